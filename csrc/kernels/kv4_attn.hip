// Decode attention over the 4-bit KV cache (kv4.h): one new query token per sequence, window + sinks.
//
// Work: one wave takes whole records (32 tokens of a kv head) for all query heads of the group, on the matrix
// cores; the visible records of a sequence are split over workgroups and the partials joined by a second
// kernel in a fixed order.
//   columns of every MFMA = (query head h, value group g of 32): B = the head's q in group g's rows, zero
//     elsewhere, so one chain of MFMAs over the head dimension gives the NG partial scores of a key apart and
//     the group scales apply to the 32-bit results;
//   scores  C[token][(h,g)] = sum_d (16 + code) q  - 24 sum_d q   (codes are fed as the bf16 16 + code: kv4.h; the
//     accumulator starts at the constant), times the key's scale, summed over g by two quad permutes;
//   the score tiles' rows are chosen (kv4.h) so that a lane's 8 scores are the 8 tokens that it supplies to the
//     PV product: P needs no exchange between lanes.  P s_v (rounded to bf16, as P itself would be) is its B
//     operand in the same (h, g) columns, and of each result only the column of the row's own group is kept;
//   O[d][(h,g)] = sum_t (16 + code) P s_v - 24 sum_t P s_v, the last sum by an MFMA with a matrix of ones so that it
//     is over the same rounded values.
// Statistics: running maximum per head with a deferred rescale (moves when a score exceeds it by 2^8), sums in
// 32 bits.
#include "kv4.h"

using namespace ftc;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
constexpr float LOG2E = 1.4426950408889634f;

struct Dec4Args {
  const uint16_t* q;
  const uint8_t* data;
  const int* lens;
  uint16_t* out;
  float* opart;  // [B*H, nsplit, D] unnormalised partial outputs
  float* ml;     // [B*H, nsplit, 2] their maximum (log2 domain) and sum
  long long q_rs, o_rs;
  int B, H, KV, tiles, max_len, window, sinks, nsplit;
  float c;  // scale * log2(e)
};

// The visible records of a sequence: sink records [0, ts), then [tl, te); split evenly into parts of `per`
// records (a multiple of the 4 waves).
struct Span {
  int len, lo, ts, tl, n, per;
};
DEV_INLINE Span span_of(const Dec4Args& a, int b) {
  Span s;
  s.len = min(a.lens[b], a.max_len);
  s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
  s.tl = s.lo / KV4_TILE;
  s.ts = min((min(a.sinks, s.lo) + KV4_TILE - 1) / KV4_TILE, s.tl);
  s.n = s.len > 0 ? s.ts + (s.len + KV4_TILE - 1) / KV4_TILE - s.tl : 0;
  s.per = ((s.n + a.nsplit - 1) / a.nsplit + 3) / 4 * 4;
  return s;
}

DEV_INLINE float dpp_xor1(float v) {  // + the neighbouring lane's (quad_perm 1,0,3,2)
  return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xf, 0xf, true));
}
DEV_INLINE float dpp_xor2(float v) {  // quad_perm 2,3,0,1
  return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xf, 0xf, true));
}
DEV_INLINE float max_q(float v) {  // over the lanes of a column (q = 0..3)
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
DEV_INLINE float sum_q(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// nibble pair i of a word as two bf16 16 + code
template <int I>
DEV_INLINE uint32_t pair16(uint32_t w) {
  const uint32_t x = I == 0 ? w << 3 : w >> (4 * I - 3);
  return (x & 0x00780078u) | 0x41804180u;
}
DEV_INLINE bf16x8 frag(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(bf16x8, make_uint4(a, b, c, d));
}

template <int D>
struct Rec {
  uint4 k[Kv4<D>::CH], v[Kv4<D>::CH], ks, vs;
};
template <int D>
DEV_INLINE void load_rec(Rec<D>& t, const uint8_t* rec, int lane, int so) {
  using L = Kv4<D>;
#pragma unroll
  for (int c = 0; c < L::CH; ++c) t.k[c] = *reinterpret_cast<const uint4*>(rec + L::KC + c * 1024 + lane * 16);
  t.ks = *reinterpret_cast<const uint4*>(rec + L::KS + so);
#pragma unroll
  for (int c = 0; c < L::CH; ++c) t.v[c] = *reinterpret_cast<const uint4*>(rec + L::VC + c * 1024 + lane * 16);
  t.vs = *reinterpret_cast<const uint4*>(rec + L::VS + so);
}

// CS sets of 16 columns: HPS = 16 / NG query heads each (4 at D = 128, 8 at D = 64)
template <int D, int CS>
__global__ __launch_bounds__(256) void kv4_decode_kernel(Dec4Args a) {
  using L = Kv4<D>;
  constexpr int NG = L::NG, NJ = L::NJ, HPS = 16 / NG;
  __shared__ float red_m[4][CS][16], red_l[4][CS][16];
  __shared__ float red_o[4][CS][HPS][D];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, q = lane >> 4, g = col % NG, hc = col / NG;
  const int G = a.H / a.KV, nhs = (G + HPS * CS - 1) / (HPS * CS);
  const int split = blockIdx.x % a.nsplit, item = blockIdx.x / a.nsplit;
  const int hs = item % nhs, kvh = item / nhs % a.KV, b = item / nhs / a.KV;
  const int h0 = kvh * G + hs * HPS * CS, hn = min(HPS * CS, G - hs * HPS * CS);  // heads of this workgroup
  const Span sp = span_of(a, b);
  const int v0 = split * sp.per, v1 = min(sp.n, v0 + sp.per);
  if (v0 >= v1) return;  // the join skips this part too

  // q of column (h, g): values 32 g + 8 q + 0..7 of its head; zero in the other groups' MFMA steps
  bf16x8 qf[CS][NG];
  float bias[CS];
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    const int h = s * HPS + hc;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (h < hn) u = *reinterpret_cast<const uint4*>(a.q + (long long)b * a.q_rs + (long long)(h0 + h) * D + 32 * g + 8 * q);
    float f[8], t = 0.f;
    unpack8(u, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) t += f[e];
    bias[s] = -24.0f * sum_q(t);
#pragma unroll
    for (int j = 0; j < NG; ++j) qf[s][j] = __builtin_bit_cast(bf16x8, j == g ? u : make_uint4(0, 0, 0, 0));
  }
  const bf16x8 ones = frag(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);

  f32x4 acc[CS][NJ], accs[CS];
  float m[CS], l[CS];
#pragma unroll
  for (int s = 0; s < CS; ++s) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[s][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    accs[s] = (f32x4){0.f, 0.f, 0.f, 0.f};
    m[s] = -INFINITY;
    l[s] = 0.f;
  }
  const uint8_t* base = a.data + ((long long)b * a.KV + kvh) * a.tiles * L::REC;
  const int so = (q * NG + g) * 16;
  auto tile_of = [&](int v) { return v < sp.ts ? v : v - sp.ts + sp.tl; };

  Rec<D> cur, nxt;
  int v = v0 + wave;
  if (v < v1) load_rec<D>(cur, base + (long long)tile_of(v) * L::REC, lane, so);
  for (; v < v1; v += 4) {
    const int tile = tile_of(v);
    if (v + 4 < v1) load_rec<D>(nxt, base + (long long)tile_of(v + 4) * L::REC, lane, so);
    float ks[8], vs[8];
    unpack8(cur.ks, ks);
    unpack8(cur.vs, vs);
    // tokens outside the length, or before the window and past the sinks: no weight, whatever their bytes hold
    const int t0 = tile * KV4_TILE;
    const bool edge = t0 + KV4_TILE > sp.len || (t0 < sp.lo && t0 + KV4_TILE > min(a.sinks, sp.lo));
    bool ok[8];
    if (edge) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + 8 * q + i;
        ok[i] = t < sp.len && (t >= sp.lo || t < a.sinks);
        vs[i] = ok[i] ? vs[i] : 0.f;
      }
    }
    bf16x8 pf[CS];
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      f32x4 c[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        c[half] = (f32x4){bias[s], bias[s], bias[s], bias[s]};
        uint32_t w[NG];
        if constexpr (D == 128) {
          w[0] = cur.k[half].x; w[1] = cur.k[half].y; w[2] = cur.k[half].z; w[3] = cur.k[half].w;
        } else {
          w[0] = half ? cur.k[0].z : cur.k[0].x;
          w[1] = half ? cur.k[0].w : cur.k[0].y;
        }
#pragma unroll
        for (int j = 0; j < NG; ++j)
          c[half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(pair16<0>(w[j]), pair16<1>(w[j]), pair16<2>(w[j]), pair16<3>(w[j])),
                                                            qf[s][j], c[half], 0, 0, 0);
      }
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = dpp_xor1(c[i >> 2][i & 3] * ks[i]);
        if constexpr (NG == 4) x[i] = dpp_xor2(x[i]);
        x[i] *= a.c;
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ok[i] ? x[i] : -INFINITY;
      }
      float mt = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      if (__builtin_amdgcn_ballot_w64(mt > m[s] + 8.0f) != 0) {
        const float mn = fmaxf(m[s], max_q(mt));
        const float al = __builtin_amdgcn_exp2f(m[s] - (mn == -INFINITY ? 0.f : mn));
        m[s] = mn;
        l[s] *= al;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[s][j][i] *= al;
#pragma unroll
        for (int i = 0; i < 4; ++i) accs[s][i] *= al;
      }
      const float mref = m[s] == -INFINITY ? 0.f : m[s];
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(x[i] - mref);
        l[s] += p[i];
        p[i] *= vs[i];
      }
      pf[s] = frag(pack_bf2(p[0], p[1]), pack_bf2(p[2], p[3]), pack_bf2(p[4], p[5]), pack_bf2(p[6], p[7]));
      accs[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[s], accs[s], 0, 0, 0);
    }
#pragma unroll
    for (int c = 0; c < L::CH; ++c) {
      const uint4 w = cur.v[c];
      const bf16x8 vf[4] = {frag(pair16<0>(w.x), pair16<0>(w.y), pair16<0>(w.z), pair16<0>(w.w)),
                            frag(pair16<1>(w.x), pair16<1>(w.y), pair16<1>(w.z), pair16<1>(w.w)),
                            frag(pair16<2>(w.x), pair16<2>(w.y), pair16<2>(w.z), pair16<2>(w.w)),
                            frag(pair16<3>(w.x), pair16<3>(w.y), pair16<3>(w.z), pair16<3>(w.w))};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int s = 0; s < CS; ++s)
          acc[s][4 * c + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[i], pf[s], acc[s][4 * c + i], 0, 0, 0);
    }
    cur = nxt;
  }

  // ---- join the four waves: common maximum per column, then the sums
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    l[s] = sum_q(l[s]);
    if (q == 0) red_m[wave][s][col] = m[s];
  }
  __syncthreads();
  const bool mine = g == (NG == 4 ? q : q >> 1);  // this lane's rows (d) are in its column's group
  float M[CS];
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    M[s] = fmaxf(fmaxf(red_m[0][s][col], red_m[1][s][col]), fmaxf(red_m[2][s][col], red_m[3][s][col]));
    const float al = __builtin_amdgcn_exp2f(m[s] - (M[s] == -INFINITY ? 0.f : M[s]));
    if (q == 0) red_l[wave][s][col] = l[s] * al;
    if (mine) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) red_o[wave][s][hc][NJ * (4 * q + i) + j] = (acc[s][j][i] - 24.0f * accs[s][i]) * al;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < hn * D; e += 256) {
    const int h = e / D, d = e % D, s = h / HPS, c = (h % HPS);
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) o += red_o[w][s][c][d];
    const long long row = ((long long)b * a.H + h0 + h) * a.nsplit + split;
    a.opart[row * D + d] = o;
    if (d == 0) {
      a.ml[row * 2] = fmaxf(fmaxf(red_m[0][s][c * NG], red_m[1][s][c * NG]), fmaxf(red_m[2][s][c * NG], red_m[3][s][c * NG]));
      a.ml[row * 2 + 1] = red_l[0][s][c * NG] + red_l[1][s][c * NG] + red_l[2][s][c * NG] + red_l[3][s][c * NG];
    }
  }
}

// Partials of a (sequence, head) joined in split order.
template <int D>
__global__ __launch_bounds__(D) void kv4_join_kernel(Dec4Args a) {
  const int bh = blockIdx.x, d = threadIdx.x;
  const Span sp = span_of(a, bh / a.H);
  const int parts = sp.n > 0 ? (sp.n + sp.per - 1) / sp.per : 0;
  const long long base = (long long)bh * a.nsplit;
  float M = -INFINITY;
  for (int s = 0; s < parts; ++s) M = fmaxf(M, a.ml[(base + s) * 2]);
  float l = 0.f, o = 0.f;
  for (int s = 0; s < parts; ++s) {
    const float w = __builtin_amdgcn_exp2f(a.ml[(base + s) * 2] - (M == -INFINITY ? 0.f : M));
    l += w * a.ml[(base + s) * 2 + 1];
    o += w * a.opart[(base + s) * D + d];
  }
  a.out[(long long)(bh / a.H) * a.o_rs + (long long)(bh % a.H) * D + d] = f2bf(parts > 0 ? o / l : 0.f);
}

// column sets a workgroup takes: enough for the group's query heads, at most 4 (16 heads at D = 128)
int kv4_sets(int D, int G) {
  const int hps = D == 128 ? 4 : 8, need = (G + hps - 1) / hps;
  return need >= 3 ? 4 : need;
}
// parts a sequence is split into: ~1024 workgroups (16 waves a CU), each wave at least one record
int kv4_nsplit(int B, int H, int KV, int D, int max_len, int window, int sinks) {
  const int G = H / KV, cs = kv4_sets(D, G), hps = D == 128 ? 4 : 8;
  const long long items = (long long)B * KV * ((G + hps * cs - 1) / (hps * cs));
  long long vis = (max_len + KV4_TILE - 1) / KV4_TILE;
  if (window > 0) {
    const long long w = ((long long)sinks + KV4_TILE - 1) / KV4_TILE + ((long long)window + KV4_TILE - 1) / KV4_TILE + 1;
    vis = w < vis ? w : vis;
  }
  long long n = (1024 + items - 1) / items;
  const long long most = (vis + 3) / 4;
  return (int)(n < most ? n : most);
}

}  // namespace

extern "C" int ftc_kv4_store(void* data, const void* k, const void* v, const int* start, const int* count, int B, int KV,
                             int D, int n, int tiles, long long k_bs, long long k_rs, long long v_bs, long long v_rs,
                             int bias, int limit, hipStream_t stream);

extern "C" long long ftc_kv4_decode_workspace_floats(int B, int H, int KV, int D, int max_len, int window, int sinks) {
  return (long long)B * H * kv4_nsplit(B, H, KV, D, max_len, window, sinks) * (D + 2);
}

extern "C" int ftc_kv4_decode(const void* qkv, void* data, const int* lens, void* out, float* workspace, int B, int H,
                              int KV, int D, int tiles, int max_len, long long q_rs, long long o_rs, float scale, int window,
                              int sinks, hipStream_t stream) {
  if ((D != 64 && D != 128) || B < 1 || KV < 1 || H < KV || H % KV || max_len < 1 || max_len > (long long)tiles * KV4_TILE)
    return -1;
  const int nsplit = kv4_nsplit(B, H, KV, D, max_len, window, sinks), G = H / KV, cs = kv4_sets(D, G), hps = D == 128 ? 4 : 8;
  const long long blocks = (long long)B * KV * ((G + hps * cs - 1) / (hps * cs)) * nsplit;
  if (blocks > 0x7fffffffLL || (long long)B * H > 0x7fffffffLL) return -1;
  const uint16_t* qp = (const uint16_t*)qkv;
  // the new token's row: position lens - 1
  const int rc = ftc_kv4_store(data, qp + (long long)H * D, qp + (long long)(H + KV) * D, lens, nullptr, B, KV, D, 1,
                               tiles, q_rs, 0, q_rs, 0, -1, max_len, stream);
  if (rc) return rc;
  Dec4Args a{qp, (const uint8_t*)data, lens, (uint16_t*)out, workspace, workspace + (long long)B * H * nsplit * D, q_rs, o_rs,
             B, H, KV, tiles, max_len, window, sinks, nsplit, scale * LOG2E};
  const dim3 grid((unsigned)blocks), join((unsigned)(B * H));
#define KV4_LAUNCH(DD, CC) hipLaunchKernelGGL((kv4_decode_kernel<DD, CC>), grid, dim3(256), 0, stream, a)
  if (D == 128) {
    if (cs == 1) KV4_LAUNCH(128, 1); else if (cs == 2) KV4_LAUNCH(128, 2); else KV4_LAUNCH(128, 4);
    hipLaunchKernelGGL(kv4_join_kernel<128>, join, dim3(128), 0, stream, a);
  } else {
    if (cs == 1) KV4_LAUNCH(64, 1); else if (cs == 2) KV4_LAUNCH(64, 2); else KV4_LAUNCH(64, 4);
    hipLaunchKernelGGL(kv4_join_kernel<64>, join, dim3(64), 0, stream, a);
  }
#undef KV4_LAUNCH
  return (int)hipGetLastError();
}
