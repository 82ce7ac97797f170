// Decode attention over the 4-bit KV cache (kv4.h): one new query token per sequence, window + sinks.
//
// Work: one wave takes whole records (32 tokens of a kv head) for all query heads of the group, on the matrix
// cores; the visible records of a sequence are split over workgroups and the partials joined by a second
// kernel in a fixed order.
//   columns of every MFMA = HPS query heads h x NGC = 16 / HPS value groups (of 32 d); NCH = NG / NGC chains take the
//     groups NGC at a time.  B = the head's q in its column's group's rows, zero elsewhere, so a chain of MFMAs gives the
//     partial scores of its groups apart and the group scales apply to the 32-bit results;
//   scores  C[token][(h,g)] = sum_d (16 + code) q  - 24 sum_d q   (codes are fed as the bf16 16 + code: kv4.h; the
//     accumulator starts at the constant), times the key's scale, summed over chains and, by quad permutes, columns;
//   the score tiles' rows are chosen (kv4.h) so that a lane's 8 scores are the 8 tokens that it supplies to the
//     PV product: P needs no exchange between lanes.  P s_v (rounded to bf16, as P itself would be) is its B
//     operand in the same columns, one for each chain; of a result the columns of the row's own group are kept;
//   O[d][(h,g)] = sum_t (16 + code) P s_v - 24 sum_t P s_v, the last sum by an MFMA with a matrix of ones so that it
//     is over the same rounded values.
// HPS is the smallest that holds the group's query heads (4, 8 or 16 at D = 128; 8 or 16 at 64; larger groups take
// several workgroups): with the columns of 4 heads for every group size, 8 heads took two column sets, 210 registers
// (2 waves per SIMD) and twice the softmax: 137 us at 64 x 8192 tokens, 64 / 8 heads x 128, instead of 110 (4.4 TB/s).
// Statistics: running maximum per head with a deferred rescale (moves when a score exceeds it by 2^8), sums in
// 32 bits.
// Bound: HBM, 4.5 bits of each visible value -- 64 x 16384 tokens, 32 / 8 heads x 128: 193 us, 5.3 TB/s (MFMA busy 0.13,
// VALU 0.16); 32 x 4096: 26.5 us; below some 10 MB of cache, latency (one sequence of 2000 tokens: 6.7 us + 3.5 of the join).
#include "kv4.h"

using namespace ftc;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
constexpr float LOG2E = 1.4426950408889634f;

struct Dec4Args {
  const uint16_t* q;
  const uint16_t *knew, *vnew;  // the current tokens' rows (row stride q_rs)
  uint8_t* data;
  const int* lens;
  uint16_t* out;
  float* opart;  // [B*H, nsplit, D] unnormalised partial outputs
  float* ml;     // [B*H, nsplit, 2] their maximum (log2 domain) and sum
  long long q_rs, o_rs;
  int B, H, KV, tiles, max_len, window, sinks, nsplit;
  float c;  // scale * log2(e)
};

// The visible records of a sequence: sink records [0, ts), then [tl, te); split evenly into parts of `per`
// records (a multiple of the workgroup's NW waves).
struct Span {
  int len, lo, ts, tl, n, per;
  bool append;  // the current token is written (a length within max_len)
};
template <int NW>
DEV_INLINE Span span_of(const Dec4Args& a, int b) {
  Span s;
  const int len = a.lens[b];
  s.append = len > 0 && len <= a.max_len;
  s.len = min(len, a.max_len);
  s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
  s.tl = s.lo / KV4_TILE;
  s.ts = min((min(a.sinks, s.lo) + KV4_TILE - 1) / KV4_TILE, s.tl);
  s.n = s.len > 0 ? s.ts + (s.len + KV4_TILE - 1) / KV4_TILE - s.tl : 0;
  s.per = ((s.n + a.nsplit - 1) / a.nsplit + NW - 1) / NW * NW;
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

// One record as a lane holds it: its chunks, and the scales of its column's group of every chain (so: the first's offset)
template <int D, int NCH>
struct Rec {
  uint4 k[Kv4<D>::CH], v[Kv4<D>::CH], ks[NCH], vs[NCH];
};
template <int D, int NCH>
DEV_INLINE void load_k(Rec<D, NCH>& t, const uint8_t* rec, int lane, int so) {
  using L = Kv4<D>;
#pragma unroll
  for (int c = 0; c < L::CH; ++c) t.k[c] = *reinterpret_cast<const uint4*>(rec + L::KC + c * 1024 + lane * 16);
#pragma unroll
  for (int c = 0; c < NCH; ++c) t.ks[c] = *reinterpret_cast<const uint4*>(rec + L::KS + so + c * (L::NG / NCH) * 16);
}
template <int D, int NCH>
DEV_INLINE void load_v(Rec<D, NCH>& t, const uint8_t* rec, int lane, int so) {
  using L = Kv4<D>;
#pragma unroll
  for (int c = 0; c < L::CH; ++c) t.v[c] = *reinterpret_cast<const uint4*>(rec + L::VC + c * 1024 + lane * 16);
#pragma unroll
  for (int c = 0; c < NCH; ++c) t.vs[c] = *reinterpret_cast<const uint4*>(rec + L::VS + so + c * (L::NG / NCH) * 16);
}

// The current token's codes put into the registers of the wave that read its record (token t of 32): the lanes
// that hold its chunks take them from the lanes that quantised it, so nothing waits for the store.
template <int D, int NCH>
DEV_INLINE void patch_rec(Rec<D, NCH>& x, int t, const Kv4Token& n, int lane) {
  using L = Kv4<D>;
  constexpr int NGC = L::NG / NCH;
  const int r = lane & 15, q = lane >> 4, g = r % NGC;
  uint32_t w[L::NG], v[L::CH], ks[NCH], vs[NCH];
#pragma unroll
  for (int j = 0; j < L::NG; ++j) w[j] = __shfl(n.code, 8 * j + 2 * q, 64);
#pragma unroll
  for (int c = 0; c < L::CH; ++c) v[c] = __shfl(n.code, 32 + 16 * c + r, 64);
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    ks[c] = __shfl(n.scale, 8 * (c * NGC + g), 64);
    vs[c] = __shfl(n.scale, 32 + 8 * (c * NGC + g), 64);
  }
  const int half = (t >> 2) & 1;
  if (r == 4 * (t >> 3) + (t & 3)) {
    if constexpr (D == 128) {
      if (half) x.k[1] = make_uint4(w[0], w[1], w[2], w[3]);
      else x.k[0] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      if (half) { x.k[0].z = w[0]; x.k[0].w = w[1]; }
      else { x.k[0].x = w[0]; x.k[0].y = w[1]; }
    }
  }
  if (q == t >> 3) {
    const int p = (t & 7) >> 1, sh = 16 * (t & 1);
    auto put = [&](uint4& u, uint32_t y) __attribute__((always_inline)) {
      const uint32_t m = 0xffffu << sh, z = y << sh;
      u.x = p == 0 ? (u.x & ~m) | z : u.x;
      u.y = p == 1 ? (u.y & ~m) | z : u.y;
      u.z = p == 2 ? (u.z & ~m) | z : u.z;
      u.w = p == 3 ? (u.w & ~m) | z : u.w;
    };
#pragma unroll
    for (int c = 0; c < L::CH; ++c) put(x.v[c], v[c]);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      put(x.ks[c], ks[c]);
      put(x.vs[c], vs[c]);
    }
  }
}

template <int D, int HPS, int NW>
__global__ __launch_bounds__(64 * NW) void kv4_decode_kernel(Dec4Args a) {
  using L = Kv4<D>;
  constexpr int NG = L::NG, NGC = 16 / HPS, NCH = NG / NGC;
  constexpr int NP = NGC == 1 ? 2 : 1;  // PV products a chunk of 64 d: its two groups are in one chain, or in two
  static_assert(NGC <= NG && NGC * NCH == NG, "columns");
  __shared__ float red_m[NW][16], red_l[NW][16];
  __shared__ float red_o[NW][HPS][D];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, q = lane >> 4, g = col % NGC, hc = col / NGC;
  const int G = a.H / a.KV, nhs = (G + HPS - 1) / HPS;
  const int split = blockIdx.x % a.nsplit, item = blockIdx.x / a.nsplit;
  const int hs = item % nhs, kvh = item / nhs % a.KV, b = item / nhs / a.KV;
  const int h0 = kvh * G + hs * HPS, hn = min(HPS, G - hs * HPS);  // heads of this workgroup
  const Span sp = span_of<NW>(a, b);
  const int v0 = split * sp.per, v1 = min(sp.n, v0 + sp.per);
  if (v0 >= v1) {  // the join skips this part too
    if (a.nsplit == 1) {  // an empty sequence
      for (int e = threadIdx.x; e < hn * D; e += 64 * NW) a.out[(long long)b * a.o_rs + (long long)h0 * D + e] = 0;
    }
    return;
  }

  // q of column (h, g): in chain c values 32 (c NGC + g) + 8 q + 0..7 of its head; zero in the other groups' MFMA steps
  bf16x8 qf[NG];
  float bias[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (hc < hn)
      u = *reinterpret_cast<const uint4*>(a.q + (long long)b * a.q_rs + (long long)(h0 + hc) * D + 32 * (c * NGC + g) + 8 * q);
    float f[8], t = 0.f;
    unpack8(u, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) t += f[e];
    bias[c] = -24.0f * sum_q(t);
#pragma unroll
    for (int j = 0; j < NGC; ++j) qf[c * NGC + j] = __builtin_bit_cast(bf16x8, j == g ? u : make_uint4(0, 0, 0, 0));
  }
  const bf16x8 ones = frag(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);

  f32x4 acc[NP][L::CH][4], accs[NCH];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int c = 0; c < L::CH; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[p][c][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < NCH; ++c) accs[c] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  uint8_t* base = a.data + ((long long)b * a.KV + kvh) * a.tiles * L::REC;
  const int so = (q * NG + g) * 16;
  auto tile_of = [&](int v) { return v < sp.ts ? v : v - sp.ts + sp.tl; };

  // One record in registers; its K is loaded again for the next record as soon as it is used up, its V likewise.
  // The loads are unconditional (the last record is read once more): under a condition the compiler sinks them to
  // their use, which cost 294 instead of 193 us at 64 x 16384 tokens (32 / 8 heads x 128); two records in
  // registers spill their way to 594.
  Rec<D, NCH> cur;
  {
    const uint8_t* rec = base + (long long)tile_of(min(v0 + wave, v1 - 1)) * L::REC;
    load_k(cur, rec, lane, so);
    load_v(cur, rec, lane, so);
  }
  // the wave of the last record quantises the current token, writes it and keeps its codes for that record
  const bool last = sp.append && v1 == sp.n && (sp.n - 1 - v0) % NW == wave;
  const int tok = (sp.len - 1) % KV4_TILE;
  Kv4Token fresh;
  if (last) {
    const int d = (4 * (lane & 31)) % D;
    fresh = kv4_token(*reinterpret_cast<const uint2*>((lane < 32 ? a.knew : a.vnew) + (long long)b * a.q_rs + (long long)kvh * D + d), lane);
    if (hs == 0) kv4_put_token<D>(base + (long long)((sp.len - 1) / KV4_TILE) * L::REC, tok, fresh, lane);
  }
  auto record = [&](int v, bool more) __attribute__((always_inline)) {
    const int t0 = tile_of(v) * KV4_TILE;
    const uint8_t* next = base + (long long)tile_of(min(v + NW, v1 - 1)) * L::REC;
    f32x4 c[NCH][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) c[ch][half] = (f32x4){bias[ch], bias[ch], bias[ch], bias[ch]};
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        uint32_t w;
        if constexpr (D == 128)
          w = j == 0 ? cur.k[half].x : j == 1 ? cur.k[half].y : j == 2 ? cur.k[half].z : cur.k[half].w;
        else
          w = half ? (j ? cur.k[0].w : cur.k[0].z) : (j ? cur.k[0].y : cur.k[0].x);
        c[j / NGC][half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            frag(pair16<0>(w), pair16<1>(w), pair16<2>(w), pair16<3>(w)), qf[j], c[j / NGC][half], 0, 0, 0);
      }
    }
    float x[8];
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      float ks[8];
      unpack8(cur.ks[ch], ks);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = ch ? x[i] + c[ch][i >> 2][i & 3] * ks[i] : c[ch][i >> 2][i & 3] * ks[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (NGC >= 2) x[i] = dpp_xor1(x[i]);
      if constexpr (NGC == 4) x[i] = dpp_xor2(x[i]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_k(cur, next, lane, so);
    __builtin_amdgcn_sched_barrier(0);
    // tokens outside the length, or before the window and past the sinks: no weight, whatever their bytes hold
    const bool edge = t0 + KV4_TILE > sp.len || (t0 < sp.lo && t0 + KV4_TILE > min(a.sinks, sp.lo));
    uint32_t hidden = 0;  // tokens without weight, one bit each
    if (edge) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + 8 * q + i;
        const bool ok = t < sp.len && (t >= sp.lo || t < a.sinks);
        hidden |= ok ? 0u : 1u << i;
        x[i] = ok ? x[i] : -INFINITY;
      }
    }
    // c > 0: the maximum commutes with the scale
    const float mt = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * a.c;
    if (__builtin_amdgcn_ballot_w64(mt > m + 8.0f) != 0) {
      const float mn = fmaxf(m, max_q(mt));
      const float al = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= al;
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int ch = 0; ch < L::CH; ++ch)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[p][ch][i][e] *= al;
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
        for (int e = 0; e < 4; ++e) accs[ch][e] *= al;
    }
    const float mref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], a.c, -mref));
      l += x[i];
    }
    bf16x8 pf[NCH];
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      float vs[8];
      unpack8(cur.vs[ch], vs);
      if (edge) {
#pragma unroll
        for (int i = 0; i < 8; ++i) vs[i] = (hidden >> i) & 1 ? 0.f : vs[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) vs[i] *= x[i];
      pf[ch] = frag(pack_bf2(vs[0], vs[1]), pack_bf2(vs[2], vs[3]), pack_bf2(vs[4], vs[5]), pack_bf2(vs[6], vs[7]));
      accs[ch] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[ch], accs[ch], 0, 0, 0);
    }
#pragma unroll
    for (int ch = 0; ch < L::CH; ++ch) {
      const uint4 w = cur.v[ch];
      auto pv = [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < NP; ++p)  // the chain of group 2 ch + p
          acc[p][ch][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(a0, a1, a2, a3), pf[(2 * ch + p) / NGC], acc[p][ch][i], 0, 0, 0);
      };
      pv(0, pair16<0>(w.x), pair16<0>(w.y), pair16<0>(w.z), pair16<0>(w.w));
      pv(1, pair16<1>(w.x), pair16<1>(w.y), pair16<1>(w.z), pair16<1>(w.w));
      pv(2, pair16<2>(w.x), pair16<2>(w.y), pair16<2>(w.z), pair16<2>(w.w));
      pv(3, pair16<3>(w.x), pair16<3>(w.y), pair16<3>(w.z), pair16<3>(w.w));
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_v(cur, next, lane, so);
  };
  // the current token's record is peeled off: patching it inside the loop makes every record's loads wait
  int v = v0 + wave;
  for (const int ve = last ? v1 - 1 : v1; v < ve; v += NW) record(v, true);
  if (last) {
    patch_rec(cur, tok, fresh, lane);
    record(v, false);
  }

  // ---- join the waves: common maximum per column, then the sums in wave order
  l = sum_q(l);
  if (q == 0) red_m[wave][col] = m;
  __syncthreads();
  {
    float M = red_m[0][col];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, red_m[w][col]);
    const float al = __builtin_amdgcn_exp2f(m - (M == -INFINITY ? 0.f : M));
    if (q == 0) red_l[wave][col] = l * al;
#pragma unroll
    for (int ch = 0; ch < L::CH; ++ch) {
      // this lane's rows r = 4 q + 0..3 are values of group 2 ch + (q >> 1): kept in that group's column
      const bool mine = NGC == 1 || g == (2 * ch + (q >> 1)) % NGC;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[i] = (acc[0][ch][i][e] - 24.0f * accs[2 * ch / NGC][e]) * al;
          if constexpr (NP == 2) o[i] = q >> 1 ? (acc[1][ch][i][e] - 24.0f * accs[2 * ch + 1][e]) * al : o[i];
        }
        if (mine)
          *reinterpret_cast<float4*>(&red_o[wave][hc][64 * ch + 4 * (4 * q + e)]) = make_float4(o[0], o[1], o[2], o[3]);
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < hn * D; e += 64 * NW) {
    const int h = e / D, d = e % D, c = h * NGC;
    float o = 0.f, lt = 0.f, M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      o += red_o[w][h][d];
      lt += red_l[w][c];
      M = fmaxf(M, red_m[w][c]);
    }
    if (a.nsplit == 1) {
      a.out[(long long)b * a.o_rs + (long long)(h0 + h) * D + d] = f2bf(o / lt);
    } else {
      const long long row = ((long long)b * a.H + h0 + h) * a.nsplit + split;
      a.opart[row * D + d] = o;
      if (d == 0) {
        a.ml[row * 2] = M;
        a.ml[row * 2 + 1] = lt;
      }
    }
  }
}

// Partials of a (sequence, head) joined: 256 threads = 256 / D groups of parts side by side, summed in a fixed
// order.
template <int D, int NW>
__global__ __launch_bounds__(256) void kv4_join_kernel(Dec4Args a) {
  constexpr int PG = 256 / D;
  __shared__ float ol[PG][D], ll[PG];
  const int bh = blockIdx.x, d = threadIdx.x % D, pg = threadIdx.x / D;
  const Span sp = span_of<NW>(a, bh / a.H);
  const int parts = sp.n > 0 ? (sp.n + sp.per - 1) / sp.per : 0;
  const float* ml = a.ml + (long long)bh * a.nsplit * 2;
  const float* op = a.opart + (long long)bh * a.nsplit * D + d;
  float M = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < parts; ++s) M = fmaxf(M, ml[2 * s]);
  if (M == -INFINITY) M = 0.f;
  float l = 0.f, o = 0.f;
#pragma unroll 8
  for (int s = pg; s < parts; s += PG) {
    const float w = __builtin_amdgcn_exp2f(ml[2 * s] - M);
    l += w * ml[2 * s + 1];
    o += w * op[(long long)s * D];
  }
  ol[pg][d] = o;
  if (d == 0) ll[pg] = l;
  __syncthreads();
  if (pg == 0) {
#pragma unroll
    for (int i = 1; i < PG; ++i) {
      o += ol[i][d];
      l += ll[i];
    }
    a.out[(long long)(bh / a.H) * a.o_rs + (long long)(bh % a.H) * D + d] = f2bf(parts > 0 ? o / l : 0.f);
  }
}

struct Plan {
  int hps, nhs, nw, nsplit;
};
Plan kv4_plan(int B, int H, int KV, int D, int max_len, int window, int sinks) {
  Plan p;
  const int G = H / KV;
  p.hps = G <= 4 && D == 128 ? 4 : G <= 8 ? 8 : 16;
  p.nhs = (G + p.hps - 1) / p.hps;
  const long long items = (long long)B * KV * p.nhs;
  long long vis = (max_len + KV4_TILE - 1) / KV4_TILE;
  if (window > 0) {
    const long long w = ((long long)sinks + KV4_TILE - 1) / KV4_TILE + ((long long)window + KV4_TILE - 1) / KV4_TILE + 1;
    vis = w < vis ? w : vis;
  }
  // 8 waves share an item's records (one workgroup a CU), 4 where there are many short items (64 sequences of 300
  // tokens, 512 items: 8.9 us with 4 waves, 11.5 with 8).
  p.nw = items > 256 && vis < 32 ? 4 : 8;
  // Parts: the number that a model of the launch finds quickest -- rounds of 256 workgroups, 1.8 us a record and
  // wave plus 2.5 us a workgroup, and 3 us for the join.  The 1.8 us are a record's latency: a wave takes 1.5 to 1.8
  // whether 8 CUs are busy or all (192 us for 128 records a wave on 8); with all of them busy that is 5.2 TB/s as well.  Measured against every
  // split from 1 to 128: it picks the quickest or one within 4 % (one 32768-token sequence, 8 items: 32 parts
  // 15.0 us, 24 parts 16.4, unsplit 192; 16 sequences at a 4096 window: 2 parts 18.9, 1 part 30.9; 32 x 4096
  // tokens: unsplit 25.3, 2 parts 30.0).
  const long long most = (vis + p.nw - 1) / p.nw;
  auto model = [&](long long n) {
    const long long rounds = (items * n + 255) / 256, per = ((vis + n - 1) / n + p.nw - 1) / p.nw;
    return rounds * (per * 1.8f + 2.5f) + (n > 1 ? 3.f : 0.f);
  };
  p.nsplit = 1;
  float best = model(1);
  for (int r = 1; r <= 8; ++r) {  // the most parts that r rounds hold
    const long long full = 256LL * r / items, n = full < most ? full : most;
    if (n > 1 && n <= 256 && model(n) < best) {
      best = model(n);
      p.nsplit = (int)n;
    }
  }
  return p;
}

template <int D, int HPS, int NW>
void launch(const Dec4Args& a, const Plan& p, hipStream_t stream) {
  hipLaunchKernelGGL((kv4_decode_kernel<D, HPS, NW>), dim3((unsigned)((long long)a.B * a.KV * p.nhs * p.nsplit)), dim3(64 * NW),
                     0, stream, a);
  if (p.nsplit > 1)
    hipLaunchKernelGGL((kv4_join_kernel<D, NW>), dim3((unsigned)(a.B * a.H)), dim3(256), 0, stream, a);
}
template <int D>
void launch_d(const Dec4Args& a, const Plan& p, hipStream_t stream) {
  if constexpr (D == 128) {
    if (p.hps == 4) {
      p.nw == 8 ? launch<D, 4, 8>(a, p, stream) : launch<D, 4, 4>(a, p, stream);
      return;
    }
  }
  if (p.hps == 8)
    p.nw == 8 ? launch<D, 8, 8>(a, p, stream) : launch<D, 8, 4>(a, p, stream);
  else
    p.nw == 8 ? launch<D, 16, 8>(a, p, stream) : launch<D, 16, 4>(a, p, stream);
}

}  // namespace

extern "C" long long ftc_kv4_decode_workspace_floats(int B, int H, int KV, int D, int max_len, int window, int sinks) {
  const Plan p = kv4_plan(B, H, KV, D, max_len, window, sinks);
  return p.nsplit > 1 ? (long long)B * H * p.nsplit * (D + 2) : 0;
}

extern "C" int ftc_kv4_decode(const void* qkv, void* data, const int* lens, void* out, float* workspace, int B, int H,
                              int KV, int D, int tiles, int max_len, long long q_rs, long long o_rs, float scale, int window,
                              int sinks, hipStream_t stream) {
  if ((D != 64 && D != 128) || B < 1 || KV < 1 || H < KV || H % KV || max_len < 1 || max_len > (long long)tiles * KV4_TILE)
    return -1;
  const Plan p = kv4_plan(B, H, KV, D, max_len, window, sinks);
  if ((long long)B * KV * p.nhs * p.nsplit > 0x7fffffffLL || (long long)B * H > 0x7fffffffLL) return -1;
  const uint16_t* qp = (const uint16_t*)qkv;
  Dec4Args a{qp, qp + (long long)H * D, qp + (long long)(H + KV) * D, (uint8_t*)data, lens, (uint16_t*)out, workspace,
             workspace + (long long)B * H * p.nsplit * D, q_rs, o_rs, B, H, KV, tiles, max_len, window, sinks, p.nsplit,
             scale * LOG2E};
  D == 128 ? launch_d<128>(a, p, stream) : launch_d<64>(a, p, stream);
  return (int)hipGetLastError();
}
