// Rows of K and V quantised to 4 bits as they are written into a cache, and read back (layout and
// quantisation: kv4.h).
//
// One wave = one record (32 tokens of one kv head), at D = 128 its K or its V (8192 tokens of 8 heads: written 11.3 -> 10.7
// us, read back 10.0 -> 8.9; 64 x 2048: 133.9 -> 130.4, 129.7 -> 125.8; at D = 64, where half a record is a kilobyte, as
// fast or 1 % slower).  A lane quantises exactly the 16-byte chunks that the layout gives it: for K its token's 8-value
// runs of every group (the group maximum is shared by the 4 lanes of that token), for V 8 tokens x 4 values of each 64
// (shared by 8 lanes), so nothing goes through LDS and whole records are written as linear 16-byte stores.  Records that
// are only partly covered by the call (its first and last) store token by token; other tokens' bytes stay.
// Bound: HBM -- 2 bytes read and 0.5625 written per value (and back).
#include "kv4.h"

using namespace ftc;

namespace {

struct StoreArgs {
  uint8_t* data;
  const uint16_t *k, *v;
  const int *start, *count;
  long long k_bs, k_rs, v_bs, v_rs;  // batch / row strides in elements
  int B, KV, n, tiles, span;         // span: records a sequence's rows can touch
};

// maximum of packed keys (both halves) over lanes l, l ^ 16, l ^ 32, l ^ 48: row swaps, no LDS
DEV_INLINE uint32_t key_max_q(uint32_t k) {
  const auto a = __builtin_amdgcn_permlane16_swap(k, k, false, false);
  k = kv4_max2(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(k, k, false, false);
  return kv4_max2(b[0], b[1]);
}
DEV_INLINE uint32_t key_top(uint32_t k) {
  const uint32_t a = k & 0xffffu, b = k >> 16;
  return a > b ? a : b;
}
DEV_INLINE uint32_t keys8(const uint4& u) {
  return kv4_max2(kv4_max2(kv4_keys(u.x), kv4_keys(u.y)), kv4_max2(kv4_keys(u.z), kv4_keys(u.w)));
}

template <int D>
__global__ __launch_bounds__(256) void kv4_store_kernel(StoreArgs a) {
  using L = Kv4<D>;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const unsigned item = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));  // < 2^31 (launcher)
  constexpr int W = L::WAVES;
  if (item >= (unsigned)W * a.B * a.span * a.KV) return;
  const bool keys = W == 1 || !(item & 1), values = W == 1 || (item & 1);  // what this wave takes of the record
  const int kvh = item / W % (unsigned)a.KV, bs = item / W / (unsigned)a.KV;
  const int sp = bs % (unsigned)a.span, b = bs / (unsigned)a.span;
  const long long start = a.start[b];
  const int n = a.count ? min(a.n, a.count[b]) : a.n;
  // first record that the rows touch inside the cache (rows before position 0 are not written)
  const long long p0 = start > 0 ? start : 0;
  const long long tile = p0 / KV4_TILE + sp;
  if (tile >= a.tiles) return;
  const long long row0 = tile * KV4_TILE - start;  // row index of the record's token 0
  if (n < 1 || row0 >= n || row0 + KV4_TILE <= 0) return;
  const bool whole = row0 >= 0 && row0 + KV4_TILE <= n;
  uint8_t* rec = a.data + (((long long)b * a.KV + kvh) * a.tiles + tile) * L::REC;
  const uint16_t* kp = a.k + b * a.k_bs + (long long)kvh * D;
  const uint16_t* vp = a.v + b * a.v_bs + (long long)kvh * D;
  auto valid = [&](int t) { return row0 + t >= 0 && row0 + t < n; };

  // every load of the record first: under per-row conditions and loops the compiler waits for each (rows that are not
  // written are read as a row that is)
  auto row_of = [&](int t) { return min(max(row0 + t, 0LL), (long long)n - 1); };
  uint4 ku[2][L::NG];
  uint2 vu[8][L::CH];
  if (keys) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint16_t* p = kp + row_of(8 * (r >> 2) + 4 * half + (r & 3)) * a.k_rs + 8 * q;
#pragma unroll
      for (int j = 0; j < L::NG; ++j) ku[half][j] = *reinterpret_cast<const uint4*>(p + 32 * j);
    }
  }
  if (values) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t* p = vp + row_of(8 * q + i) * a.v_rs + 4 * r;
#pragma unroll
      for (int c = 0; c < L::CH; ++c) vu[i][c] = *reinterpret_cast<const uint2*>(p + 64 * c);
    }
  }

  // ---- K: this lane's token of each half, 8 values of every group
  if (keys) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int t = 8 * (r >> 2) + 4 * half + (r & 3);
      const bool ok = whole || valid(t);
      uint32_t w[L::NG], sc[L::NG];
#pragma unroll
      for (int j = 0; j < L::NG; ++j) {
        float rinv, f[8];
        sc[j] = kv4_scale(key_top(key_max_q(keys8(ku[half][j]))), &rinv);
        unpack8(ku[half][j], f);
        w[j] = kv4_pack_k(f, rinv);
      }
      if (ok) {
        uint32_t s = sc[0];  // lane q stores the scale of group q
#pragma unroll
        for (int j = 1; j < L::NG; ++j) s = q == j ? sc[j] : s;
        if (q < L::NG)
          *reinterpret_cast<uint16_t*>(rec + L::KS + ((r >> 2) * L::NG + q) * 16 + (4 * half + (r & 3)) * 2) = (uint16_t)s;
        if constexpr (D == 128)
          *reinterpret_cast<uint4*>(rec + L::KC + half * 1024 + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        else
          *reinterpret_cast<uint2*>(rec + L::KC + lane * 16 + half * 8) = make_uint2(w[0], w[1]);
      }
    }
  }
  if (!values) return;

  // ---- V: tokens 8 q + 0..7, 4 values of each 64 (their group's maximum over the 8 lanes that share it)
#pragma unroll
  for (int c = 0; c < L::CH; ++c) {
    uint32_t w[4], sc[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint2 u = vu[i][c];
      uint32_t key = kv4_max2(kv4_keys(u.x), kv4_keys(u.y));
      key = kv4_max2(key, kv4_dpp(key, 1));
      key = kv4_max2(key, kv4_dpp(key, 2));
      key = kv4_max2(key, kv4_dpp(key, 3));
      float rinv;
      const uint32_t s = kv4_scale(key_top(key), &rinv);
      const float f[4] = {bf_lo(u.x), bf_hi(u.x), bf_lo(u.y), bf_hi(u.y)};
      const uint32_t n = kv4_pack_v(f, rinv);
      if (i & 1) {
        w[i >> 1] |= n << 16;
        sc[i >> 1] |= s << 16;
      } else {
        w[i >> 1] = n;
        sc[i >> 1] = s;
      }
    }
    uint8_t* wp = rec + L::VC + c * 1024 + lane * 16;
    uint8_t* sp = rec + L::VS + (q * L::NG + 2 * c + (r >> 3)) * 16;
    if (whole) {
      *reinterpret_cast<uint4*>(wp) = make_uint4(w[0], w[1], w[2], w[3]);
      if (!(r & 7)) *reinterpret_cast<uint4*>(sp) = make_uint4(sc[0], sc[1], sc[2], sc[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!valid(8 * q + i)) continue;
        *reinterpret_cast<uint16_t*>(wp + 2 * i) = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        if (!(r & 7)) *reinterpret_cast<uint16_t*>(sp + 2 * i) = (uint16_t)(sc[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

// Few rows a sequence (a decode step's append): one wave = one token of one kv head, 4 values a lane.  A
// record's wave would keep 31 of 32 tokens' work idle and its bytewise stores serial.
template <int D>
__global__ __launch_bounds__(256) void kv4_store_token_kernel(StoreArgs a) {
  using L = Kv4<D>;
  const int lane = threadIdx.x & 63;
  const unsigned item = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (item >= (unsigned)a.B * a.n * a.KV) return;
  const int kvh = item % (unsigned)a.KV, bi = item / (unsigned)a.KV;
  const int i = bi % (unsigned)a.n, b = bi / (unsigned)a.n;
  const int d = (4 * (lane & 31)) % D;
  const uint16_t* p = (lane < 32 ? a.k + b * a.k_bs + i * a.k_rs : a.v + b * a.v_bs + i * a.v_rs) + (long long)kvh * D + d;
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const long long pos = (long long)a.start[b] + i;
  if (pos < 0 || pos >= (long long)a.tiles * KV4_TILE || (a.count && i >= a.count[b])) return;
  kv4_put_token<D>(a.data + (((long long)b * a.KV + kvh) * a.tiles + pos / KV4_TILE) * L::REC, (int)(pos % KV4_TILE),
                   kv4_token(u, lane), lane);
}

struct LoadArgs {
  const uint8_t* data;
  uint16_t *k, *v;  // [B, n, KV*D] contiguous
  const int* start;
  int B, KV, n, tiles, span;
};

// Values of one record's tokens as bf16 rows (s * c has 12 significant bits: one rounding).  Rows outside the
// cache are zeros.  Records are counted from the one of position start[b], which may be negative.
template <int D>
__global__ __launch_bounds__(256) void kv4_load_kernel(LoadArgs a) {
  using L = Kv4<D>;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const unsigned item = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));  // < 2^31 (launcher)
  constexpr int W = L::WAVES;
  if (item >= (unsigned)W * a.B * a.span * a.KV) return;
  const bool keys = W == 1 || !(item & 1), values = W == 1 || (item & 1);  // what this wave takes of the record
  const int kvh = item / W % (unsigned)a.KV, bs = item / W / (unsigned)a.KV;
  const int sp = bs % (unsigned)a.span, b = bs / (unsigned)a.span;
  const long long start = a.start[b];
  const long long tile = (start >= 0 ? start / KV4_TILE : -((-start + KV4_TILE - 1) / KV4_TILE)) + sp;
  const long long row0 = tile * KV4_TILE - start;
  if (row0 >= a.n) return;
  const bool in = tile >= 0 && tile < a.tiles;
  const uint8_t* rec = a.data + (((long long)b * a.KV + kvh) * a.tiles + (in ? tile : 0)) * L::REC;
  const long long rs = (long long)a.KV * D;
  uint16_t* kp = a.k + (long long)b * a.n * rs + (long long)kvh * D;
  uint16_t* vp = a.v + (long long)b * a.n * rs + (long long)kvh * D;
  auto valid = [&](int t) { return row0 + t >= 0 && row0 + t < a.n; };

  // K: whole rows per store instruction (16 bytes a lane), from 4-byte reads of the record: 5.3 TB/s of record and row
  // bytes at 64 x 2048 tokens of 8 heads x 128, 3.9 where each lane writes out its own chunk (64-byte pieces)
  constexpr int CPR = D / 8, RPI = 64 / CPR;  // 16-byte pieces a row, rows an instruction
  uint32_t kw[32 / RPI];
  float ks[32 / RPI];
  const int kc = lane % CPR;
  uint4 w[L::CH], sc[L::CH];
  if (keys) {
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      int off, sh, so;
      L::k_at(i * RPI + lane / CPR, 8 * kc, &off, &sh, &so);
      kw[i] = *reinterpret_cast<const uint32_t*>(rec + off);
      ks[i] = bf2f(*reinterpret_cast<const uint16_t*>(rec + so));
    }
  }
  if (values) {
#pragma unroll
    for (int c = 0; c < L::CH; ++c) {
      w[c] = *reinterpret_cast<const uint4*>(rec + L::VC + c * 1024 + lane * 16);
      sc[c] = *reinterpret_cast<const uint4*>(rec + L::VS + (q * L::NG + 2 * c + (r >> 3)) * 16);
    }
  }
  if (keys) {
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int t = i * RPI + lane / CPR;
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = ks[i] * ((float)(int)((kw[i] >> (16 * (e & 1) + 4 * (e >> 1))) & 15u) - 8.0f);
      if (valid(t)) *reinterpret_cast<uint4*>(kp + (row0 + t) * rs + 8 * kc) = in ? pack8(f) : make_uint4(0, 0, 0, 0);
    }
  }
  if (!values) return;
#pragma unroll
  for (int c = 0; c < L::CH; ++c) {
    const uint32_t words[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
    float s[8];
    unpack8(sc[c], s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = s[i] * ((float)(int)((words[i >> 1] >> (16 * (i & 1) + 4 * e)) & 15u) - 8.0f);
      if (valid(8 * q + i))
        *reinterpret_cast<uint2*>(vp + (row0 + 8 * q + i) * rs + 64 * c + 4 * r) =
            in ? make_uint2(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3])) : make_uint2(0, 0);
    }
  }
}

}  // namespace

// calls of fewer rows go token by token
constexpr int KV4_STORE_TOKENS = 32;

// records that n consecutive positions can touch, wherever they start
static int waves_of(int D) { return D == 128 ? Kv4<128>::WAVES : Kv4<64>::WAVES; }
static int kv4_span(int n) { return (n + KV4_TILE - 2) / KV4_TILE + 1; }

extern "C" int ftc_kv4_store(void* data, const void* k, const void* v, const int* start, const int* count, int B, int KV,
                             int D, int n, int tiles, long long k_bs, long long k_rs, long long v_bs, long long v_rs,
                             hipStream_t stream) {
  if ((D != 64 && D != 128) || B < 1 || KV < 1 || n < 1 || tiles < 1) return -1;
  const int span = kv4_span(n);
  const bool tokens = n < KV4_STORE_TOKENS;
  const long long waves = (long long)B * KV * (tokens ? n : (long long)span * waves_of(D)), blocks = (waves + 3) / 4;
  if (blocks > 0x1fffffffLL) return -1;  // a wave's index stays below 2^31
  StoreArgs a{(uint8_t*)data, (const uint16_t*)k, (const uint16_t*)v, start, count, k_bs, k_rs, v_bs, v_rs,
              B, KV, n, tiles, span};
  if (tokens && D == 128)
    hipLaunchKernelGGL(kv4_store_token_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else if (tokens)
    hipLaunchKernelGGL(kv4_store_token_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else if (D == 128)
    hipLaunchKernelGGL(kv4_store_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(kv4_store_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

extern "C" int ftc_kv4_load(const void* data, void* k, void* v, const int* start, int B, int KV, int D, int n, int tiles,
                            hipStream_t stream) {
  if ((D != 64 && D != 128) || B < 1 || KV < 1 || n < 1 || tiles < 1) return -1;
  const int span = kv4_span(n);
  const long long waves = (long long)B * KV * span * waves_of(D), blocks = (waves + 3) / 4;
  if (blocks > 0x1fffffffLL) return -1;  // a wave's index stays below 2^31
  LoadArgs a{(const uint8_t*)data, (uint16_t*)k, (uint16_t*)v, start, B, KV, n, tiles, span};
  if (D == 128)
    hipLaunchKernelGGL(kv4_load_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(kv4_load_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}
