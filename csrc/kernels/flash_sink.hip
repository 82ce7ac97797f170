// Attention with a sliding window and sinks: query q sees key k iff k <= q and (q - k < window or k < sinks).
// Causal GQA, bf16, forward and backward, on the tiles and MFMA orientations of flash_attn_fwd.hip /
// flash_attn_bwd.hip (where the layout choices are explained and measured).  Different here:
//   * a query block's key tiles are the sink keys' (at most ceil(sinks / 64)) and then its window's, so a block of
//     128 queries costs (window + 128) / 64 + 1 tiles whatever the length;
//   * any S: rows past the end are read as the last one (an offset clamp per DMA piece), masked, and not stored, so
//     odd lengths need no padded copy of q, k, v and the gradients;
//   * dK / dV of the sink keys: the key-block kernel takes the queries whose window reaches the block; the queries
//     past it are summed by sink_far_kernel over parts of the sequence and joined in part order.  The first block would
//     otherwise sweep the whole sequence while the others sweep a window.
// No float atomics: results do not depend on the order of workgroups.
// Bound: MFMA with the softmax's VALU in the same waves.  32 / 8 heads x 128, 4 sinks: forward of 16384 tokens, window
// 4096: 912 to 956 us on different cards, 1007 to 1056 TF/s (MFMA busy 0.55); 4 x 4096, window 1024: forward 314 to 323 us,
// dQ 427 to 434, dK / dV 600 to 613, far queries 55 (MFMA busy 0.38, 0.48, 0.36: blocks of 128 queries or 256 keys reach
// past a window of 1024 by 12 or 18 %, and dK / dV's workgroups fill two rounds unevenly).
#include "flash_tiles.h"

using namespace ftc;

namespace {

// ---------------------------------------------------------------- forward
constexpr int WAVES = 4;  // x 32 query rows
constexpr int BK = 64;    // keys per tile
constexpr int KPRE = 4;   // K-fragment reads issued ahead of the S MFMA chain

struct FwdArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  uint8_t* olow;  // [B*S, H*D] GRAD: the 8 significand bits of O below bf16's (low_byte)
  float* lse;
  long long q_rs, kv_rs, o_rs;
  int B, S, H, KV, nqb;
  float scale_log2;
  int window, sinks;
};

// logical block -> (qb, b, kvh, g) with heavy-first order and GQA groups co-located on one XCD
DEV_INLINE void decode_block(const FwdArgs& a, int& qb, int& b, int& hq, int& kvh) {
  const int G = a.H / a.KV;
  const int bid = blockIdx.x;
  const int ngroups = a.nqb * a.B * a.KV;
  int j, g;
  if ((ngroups & 7) == 0) {
    const int xcd = bid & 7, slot = bid >> 3;
    g = slot % G;
    j = (slot / G) * 8 + xcd;
  } else {
    g = bid % G;
    j = bid / G;
  }
  kvh = j % a.KV;
  const int t = j / a.KV;
  b = t % a.B;
  const int qr = t / a.B;
  qb = a.nqb - 1 - qr;  // heaviest (latest) query blocks first
  hq = kvh * G + g;
}

// Signed distance of a float from its bf16 rounding in units of 2^-8 of a bf16 step, as a byte, and back: with it O
// has a 16-bit significand.  The backward's delta = rowsum(dO * O) cancels against dP; from the rounded O alone it put
// half again the other roundings' error into dQ and dK (relative error of dqkv 0.0028 against 64 bits, 0.0024 with the
// byte; the output's own rounding is 0.0017).
DEV_INLINE uint32_t low_byte(float x) {
  const int r = (int)(__float_as_uint(x) - ((uint32_t)f2bf(x) << 16)) >> 8;
  return (uint32_t)min(r, 127) & 0xffu;
}
DEV_INLINE float with_low_byte(uint32_t hi, uint32_t byte) {  // hi: the bf16 in the high half
  return __uint_as_float(hi + ((uint32_t)((int)(byte << 24) >> 24) << 8));
}

// O is normalised by the sum of the weights as they were rounded for the PV product, so that the rounding of a row's
// largest weights cancels (and 16 two-element dot products replace 32 adds a tile).  GRAD: a backward pass follows --
// the output's low bits are kept, and the LSE of the unrounded weights.
// GR = 2: two groups of WAVES waves take the block's key tiles in turn, each with its own buffers, and join their O, m, l
// through LDS at the end -- for grids that leave most of the chip idle, where the chain of tiles is the time.
template <int D, bool GRAD, int GR>
__global__ __launch_bounds__(64 * WAVES * GR, 8 / WAVES) void sink_fwd_kernel(FwdArgs a) {
  constexpr int BQ = 32 * WAVES;
  constexpr int NCH = D / 8;           // 16-byte chunks per row
  constexpr int DSTEPS = D / 16;       // k-steps of the S MFMA
  constexpr int DT = D / 32;           // 32-wide d tiles of O
  constexpr int TILE_BYTES = BK * D * 2;
  constexpr int NGT = TILE_BYTES / 1024 / WAVES;  // 1 KiB DMA pieces per wave per matrix
  constexpr int RPG = 1024 / (D * 2);             // rows per piece
  static_assert(NGT >= 1, "tile too small for the wave count");
  // K/V tiles double-buffered in four DISTINCT __shared__ objects: reading one does not make the
  // compiler drain the DMA still filling the other pair (LDS alias scopes)
  __shared__ __attribute__((aligned(16))) char K0[GR * TILE_BYTES];
  __shared__ __attribute__((aligned(16))) char V0[GR * TILE_BYTES];
  __shared__ __attribute__((aligned(16))) char K1[GR * TILE_BYTES];
  __shared__ __attribute__((aligned(16))) char V1[GR * TILE_BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);  // provably wave-uniform -> scalar branches
  const int wave = GR == 1 ? wid : wid % WAVES, grp = GR == 1 ? 0 : wid / WAVES;
  char *const K0g = K0 + grp * TILE_BYTES, *const V0g = V0 + grp * TILE_BYTES;
  char *const K1g = K1 + grp * TILE_BYTES, *const V1g = V1 + grp * TILE_BYTES;
  const int hh = lane >> 5, lr = lane & 31;
  int qb, b, hq, kvh;
  decode_block(a, qb, b, hq, kvh);
  const int S = a.S;
  const int q0 = qb * BQ;
  const int qrow = q0 + wave * 32 + lr;
  const bool qvalid = qrow < S;

  bf16x8 qf[DSTEPS];
  auto load_q = [&]() __attribute__((always_inline)) {
    // ---- Q^T fragments (B operand of S^T = K Q^T): lane holds Q[qrow][16s + 8hh .. +8)
    const uint16_t* qp = a.q + ((long long)b * S + (qvalid ? qrow : 0)) * a.q_rs + (long long)hq * D + 8 * hh;
#pragma unroll
    for (int s = 0; s < DSTEPS; ++s) {
      uint4 v = qvalid ? *reinterpret_cast<const uint4*>(qp + 16 * s) : make_uint4(0, 0, 0, 0);
      qf[s] = as_bf8(v);
    }
  };
  load_q();

  // ---- key tiles: those of the sink keys, then from the window's first
  const int kv_end = min(S, q0 + BQ);
  const int kv_begin = max(0, q0 - a.window + 1) / BK * BK;
  const int nsink = min((a.sinks + BK - 1) / BK, kv_begin / BK);
  const int ntiles = nsink + (kv_end - kv_begin + BK - 1) / BK;
  auto tile_key = [&](const int t) __attribute__((always_inline)) {  // first key of tile t
    return t < nsink ? t * BK : kv_begin + (t - nsink) * BK;
  };

  const uint16_t* kbase = a.k + (long long)b * S * a.kv_rs + (long long)kvh * D;
  const uint16_t* vbase = a.v + (long long)b * S * a.kv_rs + (long long)kvh * D;
  // rows of one (b, kv head) span < 2 GiB (S * kv_rs * 2 bytes): 32-bit buffer offsets
  const auto krs = make_rsrc(kbase), vrs = make_rsrc(vbase);
  // per-lane source offsets of a tile's pieces: row and (pre-swizzled) chunk apart, so that rows past the end of
  // the sequence can be read as its last one
  int vrow[NGT], vcol[NGT];
#pragma unroll
  for (int i = 0; i < NGT; ++i) {
    const int row = (wave * NGT + i) * RPG + lane / NCH, pc = lane % NCH;
    vrow[i] = row * (int)a.kv_rs * 2;
    vcol[i] = ((pc ^ swz(row)) & (NCH - 1)) * 16;
  }
  auto dma = [&](const int kv0, char* Kd, char* Vd) __attribute__((always_inline)) {
    const int last = (S - 1 - kv0) * (int)a.kv_rs * 2;
    int vo[NGT];
#pragma unroll
    for (int i = 0; i < NGT; ++i) vo[i] = min(vrow[i], last) + vcol[i];
    kv_dma<D, NGT, RPG>(krs, vrs, vo, kv0 * (int)a.kv_rs * 2, Kd, Vd, wave);
  };

  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float c = a.scale_log2;
  float lw = 0.f;  // sum of the weights as rounded for the PV product

  __builtin_amdgcn_s_waitcnt(0x0F70);  // Q fragments (plain loads) retired before any DMA: vmcnt(0)
  if (GR == 1 || grp < ntiles) dma(tile_key(grp), K0g, V0g);

  // tr-read addressing (V^T A operand): 16-lane group gi = lane>>4 covers d cols [16*(gi&1), +16)
  // of the 32-wide d tile and key rows [16ks + 4*hh (+8), +4)
  const int gi = lane >> 4, li = lane & 15;
  const int trq = li >> 2, trp = li & 3;
  // lane byte offsets of the transposed V reads, hoisted out of the tile loop: row r1 = 16 ks + 4 hh
  // + trq has swizzle (trq << 2) | hh for every ks (r1 + 8: | (hh + 2)), so ks only moves the row by
  // a compile-time 16 * D * 2 bytes (the ds_read's immediate offset) and the 2 * DT lane offsets below
  // are the only per-lane addressing left in phase B2 (was ~20 address adds per tile)
  int vto[DT][2];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int col = dt * 32 + 16 * (gi & 1) + 4 * trp;
    const int chunk = col >> 3, half8 = (col & 7) ? 8 : 0;
    vto[dt][0] = lds_off<D>(4 * hh + trq, chunk) + half8;
    vto[dt][1] = lds_off<D>(4 * hh + trq + 8, chunk) + half8;
  }

  f32x16 s[2];   // S^T of the current tile, then its P (registers between the phases)
  bf16x8 pf[4];  // packed P^T operand of the PV MFMAs
  // wait for tile t, barrier, then DMA the group's next tile into the slots that held the one before
  auto sync_tile = [&](const int t, char* Kn, char* Vn) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // this wave's pieces of tile t landed (vmcnt(0))
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();        // ... and everyone's
    if (t + GR < ntiles) dma(tile_key(t + GR), Kn, Vn);
  };
  // ---- phase A: S^T = K Q^T, two 32-key blocks
  auto phaseA = [&](const char* Kc) __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      // issue all LDS reads of this 32-key block before its MFMA chain (no read->wait->mfma serialisation)
      const int r = kt * 32 + lr;
      uint4 kf[DSTEPS];
#pragma unroll
      for (int st = 0; st < DSTEPS; ++st) kf[st] = *reinterpret_cast<const uint4*>(Kc + lds_off<D>(r, 2 * st + hh));
      f32x16 acc;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll
      for (int st = 0; st < DSTEPS; ++st) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(kf[st]), qf[st], acc, 0, 0, 0);
      s[kt] = acc;
    }
    // software pipeline of the 2*DSTEPS K-fragment reads against the MFMA chain, 4 reads in flight
    // (the default scheduler serialises read -> wait -> mfma to save registers)
    __builtin_amdgcn_sched_group_barrier(0x100, KPRE, 0);
#pragma unroll
    for (int i = 0; i < 2 * DSTEPS - KPRE; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, KPRE, 0);
  };
  // ---- phase B1: mask (wave-uniform branch, branch-free selects inside) + online softmax in the log2
  // domain; P packed as the bf16 B operand of the PV MFMAs
  auto phaseB1 = [&](const int t) __attribute__((always_inline)) {
    const int kv0 = tile_key(t);
    const int qmin_w = q0 + wave * 32;
    const bool need_mask = kv0 + BK - 1 > qmin_w || (qmin_w + 31 - kv0 >= a.window && kv0 + BK > a.sinks);
    if (need_mask) {
      // key k of element (kt, i) = kv0 + kt*32 + (i&3) + 8*(i>>2) + 4*hh; seen iff k <= q and (q - k < window or k < sinks)
      const int base = kv0 + 4 * hh;
      const int hi = qrow - base, lo = qrow - a.window + 1 - base, snk = a.sinks - base;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int off = kt * 32 + (i & 3) + 8 * (i >> 2);
          s[kt][i] = ((off >= lo || off < snk) && off <= hi) ? s[kt][i] : -INFINITY;
        }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[kt][i]);  // (a depth-5 fmaxf tree measured 3-4 % slower)
    mt = xhalf_max(mt) * c;  // c > 0: max commutes with the scale
    // deferred rescale: the running reference m moves -- and O, l are rescaled -- only
    // when some row's max grew by more than 2^8; otherwise P <= 256 (exact in bf16's exponent range,
    // fp32 accumulation) and the 64 multiplies of O are skipped.  Wave-uniform branch.
    if (__builtin_amdgcn_ballot_w64(mt > m + 8.0f) != 0) {
      const float mn = fmaxf(m, mt);
      const float alpha = __builtin_amdgcn_exp2f(m - ((mn == -INFINITY) ? 0.f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
      lw *= alpha;
    }
    const float mref = (m == -INFINITY) ? 0.f : m;
    float rs = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], c, -mref));
        s[kt][i] = p;
        if constexpr (GRAD) rs += p;
      }
    if constexpr (GRAD) l += rs;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      uint32_t w[4];  // summed from the words: taken back out of the operand vector, hipcc 7.2 sums its first word 4 times
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = pack_bf2(s[ks >> 1][8 * (ks & 1) + 2 * i], s[ks >> 1][8 * (ks & 1) + 2 * i + 1]);
        lw = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w[i]), __builtin_bit_cast(bf16x2, 0x3f803f80u), lw, false);
      }
      pf[ks] = as_bf8(make_uint4(w[0], w[1], w[2], w[3]));
    }
  };
  // ---- phase B2: O^T += V^T P^T, 4 k-steps of 16 keys
  auto phaseB2 = [&](const char* Vc) __attribute__((always_inline)) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      s16x4 vt[8];  // all 8 transposed reads of this 32-wide d tile in flight before the MFMA chain
      const char* v0 = Vc + vto[dt][0];
      const char* v8 = Vc + vto[dt][1];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        vt[2 * ks] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(v0 + ks * 16 * D * 2));
        vt[2 * ks + 1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(v8 + ks * 16 * D * 2));
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const s16x4 v1 = vt[2 * ks], v2 = vt[2 * ks + 1];
        s16x8 va = {v1[0], v1[1], v1[2], v1[3], v2[0], v2[1], v2[2], v2[3]};
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, va), pf[ks], o[dt], 0, 0, 0);
      }
    }
  };
  // tile t reads (Kc, Vc); tile t+1 is DMA'd into (Kn, Vn), which held tile t-1 -- free once every
  // wave passed this tile's barrier
  auto tile = [&](const int t, const char* Kc, const char* Vc, char* Kn, char* Vn) __attribute__((always_inline)) {
    sync_tile(t, Kn, Vn);
    if (GR > 1 && t >= ntiles) return;  // (the groups meet at the same barriers)
    // a wave sees nothing of the tiles past its rows and before its window: with a short window they are many (341 us
    // instead of 362 at 4 x 4096 tokens, window 1024, 32 heads x 128; 0-1 % at 4096 of 8192 and 16384)
    const int kv0 = tile_key(t), qw = q0 + wave * 32;
    if (kv0 > qw + 31 || (qw - (kv0 + BK - 1) >= a.window && kv0 >= a.sinks)) return;
    phaseA(Kc);
    phaseB1(t);
    phaseB2(Vc);
  };
  const int steps = (ntiles + GR - 1) / GR;
  for (int i = 0; i < steps; i += 2) {
    tile(GR * i + grp, K0g, V0g, K1g, V1g);
    if (i + 1 < steps) tile(GR * (i + 1) + grp, K1g, V1g, K0g, V0g);
  }

  // ---- join the groups: a lane holds the same row and elements in both; one shared object for each wave of a group
  if constexpr (GR == 2) {
    static_assert(WAVES == 4 && 64 * (DT * 16 + 3) * 4 <= GR * TILE_BYTES, "join buffers");
    float* const jb = reinterpret_cast<float*>(wave == 0 ? K0 : wave == 1 ? V0 : wave == 2 ? K1 : V1);
    __syncthreads();  // every wave is past its last tile
    if (grp == 1) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(jb + ((t * 4 + i) * 64 + lane) * 4) =
              make_float4(o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]);
      jb[DT * 1024 + lane] = m;
      jb[DT * 1024 + 64 + lane] = lw;
      jb[DT * 1024 + 128 + lane] = l;
    }
    __syncthreads();
    if (grp == 1) return;
    const float m1 = jb[DT * 1024 + lane], mn = fmaxf(m, m1), mref = mn == -INFINITY ? 0.f : mn;
    const float a0 = __builtin_amdgcn_exp2f(m - mref), a1 = __builtin_amdgcn_exp2f(m1 - mref);
    m = mn;
    lw = lw * a0 + jb[DT * 1024 + 64 + lane] * a1;
    l = l * a0 + jb[DT * 1024 + 128 + lane] * a1;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(jb + ((t * 4 + i) * 64 + lane) * 4);
        o[t][4 * i] = o[t][4 * i] * a0 + x.x * a1;
        o[t][4 * i + 1] = o[t][4 * i + 1] * a0 + x.y * a1;
        o[t][4 * i + 2] = o[t][4 * i + 2] * a0 + x.z * a1;
        o[t][4 * i + 3] = o[t][4 * i + 3] * a0 + x.w * a1;
      }
  }

  // ---- epilogue: normalise, store O (bf16) and LSE (natural log)
  lw += __shfl_xor(lw, 32, 64);
  const float inv = lw > 0.f ? 1.0f / lw : 0.f;
  uint16_t* op = a.o + ((long long)b * S + (qvalid ? qrow : 0)) * a.o_rs + (long long)hq * D;
  if constexpr (GRAD) {
    // the 4 bytes of each g4 are a dword; two swaps give lane half hh the 16 bytes of d [16 hh, 16 hh + 16)
    uint8_t* lp = a.olow + ((long long)b * S + (qvalid ? qrow : 0)) * ((long long)a.H * D) + (long long)hq * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      uint32_t w[4];
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        w[g4] = low_byte(o[dt][4 * g4] * inv) | low_byte(o[dt][4 * g4 + 1] * inv) << 8 |
                low_byte(o[dt][4 * g4 + 2] * inv) << 16 | low_byte(o[dt][4 * g4 + 3] * inv) << 24;
      const auto a0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
      const auto b0 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      if (qvalid) *reinterpret_cast<uint4*>(lp + dt * 32 + 16 * hh) = make_uint4(a0[0], a0[1], b0[0], b0[1]);
    }
  }
  // 16-byte stores (the store tail is issue-bound): lanes l and l ^ 32 hold the same
  // query row, d runs {8 g4 + 4 hh + 0..3}; two v_permlane32_swap per dword pair give lane half hh
  // the 16 contiguous d [16 hh, 16 hh + 16) of each 32-wide tile -> 2 x dwordx4 instead of 4 x dwordx2
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    uint32_t w[4][2];
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      w[g4][0] = pack_bf2(o[dt][4 * g4 + 0] * inv, o[dt][4 * g4 + 1] * inv);
      w[g4][1] = pack_bf2(o[dt][4 * g4 + 2] * inv, o[dt][4 * g4 + 3] * inv);
    }
    // swap(x, y): lanes 0-31 keep x and receive the upper half's x; lanes 32-63 receive the lower
    // half's y and keep y -> (x_own | x_partner) below, (y_partner | y_own) above
    const auto a0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[2][0], false, false);
    const auto a1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[2][1], false, false);
    const auto b0 = __builtin_amdgcn_permlane32_swap(w[1][0], w[3][0], false, false);
    const auto b1 = __builtin_amdgcn_permlane32_swap(w[1][1], w[3][1], false, false);
    if (qvalid) {
      const int d = dt * 32 + 16 * hh;
      *reinterpret_cast<uint4*>(op + d) = make_uint4(a0[0], a1[0], a0[1], a1[1]);
      *reinterpret_cast<uint4*>(op + d + 8) = make_uint4(b0[0], b1[0], b0[1], b1[1]);
    }
  }
  if constexpr (GRAD) {
    const float ltot = l + __shfl_xor(l, 32, 64);
    if (qvalid && hh == 0) {
      const float lse2 = (m == -INFINITY) ? -INFINITY : m + __log2f(ltot);
      a.lse[((long long)b * a.H + hq) * S + qrow] = lse2 * LN2;
    }
  }
}

// ---------------------------------------------------------------- backward
struct BwdArgs {
  const uint16_t *q, *k, *v, *o, *dout;
  const uint8_t* olow;  // O's bits below bf16's (low_byte)
  const float* lse;
  float* delta;  // workspace [-delta | -lse/scale], B*H*S each
  uint16_t *dq, *dk, *dv;
  long long q_rs, kv_rs, o_rs, dq_rs, dkv_rs, do_rs;
  int B, S, H, KV;
  float scale, c;  // c = scale * log2(e)
  int window, sinks;
  float* far;  // [B * KV, nfar, sinks, 2 (dK before the scale, dV), D] sums of the sink keys' far queries (null: none)
  int nfar;
  float* ksum;  // [B * KV, kparts, S, 2, D] sums of key blocks swept in parts (kparts > 1)
  int kparts;
  const float* rcos;  // RoPE folded into the dQ / dK epilogues (rope_inv_rows), or null
  const float* rsin;
  const int* rpos;
};

// ---------------------------------------------------------------- dK / dV
// As bwd_dkdv8_kernel (8 waves x 32 keys in ping-pong phase order, 5-slot DMA ring), windowed.
// PARTS: the workgroup sweeps one part of the block's slices and leaves 32-bit sums for sink_join_kernel.
template <int D, int QR, bool PARTS>
__global__ __launch_bounds__(512, 1) void sink_dkdv_kernel(BwdArgs a) {
  constexpr int DIST = 3;
  static_assert(QR == 1 || QR == 2, "one or two 32-row query blocks per slice");
  constexpr int NCH = D / 8, DSTEPS = D / 16, DT = D / 32;
  constexpr int BKV = 256, BQ2 = 32 * QR;
  constexpr int WAVES = 8, NT = 64 * WAVES;
  constexpr int KBYTES = BKV * D * 2, QBYTES = BQ2 * D * 2;
  constexpr int SLICE = 2 * QBYTES + 2 * BQ2 * 4;  // Q | dO | -lse/scale | -delta
  // K and the five ring slots are DISTINCT __shared__ objects: the compiler then knows (LDS alias
  // scopes) that reading one slot does not depend on the DMA still writing the others, instead of
  // draining every DMA (vmcnt(0)) before the first ds_read of each slice
  __shared__ __attribute__((aligned(16))) char Ks[KBYTES];
  __shared__ __attribute__((aligned(16))) char slot0[SLICE];
  __shared__ __attribute__((aligned(16))) char slot1[SLICE];
  __shared__ __attribute__((aligned(16))) char slot2[SLICE];
  __shared__ __attribute__((aligned(16))) char slot3[SLICE];
  __shared__ __attribute__((aligned(16))) char slot4[SLICE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hh = lane >> 5, lr = lane & 31;
  const int S = a.S, G = a.H / a.KV;
  const int npairs = a.B * a.KV;
  int kb, pair;
  const int part = PARTS ? blockIdx.x % a.kparts : 0;
  {
    const int bid = PARTS ? blockIdx.x / a.kparts : blockIdx.x;
    if ((npairs & 7) == 0) {
      const int xcd = bid & 7, slot = bid >> 3, ppx = npairs >> 3;
      kb = slot / ppx;
      pair = (slot % ppx) * 8 + xcd;
    } else {
      kb = bid / npairs;
      pair = bid % npairs;
    }
  }
  const int kvh = pair % a.KV, b = pair / a.KV;
  const int kv0 = kb * BKV;
  const int wkey0 = kv0 + wave * 32;  // this wave's first key

  // stage the block's K rows into LDS; V^T fragments (B operand of dP) to registers
  const uint16_t* kbase = a.k + ((long long)b * S) * a.kv_rs + (long long)kvh * D;
  {
    constexpr int RPP = NT / NCH;
    const int lrow = tid / NCH, lch = tid % NCH;
    const auto krs = make_rsrc(kbase + (long long)kv0 * a.kv_rs);
#pragma unroll
    for (int p = 0; p < BKV / RPP; ++p)  // rows past the end of the sequence are read as its last one, here and below
      *reinterpret_cast<u32x4*>(Ks + lds_off<D>(p * RPP + lrow, lch)) =
          buf_load16(krs, (min(p * RPP + lrow, S - 1 - kv0) * (int)a.kv_rs + lch * 8) * 2, 0);
  }
  bf16x8 vf[DSTEPS];
  {
    const int vrow = min(wkey0 + lr, S - 1);
    const uint16_t* vp = a.v + ((long long)b * S + vrow) * a.kv_rs + (long long)kvh * D + 8 * hh;
#pragma unroll
    for (int s = 0; s < DSTEPS; ++s) vf[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(vp + 16 * s));
  }

  f32x16 dv[DT], dk[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) { dv[t][i] = 0.f; dk[t][i] = 0.f; }

  // queries whose window reaches this key block (the sink keys' later queries: sink_far_kernel)
  const int qbeg = kv0 / BQ2 * BQ2, qend = min(S, kv0 + BKV - 1 + a.window);
  const int nqt = (qend - qbeg + BQ2 - 1) / BQ2;
  const int per = PARTS ? (G * nqt + a.kparts - 1) / a.kparts : G * nqt, it0 = part * per;
  const int total = PARTS ? min(per, G * nqt - it0) : per;
  // Q / dO / row-constant slices arrive by LDS-DMA (global_load_lds_dwordx4: no staging VGPRs) into a
  // 5-slot ring, three slices ahead of the compute; one raw barrier per slice with a COUNTED vmcnt so the
  // next slice's DMA stays in flight across it.  The swizzled
  // LDS image is produced by pre-swizzling the per-lane global source (the DMA writes lane-linearly).
  constexpr int PIECES = BQ2 * D * 2 / 1024;         // 1 KiB pieces per matrix per slice
  constexpr bool SPLIT = PIECES < WAVES;             // D = 64, 8 waves: one piece of Q OR dO per wave
  static_assert(!SPLIT || 2 * PIECES == WAVES, "split DMA: one piece per wave");
  constexpr int NG = SPLIT ? 1 : PIECES / WAVES;     // 1 KiB DMA pieces per wave per matrix
  static_assert(NG >= 1, "each wave DMAs at least one 1 KiB piece of Q and of dO");
  constexpr int PER_SLICE = (SPLIT ? 1 : 2 * NG) + QR;  // DMA instructions per wave per slice (+ row constants)
  constexpr int RPG = 1024 / (D * 2);                // rows per 1 KiB piece
  // DMA sources as buffer resources (SGPRs) + per-lane loop-invariant 32-bit offsets: the slice's head
  // and row position go into the scalar offset, so no 64-bit address VGPRs stay live in the loop
  const auto qrsrc = make_rsrc(a.q + (long long)b * S * a.q_rs);
  const auto drsrc = make_rsrc(a.dout + (long long)b * S * a.do_rs);
  const auto crsrc = make_rsrc(a.delta);  // workspace [-delta | -lse/scale]
  int qrow[NG], drow[NG], ccol[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int row = ((SPLIT ? wave % PIECES : wave * NG) + i) * RPG + lane / NCH, pc = lane % NCH;
    qrow[i] = row * (int)a.q_rs * 2;
    drow[i] = row * (int)a.do_rs * 2;
    ccol[i] = ((pc ^ swz(row)) & (NCH - 1)) * 16;  // pre-swizzled source, lane-linear destination
  }
  // QR = 1: lanes 0..31 -lse/scale of the 32 rows, lanes 32..63 -delta (every wave issues the same
  // piece); QR = 2: one piece of the 64 rows' -lse/scale and one of their -delta
  auto issue = [&](int it_, char* base_) {
    const int g_ = (it0 + it_) / nqt, qt_ = qbeg + ((it0 + it_) % nqt) * BQ2;
    const int hq_ = kvh * G + g_, left = S - 1 - qt_;
    int qvo[NG], dvo[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      qvo[i] = min(qrow[i], left * (int)a.q_rs * 2) + ccol[i];
      dvo[i] = min(drow[i], left * (int)a.do_rs * 2) + ccol[i];
    }
    const int cvo = QR == 1 ? (min(lr, left) + (hh ? 0 : a.B * a.H * S)) * 4 : (min(lane, left) + a.B * a.H * S) * 4;
    dkdv_dma<D, NG, RPG, QBYTES, SPLIT, QR>(qrsrc, drsrc, crsrc, qvo, dvo, cvo, min(lane, left) * 4,
                                            (hq_ * D + qt_ * (int)a.q_rs) * 2, (hq_ * D + qt_ * (int)a.do_rs) * 2,
                                            ((b * a.H + hq_) * S + qt_) * 4, base_, wave);
  };
  constexpr int VM_ONE = 0x0F70 | (PER_SLICE & 15) | ((PER_SLICE >> 4) << 14);  // vmcnt(PER_SLICE)
  constexpr int VM_TWO = 0x0F70 | ((2 * PER_SLICE) & 15) | (((2 * PER_SLICE) >> 4) << 14);  // vmcnt(2 PER_SLICE)
  constexpr int VM_ZERO = 0x0F70;                                               // vmcnt(0)
  constexpr int LGKM_ZERO = 0xC07F;                                             // lgkmcnt(0)

  // K staging and the V fragments are ordinary loads: retire them before the first DMA so no
  // compiler-inserted wait inside the loop has to count them
  __builtin_amdgcn_s_waitcnt(VM_ZERO);
  __syncthreads();  // K staged (no DMA in flight yet: a plain barrier is fine here)
  if (total > 0) issue(0, slot0);
  if (total > 1) issue(1, slot1);
  if (total > 2) issue(2, slot2);
  f32x16 s[QR], dp[QR];  // S / dP' of the slice between phase A and phase B (registers)
  // phase A: S[q][k], dP'[q][k] in one k-loop (rows q in registers, key on the lane), the K fragments read once
  // for all row blocks -- 2 QR independent MFMA chains
  auto phaseA = [&](const char* Qs) __attribute__((always_inline)) {
    const char* Ds = Qs + QBYTES;
    const float* lse_s = reinterpret_cast<const float*>(Ds + QBYTES);
    const float* dlt_s = lse_s + BQ2;
#pragma unroll
    for (int r = 0; r < QR; ++r)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const float4 lv = *reinterpret_cast<const float4*>(lse_s + 32 * r + 8 * g4 + 4 * hh);
        const float4 dv4 = *reinterpret_cast<const float4*>(dlt_s + 32 * r + 8 * g4 + 4 * hh);
        s[r][4 * g4 + 0] = lv.x; s[r][4 * g4 + 1] = lv.y; s[r][4 * g4 + 2] = lv.z; s[r][4 * g4 + 3] = lv.w;
        dp[r][4 * g4 + 0] = dv4.x; dp[r][4 * g4 + 1] = dv4.y; dp[r][4 * g4 + 2] = dv4.z; dp[r][4 * g4 + 3] = dv4.w;
      }
#pragma unroll
    for (int st = 0; st < DSTEPS; ++st) {
      u32x4 qa[QR], da[QR];
#pragma unroll
      for (int r = 0; r < QR; ++r) {
        qa[r] = *reinterpret_cast<const u32x4*>(Qs + lds_off<D>(32 * r + lr, 2 * st + hh));
        da[r] = *reinterpret_cast<const u32x4*>(Ds + lds_off<D>(32 * r + lr, 2 * st + hh));
      }
      const u32x4 kk = *reinterpret_cast<const u32x4*>(Ks + lds_off<D>(wave * 32 + lr, 2 * st + hh));
#pragma unroll
      for (int r = 0; r < QR; ++r)
        s[r] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, qa[r]), __builtin_bit_cast(bf16x8, kk), s[r], 0, 0, 0);
#pragma unroll
      for (int r = 0; r < QR; ++r)
        dp[r] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, da[r]), vf[st], dp[r], 0, 0, 0);
    }
    // fragment reads of two k-steps in flight ahead of the MFMA chain, the rest interleaved
    {
      constexpr int NDS = (2 * QR + 1) * DSTEPS, NMF = 2 * QR * DSTEPS, PRE = (2 * QR + 1);
      constexpr int REM = NDS - PRE, Q = REM / NMF, X = REM % NMF;
      __builtin_amdgcn_sched_group_barrier(0x100, PRE, 0);
#pragma unroll
      for (int i = 0; i < X; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, Q + 1, 0);
      }
#pragma unroll
      for (int i = X; i < NMF; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr (Q > 0) __builtin_amdgcn_sched_group_barrier(0x100, Q, 0);
      }
    }
  };
  // phase B1: P, dS (bf16 B operands of the accumulating products) -- exp / mask / pack VALU work
  bf16x8 pb[QR][2], sb[QR][2];
  auto phaseB1 = [&](const int it) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < QR; ++r) {
      const int qt = qbeg + ((it0 + it) % nqt) * BQ2 + 32 * r;
      const int key = wkey0 + lr;
      const bool need_mask = qt < wkey0 + 31 || qt + 31 - wkey0 >= a.window || qt + 32 > S;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[r][i] = __builtin_amdgcn_exp2f(a.c * s[r][i]);
      if (need_mask) {  // wave-uniform; query q = qt + (i&3) + 8(i>>2) + 4hh valid iff key <= q < key + window
        const int base = qt + 4 * hh;
        const int lo = key - base, hi = min(key + a.window, S) - 1 - base;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int off = (i & 3) + 8 * (i >> 2);
          s[r][i] = (off >= lo && off <= hi) ? s[r][i] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[r][i] = s[r][i] * dp[r][i];
      pb[r][0] = pack8_bf(s[r], 0);
      pb[r][1] = pack8_bf(s[r], 8);
      sb[r][0] = pack8_bf(dp[r], 0);
      sb[r][1] = pack8_bf(dp[r], 8);
    }
  };
  // phase B2: dV^T += dO^T P ; dK^T += Q^T dS (k of these MFMAs = the slice's query rows)
  auto phaseB2 = [&](const char* Qs) __attribute__((always_inline)) {
    const char* Ds = Qs + QBYTES;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int2 to = tr_offsets<D>(dt * 32, lane);
#pragma unroll
      for (int r = 0; r < QR; ++r) {
        const bf16x8 a0 = tr_read<D>(Ds, 32 * r, to);
        const bf16x8 a1 = tr_read<D>(Ds, 32 * r + 16, to);
        const bf16x8 q0v = tr_read<D>(Qs, 32 * r, to);
        const bf16x8 q1v = tr_read<D>(Qs, 32 * r + 16, to);
        dv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a0, pb[r][0], dv[dt], 0, 0, 0);
        dv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a1, pb[r][1], dv[dt], 0, 0, 0);
        dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q0v, sb[r][0], dk[dt], 0, 0, 0);
        dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q1v, sb[r][1], dk[dt], 0, 0, 0);
      }
    }
  };
  // some key of this wave is seen by some query of the slice (the others are skipped: backward 1113 instead of 1151 us at
  // 4 x 4096 tokens, window 1024; 741 instead of 798 at 2 x 8192, window 512; 1 % slower at 8192, window 4096); not in
  // parts, whose kernel would spill 374 registers for it
  auto seen = [&](const int it) __attribute__((always_inline)) {
    if constexpr (PARTS) return true;
    const int qt = qbeg + ((it0 + it) % nqt) * BQ2;
    return qt + BQ2 - 1 >= wkey0 && qt - (wkey0 + 31) < a.window;
  };
  // one barrier per slice: slice it is in LDS for every wave, the DMA of slice it + DIST goes out
  auto sync_slice = [&](const int it, char* dma_slot) __attribute__((always_inline)) {
    if (it + 2 < total) {
      __builtin_amdgcn_s_waitcnt(VM_TWO);  // slices it+1, it+2 may fly on
    } else if (it + 1 < total) {
      __builtin_amdgcn_s_waitcnt(VM_ONE);  // slice it landed, it+1 may fly on
    } else {
      __builtin_amdgcn_s_waitcnt(VM_ZERO);
    }
    __builtin_amdgcn_s_waitcnt(LGKM_ZERO);
    __builtin_amdgcn_s_barrier();  // every wave's pieces of slice it are in
    if (it + DIST < total) issue(it + DIST, dma_slot);
  };
  // ping-pong over a 5-slot ring, DMA three slices ahead: slice it in slot it % 5; the DMA of slice it + 3
  // reuses the slot of slice it - 2, whose last reader (half 1's phase B2) finished before this slice's
  // barrier.  Half 1 carries only the packed P / dS operands (16 VGPRs) across the barrier:
  // ... [B2(it-1) A(it) B1(it)] ...; the halves run separate straight-line loops (one branch outside the
  // loop, not one per slice: the register allocator then sees two independent paths) with the same
  // barrier count
  if (wave < 4) {  // waves w and w + 4 share a SIMD
    auto body = [&](const int it, const char* Qs, char* dma_slot) __attribute__((always_inline)) {
      sync_slice(it, dma_slot);
      if (!seen(it)) return;
      phaseA(Qs);
      phaseB1(it);
      phaseB2(Qs);
    };
    for (int it = 0; it < total; it += 5) {
      body(it, slot0, slot3);
      if (it + 1 < total) body(it + 1, slot1, slot4);
      if (it + 2 < total) body(it + 2, slot2, slot0);
      if (it + 3 < total) body(it + 3, slot3, slot1);
      if (it + 4 < total) body(it + 4, slot4, slot2);
    }
  } else {
    auto body = [&](const int it, const char* Qs, const char* Qprev, char* dma_slot) __attribute__((always_inline)) {
      sync_slice(it, dma_slot);
      if (it > 0 && seen(it - 1)) phaseB2(Qprev);
      if (!seen(it)) return;
      phaseA(Qs);
      phaseB1(it);
    };
    for (int it = 0; it < total; it += 5) {
      body(it, slot0, slot4, slot3);
      if (it + 1 < total) body(it + 1, slot1, slot0, slot4);
      if (it + 2 < total) body(it + 2, slot2, slot1, slot0);
      if (it + 3 < total) body(it + 3, slot3, slot2, slot1);
      if (it + 4 < total) body(it + 4, slot4, slot3, slot2);
    }
    if (total > 0 && seen(total - 1)) {
      const int r = (total - 1) % 5;
      phaseB2(r == 0 ? slot0 : r == 1 ? slot1 : r == 2 ? slot2 : r == 3 ? slot3 : slot4);
    }
  }

  // ---- epilogue: dK = scale * dK^T^T, dV; lane owns one key row
  const int key = wkey0 + lr;
  if (key >= S) return;
  if constexpr (PARTS) {
    float* p = a.ksum + (((long long)pair * a.kparts + part) * S + key) * 2 * D + 4 * hh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        *reinterpret_cast<float4*>(p + 32 * dt + 8 * g4) =
            make_float4(dk[dt][4 * g4], dk[dt][4 * g4 + 1], dk[dt][4 * g4 + 2], dk[dt][4 * g4 + 3]);
        *reinterpret_cast<float4*>(p + D + 32 * dt + 8 * g4) =
            make_float4(dv[dt][4 * g4], dv[dt][4 * g4 + 1], dv[dt][4 * g4 + 2], dv[dt][4 * g4 + 3]);
      }
    return;
  }
  if (a.far && key < a.sinks) {  // queries past this key's window
    const float* fp = a.far + ((long long)pair * a.nfar * a.sinks + key) * 2 * D + 4 * hh;
    for (int n = 0; n < a.nfar; ++n, fp += (long long)a.sinks * 2 * D) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const float4 x = *reinterpret_cast<const float4*>(fp + 32 * dt + 8 * g4);
          const float4 y = *reinterpret_cast<const float4*>(fp + D + 32 * dt + 8 * g4);
          dk[dt][4 * g4] += x.x; dk[dt][4 * g4 + 1] += x.y; dk[dt][4 * g4 + 2] += x.z; dk[dt][4 * g4 + 3] += x.w;
          dv[dt][4 * g4] += y.x; dv[dt][4 * g4 + 1] += y.y; dv[dt][4 * g4 + 2] += y.z; dv[dt][4 * g4 + 3] += y.w;
        }
    }
  }
  uint16_t* dkp = a.dk + ((long long)b * S + key) * a.dkv_rs + (long long)kvh * D;
  uint16_t* dvp = a.dv + ((long long)b * S + key) * a.dkv_rs + (long long)kvh * D;
  if constexpr (D == 128) {
    if (a.rcos) rope_inv_rows<DT>(dk, a, (long long)b * S + key, hh);
  }
  store_rows<DT>(dkp, dk, a.scale, hh, true);
  store_rows<DT>(dvp, dv, 1.0f, hh, true);
}

// dK / dV rows of key blocks that were swept in parts: the parts' sums and the sink keys' far sums in order, then the
// same epilogue.  A thread holds 4 columns of each half of a row (RoPE pairs d with d + 64).
template <int D>
__global__ __launch_bounds__(256) void sink_join_kernel(BwdArgs a) {
  constexpr int TPK = D / 8;  // threads a key
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = id / TPK;  // pair * S + key
  const int d0 = (int)(id % TPK) * 4;
  if (row >= (long long)a.B * a.KV * a.S) return;
  const int key = (int)(row % a.S), pair = (int)(row / a.S), kvh = pair % a.KV, b = pair / a.KV;
  float acc[2][2][4] = {};  // dK | dV, halves of the row
  auto add = [&](const float* p) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 x = *reinterpret_cast<const float4*>(p + m * D + h * (D / 2) + d0);
        acc[m][h][0] += x.x; acc[m][h][1] += x.y; acc[m][h][2] += x.z; acc[m][h][3] += x.w;
      }
  };
#pragma unroll 4
  for (int n = 0; n < a.kparts; ++n) add(a.ksum + (((long long)pair * a.kparts + n) * a.S + key) * 2 * D);
  if (a.far && key < a.sinks) {
#pragma unroll 4
    for (int n = 0; n < a.nfar; ++n) add(a.far + (((long long)pair * a.nfar + n) * a.sinks + key) * 2 * D);
  }
  const long long token = (long long)b * a.S + key;
  if constexpr (D == 128) {
    if (a.rcos) {
      const long long t = (long long)(a.rpos ? a.rpos[token] : key) * 64 + d0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float c = a.rcos[t + e], sn = a.rsin[t + e], g1 = acc[0][0][e], g2 = acc[0][1][e];
        acc[0][0][e] = g1 * c + g2 * sn;
        acc[0][1][e] = g2 * c - g1 * sn;
      }
    }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    uint16_t* o = (m ? a.dv : a.dk) + token * a.dkv_rs + (long long)kvh * D + d0;
    const float sc = m ? 1.0f : a.scale;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<uint2*>(o + h * (D / 2)) = make_uint2(pack_bf2(acc[m][h][0] * sc, acc[m][h][1] * sc),
                                                              pack_bf2(acc[m][h][2] * sc, acc[m][h][3] * sc));
  }
}

// ---------------------------------------------------------------- dK / dV of the sink keys, far queries
// The pairs (q, k) with k < sinks and q - k >= window, which the key-block kernel above leaves out: its block of
// the first 256 keys would otherwise sweep every query while the others sweep a window's worth.  One workgroup
// = 32 sink keys of one (batch, kv head) x one part of the queries; its waves take 32-row slices (of all G query
// heads), staged in wave-private LDS for the transposed reads, with K and V of the keys in registers; partial
// sums per workgroup in 32 bits, added in part order by the key-block kernel.  Bound by reading Q and dO once more.
constexpr int FAR_WAVES = 4;
template <int D>
__global__ __launch_bounds__(64 * FAR_WAVES, 1) void sink_far_kernel(BwdArgs a) {
  constexpr int DSTEPS = D / 16, DT = D / 32, QB = 32 * D * 2;
  // per wave: Q | dO | -lse/scale | -delta of one slice; afterwards the sums of two waves
  constexpr int SL = 2 * QB + 256, SUMS = 2 * 32 * D * 4;
  constexpr int LDS = FAR_WAVES * SL > 2 * SUMS ? FAR_WAVES * SL : 2 * SUMS;
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hh = lane >> 5, lr = lane & 31, S = a.S, G = a.H / a.KV;
  const int part = blockIdx.x % a.nfar, pair = blockIdx.x / a.nfar % (a.B * a.KV), kt = blockIdx.x / a.nfar / (a.B * a.KV);
  const int kvh = pair % a.KV, b = pair / a.KV, key0 = 32 * kt, key = key0 + lr, krow = min(key, S - 1);
  char* Qs = lds + wave * SL;
  char* Ds = Qs + QB;
  float* Cs = reinterpret_cast<float*>(Ds + QB);

  bf16x8 kf[DSTEPS], vf[DSTEPS];
#pragma unroll
  for (int st = 0; st < DSTEPS; ++st) {
    const long long off = ((long long)b * S + krow) * a.kv_rs + (long long)kvh * D + 16 * st + 8 * hh;
    kf[st] = as_bf8(*reinterpret_cast<const uint4*>(a.k + off));
    vf[st] = as_bf8(*reinterpret_cast<const uint4*>(a.v + off));
  }
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) { dk[t][i] = 0.f; dv[t][i] = 0.f; }

  const int sl0 = (key0 + a.window) / 32, nsl = (S + 31) / 32 - sl0;  // slices that hold far queries of these keys
  const int total = nsl > 0 ? nsl * G : 0, per = (total + a.nfar - 1) / a.nfar;
  const int t1 = min(total, (part + 1) * per);
  uint4 qa[DSTEPS], da[DSTEPS], qn[DSTEPS], dn[DSTEPS];
  float cst = 0.f, cn = 0.f;
  auto fetch = [&](int t) __attribute__((always_inline)) {  // slice t's rows, into the next registers
    const int qt = (sl0 + t / G) * 32, hq = kvh * G + t % G, row = min(qt + lr, S - 1);
    const uint16_t* qp = a.q + ((long long)b * S + row) * a.q_rs + (long long)hq * D + 8 * hh;
    const uint16_t* dp = a.dout + ((long long)b * S + row) * a.do_rs + (long long)hq * D + 8 * hh;
#pragma unroll
    for (int st = 0; st < DSTEPS; ++st) {
      qn[st] = *reinterpret_cast<const uint4*>(qp + 16 * st);
      dn[st] = *reinterpret_cast<const uint4*>(dp + 16 * st);
    }
    // lanes 0..31 -lse/scale, 32..63 -delta
    cn = a.delta[((long long)b * a.H + hq) * S + row + (hh ? 0 : (long long)a.B * a.H * S)];
  };
  int t = part * per + wave;
  if (t < t1) fetch(t);
  for (; t < t1; t += FAR_WAVES) {
    const int qt = (sl0 + t / G) * 32;
#pragma unroll
    for (int st = 0; st < DSTEPS; ++st) {
      qa[st] = qn[st];
      da[st] = dn[st];
    }
    cst = cn;
    fetch(min(t + FAR_WAVES, t1 - 1));
#pragma unroll
    for (int st = 0; st < DSTEPS; ++st) {
      *reinterpret_cast<uint4*>(Qs + lds_off<D>(lr, 2 * st + hh)) = qa[st];
      *reinterpret_cast<uint4*>(Ds + lds_off<D>(lr, 2 * st + hh)) = da[st];
    }
    Cs[lane] = cst;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    f32x16 s, dp;
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const float4 lv = *reinterpret_cast<const float4*>(Cs + 8 * g4 + 4 * hh);
      const float4 de = *reinterpret_cast<const float4*>(Cs + 32 + 8 * g4 + 4 * hh);
      s[4 * g4] = lv.x; s[4 * g4 + 1] = lv.y; s[4 * g4 + 2] = lv.z; s[4 * g4 + 3] = lv.w;
      dp[4 * g4] = de.x; dp[4 * g4 + 1] = de.y; dp[4 * g4 + 2] = de.z; dp[4 * g4 + 3] = de.w;
    }
#pragma unroll
    for (int st = 0; st < DSTEPS; ++st) {
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(qa[st]), kf[st], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(da[st]), vf[st], dp, 0, 0, 0);
    }
    // query qt + (i & 3) + 8 (i >> 2) + 4 hh counts if it is past the key's window and inside the sequence (columns of
    // keys >= sinks are never stored)
    const int lo = key + a.window - qt - 4 * hh, hi = S - qt - 4 * hh;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int off = (i & 3) + 8 * (i >> 2);
      const float p = __builtin_amdgcn_exp2f(a.c * s[i]);
      s[i] = off >= lo && off < hi ? p : 0.f;
      dp[i] = s[i] * dp[i];
    }
    const bf16x8 p0 = pack8_bf(s, 0), p1 = pack8_bf(s, 8), d0 = pack8_bf(dp, 0), d1 = pack8_bf(dp, 8);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int2 to = tr_offsets<D>(dt * 32, lane);
      dv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_read<D>(Ds, 0, to), p0, dv[dt], 0, 0, 0);
      dv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_read<D>(Ds, 16, to), p1, dv[dt], 0, 0, 0);
      dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_read<D>(Qs, 0, to), d0, dk[dt], 0, 0, 0);
      dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_read<D>(Qs, 16, to), d1, dk[dt], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the slice is read before the next one overwrites it
  }
  // join the waves pairwise: 2 -> 0 and 3 -> 1, then 1 -> 0 (lane = key, d = 32 dt + 8 g4 + 4 hh + e)
  float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int step = 2; step >= 1; step >>= 1) {
    __syncthreads();
    if (wave >= step && wave < 2 * step) {
      float* o = sums + (wave - step) * (SUMS / 4) + lane;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[(dt * 16 + i) * 64] = dk[dt][i];
          o[(DT * 16 + dt * 16 + i) * 64] = dv[dt][i];
        }
    }
    __syncthreads();
    if (wave < step) {
      const float* o = sums + wave * (SUMS / 4) + lane;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          dk[dt][i] += o[(dt * 16 + i) * 64];
          dv[dt][i] += o[(DT * 16 + dt * 16 + i) * 64];
        }
    }
  }
  if (wave == 0 && key < a.sinks) {
    float* fp = a.far + (((long long)pair * a.nfar + part) * a.sinks + key) * 2 * D + 4 * hh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        *reinterpret_cast<float4*>(fp + 32 * dt + 8 * g4) =
            make_float4(dk[dt][4 * g4], dk[dt][4 * g4 + 1], dk[dt][4 * g4 + 2], dk[dt][4 * g4 + 3]);
        *reinterpret_cast<float4*>(fp + D + 32 * dt + 8 * g4) =
            make_float4(dv[dt][4 * g4], dv[dt][4 * g4 + 1], dv[dt][4 * g4 + 2], dv[dt][4 * g4 + 3]);
      }
  }
}

// ---------------------------------------------------------------- dQ (launched first: forms delta)
template <int D>
__global__ __launch_bounds__(256, 2) void sink_dq_kernel(BwdArgs a) {
  constexpr int NCH = D / 8, DSTEPS = D / 16, DT = D / 32;
  constexpr int BQ = 128, BK = 64;
  constexpr int TILE = BK * D * 2;
  // K/V tiles arrive by LDS-DMA (global_load_lds_dwordx4) into two distinct buffer pairs: no staging
  // registers (the register-staged version spilled at D=128) and no ds_write pass
  __shared__ __attribute__((aligned(16))) char Kt0[TILE];
  __shared__ __attribute__((aligned(16))) char Vt0[TILE];
  __shared__ __attribute__((aligned(16))) char Kt1[TILE];
  __shared__ __attribute__((aligned(16))) char Vt1[TILE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // wave-uniform -> scalar branches
  const int hh = lane >> 5, lr = lane & 31;
  const int S = a.S, G = a.H / a.KV;
  const int nqb = (S + BQ - 1) / BQ;
  // heaviest (latest) query blocks first; q heads of one kv group adjacent
  const int qr = blockIdx.x / (a.B * a.H);
  const int rem = blockIdx.x % (a.B * a.H);
  const int b = rem / a.H, hq = rem % a.H;
  const int kvh = hq / G;
  const int qb = nqb - 1 - qr;
  const int q0 = qb * BQ;
  const int qpos = q0 + wave * 32 + lr;
  const bool qvalid = qpos < S;
  const int qrow = min(qpos, S - 1);  // rows past the end work on the last one and store nothing

  bf16x8 qf[DSTEPS], df[DSTEPS];
  {
    const uint16_t* qp = a.q + ((long long)b * S + qrow) * a.q_rs + (long long)hq * D + 8 * hh;
    const uint16_t* dp = a.dout + ((long long)b * S + qrow) * a.do_rs + (long long)hq * D + 8 * hh;
#pragma unroll
    for (int s = 0; s < DSTEPS; ++s) {
      qf[s] = as_bf8(*reinterpret_cast<const uint4*>(qp + 16 * s));
      df[s] = as_bf8(*reinterpret_cast<const uint4*>(dp + 16 * s));
    }
  }
  const long long sidx = ((long long)b * a.H + hq) * S + qrow;
  const float lse = a.lse[sidx];
  const float lse2 = lse * LOG2E;
  // delta = rowsum(dO * O) and the row constants [-delta | -lse/scale] that the dK/dV kernels read
  float dsum = 0.f;
  {
    const uint16_t* op = a.o + ((long long)b * S + qrow) * a.o_rs + (long long)hq * D + 8 * hh;
    const uint8_t* lp = a.olow + ((long long)b * S + qrow) * ((long long)a.H * D) + (long long)hq * D + 8 * hh;
#pragma unroll
    for (int s = 0; s < DSTEPS; ++s) {
      float fd[8];
      const uint4 u = *reinterpret_cast<const uint4*>(op + 16 * s);
      const uint2 w = *reinterpret_cast<const uint2*>(lp + 16 * s);
      const uint32_t hi[4] = {u.x, u.y, u.z, u.w}, lo[2] = {w.x, w.y};
      unpack8(__builtin_bit_cast(uint4, df[s]), fd);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        dsum += with_low_byte(j & 1 ? hi[j >> 1] & 0xffff0000u : hi[j >> 1] << 16, (lo[j >> 2] >> (8 * (j & 3))) & 0xffu) * fd[j];
    }
  }
  dsum += __shfl_xor(dsum, 32, 64);
  const float ndlt = -dsum;
  if (hh == 0 && qvalid) {
    a.delta[sidx] = ndlt;
    a.delta[(long long)a.B * S * a.H + sidx] = -lse / a.scale;
  }

  const int kv_end = min(S, q0 + BQ);
  const int kv_begin = max(0, q0 - a.window + 1) / BK * BK;
  const int nsink = min((a.sinks + BK - 1) / BK, kv_begin / BK);  // tiles of sink keys, as in the forward
  const int ntiles = nsink + (kv_end - kv_begin + BK - 1) / BK;
  auto tile_key = [&](const int t) __attribute__((always_inline)) {
    return t < nsink ? t * BK : kv_begin + (t - nsink) * BK;
  };
  const uint16_t* kbase = a.k + (long long)b * S * a.kv_rs + (long long)kvh * D;
  const uint16_t* vbase = a.v + (long long)b * S * a.kv_rs + (long long)kvh * D;
  constexpr int NGT = TILE / 1024 / 4;  // 1 KiB DMA pieces per wave per matrix
  constexpr int RPG = 1024 / (D * 2);  // rows per piece
  const auto krs = make_rsrc(kbase), vrs = make_rsrc(vbase);
  int vrow[NGT], vcol[NGT];
#pragma unroll
  for (int i = 0; i < NGT; ++i) {
    const int row = (wave * NGT + i) * RPG + lane / NCH, pc = lane % NCH;
    vrow[i] = row * (int)a.kv_rs * 2;
    vcol[i] = ((pc ^ swz(row)) & (NCH - 1)) * 16;
  }
  auto issue = [&](const int kv0, char* kdst, char* vdst) __attribute__((always_inline)) {
    const int last = (S - 1 - kv0) * (int)a.kv_rs * 2;  // rows past the end are read as the last one
    int vo[NGT];
#pragma unroll
    for (int i = 0; i < NGT; ++i) vo[i] = min(vrow[i], last) + vcol[i];
    kv_dma<D, NGT, RPG>(krs, vrs, vo, kv0 * (int)a.kv_rs * 2, kdst, vdst, wave);
  };

  f32x16 dq[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[t][i] = 0.f;
  // the dP^T chains start from -delta, so dS^T = P (dP - delta) needs no per-element add
  f32x16 ndv;
#pragma unroll
  for (int i = 0; i < 16; ++i) ndv[i] = ndlt;

  __builtin_amdgcn_s_waitcnt(0x0F70);  // retire the Q/dO/lse loads before any DMA (vmcnt(0))
  if (ntiles > 0) issue(tile_key(0), Kt0, Vt0);
  auto tile = [&](const int t, const char* Kc, const char* Vc, char* Kn, char* Vn) __attribute__((always_inline)) {
    const int kv0 = tile_key(t);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // this wave's pieces of tile t landed (vmcnt(0))
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();        // ... everyone's; and tile t-1's buffers are free
    if (t + 1 < ntiles) issue(tile_key(t + 1), Kn, Vn);  // flies under this tile's compute
    f32x16 s[2], dp[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kt][i] = 0.f;
      dp[kt] = ndv;
      const int r = kt * 32 + lr;
#pragma unroll
      for (int st = 0; st < DSTEPS; ++st) {
        const u32x4 kv = *reinterpret_cast<const u32x4*>(Kc + lds_off<D>(r, 2 * st + hh));
        const u32x4 vv = *reinterpret_cast<const u32x4*>(Vc + lds_off<D>(r, 2 * st + hh));
        s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kv), qf[st], s[kt], 0, 0, 0);
        dp[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vv), df[st], dp[kt], 0, 0, 0);
      }
    }
    // keep 2 K/V fragment reads in flight against the MFMA chain (deeper ones spill at D=128)
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
    for (int i = 0; i < 4 * DSTEPS - 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kt][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(a.c, s[kt][i], -lse2));
    const int qmin_w = q0 + wave * 32;
    const bool need_mask = kv0 + BK - 1 > qmin_w || (qmin_w + 31 - kv0 >= a.window && kv0 + BK > a.sinks);
    if (need_mask) {  // wave-uniform; selects inside
      const int base = kv0 + 4 * hh;
      const int hi = qrow - base, lo = qrow - a.window + 1 - base, snk = a.sinks - base;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int off = kt * 32 + (i & 3) + 8 * (i >> 2);
          s[kt][i] = ((off >= lo || off < snk) && off <= hi) ? s[kt][i] : 0.f;
        }
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[kt][i] = s[kt][i] * dp[kt][i];  // dS^T
    bf16x8 sb[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) sb[ks] = pack8_bf(dp[ks >> 1], 8 * (ks & 1));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      bf16x8 ka[4];
      const int2 to = tr_offsets<D>(dt * 32, lane);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) ka[ks] = tr_read<D>(Kc, 16 * ks, to);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) dq[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[ks], sb[ks], dq[dt], 0, 0, 0);
    }
  };
  for (int t = 0; t < ntiles; t += 2) {
    tile(t, Kt0, Vt0, Kt1, Vt1);
    if (t + 1 < ntiles) tile(t + 1, Kt1, Vt1, Kt0, Vt0);
  }
  if (!qvalid) return;
  uint16_t* op = a.dq + ((long long)b * S + qrow) * a.dq_rs + (long long)hq * D;
  if constexpr (D == 128) {
    if (a.rcos) rope_inv_rows<DT>(dq, a, (long long)b * S + qrow, hh);
  }
  store_rows<DT>(op, dq, a.scale, hh, true);
}

template <int D, bool GRAD>
void launch_fwd(const FwdArgs& a, long long blocks, bool two, hipStream_t stream) {
  if (two) hipLaunchKernelGGL((sink_fwd_kernel<D, GRAD, 2>), dim3((unsigned)blocks), dim3(128 * WAVES), 0, stream, a);
  else hipLaunchKernelGGL((sink_fwd_kernel<D, GRAD, 1>), dim3((unsigned)blocks), dim3(64 * WAVES), 0, stream, a);
}

}  // namespace

extern "C" int ftc_sink_fwd(const void* q, const void* k, const void* v, void* o, void* olow, float* lse, int B, int S, int H, int KV,
                            int D, long long q_rs, long long kv_rs, long long o_rs, float scale, int window, int sinks,
                            hipStream_t stream) {
  // the rows of one (batch, kv head) are addressed with 32-bit buffer offsets; every row starts on 16 bytes
  if (B < 1 || S < 1 || KV < 1 || H % KV != 0 || (D != 128 && D != 64) || window < 1 || sinks < 0 ||
      ((q_rs | kv_rs | o_rs) & 7) || (long long)S * kv_rs * 2 >= (1LL << 31))
    return -1;
  const int BQ = 32 * WAVES;
  FwdArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (uint16_t*)o, (uint8_t*)olow, lse, q_rs,
            kv_rs, o_rs, B, S, H, KV, (S + BQ - 1) / BQ, scale * LOG2E, window < S ? window : S, sinks < S ? sinks : S};
  const long long blocks = (long long)a.nqb * B * H;
  if (blocks > 0x7fffffffLL) return -1;
  // One group where the blocks fill the chip, two where each has a CU to itself and the sequence is longer than a block (in
  // one block of queries there are at most two tiles to share) (one group, two groups, us): 1 x 1000 tokens, 32 / 8 heads x 128 (256 blocks), window 999: 23.5, 19.9; 512: 20.1, 18.3; 16: 11.8, 11.7;
  // 1 x 1001, 8 / 2 heads, window 256 (64 blocks): 15.0, 14.4; 320 blocks, window 512: 21.6, 21.5; 512 blocks: 35.7, 42.8;
  // 1 x 100, 8 heads: 6.8, 7.7.
  const bool two = blocks <= 256 && S > BQ;
  if (D == 128)
    olow ? launch_fwd<128, true>(a, blocks, two, stream) : launch_fwd<128, false>(a, blocks, two, stream);
  else
    olow ? launch_fwd<64, true>(a, blocks, two, stream) : launch_fwd<64, false>(a, blocks, two, stream);
  return (int)hipGetLastError();
}

// Parts of the sink keys' far queries (0: no query is past a sink key's window)
static int far_parts(int B, int S, int H, int KV, int window, int sinks) {
  const int n = sinks < S ? sinks : S;
  if (n < 1 || window >= S) return 0;
  const long long slices = ((long long)(S + 31) / 32 - window / 32) * (H / KV);
  const long long pairs = (long long)B * KV * ((n + 31) / 32);
  const long long p = (512 + pairs - 1) / pairs, most = (slices + FAR_WAVES - 1) / FAR_WAVES;  // a slice a wave at least
  const long long r = p < most ? p : most;
  return (int)(r < 1 ? 1 : r);
}

// Parts that a key block's sweep is split into where there are few blocks: one workgroup a CU, at least 4 slices a part.
// Measured against 1 to 32 parts (whole backward): 1 x 2048 tokens, 32 / 8 heads x 128, window 512 (64 blocks): 4 parts
// 139 us, 3 145, 6 168, unsplit 247; 1 x 4096, window 1024 (128 blocks): 2 parts 310, 3 366, unsplit 438; 1 x 1001, 8 / 2
// heads, window 256 (8 blocks): 16 parts 62, 32 64, unsplit 146; 144 blocks: 2 parts 59, unsplit 53.
static int key_parts(int B, int S, int H, int KV, int D, int window) {
  const long long blocks = (long long)B * KV * ((S + 255) / 256);
  const int rows = D == 128 ? 32 : 64;  // a slice
  const long long span = 255LL + window < S ? 255 + window : S, slices = (span + rows - 1) / rows * (H / KV);
  const long long p = 256 / blocks, most = slices / 4, r = p < most ? p : most;
  return (int)(r < 1 ? 1 : r);
}
struct Ws {
  int nfar, kparts;
  long long far, ksum, total;  // floats: [-delta | -lse/scale], far sums, part sums
};
static Ws bwd_ws(int B, int S, int H, int KV, int D, int window, int sinks) {
  Ws w;
  const long long n = sinks < S ? sinks : S;
  w.nfar = far_parts(B, S, H, KV, window, sinks);
  w.kparts = key_parts(B, S, H, KV, D, window);
  w.far = (2LL * B * H * S + 3) / 4 * 4;
  w.ksum = w.far + (long long)B * KV * w.nfar * n * 2 * D;
  w.total = w.ksum + (w.kparts > 1 ? (long long)B * KV * w.kparts * S * 2 * D : 0);
  return w;
}
extern "C" long long ftc_sink_bwd_workspace(int B, int S, int H, int KV, int D, int window, int sinks) {
  return bwd_ws(B, S, H, KV, D, window, sinks).total;
}

extern "C" int ftc_sink_bwd(const void* q, const void* k, const void* v, const void* o, const void* olow, const void* dout,
                            const float* lse, void* dq, void* dk, void* dv, float* workspace, int B, int S, int H, int KV, int D,
                            long long q_rs, long long kv_rs, long long o_rs, long long do_rs, long long dq_rs,
                            long long dkv_rs, float scale, int window, int sinks, const float* rope_cos,
                            const float* rope_sin, const int* rope_pos, hipStream_t stream) {
  if (B < 1 || S < 1 || KV < 1 || H % KV != 0 || (D != 128 && D != 64) || window < 1 || sinks < 0) return -1;
  if ((q_rs | kv_rs | o_rs | do_rs | dq_rs | dkv_rs) & 7) return -1;  // every row starts on 16 bytes
  if (rope_cos && (D != 128 || !rope_sin || ((reinterpret_cast<uintptr_t>(rope_cos) |
                                               reinterpret_cast<uintptr_t>(rope_sin)) & 15)))
    return -1;
  // one batch's Q / dO / K / V rows and the row constants are addressed with 32-bit buffer offsets
  const long long max_rs = q_rs > do_rs ? (q_rs > kv_rs ? q_rs : kv_rs) : (do_rs > kv_rs ? do_rs : kv_rs);
  if ((long long)S * max_rs * 2 >= (1LL << 31) || 2LL * B * H * S * 4 >= (1LL << 31)) return -1;
  const Ws w = bwd_ws(B, S, H, KV, D, window, sinks);
  const int nfar = w.nfar;
  BwdArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (const uint16_t*)o, (const uint16_t*)dout,
            (const uint8_t*)olow, lse, workspace, (uint16_t*)dq, (uint16_t*)dk, (uint16_t*)dv, q_rs, kv_rs, o_rs, dq_rs, dkv_rs, do_rs,
            B, S, H, KV, scale, scale * LOG2E, window < S ? window : S, sinks < S ? sinks : S,
            nfar ? workspace + w.far : nullptr, nfar, workspace + w.ksum, w.kparts, rope_cos, rope_sin, rope_pos};
  const dim3 g_kv(B * KV * ((S + 255) / 256) * w.kparts), g_q(B * H * ((S + 127) / 128));
  const dim3 g_far(B * KV * nfar * ((a.sinks + 31) / 32));
  const dim3 g_join((unsigned)(((long long)B * KV * S * (D / 8) + 255) / 256));
  // dQ first: it writes the row constants that the other two read
  if (D == 128) {
    hipLaunchKernelGGL((sink_dq_kernel<128>), g_q, dim3(256), 0, stream, a);
    if (nfar) hipLaunchKernelGGL((sink_far_kernel<128>), g_far, dim3(64 * FAR_WAVES), 0, stream, a);
    if (w.kparts > 1) {
      hipLaunchKernelGGL((sink_dkdv_kernel<128, 1, true>), g_kv, dim3(512), 0, stream, a);
      hipLaunchKernelGGL((sink_join_kernel<128>), g_join, dim3(256), 0, stream, a);
    } else {
      hipLaunchKernelGGL((sink_dkdv_kernel<128, 1, false>), g_kv, dim3(512), 0, stream, a);
    }
  } else {
    hipLaunchKernelGGL((sink_dq_kernel<64>), g_q, dim3(256), 0, stream, a);
    if (nfar) hipLaunchKernelGGL((sink_far_kernel<64>), g_far, dim3(64 * FAR_WAVES), 0, stream, a);
    if (w.kparts > 1) {
      hipLaunchKernelGGL((sink_dkdv_kernel<64, 2, true>), g_kv, dim3(512), 0, stream, a);
      hipLaunchKernelGGL((sink_join_kernel<64>), g_join, dim3(256), 0, stream, a);
    } else {
      hipLaunchKernelGGL((sink_dkdv_kernel<64, 2, false>), g_kv, dim3(512), 0, stream, a);
    }
  }
  return (int)hipGetLastError();
}
