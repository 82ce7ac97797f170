// Helpers shared by the flash-attention kernels (flash_attn_fwd.hip, flash_attn_bwd.hip, flash_sink.hip): LDS tile
// images, MFMA operand reads, K / V tile DMA, row stores, the RoPE epilogue.
#pragma once
#include "common.h"

namespace ftc {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

DEV_INLINE int swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
template <int D>
DEV_INLINE int lds_off(int r, int chunk) {  // byte offset of 16-byte chunk `chunk` of row r
  constexpr int NCH = D / 8;
  return r * (D * 2) + 16 * ((chunk ^ swz(r)) & (NCH - 1));
}
DEV_INLINE bf16x8 as_bf8(const uint4& v) { return __builtin_bit_cast(bf16x8, v); }
DEV_INLINE bf16x8 pack8_bf(const f32x16& p, int base) {
  uint4 u;
  u.x = pack_bf2(p[base + 0], p[base + 1]);
  u.y = pack_bf2(p[base + 2], p[base + 3]);
  u.z = pack_bf2(p[base + 4], p[base + 5]);
  u.w = pack_bf2(p[base + 6], p[base + 7]);
  return as_bf8(u);
}
// Epilogue rows (lanes l and l ^ 32 hold the same row, d runs {8 g4 + 4 hh + 0..3} of each 32-wide tile):
// WIDE swaps dword pairs across the lane halves (v_permlane32_swap) so each lane stores 16 contiguous
// d as 2 x dwordx4 per tile instead of 4 x dwordx2 (the store tail is issue-bound; forward: -1 %).
#ifndef BWD_WIDE_STORE
#define BWD_WIDE_STORE 1
#endif
template <int DT>
DEV_INLINE void store_rows(uint16_t* p, const f32x16* acc, float sc, int hh, bool wide) {
  if (BWD_WIDE_STORE && wide) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      uint32_t w[4][2];
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        w[g4][0] = pack_bf2(acc[dt][4 * g4 + 0] * sc, acc[dt][4 * g4 + 1] * sc);
        w[g4][1] = pack_bf2(acc[dt][4 * g4 + 2] * sc, acc[dt][4 * g4 + 3] * sc);
      }
      const auto a0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[2][0], false, false);
      const auto a1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[2][1], false, false);
      const auto b0 = __builtin_amdgcn_permlane32_swap(w[1][0], w[3][0], false, false);
      const auto b1 = __builtin_amdgcn_permlane32_swap(w[1][1], w[3][1], false, false);
      const int d = dt * 32 + 16 * hh;
      *reinterpret_cast<uint4*>(p + d) = make_uint4(a0[0], a1[0], a0[1], a1[1]);
      *reinterpret_cast<uint4*>(p + d + 8) = make_uint4(b0[0], b1[0], b0[1], b1[1]);
    }
  } else {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        uint2 w;
        w.x = pack_bf2(acc[dt][4 * g4 + 0] * sc, acc[dt][4 * g4 + 1] * sc);
        w.y = pack_bf2(acc[dt][4 * g4 + 2] * sc, acc[dt][4 * g4 + 3] * sc);
        *reinterpret_cast<uint2*>(p + dt * 32 + 8 * g4 + 4 * hh) = w;
      }
  }
}
// A operand (32 rows x 16 k, permuted k) via two transposed reads of an LDS image whose rows are k
// and columns are the A rows: elements 0..3 <- image rows kb+4h+0..3, elements 4..7 <- +8.
// tr_offsets() gives the lane's two byte offsets for kb = 0; since the swizzle depends on r & 15 only,
// kb (a multiple of 16) is a plain immediate on top (few live address VGPRs).
template <int D>
DEV_INLINE int2 tr_offsets(int colbase, int lane) {
  const int hh = lane >> 5, gi = (lane >> 4) & 3, li = lane & 15;
  const int trq = li >> 2, trp = li & 3;
  const int col = colbase + 16 * (gi & 1) + 4 * trp;
  const int chunk = col >> 3, half8 = (col & 7) ? 8 : 0;
  const int r1 = 4 * hh + trq;
  return make_int2(lds_off<D>(r1, chunk) + half8, lds_off<D>(r1 + 8, chunk) + half8);
}
template <int D>
DEV_INLINE bf16x8 tr_read(const char* img, int kb, int2 off) {
  s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(img + off.x + kb * D * 2));
  s16x4 v2 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(img + off.y + kb * D * 2));
  s16x8 va = {v1[0], v1[1], v1[2], v1[3], v2[0], v2[1], v2[2], v2[3]};
  return __builtin_bit_cast(bf16x8, va);
}

// Inverse rotation of one row's gradient held as store_rows' accumulators: element i of tile dt is
// d = 32 dt + 8 (i >> 2) + 4 hh + (i & 3), so d and d + 64 are tiles dt and dt + 2 of the same lane.
// (y1, y2) = (u1 c - u2 s, u2 c + u1 s)  =>  (du1, du2) = (g1 c + g2 s, g2 c - g1 s)
template <int DT, typename Args>
DEV_INLINE void rope_inv_rows(f32x16* acc, const Args& a, long long token, int hh) {
  static_assert(DT == 4, "RoPE epilogue: head_dim 128");
  const int pos = a.rpos ? a.rpos[token] : (int)(token % a.S);
  const float* cr = a.rcos + (long long)pos * 64 + 4 * hh;
  const float* sr = a.rsin + (long long)pos * 64 + 4 * hh;
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const float4 c = *reinterpret_cast<const float4*>(cr + 32 * dt + 8 * g4);
      const float4 sn = *reinterpret_cast<const float4*>(sr + 32 * dt + 8 * g4);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * g4 + e;
        const float g1 = acc[dt][i], g2 = acc[dt + 2][i];
        acc[dt][i] = g1 * cc[e] + g2 * ss[e];
        acc[dt + 2][i] = g2 * cc[e] - g1 * ss[e];
      }
    }
}

// max over lanes l and l ^ 32: v_permlane32_swap (gfx950 VALU, one instruction) instead of
// ds_bpermute -- the row max sits on the softmax's dependency chain every tile, and the LDS permute's
// round trip was part of it.
DEV_INLINE float xhalf_max(float v) {
  const auto pr = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float a = __uint_as_float(pr[0]), b = __uint_as_float(pr[1]);
  return a > b ? a : b;  // lane l holds {v_l, v_(l^32)} in some order
}

// one 4-byte-per-lane LDS-DMA piece (the row constants), inline asm like common.h lds_dma16
DEV_INLINE void lds_dma4(__amdgpu_buffer_rsrc_t r, const void* lds, int voff, int soff) {
  const unsigned dst = (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"
      "buffer_load_dword %1, %2, %4 offen lds\n\ts_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(voff), "s"(r), "s"(dst), "s"(soff)
      : "memory");
}

// One slice's LDS-DMA for a dK/dV wave: NG 1 KiB pieces of Q and of dO (lane-linear destinations,
// pre-swizzled per-lane source offsets qvo/dvo) and the 256-byte row-constant piece.  A device-only
// function rather than a lambda in the kernel: the host pass cannot instantiate these builtins.
// SPLIT (a slice of fewer 1 KiB pieces per matrix than waves, D = 64 with 8 waves): each wave DMAs ONE
// piece -- waves [0, P) a piece of Q, waves [P, 2P) the same piece of dO -- so every wave still issues
// the same number of DMA instructions per slice (the counted vmcnt stays wave-uniform).
// QR = 2 (64-row slices): the row constants are two 256-byte pieces (-lse/scale rows, then -delta rows).
template <int D, int NG, int RPG, int QBYTES, bool SPLIT = false, int QR = 1>
DEV_INLINE void dkdv_dma(__amdgpu_buffer_rsrc_t qr, __amdgpu_buffer_rsrc_t dr, __amdgpu_buffer_rsrc_t cr, const int* qvo,
                      const int* dvo, int cvo, int cvo2, int qso, int dso, int cso, char* base, int wave) {
  // inline asm (lds_dma16 / lds_dma4), not the builtin: hipcc tracks builtin LDS-DMA and, unable to prove
  // the ring slots disjoint from the row-constant reads, drained every in-flight slice (vmcnt(0)) at the
  // start of each phase A -- the counted waits in sync_slice are the only ones the ring needs
  if constexpr (SPLIT) {
    constexpr int P = QBYTES / 1024;
    if (wave < P)
      lds_dma16(qr, base + wave * 1024, qvo[0], qso);
    else
      lds_dma16(dr, base + QBYTES + (wave - P) * 1024, dvo[0], dso);
  } else {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int r0 = (wave * NG + i) * RPG;
      lds_dma16(qr, base + r0 * D * 2, qvo[i], qso);
      lds_dma16(dr, base + QBYTES + r0 * D * 2, dvo[i], dso);
    }
  }
  lds_dma4(cr, base + 2 * QBYTES, cvo, cso);
  if constexpr (QR == 2)  // second piece: -delta of the 64 rows (cvo addressed the -lse/scale rows)
    lds_dma4(cr, base + 2 * QBYTES + 256, cvo2, cso);
}

// One K/V tile by LDS-DMA: NGT 1 KiB pieces per matrix per wave (device-only functions: the host pass of
// hipcc cannot instantiate these builtins inside a kernel lambda)
template <int D, int NGT, int RPG>
DEV_INLINE void kv_dma(__amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t vr, const int* voff, int toff, char* kdst,
                    char* vdst, int wave) {
#pragma unroll
  for (int i = 0; i < NGT; ++i) {
    const int r0 = (wave * NGT + i) * RPG;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (__attribute__((address_space(3))) void*)(kdst + r0 * D * 2), 16,
                                             voff[i], toff, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (__attribute__((address_space(3))) void*)(vdst + r0 * D * 2), 16,
                                             voff[i], toff, 0, 0);
  }
}

}  // namespace ftc
