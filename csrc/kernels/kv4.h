// The 4-bit KV cache's record: 32 tokens of one (sequence, kv head), K codes | K scales | V codes | V scales.
//
// A 16-byte chunk of codes is what one lane of a 64-lane wave feeds to v_mfma_f32_16x16x32_bf16, and the
// chunks of a wave lie in lane order (lane = 16 q + r), so every load and store is one linear 1 KiB access:
//   K  chunk of lane (r, q): token t(half, r) = 8 (r >> 2) + 4 half + (r & 3); word j holds d = 32 j + 8 q
//      + 0..7, even d in the low 16 bits (nibbles d/2), odd d in the high 16 bits.
//      D = 128: chunk half = 4 words (j = 0..3), two chunks 1 KiB apart; D = 64: one chunk, words [half][j].
//   V  chunk c of lane (r, q): tokens 8 q + 0..7, d = 64 c + 4 r + 0..3; word p holds tokens 2p (low 16 bits) and
//      2p + 1 (high), nibble i = d0 + i.  The 16 rows r of an MFMA so lie in two value groups, 2 c + (r >> 3).
//      Chunks are 1 KiB apart.
//   scales (bf16): chunk (q, g) of 8 tokens 8 q + 0..7 of value group g = d / 32.
// (x >> 4 i) & 0x000f000f of a word is therefore a pair of adjacent MFMA k elements: two d of one token (K), two
// tokens of one d (V) -- unpacking costs one shift and one and-or a pair and no cross-lane traffic.
// A byte never holds values of two tokens, so tokens are written without reading what is there.
// Codes are stored + 8 (0..15); 16 + code is exactly the bf16 with the code in the top mantissa bits
// (0x4180 | code << 3), which the attention kernel feeds to the MFMA as it is.
#pragma once
#include "common.h"

namespace ftc {

constexpr int KV4_TILE = 32, KV4_GROUP = 32;
template <int D>
struct Kv4 {
  static constexpr int NG = D / 32;                 // value groups (scales) per row
  static constexpr int CH = D / 64;                 // 16-byte chunks per lane and matrix
  static constexpr int CODES = KV4_TILE * D / 2;    // bytes
  static constexpr int SCALES = KV4_TILE * NG * 2;  // bytes
  static constexpr int REC = 2 * (CODES + SCALES);
  static constexpr int WAVES = D == 128 ? 2 : 1;    // waves that write a record or read it back (kv4.hip)
  static constexpr int KC = 0, KS = CODES, VC = CODES + SCALES, VS = 2 * CODES + SCALES;
  // byte offset and shift of one value's code, and byte offset of its scale, within a record
  DEV_INLINE static void k_at(int t, int d, int* off, int* shift, int* soff) {
    const int half = (t >> 2) & 1, r = 4 * (t >> 3) + (t & 3), j = d >> 5, q = (d >> 3) & 3, e = d & 7;
    *off = KC + q * 256 + r * 16 + j * 4 + (D == 128 ? half * 1024 : half * 8) + 2 * (e & 1) + (e >> 2);
    *shift = 4 * ((e >> 1) & 1);
    *soff = KS + ((t >> 3) * NG + j) * 16 + (t & 7) * 2;
  }
  DEV_INLINE static void v_at(int t, int d, int* off, int* shift, int* soff) {
    *off = VC + (d >> 6) * 1024 + (t >> 3) * 256 + ((d & 63) >> 2) * 16 + (t & 7) * 2 + ((d >> 1) & 1);
    *shift = 4 * (d & 1);
    *soff = VS + ((t >> 3) * NG + (d >> 5)) * 16 + (t & 7) * 2;
  }
};

// ---- quantisation: s = -e / 8 with e the group's element of largest magnitude (positive if both signs
// have it), code = clamp(round_half_even(x / s), -8, 7) + 8.
// Magnitude keys as integers: |x| bits << 1 | (x >= 0), two per dword; infinities and NaN order above all.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
DEV_INLINE uint32_t kv4_keys(uint32_t w) {
  return (((w << 1) & 0xfffefffeu) | ((w >> 15) & 0x00010001u)) ^ 0x00010001u;
}
DEV_INLINE uint32_t kv4_max2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// Scale bits and reciprocal from a group's largest key.  e / 8 is exact in bf16 above 2^-100; smaller groups
// are held as zeros (s = 0), non-finite ones get a NaN scale.
DEV_INLINE uint32_t kv4_scale(uint32_t key, float* rinv) {
  const uint32_t mag = (key >> 1) << 16;  // |e| as float bits
  const bool dead = mag < 0x0d800000u;    // 2^-100
  const bool bad = mag >= 0x7f800000u;
  const float s = __uint_as_float(mag) * ((key & 1) ? -0.125f : 0.125f);
  *rinv = (dead || bad) ? 0.f : 1.0f / s;
  return dead ? 0u : bad ? 0x7fc0u : (__float_as_uint(s) >> 16);
}
// code + 8 in 0..15, with 0x4b400000 on top.  x and s have 8-bit significands, so x / s is a half integer or at least
// 2^-10 away from one: the product with the rounded reciprocal (error under 2^-19) is first rounded to a multiple of
// 2^-11 (6144 = 1.5 * 2^12 is added), which puts it exactly on the ties it stands for and moves it over none; the second
// sum, x / s + 1.5 * 2^23 + 8, rounds half to even and leaves the integer in the low bits.
DEV_INLINE uint32_t kv4_code(float x, float rinv) {
  const uint32_t n = __float_as_uint((x * rinv + 6144.0f) + 12576776.0f);
  return n < 0x4b40000fu ? n : 0x4b40000fu;
}
// Codes are packed by shift-and-add; the constants on top add up to a known sum that is taken off at the end.
constexpr uint32_t kv4_top(int s0, int s1, int s2, int s3) {
  return (0x4b400000u << s0) + (0x4b400000u << s1) + (0x4b400000u << s2) + (0x4b400000u << s3);
}
// 8 values of a K word: even d in the low half, odd d in the high half
DEV_INLINE uint32_t kv4_pack_k(const float* f, float rinv) {
  uint32_t w = 0u - kv4_top(0, 4, 8, 12) - kv4_top(16, 20, 24, 28);
#pragma unroll
  for (int e = 0; e < 8; ++e) w += kv4_code(f[e], rinv) << (16 * (e & 1) + 4 * (e >> 1));
  return w;
}
// 4 values of a V half word
DEV_INLINE uint32_t kv4_pack_v(const float* f, float rinv) {
  uint32_t w = 0u - kv4_top(0, 4, 8, 12);
#pragma unroll
  for (int e = 0; e < 4; ++e) w += kv4_code(f[e], rinv) << (4 * e);
  return w;  // (below 2^16: the tops cancel modulo 2^32)
}

// ---- one token's row, quantised by one wave: lanes 0..31 hold K, 32..63 V, 4 values from d = 4 (lane & 31) each
// (D = 64: the first 16 of each half).  A group of 32 is 8 lanes: its maximum takes two quad permutes and a
// mirror of 8.
DEV_INLINE uint32_t kv4_dpp(uint32_t v, int ctrl_is) {  // (a constant in every call)
  return ctrl_is == 1   ? (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true)   // lane ^ 1
         : ctrl_is == 2 ? (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true)   // lane ^ 2
                        : (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true);  // 7 - lane of 8
}
struct Kv4Token {
  uint32_t code;   // K: the whole word of the lane pair's 8 values (both lanes); V: 4 nibbles, natural order
  uint32_t scale;  // bf16 bits of the lane's group
};
DEV_INLINE Kv4Token kv4_token(uint2 u, int lane) {
  uint32_t k2 = kv4_max2(kv4_keys(u.x), kv4_keys(u.y));
  k2 = kv4_max2(k2, kv4_dpp(k2, 1));
  k2 = kv4_max2(k2, kv4_dpp(k2, 2));
  k2 = kv4_max2(k2, kv4_dpp(k2, 3));
  const uint32_t a = k2 & 0xffffu, b = k2 >> 16;
  float rinv;
  Kv4Token t;
  t.scale = kv4_scale(a > b ? a : b, &rinv);
  const float f[4] = {bf_lo(u.x), bf_hi(u.x), bf_lo(u.y), bf_hi(u.y)};
  const uint32_t n = kv4_pack_v(f, rinv);  // nibbles d 0 1 2 3
  const uint32_t kw = ((n & 0xfu) | (n & 0xf00u) >> 4 | (n & 0xf0u) << 12 | (n & 0xf000u) << 8) << (8 * (lane & 1));
  t.code = lane < 32 ? (kw | kv4_dpp(kw, 1)) : n;
  return t;
}
template <int D>
DEV_INLINE void kv4_put_token(uint8_t* rec, int t, const Kv4Token& x, int lane) {
  using L = Kv4<D>;
  const int i5 = lane & 31, d = 4 * i5;
  if (d >= D) return;
  const int so = ((t >> 3) * L::NG + (d >> 5)) * 16 + (t & 7) * 2;
  if (lane < 32) {
    int off, sh, s;
    L::k_at(t, d & ~7, &off, &sh, &s);
    if (!(lane & 1)) *reinterpret_cast<uint32_t*>(rec + off) = x.code;
    if (!(i5 & 7)) *reinterpret_cast<uint16_t*>(rec + L::KS + so) = (uint16_t)x.scale;
  } else {
    int off, sh, s;
    L::v_at(t, d, &off, &sh, &s);
    *reinterpret_cast<uint16_t*>(rec + off) = (uint16_t)x.code;
    if (!(i5 & 7)) *reinterpret_cast<uint16_t*>(rec + L::VS + so) = (uint16_t)x.scale;
  }
}

}  // namespace ftc
