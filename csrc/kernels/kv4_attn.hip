// Decode attention over the 4-bit KV cache (kv4.h): one new query token per sequence, window + sinks.
//
// One wave per (sequence, query head): lanes over the head dimension, an online softmax over the visible
// tokens, one at a time.
#include "kv4.h"

using namespace ftc;

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct Dec4Args {
  const uint16_t* q;
  const uint8_t* data;
  const int* lens;
  uint16_t* out;
  long long q_rs, o_rs;
  int B, H, KV, tiles, max_len, window, sinks;
  float c;  // scale * log2(e)
};

template <int D>
__global__ __launch_bounds__(64) void kv4_decode_kernel(Dec4Args a) {
  using L = Kv4<D>;
  constexpr int E = D / 64;
  const int lane = threadIdx.x;
  const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, kvh = h / (a.H / a.KV);
  const int len = min(a.lens[b], a.max_len);
  const int lo = a.window > 0 ? max(0, len - a.window) : 0;
  const uint8_t* base = a.data + ((long long)b * a.KV + kvh) * a.tiles * L::REC;
  float q[E], o[E], m = -INFINITY, l = 0.f;
  int off, sh, so;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = bf2f(a.q[(long long)b * a.q_rs + (long long)h * D + lane + 64 * e]);
    o[e] = 0.f;
  }
  for (int t = 0; t < len; ++t) {
    if (t < lo && t >= a.sinks) continue;
    const uint8_t* rec = base + (long long)(t / KV4_TILE) * L::REC;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      L::k_at(t % KV4_TILE, lane + 64 * e, &off, &sh, &so);
      s += q[e] * bf2f(*reinterpret_cast<const uint16_t*>(rec + so)) * ((float)((rec[off] >> sh) & 15) - 8.0f);
    }
    s = wave_sum(s) * a.c;
    const float mn = fmaxf(m, s), al = __builtin_amdgcn_exp2f(m - mn), p = __builtin_amdgcn_exp2f(s - mn);
    m = mn;
    l = l * al + p;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      L::v_at(t % KV4_TILE, lane + 64 * e, &off, &sh, &so);
      o[e] = o[e] * al + p * bf2f(*reinterpret_cast<const uint16_t*>(rec + so)) * ((float)((rec[off] >> sh) & 15) - 8.0f);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.out[(long long)b * a.o_rs + (long long)h * D + lane + 64 * e] = f2bf(len > 0 ? o[e] / l : 0.f);
}

}  // namespace

extern "C" int ftc_kv4_store(void* data, const void* k, const void* v, const int* start, const int* count, int B, int KV,
                             int D, int n, int tiles, long long k_bs, long long k_rs, long long v_bs, long long v_rs,
                             int bias, int limit, hipStream_t stream);

extern "C" int ftc_kv4_decode(const void* qkv, void* data, const int* lens, void* out, int B, int H, int KV, int D,
                              int tiles, int max_len, long long q_rs, long long o_rs, float scale, int window, int sinks,
                              hipStream_t stream) {
  if ((D != 64 && D != 128) || B < 1 || KV < 1 || H < KV || H % KV || max_len < 1 || max_len > (long long)tiles * KV4_TILE ||
      (long long)B * H > 0x7fffffffLL)
    return -1;
  const uint16_t* qp = (const uint16_t*)qkv;
  // the new token's row: position lens - 1
  const int rc = ftc_kv4_store(data, qp + (long long)H * D, qp + (long long)(H + KV) * D, lens, nullptr, B, KV, D, 1,
                               tiles, q_rs, 0, q_rs, 0, -1, max_len, stream);
  if (rc) return rc;
  Dec4Args a{qp, (const uint8_t*)data, lens, (uint16_t*)out, q_rs, o_rs, B, H, KV, tiles, max_len, window, sinks,
             scale * LOG2E};
  if (D == 128)
    hipLaunchKernelGGL(kv4_decode_kernel<128>, dim3(B * H), dim3(64), 0, stream, a);
  else
    hipLaunchKernelGGL(kv4_decode_kernel<64>, dim3(B * H), dim3(64), 0, stream, a);
  return (int)hipGetLastError();
}
