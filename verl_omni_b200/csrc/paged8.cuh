// e4m3 conversions, page scales and the attention arguments of the 8-bit paged KV cache (no torch dependency).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace vo {
namespace p8 {

constexpr int kMinExp = -100;  // smallest exponent of a page scale: scale and reciprocal stay normal fp32 numbers

// 2^e, e in [-126, 127]
__host__ __device__ __forceinline__ float pow2(int e) {
#ifdef __CUDA_ARCH__
  return __int_as_float((e + 127) << 23);
#else
  union {
    int i;
    float f;
  } u;
  u.i = (e + 127) << 23;
  return u.f;
#endif
}

// smallest 2^e, e >= kMinExp, with amax <= 448 * 2^e.  448 = 0.875 * 2^9: with amax = m 2^x, m in [0.5, 1),
// e is x - 9 where m <= 0.875 and x - 8 above.
__device__ __forceinline__ float scale_of(float amax) {
  const int bits = __float_as_int(amax);
  const int x = (bits >> 23) - 126;                                       // subnormal amax: far below kMinExp
  const int e = x - 9 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);           // fraction of 0.875: 0x600000
  return pow2(e < kMinExp ? kMinExp : e);
}

__device__ __forceinline__ float e4m3_to_float(uint8_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint16_t c) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// nearest e4m3, ties to even; beyond 448 (infinities too) +-448, NaN stays NaN.  x: low byte, y: high byte
__device__ __forceinline__ uint16_t float2_to_e4m3x2(float x, float y) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ void unpack_e4m3x8(uint2 w, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = i < 2 ? w.x : w.y;
    const float2 t = e4m3x2_to_float2((uint16_t)(i & 1 ? u >> 16 : u & 0xffff));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint2 pack_e4m3x8(const float* f) {
  uint2 w;
  w.x = (uint32_t)float2_to_e4m3x2(f[0], f[1]) | ((uint32_t)float2_to_e4m3x2(f[2], f[3]) << 16);
  w.y = (uint32_t)float2_to_e4m3x2(f[4], f[5]) | ((uint32_t)float2_to_e4m3x2(f[6], f[7]) << 16);
  return w;
}

struct AttendArgs {
  const __nv_bfloat16* q;  // [B, Hq, S, hd] with these strides, last dim contiguous
  int64_t qsb, qsh, qss;
  const uint8_t *kp, *vp;  // [pages, Hk, block, hd] e4m3
  const float *ks, *vs;    // [pages, Hk]
  const int *table;        // [B, width]
  const int *lens, *q_lens;
  __nv_bfloat16* out;      // [B, S, Hq, hd]
  int width, pages, block, B, Hq, Hk, rep, S, hd, len_add;
  float scale_log2;
};

// cached rows of sequence b, clamped to the block table's reach
__device__ __forceinline__ int seq_len(const AttendArgs& a, int b) {
  const int64_t cap = (int64_t)a.width * a.block;
  const int64_t len = (int64_t)a.lens[b] + a.len_add;
  return (int)(len < 0 ? 0 : len > cap ? cap : len);
}
__device__ __forceinline__ int seq_q(const AttendArgs& a, int b) {
  if (!a.q_lens) return a.S;
  const int n = a.q_lens[b];
  return n < 0 ? 0 : n > a.S ? a.S : n;
}
// number of leading cached rows that query token s of sequence b sees (0: an empty row)
__device__ __forceinline__ int row_limit(const AttendArgs& a, int b, int s) {
  const int nq = seq_q(a, b);
  if (s >= nq) return 0;
  const int lim = seq_len(a, b) - nq + s + 1;
  return lim < 0 ? 0 : lim;
}

}  // namespace p8
}  // namespace vo
