// Codes and scales of the page-scaled 8-bit KV cache (device side).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace lk {

// KV: 1 = e4m3, 2 = int8 (the numbers of the per-token cache's kv_dtype)

// The page scale of a finite amax >= 0: with amax = f 2^k, f in [1/2, 1), and
// QMAX = 0.875 * 2^9 (e4m3) or 0.9921875 * 2^7 (int8), the exponent is k - 9
// or k - 7, one more when f is above QMAX's fraction.
template <int KV>
__device__ __forceinline__ float page_scale(float amax) {
  constexpr uint32_t FRAC = KV == 1 ? 0x600000u : 0x7E0000u;  // mantissa bits of QMAX
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 126 - (KV == 1 ? 9 : 7) + ((u & 0x7FFFFFu) > FRAC ? 1 : 0);
  e = e < -126 ? -126 : e;  // zero, subnormal and tiny pages
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// x (already divided by the scale) -> code, round to nearest even; beyond the
// range the largest code, NaN 0: a code is always a finite value, so that one
// bad token does not spoil the pages that other requests share with it.
template <int KV>
__device__ __forceinline__ uint8_t page_encode(float x) {
  if (x != x) return 0;
  if constexpr (KV == 1) {
    return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  } else {
    return (uint8_t)(int8_t)fminf(fmaxf(rintf(x), -127.f), 127.f);
  }
}

template <int KV>
__device__ __forceinline__ float page_decode(uint8_t c) {
  if constexpr (KV == 1) return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
  else return (float)(int8_t)c;
}

// n / d = (n * magic) >> shift for 0 <= n < 2^31, with l = ceil(log2 d), shift = 31 + l
// and magic = ceil(2^shift / d): magic * d exceeds 2^shift by less than 2^l, so the product
// exceeds n 2^shift / d by less than 2^31 2^l / d = 2^shift / d.
struct FastDiv {
  uint32_t magic;
  int shift, d;
  explicit FastDiv(int divisor) : magic(0), shift(31), d(divisor) {
    while ((1ll << (shift - 31)) < divisor) ++shift;
    magic = (uint32_t)(((1ull << shift) + divisor - 1) / divisor);
  }
  __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * magic) >> shift); }
};

}  // namespace lk
