// Device helpers of the 8-bit cache: e4m3 / e5m2 conversions, block scales, table lookups with bounds.
#pragma once
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "kv8.h"

namespace lb {

constexpr float KV8_MOST = 3.3895313892515355e38f;   // largest finite bf16 value: infinities count as this

// two e4m3 codes in the low 16 bits, `lo` in the first byte
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ __half2 e4m3x2_to_half2(uint32_t b) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(uint16_t(b)));
  return *reinterpret_cast<__half2*>(&r);
}
__device__ __forceinline__ uint32_t e5m2x2(__half2 h) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<uint32_t*>(&h)));
  return r;
}
// e5m2 is the upper byte of a half
__device__ __forceinline__ __half2 e5m2x2_to_half2(uint32_t b) {
  const uint32_t r = __byte_perm(b, 0, 0x1404);
  return *reinterpret_cast<const __half2*>(&r);
}

// 2^(e - 7) for a largest magnitude in [2^e, 2^(e+1)), at least 2^-60; 0 for 0. A code of the largest magnitude then lies in
// [128, 256]: e4m3 is a floating format, so a power of two costs no precision, and a block whose scale grows keeps its older
// codes bit for bit, apart from those that fall below its smallest normal value.
__device__ __forceinline__ float kv8_scale_of(float amax) {
  if (!(amax > 0.f)) return 0.f;
  const int e = int(__float_as_uint(amax) >> 23) - 127;
  return __uint_as_float(uint32_t(max(e - 7, -60) + 127) << 23);
}
// 1 / scale of a power of two (2^-60 .. 2^120), 0 for 0: the exponent turned round, without a division's code
__device__ __forceinline__ float kv8_inverse(float scale) { return scale > 0.f ? __uint_as_float(0x7f000000u - __float_as_uint(scale)) : 0.f; }
// A value scale joins the exponents of its keys' weights. A scale of 0, nothing but zeros, counts as 2^-80: its keys belong to the
// denominator alone, and with a larger scale they would set the reference that other blocks' weights keep their bits below (with 2^0 a
// block of zeros cost values of 2^-20 a fifth of their size in decode, with 2^-60 a weight of 2^-60 beside it most of its bits). With a
// smaller one their own exponentials would run out of range beside scales above 2^20.
__device__ __forceinline__ float kv8_value_scale(float scale) { return scale > 0.f ? scale : 0x1p-80f; }
__device__ __forceinline__ int kv8_log2(float scale) { return max(-120, min(120, int(__float_as_uint(scale) >> 23) - 127)); }

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A sink (log2) joins a denominator of exponentials relative to 2^top, both then relative to the larger: what the factor returned leaves
// of sums so far. (Relative to `top` alone a sink 2^40 above keys of zero values would be infinite.)
__device__ __forceinline__ float kv8_add_sink(float sk, float& top, float& den) {
  if (top == -INFINITY && den == 0.f) {
    top = sk;
    den = 1.f;
    return 0.f;
  }
  const float m = fmaxf(top, sk), f = ex2(top - m);
  den = den * f + ex2(sk - m);
  top = m;
  return f;
}

// A kernel's shared memory limit is a setting per device: set at its first launch on each.
struct DeviceOnce {
  std::atomic<uint64_t> done{0};
  cudaError_t shared_memory(const void* fn, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
  }
};

}  // namespace lb
