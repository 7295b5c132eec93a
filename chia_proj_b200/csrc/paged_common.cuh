// paged_common.cuh -- what the kernels of the paged 8-bit K/V cache share: the
// cache's number formats, its scales, and the bounds checks on what the host
// cannot see (lengths, pages, offsets).
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx.cuh"

namespace chia {

enum CacheType : int { CACHE_E4M3 = 0, CACHE_INT8 = 1 };

constexpr int kStatusBadIndex = 8;   // CHIA_ERR_BAD_INDEX
constexpr int kStatusNoPages = 16;   // CHIA_ERR_NO_PAGES
constexpr int kMinScaleExp = -64;    // the smallest scale is 2^-64

__device__ __forceinline__ void report(int32_t *status, int bits) {
  if (status != nullptr) atomicOr(status, bits);
}

// The kernels of a serving step follow one another on a stream and take some
// microseconds each, so each is launched while the one before still runs
// (programmatic stream serialisation) and waits for its completion, memory
// included, before it touches any: follow() is the first thing a kernel does.
// It lets the next one be set up in turn, whose own wait is for all of this.
__device__ __forceinline__ void follow() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <class... P, class... A>
inline cudaError_t launch_after(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s,
                                A &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }

// The smallest e >= kMinScaleExp with amax <= top * 2^e, from the bits of
// amax = m 2^k (1 <= m < 2): top is 1.75 * 2^8 (e4m3) or 1.984375 * 2^6 (int8),
// so e = k - 8 (k - 6), one more where m exceeds top's own significand. Exact:
// the scale is a power of two, so that a stored value is x 2^-e rounded once,
// and a page whose scale grows is re-expressed by a change of exponent.
template <int CT>
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t b = __float_as_uint(amax);
  constexpr uint32_t M = CT == CACHE_E4M3 ? 0x600000u : 0x7E0000u;
  constexpr int K = CT == CACHE_E4M3 ? 8 : 6;
  const int e = static_cast<int>(b >> 23) - 127 - K + ((b & 0x7fffffu) > M ? 1 : 0);
  return e < kMinScaleExp ? kMinScaleExp : e;
}

// two fp32 values to two e4m3 bytes (to nearest even, saturating; lo in the low byte)
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// two e4m3 bytes to two halves: exact, e4m3's numbers are halves too
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
  return r;
}
__device__ __forceinline__ uint32_t to_int8(float x) {
  const int v = __float2int_rn(x);  // NaN: 0; beyond the range: saturates
  return static_cast<uint32_t>(max(-127, min(127, v))) & 0xffu;
}

// four fp32 values to four bytes of the cache
template <int CT>
__device__ __forceinline__ uint32_t to_cache4(float a, float b, float c, float d) {
  if (CT == CACHE_E4M3) return to_e4m3x2(a, b) | (to_e4m3x2(c, d) << 16);
  return to_int8(a) | (to_int8(b) << 8) | (to_int8(c) << 16) | (to_int8(d) << 24);
}

// four bytes of the cache to two pairs of halves: (0, 1) and (2, 3). int8: a
// byte with its sign bit flipped, u = v + 128, put under the exponent of 1024
// is the half 1024 + u; 1152 less is v, exactly.
template <int CT>
__device__ __forceinline__ void cache4_to_f16(uint32_t four, uint32_t &p01, uint32_t &p23) {
  if (CT == CACHE_E4M3) {
    p01 = e4m3x2_to_f16x2(four & 0xffffu);
    p23 = e4m3x2_to_f16x2(four >> 16);
  } else {
    const uint32_t u = four ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), bias);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), bias);
    p01 = *reinterpret_cast<const uint32_t *>(&x);
    p23 = *reinterpret_cast<const uint32_t *>(&y);
  }
}

__device__ __forceinline__ float2 f16x2_to_float2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// two 16-bit input values (bf16 or fp16) to fp32
template <bool BF16>
__device__ __forceinline__ float2 in16x2_to_float2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return f16x2_to_float2(v);
}

// A value scale as the attention kernels use it: for the softmax kinds its
// logarithm, exact for a power of two and at least -100 (a scale of zero).
template <bool SOFTMAX>
__device__ __forceinline__ float value_factor(float v) {
  if (!SOFTMAX) return v;
  const uint32_t b = __float_as_uint(v);
  if (v < 7.9e-31f) return -100.f;
  return (b & 0x7fffffu) == 0 && b < 0x7f800000u ? static_cast<float>(static_cast<int>(b >> 23) - 127)
                                                 : __log2f(v);
}

// Largest r in [0, n) with off[r] <= x (off rises, off[0] <= x).
__device__ __forceinline__ int last_not_above(const int32_t *off, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

}  // namespace chia
