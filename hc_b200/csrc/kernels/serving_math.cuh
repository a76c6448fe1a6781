// Shared by the serving kernels (add_rms_norm.cu, gemm_w4.cu, kv_append.cu,
// kv_attention.cu): 8-bit element types, packed loads, warp and CTA reductions.
#pragma once

#include "hc_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace hcs {

struct I8 {};   // two's complement, -127..127 in use
struct E4M3 {}; // 8-bit float: 4 exponent bits (bias 7), 3 fraction bits, largest 448

template <class Q> struct Peak;
template <> struct Peak<I8> {
  static constexpr float value = 127.0f;
};
template <> struct Peak<E4M3> {
  static constexpr float value = 448.0f;
};

// Nearest representable value (ties to even), saturating; NaN becomes 0 (int8) or
// the NaN pattern (e4m3).
template <class Q> __device__ __forceinline__ uint32_t quantise(float v);
template <> __device__ __forceinline__ uint32_t quantise<I8>(float v) {
  const int q = __float2int_rn(fminf(fmaxf(v, -127.0f), 127.0f));
  return uint32_t(v == v ? q : 0) & 0xffu;
}
// Two values into the low and the high byte of a 16-bit result.
__device__ __forceinline__ uint32_t e4m3Pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t quantise<E4M3>(float v) {
  return e4m3Pair(v, 0.0f) & 0xffu;
}

template <class Q>
__device__ __forceinline__ uint32_t quantise4(float a, float b, float c, float d) {
  if constexpr (sizeof(Q) && __is_same(Q, E4M3))
    return e4m3Pair(a, b) | (e4m3Pair(c, d) << 16);
  else
    return quantise<Q>(a) | (quantise<Q>(b) << 8) | (quantise<Q>(c) << 16) |
           (quantise<Q>(d) << 24);
}

template <class Q> __device__ __forceinline__ float dequantise(uint32_t byte);
template <> __device__ __forceinline__ float dequantise<I8>(uint32_t byte) {
  return float(int8_t(byte));
}
template <> __device__ __forceinline__ float dequantise<E4M3>(uint32_t byte) {
  uint32_t h;
  asm("{ .reg .b16 p; cvt.u16.u32 p, %1; cvt.rn.f16x2.e4m3x2 %0, p; }"
      : "=r"(h)
      : "r"(byte & 0xffu));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

__device__ __forceinline__ uint4 loadStream16(const void *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ float warpSum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// log2(2^top * sum) with the error of a logarithm of 1..2, however far top and the sum's
// exponent are from 0: they cancel exactly.
__device__ __forceinline__ float log2Of(float top, float sum) {
  const uint32_t bits = __float_as_uint(sum), e = bits >> 23;
  if (e == 0 || e >= 255) // subnormal or not finite
    return top + __log2f(sum);
  return (top + float(int(e) - 127)) +
         __log2f(__uint_as_float((bits & 0x007fffffu) | 0x3f800000u));
}

// What a block's value scale adds to its scores where the reference of the exponentials
// is chosen: exponential times scale then fits f16 whatever the scales are.  Scales below
// 2^-96, and 0, count as that: their sums of exponentials stay below float32's end, and
// blocks of zeros do not push the others' weights among f16's subnormals.
__device__ __forceinline__ float logOfScale(float scale) {
  const float s = fabsf(scale);
  return s < INFINITY ? fmaxf(__log2f(s), -96.0f) : 0.0f;
}

// Maximum over aligned segments of `width` lanes (a power of two); NaN if any is.
__device__ __forceinline__ float segmentMax(float v, int width) {
  for (int d = width >> 1; d > 0; d >>= 1)
    v = hc::maxNan(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// Over the whole CTA; every thread gets the result.  `scratch`: one float per warp.
// The caller puts a __syncthreads between two uses of one scratch array.
template <bool Max> __device__ __forceinline__ float blockReduce(float v, float *scratch) {
  v = Max ? segmentMax(v, 32) : warpSum(v);
  const int warps = int(blockDim.x) >> 5;
  if ((threadIdx.x & 31) == 0)
    scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = scratch[0];
  for (int w = 1; w < warps; ++w)
    r = Max ? hc::maxNan(r, scratch[w]) : r + scratch[w];
  return r;
}

} // namespace hcs
