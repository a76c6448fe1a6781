// Root-mean-square norm of the rows of x + residual, with an output in the input's
// type or in 8 bits with scales:
//
//   s = x + residual                      (s is x where there is no residual)
//   y = s / sqrt(mean(s^2) + eps) * gain  (mean over the row)
//   out = y, or per group of columns  scale = max|y| / peak, out = round(y / scale)
//
// s, the sum of squares and y stay in fp32 (the sum that is written out is s rounded
// to the input's type; the norm uses s itself), each value is rounded once.  Rows whose
// squares overflow or vanish are scaled by a power of two and summed again.  peak is
// 127 (int8) or 448 (e4m3).  A group that holds NaN gets the scale NaN, one that
// holds an infinity the scale infinity: no value of such a group comes out finite.
//
// HBM bound: per element x and the residual are read once and the sum and the output
// written once (7 bytes for bf16 with an 8-bit output).  So a row is read into
// registers by one CTA, 8 elements per packet and V packets per thread, all loads
// issued before the first use; the two reductions (squares, then the largest
// magnitude) go through shuffles and one shared-memory exchange each.  A group of
// 32..256 columns is 4..32 neighbouring packets, which neighbouring lanes hold: its
// maximum takes shuffles alone.  Measured: 16384 x 8192 bf16 with residual to e4m3 in 162
// us, 5.8 TB/s, 0.90 of a plain copy's rate, float32 in 257 (5.7 TB/s), bf16 to int8 in
// groups of 128 in 220; 1 x 4096 in 2.2 us, which is one launch.  Odd widths go element by
// element: 16384 x 8191 in 367 us from bf16, 423 from float32, 16384 x 1001 in 103.
#include "serving_math.cuh"

using namespace hcs;

namespace {

struct NormParams {
  const void *x;
  const void *residual; // may be null
  void *summed;         // null with residual; may be residual itself
  const void *gain;
  void *out;
  float *scale; // [rows, groups], 8-bit outputs only
  long long rows, cols;
  long long xPitch, residualPitch, summedPitch, outPitch, scalePitch; // elements
  float eps;
  int group; // columns per scale; 0: the whole row
};

// Eight consecutive elements as floats.
template <class T> struct Packet;
template <> struct Packet<__nv_bfloat16> {
  uint4 raw;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) { raw = loadStream16(p); }
  __device__ __forceinline__ void loadCached(const __nv_bfloat16 *p) {
    raw = __ldg(reinterpret_cast<const uint4 *>(p));
  }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = i < 2 ? raw.x : i < 4 ? raw.y : i < 6 ? raw.z : raw.w;
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
};
template <> struct Packet<float> {
  uint4 a, b;
  __device__ __forceinline__ void load(const float *p) {
    a = loadStream16(p);
    b = loadStream16(p + 4);
  }
  __device__ __forceinline__ void loadCached(const float *p) {
    a = __ldg(reinterpret_cast<const uint4 *>(p));
    b = __ldg(reinterpret_cast<const uint4 *>(p + 4));
  }
  __device__ __forceinline__ float get(int i) const {
    const uint4 &v = i < 4 ? a : b;
    const int j = i & 3;
    return __uint_as_float(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w);
  }
};

__device__ __forceinline__ uint32_t bf16Pair(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}

__device__ __forceinline__ void storeStream16(void *p, uint4 v) {
  asm volatile("st.global.cs.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}

__device__ __forceinline__ void storePacket(__nv_bfloat16 *p, const float (&v)[8]) {
  storeStream16(p, make_uint4(bf16Pair(v[0], v[1]), bf16Pair(v[2], v[3]), bf16Pair(v[4], v[5]),
                              bf16Pair(v[6], v[7])));
}
__device__ __forceinline__ void storePacket(float *p, const float (&v)[8]) {
  storeStream16(p, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]),
                              __float_as_uint(v[2]), __float_as_uint(v[3])));
  storeStream16(p + 4, make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]),
                                  __float_as_uint(v[6]), __float_as_uint(v[7])));
}

// What y is multiplied with to be stored, peak / most (one rounding, where 1 / scale
// would take two); 0 where that is not a finite number: the values of such groups
// (below 2^-118, or not finite) are stored as 0 or NaN.
template <class Out> __device__ __forceinline__ float inverse(float most) {
  return most >= 3.0e-36f && most < __int_as_float(0x7f800000) ? Peak<Out>::value / most : 0.0f;
}

// A power of two for the values of a row whose squares leave float32, 1 for the others:
// where their sum has overflowed (the values then reach 2^64 / sqrt(cols) at least), or is
// so small that squares may have vanished and eps does not stand above them.
__device__ __forceinline__ float rescale(float total, float eps) {
  if (total == __int_as_float(0x7f800000))
    return 1.3234889800848443e-23f; // 2^-76
  if (total < 7.8886090522101181e-31f && eps < 5.2939559203393771e-23f) // 2^-100, 2^-74
    return 1.2676506002282294e30f; // 2^100
  return 1.0f;
}

template <class T> struct Same {};

template <class T, class Out, int Threads, int V>
__device__ __forceinline__ void normRow(const NormParams &p) {
  __shared__ float scratch[2][Threads / 32];
  const T *x = static_cast<const T *>(p.x);
  const T *res = static_cast<const T *>(p.residual);
  T *summed = static_cast<T *>(p.summed);
  const T *gain = static_cast<const T *>(p.gain);
  const int packets = int(p.cols >> 3);
  const int tid = int(threadIdx.x);
  const long long row = blockIdx.x;
  constexpr bool kSame = !__is_same(Out, I8) && !__is_same(Out, E4M3);

  float v[V][8];
  {
    Packet<T> a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = i * Threads + tid;
      if (c < packets) {
        a[i].load(x + row * p.xPitch + c * 8);
        if (res)
          b[i].load(res + row * p.residualPitch + c * 8);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool in = i * Threads + tid < packets;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[i][k] = in ? (res ? a[i].get(k) + b[i].get(k) : a[i].get(k)) : 0.0f;
    }
  }
  float squares = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float part = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      part = fmaf(v[i][k], v[i][k], part);
    squares += part;
  }
  if (summed) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = i * Threads + tid;
      if (c < packets)
        storePacket(summed + row * p.summedPitch + c * 8, v[i]);
    }
  }
  float total = blockReduce<false>(squares, scratch[0]);
  const float pre = rescale(total, p.eps);
  if (pre != 1.0f) { // (the same for the whole CTA)
    squares = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[i][k] *= pre;
        squares = fmaf(v[i][k], v[i][k], squares);
      }
    __syncthreads();
    total = blockReduce<false>(squares, scratch[0]);
  }
  const float rms = __frsqrt_rn(total / float(p.cols) + p.eps * pre * pre);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = i * Threads + tid;
    if (c < packets) {
      Packet<T> g;
      g.loadCached(gain + c * 8);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[i][k] = v[i][k] * rms * g.get(k);
    }
  }
  if constexpr (kSame) {
    T *out = static_cast<T *>(p.out);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = i * Threads + tid;
      if (c < packets)
        storePacket(out + row * p.outPitch + c * 8, v[i]);
    }
  } else {
    float top[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      top[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        top[i] = hc::maxNan(top[i], fabsf(v[i][k]));
    }
    float rowTop = 0.0f;
    if (p.group == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        rowTop = hc::maxNan(rowTop, top[i]);
      rowTop = blockReduce<true>(rowTop, scratch[1]);
    }
    const int lanes = p.group >> 3;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = i * Threads + tid;
      const float most = p.group ? segmentMax(top[i], lanes) : rowTop;
      const float scale = most / Peak<Out>::value;
      const float inv = inverse<Out>(most);
      if (c < packets) {
        uint2 q;
        q.x = quantise4<Out>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
        q.y = quantise4<Out>(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
        asm volatile("st.global.cs.v2.u32 [%0], {%1, %2};" ::"l"(
                         static_cast<uint8_t *>(p.out) + row * p.outPitch + c * 8),
                     "r"(q.x), "r"(q.y)
                     : "memory");
        if (p.group ? tid % lanes == 0 : c == 0)
          p.scale[row * p.scalePitch + (p.group ? c / lanes : 0)] = scale;
      }
    }
  }
}

// Any column count, pitch and alignment, one element at a time: a CTA per row.  With
// `cached` the row's values live in shared memory (cols floats); without, they are
// computed anew from the inputs in every pass, and the sum is written in the last
// one, so that it may go where the residual lies.
template <class T, class Out>
__device__ __forceinline__ void normRowGeneric(const NormParams &p, int cached) {
  extern __shared__ float held[];
  __shared__ float scratch[2][8];
  const T *gain = static_cast<const T *>(p.gain);
  const int tid = int(threadIdx.x);
  const long long row = blockIdx.x;
  const T *x = static_cast<const T *>(p.x) + row * p.xPitch;
  const T *res =
      p.residual ? static_cast<const T *>(p.residual) + row * p.residualPitch : nullptr;
  T *summed = p.summed ? static_cast<T *>(p.summed) + row * p.summedPitch : nullptr;
  constexpr bool kSame = !__is_same(Out, I8) && !__is_same(Out, E4M3);
  auto value = [&](long long c) {
    return cached ? held[c] : float(x[c]) + (res ? float(res[c]) : 0.0f);
  };
  float squares = 0.0f;
  for (long long c = tid; c < p.cols; c += blockDim.x) {
    const float s = res ? float(x[c]) + float(res[c]) : float(x[c]);
    if (cached)
      held[c] = s;
    squares = fmaf(s, s, squares);
  }
  float total = blockReduce<false>(squares, scratch[0]); // (a barrier: held is complete)
  const float pre = rescale(total, p.eps);
  if (pre != 1.0f) { // (the same for the whole CTA)
    squares = 0.0f;
    for (long long c = tid; c < p.cols; c += blockDim.x) {
      const float s = value(c) * pre;
      squares = fmaf(s, s, squares);
    }
    __syncthreads();
    total = blockReduce<false>(squares, scratch[0]);
  }
  const float rms = __frsqrt_rn(total / float(p.cols) + p.eps * pre * pre);
  auto norm = [&](long long c, float s) { return s * pre * rms * float(gain[c]); };
  auto put = [&](long long c, float inv) {
    const float s = value(c);
    const float y = norm(c, s);
    if (summed)
      summed[c] = T(s);
    if constexpr (kSame)
      static_cast<T *>(p.out)[row * p.outPitch + c] = T(y);
    else
      static_cast<uint8_t *>(p.out)[row * p.outPitch + c] = uint8_t(quantise<Out>(y * inv));
  };
  if constexpr (kSame) {
    for (long long c = tid; c < p.cols; c += blockDim.x)
      put(c, 0.0f);
  } else if (p.group == 0) {
    float top = 0.0f;
    for (long long c = tid; c < p.cols; c += blockDim.x)
      top = hc::maxNan(top, fabsf(norm(c, value(c))));
    const float most = blockReduce<true>(top, scratch[1]);
    const float scale = most / Peak<Out>::value;
    const float inv = inverse<Out>(most);
    if (tid == 0)
      p.scale[row * p.scalePitch] = scale;
    for (long long c = tid; c < p.cols; c += blockDim.x)
      put(c, inv);
  } else {
    const int lane = tid & 31, warps = int(blockDim.x) >> 5;
    const long long groups = (p.cols + p.group - 1) / p.group;
    for (long long g = tid >> 5; g < groups; g += warps) {
      const long long end = min((g + 1) * p.group, p.cols);
      float top = 0.0f;
      for (long long c = g * p.group + lane; c < end; c += 32)
        top = hc::maxNan(top, fabsf(norm(c, value(c))));
      const float most = segmentMax(top, 32);
      const float scale = most / Peak<Out>::value;
      const float inv = inverse<Out>(most);
      if (lane == 0)
        p.scale[row * p.scalePitch + g] = scale;
      for (long long c = g * p.group + lane; c < end; c += 32)
        put(c, inv);
    }
  }
}

} // namespace

#define HC_NORM(tname, T, oname, Out, threads, v)                                         \
  extern "C" __global__ void __launch_bounds__(threads)                                   \
      hc_add_rms_norm_##tname##_##oname##_t##threads##_v##v(const __grid_constant__       \
                                                                NormParams p) {           \
    normRow<T, Out, threads, v>(p);                                                       \
  }
#define HC_NORM_SIZES(tname, T, oname, Out)                                               \
  HC_NORM(tname, T, oname, Out, 64, 1)                                                    \
  HC_NORM(tname, T, oname, Out, 128, 1)                                                   \
  HC_NORM(tname, T, oname, Out, 128, 2)                                                   \
  HC_NORM(tname, T, oname, Out, 256, 1)                                                   \
  HC_NORM(tname, T, oname, Out, 256, 2)                                                   \
  HC_NORM(tname, T, oname, Out, 512, 1)                                                   \
  HC_NORM(tname, T, oname, Out, 256, 4)                                                   \
  HC_NORM(tname, T, oname, Out, 512, 2)                                                   \
  HC_NORM(tname, T, oname, Out, 512, 4)                                                   \
  extern "C" __global__ void __launch_bounds__(256)                                       \
      hc_add_rms_norm_##tname##_##oname##_generic(const __grid_constant__ NormParams p,   \
                                                  int cached) {                           \
    normRowGeneric<T, Out>(p, cached);                                                    \
  }
#define HC_NORM_TYPES(tname, T)                                                           \
  HC_NORM_SIZES(tname, T, same, Same<T>)                                                  \
  HC_NORM_SIZES(tname, T, i8, I8)                                                         \
  HC_NORM_SIZES(tname, T, e4m3, E4M3)

HC_NORM_TYPES(bf16, __nv_bfloat16)
HC_NORM_TYPES(f32, float)
