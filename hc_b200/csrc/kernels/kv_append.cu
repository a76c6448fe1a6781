// New keys and values into the paged 8-bit cache, one scale per block of tokens and
// head:
//
//   need  = max |x| over the block's new tokens * fl(1 / peak)   (e4m3: the next power of two)
//   s     = max(scale of the block's earlier tokens, need)
//   new   = round(x / s);  earlier tokens, where s grew: round(q * (old / s))
//
// A block without earlier tokens starts from the new ones alone.  With e4m3 the scales
// are powers of two, so that a growing scale moves exponents only (exact until a value
// reaches the subnormals); int8 is rounded again when its scale grows.  Infinities take
// the largest finite value, they do not enter the scale (in a block of nothing but zeros
// and infinities they count as NaN); NaN is stored as 0 in int8 and as NaN in e4m3.  Every step is one correctly rounded fp32 operation, so the stored
// bytes are determined by the inputs alone.
//
// HBM bound (2 bytes read and 1 written per element), for one new token per sequence
// latency bound.  A CTA owns one (sequence, block, head) of keys or of values: it reads
// the new rows twice, the second time from L1, and nobody else writes its bytes.
#include "kv_params.h"
#include "serving_math.cuh"

using namespace hcs;

namespace {

struct AppendParams {
  HcKvCacheDev cache;
  HcKvPlaceDev place;
  const __nv_bfloat16 *k, *v;    // [tokens, heads, dim]
  long long tokenStride, headStride;   // of k, elements
  long long tokenStrideV, headStrideV; // of v
  int touched; // blocks per sequence the grid covers
  int vec;     // 16-byte aligned rows of k and v
};

struct Eight {
  float v[8];
};

__device__ __forceinline__ Eight loadEight(const __nv_bfloat16 *p, int vec) {
  Eight e;
  if (vec) {
    const uint4 r = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e.v[2 * i] = __uint_as_float(w[i] << 16);
      e.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      e.v[i] = __bfloat162float(p[i]);
  }
  return e;
}

// Smallest power of two that is not below x (x >= 0, finite), as a float; 0 for 0.
__device__ __forceinline__ float powerAbove(float x) {
  const uint32_t bits = __float_as_uint(x);
  if (bits == 0)
    return 0.0f;
  if (bits < 0x00800000u) // below the smallest normal number
    return __uint_as_float(0x00800000u);
  return __uint_as_float((bits + 0x007fffffu) & 0x7f800000u);
}

template <class Q> __device__ __forceinline__ void appendBlock(const AppendParams &p) {
  __shared__ float scratch[4];
  const HcKvCacheDev &c = p.cache;
  const int seq = int(blockIdx.x) / p.touched, nth = int(blockIdx.x) % p.touched;
  const int head = int(blockIdx.y), values = int(blockIdx.z);
  const int tid = int(threadIdx.x), threads = int(blockDim.x);

  const HcKvSpan s = hcKvLoadSpan(p.place, c.block, seq);
  const int b = s.first / c.block + nth;
  const int base = b * c.block;
  const int lo = max(s.first, base), hi = min(s.first + s.count, base + c.block);
  if (lo >= hi)
    return;
  const int page = hcKvPageOf(p.place.table[(long long)seq * p.place.tablePitch + b], c.pages);
  if (page < 0)
    return;
  uint8_t *dst = static_cast<uint8_t *>(values ? c.v : c.k) + (long long)page * c.pageStride +
                 (long long)head * c.headStride;
  float *scaleAt =
      (values ? c.vScale : c.kScale) + (long long)page * c.scalePitch + head;
  const long long rowStride = values ? p.tokenStrideV : p.tokenStride;
  const __nv_bfloat16 *src = (values ? p.v : p.k) + (long long)(s.row + lo - s.first) * rowStride +
                             (long long)head * (values ? p.headStrideV : p.headStride);

  const bool held = lo > base;
  float old = held ? *scaleAt : 0.0f;
  old = old > 0.0f ? old : 0.0f;
  const int perRow = c.dim >> 3;
  const int pieces = (hi - lo) * perRow;
  float top = 0.0f;
  for (int i = tid; i < pieces; i += threads) {
    const int r = i / perRow, q = i - r * perRow;
    const Eight e = loadEight(src + r * rowStride + q * 8, p.vec);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float a = fabsf(e.v[k]);
      top = a < __int_as_float(0x7f800000) ? fmaxf(top, a) : top;
    }
  }
  top = blockReduce<true>(top, scratch); // (a barrier: every thread has read the old scale)
  float need = __fmul_rn(top, 1.0f / Peak<Q>::value);
  if constexpr (__is_same(Q, E4M3))
    need = powerAbove(need);
  const float scale = fmaxf(old, need);
  if (tid == 0)
    *scaleAt = scale;

  if (held && scale > old) {
    const float ratio = __fdiv_rn(old, scale);
    const int words = (lo - base) * (c.dim >> 2);
    const int wordsPerRow = c.dim >> 2;
    for (int i = tid; i < words; i += threads) {
      const int r = i / wordsPerRow, w = i - r * wordsPerRow;
      uint32_t *at = reinterpret_cast<uint32_t *>(dst + r * c.tokenStride) + w;
      const uint32_t q = *at;
      *at = quantise4<Q>(dequantise<Q>(q) * ratio, dequantise<Q>(q >> 8) * ratio,
                         dequantise<Q>(q >> 16) * ratio, dequantise<Q>(q >> 24) * ratio);
    }
  }
  // A power of two (every e4m3 scale this kernel makes) divides exactly by its inverse.
  const uint32_t bits = __float_as_uint(scale);
  const bool exact = (bits & 0x007fffffu) == 0 && bits >= 0x01000000u && bits < 0x7e000000u;
  const float inv = exact ? 1.0f / scale : 0.0f;
  for (int i = tid; i < pieces; i += threads) {
    const int r = i / perRow, q = i - r * perRow;
    Eight e = loadEight(src + r * rowStride + q * 8, p.vec);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      e.v[k] = exact || !(scale > 0.0f) ? e.v[k] * inv : __fdiv_rn(e.v[k], scale);
    *reinterpret_cast<uint2 *>(dst + (long long)(lo - base + r) * c.tokenStride + q * 8) =
        make_uint2(quantise4<Q>(e.v[0], e.v[1], e.v[2], e.v[3]),
                   quantise4<Q>(e.v[4], e.v[5], e.v[6], e.v[7]));
  }
}

} // namespace

extern "C" __global__ void __launch_bounds__(128)
    hc_kv_append_i8(const __grid_constant__ AppendParams p) {
  appendBlock<I8>(p);
}
extern "C" __global__ void __launch_bounds__(128)
    hc_kv_append_e4m3(const __grid_constant__ AppendParams p) {
  appendBlock<E4M3>(p);
}
