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
// latency bound.  A warp owns one unit, a (sequence, block, head) of keys or of values: it
// reads the new rows once into registers (what does not fit there again from L1), reduces
// by shuffles alone, and nobody else writes its bytes.  Where that gives the GPU too few
// warps a CTA takes a unit.  Measured: 16 prompts of up to 2048 tokens, 8 heads of 128, to
// e4m3 in 25 us by warps (4.4 TB/s of reads and writes; when both were tried, 31 by warps
// and 38 by CTAs, which spend most instructions on setting up), to int8, which divides, in
// 55; one chunk of 512 tokens in 4.5 us by CTAs (19 by warps); one token in 2.8 us.
#include "kv_params.h"
#include "serving_math.cuh"

#include <type_traits>

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

// Eight bf16 elements as they lie in memory.
struct Raw {
  uint32_t w[4] = {0, 0, 0, 0};
};

__device__ __forceinline__ Raw loadRaw(const __nv_bfloat16 *p, int vec) {
  Raw x;
  if (vec) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    x.w[0] = v.x;
    x.w[1] = v.y;
    x.w[2] = v.z;
    x.w[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x.w[i] = uint32_t(__bfloat16_as_ushort(p[2 * i])) |
               uint32_t(__bfloat16_as_ushort(p[2 * i + 1])) << 16;
  }
  return x;
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

constexpr int kWarps = 4;
constexpr int kHeld = 16; // pieces of 8 elements per lane in registers

// Threads: 32, a warp per unit and four units per CTA; 256, a CTA per unit.
template <class Q, int Threads> __device__ __forceinline__ void appendBlock(const AppendParams &p) {
  __shared__ uint32_t sTop[8];
  const HcKvCacheDev &c = p.cache;
  const int seq = int(blockIdx.x) / p.touched, nth = int(blockIdx.x) - seq * p.touched;
  const int lane = int(threadIdx.x) & (Threads - 1);
  const int unit =
      Threads == 32 ? int(blockIdx.y) * kWarps + (int(threadIdx.x) >> 5) : int(blockIdx.y);
  if (unit >= 2 * c.heads)
    return;
  const int head = unit >> 1, values = unit & 1;
  // The largest over the unit's threads.
  auto largest = [&](uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (Threads > 32) {
      __syncthreads(); // (an earlier result has been read)
      if ((threadIdx.x & 31) == 0)
        sTop[threadIdx.x >> 5] = v;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < Threads / 32; ++w)
        v = max(v, sTop[w]);
    }
    return v;
  };

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
  float *scaleAt = (values ? c.vScale : c.kScale) + (long long)page * c.scalePitch + head;
  const long long rowStride = values ? p.tokenStrideV : p.tokenStride;
  const __nv_bfloat16 *src = (values ? p.v : p.k) + (long long)(s.row + lo - s.first) * rowStride +
                             (long long)head * (values ? p.headStrideV : p.headStride);

  const bool held = lo > base;
  float old = held ? *scaleAt : 0.0f;
  old = old > 0.0f ? old : 0.0f;
  // Pieces of 8 elements, lane by lane along the rows; a lane's next piece by addition.
  const int perRow = c.dim >> 3, rows = hi - lo;
  const int stepRow = Threads / perRow, stepCol = Threads - stepRow * perRow;
  struct At {
    int row, col;
    const __nv_bfloat16 *from;
    uint8_t *to;
  };
  At first{lane / perRow, lane - lane / perRow * perRow, nullptr, nullptr};
  first.from = src + first.row * rowStride + first.col * 8;
  first.to = dst + (long long)(lo - base + first.row) * c.tokenStride + first.col * 8;
  const long long stepFrom = stepRow * rowStride + stepCol * 8, wrapFrom = rowStride - 8 * perRow;
  const long long stepTo = stepRow * c.tokenStride + stepCol * 8, wrapTo = c.tokenStride - 8 * perRow;
  auto advance = [&](At &at) {
    at.row += stepRow;
    at.from += stepFrom;
    at.to += stepTo;
    if (stepCol) {
      at.col += stepCol;
      if (at.col >= perRow) {
        at.col -= perRow;
        ++at.row;
        at.from += wrapFrom;
        at.to += wrapTo;
      }
    }
  };
  auto fetch = [&](const At &at) { return loadRaw(at.from, p.vec); };

  Raw raw[kHeld];
  uint32_t top2 = 0; // magnitudes, as bits: they order like unsigned numbers
  auto magnitude = [&](const Raw &x) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      top2 = __vmaxu2(top2, x.w[k] & 0x7fff7fffu);
  };
  // (One token is one turn: leaving early keeps the code that runs short, and at one
  // token per sequence fetching instructions is what takes the time.)
  // Only rows of 16-byte loads are held, and only for the usual way of storing them is the
  // code unrolled: with every combination of the two unrolled, fetching instructions took
  // half of the time.
  const int turns = p.vec ? (rows * perRow + Threads - 1) / Threads : 0;
  At at = first;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    if (i >= turns)
      break;
    raw[i] = at.row < rows ? loadRaw(at.from, 1) : Raw{};
    advance(at);
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    if (i >= turns)
      break;
    magnitude(raw[i]);
  }
#pragma unroll 1
  for (; at.row < rows; advance(at))
    magnitude(fetch(at));
  uint32_t top16 = max(top2 & 0xffffu, top2 >> 16);
  top16 = largest(top16);
  if (top16 >= 0x7f80u) { // something is not finite: the largest of the others
    uint32_t best = 0;
#pragma unroll 1
    for (at = first; at.row < rows; advance(at)) {
      const Raw x = fetch(at);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t m = (x.w[k >> 1] >> (16 * (k & 1))) & 0x7fffu;
        best = m < 0x7f80u ? max(best, m) : best;
      }
    }
    top16 = largest(best);
  }
  float need = __fmul_rn(__uint_as_float(top16 << 16), 1.0f / Peak<Q>::value);
  if constexpr (__is_same(Q, E4M3))
    need = powerAbove(need);
  const float scale = fmaxf(old, need);
  if constexpr (Threads == 32)
    __syncwarp(); // every lane has read the old scale (in a CTA: before `largest`)
  if (lane == 0)
    *scaleAt = scale;

  if (held && scale > old) {
    const float ratio = __fdiv_rn(old, scale);
    const int wordsPerRow = c.dim >> 2, words = (lo - base) * wordsPerRow;
    for (int i = lane; i < words; i += Threads) {
      const int row = i / wordsPerRow, w = i - row * wordsPerRow;
      uint32_t *word = reinterpret_cast<uint32_t *>(dst + row * c.tokenStride) + w;
      const uint32_t x = *word;
      *word = quantise4<Q>(dequantise<Q>(x) * ratio, dequantise<Q>(x >> 8) * ratio,
                           dequantise<Q>(x >> 16) * ratio, dequantise<Q>(x >> 24) * ratio);
    }
  }
  // A power of two (every e4m3 scale this kernel makes) divides exactly by its inverse;
  // a scale of 0 leaves zeros (and NaN of what is not finite).
  const uint32_t bits = __float_as_uint(scale);
  const bool exact = (bits & 0x007fffffu) == 0 && bits >= 0x01000000u && bits < 0x7e000000u;
  const float inv = exact ? 1.0f / scale : 0.0f;
  const bool product = exact || !(scale > 0.0f);
  auto store = [&](auto multiply, const Raw &x, const At &to) {
    float e[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      e[2 * k] = __uint_as_float(x.w[k] << 16);
      e[2 * k + 1] = __uint_as_float(x.w[k] & 0xffff0000u);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      e[k] = decltype(multiply)::value ? e[k] * inv : __fdiv_rn(e[k], scale);
    *reinterpret_cast<uint2 *>(to.to) =
        make_uint2(quantise4<Q>(e[0], e[1], e[2], e[3]), quantise4<Q>(e[4], e[5], e[6], e[7]));
  };
  at = first;
  if (product) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (i >= turns)
        break;
      if (at.row < rows)
        store(std::true_type{}, raw[i], at);
      advance(at);
    }
#pragma unroll 1
    for (; at.row < rows; advance(at))
      store(std::true_type{}, fetch(at), at);
  } else {
#pragma unroll 1
    for (; at.row < rows; advance(at)) // (the rows come from L1 again)
      store(std::false_type{}, fetch(at), at);
  }
}

} // namespace

#define HC_APPEND(name, Q)                                                                 \
  extern "C" __global__ void __launch_bounds__(128)                                         \
      hc_kv_append_##name##_warp(const __grid_constant__ AppendParams p) {                  \
    appendBlock<Q, 32>(p);                                                                  \
  }                                                                                         \
  extern "C" __global__ void __launch_bounds__(256)                                         \
      hc_kv_append_##name##_cta(const __grid_constant__ AppendParams p) {                   \
    appendBlock<Q, 256>(p);                                                                 \
  }
HC_APPEND(i8, I8)
HC_APPEND(e4m3, E4M3)
