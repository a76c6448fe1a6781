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
// latency bound.  A warp owns one (sequence, block, head) of keys or of values: it reads
// the new rows once into registers (what does not fit there again from L1), reduces by
// shuffles alone, and nobody else writes its bytes.  (A CTA per unit spent two thirds of
// its instructions on setting up: 41 us instead of 26 for 16 prompts of 2048 tokens.)
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

template <class Q> __device__ __forceinline__ void appendBlock(const AppendParams &p) {
  const HcKvCacheDev &c = p.cache;
  const int seq = int(blockIdx.x) / p.touched, nth = int(blockIdx.x) - seq * p.touched;
  const int lane = int(threadIdx.x) & 31;
  const int unit = int(blockIdx.y) * kWarps + (int(threadIdx.x) >> 5);
  if (unit >= 2 * c.heads)
    return;
  const int head = unit >> 1, values = unit & 1;

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
  const int stepRow = 32 / perRow, stepCol = 32 - stepRow * perRow;
  struct At {
    int row, col;
  };
  const At first{lane / perRow, lane - lane / perRow * perRow};
  auto advance = [&](At &at) {
    at.row += stepRow;
    at.col += stepCol;
    if (at.col >= perRow) {
      at.col -= perRow;
      ++at.row;
    }
  };
  auto fetch = [&](const At &at) { return loadRaw(src + at.row * rowStride + at.col * 8, p.vec); };

  Raw raw[kHeld];
  uint32_t top2 = 0; // magnitudes, as bits: they order like unsigned numbers
  auto magnitude = [&](const Raw &x) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      top2 = __vmaxu2(top2, x.w[k] & 0x7fff7fffu);
  };
  // (One token is one turn: leaving early keeps the code that runs short, and at one
  // token per sequence fetching instructions is what takes the time.)
  const int turns = (rows * perRow + 31) >> 5;
  At at = first;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    if (i >= turns)
      break;
    raw[i] = at.row < rows ? fetch(at) : Raw{};
    advance(at);
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    if (i >= turns)
      break;
    magnitude(raw[i]);
  }
  for (; at.row < rows; advance(at))
    magnitude(fetch(at));
  uint32_t top16 = max(top2 & 0xffffu, top2 >> 16);
  top16 = __reduce_max_sync(0xffffffffu, top16);
  if (top16 >= 0x7f80u) { // something is not finite: the largest of the others
    uint32_t best = 0;
    for (at = first; at.row < rows; advance(at)) {
      const Raw x = fetch(at);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t m = (x.w[k >> 1] >> (16 * (k & 1))) & 0x7fffu;
        best = m < 0x7f80u ? max(best, m) : best;
      }
    }
    top16 = __reduce_max_sync(0xffffffffu, best);
  }
  float need = __fmul_rn(__uint_as_float(top16 << 16), 1.0f / Peak<Q>::value);
  if constexpr (__is_same(Q, E4M3))
    need = powerAbove(need);
  const float scale = fmaxf(old, need);
  __syncwarp(); // every lane has read the old scale
  if (lane == 0)
    *scaleAt = scale;

  if (held && scale > old) {
    const float ratio = __fdiv_rn(old, scale);
    const int wordsPerRow = c.dim >> 2, words = (lo - base) * wordsPerRow;
    for (int i = lane; i < words; i += 32) {
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
  uint8_t *out = dst + (long long)(lo - base) * c.tokenStride;
  auto store = [&](const Raw &x, const At &to) {
    float e[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      e[2 * k] = __uint_as_float(x.w[k] << 16);
      e[2 * k + 1] = __uint_as_float(x.w[k] & 0xffff0000u);
    }
    if (product) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        e[k] *= inv;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        e[k] = __fdiv_rn(e[k], scale);
    }
    *reinterpret_cast<uint2 *>(out + to.row * c.tokenStride + to.col * 8) =
        make_uint2(quantise4<Q>(e[0], e[1], e[2], e[3]), quantise4<Q>(e[4], e[5], e[6], e[7]));
  };
  at = first;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    if (i >= turns)
      break;
    if (at.row < rows)
      store(raw[i], at);
    advance(at);
  }
  for (; at.row < rows; advance(at))
    store(fetch(at), at);
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
