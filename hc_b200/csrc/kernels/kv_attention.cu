// Attention over the paged 8-bit key/value cache:
//
//   out[i] = sum_j p_ij v_j,  p = softmax over the visible j of  scale * q_i . k_j
//
// with k_j = kScale[page(j), head] * K[j] and v_j alike, K and V int8 or e4m3.  Token j
// is visible to the query at position i when j <= i and, with a window, i - j < window;
// a row that sees nothing gives zeros and lse = -inf.
//
// For single tokens and drafts the cache is the traffic: 2 * dim bytes per token and
// key/value head, each read once for all the query rows that share the head.
//   * A warp takes 16 tokens at a time and loads their keys and values straight from
//     HBM into registers, 16 bytes per lane and row in the layout they are stored in.
//     mma.sync m16n8k16 (f16 in, fp32 out) computes S^T = K Q^T with the tokens as the
//     16 rows and 8 query rows as the columns, then O^T += V^T P^T; a sum does not care
//     about the order of its terms, so the head dimension is permuted to what each lane
//     holds, and P only needs an 8 x 8 transpose of halves (movmatrix) in between.
//     Eight query rows fill the MMA: with tcgen05 they would be 8 of 128 rows, and the
//     operands would need a detour through shared memory.
//   * 8-bit values are exact in f16 (int8 by byte permutes, e4m3 by the hardware
//     conversion); q is brought into f16 range by a power of two per row, exact down to
//     2^-14 of the row's largest element; the block's key scale multiplies the fp32
//     scores; its value scale goes into the probabilities before they are rounded to
//     f16: w = 2^11 * exp2(x - m) * vScale, where m follows the running maximum of
//     x + log2(vScale) and is at most 4 behind it, so w <= 2^15 whatever the scales are
//     and the outputs are rescaled a few times per sequence only.  The sum of
//     exp2(x - m), the maxima and the output are fp32; rounding w costs 2^-12 of a term
//     (terms below 2^-25 of the largest lose more, by at most 2^-36 of it).
//   * The tiles (128 tokens: 16 per warp of a CTA) of all (sequence, head, row tile)
//     units stand in one line that is cut into equal shares, one per resident CTA, so a
//     ragged batch is balanced and a single long sequence uses the whole GPU.  A unit
//     that is cut is joined by the last of its CTAs to finish, from partial results in
//     global memory, added in the order of the shares: the result does not depend on
//     which one that is.
#include "kv_params.h"
#include "serving_math.cuh"

using namespace hcs;

namespace {

struct AttentionParams {
  HcKvCacheDev cache;
  HcKvPlaceDev place;
  const __nv_bfloat16 *q; // [tokens, heads * share, dim]
  __nv_bfloat16 *out;
  float *lse; // [tokens, heads * share] or null
  long long qTokenStride, qHeadStride, outTokenStride, outHeadStride, lseStride;
  float scaleLog2; // scale * log2(e)
  int share;       // query heads per key/value head
  int window;      // 0: none
  int rowTiles;    // row tiles that maxNew * share rows can take
  int sixteenths;  // block / 16, and ceil(2^32 / that) for more than one
  uint32_t blockInverse;
  unsigned *counters; // [CTAs], zero between calls
  float *partial;     // [CTAs][2] slots
};

constexpr int kWarps = 8;
constexpr int kTile = 16 * kWarps;
constexpr float kNegInf = -INFINITY;
// The reference that the exponentials are taken against follows the running maximum
// only when that has grown by more than 2^kSlack: probabilities reach 2^kSlack, times
// kWeight they fit f16.
constexpr float kSlack = 4.0f;
constexpr float kWeight = 2048.0f; // 2^(15 - kSlack)

__device__ __forceinline__ void mmaF16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                       uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float exp2Approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t halfPair(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// The low (high) two bytes of w as an f16 pair, exactly.
template <class Q> __device__ __forceinline__ uint32_t widenLow(uint32_t w);
template <class Q> __device__ __forceinline__ uint32_t widenHigh(uint32_t w);
// int8: 0x6400 | u is 1024 + u in f16 for a byte u; the caller flips the sign bits, so
// u = x + 128 and 1152 comes off again.
__device__ __forceinline__ uint32_t sub1152(uint32_t v) {
  const uint32_t bias = 0x64806480u;
  const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&v),
                            *reinterpret_cast<const __half2 *>(&bias));
  return *reinterpret_cast<const uint32_t *>(&d);
}
template <> __device__ __forceinline__ uint32_t widenLow<I8>(uint32_t w) {
  return sub1152(__byte_perm(w, 0x64646464u, 0x4140));
}
template <> __device__ __forceinline__ uint32_t widenHigh<I8>(uint32_t w) {
  return sub1152(__byte_perm(w, 0x64646464u, 0x4342));
}
__device__ __forceinline__ uint32_t widenE4M3(uint16_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(w));
  return r;
}
template <> __device__ __forceinline__ uint32_t widenLow<E4M3>(uint32_t w) {
  return widenE4M3(uint16_t(w));
}
template <> __device__ __forceinline__ uint32_t widenHigh<E4M3>(uint32_t w) {
  return widenE4M3(uint16_t(w >> 16));
}
template <class Q> __device__ __forceinline__ uint32_t prepare(uint32_t w) {
  return __is_same(Q, I8) ? w ^ 0x80808080u : w;
}

template <int DimCap, int NT> struct Shape {
  static constexpr int rows = 8 * NT;
  static constexpr int keyPieces = DimCap / 64;                 // 16 bytes per lane and row
  static constexpr int valueBytes = DimCap == 64 ? 8 : 16;      // per lane, row and piece
  static constexpr int valuePieces = DimCap == 256 ? 2 : 1;
  static constexpr int valueWords = valueBytes / 4;
  static constexpr int mTiles = DimCap / 16;
  static constexpr int qPitch = DimCap + 8; // halves: rows 4 banks apart
  static constexpr int slotFloats = rows * DimCap + 2 * rows;
  // (Shared memory, launched with kWarps * rows * DimCap * 4 bytes: the query rows, and
  // at the end of a segment the warps' partial outputs [warps][rows][DimCap].)
};

// Whole: the head dimension is DimCap.
template <class Q, int DimCap, int NT, bool Whole>
__device__ __forceinline__ void attend(const AttentionParams &p) {
  using S = Shape<DimCap, NT>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ long long sPrefix[kWarps * 32];
  __shared__ float sRowFactor[S::rows];
  __shared__ float sMax[kWarps][S::rows], sSum[kWarps][S::rows];
  __shared__ float sFactor[kWarps][S::rows], sTop[S::rows], sTotal[S::rows];
  __shared__ long long sWarpTotal[kWarps];
  __shared__ int sLast;
  __half *sQ = reinterpret_cast<__half *>(smem);
  float *sOut = reinterpret_cast<float *>(smem);

  const HcKvCacheDev &c = p.cache;
  const int tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  // This lane's bytes within 16 tokens (a page spans less than 2^31 bytes).
  const uint32_t kOffset = uint32_t(g) * uint32_t(c.tokenStride) + 16 * t;
  const uint32_t vOffset = uint32_t(2 * t) * uint32_t(c.tokenStride) + S::valueBytes * g;

  // Tiles of one unit of a sequence, and its row tiles.
  auto tilesOf = [&](int seq, HcKvSpan &s, int &begin, int &rowTiles) -> int {
    s = hcKvLoadSpan(p.place, c.block, seq);
    rowTiles = (s.count * p.share + S::rows - 1) / S::rows;
    begin = 0;
    if (p.window > 0)
      begin = max(0, s.first - p.window + 1) & ~15;
    const int end = s.first + s.count;
    return s.count > 0 && end > begin ? (end - begin + kTile - 1) / kTile : 0;
  };

  // The line's length, and the sequence in which this CTA's share begins.
  long long total = 0;
  bool placeless = false; // rows without a place in the cache
  for (int base = 0; base < p.place.seqs; base += 256) {
    long long mine = 0;
    if (base + tid < p.place.seqs) {
      HcKvSpan s;
      int begin, rt;
      const int n = tilesOf(base + tid, s, begin, rt);
      mine = (long long)n * rt * c.heads;
      placeless = placeless || s.count != s.allCount;
    }
    // Inclusive scan over the CTA.
    long long scan = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= d)
        scan += other;
    }
    if (lane == 31)
      sWarpTotal[warp] = scan;
    __syncthreads();
    long long before = total;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp)
        before += sWarpTotal[w];
      total += sWarpTotal[w];
    }
    sPrefix[tid] = before + scan; // inclusive, from the start of the line
    __syncthreads();
  }
  if (blockIdx.x == 0 && __syncthreads_or(placeless)) {
    // They see nothing: zeros.
    const int heads = c.heads * p.share;
    for (int seq = 0; seq < p.place.seqs; ++seq) {
      const HcKvSpan s = hcKvLoadSpan(p.place, c.block, seq);
      for (int row = s.allRow; row < s.allRow + s.allCount; ++row) {
        if (row >= s.row && row < s.row + s.count)
          continue;
        for (int i = tid; i < heads * c.dim; i += 256) {
          const int h = i / c.dim, d = i - h * c.dim;
          p.out[row * p.outTokenStride + h * p.outHeadStride + d] = __float2bfloat16_rn(0.0f);
          if (d == 0 && p.lse)
            p.lse[row * p.lseStride + h] = kNegInf;
        }
      }
    }
  }
  const long long shares = min((long long)gridDim.x, total);
  if ((long long)blockIdx.x >= shares)
    return;
  long long at = hcKvShareBegin(blockIdx.x, total, shares);
  const long long shareEnd = hcKvShareBegin((long long)blockIdx.x + 1, total, shares);
  int seq = 0;
  long long seqBegin = 0; // where that sequence begins in the line
  if (p.place.seqs <= 256) {
    // sPrefix holds the whole line: count the sequences that end at or before `at`.
    const int done = tid < p.place.seqs && sPrefix[tid] <= at;
    seq = __syncthreads_count(done);
    seqBegin = seq > 0 ? sPrefix[seq - 1] : 0;
  } else {
    for (int base = 0;; base += 256) {
      HcKvSpan s;
      int begin, rt;
      long long mine = 0;
      if (base + tid < p.place.seqs)
        mine = (long long)tilesOf(base + tid, s, begin, rt) * rt * c.heads;
      long long scan = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long other = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d)
          scan += other;
      }
      __syncthreads();
      if (lane == 31)
        sWarpTotal[warp] = scan;
      __syncthreads();
      long long before = seqBegin, all = seqBegin;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp)
          before += sWarpTotal[w];
        all += sWarpTotal[w];
      }
      sPrefix[tid] = before + scan;
      __syncthreads();
      if (all > at || base + 256 >= p.place.seqs) {
        const int done = base + tid < p.place.seqs && sPrefix[tid] <= at;
        const int n = __syncthreads_count(done);
        seq = base + n;
        seqBegin = n > 0 ? sPrefix[n - 1] : seqBegin;
        break;
      }
      seqBegin = all;
    }
  }

  while (at < shareEnd) {
    HcKvSpan span;
    int kvBegin, rowTiles;
    int unitTiles = tilesOf(seq, span, kvBegin, rowTiles);
    const long long inSeq = (long long)unitTiles * rowTiles * c.heads;
    if (at - seqBegin >= inSeq) { // next sequence (those without tiles are passed over)
      seqBegin += inSeq;
      ++seq;
      continue;
    }
    const int unit = int((at - seqBegin) / unitTiles);
    const int head = unit / rowTiles, rowTile = unit - head * rowTiles;
    const long long unitBegin = seqBegin + (long long)unit * unitTiles;
    const int tile0 = int(at - unitBegin);
    const int tile1 = int(min((long long)unitTiles, shareEnd - unitBegin));
    const int row0 = rowTile * S::rows;
    const int rowsHere = min(S::rows, span.count * p.share - row0);
    const int *table = p.place.table + (long long)seq * p.place.tablePitch;

    // ---- query rows into shared memory as f16, a power of two per row ----------------
    __syncthreads(); // the previous segment's shared memory has been read
    for (int r = warp; r < S::rows; r += kWarps) {
      float v[DimCap / 32];
      float top = 0.0f;
      if (r < rowsHere) {
        const int qi = (row0 + r) / p.share, gh = (row0 + r) - qi * p.share;
        const __nv_bfloat16 *src = p.q + (long long)(span.row + qi) * p.qTokenStride +
                                   (long long)(head * p.share + gh) * p.qHeadStride;
#pragma unroll
        for (int i = 0; i < DimCap / 32; ++i) {
          const int d = i * 32 + lane;
          v[i] = d < c.dim ? __bfloat162float(src[d]) : 0.0f;
          top = fmaxf(top, fabsf(v[i]));
        }
        top = segmentMax(top, 32);
      } else {
#pragma unroll
        for (int i = 0; i < DimCap / 32; ++i)
          v[i] = 0.0f;
      }
      // 2^e <= top < 2^(e+1); zero, subnormal and infinite rows keep their values.
      const int e = int(__float_as_uint(top) >> 23);
      const bool plain = e == 0 || e == 255;
      const float down = plain ? 1.0f : __uint_as_float(uint32_t(max(254 - e, 1)) << 23);
      const float up = plain ? 1.0f : 1.0f / down;
      if (lane == 0)
        sRowFactor[r] = p.scaleLog2 * up;
#pragma unroll
      for (int i = 0; i < DimCap / 32; ++i)
        sQ[r * S::qPitch + i * 32 + lane] = __float2half_rn(v[i] * down);
    }
    __syncthreads();

    // ---- this lane's columns: query rows 2t and 2t + 1 of each n-tile ------------------
    float colFactor[NT][2], m[NT][2], l[NT][2];
    int seenHi[NT][2], seenLo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = n * 8 + 2 * t + h;
        colFactor[n][h] = sRowFactor[r];
        m[n][h] = kNegInf;
        l[n][h] = 0.0f;
        const int qi = min(row0 + r, row0 + rowsHere - 1) / p.share;
        seenHi[n][h] = span.first + qi;
        seenLo[n][h] = p.window > 0 ? max(0, span.first + qi - p.window + 1) : 0;
      }
    const int firstPos = span.first + row0 / p.share;
    const int lastPos = span.first + (row0 + rowsHere - 1) / p.share;
    // Positions that every row sees: [allLo, firstPos].
    const int allLo = p.window > 0 ? max(0, lastPos - p.window + 1) : 0;
    const int anyLo = p.window > 0 ? max(0, firstPos - p.window + 1) : 0;

    const uint8_t *kHead = static_cast<const uint8_t *>(c.k) + (long long)head * c.headStride;
    const uint8_t *vHead = static_cast<const uint8_t *>(c.v) + (long long)head * c.headStride;
    const float *kScales = c.kScale + head, *vScales = c.vScale + head;

    float o[S::mTiles][NT][4];
#pragma unroll
    for (int i = 0; i < S::mTiles; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          o[i][n][k] = 0.0f;

    // ---- the warp's 16 tokens of each tile -----------------------------------------------
    auto posOf = [&](int tile) { return kvBegin + tile * kTile + warp * 16; };
    // Blocks are multiples of 16 tokens: the quotient of two small numbers by a product.
    auto blockOf = [&](int pos) {
      return p.sixteenths == 1 ? pos >> 4
                               : int(__umulhi(uint32_t(pos) >> 4, p.blockInverse));
    };
    auto pageAt = [&](int tile) -> int {
      const int pos = posOf(tile);
      // Tokens that no row of this unit sees are passed over like missing pages.
      if (tile >= tile1 || pos > lastPos || pos + 15 < anyLo)
        return -1;
      return hcKvPageOf(__ldg(table + blockOf(pos)), c.pages);
    };
    // All 16 rows lie inside the page, written or not: what is not visible is masked.
    uint4 kReg[2][S::keyPieces];
    uint32_t vReg[4][S::valuePieces][S::valueWords];
    float kScale = 0.0f, vScale = 0.0f;
    auto loadKeys = [&](int tile, int page) {
      if (page < 0)
        return;
      const int pos = posOf(tile);
      const uint8_t *k = kHead + (long long)page * c.pageStride +
                         uint32_t(pos - blockOf(pos) * c.block) * uint32_t(c.tokenStride);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < S::keyPieces; ++j)
          kReg[h][j] = Whole || 64 * j + 16 * t < c.dim
                           ? loadStream16(k + (h ? kOffset + 8 * uint32_t(c.tokenStride) : kOffset) +
                                          64 * j)
                           : make_uint4(0, 0, 0, 0);
      kScale = __ldg(kScales + (long long)page * c.scalePitch);
    };
    auto loadValues = [&](int tile, int page) {
      if (page < 0)
        return;
      const int pos = posOf(tile);
      const uint8_t *v = vHead + (long long)page * c.pageStride +
                         uint32_t(pos - blockOf(pos) * c.block) * uint32_t(c.tokenStride);
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int j = 0; j < S::valuePieces; ++j) {
          const uint8_t *at =
              v + (vOffset + ((h & 1) + 8 * (h >> 1)) * uint32_t(c.tokenStride)) + 128 * j;
          const bool in = Whole || 128 * j + S::valueBytes * g < c.dim;
          if constexpr (S::valueBytes == 16) {
            const uint4 w = in ? loadStream16(at) : make_uint4(0, 0, 0, 0);
            vReg[h][j][0] = w.x;
            vReg[h][j][1] = w.y;
            vReg[h][j][2] = w.z;
            vReg[h][j][3] = w.w;
          } else {
            uint2 w = make_uint2(0, 0);
            if (in)
              asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
                           : "=r"(w.x), "=r"(w.y)
                           : "l"(at));
            vReg[h][j][0] = w.x;
            vReg[h][j][1] = w.y;
          }
        }
      vScale = __ldg(vScales + (long long)page * c.scalePitch);
    };

    int page = pageAt(tile0), nextPage = pageAt(tile0 + 1);
    loadKeys(tile0, page);
    loadValues(tile0, page);
    for (int tile = tile0; tile < tile1; ++tile) {
      const int pos = posOf(tile);
      const int afterPage = pageAt(tile + 2);
      const float sk = kScale, sv = vScale;
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          s[n][k] = 0.0f;
      if (page >= 0) {
#pragma unroll
        for (int j = 0; j < S::keyPieces; ++j) {
          const uint32_t w0[4] = {kReg[0][j].x, kReg[0][j].y, kReg[0][j].z, kReg[0][j].w};
          const uint32_t w1[4] = {kReg[1][j].x, kReg[1][j].y, kReg[1][j].z, kReg[1][j].w};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint4 b[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n)
              b[n] = *reinterpret_cast<const uint4 *>(sQ + (n * 8 + g) * S::qPitch + 64 * j +
                                                      16 * t + 8 * half);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const uint32_t x = prepare<Q>(w0[2 * half + q]), y = prepare<Q>(w1[2 * half + q]);
              const uint32_t a[4] = {widenLow<Q>(x), widenLow<Q>(y), widenHigh<Q>(x),
                                     widenHigh<Q>(y)};
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mmaF16(s[n], a, q ? b[n].z : b[n].x, q ? b[n].w : b[n].y);
            }
          }
        }
      }
      const int nowPage = page;
      page = nextPage;
      nextPage = afterPage;
      loadKeys(tile + 1, page);
      if (nowPage >= 0) {
        // Scores in units of log2, masked; the largest one with its value scale.
        float lsv = 0.0f;
        if (sv > 0.0f && sv < INFINITY)
          lsv = fmaxf(__log2f(sv), -96.0f);
        const bool whole = pos >= allLo && pos + 15 <= firstPos;
        float top[NT][2];
        bool grows = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            s[n][k] *= sk * colFactor[n][k & 1];
            if (!whole) {
              const int at = pos + g + 8 * (k >> 1);
              if (at > seenHi[n][k & 1] || at < seenLo[n][k & 1])
                s[n][k] = kNegInf;
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v = fmaxf(s[n][h], s[n][h + 2]) + lsv;
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
            top[n][h] = v;
            grows = grows || v > m[n][h] + kSlack;
          }
        }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float now = fmaxf(m[n][h], top[n][h]);
              f[h] = now == kNegInf ? 1.0f : exp2Approx(m[n][h] - now);
              m[n][h] = now;
              l[n][h] *= f[h];
            }
#pragma unroll
            for (int i = 0; i < S::mTiles; ++i)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                o[i][n][k] *= f[k & 1];
          }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float ref = m[n][k & 1] == kNegInf ? 0.0f : m[n][k & 1];
            const float e = exp2Approx(s[n][k] - ref);
            l[n][k & 1] += e;
            w[k] = whole || s[n][k] != kNegInf ? e * (sv * kWeight) : 0.0f;
          }
          pb[n][0] = transpose8x8(halfPair(w[0], w[1]));
          pb[n][1] = transpose8x8(halfPair(w[2], w[3]));
        }
        // NaN among the values (e4m3 only) must not reach rows that do not see its
        // token: 0 * NaN is NaN.  Then each column takes the values it sees alone.
        bool poisoned = false;
        if constexpr (__is_same(Q, E4M3)) {
          if (!whole) {
            uint32_t bad = 0;
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
              for (int j = 0; j < S::valuePieces; ++j)
#pragma unroll
                for (int w = 0; w < S::valueWords; ++w)
                  bad |= __vcmpeq4(vReg[h][j][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
            poisoned = __any_sync(0xffffffffu, bad != 0);
          }
        }
        auto addValues = [&](const uint32_t (&vr)[4][S::valuePieces][S::valueWords],
                             const uint32_t (&pr)[NT][2]) {
#pragma unroll
          for (int j = 0; j < S::valuePieces; ++j)
#pragma unroll
            for (int w = 0; w < S::valueWords; ++w) {
              uint32_t lo[2], hi[2]; // [tokens 2t.., tokens 2t + 8..]: bytes 0,1 and 2,3
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t x = prepare<Q>(vr[2 * h][j][w]), y = prepare<Q>(vr[2 * h + 1][j][w]);
                lo[h] = __byte_perm(x, y, 0x5140);
                hi[h] = __byte_perm(x, y, 0x7362);
              }
              const uint32_t a0[4] = {widenLow<Q>(lo[0]), widenHigh<Q>(lo[0]), widenLow<Q>(lo[1]),
                                      widenHigh<Q>(lo[1])};
              const uint32_t a1[4] = {widenLow<Q>(hi[0]), widenHigh<Q>(hi[0]), widenLow<Q>(hi[1]),
                                      widenHigh<Q>(hi[1])};
              const int i = (j * S::valueWords + w) * 2;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mmaF16(o[i][n], a0, pr[n][0], pr[n][1]);
                mmaF16(o[i + 1][n], a1, pr[n][0], pr[n][1]);
              }
            }
        };
        if (!poisoned) {
          addValues(vReg, pb);
        } else {
          for (int col = 0; col < S::rows; ++col) {
            const int qi = min(row0 + col, row0 + rowsHere - 1) / p.share;
            const int hiPos = span.first + qi;
            const int loPos = p.window > 0 ? max(0, hiPos - p.window + 1) : 0;
            uint32_t vr[4][S::valuePieces][S::valueWords];
            uint32_t pr[NT][2];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const int tok = pos + 2 * t + (h & 1) + 8 * (h >> 1);
              const bool in = tok <= hiPos && tok >= loPos;
#pragma unroll
              for (int j = 0; j < S::valuePieces; ++j)
#pragma unroll
                for (int w = 0; w < S::valueWords; ++w)
                  vr[h][j][w] = in ? vReg[h][j][w] : 0u;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) { // the B operand's column is lane / 4
              pr[n][0] = n * 8 + g == col ? pb[n][0] : 0u;
              pr[n][1] = n * 8 + g == col ? pb[n][1] : 0u;
            }
            // NaN * 0 in the other columns: keep what they had.
            float keep[S::mTiles][NT][4];
#pragma unroll
            for (int i = 0; i < S::mTiles; ++i)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  keep[i][n][k] = o[i][n][k];
            addValues(vr, pr);
#pragma unroll
            for (int i = 0; i < S::mTiles; ++i)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  if (n * 8 + 2 * t + (k & 1) != col)
                    o[i][n][k] = keep[i][n][k];
          }
        }
      }
      loadValues(tile + 1, page);
    }

    // ---- join the warps -------------------------------------------------------------------
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v = l[n][h];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) {
          sMax[warp][n * 8 + 2 * t + h] = m[n][h];
          sSum[warp][n * 8 + 2 * t + h] = v;
        }
      }
    __syncthreads(); // also: the query rows in sOut's place have been read
    if (tid < S::rows) {
      float top = kNegInf, sum = 0.0f;
      for (int w = 0; w < kWarps; ++w)
        top = fmaxf(top, sMax[w][tid]);
      for (int w = 0; w < kWarps; ++w) {
        const float f = sMax[w][tid] == kNegInf ? 0.0f : exp2Approx(sMax[w][tid] - top);
        sFactor[w][tid] = f;
        // (a warp whose scores are NaN has a sum but no maximum)
        sum += sMax[w][tid] == kNegInf ? sSum[w][tid] : sSum[w][tid] * f;
      }
      sTop[tid] = top;
      sTotal[tid] = sum;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = n * 8 + 2 * t + h;
        float *dst = sOut + (warp * S::rows + col) * DimCap;
#pragma unroll
        for (int j = 0; j < S::valuePieces; ++j)
#pragma unroll
          for (int w = 0; w < S::valueWords; ++w) {
            const int i = (j * S::valueWords + w) * 2;
            // dims 4w .. 4w + 3 of the lane's run
            *reinterpret_cast<float4 *>(dst + 128 * j + S::valueBytes * g + 4 * w) =
                make_float4(o[i][n][h], o[i][n][h + 2], o[i + 1][n][h], o[i + 1][n][h + 2]);
          }
      }
    __syncthreads();

    const bool split = tile0 > 0 || tile1 < unitTiles;
    constexpr int kQuads = S::rows * DimCap / 4;
    auto finish = [&](int col, int d, float4 v, float top, float sum) {
      // v: sum of kWeight w V; sum: of exp2(x - top).
      const int r = row0 + col;
      const int qi = r / p.share, gh = r - qi * p.share;
      const long long token = span.row + qi;
      const int qHead = head * p.share + gh;
      const float f = sum == 0.0f ? 0.0f : 1.0f / (kWeight * sum);
      __nv_bfloat162 a = __floats2bfloat162_rn(v.x * f, v.y * f);
      __nv_bfloat162 b = __floats2bfloat162_rn(v.z * f, v.w * f);
      uint2 packed;
      packed.x = *reinterpret_cast<uint32_t *>(&a);
      packed.y = *reinterpret_cast<uint32_t *>(&b);
      if (d < c.dim)
        *reinterpret_cast<uint2 *>(p.out + token * p.outTokenStride + qHead * p.outHeadStride + d) =
            packed;
      if (d == 0 && p.lse)
        p.lse[token * p.lseStride + qHead] =
            sum == 0.0f ? kNegInf : (top + __log2f(sum)) * 0.693147180559945309f;
    };
    auto joined = [&](int col, int d) {
      float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4 *>(sOut + (w * S::rows + col) * DimCap + d);
        const float f = sFactor[w][col];
        v.x = fmaf(x.x, f, v.x);
        v.y = fmaf(x.y, f, v.y);
        v.z = fmaf(x.z, f, v.z);
        v.w = fmaf(x.w, f, v.w);
      }
      return v;
    };
    if (!split) {
      for (int i = tid; i < kQuads; i += 256) {
        const int col = i / (DimCap / 4), d = (i - col * (DimCap / 4)) * 4;
        if (col < rowsHere)
          finish(col, d, joined(col, d), sTop[col], sTotal[col]);
      }
    } else {
      const int firstShare = hcKvShareOf(unitBegin, total, shares);
      const int lastShare = hcKvShareOf(unitBegin + unitTiles - 1, total, shares);
      auto slotOf = [&](int share) {
        return p.partial + ((long long)share * 2 + (share == firstShare)) * S::slotFloats;
      };
      float *slot = slotOf(int(blockIdx.x));
      for (int i = tid; i < kQuads; i += 256) {
        const int col = i / (DimCap / 4), d = (i - col * (DimCap / 4)) * 4;
        if (col < rowsHere)
          __stcg(reinterpret_cast<float4 *>(slot + col * DimCap + d), joined(col, d));
      }
      if (tid < rowsHere) {
        __stcg(slot + S::rows * DimCap + tid, sTop[tid]);
        __stcg(slot + S::rows * DimCap + S::rows + tid, sTotal[tid]);
      }
      __threadfence();
      __syncthreads();
      if (tid == 0) // wraps to 0 with the last arrival
        sLast = atomicInc(p.counters + firstShare, unsigned(lastShare - firstShare)) ==
                unsigned(lastShare - firstShare);
      __syncthreads();
      if (sLast) {
        __threadfence();
        for (int i = tid; i < kQuads; i += 256) {
          const int col = i / (DimCap / 4), d = (i - col * (DimCap / 4)) * 4;
          if (col >= rowsHere)
            continue;
          float top = kNegInf;
          for (int x = firstShare; x <= lastShare; ++x)
            top = fmaxf(top, __ldcg(slotOf(x) + S::rows * DimCap + col));
          float sum = 0.0f;
          float4 v = make_float4(0, 0, 0, 0);
          for (int x = firstShare; x <= lastShare; ++x) {
            const float *from = slotOf(x);
            const float part = __ldcg(from + S::rows * DimCap + col);
            const float4 y = __ldcg(reinterpret_cast<const float4 *>(from + col * DimCap + d));
            const float add = __ldcg(from + S::rows * DimCap + S::rows + col);
            const float f = part == kNegInf ? 0.0f : exp2Approx(part - top);
            sum += part == kNegInf ? add : add * f;
            v.x = fmaf(y.x, f, v.x);
            v.y = fmaf(y.y, f, v.y);
            v.z = fmaf(y.z, f, v.z);
            v.w = fmaf(y.w, f, v.w);
          }
          finish(col, d, v, top, sum);
        }
      }
    }
    at = unitBegin + tile1;
  }
}

} // namespace

#define HC_ATTENTION(qname, Q, dim, nt, ctas)                                              \
  extern "C" __global__ void __launch_bounds__(256, ctas)                                   \
      hc_kv_attention_##qname##_d##dim##_r##nt(const __grid_constant__ AttentionParams p) { \
    attend<Q, dim, nt, true>(p);                                                            \
  }                                                                                         \
  extern "C" __global__ void __launch_bounds__(256, ctas)                                   \
      hc_kv_attention_##qname##_d##dim##_r##nt##_any(                                       \
          const __grid_constant__ AttentionParams p) {                                      \
    attend<Q, dim, nt, false>(p);                                                           \
  }
#define HC_ATTENTION_DIMS(qname, Q)                                                        \
  HC_ATTENTION(qname, Q, 64, 1, 2)                                                          \
  HC_ATTENTION(qname, Q, 64, 2, 2)                                                          \
  HC_ATTENTION(qname, Q, 128, 1, 2)                                                         \
  HC_ATTENTION(qname, Q, 128, 2, 1)                                                         \
  HC_ATTENTION(qname, Q, 256, 1, 1)
HC_ATTENTION_DIMS(i8, I8)
HC_ATTENTION_DIMS(e4m3, E4M3)
