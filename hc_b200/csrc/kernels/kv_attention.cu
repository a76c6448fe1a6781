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
//     x + log2(vScale) and is at most 4 behind it (a scale below 2^-96, or 0, counts as
//     that), so w <= 2^15 whatever the scales are and the outputs are rescaled a few times per sequence only.  The sum of
//     exp2(x - m), the maxima and the output are fp32; rounding w costs 2^-12 of a term
//     (terms below 2^-25 of the largest lose more, by at most 2^-36 of it).
//   * The tiles (16 tokens) of all (sequence, head, row tile) units stand in one line
//     that is cut into equal shares, one per resident CTA, and a share into eight, one
//     per warp: a ragged batch is balanced to a tile, and a single long sequence uses the
//     whole GPU.  A warp walks through its part alone, whatever units it crosses (when
//     the warps of a CTA went through units together, meeting at each one's end, the
//     meetings took a third of the time); at the end the CTA joins the pieces of units
//     that its warps share, and a unit that several CTAs share is joined by the last of
//     them to finish, from partial results in global memory - all in the order of the
//     line, so the result does not depend on timing.
// Measured: 64 sequences of up to 8192 tokens, one new token each, int8, dim 128: 145 us,
// 4.6 TB/s, bound by instructions (widening, transposing and scaling per 16 tokens take
// the issue slots that loads leave); one sequence of 1500 tokens 13.6 us, of which setting
// up and the first fetch of instructions are most.  More than 16 query rows per sequence
// and key/value head go to kv_attention_umma.cu.
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
  int stepBlocks, stepRows; // of a tile: whole blocks, and rows beyond them
  // Quotients by products (ceil(2^32 / n), 0 for n = 1): of a position's sixteens by a
  // block's, of a query row by `share`.
  uint32_t blockInverse, shareInverse;
  int vecQ; // rows of q that 16-byte loads can take
  unsigned *counters; // [CTAs], zero between calls
  float *partial;     // [CTAs][2] slots
};

constexpr int kWarps = 8;
constexpr int kChunks = 64; // of 256 sequences whose places in the line are kept
constexpr int kTile = 16;
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
  // (Shared memory: every warp's query rows, its two pieces [rows][DimCap] of floats, and
  // a factor per row of the pieces, or of the shares, that are joined:
  // kWarps * rows * (2 * qPitch + 8 * DimCap) + 4 * rows * max(2 * kWarps, CTAs) bytes.)
};

// What a warp leaves of a unit that it does not have all of.
struct Piece {
  int unitBegin; // names the unit; -1: none
  int tile0, tile1, unitTiles;
  int head, row0, rowsHere, spanRow;
};

// Whole: the head dimension is DimCap.
template <class Q, int DimCap, int NT, bool Whole>
__device__ __forceinline__ void attend(const AttentionParams &p) {
  using S = Shape<DimCap, NT>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int sChunk[kChunks + 1]; // where every 256 sequences begin in the line
  __shared__ int sWarpTotal[kWarps], sWarpUnits[kWarps];
  __shared__ float sTop[S::rows], sTotal[S::rows];
  __shared__ float sRowFactor[kWarps][S::rows];
  __shared__ float sMax[kWarps][2][S::rows], sSum[kWarps][2][S::rows];
  __shared__ Piece sPiece[kWarps][2];
  __shared__ int sLast;
  const HcKvCacheDev &c = p.cache;
  const int tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  __half *sQ = reinterpret_cast<__half *>(smem) + warp * S::rows * S::qPitch;
  float *const sPieces = reinterpret_cast<float *>(smem + kWarps * S::rows * S::qPitch * 2);
  float *const sWeight = sPieces + 2 * kWarps * S::rows * DimCap; // [part][rows], when joining
  // This lane's bytes within 16 tokens (a page spans less than 2^31 bytes).
  const uint32_t kOffset = uint32_t(g) * uint32_t(c.tokenStride) + 16 * t;
  const uint32_t vOffset = uint32_t(2 * t) * uint32_t(c.tokenStride) + S::valueBytes * g;

  auto queryOf = [&](int r) { // of a unit's sequence: row r of the `share` rows per query
    return p.share == 1 ? r : int(__umulhi(uint32_t(r), p.shareInverse));
  };

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
  int total = 0, units = 0; // (the host has checked that they fit)
  bool placeless = false; // rows without a place in the cache
  for (int base = 0; base < p.place.seqs; base += 256) {
    int mine = 0, mineUnits = 0;
    if (base + tid < p.place.seqs) {
      HcKvSpan s;
      int begin, rt;
      const int n = tilesOf(base + tid, s, begin, rt);
      mineUnits = n > 0 ? rt * c.heads : 0;
      mine = n * mineUnits;
      placeless = placeless || s.count != s.allCount;
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    mineUnits = __reduce_add_sync(0xffffffffu, mineUnits);
    if (lane == 0) {
      sWarpTotal[warp] = mine;
      sWarpUnits[warp] = mineUnits;
    }
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) {
      total += sWarpTotal[w];
      units += sWarpUnits[w];
    }
    if (tid == 0 && base / 256 < kChunks)
      sChunk[base / 256 + 1] = total;
    __syncthreads();
  }
  if (tid == 0)
    sChunk[0] = 0;
  if (tid < 2 * kWarps)
    sPiece[tid >> 1][tid & 1].unitBegin = -1;
  __syncthreads();
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
  // A share is a tile per warp at least.  A unit of n tiles is cut into about sqrt(n)
  // shares at most: joining s of them costs as much as s tiles of a warp.
  unsigned shares =
      min(gridDim.x, min(unsigned(total + kWarps - 1) / kWarps,
                         unsigned(ceilf(sqrtf(float(total)) * sqrtf(float(units))))));
  // The units of a single sequence are alike: cut evenly, no CTA has two to join (one
  // token of a sequence of 1500: 13 us instead of 18).
  const bool alike = p.place.seqs == 1 && units > 0 && unsigned(units) <= shares;
  const unsigned perUnit = alike ? shares / unsigned(units) : 0;
  if (alike)
    shares = perUnit * unsigned(units);
  if (blockIdx.x >= shares)
    return;
  const HcKvShares line = alike ? hcKvSharesOfUnits(unsigned(total) / unsigned(units), perUnit)
                                : hcKvSharesOf(unsigned(total), shares);
  const int shareBegin = int(hcKvShareBegin(line, blockIdx.x));
  const int shareTiles = int(hcKvShareBegin(line, blockIdx.x + 1)) - shareBegin;
  int at = shareBegin + int((unsigned)shareTiles * unsigned(warp) / kWarps);
  const int myEnd = shareBegin + int((unsigned)shareTiles * unsigned(warp + 1) / kWarps);

  // The sequence in which this warp's part begins, and where that begins in the line.
  int seq = 0, seqBegin = 0;
  if (at < myEnd) {
    const int chunks = min((p.place.seqs + 255) / 256, kChunks);
    while (seq / 256 + 1 < chunks && sChunk[seq / 256 + 1] <= at)
      seq += 256;
    seqBegin = sChunk[seq / 256];
    for (;; seq += 32) { // (ends: `at` lies before the line's end)
      HcKvSpan s;
      int begin, rt;
      int mine = 0;
      if (seq + lane < p.place.seqs) {
        const int n = tilesOf(seq + lane, s, begin, rt);
        mine = n * rt * c.heads;
      }
      int scan = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d)
          scan += other;
      }
      const unsigned beyond = __ballot_sync(0xffffffffu, seqBegin + scan > at);
      if (beyond) {
        const int first = __ffs(beyond) - 1;
        seqBegin += __shfl_sync(0xffffffffu, scan - mine, first);
        seq += first;
        break;
      }
      seqBegin += __shfl_sync(0xffffffffu, scan, 31);
      if (seq + 32 >= p.place.seqs)
        break;
    }
  }

  // sum: of exp2(x - top); v: four outputs, times kWeight * sum.
  auto finish = [&](const Piece &u, int col, int d, float4 v, float top, float sum) {
    const int r = u.row0 + col;
    const int qi = queryOf(r), gh = r - qi * p.share;
    const long long token = u.spanRow + qi;
    const int qHead = u.head * p.share + gh;
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
          sum == 0.0f ? kNegInf : log2Of(top, sum) * 0.693147180559945309f;
  };

  int slot = 0; // of the warp's next piece
  while (at < myEnd) {
    HcKvSpan span;
    int kvBegin, rowTiles;
    const int unitTiles = tilesOf(seq, span, kvBegin, rowTiles);
    const int inSeq = unitTiles * rowTiles * c.heads;
    if (at - seqBegin >= inSeq) { // next sequence (those without tiles are passed over)
      seqBegin += inSeq;
      ++seq;
      continue;
    }
    const int unit = (at - seqBegin) / unitTiles;
    const int head = rowTiles == 1 ? unit : unit / rowTiles;
    const int rowTile = unit - head * rowTiles;
    const int unitBegin = seqBegin + unit * unitTiles;
    const int tile0 = at - unitBegin;
    const int tile1 = min(unitTiles, myEnd - unitBegin);
    const int row0 = rowTile * S::rows;
    const int rowsHere = min(S::rows, span.count * p.share - row0);
    const int *table = p.place.table + (long long)seq * p.place.tablePitch;

    // ---- query rows into shared memory as f16, a power of two per row ----------------
    __syncwarp(); // the previous unit's have been read
    constexpr int kPer = DimCap / 32; // consecutive elements of a lane
#pragma unroll 1
    for (int r0 = 0; r0 < S::rows; r0 += 4) {
      uint32_t v[4][kPer / 2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j)
          v[i][j] = 0;
        if (r0 + i < rowsHere && lane * kPer < c.dim) {
          const int qi = queryOf(row0 + r0 + i), gh = row0 + r0 + i - qi * p.share;
          const __nv_bfloat16 *src = p.q + (long long)(span.row + qi) * p.qTokenStride +
                                     (long long)(head * p.share + gh) * p.qHeadStride +
                                     lane * kPer;
          if (p.vecQ) {
            if constexpr (kPer == 2) {
              v[i][0] = *reinterpret_cast<const uint32_t *>(src);
            } else if constexpr (kPer == 4) {
              const uint2 x = *reinterpret_cast<const uint2 *>(src);
              v[i][0] = x.x;
              v[i][1] = x.y;
            } else {
              const uint4 x = *reinterpret_cast<const uint4 *>(src);
              v[i][0] = x.x;
              v[i][1] = x.y;
              v[i][2] = x.z;
              v[i][3] = x.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j)
              v[i][j >> 1] |= uint32_t(__bfloat16_as_ushort(src[j])) << (16 * (j & 1));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t top2 = 0; // magnitudes order like their bits
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j)
          top2 = __vmaxu2(top2, v[i][j] & 0x7fff7fffu);
        const uint32_t top =
            __reduce_max_sync(0xffffffffu, max(top2 & 0xffffu, top2 >> 16)) << 16;
        // 2^e <= top < 2^(e+1); zero, subnormal and infinite rows keep their values.
        const int e = int(top >> 23);
        const bool plain = e == 0 || e == 255;
        const float down = plain ? 1.0f : __uint_as_float(uint32_t(max(254 - e, 1)) << 23);
        const float up = plain ? 1.0f : __uint_as_float(uint32_t(min(e, 253)) << 23);
        if (lane == 0)
          sRowFactor[warp][r0 + i] = p.scaleLog2 * up;
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j)
          *reinterpret_cast<uint32_t *>(sQ + (r0 + i) * S::qPitch + lane * kPer + 2 * j) =
              halfPair(__uint_as_float(v[i][j] << 16) * down,
                       __uint_as_float(v[i][j] & 0xffff0000u) * down);
      }
    }
    __syncwarp();

    // ---- this lane's columns: query rows 2t and 2t + 1 of each n-tile ------------------
    float colFactor[NT][2], m[NT][2], l[NT][2];
    int seenHi[NT][2], seenLo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = n * 8 + 2 * t + h;
        colFactor[n][h] = sRowFactor[warp][r];
        m[n][h] = kNegInf;
        l[n][h] = 0.0f;
        const int qi = queryOf(row0 + min(r, rowsHere - 1));
        seenHi[n][h] = span.first + qi;
        seenLo[n][h] = p.window > 0 ? max(0, span.first + qi - p.window + 1) : 0;
      }
    const int firstPos = span.first + queryOf(row0);
    const int lastPos = span.first + queryOf(row0 + rowsHere - 1);
    // Positions that every row sees: [allLo, firstPos].
    const int allLo = p.window > 0 ? max(0, lastPos - p.window + 1) : 0;
    const int anyLo = p.window > 0 ? max(0, firstPos - p.window + 1) : 0;

    const uint8_t *kLane =
        static_cast<const uint8_t *>(c.k) + (long long)head * c.headStride + kOffset;
    const uint8_t *vLane =
        static_cast<const uint8_t *>(c.v) + (long long)head * c.headStride + vOffset;
    // Tokens of this segment's tiles that some row sees: [anyLo, lookEnd).
    const int lookEnd = min(lastPos + 1, kvBegin + tile1 * kTile);
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
    // The tile that is looked up next (two ahead of the one at work): its first position,
    // the block it lies in and its place there, stepped along without divisions.
    int lookPos = kvBegin + tile0 * kTile;
    int lookBlock = lookPos >> 4;
    if (c.block > 16)
      lookBlock = int(__umulhi(uint32_t(lookBlock), p.blockInverse));
    int lookRow = lookPos - lookBlock * c.block;
    // Where a tile's rows lie in the cache; page < 0: not there, or seen by no row.
    struct Spot {
      int page;
      uint64_t at;
    };
    auto look = [&]() -> Spot {
      Spot s{-1, 0};
      if (lookPos < lookEnd && lookPos + 15 >= anyLo)
        s.page = hcKvPageOf(__ldg(table + lookBlock), c.pages);
      s.at = uint32_t(lookRow) * uint32_t(c.tokenStride);
      lookPos += kTile;
      lookBlock += p.stepBlocks;
      lookRow += p.stepRows;
      if (lookRow >= c.block) {
        lookRow -= c.block;
        ++lookBlock;
      }
      return s;
    };
    // All 16 rows lie inside the page, written or not: what is not visible is masked.
    uint4 kReg[2][S::keyPieces];
    uint32_t vReg[4][S::valuePieces][S::valueWords];
    float kScale = 0.0f, vScale = 0.0f;
    auto loadKeys = [&](Spot &s) {
      if (s.page < 0)
        return;
      s.at += uint64_t(uint32_t(s.page)) * uint32_t(c.pageStride);
      const uint8_t *k = kLane + s.at;
      const uint8_t *k8 = k + 8 * uint32_t(c.tokenStride);
#pragma unroll
      for (int j = 0; j < S::keyPieces; ++j) {
        const bool in = Whole || 64 * j + 16 * t < c.dim;
        kReg[0][j] = in ? loadStream16(k + 64 * j) : make_uint4(0, 0, 0, 0);
        kReg[1][j] = in ? loadStream16(k8 + 64 * j) : make_uint4(0, 0, 0, 0);
      }
      kScale = __ldg(kScales + uint64_t(uint32_t(s.page)) * uint32_t(c.scalePitch));
    };
    auto loadValues = [&](const Spot &s) {
      if (s.page < 0)
        return;
      const uint8_t *v = vLane + s.at;
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int j = 0; j < S::valuePieces; ++j) {
          const uint8_t *at =
              v + uint64_t(((h & 1) + 8 * (h >> 1)) * uint32_t(c.tokenStride)) + 128 * j;
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
      vScale = __ldg(vScales + uint64_t(uint32_t(s.page)) * uint32_t(c.scalePitch));
    };

    Spot now = look(), next = look();
    loadKeys(now);
    loadValues(now);
    int pos = kvBegin + tile0 * kTile;
#pragma unroll 1
    for (int tile = tile0; tile < tile1; ++tile, pos += kTile) {
      const Spot after = look();
      const float sk = kScale, sv = vScale;
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          s[n][k] = 0.0f;
      if (now.page >= 0) {
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
      const bool there = now.page >= 0;
      now = next;
      next = after;
      loadKeys(now);
      if (there) {
        // Scores in units of log2, masked; the largest one with its value scale.
        const float lsv = logOfScale(sv);
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
            const int qi = queryOf(row0 + min(col, rowsHere - 1));
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
      loadValues(now);
    }

    // ---- a whole unit is finished, a piece is kept -----------------------------------------
    const Piece piece{unitBegin, tile0, tile1, unitTiles, head, row0, rowsHere, span.row};
    float *const held = sPieces + (warp * 2 + slot) * S::rows * DimCap;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[n][h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int col = n * 8 + 2 * t + h;
        if (g == 0) {
          sMax[warp][slot][col] = m[n][h];
          sSum[warp][slot][col] = sum;
        }
        float *dst = held + col * DimCap + S::valueBytes * g;
#pragma unroll
        for (int j = 0; j < S::valuePieces; ++j)
#pragma unroll
          for (int w = 0; w < S::valueWords; ++w) {
            const int i = (j * S::valueWords + w) * 2;
            *reinterpret_cast<float4 *>(dst + 128 * j + 4 * w) =
                make_float4(o[i][n][h], o[i][n][h + 2], o[i + 1][n][h], o[i + 1][n][h + 2]);
          }
      }
    if (tile0 == 0 && tile1 == unitTiles) {
      __syncwarp();
#pragma unroll 1
      for (int i = lane; i < rowsHere * (DimCap / 4); i += 32) {
        const int col = i / (DimCap / 4), d = (i - col * (DimCap / 4)) * 4;
        finish(piece, col, d, *reinterpret_cast<const float4 *>(held + col * DimCap + d),
               sMax[warp][slot][col], sSum[warp][slot][col]);
      }
      __syncwarp();
    } else {
      if (lane == 0)
        sPiece[warp][slot] = piece;
      ++slot; // (a part has two ends: at most two pieces)
    }
    at = unitBegin + tile1;
  }

  // ---- join the warps' pieces, unit by unit -----------------------------------------------------
  __syncthreads();
  constexpr int kQuads = S::rows * DimCap / 4;
  for (int e0 = 0; e0 < 2 * kWarps;) {
    const Piece u = sPiece[e0 >> 1][e0 & 1];
    if (u.unitBegin < 0) {
      ++e0;
      continue;
    }
    int e1 = e0 + 1, lastTile = u.tile1; // pieces [e0, e1) are the unit's (or empty)
    for (; e1 < 2 * kWarps; ++e1) {
      const Piece &x = sPiece[e1 >> 1][e1 & 1];
      if (x.unitBegin >= 0) {
        if (x.unitBegin != u.unitBegin)
          break;
        lastTile = x.tile1;
      }
    }
    // Factors of the pieces: thread (row, piece), sixteen neighbours hold a row's.
    static_assert(2 * kWarps == 16, "a row's pieces are reduced over sixteen lanes");
    for (int i = tid; i < 16 * S::rows; i += 256) {
      const int col = i >> 4, e = i & 15;
      const bool in = e >= e0 && e < e1 && sPiece[e >> 1][e & 1].unitBegin >= 0;
      const float part = in ? sMax[e >> 1][e & 1][col] : kNegInf;
      float top = part;
#pragma unroll
      for (int d = 8; d > 0; d >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float f = part == kNegInf ? 0.0f : exp2Approx(part - top);
      // (a piece whose scores are NaN has a sum but no maximum)
      float sum = in ? sSum[e >> 1][e & 1][col] * (part == kNegInf ? 1.0f : f) : 0.0f;
#pragma unroll
      for (int d = 8; d > 0; d >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
      sWeight[e * S::rows + col] = f;
      if (e == 0) {
        sTop[col] = top;
        sTotal[col] = sum;
      }
    }
    __syncthreads();
    const bool split = u.tile0 > 0 || lastTile < u.unitTiles;
    const int firstShare = split ? int(hcKvShareOf(line, u.unitBegin)) : 0;
    const int lastShare = split ? int(hcKvShareOf(line, u.unitBegin + u.unitTiles - 1)) : 0;
    auto slotOf = [&](int share) {
      return p.partial + ((long long)share * 2 + (share == firstShare)) * S::slotFloats;
    };
    auto add = [](float4 &v, const float4 &x, float f) {
      v.x = fmaf(x.x, f, v.x);
      v.y = fmaf(x.y, f, v.y);
      v.z = fmaf(x.z, f, v.z);
      v.w = fmaf(x.w, f, v.w);
    };
    float *mine = slotOf(int(blockIdx.x));
    for (int i = tid; i < kQuads; i += 256) {
      const int col = i / (DimCap / 4), d = (i - col * (DimCap / 4)) * 4;
      if (col >= u.rowsHere)
        continue;
      float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
      for (int e = e0; e < e1; ++e) {
        const float f = sWeight[e * S::rows + col];
        if (f != 0.0f) // (0 also for slots that hold nothing)
          add(v, *reinterpret_cast<const float4 *>(sPieces + (e * S::rows + col) * DimCap + d), f);
      }
      if (!split) {
        finish(u, col, d, v, sTop[col], sTotal[col]);
      } else {
        __stcg(reinterpret_cast<float4 *>(mine + col * DimCap + d), v);
        if (d == 0) {
          __stcg(mine + S::rows * DimCap + col, sTop[col]);
          __stcg(mine + S::rows * DimCap + S::rows + col, sTotal[col]);
        }
      }
    }
    if (split) {
      __threadfence();
      __syncthreads();
      if (tid == 0) // wraps to 0 with the last arrival
        sLast = atomicInc(p.counters + firstShare, unsigned(lastShare - firstShare)) ==
                unsigned(lastShare - firstShare);
      __syncthreads();
      if (sLast) {
        __threadfence();
        // A warp per row: the shares' maxima and sums, 32 at a time.
        const int parts = lastShare - firstShare + 1;
        for (int col = warp; col < u.rowsHere; col += kWarps) {
          float top = kNegInf;
          for (int x = lane; x < parts; x += 32)
            top = fmaxf(top, __ldcg(slotOf(firstShare + x) + S::rows * DimCap + col));
#pragma unroll
          for (int d = 16; d > 0; d >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          float sum = 0.0f;
          for (int x = lane; x < parts; x += 32) {
            const float *from = slotOf(firstShare + x) + S::rows * DimCap;
            const float part = __ldcg(from + col), more = __ldcg(from + S::rows + col);
            const float f = part == kNegInf ? 0.0f : exp2Approx(part - top);
            sum += part == kNegInf ? more : more * f;
            sWeight[x * S::rows + col] = f;
          }
          sum = warpSum(sum);
          if (lane == 0) {
            sTop[col] = top;
            sTotal[col] = sum;
          }
        }
        __syncthreads();
        for (int i = tid; i < kQuads; i += 256) {
          const int col = i / (DimCap / 4), d = (i - col * (DimCap / 4)) * 4;
          if (col >= u.rowsHere)
            continue;
          float4 v = make_float4(0, 0, 0, 0);
          int x = 0;
          for (; x + 8 <= parts; x += 8) { // (eight loads travel together)
            float4 y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
              y[k] = __ldcg(reinterpret_cast<const float4 *>(slotOf(firstShare + x + k) +
                                                             col * DimCap + d));
#pragma unroll
            for (int k = 0; k < 8; ++k)
              add(v, y[k], sWeight[(x + k) * S::rows + col]);
          }
          for (; x < parts; ++x)
            add(v,
                __ldcg(reinterpret_cast<const float4 *>(slotOf(firstShare + x) + col * DimCap + d)),
                sWeight[x * S::rows + col]);
          finish(u, col, d, v, sTop[col], sTotal[col]);
        }
      }
    }
    __syncthreads(); // the factors and sLast have been read
    e0 = e1;
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
