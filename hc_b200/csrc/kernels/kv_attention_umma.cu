// Attention over the paged 8-bit key/value cache for many query rows per key/value head
// (chunks of a prompt, and drafts whose query heads share a head); the formula, the
// scales, the masks and the roundings are those of kv_attention.cu.
//
// 128 query rows against T tokens (128, or 64 for heads of 256) at a time on tcgen05:
//   S[128, T] = Q K^T       Q and K in shared memory, f16
//   O[128, D] += P V        P in tensor memory (f16, over its scores), V in shared memory
//                           as it lies in the cache, tokens by dims: an MN-major operand
// Roles of a CTA, which keeps to one unit (sequence, head, 128 rows), or a part of its
// tokens where there are few units:
//   * 4 warps bring the keys of a tile from the cache into registers a tile ahead, widen
//     them to f16 (exact) and store them in the swizzled layout; 4 others the values;
//   * one thread issues the MMAs: the outputs of tile j, then the scores of tile j + 3;
//   * two groups of 4 warps take the score tiles in turn, a thread per row: maximum,
//     exponentials, sum, and P back to tensor memory.  Only the reference that the
//     exponentials are taken against is handed from tile to tile; it is kept until the
//     maximum has grown by 2^4 over it, so O is rescaled in place a few times per unit.
// Per tile of 128 x 128 x 128 the MMAs take 1024 cycles, the exponentials 1024 (16 per
// cycle), and the instructions of widening and softmax about as many issue slots: the
// three run beside each other.  Reading the cache is small beside that (32 KiB a tile,
// mostly from L2).
// Measured: 512 new tokens of 32 heads (8 for keys and values, dim 128) at 16384 tokens in
// 196 us with int8 and 198 to 201 with e4m3 (690 TFLOP/s; the compiler's order of the same
// code moves either by 5 %), against 1143 and 1020 us with kv_attention.cu; dim 64 168 us,
// dim 256 408.  Eight whole prompts of 2048: 670.  Counters show half of the issue slots
// taken (8600 instructions per tile, half of them conversion), the tensor pipe at a
// quarter and no single pipe full: what is left are the latencies of the hand-overs
// between the roles.
#include "kv_params.h"
#include "serving_math.cuh"

using namespace hc;
using namespace hcs;

namespace {

struct KvRowsParams {
  HcKvCacheDev cache;
  HcKvPlaceDev place;
  const __nv_bfloat16 *q; // [tokens, heads * share, dim]
  __nv_bfloat16 *out;
  float *lse; // [tokens, heads * share] or null
  long long qTokenStride, qHeadStride, outTokenStride, outHeadStride, lseStride;
  float scaleLog2; // scale * log2(e)
  int share;       // query heads per key/value head
  int window;      // 0: none
  int rowTiles;    // tiles of 128 rows that maxNew * share rows can take
  int compact;     // units of the rows that there are, not of rowTiles per sequence
  int splits;      // parts that a unit's tokens may be divided into
  // Quotients by products (ceil(2^32 / n), 0 for n = 1): of a position's sixteens by a
  // block's, of a query row by `share`.
  uint32_t blockInverse, shareInverse;
  int vecQ, vecOut;   // rows of q and of out that 16-byte accesses can take
  unsigned *counters; // [units], zero between calls
  float *partial;     // [units][splits] slots
  int *status;
};

constexpr int kThreads = 17 * 32;
constexpr int kMmaWarp = 16; // warps 8..11 convert keys, 12..15 values
constexpr float kNegInf = -INFINITY;
constexpr float kSlack = 4.0f;
constexpr float kWeight = 2048.0f; // 2^(15 - kSlack): probabilities fit f16
constexpr int kStatusRowsConvert = 9, kStatusRowsSoftmax = 10;

__device__ __forceinline__ float exp2Approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t halfPair(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Two floats at a time.
__device__ __forceinline__ uint64_t pairOf(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Four stored elements -> two f16 pairs, exactly.  int8: 0x6400 | u is 1024 + u in f16,
// with the sign bit flipped u = x + 128, and 1152 comes off again.
template <class Q> __device__ __forceinline__ uint2 widen(uint32_t w) {
  uint2 r;
  if constexpr (__is_same(Q, I8)) {
    const uint32_t bias = 0x64806480u, x = w ^ 0x80808080u;
    const __half2 b = *reinterpret_cast<const __half2 *>(&bias);
    const uint32_t lo = __byte_perm(x, 0x64646464u, 0x4140);
    const uint32_t hi = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 l = __hsub2(*reinterpret_cast<const __half2 *>(&lo), b);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&hi), b);
    r.x = *reinterpret_cast<const uint32_t *>(&l);
    r.y = *reinterpret_cast<const uint32_t *>(&h);
  } else {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r.x) : "h"(uint16_t(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r.y) : "h"(uint16_t(w >> 16)));
  }
  return r;
}

// Instruction descriptor of kind::f16 with f16 inputs and f32 accumulation.
__host__ __device__ constexpr uint32_t instrDescF16(int m, int n, bool bMnMajor) {
  return (1u << 4) | (uint32_t(bMnMajor) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(m >> 4) << 24);
}
// D[tmem] (+)= A[tmem] * B[smem], f16.
__device__ __forceinline__ void ummaTmemA(uint32_t dTmem, uint32_t aTmem, uint64_t bDesc,
                                          uint32_t iDesc, uint32_t accumulate) {
  asm volatile("{\n"
               ".reg .pred p;\n"
               "setp.ne.b32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
               "}\n" ::"r"(dTmem),
               "r"(aTmem), "l"(bDesc), "r"(iDesc), "r"(accumulate)
               : "memory");
}

// 32 lanes x 16 columns.
__device__ __forceinline__ void tmemLoad32x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]),
                 "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                 "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(taddr)
               : "memory");
}

// Waits for the loads in flight; what depends on `v` stays behind it.
__device__ __forceinline__ void tmemLoadWaitFor(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]),
                 "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}

// mbarWait (hc_ptx.cuh) with a shorter sleep between its looks: what waits here waits for
// hundreds of cycles (20 us as there took 8 % more of the kernel's time).
__device__ __forceinline__ bool waitFor(uint32_t bar, uint32_t parity, volatile int *abortFlag,
                                        int *status, int code) {
  if (mbarTryWait(bar, parity))
    return true;
  const unsigned long long start = globalTimerNs();
  for (uint32_t spin = 1;; ++spin) {
    if (mbarTryWaitFor(bar, parity, 500u))
      return true;
    if ((spin & 63u) == 0) {
      if (*abortFlag)
        return false;
      if (globalTimerNs() - start > kWaitLimitNs) {
        *abortFlag = 1;
        atomicCAS(status, kStatusOk, code);
        return false;
      }
    }
  }
}

struct alignas(8) RowsBarriers {
  uint64_t queriesFull;                // the softmax warps
  uint64_t keysFull[2], valuesFull[2]; // the converting warps
  uint64_t scored[3];                  // S written, the keys read (MMA commit)
  uint64_t weighted[2];                // P written (the warps of a group)
  uint64_t decided[2];                 // the reference of a tile stands
  uint64_t added[2];                   // P and the values read, O complete (MMA commit)
  uint64_t done;                       // all of it
  uint32_t tmemBase;
  int abortFlag;
};

// The scales of 16 tokens; there = 0: the table names no page for them.
struct alignas(16) Group {
  float key, value, logValue, there; // value: times kWeight
};

template <int DimCap> struct RowsShape {
  static constexpr int tokens = DimCap == 256 ? 64 : 128;
  static constexpr int groups = tokens / 16;
  static constexpr uint32_t chunkBytes = tokens * 128; // 64 dims of a tile's tokens
  static constexpr uint32_t tileBytes = chunkBytes * (DimCap / 64);
  static constexpr uint32_t qBytes = 128 * 128 * (DimCap / 64);
  // (Shared memory: qBytes + 4 * tileBytes + 1024 to align.)
  // Tensor memory columns: three tiles of scores (a tile's weights overwrite them), the
  // outputs.
  static constexpr uint32_t atO = 3 * tokens;
  static constexpr int lanesPerRow = DimCap / 16;
  static constexpr int rowsPerTurn = 128 / lanesPerRow;
  static constexpr int turns = tokens / rowsPerTurn;
  static constexpr int slotFloats = 128 * (DimCap + 2);
};

template <class Q, int DimCap> __device__ __forceinline__ void attendRows(const KvRowsParams &p) {
  using S = RowsShape<DimCap>;
  constexpr int T = S::tokens;
  extern __shared__ __align__(16) unsigned char smemRaw[];
  __shared__ RowsBarriers bars;
  __shared__ Group sGroup[8][S::groups];
  __shared__ int sPlain[8]; // every group of the tile is there, with a key scale >= 0
  __shared__ float sFactor[128]; // of a query row: its power of two, scale * log2(e)
  __shared__ float sRef[128], sSum[2][128], sSumRef[2][128];
  __shared__ int sPoisoned, sLast;
  __shared__ uint64_t sPlace[8][2][S::groups]; // of the converting warps
  const HcKvCacheDev &c = p.cache;
  const int tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5;

  // ---- the unit ------------------------------------------------------------------------
  // Later rows see more tokens: they go first.
  const unsigned lower = unsigned(blockIdx.x) / unsigned(c.heads);
  const int head = int(blockIdx.x - lower * unsigned(c.heads));
  int seq, rowTile;
  if (!p.compact) {
    const unsigned higher = lower / unsigned(p.place.seqs);
    seq = int(lower - higher * unsigned(p.place.seqs));
    rowTile = p.rowTiles - 1 - int(higher);
  } else {
    // The sequence whose row tiles hold number `lower`; one without rows counts as one, for
    // its rows without a place.
    __shared__ int sTiles[kThreads / 32];
    __shared__ int sFound[2];
    if (tid == 0)
      sFound[0] = -1;
    int before = 0;
    for (int base = 0; base < p.place.seqs; base += kThreads) {
      int mine = 0;
      if (base + tid < p.place.seqs) {
        const HcKvSpan s = hcKvLoadSpan(p.place, c.block, base + tid);
        mine = max(1, int(((long long)s.count * p.share + 127) / 128));
      }
      int scan = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d)
          scan += other;
      }
      if (lane == 31)
        sTiles[warp] = scan;
      __syncthreads();
      int total = 0, ahead = before;
      for (int w = 0; w < kThreads / 32; ++w) {
        ahead += w < warp ? sTiles[w] : 0;
        total += sTiles[w];
      }
      const int at = int(lower) - (ahead + scan - mine);
      if (mine > 0 && at >= 0 && at < mine) {
        sFound[0] = base + tid;
        sFound[1] = mine - 1 - at;
      }
      before += total;
      __syncthreads();
      if (int(lower) < before)
        break;
    }
    seq = sFound[0];
    if (seq < 0)
      return;
    rowTile = sFound[1];
  }
  const HcKvSpan span = hcKvLoadSpan(p.place, c.block, seq);
  auto queryOf = [&](int r) {
    return p.share == 1 ? r : int(__umulhi(uint32_t(r), p.shareInverse));
  };
  if (rowTile == 0 && blockIdx.y == 0 && span.count != span.allCount) {
    // Rows without a place in the cache see nothing: zeros.
    for (int row = span.allRow; row < span.allRow + span.allCount; ++row) {
      if (row >= span.row && row < span.row + span.count)
        continue;
      for (int i = tid; i < p.share * c.dim; i += kThreads) {
        const int h = i / c.dim, d = i - h * c.dim;
        p.out[row * p.outTokenStride + (head * p.share + h) * p.outHeadStride + d] =
            __float2bfloat16_rn(0.0f);
        if (d == 0 && p.lse)
          p.lse[row * p.lseStride + head * p.share + h] = kNegInf;
      }
    }
  }
  const int row0 = rowTile * 128;
  const int rowsHere = min(128, span.count * p.share - row0);
  if (rowsHere <= 0)
    return;
  const int firstPos = span.first + queryOf(row0);
  const int lastPos = span.first + queryOf(row0 + rowsHere - 1);
  // Some row sees positions [anyLo, lastPos], every row sees [allLo, firstPos].
  const int anyLo = p.window > 0 ? max(0, firstPos - p.window + 1) : 0;
  const int allLo = p.window > 0 ? max(0, lastPos - p.window + 1) : 0;
  const int kvBegin = anyLo & ~15;
  const int unitTiles = (lastPos - kvBegin) / T + 1;
  // A part has four tiles at least.
  const int parts = min(p.splits, max(1, unitTiles / 4));
  if (int(blockIdx.y) >= parts)
    return;
  const int tile0 = int((long long)unitTiles * blockIdx.y / parts);
  const int tiles = int((long long)unitTiles * (blockIdx.y + 1) / parts) - tile0;
  const int pos0 = kvBegin + tile0 * T; // of the part's first tile

  // ---- setting up -------------------------------------------------------------------------
  const uint32_t smemBase = (smemAddr(smemRaw) + 1023u) & ~1023u;
  unsigned char *smem = smemRaw + (smemBase - smemAddr(smemRaw));
  volatile int *abortFlag = &bars.abortFlag;
  int *status = p.status;
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbarInit(smemAddr(&bars.keysFull[s]), 4);
      mbarInit(smemAddr(&bars.valuesFull[s]), 4);
      mbarInit(smemAddr(&bars.weighted[s]), 4);
      mbarInit(smemAddr(&bars.decided[s]), 4);
      mbarInit(smemAddr(&bars.added[s]), 1);
    }
    for (int s = 0; s < 3; ++s)
      mbarInit(smemAddr(&bars.scored[s]), 1);
    mbarInit(smemAddr(&bars.queriesFull), 8);
    mbarInit(smemAddr(&bars.done), 1);
    bars.abortFlag = 0;
    sPoisoned = 0;
    fenceBarrierInit();
  }
  if (warp == kMmaWarp) {
    tmemAlloc<1>(smemAddr(&bars.tmemBase), 512);
    tmemRelinquish<1>();
  }
  tcgen05FenceBefore();
  __syncthreads();
  tcgen05FenceAfter();
  const uint32_t tmemBase = bars.tmemBase;
  const uint32_t kBase = smemBase + S::qBytes, vBase = kBase + 2 * S::tileBytes;

  // Lane 0 waits for the warp.
  auto await = [&](uint64_t &bar, int use, int code) {
    bool ok = true;
    if (lane == 0)
      ok = waitFor(smemAddr(&bar), uint32_t(use) & 1u, abortFlag, status, code);
    return __shfl_sync(0xffffffffu, int(ok), 0) != 0;
  };

  bool ok = true;
  if (warp == kMmaWarp) {
    // ------------------------------- MMA issuer ---------------------------------
    if (lane == 0) {
      constexpr uint32_t scoreDesc = instrDescF16(128, T, false);
      constexpr uint32_t outDesc = instrDescF16(128, DimCap, true);
      // K-major rows of 128 bytes (64 dims), 8-row groups 1024 bytes apart; the values are
      // MN-major: chunks of 64 dims apart, 8-token groups 1024 bytes.
      const uint64_t qDesc = makeSmemDesc(smemBase, 16, 1024);
      const uint64_t kDesc = makeSmemDesc(kBase, 16, 1024);
      const uint64_t vDesc = makeSmemDesc(vBase, S::chunkBytes, 1024);
      int scoreAt = 0, weightAt = 0; // of three
      auto score = [&](int j) {
        const int b = j & 1;
        if (!waitFor(smemAddr(&bars.keysFull[b]), uint32_t(j >> 1) & 1u, abortFlag, status,
                     kStatusMmaWaitData))
          return false;
        tcgen05FenceAfter();
        const uint64_t k = kDesc + uint32_t(b) * (S::tileBytes >> 4);
        const uint32_t to = tmemBase + uint32_t(scoreAt * T);
#pragma unroll
        for (int kk = 0; kk < DimCap / 16; ++kk)
          umma<1>(to, qDesc + uint64_t((kk >> 2) * (128 * 128 >> 4) + (kk & 3) * 2),
                  k + uint64_t((kk >> 2) * (S::chunkBytes >> 4) + (kk & 3) * 2), scoreDesc,
                  kk != 0);
        ummaCommit(smemAddr(&bars.scored[scoreAt]));
        scoreAt = scoreAt == 2 ? 0 : scoreAt + 1;
        return true;
      };
      ok = waitFor(smemAddr(&bars.queriesFull), 0, abortFlag, status, kStatusMmaWaitData);
      for (int j = 0; ok && j < min(3, tiles); ++j)
        ok = score(j);
      for (int j = 0; ok && j < tiles; ++j) {
        const int b = j & 1;
        ok = waitFor(smemAddr(&bars.valuesFull[b]), uint32_t(j >> 1) & 1u, abortFlag, status,
                     kStatusMmaWaitData) &&
             waitFor(smemAddr(&bars.weighted[b]), uint32_t(j >> 1) & 1u, abortFlag, status,
                     kStatusMmaWaitTmem);
        if (!ok)
          break;
        tcgen05FenceAfter();
        const uint64_t v = vDesc + uint32_t(b) * (S::tileBytes >> 4);
        const uint32_t from = tmemBase + uint32_t(weightAt * T);
        weightAt = weightAt == 2 ? 0 : weightAt + 1;
#pragma unroll
        for (int kk = 0; kk < T / 16; ++kk)
          ummaTmemA(tmemBase + S::atO, from + uint32_t(kk * 8), v + uint64_t(kk * 128), outDesc,
                    (j | kk) != 0);
        ummaCommit(smemAddr(&bars.added[b]));
        // The place of tile j's scores and weights is free behind these MMAs.
        ok = j + 3 >= tiles || score(j + 3);
      }
      if (ok)
        ummaCommit(smemAddr(&bars.done));
      if (!ok) { // MMAs may still be reading
        const unsigned long long t0 = globalTimerNs();
        while (globalTimerNs() - t0 < 1000000ull) {
        }
      }
    }
  } else if (warp >= 8) {
    // ------------------------------- converters ---------------------------------
    // A lane takes 16 bytes of a token: four lanes 64 dims of one, neighbouring fours
    // neighbouring tokens, so that no two lanes of a store phase share banks; a warp takes
    // whole rows.
    constexpr int kRowBits = S::lanesPerRow == 4 ? 3 : S::lanesPerRow == 8 ? 2 : 1;
    const int chunk = lane >> (2 + kRowBits), first16 = (lane & 3) * 2;
    const int piece = chunk * 4 + (lane & 3);
    const int rowOf = ((warp & 3) << kRowBits) + ((lane >> 2) & ((1 << kRowBits) - 1));
    const bool inDim = piece * 16 < c.dim;
    const int *table = p.place.table + (long long)seq * p.place.tablePitch;
    const bool ofKeys = warp < 12;
    const uint8_t *const source = static_cast<const uint8_t *>(ofKeys ? c.k : c.v) +
                                  (long long)head * c.headStride + piece * 16;
    const uint32_t inGroup = uint32_t(rowOf & 15) * uint32_t(c.tokenStride);
    const uint32_t storeAt = uint32_t(chunk) * S::chunkBytes + uint32_t(rowOf) * 128;
    const uint32_t store0 = storeAt + ((first16 ^ (rowOf & 7)) << 4);
    const uint32_t store1 = storeAt + (((first16 + 1) ^ (rowOf & 7)) << 4);

    // Lane g of a warp looks up the place of the tile's sixteen tokens g; the table is read
    // a tile ahead of that.
    int page = -1, entry = -1, rowAt = 0;
    float kScale = 0.0f, vScale = 0.0f;
    bool clear[2] = {false, false}; // of a tile (even, odd): every token is there and seen
    uint4 reg[S::turns];            // a tile is in flight
    auto find = [&](int j) {
      const int pos = pos0 + j * T + lane * 16;
      entry = -1;
      if (lane < S::groups && j < tiles && pos + 15 >= anyLo && pos <= lastPos) {
        int block = pos >> 4;
        if (c.block > 16)
          block = int(__umulhi(uint32_t(block), p.blockInverse));
        entry = __ldg(table + block);
        rowAt = pos - block * c.block;
      }
    };
    auto look = [&](int j) {
      page = hcKvPageOf(entry, c.pages);
      const uint64_t base = page < 0 ? ~0ull
                                     : uint64_t(uint32_t(page)) * uint32_t(c.pageStride) +
                                           uint32_t(rowAt) * uint32_t(c.tokenStride);
      if (lane < S::groups)
        sPlace[warp - 8][j & 1][lane] = base;
      const int first = pos0 + j * T;
      const bool inside = first >= anyLo && first + T - 1 <= lastPos && c.dim == DimCap;
      const bool whole = __all_sync(0xffffffffu, inside && (lane >= S::groups || page >= 0));
      clear[0] = j & 1 ? clear[0] : whole;
      clear[1] = j & 1 ? whole : clear[1];
      find(j + 1);
      __syncwarp();
    };
    // A turn of tile j.
    auto load = [&](int j, int i) {
      const int row = i * S::rowsPerTurn + rowOf;
      const uint64_t at = sPlace[warp - 8][j & 1][row >> 4];
      bool in = true;
      if (!(j & 1 ? clear[1] : clear[0])) {
        const int pos = pos0 + j * T + row;
        in = at != ~0ull && inDim && pos >= anyLo && pos <= lastPos;
      }
      reg[i] = make_uint4(0, 0, 0, 0);
      if (in)
        reg[i] = __ldg(reinterpret_cast<const uint4 *>(
            source + at +
            (inGroup + ((i * S::rowsPerTurn) & 15) * uint32_t(c.tokenStride))));
    };
    auto loadScales = [&]() { // the first warp hands them on
      kScale = vScale = 0.0f;
      if (warp == 8 && page >= 0) {
        const uint64_t at = uint64_t(uint32_t(page)) * uint32_t(c.scalePitch) + head;
        kScale = __ldg(c.kScale + at);
        vScale = __ldg(c.vScale + at);
      }
    };
    // NaN among the values (e4m3 only) must not reach rows that do not see its token:
    // 0 * NaN is NaN.  Where some rows see the token and others do not, zeros stand in
    // for them and the rows that do are mended at the end.
    auto clean = [&](int at, uint4 &v) {
      if constexpr (__is_same(Q, E4M3)) {
        if (at >= allLo && at <= firstPos)
          return;
        uint32_t *w = &v.x, bad = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t nan = __vcmpeq4(w[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
          w[k] &= ~nan;
          bad |= nan;
        }
        if (bad)
          sPoisoned = 1;
      }
    };

    find(0);
    look(0);
#pragma unroll
    for (int i = 0; i < S::turns; ++i)
      load(0, i);
    loadScales();
    uint64_t *const full = ofKeys ? bars.keysFull : bars.valuesFull;
    unsigned char *const ring = smem + ((ofKeys ? kBase : vBase) - smemBase);
    int scoredAt = 0, scoredUse = 0; // of tile j - 2, in a ring of three
    for (int j = 0; j < tiles; ++j) {
      const int b = j & 1;
      if (j >= 2) {
        ok = ofKeys ? await(bars.scored[scoredAt], scoredUse, kStatusRowsConvert)
                    : await(bars.added[b], (j >> 1) - 1, kStatusRowsConvert);
        if (!ok)
          break;
        if (++scoredAt == 3) {
          scoredAt = 0;
          ++scoredUse;
        }
      }
      if (warp == 8) {
        // (Slot j - 8 has been read: the scores of tile j - 2 came behind its weights.)
        Group g;
        g.key = kScale;
        g.value = vScale * kWeight;
        g.logValue = logOfScale(vScale);
        g.there = page >= 0 ? 1.0f : 0.0f;
        const bool plain = __all_sync(
            0xffffffffu, lane >= S::groups || (page >= 0 && kScale >= 0.0f && p.scaleLog2 >= 0.0f));
        if (lane < S::groups)
          sGroup[j & 7][lane] = g;
        if (lane == 0)
          sPlain[j & 7] = plain;
      }
      look(j + 1);
      loadScales();
      const int first = pos0 + j * T + rowOf;
      const bool edge = !ofKeys && (pos0 + j * T < allLo || pos0 + j * T + T - 1 > firstPos);
      if (edge) {
#pragma unroll
        for (int i = 0; i < S::turns; ++i)
          clean(first + i * S::rowsPerTurn, reg[i]);
      }
      unsigned char *const to = ring + b * S::tileBytes;
#pragma unroll
      for (int i = 0; i < S::turns; ++i) {
        const uint2 w0 = widen<Q>(reg[i].x), w1 = widen<Q>(reg[i].y);
        const uint2 w2 = widen<Q>(reg[i].z), w3 = widen<Q>(reg[i].w);
        load(j + 1, i); // (four turns ahead only: 242 us instead of 210)
        *reinterpret_cast<uint4 *>(to + store0 + i * S::rowsPerTurn * 128) =
            make_uint4(w0.x, w0.y, w1.x, w1.y);
        *reinterpret_cast<uint4 *>(to + store1 + i * S::rowsPerTurn * 128) =
            make_uint4(w2.x, w2.y, w3.x, w3.y);
      }
      fenceProxyAsync();
      __syncwarp();
      if (lane == 0)
        mbarArrive(smemAddr(&full[b]));
    }
  } else {
    // --------------------------------- softmax -----------------------------------
    // Query rows as f16, a power of two per row, K-major and swizzled: a warp takes 16.
    constexpr int kPer = DimCap / 32; // consecutive elements of a lane
#pragma unroll 1
    for (int r0 = warp * 16; r0 < warp * 16 + 16; r0 += 8) {
      uint32_t v[8][kPer / 2];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
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
      for (int i = 0; i < 8; ++i) {
        const int r = r0 + i;
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
          sFactor[r] = p.scaleLog2 * up;
        const int byte = lane * kPer * 2, chunk = byte >> 7, in = byte & 127;
        unsigned char *dst = smem + chunk * (128 * 128) + r * 128 +
                             ((((in >> 4) ^ (r & 7)) << 4) | (in & 15));
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j)
          *reinterpret_cast<uint32_t *>(dst + 4 * j) =
              halfPair(__uint_as_float(v[i][j] << 16) * down,
                       __uint_as_float(v[i][j] & 0xffff0000u) * down);
      }
    }
    fenceProxyAsync();
    __syncwarp();
    if (lane == 0)
      mbarArrive(smemAddr(&bars.queriesFull));
    ok = await(bars.queriesFull, 0, kStatusRowsSoftmax); // (the rows' factors)
    const int group = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t laneBase = uint32_t((warp & 3) * 32) << 16;
    const float rowFactor = sFactor[r];
    const int qi = queryOf(row0 + min(r, rowsHere - 1));
    const int seenHi = span.first + qi;
    const int seenLo = p.window > 0 ? max(0, seenHi - p.window + 1) : 0;
    float ref = kNegInf; // what `sum` was taken against
    float sum = 0.0f;
    int at3 = group, use3 = 0; // of tile j in the ring of three
    for (int j = group; ok && j < tiles; j += 2) {
      const int b = j & 1, pos = pos0 + j * T;
      if (!(ok = await(bars.scored[at3], use3, kStatusRowsSoftmax)))
        break;
      tcgen05FenceAfter();
      const Group *const groups = sGroup[j & 7];
      // The weights overwrite the scores, 16 columns per 32: those have been loaded then.
      const uint32_t sAt = tmemBase + laneBase + uint32_t(at3 * T), pAt = sAt;
      at3 += 2;
      if (at3 >= 3) {
        at3 -= 3;
        ++use3;
      }
      const bool whole = pos >= allLo && pos + T - 1 <= firstPos;
      const bool plain = whole && sPlain[j & 7];
      uint32_t v[16], u[16];

      // The largest score with its value scale, in loops that are not unrolled further.
      // (No load stays in flight across a branch or a loop's end, where the compiler might
      // move a register that it has not reached yet; and the warp is brought together in
      // front of each load behind code whose path differs by lane: all 32 lanes have to
      // reach it at once.)
      float top = kNegInf;
      auto seen = [&](int at) { return at >= seenLo && at <= seenHi; };
      auto most16 = [&](const uint32_t (&x)[16], const Group &g) {
        float a = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
        float c = fmaxf(__uint_as_float(x[2]), __uint_as_float(x[3]));
#pragma unroll
        for (int i = 4; i < 16; i += 4) {
          a = max3(a, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
          c = max3(c, __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
        }
        top = fmaxf(top, fmaf(fmaxf(a, c), g.key * rowFactor, g.logValue));
      };
      if (plain) {
#pragma unroll 1
        for (int k = 0; k < T / 32; ++k) {
          tmemLoad32x16(sAt + uint32_t(32 * k), v);
          tmemLoad32x16(sAt + uint32_t(32 * k + 16), u);
          const Group g0 = groups[2 * k], g1 = groups[2 * k + 1];
          tmemLoadWaitFor(v);
          tmemLoadWaitFor(u);
          most16(v, g0);
          most16(u, g1);
        }
      } else {
#pragma unroll 1
        for (int k = 0; k < T / 16; ++k) {
          const Group g = groups[k];
          if (g.there == 0.0f)
            continue;
          __syncwarp();
          tmemLoad32x16(sAt + uint32_t(16 * k), v);
          tmemLoadWaitFor(v);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (seen(pos + 16 * k + i))
              top = fmaxf(top, fmaf(__uint_as_float(v[i]), g.key * rowFactor, g.logValue));
        }
      }

      // The reference: handed on by the tile before.
      float old = kNegInf;
      if (j > 0) {
        if (!(ok = await(bars.decided[b ^ 1], (j - 1) >> 1, kStatusRowsSoftmax)))
          break;
        old = sRef[r];
      }
      const float now = top > old + kSlack ? top : old;
      if (now != old || j == 0)
        sRef[r] = now;
      __syncwarp();
      if (lane == 0)
        mbarArrive(smemAddr(&bars.decided[b]));
      if (now != ref) {
        sum *= exp2Approx(ref - now); // (0 against -inf: there was no sum)
        ref = now;
      }
      __syncwarp();
      const float base = now == kNegInf ? 0.0f : now;
      const uint64_t minusBase = pairOf(-base, -base);
      uint64_t sum2 = pairOf(0.0f, 0.0f);
      auto weigh16 = [&](const uint32_t (&x)[16], const Group &g, uint32_t at) {
        const float f = g.key * rowFactor;
        const uint64_t f2 = pairOf(f, f), v2 = pairOf(g.value, g.value);
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint64_t y =
              fma2(pairOf(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), f2, minusBase);
          float lo, hi;
          unpair(y, lo, hi);
          y = pairOf(exp2Approx(lo), exp2Approx(hi));
          sum2 = add2(sum2, y);
          unpair(mul2(y, v2), lo, hi);
          w[i] = halfPair(lo, hi);
        }
        tmemStore32x8(pAt + at, w);
      };
      if (plain) {
#pragma unroll 1
        for (int k = 0; k < T / 32; ++k) {
          tmemLoad32x16(sAt + uint32_t(32 * k), v);
          tmemLoad32x16(sAt + uint32_t(32 * k + 16), u);
          const Group g0 = groups[2 * k], g1 = groups[2 * k + 1];
          tmemLoadWaitFor(v);
          tmemLoadWaitFor(u);
          weigh16(v, g0, uint32_t(16 * k));
          weigh16(u, g1, uint32_t(16 * k + 8));
        }
      } else {
#pragma unroll 1
        for (int k = 0; k < T / 16; ++k) {
          const Group g = groups[k];
          uint32_t w[8];
          __syncwarp();
          tmemLoad32x16(sAt + uint32_t(16 * k), v);
          tmemLoadWaitFor(v);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float e[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const bool in = g.there != 0.0f && seen(pos + 16 * k + i + h);
              const float x =
                  exp2Approx(fmaf(__uint_as_float(v[i + h]), g.key * rowFactor, -base));
              sum += in ? x : 0.0f;
              e[h] = in ? x * g.value : 0.0f;
            }
            w[i >> 1] = halfPair(e[0], e[1]);
          }
          tmemStore32x8(pAt + uint32_t(8 * k), w);
        }
      }
      float lo, hi;
      unpair(sum2, lo, hi);
      sum += lo + hi;
      // O, where the reference has moved: the outputs of the tile before are in it by now.
      if (__any_sync(0xffffffffu, now != old) && j > 0) {
        // (Use before last: complete, the scores of tile j came behind it.)
        if (!(ok = await(bars.added[b ^ 1], (j - 1) >> 1, kStatusRowsSoftmax)))
          break;
        tcgen05FenceAfter();
        const float f = now == old ? 1.0f : exp2Approx(old - now);
#pragma unroll 1
        for (int d = 0; d < DimCap; d += 16) {
          tmemLoad32x16(tmemBase + laneBase + S::atO + uint32_t(d), u);
          tmemLoadWaitFor(u);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              o[i] = __float_as_uint(__uint_as_float(u[8 * k + i]) * f);
            tmemStore32x8(tmemBase + laneBase + S::atO + uint32_t(d + 8 * k), o);
          }
        }
      }
      tmemStoreWait();
      tcgen05FenceBefore();
      __syncwarp();
      if (lane == 0)
        mbarArrive(smemAddr(&bars.weighted[b]));
    }
    sSum[group][r] = sum;
    sSumRef[group][r] = ref;
  }
  __syncwarp();
  __syncthreads();

  // ---- the outputs ---------------------------------------------------------------------------
  const int unit = int(blockIdx.x);
  auto slotOf = [&](int part) {
    return p.partial + ((long long)unit * p.splits + part) * S::slotFloats;
  };
  // Rows go out through shared memory (the queries' place), 16 bytes per thread and whole
  // rows per warp: a thread per row storing its own took 4 us per unit.  The 16-byte
  // chunks of a row are exchanged by an XOR with the row.
  auto keep = [&](int r, int d, float4 v, float f) {
    __nv_bfloat162 x = __floats2bfloat162_rn(v.x * f, v.y * f);
    __nv_bfloat162 y = __floats2bfloat162_rn(v.z * f, v.w * f);
    uint2 packed;
    packed.x = *reinterpret_cast<uint32_t *>(&x);
    packed.y = *reinterpret_cast<uint32_t *>(&y);
    *reinterpret_cast<uint2 *>(smem + r * (2 * DimCap) + (((d >> 3) ^ (r & 7)) << 4) +
                               (d & 4) * 2) = packed;
  };
  auto writeRows = [&]() {
    for (int i = tid; i < rowsHere * (DimCap / 8); i += kThreads) {
      const int r = i / (DimCap / 8), ch = i - r * (DimCap / 8);
      if (ch * 8 >= c.dim)
        continue;
      const uint4 v =
          *reinterpret_cast<const uint4 *>(smem + r * (2 * DimCap) + ((ch ^ (r & 7)) << 4));
      const int qi = queryOf(row0 + r), gh = row0 + r - qi * p.share;
      __nv_bfloat16 *to = p.out + (long long)(span.row + qi) * p.outTokenStride +
                          (long long)(head * p.share + gh) * p.outHeadStride + ch * 8;
      if (p.vecOut) {
        *reinterpret_cast<uint4 *>(to) = v;
      } else {
        *reinterpret_cast<uint2 *>(to) = make_uint2(v.x, v.y);
        *reinterpret_cast<uint2 *>(to + 4) = make_uint2(v.z, v.w);
      }
    }
  };
  auto finishSum = [&](int r, float top, float sum) {
    const int qi = queryOf(row0 + r), gh = row0 + r - qi * p.share;
    if (p.lse)
      p.lse[(long long)(span.row + qi) * p.lseStride + head * p.share + gh] =
          sum == 0.0f ? kNegInf : log2Of(top, sum) * 0.693147180559945309f;
  };
  const bool aborted = *abortFlag != 0;
  if (warp < 8 && !aborted) {
    // (A barrier of its own: a wait for the last use of `added` would also pass while the
    // use before the last but one is incomplete.)
    if (await(bars.done, 0, kStatusEpilogueWait)) {
      tcgen05FenceAfter();
      const int group = warp >> 2, r = (warp & 3) * 32 + lane;
      const float top = sRef[r];
      float sum = 0.0f;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float part = sSum[g][r], against = sSumRef[g][r];
        sum += against == top ? part : part * exp2Approx(against - top);
      }
      const float f = sum == 0.0f ? 0.0f : 1.0f / (kWeight * sum);
      float *slot = slotOf(int(blockIdx.y));
      const int qi = queryOf(row0 + min(r, rowsHere - 1));
      const int seenHi = span.first + qi;
      const int seenLo = p.window > 0 ? max(0, seenHi - p.window + 1) : 0;
#pragma unroll 1
      for (int d0 = group * (DimCap / 2); d0 < (group + 1) * (DimCap / 2); d0 += 16) {
        uint32_t v[16];
        __syncwarp(); // (the lanes' paths through the turn before differ)
        tmemLoad32x16(tmemBase + (uint32_t((warp & 3) * 32) << 16) + S::atO + d0, v);
        tmemLoadWaitFor(v);
#pragma unroll
        for (int i = 0; i < 4 && r < rowsHere; ++i) {
          float4 o = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                 __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
          if (__is_same(Q, E4M3) && sPoisoned && d0 + 4 * i < c.dim) {
            // The row's tokens that not every row sees: [seenLo, allLo) and (firstPos, seenHi].
            const int *table = p.place.table + (long long)seq * p.place.tablePitch;
            const int end = min(seenHi, pos0 + tiles * T - 1);
#pragma unroll 1
            for (int at = max(seenLo, pos0); at <= end; ++at) {
              if (at >= allLo && at <= firstPos) {
                at = firstPos;
                continue;
              }
              const int page = hcKvPageOf(table[at / c.block], c.pages);
              if (page < 0)
                continue;
              const uint32_t w = *reinterpret_cast<const uint32_t *>(
                  static_cast<const uint8_t *>(c.v) + (long long)page * c.pageStride +
                  (long long)head * c.headStride + (long long)(at % c.block) * c.tokenStride +
                  d0 + 4 * i);
              const uint32_t nan = __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
              const float bad = __uint_as_float(0x7fc00000u);
              o.x = nan & 0xffu ? bad : o.x;
              o.y = nan & 0xff00u ? bad : o.y;
              o.z = nan & 0xff0000u ? bad : o.z;
              o.w = nan & 0xff000000u ? bad : o.w;
            }
          }
          if (parts == 1)
            keep(r, d0 + 4 * i, o, f);
          else // [dims / 4][rows]
            __stcg(reinterpret_cast<float4 *>(slot) + (d0 / 4 + i) * 128 + r, o);
        }
      }
      if (group == 0 && r < rowsHere) {
        if (parts == 1) {
          finishSum(r, top, sum);
        } else {
          __stcg(slot + 128 * DimCap + r, top);
          __stcg(slot + 128 * DimCap + 128 + r, sum);
        }
      }
      __syncwarp();
      tcgen05FenceBefore();
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == kMmaWarp) {
    tcgen05FenceAfter();
    tmemFree<1>(tmemBase, 512);
  }
  // A wait that was given up must not leave rows that look like results: this unit's become
  // NaN, or the part's share of the joint sums does.
  const bool lost = *abortFlag != 0; // (nobody waits from here on)
  if (parts == 1) {
    if (lost) {
      const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll 1
      for (int i = tid; i < rowsHere * (DimCap / 4); i += kThreads)
        keep(i / (DimCap / 4), i % (DimCap / 4) * 4, make_float4(nan, nan, nan, nan), 1.0f);
      if (tid < rowsHere)
        finishSum(tid, nan, nan);
      __syncthreads();
    }
    writeRows();
    return;
  }
  if (lost && tid < 128) {
    const HcKvPart none = hcKvLostPart();
    float *slot = slotOf(int(blockIdx.y));
    __stcg(slot + 128 * DimCap + tid, none.top);
    __stcg(slot + 128 * DimCap + 128 + tid, none.sum);
  }

  // ---- the last part to finish joins them, in their order ------------------------------------
  __threadfence();
  __syncthreads();
  if (tid == 0) // wraps to 0 with the last arrival
    sLast = atomicInc(p.counters + unit, unsigned(parts - 1)) == unsigned(parts - 1);
  __syncthreads();
  if (!sLast)
    return;
  __threadfence();
  float *const sWeight = reinterpret_cast<float *>(smem + S::qBytes); // [part][rows]
  if (tid < rowsHere) {
    float top = kNegInf;
    for (int x = 0; x < parts; ++x)
      top = fmaxf(top, __ldcg(slotOf(x) + 128 * DimCap + tid));
    float sum = 0.0f;
    for (int x = 0; x < parts; ++x) {
      // (a part whose scores are NaN has a sum but no maximum)
      const HcKvPart part{__ldcg(slotOf(x) + 128 * DimCap + tid),
                          __ldcg(slotOf(x) + 128 * DimCap + 128 + tid)};
      const float power = exp2Approx(part.top - top);
      sum += hcKvPartSum(part, power);
      sWeight[x * 128 + tid] = hcKvPartWeight(part, power);
    }
    sSum[0][tid] = sum;
    finishSum(tid, top, sum);
  }
  __syncthreads();
  for (int i = tid; i < 128 * (DimCap / 4); i += kThreads) {
    const int r = i & 127, d = (i >> 7) * 4;
    if (r >= rowsHere)
      continue;
    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int x = 0; x < parts; ++x) {
      const float4 y = __ldcg(reinterpret_cast<const float4 *>(slotOf(x)) + i);
      const float f = sWeight[x * 128 + r];
      if (f != 0.0f) {
        v.x = fmaf(y.x, f, v.x);
        v.y = fmaf(y.y, f, v.y);
        v.z = fmaf(y.z, f, v.z);
        v.w = fmaf(y.w, f, v.w);
      }
    }
    keep(r, d, v, sSum[0][r] == 0.0f ? 0.0f : 1.0f / (kWeight * sSum[0][r]));
  }
  __syncthreads();
  writeRows();
}

} // namespace

#define HC_ATTENTION_ROWS(qname, Q, dim)                                                   \
  extern "C" __global__ void __launch_bounds__(kThreads, 1)                                 \
      hc_kv_attention_rows_##qname##_d##dim(const __grid_constant__ KvRowsParams p) {       \
    attendRows<Q, dim>(p);                                                                  \
  }
HC_ATTENTION_ROWS(i8, I8, 64)
HC_ATTENTION_ROWS(i8, I8, 128)
HC_ATTENTION_ROWS(i8, I8, 256)
HC_ATTENTION_ROWS(e4m3, E4M3, 64)
HC_ATTENTION_ROWS(e4m3, E4M3, 128)
HC_ATTENTION_ROWS(e4m3, E4M3, 256)
