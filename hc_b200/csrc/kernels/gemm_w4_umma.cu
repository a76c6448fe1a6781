// Products with 4-bit weights for more than a few rows (hcGemmW4), the weights converted
// inside the GEMM's pipeline:
//
//   out[m, n] = bf16( as[m] * sum_k a[m, k] * bf16((u[n, k] - z[n, k/g]) * s[n, k/g]) )
//
// The product is formed transposed: the weights are the M = 128 rows of tcgen05.mma, the
// activations its N columns (16..256 of them), so a CTA reads its weight rows once for
// up to 256 activation rows, and the accumulator's columns are what few rows leave empty.
//   * The packed weights come by TMA (128 rows x 256 k, 16 KiB) into a ring of their
//     own; converted ones never touch shared memory: a converter thread owns one weight
//     row, turns its 64 bytes of a stage (128 k) into 64 bf16 pairs in registers and
//     stores them into tensor memory (tcgen05.st), from where the MMA takes its A
//     operand.  u becomes 128 + u in bf16 by a shift, a mask and a bias; subtracting
//     128 + z is exact, multiplying by the scale rounds once (bf16, half a step of 2^-8:
//     accumulating in tensor memory leaves no place for a scale per group), and a byte
//     permute puts neighbours in K side by side: 19 instructions for 8 weights, which is
//     what bounds few columns.
//   * The activations (bf16, K-major) come by TMA into 128-byte-swizzled stages.
//   * Warps 0 and 2 issue the copies, warp 1 the MMAs, the others convert stages
//     in turn and drain the accumulator.  Few columns: two CTAs per SM of 256 tensor memory
//     columns each; many: one with twice the converters.
//   * Where the tiles alone do not fill the GPU a cluster of CTAs shares the K of a tile;
//     the partial tiles meet through distributed shared memory, added in rank order.
// Few columns are bound by the stream of weights and its conversion, many by the tensor
// pipe.  Measured, N = K = 8192, groups of 128: 24 us for 16 and 32 rows (1.5 TB/s of packed
// weights), 26 for 64 (the last with two CTAs per SM: 128 take 35), 45 for 256, 64 for 512
// (1.07 PFLOP/s); a launch costs 6.7 us before the first weight arrives.  Up to 1024 rows
// run here, more are converted first (gemm_w4.cu, gemm_bf16_umma.cu); us, here / converted
// first, groups of 128:
//   rows           512       1024        1280        1536        2048        4096
//   8192 x 8192    64 / 98   122 / 137   178 / 182   179 / 182   240 / 229   506 / 435
//   4096 x 4096    31 / 49    39 /  41    71 /  60    72 /  60    73 /  61   141 / 106
//   14336 x 4096   73 / 95   139 / 133   141 / 137   176 / 159   241 / 201   459 / 349
// Waits are bounded as in the other tcgen05 kernels (hc_ptx.cuh); one that is given up
// leaves NaN.
#include "serving_math.cuh"

#include <cooperative_groups.h>

using namespace hc;
namespace cg = cooperative_groups;

namespace {

struct W4UmmaParams {
  const void *scale;
  const uint8_t *zero;
  const float *rowScale; // [M] at rowScaleStride, or null
  __nv_bfloat16 *out;
  long long lds, ldz, rowScaleStride, ldc;
  int M, N, K;
  int group32;      // group / 32
  uint32_t inverse; // 2^32 / group32, rounded down, for group32 > 1
  int groups;       // per row
  int cols;         // activation rows of a tile, a multiple of 16 up to 256
  int tilesM;
  int stagesA, stagesB, stagesW; // tensor memory; shared memory: activations, weights
  int tmemCols;                  // 256 or 512
  int packed;                    // groups of 32 whose four scales of 128 k load together
  int *status;
};

constexpr int kBK = 128; // K of a stage: 64 columns of packed pairs in tensor memory
constexpr int kMaxStages = 6;
constexpr uint32_t kWBytes = 128 * 128; // a stage of weights: 128 rows x 256 k

struct alignas(8) W4Barriers {
  uint64_t fullA[kMaxStages], emptyA[kMaxStages];
  uint64_t fullB[kMaxStages], emptyB[kMaxStages];
  uint64_t fullW[kMaxStages], emptyW[kMaxStages];
  uint64_t done;
  uint32_t tmemBase;
  int abortFlag;
};

constexpr int kStatusConvertWait = 8; // a converter waiting for a free stage

// D[tmem] (+)= A[tmem] * B[smem], bf16.
__device__ __forceinline__ void ummaBf16TmemA(uint32_t dTmem, uint32_t aTmem, uint64_t bDesc,
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

__device__ __forceinline__ __nv_bfloat162 asPair(uint32_t v) {
  return *reinterpret_cast<const __nv_bfloat162 *>(&v);
}
__device__ __forceinline__ uint32_t asWord(__nv_bfloat162 v) {
  return *reinterpret_cast<const uint32_t *>(&v);
}

// A stage of a ring and the parity of its barriers' phase, counted along: dividing the
// use's number by the ring's length took half of a converter's instructions.
struct RingAt {
  int stage = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void step(int stages) {
    if (++stage == stages) {
      stage = 0;
      parity ^= 1;
    }
  }
};

// (v & mask) | bias in one instruction: an immediate may stand in one place only, so the
// bias comes as a value that the compiler does not see through.
__device__ __forceinline__ uint32_t maskBias(uint32_t v, uint32_t bias) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(r) : "r"(v), "r"(bias));
  return r;
}

// Eight weights -> four bf16 pairs in the order of K.  one28: the pair 128, 128.
template <bool ScaleF32>
__device__ __forceinline__ void convert(uint32_t w, uint32_t one28, uint32_t bias, uint32_t scale,
                                        uint32_t *out) {
  uint32_t d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = maskBias(w >> (4 * i), one28);
    const __nv_bfloat162 x = __hsub2(asPair(t), asPair(bias));
    if constexpr (ScaleF32) {
      const float s = __uint_as_float(scale);
      d[i] = asWord(__floats2bfloat162_rn(__low2float(x) * s, __high2float(x) * s));
    } else {
      d[i] = asWord(__hmul2(x, asPair(scale)));
    }
  }
  out[0] = __byte_perm(d[0], d[1], 0x5410);
  out[1] = __byte_perm(d[2], d[3], 0x5410);
  out[2] = __byte_perm(d[0], d[1], 0x7632);
  out[3] = __byte_perm(d[2], d[3], 0x7632);
}

// Two groups of converter warps take the stages in turn; with Halves = 2 a group is eight
// warps, four for each half of a stage's K.
template <int Halves, bool Fine, bool ScaleF32>
__device__ __forceinline__ void w4Umma(const CUtensorMap *mapB, const CUtensorMap *mapW,
                                       const W4UmmaParams &p) {
  extern __shared__ __align__(16) unsigned char smemRaw[];
  __shared__ W4Barriers bars;
  const uint32_t smemBase = (smemAddr(smemRaw) + 1023u) & ~1023u;
  unsigned char *smem = smemRaw + (smemBase - smemAddr(smemRaw));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abortFlag = &bars.abortFlag;
  int *status = p.status;
  const uint32_t stageBytes = uint32_t(p.cols) * kBK * 2;
  const uint32_t wBase = p.stagesB * stageBytes; // of the weights' ring

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbarInit(smemAddr(&bars.fullA[s]), 4 * Halves); // the warps of a group
      mbarInit(smemAddr(&bars.emptyA[s]), 1); // one MMA commit
      mbarInit(smemAddr(&bars.fullB[s]), 1);
      mbarInit(smemAddr(&bars.emptyB[s]), 1);
      mbarInit(smemAddr(&bars.fullW[s]), 1);
      mbarInit(smemAddr(&bars.emptyW[s]), 8 * Halves); // those of both groups
    }
    mbarInit(smemAddr(&bars.done), 1);
    bars.abortFlag = 0;
    fenceBarrierInit();
    prefetchTensorMap(mapB);
    prefetchTensorMap(mapW);
  }
  if (warp == 1) {
    tmemAlloc<1>(smemAddr(&bars.tmemBase), uint32_t(p.tmemCols));
    tmemRelinquish<1>();
  }
  tcgen05FenceBefore();
  __syncthreads();
  tcgen05FenceAfter();
  const uint32_t tmemBase = bars.tmemBase;
  // The accumulator's columns, then 64 columns per stage of A.
  const uint32_t aBase = tmemBase + ((uint32_t(p.cols) + 31u) & ~31u);

  const int tn = int(blockIdx.x) / p.tilesM, tm = int(blockIdx.x) - tn * p.tilesM;
  const int n0 = tn * 128, m0 = tm * p.cols;
  // K in pairs of stages (256 k); behind K both operands read zeros.
  const int pairs = (p.K + 2 * kBK - 1) / (2 * kBK);
  const int splits = int(gridDim.y), split = int(blockIdx.y);
  const int kb0 = 2 * int((long long)split * pairs / splits);
  const int blocks = 2 * int((long long)(split + 1) * pairs / splits) - kb0;

  // Waits for a ring's stage to be free, or filled.
  auto freeOf = [&](uint64_t *bar, const RingAt &at, int code) {
    return mbarWait(smemAddr(&bar[at.stage]), at.parity ^ 1, abortFlag, status, code);
  };
  auto filled = [&](uint64_t *bar, const RingAt &at, int code) {
    return mbarWait(smemAddr(&bar[at.stage]), at.parity, abortFlag, status, code);
  };
  auto settle = [&]() { // after a wait gave up: copies may still be landing, MMAs reading
    if (*abortFlag) {
      const unsigned long long t0 = globalTimerNs();
      while (globalTimerNs() - t0 < 1000000ull) {
      }
    }
  };

  if (warp == 0) {
    // --------------------------- activations by TMA ---------------------------
    if (lane == 0) {
      RingAt ring;
      for (int i = 0; i < blocks; ++i, ring.step(p.stagesB)) {
        if (!freeOf(bars.emptyB, ring, kStatusProducerWait))
          break;
        const int s = ring.stage;
        const uint32_t full = smemAddr(&bars.fullB[s]), at = smemBase + s * stageBytes;
        mbarExpectTx(full, stageBytes);
        tmaLoad2D(at, mapB, full, (kb0 + i) * kBK, m0);
        tmaLoad2D(at + stageBytes / 2, mapB, full, (kb0 + i) * kBK + 64, m0);
      }
      settle();
    }
  } else if (warp == 2) {
    // ----------------------------- weights by TMA ------------------------------
    if (lane == 0) {
      RingAt ring;
      for (int i = 0; i < blocks / 2; ++i, ring.step(p.stagesW)) {
        if (!freeOf(bars.emptyW, ring, kStatusProducerWait))
          break;
        const int s = ring.stage;
        const uint32_t full = smemAddr(&bars.fullW[s]);
        mbarExpectTx(full, kWBytes);
        tmaLoad2D(smemBase + wBase + s * kWBytes, mapW, full, (kb0 / 2 + i) * 128, n0);
      }
      settle();
    }
  } else if (warp == 1) {
    // -------------------------------- MMA issuer -------------------------------
    if (lane == 0) {
      const uint32_t iDesc = makeInstrDescBf16(128, p.cols, false, false);
      bool ok = true;
      RingAt ringA, ringB;
      for (int i = 0; i < blocks; ++i, ringA.step(p.stagesA), ringB.step(p.stagesB)) {
        const int sa = ringA.stage, sb = ringB.stage;
        ok = filled(bars.fullB, ringB, kStatusMmaWaitData) &&
             filled(bars.fullA, ringA, kStatusMmaWaitData);
        if (!ok)
          break;
        tcgen05FenceAfter();
        const uint32_t stage = smemBase + sb * stageBytes;
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk) {
          // K-major rows of 128 bytes (64 k), 8-row groups 1024 bytes apart.
          const uint64_t bDesc =
              makeSmemDesc(stage + (kk >> 2) * (stageBytes / 2), 16, 1024) + uint64_t((kk & 3) * 2);
          ummaBf16TmemA(tmemBase, aBase + uint32_t(sa * 64 + kk * 8), bDesc, iDesc,
                        (i | kk) != 0);
        }
        ummaCommit(smemAddr(&bars.emptyA[sa]));
        ummaCommit(smemAddr(&bars.emptyB[sb]));
      }
      if (ok)
        ummaCommit(smemAddr(&bars.done));
      settle();
    }
  } else if (warp >= 4) {
    // -------------------------------- converters -------------------------------
    // (Every group reads every stage of the weights' ring and there are at least two
    // stages of A, so no wait can be two phases behind its barrier.)
    const int grp = ((warp - 4) >> 2) & 1, firstHalf = (warp - 4) >> 3;
    const int quad = warp & 3, r = quad * 32 + lane;
    const int n = min(n0 + r, p.N - 1); // rows past N: not stored
    const long long atScale = (long long)n * p.lds, atZero = (long long)n * p.ldz;
    const uint32_t laneBase = uint32_t(quad * 32) << 16;
    // Scales (as bf16 or float bits) and zero points of a stage, loaded a turn ahead.
    constexpr int kScales = Fine ? 4 : 1;
    uint32_t scale[kScales], zero[kScales];
    auto loadScales = [&](int i) {
      const int kb = kb0 + i;
      if constexpr (Fine && !ScaleF32) {
        if (p.packed && 4 * kb + 4 <= p.groups) {
          const uint2 s = __ldg(reinterpret_cast<const uint2 *>(
              static_cast<const unsigned short *>(p.scale) + atScale + 4 * kb));
          const uint32_t z =
              p.zero ? __ldg(reinterpret_cast<const uint32_t *>(p.zero + atZero + 4 * kb))
                     : 0x08080808u;
          scale[0] = s.x & 0xffffu;
          scale[1] = s.x >> 16;
          scale[2] = s.y & 0xffffu;
          scale[3] = s.y >> 16;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            zero[j] = (z >> (8 * j)) & 0xffu;
          return;
        }
      }
#pragma unroll
      for (int j = 0; j < kScales; ++j) {
        const uint32_t k32 = uint32_t(kb) * 4 + j;
        // The product's high word is the quotient or one less.
        uint32_t g = k32;
        if (p.group32 > 1) {
          g = __umulhi(k32, p.inverse);
          g += (g + 1) * uint32_t(p.group32) <= k32 ? 1 : 0;
        }
        const int gi = min(int(g), p.groups - 1);
        if constexpr (ScaleF32)
          scale[j] = __float_as_uint(__ldg(static_cast<const float *>(p.scale) + atScale + gi));
        else
          scale[j] = __ldg(static_cast<const unsigned short *>(p.scale) + atScale + gi);
        zero[j] = p.zero ? __ldg(p.zero + atZero + gi) : 8u;
      }
    };
    bool ok = true;
    if (grp < blocks)
      loadScales(grp);
    uint32_t one28;
    asm volatile("mov.b32 %0, 0x43004300;" : "=r"(one28));
    RingAt ringW, ringA;
    if (grp)
      ringA.step(p.stagesA);
    for (int i = grp; i < blocks;
         i += 2, ringW.step(p.stagesW), ringA.step(p.stagesA), ringA.step(p.stagesA)) {
      const int sw = ringW.stage, sa = ringA.stage;
      if (lane == 0)
        ok = filled(bars.fullW, ringW, kStatusConvertWait);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok)
        break;
      // The row's 64 bytes: chunks 4 (i & 1) .. + 3 of 8, swizzled by the row.
      uint32_t w[16 / Halves];
#pragma unroll
      for (int c = 0; c < 4 / Halves; ++c) {
        const uint4 v = *reinterpret_cast<const uint4 *>(
            smem + wBase + sw * kWBytes + r * 128 +
            (((4 * (i & 1) + 2 * firstHalf + c) ^ (r & 7)) << 4));
        w[4 * c] = v.x;
        w[4 * c + 1] = v.y;
        w[4 * c + 2] = v.z;
        w[4 * c + 3] = v.w;
      }
      // 128 + z in bf16 (z <= 127: exact) and the scale, twice each; of this warp's half.
      constexpr int kUsed = Fine ? 4 / Halves : 1;
      uint32_t bias[kUsed], factor[kUsed];
#pragma unroll
      for (int j = 0; j < kUsed; ++j) {
        const uint32_t z = Fine && Halves == 2 && firstHalf ? zero[(j + 2) % kScales] : zero[j];
        const uint32_t s = Fine && Halves == 2 && firstHalf ? scale[(j + 2) % kScales] : scale[j];
        bias[j] = 0x43004300u + z * 0x00010001u;
        factor[j] = ScaleF32 ? s : s * 0x00010001u;
      }
      __syncwarp();
      if (lane == 0)
        mbarArrive(smemAddr(&bars.emptyW[sw]));
      if (i + 2 < blocks)
        loadScales(i + 2);
      if (lane == 0)
        ok = freeOf(bars.emptyA, ringA, kStatusConvertWait);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok)
        break;
      tcgen05FenceAfter(); // the MMAs that read this stage are complete
#pragma unroll
      for (int c = 0; c < 16 / Halves; c += 2) {
        uint32_t v[8];
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const int j = Fine ? (c + d) >> 2 : 0;
          convert<ScaleF32>(w[c + d], one28, bias[j], factor[j], v + 4 * d);
        }
        tmemStore32x8(aBase + laneBase + uint32_t(sa * 64 + firstHalf * 32 + c * 4), v);
      }
      tmemStoreWait();
      tcgen05FenceBefore();
      __syncwarp();
      if (lane == 0)
        mbarArrive(smemAddr(&bars.fullA[sa]));
    }
    // -------------------------------- the accumulator ----------------------------
    if (ok) {
      if (lane == 0)
        ok = mbarWait(smemAddr(&bars.done), 0, abortFlag, status, kStatusEpilogueWait);
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
    if (ok) {
      tcgen05FenceAfter();
      const int nHere = n0 + quad * 32 + lane;
      float *part = reinterpret_cast<float *>(smem); // [cols][128]
      for (int c = (grp + 2 * firstHalf) * 16; c < p.cols; c += 2 * Halves * 16) { // uniform
        uint32_t v[16];
        __syncwarp();
        tmemLoad32x16(tmemBase + laneBase + uint32_t(c), v);
        tmemLoadWait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int m = m0 + c + j;
          if (splits > 1) {
            part[(c + j) * 128 + quad * 32 + lane] = __uint_as_float(v[j]);
          } else if (m < p.M && nHere < p.N) {
            float x = __uint_as_float(v[j]);
            if (p.rowScale)
              x *= __ldg(p.rowScale + m * p.rowScaleStride);
            p.out[(long long)m * p.ldc + nHere] = __float2bfloat16_rn(x);
          }
        }
      }
      tcgen05FenceBefore();
    }
  }
  __syncwarp();
  // Tensor memory is given back before this CTA waits for the others of its cluster: a
  // CTA of another kernel that waits for it can then never hold up one this CTA waits for.
  __syncthreads();
  if (warp == 1) {
    tcgen05FenceAfter();
    tmemFree<1>(tmemBase, uint32_t(p.tmemCols));
  }
  if (*abortFlag) {
    // A wait was given up (nobody waits from here on): NaN instead of a tile, or of this
    // rank's part of one, so that nothing that looks like a result is left.
    const float nan = __uint_as_float(0x7fc00000u);
    float *part = reinterpret_cast<float *>(smem);
    for (int i = int(threadIdx.x); i < p.cols * 128; i += int(blockDim.x)) {
      const int m = m0 + (i >> 7), n = n0 + (i & 127);
      if (splits > 1)
        part[i] = nan;
      else if (m < p.M && n < p.N)
        p.out[(long long)m * p.ldc + n] = __float2bfloat16_rn(nan);
    }
  }
  if (splits > 1) {
    // Partial tiles, added in rank order; a rank finishes every splits-th row.
    cg::cluster_group cluster = cg::this_cluster();
    float *part = reinterpret_cast<float *>(smem);
    cluster.sync();
    const int rank = int(cluster.block_rank());
    for (int c = rank + int(threadIdx.x >> 7) * splits; c < p.cols;
         c += int(blockDim.x >> 7) * splits) {
      const int m = m0 + c, i = threadIdx.x & 127;
      if (m < p.M && n0 + i < p.N) {
        float sum = 0.0f;
        for (int r = 0; r < splits; ++r)
          sum += cluster.map_shared_rank(part, r)[c * 128 + i];
        if (p.rowScale)
          sum *= __ldg(p.rowScale + m * p.rowScaleStride);
        p.out[(long long)m * p.ldc + n0 + i] = __float2bfloat16_rn(sum);
      }
    }
    cluster.sync(); // no CTA leaves while its memory is read
  }
}

} // namespace

#define HC_W4_UMMA(gname, Halves, ctas, fname, Fine, sname, F32)                            \
  extern "C" __global__ void __launch_bounds__(128 + 256 * Halves, ctas)                    \
      hc_gemm_w4_umma_##gname##_##fname##_##sname(const __grid_constant__ CUtensorMap mapB, \
                                                  const __grid_constant__ CUtensorMap mapW, \
                                                  const __grid_constant__ W4UmmaParams p) { \
    w4Umma<Halves, Fine, F32>(&mapB, &mapW, p);                                             \
  }
#define HC_W4_UMMA_SCALES(gname, Halves, ctas, fname, Fine)                                 \
  HC_W4_UMMA(gname, Halves, ctas, fname, Fine, bf16, false)                                 \
  HC_W4_UMMA(gname, Halves, ctas, fname, Fine, f32, true)
HC_W4_UMMA_SCALES(narrow, 1, 2, coarse, false)
HC_W4_UMMA_SCALES(narrow, 1, 2, fine, true)
HC_W4_UMMA_SCALES(wide, 2, 1, coarse, false)
HC_W4_UMMA_SCALES(wide, 2, 1, fine, true)
