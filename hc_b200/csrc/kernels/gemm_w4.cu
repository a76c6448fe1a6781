// Products of a few activation rows with 4-bit weights that have a scale (and maybe a
// zero point) for each group of K, and the conversions that larger row counts use:
//
//   out[m, n] = bf16( sa[m, k/ga] * sum_k a[m, k] * (u[n, k] - z[n, k/g]) * s[n, k/g] )
//
// u: 4-bit numbers 0..15, two per byte along K (even k in the low half), rows of
// weights one after another ([N, K/2]); z is 8 where there are no zero points; sa is 1
// for bf16 activations.
//
// With few rows the weights are the traffic (half a byte each, read once), so the
// kernel streams them from HBM straight into registers, in the layout they are stored
// in: no shared memory, no barrier in the stream.  The weights are the A operand of
// mma.sync m16n8k16 (16 weight rows x 16 of K) and the activations the B operand: a
// lane holds two rows' 32 consecutive weights of 128 (one 16-byte load each), and since
// a sum does not care about the order of its terms, K is permuted so that these are the
// very elements the lane feeds to 8 MMAs.  Legacy mma.sync rather than tcgen05: at
// M <= 64 the stream of weights is the bound, operand registers need no detour through
// shared memory, and one row costs what eight do.
//   * unpacking: (w >> 4i) & 0x000f000f | 0x43004300 is the bf16 pair 128 + u of
//     nibbles i and i + 4, one packed subtraction of 128 + z makes it exact (u - z);
//     with int8 activations the MMA takes the unsigned nibbles themselves
//     (m16n8k32, u8 x s8, exact int32 sums) and z * sum(a) is subtracted per group.
//   * the sum of a group is formed in the MMA's fp32 (int32) accumulators and then
//     multiplied by the group's scale into the fp32 total: no rounding of weights.
//   * groups that are not multiples of 128 (32, 64, 96 ...): the four lanes of a row
//     exchange words (a 4 x 4 transpose by shuffles) so that an MMA stays inside 32
//     consecutive k.
//   * a CTA is 8 warps on 128 (MT = 2: 256) weight rows and a slice of K; the
//     activations of its slice lie in shared memory in fragment order.  A cluster of
//     CTAs along K adds its partial sums through distributed shared memory, in a fixed
//     order, so the result does not depend on timing.
#include "serving_math.cuh"

#include <cooperative_groups.h>
#include <type_traits>

using namespace hcs;
namespace cg = cooperative_groups;

namespace {

struct W4Params {
  const void *a;       // bf16 or int8 [M, K]
  const float *aScale; // int8 activations: [M, ceil(K / aGroup)]
  const uint8_t *w;    // [N, ceil(K / 2)]
  const void *scale;   // bf16 or float [N, ceil(K / group)]
  const uint8_t *zero; // [N, ceil(K / group)] or null
  __nv_bfloat16 *out;  // [M, N]
  long long lda, ldas, ldw, lds, ldz, ldc;
  int M, N, K, group, aGroup;
  int scaleF32;
  int sliceK; // K per CTA, a multiple of 128
  int stepK;  // K staged in shared memory at a time, a multiple of 128
  int vec;    // w: 16-byte aligned rows
  int vecA;   // a: 16-byte aligned rows
};

constexpr int kSpan = 128; // K of one pair of 16-byte loads

__device__ __forceinline__ void mmaBf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mmaU8S8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The 16 bytes (32 weights) at byte `at` of a weight row that is `bytes` long; what
// lies beyond the row reads as zero (its activations are zero).  Whole: rows are
// 16-byte aligned and a multiple of 16 bytes long.
template <bool Whole>
__device__ __forceinline__ uint4 loadWeights(const uint8_t *row, long long at, int bytes,
                                             int vec) {
  if constexpr (Whole) {
    return at < bytes ? loadStream16(row + at) : make_uint4(0, 0, 0, 0);
  } else {
    if (vec && at + 16 <= bytes)
      return loadStream16(row + at);
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (at + i < bytes)
        v[i >> 2] |= uint32_t(row[at + i]) << (8 * (i & 3));
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// words[j] of lane t of a quad <-> words[t] of lane j: afterwards word c of lane t is
// word t of what lane c had, i.e. the quad's words c are 32 consecutive k.
__device__ __forceinline__ void transposeQuad(uint32_t (&v)[4], int t) {
  const bool odd = t & 1, high = t & 2;
  uint32_t s0 = odd ? v[0] : v[1], s1 = odd ? v[2] : v[3];
  s0 = __shfl_xor_sync(0xffffffffu, s0, 1);
  s1 = __shfl_xor_sync(0xffffffffu, s1, 1);
  if (odd) {
    v[0] = s0;
    v[2] = s1;
  } else {
    v[1] = s0;
    v[3] = s1;
  }
  uint32_t r0 = high ? v[0] : v[2], r1 = high ? v[1] : v[3];
  r0 = __shfl_xor_sync(0xffffffffu, r0, 2);
  r1 = __shfl_xor_sync(0xffffffffu, r1, 2);
  if (high) {
    v[0] = r0;
    v[1] = r1;
  } else {
    v[2] = r0;
    v[3] = r1;
  }
}

__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&a),
                                   *reinterpret_cast<const __nv_bfloat162 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&d);
}

// Eight weights -> four bf16 pairs (k0,k4) (k1,k5) (k2,k6) (k3,k7) of u - z; `bias` is
// the pair 128 + z.
__device__ __forceinline__ void unpackBf16(uint32_t w, uint32_t bias, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p[i] = sub2(((w >> (4 * i)) & 0x000f000fu) | 0x43004300u, bias);
}

// Shared memory: the activations of the current step in fragment order, then the
// scales and zero points of the step's groups, [group][row].
//   bf16: per span, n-tile and word j one 16-byte piece per lane: the 8 activations
//         that meet word j of that lane, as pairs (0,4) (1,5) (2,6) (3,7);
//   int8: 8 bytes per lane: bytes (0,2,4,6) and (1,3,5,7).
template <int NT, int MT, bool A8, bool Fine> struct Layout {
  static constexpr int rows = 8 * 16 * MT; // weight rows of a CTA
  static constexpr int pieceBytes = A8 ? 8 : 16;
  static constexpr int spanBytes = NT * 4 * 32 * pieceBytes;
};

template <int NT, int MT, bool A8, bool Fine, bool Whole>
__device__ __forceinline__ void w4Body(const W4Params &p) {
  using L = Layout<NT, MT, A8, Fine>;
  using Acc = typename std::conditional<A8, int, float>::type;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int row0 = int(blockIdx.x) * L::rows;
  const int kBegin = int(blockIdx.y) * p.sliceK;
  const int kEnd = min(p.K, kBegin + p.sliceK);
  const int rowBytes = (p.K + 1) >> 1;

  unsigned char *frag = smem;
  const int maxGroups = (p.stepK + p.group - 1) / p.group + 1; // (as the host computes it)
  float *sScale = reinterpret_cast<float *>(smem + size_t(p.stepK / kSpan) * L::spanBytes);
  uint32_t *sBias = reinterpret_cast<uint32_t *>(sScale + maxGroups * L::rows);
  int *sASum = reinterpret_cast<int *>(sBias + maxGroups * L::rows);       // int8: [group][8 NT]
  float *sAScale = reinterpret_cast<float *>(sASum + maxGroups * 8 * NT); // int8: [group][8 NT]

  const uint8_t *wRow[2 * MT];
  bool rowIn[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    const int r = row0 + warp * 16 * MT + (i >> 1) * 16 + (i & 1) * 8 + g;
    rowIn[i] = r < p.N;
    wRow[i] = p.w + (rowIn[i] ? (long long)r * p.ldw : 0);
  }
  float total[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        total[m][n][i] = 0.0f;

  constexpr int kAhead = MT == 1 ? 4 : 2; // spans in flight per warp
  for (int k0 = kBegin; k0 < kEnd; k0 += p.stepK) {
    const int spans = (min(kEnd, k0 + p.stepK) - k0 + kSpan - 1) / kSpan;
    uint4 ring[kAhead][2 * MT];
    auto fetch = [&](uint4 (&dst)[2 * MT], int s) {
      const long long at = ((long long)k0 + s * kSpan + t * 32) >> 1;
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i)
        dst[i] = rowIn[i] && s < spans ? loadWeights<Whole>(wRow[i], at, rowBytes, p.vec)
                                       : make_uint4(0, 0, 0, 0);
    };
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
      fetch(ring[s], s);

    // Stage the step's activations and scales while the first weights travel.
    if (k0 != kBegin)
      __syncthreads(); // the previous step's have been read
    const int firstGroup = k0 / p.group;
    const int lastK = min(kEnd, k0 + spans * kSpan) - 1;
    const int groups = lastK / p.group - firstGroup + 1;
    if constexpr (A8) {
      for (int i = tid; i < groups * 8 * NT; i += 256)
        sASum[i] = 0;
      __syncthreads();
    }
    const int pieces = spans * 16 * NT * 8; // 8 activations each
    for (int i = tid; i < pieces; i += 256) {
      const int m = i / (spans * 16), q = i - m * (spans * 16);
      const int span = q >> 4, hi = (q >> 2) & 3, lo = q & 3; // k = span*128 + hi*32 + lo*8
      const int k = k0 + span * kSpan + hi * 32 + lo * 8;
      // Coarse: lane t holds 32 consecutive k, word j its j-th eight.  Fine: word c is
      // the c-th 32 of the span, lane t its t-th eight.
      const int ft = Fine ? lo : hi, fj = Fine ? hi : lo;
      const int flane = (m & 7) * 4 + ft, nt = m >> 3;
      unsigned char *dst =
          frag + size_t(span) * L::spanBytes + ((nt * 4 + fj) * 32 + flane) * L::pieceBytes;
      if constexpr (A8) {
        const int8_t *src = static_cast<const int8_t *>(p.a) + (long long)m * p.lda + k;
        uint32_t x = 0, y = 0;
        if (m < p.M && k < kEnd) {
          if (p.vecA && k + 8 <= kEnd) {
            const uint2 v = *reinterpret_cast<const uint2 *>(src);
            x = v.x;
            y = v.y;
          } else {
            for (int b = 0; b < 8; ++b)
              if (k + b < kEnd)
                (b < 4 ? x : y) |= uint32_t(uint8_t(src[b])) << (8 * (b & 3));
          }
        }
        *reinterpret_cast<uint2 *>(dst) =
            make_uint2(__byte_perm(x, y, 0x6420), __byte_perm(x, y, 0x7531));
        // The sum of the group's activations (integers: the order does not matter).
        if (m < p.M && k < kEnd) {
          const int sum = __dp4a(int(x), 0x01010101, __dp4a(int(y), 0x01010101, 0));
          atomicAdd(&sASum[(k / p.group - firstGroup) * 8 * NT + m], sum);
        }
      } else {
        const __nv_bfloat16 *src =
            static_cast<const __nv_bfloat16 *>(p.a) + (long long)m * p.lda + k;
        uint32_t v[4] = {0, 0, 0, 0};
        if (m < p.M && k < kEnd) {
          if (p.vecA && k + 8 <= kEnd) {
            const uint4 q4 = *reinterpret_cast<const uint4 *>(src);
            v[0] = q4.x;
            v[1] = q4.y;
            v[2] = q4.z;
            v[3] = q4.w;
          } else {
            for (int b = 0; b < 8; ++b)
              if (k + b < kEnd)
                v[b >> 1] |= uint32_t(__bfloat16_as_ushort(src[b])) << (16 * (b & 1));
          }
        }
        *reinterpret_cast<uint4 *>(dst) =
            make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632),
                       __byte_perm(v[1], v[3], 0x5410), __byte_perm(v[1], v[3], 0x7632));
      }
    }
    for (int i = tid; i < groups * L::rows; i += 256) {
      const int r = i / groups, gi = i - r * groups;
      const int n = row0 + r;
      float s = 0.0f;
      int z = 8;
      if (n < p.N) {
        const long long at = (long long)n * p.lds + firstGroup + gi;
        s = p.scaleF32 ? static_cast<const float *>(p.scale)[at]
                       : __bfloat162float(static_cast<const __nv_bfloat16 *>(p.scale)[at]);
        if (p.zero)
          z = p.zero[(long long)n * p.ldz + firstGroup + gi];
      }
      sScale[gi * L::rows + r] = s;
      const uint32_t b = __bfloat16_as_ushort(__float2bfloat16_rn(128.0f + float(z)));
      sBias[gi * L::rows + r] = A8 ? uint32_t(z) : (b << 16 | b);
    }
    if constexpr (A8) {
      for (int i = tid; i < groups * 8 * NT; i += 256) {
        const int gi = i / (8 * NT), m = i - gi * 8 * NT;
        const int b = max(k0, (firstGroup + gi) * p.group);
        sAScale[i] = m < p.M ? p.aScale[(long long)m * p.ldas + b / p.aGroup] : 0.0f;
      }
    }
    __syncthreads();

    Acc acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[m][n][i] = 0;
    // Adds the group sums, times their scales, to the totals.
    auto flush = [&](int gi) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int r = warp * 16 * MT + m * 16 + g;
        const float s0 = sScale[gi * L::rows + r], s1 = sScale[gi * L::rows + r + 8];
        int z0 = 0, z1 = 0;
        if constexpr (A8) {
          z0 = int(sBias[gi * L::rows + r]);
          z1 = int(sBias[gi * L::rows + r + 8]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (A8) {
              const int at = gi * 8 * NT + n * 8 + 2 * t + (i & 1);
              const int exact = acc[m][n][i] - (i < 2 ? z0 : z1) * sASum[at];
              total[m][n][i] =
                  fmaf((i < 2 ? s0 : s1) * sAScale[at], float(exact), total[m][n][i]);
            } else {
              total[m][n][i] = fmaf(i < 2 ? s0 : s1, acc[m][n][i], total[m][n][i]);
            }
            acc[m][n][i] = 0;
          }
        }
      }
    };

    int current = 0; // group (within the step) that acc belongs to
    for (int s0 = 0; s0 < spans; s0 += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int s = s0 + u;
        if (s >= spans)
          break;
        uint32_t words[2 * MT][4];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
          words[i][0] = ring[u][i].x;
          words[i][1] = ring[u][i].y;
          words[i][2] = ring[u][i].z;
          words[i][3] = ring[u][i].w;
          if constexpr (Fine)
            transposeQuad(words[i], t);
        }
        fetch(ring[u], s + kAhead);
        const unsigned char *piece = frag + size_t(s) * L::spanBytes + lane * L::pieceBytes;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (Fine || j == 0) {
            const int gi = (k0 + s * kSpan + (Fine ? j * 32 : 0)) / p.group - firstGroup;
            // (behind the last element there is no such group, and nothing to add)
            if (gi != current && gi < groups) {
              flush(current);
              current = gi;
            }
          }
          uint32_t a[MT][2][4];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint32_t w0 = words[2 * m][j], w1 = words[2 * m + 1][j];
            if constexpr (A8) {
              a[m][0][0] = w0 & 0x0f0f0f0fu;
              a[m][0][1] = w1 & 0x0f0f0f0fu;
              a[m][0][2] = (w0 >> 4) & 0x0f0f0f0fu;
              a[m][0][3] = (w1 >> 4) & 0x0f0f0f0fu;
            } else {
              const int r = warp * 16 * MT + m * 16 + g;
              const uint32_t b0 = p.zero ? sBias[current * L::rows + r] : 0x43084308u;
              const uint32_t b1 = p.zero ? sBias[current * L::rows + r + 8] : 0x43084308u;
              uint32_t p0[4], p1[4];
              unpackBf16(w0, b0, p0);
              unpackBf16(w1, b1, p1);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                a[m][h][0] = p0[2 * h];
                a[m][h][1] = p1[2 * h];
                a[m][h][2] = p0[2 * h + 1];
                a[m][h][3] = p1[2 * h + 1];
              }
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const unsigned char *src = piece + (n * 4 + j) * 32 * L::pieceBytes;
            if constexpr (A8) {
              const uint2 b = *reinterpret_cast<const uint2 *>(src);
#pragma unroll
              for (int m = 0; m < MT; ++m)
                mmaU8S8(acc[m][n], a[m][0], b.x, b.y);
            } else {
              const uint4 b = *reinterpret_cast<const uint4 *>(src);
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                mmaBf16(acc[m][n], a[m][0], b.x, b.y);
                mmaBf16(acc[m][n], a[m][1], b.z, b.w);
              }
            }
          }
        }
      }
    }
    flush(current);
  }

  // Partial sums of the cluster's CTAs, [weight row][activation row], added in rank
  // order: rank r finishes its share of the rows.
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = int(gridDim.y);
  constexpr int pitch = 8 * NT + 1;
  if (ranks == 1) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = n * 8 + 2 * t + (i & 1);
          const int r = row0 + warp * 16 * MT + m * 16 + (i >> 1) * 8 + g;
          if (r < p.N && col < p.M)
            p.out[(long long)col * p.ldc + r] = __float2bfloat16_rn(total[m][n][i]);
        }
    return;
  }
  float *part = reinterpret_cast<float *>(smem);
  __syncthreads(); // the staged operands have been read
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        part[(warp * 16 * MT + m * 16 + (i >> 1) * 8 + g) * pitch + n * 8 + 2 * t + (i & 1)] =
            total[m][n][i];
  cluster.sync();
  const int share = L::rows / ranks, mine = int(cluster.block_rank()) * share;
  for (int i = tid; i < share * p.M; i += 256) {
    const int col = i / share, r = mine + i - col * share;
    float sum = 0.0f;
    for (int c = 0; c < ranks; ++c)
      sum += cluster.map_shared_rank(part, c)[r * pitch + col];
    if (row0 + r < p.N)
      p.out[(long long)col * p.ldc + row0 + r] = __float2bfloat16_rn(sum);
  }
  cluster.sync(); // no CTA leaves while its memory is read
}

} // namespace

#define HC_W4(nt, mt, aname, A8, fname, Fine)                                              \
  extern "C" __global__ void __launch_bounds__(256, 2)                                      \
      hc_gemm_w4_##aname##_##fname##_m##nt(const __grid_constant__ W4Params p) {            \
    w4Body<nt, mt, A8, Fine, true>(p);                                                      \
  }                                                                                         \
  extern "C" __global__ void __launch_bounds__(256)                                         \
      hc_gemm_w4_##aname##_##fname##_m##nt##_any(const __grid_constant__ W4Params p) {      \
    w4Body<nt, mt, A8, Fine, false>(p);                                                     \
  }
#define HC_W4_ROWS(aname, A8, fname, Fine)                                                  \
  HC_W4(1, 1, aname, A8, fname, Fine)                                                       \
  HC_W4(2, 1, aname, A8, fname, Fine)                                                       \
  HC_W4(4, 1, aname, A8, fname, Fine)                                                       \
  HC_W4(8, 1, aname, A8, fname, Fine)
HC_W4_ROWS(bf16, false, coarse, false)
HC_W4_ROWS(bf16, false, fine, true)
HC_W4_ROWS(i8, true, coarse, false)
HC_W4_ROWS(i8, true, fine, true)

// ---- conversions for larger row counts ----------------------------------------------------
// out[k, n] = bf16((u - z) * s): the weights transposed into the [K, N] layout of the
// bf16 GEMM, tiles of 64 weight rows x 128 k through shared memory.  The product is
// rounded to bf16 here (half a step of 2^-8), which the few-row kernel above does not do.
extern "C" __global__ void __launch_bounds__(256)
    hc_dequant_w4_bf16(const __grid_constant__ W4Params p, __nv_bfloat16 *out,
                       long long outPitch) {
  __shared__ __nv_bfloat16 tile[128][64 + 2];
  const int tid = int(threadIdx.x);
  const int rowBytes = (p.K + 1) >> 1;
  const long long n0 = (long long)blockIdx.x * 64;
  const int k0 = int(blockIdx.y) * 128;
  {
    // Thread: weight row tid / 4, 32 k at (tid % 4) * 32.
    const int r = tid >> 2, kk = (tid & 3) * 32;
    const long long n = n0 + r;
    const uint4 q = n < p.N ? loadWeights<false>(p.w + n * p.ldw, (k0 + kk) >> 1, rowBytes, p.vec)
                            : make_uint4(0, 0, 0, 0);
    const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // Groups are multiples of 32 columns: one scale for the thread's 32 weights.
      float s = 0.0f, z = 8.0f;
      const int k = k0 + kk + j * 8;
      if (n < p.N && k < p.K) {
        const long long at = k / p.group;
        s = p.scaleF32 ? static_cast<const float *>(p.scale)[n * p.lds + at]
                       : __bfloat162float(
                             static_cast<const __nv_bfloat16 *>(p.scale)[n * p.lds + at]);
        if (p.zero)
          z = float(p.zero[n * p.ldz + at]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        tile[kk + j * 8 + i][r] =
            __float2bfloat16_rn((float((words[j] >> (4 * i)) & 15u) - z) * s);
    }
  }
  __syncthreads();
  // Rows of 64 n: 32 threads per row, one bf16 pair each.
  for (int i = tid; i < 128 * 32; i += 256) {
    const int kk = i >> 5, c = (i & 31) * 2;
    const int k = k0 + kk;
    const long long n = n0 + c;
    if (k < p.K && n < outPitch) { // outPitch is even, columns past N hold zeros
      const __nv_bfloat162 pair = __halves2bfloat162(tile[kk][c], tile[kk][c + 1]);
      *reinterpret_cast<__nv_bfloat162 *>(out + (long long)k * outPitch + n) = pair;
    }
  }
}

// out[m, k] = bf16(a[m, k] * aScale[m, k / aGroup]), int8 activations.
extern "C" __global__ void __launch_bounds__(256)
    hc_dequant_a8_bf16(const __grid_constant__ W4Params p, __nv_bfloat16 *out,
                       long long outPitch) {
  const long long m = blockIdx.x;
  const int8_t *a = static_cast<const int8_t *>(p.a) + m * p.lda;
  for (int k = int(blockIdx.y) * 256 + int(threadIdx.x); k < p.K; k += 256 * int(gridDim.y))
    out[m * outPitch + k] =
        __float2bfloat16_rn(float(a[k]) * p.aScale[m * p.ldas + k / p.aGroup]);
}
