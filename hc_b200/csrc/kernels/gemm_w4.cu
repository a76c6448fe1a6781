// Products of a few activation rows with 4-bit weights that have a scale (and maybe a
// zero point) for each group of K, and the conversions that larger row counts use:
//
//   out[m, n] = bf16( sa[m, k/ga] * sum_k a[m, k] * (u[n, k] - z[n, k/g]) * s[n, k/g] )
//
// u: 4-bit numbers 0..15, two per byte along K (even k in the low half), rows of
// weights one after another ([N, K/2]); z is 8 where there are no zero points; sa is 1
// for bf16 activations.
//
// With few rows the weights are the traffic (half a byte each, read once): every warp
// streams its own rows through a private ring in shared memory (cp.async, no barrier
// between warps in the stream), in the layout they are stored in.  The weights are the A operand of
// mma.sync (16 weight rows) and the activations the B operand (8 columns): a lane holds
// two rows' 32 consecutive weights of 128 (one 16-byte load each), and since a sum does
// not care about the order of its terms, K is permuted so that these are the very
// elements the lane feeds to the MMAs.  Legacy mma.sync rather than tcgen05: the operand
// registers need no detour, and its rate is not the bound (mma.sync measured 549 TFLOP/s
// in bf16 and 1127 TOP/s in int8 on this GPU; 8 rows at full bandwidth need 210).
//   * bf16: the bits of a nibble ARE the f16 number u * 2^-24 (a subnormal, which the
//     MMA takes as it is), and 16 u * 2^-24 one place further left: one AND per two
//     weights and one shift per eight unpack them, exactly.  (The logic pipe has half
//     the issue rate; shifting, masking, biasing and subtracting per pair held the
//     stream at 1.4 TB/s.)  The activations become f16 by a power of two per row and
//     segment of 128 (Fine: 32) k, those that meet 16 u a sixteenth of it: exact down
//     to 2^-24 of the segment's largest.
//     int8: the nibbles as unsigned bytes (m16n8k32, u8 x s8, exact int32 sums).
//   * a segment's sum is formed in the MMA's accumulators; z * sum(a) comes off and the
//     scale multiplies it into the fp32 total: no rounding of weights.
//   * Fine: groups that are not multiples of 128 (32, 64, 96 ...): a lane reads its four
//     words 16 bytes apart, so that an MMA stays inside 32 consecutive k.
//   * a CTA of 16 warps per SM walks over tiles of 16 weight rows; its warps divide K
//     among themselves (all 16 where K is long enough, else groups of warps take
//     different tiles), so a warp meets the same activations in every tile and they are
//     put into shared memory once.  A warp's loads run kSlots - 1 spans ahead, across
//     tiles.
//     The partial sums of a tile's warps meet in shared memory and are added in the
//     order of K.
// Measured with weights from HBM, us, for 1 / 4 / 8 rows of bf16 (6 where 8 do not fit), and
// the tcgen05 kernel (gemm_w4_umma.cu) whatever the rows:
//                  groups of 128           64                      32
//   8192 x 8192    16.2 / 19.5 / 24.7, 23  20.5 / 23.5 / 25.8, 26  23.2 / 26.3 / 29.0, 25
//   4096 x 4096     6.6 /  8.4 / 11.2, 12   8.0 /  9.7 / 12.3, 12   8.4 / 10.1 / 12.8, 11
//   14336 x 4096   16.5 / 18.5 / 22.0, 23  21.6 / 23.3 / 26.6, 26  23.7 / 25.2 / 28.3, 25
//   1024 x 8192     6.5 /  9.6 / 14.0, 12   7.6 / 10.4 / 12.5, 12   8.2 / 11.1 / 13.1, 12
// and int8 14.3 / 17.2 / 22.3 against 26 at 8192 x 8192 in groups of 128.  So with six to
// eight rows the other kernel is up to a sixth faster; this one is taken all the same
// wherever the rows fit, because its weights are not rounded: one to eight rows are one
// accuracy class.  What bounds it (2.1 TB/s of weights with one row) is the instructions
// that unpack (all of a warp's 32 lanes work for 8 columns, of which one row uses one) and,
// at 4096, the start of the stream.
#include "serving_math.cuh"

#include <type_traits>

using namespace hcs;

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
  int warpsK;   // warps that divide K: 1, 2, 4, 8 or 16
  int perWarp;  // scales a warp keeps per weight row: groups of K it can meet
  int vec;      // w: 16-byte aligned rows
  int vecA;     // a: 16-byte (int8: 8-byte) aligned rows
};

constexpr int kSpan = 128; // K of one pair of 16-byte loads

__device__ __forceinline__ void mmaF16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                       uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
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
// lies beyond the row reads as zero.
__device__ __forceinline__ uint4 loadWeights(const uint8_t *row, long long at, int bytes,
                                             int vec) {
  if (vec && at + 16 <= bytes)
    return loadStream16(row + at);
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (at + i < bytes)
      v[i >> 2] |= uint32_t(row[at + i]) << (8 * (i & 3));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

constexpr int kWarps = 16;
// A warp's ring: spans of 16 rows x 64 bytes, the 16-byte chunks of row r exchanged by
// an XOR with (r / 2) % 4 (free of bank conflicts for 16-byte and Fine's 4-byte reads).
constexpr int kSlots = 4;
constexpr int kSlotBytes = 16 * 64;

// Shared memory: the activation rows, per span of 128 k and row the pieces of 8
// activations in the order the lanes read them (piece (lane t, word j) at (4 j + t)
// pieces), as f16 pairs (0,4) (1,5)/16 (2,6) (3,7)/16 or as bytes (0,2,4,6) (1,3,5,7);
// then per segment of K (a span; Fine: 32) and column {sum of its activations in the
// accumulator's unit, that unit in the total's, times the activations' scale}; then per
// warp {scale, zero} of its 16 weight rows and its groups; then the partial sums of two
// tiles per warp; then 256 bytes of zeros that lanes without an activation row read.
template <bool A8, bool Fine> struct Layout {
  static constexpr int pieceBytes = A8 ? 8 : 16;
  static constexpr int spanBytes = 16 * pieceBytes;
  static constexpr int unit = Fine ? 32 : 128; // K of a segment
  static constexpr int segments = kSpan / unit;
};

// Whole: weight rows are 16-byte aligned and a multiple of 32 weights long.
template <bool A8, bool Fine, bool Whole>
__device__ __forceinline__ void w4Body(const W4Params &p) {
  using L = Layout<A8, Fine>;
  using Acc = typename std::conditional<A8, int, float>::type;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rowBytes = (p.K + 1) >> 1;
  const int spans = (p.K + kSpan - 1) / kSpan;

  // This warp's share of K and its tiles of 16 weight rows.
  const int wk = warp & (p.warpsK - 1), team = warp / p.warpsK;
  const int teams = kWarps / p.warpsK;
  const int sLo = wk * spans / p.warpsK, sHi = (wk + 1) * spans / p.warpsK;
  const int tiles = (p.N + 15) >> 4;
  const int tile0 = int(blockIdx.x) * teams + team, tileStep = int(gridDim.x) * teams;

  // Rows of activations are 64 bytes (int8: 32) apart modulo the banks.
  const int aPitch = spans * L::spanBytes + 4 * L::pieceBytes;
  float2 *sAct = reinterpret_cast<float2 *>(smem + p.M * aPitch);
  float2 *sScale = sAct + spans * L::segments * 8 + warp * p.perWarp * 16;
  float *sPart = reinterpret_cast<float *>(sAct + spans * L::segments * 8 +
                                           kWarps * p.perWarp * 16); // [2][warp][16 x 8]
  unsigned char *sNone = reinterpret_cast<unsigned char *>(sPart + 2 * kWarps * 128);

  // ---- the stream of weights: (tile, span) of this warp, kSlots - 1 spans ahead -------------
  unsigned char *ring = sNone + 256 + warp * kSlots * kSlotBytes;
  const int mix = (g >> 1) & 3; // (rows g and g + 8 alike)
  const uint32_t ringAt = hc::smemAddr(ring) + g * 64 + (t ^ mix) * 16;
  const int mine = tile0 < tiles && sLo < sHi ? (tiles - 1 - tile0) / tileStep + 1 : 0;
  int fTile = tile0, fLeft = sHi - sLo, fCount = mine * (sHi - sLo);
  uint32_t fSlot = 0; // bytes
  const uint8_t *fRow[2];
  auto rowsOf = [&](int tile) {
#pragma unroll
    for (int i = 0; i < 2; ++i) // rows past N read row N - 1 again and are not stored
      fRow[i] = p.w + (long long)min(tile * 16 + i * 8 + g, p.N - 1) * p.ldw + sLo * 64 + t * 16;
  };
  rowsOf(fTile);
  // In the last span of a row that is not a multiple of 128 weights, some lanes' bytes
  // lie behind the row.
  const bool ragged = sHi == spans && (spans - 1) * 64 + t * 16 >= rowBytes;
  auto fetch = [&]() {
    if (fCount > 0) {
      --fCount;
      if constexpr (Whole) { // (zeros for what is behind the row; the address is not read)
        const int in = ragged && fLeft == 1 ? 0 : 16;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                           ringAt + fSlot + i * 512),
                       "l"(fRow[i]), "r"(in)
                       : "memory");
      } else {
        const int at = (sHi - fLeft) * 64 + t * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<uint4 *>(ring + fSlot + i * 512 + g * 64 + (t ^ mix) * 16) =
              loadWeights(fRow[i] - at, at, rowBytes, p.vec);
      }
      fRow[0] += 64;
      fRow[1] += 64;
      fSlot = (fSlot + kSlotBytes) & (kSlots * kSlotBytes - 1);
      if (--fLeft == 0) {
        fLeft = sHi - sLo;
        fTile += tileStep;
        rowsOf(fTile);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int u = 0; u < kSlots - 1; ++u)
    fetch();

  // ---- its scales, a tile ahead in registers -------------------------------------------------
  const int gLo = sLo * kSpan / p.group;
  const int groups = sLo < sHi ? (min(p.K, sHi * kSpan) - 1) / p.group - gLo + 1 : 0;
  constexpr int kHeld = Fine ? 8 : 2; // per lane; more are loaded when their tile begins
  float heldScale[kHeld];
  int heldZero[kHeld];
  auto scaleAt = [&](long long at, long long atZero, float &s, int &z) {
    s = p.scaleF32 ? static_cast<const float *>(p.scale)[at]
                   : __bfloat162float(static_cast<const __nv_bfloat16 *>(p.scale)[at]);
    z = p.zero ? p.zero[atZero] : 8;
  };
  auto loadScales = [&](int tile) {
    const long long n = min(tile * 16 + (lane & 15), p.N - 1);
    const long long at = n * p.lds + gLo + (lane >> 4), atZero = n * p.ldz + gLo + (lane >> 4);
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (tile < tiles && 2 * i + (lane >> 4) < groups)
        scaleAt(at + 2 * i, atZero + 2 * i, heldScale[i], heldZero[i]);
  };
  auto putScales = [&](int tile) {
    auto put = [&](int gi, float s, int z) {
      sScale[gi * 16 + (lane & 15)] = make_float2(s, float(z));
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int gi = 2 * i + (lane >> 4);
      if (gi < groups)
        put(gi, heldScale[i], heldZero[i]);
    }
    const long long n = min(tile * 16 + (lane & 15), p.N - 1);
    for (int gi = 2 * kHeld + (lane >> 4); gi < groups; gi += 2) {
      float s;
      int z;
      scaleAt(n * p.lds + gLo + gi, n * p.ldz + gLo + gi, s, z);
      put(gi, s, z);
    }
  };
  loadScales(tile0);

  // ---- the activations, once -----------------------------------------------------------------
  for (int i = tid; i < spans * L::segments * 8; i += 32 * kWarps)
    if ((i & 7) >= p.M)
      sAct[i] = make_float2(0.0f, 0.0f);
  if (tid < 64)
    reinterpret_cast<uint32_t *>(sNone)[tid] = 0;
  constexpr int kLanes = Fine ? 4 : 16; // that hold a segment: 8 activations each
  constexpr int kBatch = 4;             // pieces per thread whose loads travel together
  const int perRow = spans * 16, pieces = p.M * perRow; // pieces of 8
  for (int q0 = tid; q0 - tid < pieces; q0 += kBatch * 32 * kWarps) {
    uint32_t v[kBatch][4];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = q0 + u * 32 * kWarps;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        v[u][c] = 0;
      if (i >= pieces)
        continue;
      const int m = i / perRow, k = (i - m * perRow) * 8;
      const char *src = static_cast<const char *>(p.a) +
                        ((long long)m * p.lda + k) * (A8 ? 1 : 2);
      if (p.vecA && k + 8 <= p.K) {
        if constexpr (A8) {
          const uint2 x = *reinterpret_cast<const uint2 *>(src);
          v[u][0] = x.x;
          v[u][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4 *>(src);
          v[u][0] = x.x;
          v[u][1] = x.y;
          v[u][2] = x.z;
          v[u][3] = x.w;
        }
      } else {
#pragma unroll
        for (int b = 0; b < 8; ++b)
          if (k + b < p.K) {
            if constexpr (A8)
              v[u][b >> 2] |= uint32_t(uint8_t(src[b])) << (8 * (b & 3));
            else
              v[u][b >> 1] |= uint32_t(reinterpret_cast<const uint16_t *>(src)[b])
                              << (16 * (b & 1));
          }
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      // (Pieces come in sixteens: a whole or half warp is at work, segments are whole.)
      const int i = q0 + u * 32 * kWarps;
      if (i >= pieces)
        continue;
      const uint32_t mask = i - lane + 32 <= pieces ? 0xffffffffu : 0x0000ffffu;
      const int m = i / perRow, q = i - m * perRow;
      const int span = q >> 4, hi = (q >> 2) & 3, lo = q & 3; // k = span*128 + hi*32 + lo*8
      // Coarse: lane t holds 32 consecutive k, word j its j-th eight.  Fine: word c is
      // the c-th 32 of the span, lane t its t-th eight.
      const int ft = Fine ? lo : hi, fj = Fine ? hi : lo;
      unsigned char *dst = smem + m * aPitch + span * L::spanBytes + (4 * fj + ft) * L::pieceBytes;
      float2 note;
      if constexpr (A8) {
        const uint32_t x = v[u][0], y = v[u][1];
        *reinterpret_cast<uint2 *>(dst) =
            make_uint2(__byte_perm(x, y, 0x6420), __byte_perm(x, y, 0x7531));
        int sum = __dp4a(int(x), 0x01010101, __dp4a(int(y), 0x01010101, 0));
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1)
          sum += __shfl_xor_sync(mask, sum, d);
        note.x = float(sum);
        note.y = 8 * q < p.K && p.aGroup < p.K
                     ? p.aScale[(long long)m * p.ldas + 8 * q / p.aGroup]
                     : 1.0f;
      } else {
        float e[8], sum = 0.0f, top = 0.0f;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          e[2 * b] = __uint_as_float(v[u][b] << 16);
          e[2 * b + 1] = __uint_as_float(v[u][b] & 0xffff0000u);
        }
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          sum = fmaf(e[b], 0.001953125f, sum); // (2^-9: the sum of the largest overflows)
          top = fmaxf(top, fabsf(e[b]));
        }
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) {
          sum += __shfl_xor_sync(mask, sum, d);
          top = fmaxf(top, __shfl_xor_sync(mask, top, d));
        }
        // up = 2^(14 - floor(log2 top)), within what float holds; down = 1 / up.
        const int expo = int(__float_as_uint(top) >> 23);
        const int shift = expo == 0 || expo == 255 ? 0 : max(-126, min(126, 14 - (expo - 127)));
        const float up = __uint_as_float(uint32_t(127 + shift) << 23);
        const float down = __uint_as_float(uint32_t(127 - shift) << 23);
#pragma unroll
        for (int b = 0; b < 8; ++b)
          e[b] *= b & 1 ? up * 0.0625f : up;
        auto pair = [](float a, float b) {
          const __half2 h = __floats2half2_rn(a, b);
          return *reinterpret_cast<const uint32_t *>(&h);
        };
        *reinterpret_cast<uint4 *>(dst) =
            make_uint4(pair(e[0], e[4]), pair(e[1], e[5]), pair(e[2], e[6]), pair(e[3], e[7]));
        // The accumulator counts in units of 2^-24 / up, the total in units of 2^-10: 2^14
        // down is at most the segment's largest activation, so that no factor overflows.
        note.x = sum * up * 3.0517578125e-05f; // 2^9 * 2^-24
        note.y = down * 16384.0f;
      }
      if ((q & (kLanes - 1)) == 0)
        sAct[(span * L::segments + (Fine ? hi : 0)) * 8 + m] = note;
    }
  }
  __syncthreads();

  // ---- tiles ----------------------------------------------------------------------------------
  float total[4];
  const bool live = g < p.M;
  const unsigned char *aRow = live ? smem + g * aPitch + t * L::pieceBytes : sNone;
  const int aStep = live ? L::spanBytes : 0;
  const int perGroup = p.group / L::unit;
  int left = 0, gi = 0, parity = 0;
  float2 c0, c1; // {scale, zero} of the current group, rows g and g + 8
  auto scalesOf = [&]() {
    c0 = sScale[gi * 16 + g];
    c1 = sScale[gi * 16 + g + 8];
  };
  // One span; the tile's sums are in `total` after the last one.
  uint32_t slot = 0;
  auto step = [&](int s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 2) : "memory");
    __syncwarp(); // (every lane's copies have arrived, and the slot before is read)
    uint32_t words[2][4];
    const unsigned char *from = ring + slot + g * 64;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (Fine) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          words[i][j] = *reinterpret_cast<const uint32_t *>(from + i * 512 + 16 * (j ^ mix) + 4 * t);
      } else {
        const uint4 v = *reinterpret_cast<const uint4 *>(from + i * 512 + 16 * (t ^ mix));
        words[i][0] = v.x;
        words[i][1] = v.y;
        words[i][2] = v.z;
        words[i][3] = v.w;
      }
    }
    slot = (slot + kSlotBytes) & (kSlots * kSlotBytes - 1);
    fetch(); // into the slot that the step before has read
    const unsigned char *piece = aRow + s * aStep;
    Acc acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (Fine || j == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[i] = 0;
      }
      const uint32_t w0 = words[0][j], w1 = words[1][j];
      if constexpr (A8) {
        const uint32_t a[4] = {w0 & 0x0f0f0f0fu, w1 & 0x0f0f0f0fu, (w0 >> 4) & 0x0f0f0f0fu,
                               (w1 >> 4) & 0x0f0f0f0fu};
        const uint2 b = *reinterpret_cast<const uint2 *>(piece + 4 * j * L::pieceBytes);
        mmaU8S8(acc, a, b.x, b.y);
      } else {
        const uint32_t h0 = w0 >> 8, h1 = w1 >> 8;
        const uint32_t a0[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u,
                                w1 & 0x00f000f0u};
        const uint32_t a1[4] = {h0 & 0x000f000fu, h1 & 0x000f000fu, h0 & 0x00f000f0u,
                                h1 & 0x00f000f0u};
        const uint4 b = *reinterpret_cast<const uint4 *>(piece + 4 * j * L::pieceBytes);
        mmaF16(acc, a0, b.x, b.y);
        mmaF16(acc, a1, b.z, b.w);
      }
      if (Fine || j == 3) {
        if (left == 0) { // (behind the last group there is nothing: its index stays)
          gi = min(gi + 1, groups - 1);
          left = perGroup;
          scalesOf();
        }
        --left;
        const float4 v = *reinterpret_cast<const float4 *>(
            sAct + (s * L::segments + (Fine ? j : 0)) * 8 + 2 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 &c = i < 2 ? c0 : c1;
          const float sum = i & 1 ? v.z : v.x, unit = i & 1 ? v.w : v.y;
          total[i] = fmaf(c.x * unit, fmaf(-c.y, sum, float(acc[i])), total[i]);
        }
      }
    }
  };
  const int firstLeft = (p.group - sLo * kSpan % p.group) / L::unit;
  auto beginTile = [&](int tile) {
    __syncwarp(); // the previous tile's scales have been read
    putScales(tile);
    loadScales(tile + tileStep);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      total[i] = 0.0f;
    gi = 0;
    left = firstLeft;
    scalesOf();
  };
  auto endTile = [&](int tile, int turn) {
    float *mine = sPart + (parity * kWarps + warp) * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i) // [column][row]
      mine[(2 * t + (i & 1)) * 16 + (i >> 1) * 8 + g] = total[i];
    if (p.warpsK == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(32 * p.warpsK) : "memory");
    // One of the team's warps adds them, in turn; the others go on (the two halves of
    // the buffer alternate, and that warp meets the others again before its half is
    // written).
    if (turn == wk) {
      const float *from = sPart + (parity * kWarps + team * p.warpsK) * 128;
      for (int i = lane; i < 16 * p.M; i += 32) {
        float sum = 0.0f;
        for (int w = 0; w < p.warpsK; ++w)
          sum += from[w * 128 + i];
        const int m = i >> 4, n = tile * 16 + (i & 15);
        if constexpr (!A8)
          sum *= 1024.0f;
        else if (p.aGroup >= p.K && p.K > 0) // one scale per activation row
          sum *= p.aScale[(long long)m * p.ldas];
        if (n < p.N)
          p.out[(long long)m * p.ldc + n] = __float2bfloat16_rn(sum);
      }
    }
    parity ^= 1;
  };

  int turn = 0;
  if (sLo < sHi) {
    int tile = tile0;
    for (int i = 0; i < mine; ++i) {
      beginTile(tile);
#pragma unroll 1
      for (int s = sLo; s < sHi; ++s)
        step(s);
      endTile(tile, turn);
      turn = turn + 1 == p.warpsK ? 0 : turn + 1;
      tile += tileStep;
    }
  } else { // (K = 0)
    for (int tile = tile0; tile < tiles; tile += tileStep) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        total[i] = 0.0f;
      endTile(tile, turn);
    }
  }
}

} // namespace

#define HC_W4(aname, A8, fname, Fine)                                                       \
  extern "C" __global__ void __launch_bounds__(512, 1)                                      \
      hc_gemm_w4_##aname##_##fname(const __grid_constant__ W4Params p) {                    \
    w4Body<A8, Fine, true>(p);                                                              \
  }                                                                                         \
  extern "C" __global__ void __launch_bounds__(512, 1)                                      \
      hc_gemm_w4_##aname##_##fname##_any(const __grid_constant__ W4Params p) {              \
    w4Body<A8, Fine, false>(p);                                                             \
  }
HC_W4(bf16, false, coarse, false)
HC_W4(bf16, false, fine, true)
HC_W4(i8, true, coarse, false)
HC_W4(i8, true, fine, true)

// ---- conversions for larger row counts ----------------------------------------------------
// out[k, n] = bf16((u - z) * s): the weights transposed into the [K, N] layout of the
// bf16 GEMM, tiles of 128 weight rows x 128 k through shared memory.  The product is
// rounded to bf16 here (half a step of 2^-8), which the few-row kernel above does not do.
// A thread takes 32 k of two neighbouring rows, so that a pair of bf16 is a pair of the
// output's neighbours: 128 + u by a mask and a bias, exact differences, one rounded
// product.  Bound by its stores.
extern "C" __global__ void __launch_bounds__(256)
    hc_dequant_w4_bf16(const __grid_constant__ W4Params p, __nv_bfloat16 *out,
                       long long outPitch) {
  __shared__ uint32_t tile[128][64 + 4]; // [k][pairs of rows]
  const int tid = int(threadIdx.x);
  const int rowBytes = (p.K + 1) >> 1;
  const long long n0 = (long long)blockIdx.x * 128;
  const int k0 = int(blockIdx.y) * 128;
  {
    const int r = tid & 63, kk = (tid >> 6) * 32;
    uint4 q[2];
    float s[2] = {0.0f, 0.0f};
    uint32_t z[2] = {8, 8};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long n = n0 + 2 * r + i;
      q[i] = make_uint4(0, 0, 0, 0);
      if (n < p.N && k0 + kk < p.K) {
        q[i] = loadWeights(p.w + n * p.ldw, (k0 + kk) >> 1, rowBytes, p.vec);
        // Groups are multiples of 32 columns: one scale for the thread's 32 weights.
        const long long at = (k0 + kk) / p.group;
        s[i] = p.scaleF32 ? static_cast<const float *>(p.scale)[n * p.lds + at]
                          : __bfloat162float(
                                static_cast<const __nv_bfloat16 *>(p.scale)[n * p.lds + at]);
        if (p.zero)
          z[i] = p.zero[n * p.ldz + at];
      }
    }
    uint32_t one28;
    asm volatile("mov.b32 %0, 0x43004300;" : "=r"(one28));
    // 128 + z in bf16 (exact up to z = 127).
    const uint32_t biasBits = 0x43004300u + z[0] + (z[1] << 16);
    const __nv_bfloat162 bias = *reinterpret_cast<const __nv_bfloat162 *>(&biasBits);
    const __nv_bfloat162 scale = __floats2bfloat162_rn(s[0], s[1]);
    const uint32_t wa[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
    const uint32_t wb[4] = {q[1].x, q[1].y, q[1].z, q[1].w};
#pragma unroll
    for (int j = 0; j < 16; ++j) { // byte j of both rows: k of 2j and 2j + 1
      const uint32_t both = __byte_perm(wa[j >> 2], wb[j >> 2], 0x4400 + 0x1111 * (j & 3));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v;
        asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(v) : "r"(both >> (4 * h)), "r"(one28));
        const __nv_bfloat162 x = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), bias);
        const __nv_bfloat162 y =
            p.scaleF32 ? __floats2bfloat162_rn(__low2float(x) * s[0], __high2float(x) * s[1])
                       : __hmul2(x, scale);
        tile[kk + 2 * j + h][r] = *reinterpret_cast<const uint32_t *>(&y);
      }
    }
  }
  __syncthreads();
  // Rows of 128 n: 16 threads each, 16 bytes per thread.  outPitch is a multiple of 16;
  // columns past N hold zeros.
  for (int i = tid; i < 128 * 16; i += 256) {
    const int kk = i >> 4, c = (i & 15) * 8;
    if (k0 + kk < p.K && n0 + c < outPitch)
      *reinterpret_cast<uint4 *>(out + (long long)(k0 + kk) * outPitch + n0 + c) =
          *reinterpret_cast<const uint4 *>(&tile[kk][c / 2]);
  }
}

// Activations as bf16 rows that TMA can read: int8 ones, times their scales or (scaled
// 0) as the integers they are; bf16 ones whose rows are not 16-byte aligned.
extern "C" __global__ void __launch_bounds__(256)
    hc_repack_a8_bf16(const __grid_constant__ W4Params p, __nv_bfloat16 *out,
                      long long outPitch, int scaled) {
  const long long m = blockIdx.x;
  const int8_t *a = static_cast<const int8_t *>(p.a) + m * p.lda;
  for (int k = int(blockIdx.y) * 256 + int(threadIdx.x); k < p.K; k += 256 * int(gridDim.y))
    out[m * outPitch + k] = __float2bfloat16_rn(
        scaled ? float(a[k]) * p.aScale[m * p.ldas + k / p.aGroup] : float(a[k]));
}
extern "C" __global__ void __launch_bounds__(256)
    hc_repack_a16_bf16(const __grid_constant__ W4Params p, __nv_bfloat16 *out,
                       long long outPitch, int) {
  const long long m = blockIdx.x;
  const __nv_bfloat16 *a = static_cast<const __nv_bfloat16 *>(p.a) + m * p.lda;
  for (int k = int(blockIdx.y) * 256 + int(threadIdx.x); k < p.K; k += 256 * int(gridDim.y))
    out[m * outPitch + k] = a[k];
}
