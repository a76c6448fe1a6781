// Entry points of the serving operators (include/hc_b200_kernels.h): checks of the
// arguments, the choice of a kernel variant, the launch.
#include "context.hpp"

#include "../kernels/kv_params.h"

#include <cuda.h> // CUtensorMap (type only; no driver call is made here)

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <cstring>

namespace {

long long ceilDiv(long long a, long long b) { return (a + b - 1) / b; }
bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// The kernels' parameter structures, as declared in their sources.
struct NormParams {
  const void *x;
  const void *residual;
  void *summed;
  const void *gain;
  void *out;
  float *scale;
  long long rows, cols;
  long long xPitch, residualPitch, summedPitch, outPitch, scalePitch;
  float eps;
  int group;
};

struct W4Params {
  const void *a;
  const float *aScale;
  const uint8_t *w;
  const void *scale;
  const uint8_t *zero;
  void *out;
  long long lda, ldas, ldw, lds, ldz, ldc;
  int M, N, K, group, aGroup;
  int scaleF32;
  int warpsK;
  int perWarp;
  int vec;
  int vecA;
};

struct W4UmmaParams {
  const void *scale;
  const uint8_t *zero;
  const float *rowScale;
  void *out;
  long long lds, ldz, rowScaleStride, ldc;
  int M, N, K;
  int group32;
  uint32_t inverse;
  int groups;
  int cols;
  int tilesM;
  int stagesA, stagesB, stagesW;
  int tmemCols;
  int packed;
  int *status;
};

struct AppendParams {
  HcKvCacheDev cache;
  HcKvPlaceDev place;
  const void *k, *v;
  long long tokenStride, headStride;
  long long tokenStrideV, headStrideV;
  int touched;
  int vec;
};

struct AttentionParams {
  HcKvCacheDev cache;
  HcKvPlaceDev place;
  const void *q;
  void *out;
  float *lse;
  long long qTokenStride, qHeadStride, outTokenStride, outHeadStride, lseStride;
  float scaleLog2;
  int share;
  int window;
  int rowTiles;
  int stepBlocks, stepRows;
  uint32_t blockInverse, shareInverse;
  int vecQ;
  unsigned *counters;
  float *partial;
};

struct KvRowsParams {
  HcKvCacheDev cache;
  HcKvPlaceDev place;
  const void *q;
  void *out;
  float *lse;
  long long qTokenStride, qHeadStride, outTokenStride, outHeadStride, lseStride;
  float scaleLog2;
  int share;
  int window;
  int rowTiles;
  int compact;
  int splits;
  uint32_t blockInverse, shareInverse;
  int vecQ, vecOut;
  unsigned *counters;
  float *partial;
  int *status;
};

static_assert(sizeof(HcKvCache) == sizeof(HcKvCacheDev) &&
                  offsetof(HcKvCache, dtype) == offsetof(HcKvCacheDev, dtype),
              "HcKvCache and its device form differ");
static_assert(sizeof(HcKvPlace) == sizeof(HcKvPlaceDev) &&
                  offsetof(HcKvPlace, maxNew) == offsetof(HcKvPlaceDev, maxNew),
              "HcKvPlace and its device form differ");

long long roundUp(long long a, long long b) { return ceilDiv(a, b) * b; }

// The weight-streaming kernel of hcGemmW4 takes up to 8 activation rows that fit in
// shared memory beside the scales of its 16 warps.
constexpr long long kW4FewRows = 8; // (both sides measured: gemm_w4.cu)
// Up to this many the weights are converted inside the tcgen05 kernel, for more by a pass
// of their own in front of the bf16 product (both sides measured: gemm_w4_umma.cu).
constexpr long long kW4FusedRows = 1024;

// The parts of hcGemmW4's workspace: the activations in bf16 (int8 ones, and bf16 ones
// that TMA cannot describe), then the weights: converted, or packed ones that TMA cannot
// describe copied to rows of 16 bytes.
size_t w4RowBytes(long long M, long long K, bool tma) {
  return tma ? 0 : size_t(roundUp(M * roundUp(K, 8) * 2, 256));
}
size_t w4WeightBytes(long long M, long long N, long long K, bool tma) {
  if (M > kW4FusedRows)
    return size_t(roundUp(N, 16) * K * 2);
  return tma ? 0 : size_t(N * roundUp(ceilDiv(K, 2), 16));
}

struct W4Few {
  int warpsK, perWarp;
  size_t smem;
};
W4Few w4Few(long long M, long long K, bool narrow, bool fine, long long group) {
  const long long spans = ceilDiv(K, 128);
  W4Few f{1, 0, 0};
  while (f.warpsK < 16 && f.warpsK * 2 <= spans)
    f.warpsK *= 2;
  f.perWarp = int(ceilDiv(ceilDiv(spans, f.warpsK) * 128, group) + 1);
  const long long piece = narrow ? 8 : 16;
  f.smem = size_t(M * (spans * 16 * piece + 4 * piece) + spans * (fine ? 4 : 1) * 64 +
                  16ll * f.perWarp * 128 + 2 * 16 * 512 + 256 + 16 * 4 * 1024 /* rings */);
  return f;
}
bool w4FitsFew(long long M, long long K, bool narrow, bool fine, long long group) {
  return M <= kW4FewRows && K <= (1 << 20) &&
         w4Few(M, K, narrow, fine, group).smem <= 227 * 1024;
}
// Whether groups are looked up per 128 columns.
bool w4Coarse(long long K, long long group) { return group % 128 == 0 || group >= K; }
// Which kernel a call of hcGemmW4 takes: the one for few rows or those of tcgen05.
bool w4RunsFew(HcContext c, long long M, long long K, bool narrow, long long group) {
  return c->w4Variant != 2 && w4FitsFew(M, K, narrow, !w4Coarse(K, group), group);
}

// Query rows (x head dimension) of a partial result in the attention's workspace, and
// the CTAs per SM that can hold two of them each.
constexpr size_t kSlotFloats = 8 * 256 + 2 * 16;
constexpr long long kAttentionCtasPerSm = 2;

// A slot of the kernel for many query rows, in floats, one per CTA of a divided unit.
constexpr size_t rowsSlotFloats(int cap) { return size_t(128) * (cap + 2); }
// The workspace: counters, then the slots of either kernel.
constexpr long long kCounters = HC_KV_COUNTER_BYTES / 4;
size_t attentionSlotBytes(HcContext c) {
  return size_t(c->smCount * kAttentionCtasPerSm) * 2 * kSlotFloats * 4;
}
size_t rowsSlotBytes(HcContext c) { return size_t(c->smCount) * rowsSlotFloats(256) * 4; }

// Query rows of a sequence and key/value head from which the tcgen05 kernel takes over:
// one more than the other kernel takes at a time.  (Measured, us, sixteen rows a time
// against tcgen05, one sequence of 16384 tokens of int8 and 32 of 4096 of e4m3:
//   16 rows  dim 64: 29, 48 / 29, 53   dim 128: 39, 66 / 35, 76   dim 256: 48, 126 / 54, 140
//   24 rows  dim 64: 37, 66 / 31, 56   dim 128: 41, 101 / 36, 79  dim 256: 62, 160 / 55, 140)
constexpr long long kManyRows = 17;

// Parts that a unit's tiles of tokens are divided into: those whose turns through the GPU
// are shortest, a turn costing its tiles and about eight more (the rows' conversion, the
// first tile's way through, joining).  `slots`, `units`: what the workspace holds.
int rowSplits(long long units, long long tiles, long long sms, long long slots, long long most) {
  long long best = 1, bestCost = 0;
  for (long long s = 1; s <= 64; ++s) {
    if (s > 1 && (s * 4 > tiles || s * units > slots || units > most))
      break;
    const long long cost = ceilDiv(units * s, sms) * (ceilDiv(tiles, s) + 8);
    if (s == 1 || cost < bestCost) {
      best = s;
      bestCost = cost;
    }
  }
  return int(best);
}

// Checks of the cache and of the rows' place that every entry point makes; copies them.
int checkKv(HcContext c, const char *who, const HcKvCache *cache, const HcKvPlace *place,
            HcKvCacheDev &outCache, HcKvPlaceDev &outPlace) {
  if (!cache || !place)
    return c->fail("%s: null cache or place", who);
  if (cache->dtype != HC_I8 && cache->dtype != HC_E4M3)
    return c->fail("%s: unsupported cache dtype %d", who, cache->dtype);
  if (cache->block < 16 || cache->block > 256 || cache->block % 16)
    return c->fail("%s: block of %d tokens (a multiple of 16 up to 256 expected)", who,
                   cache->block);
  if (cache->dim < 16 || cache->dim > 256 || cache->dim % 16)
    return c->fail("%s: head dimension %d (a multiple of 16 up to 256 expected)", who, cache->dim);
  if (cache->pages < 0 || cache->heads < 1 || cache->heads > 32767)
    return c->fail("%s: %d pages of %d heads", who, cache->pages, cache->heads);
  if (cache->tokenStride < cache->dim || cache->headStride < 0 || cache->pageStride < 0 ||
      cache->tokenStride % 16 || cache->headStride % 16 || cache->pageStride % 16 ||
      !aligned(cache->k, 16) || !aligned(cache->v, 16))
    return c->fail("%s: the cache's rows must be 16-byte aligned", who);
  if (cache->tokenStride > 0x7fffffffLL / cache->block)
    return c->fail("%s: a page of %d tokens, %lld apart, spans 2^31 bytes or more", who,
                   cache->block, cache->tokenStride);
  if (cache->pageStride > 0x7fffffffLL || cache->scalePitch > 0x7fffffffLL)
    return c->fail("%s: pages %lld bytes (scales %lld) apart: below 2^31 expected", who,
                   cache->pageStride, cache->scalePitch);
  if (cache->scalePitch < cache->heads)
    return c->fail("%s: scale pitch %lld is below the %d heads", who, cache->scalePitch,
                   cache->heads);
  if (place->seqs < 0 || place->width < 0 || place->tokens < 0 || place->maxNew < 0 ||
      place->tablePitch < place->width ||
      (long long)place->width * cache->block > 0x7fffffffLL - 512)
    return c->fail("%s: invalid place (%d sequences, %d blocks, %d tokens, at most %d new)", who,
                   place->seqs, place->width, place->tokens, place->maxNew);
  if (!place->starts && place->tokens < place->seqs)
    return c->fail("%s: %d rows for %d sequences of one new token", who, place->tokens,
                   place->seqs);
  if (place->seqs > 0 && place->tokens > 0 &&
      (!place->lengths || (place->width > 0 && !place->table)))
    return c->fail("%s: null lengths or table", who);
  if (cache->pages > 0 && (!cache->k || !cache->v || !cache->kScale || !cache->vScale))
    return c->fail("%s: null cache buffer", who);
  std::memcpy(&outCache, cache, sizeof outCache);
  std::memcpy(&outPlace, place, sizeof outPlace);
  if (!place->starts)
    outPlace.maxNew = std::min(outPlace.maxNew, 1);
  outPlace.maxNew = std::min(outPlace.maxNew, outPlace.tokens);
  return 0;
}

// Which image defines which family of kernels (names start with `prefix`).
const struct {
  const char *prefix, *image;
} kFamilies[] = {
    // hc_add_rms_norm_{bf16,f32}_{same,i8,e4m3}_{t<threads>_v<packets>,generic}
    {"hc_add_rms_norm_", "add_rms_norm"},
    // hc_gemm_w4_{bf16,i8}_{coarse,fine}[_any]: activation type, groups that are
    // multiples of 128 or not, weight rows that 16-byte loads do not tile; and the
    // conversions
    // hc_gemm_w4_umma_{narrow,wide}_{coarse,fine}_{bf16,f32}: up to 64 activation rows per
    // tile or up to 256, groups alike, type of the scales
    {"hc_gemm_w4_umma_", "gemm_w4_umma"},
    {"hc_gemm_w4_", "gemm_w4"},
    {"hc_dequant_w4_", "gemm_w4"},
    {"hc_repack_", "gemm_w4"},
    {"hc_kv_append_", "kv_append"},       // _{i8,e4m3}_{warp,cta}
    // hc_kv_attention_rows_{i8,e4m3}_d{64,128,256}: many query rows, on tcgen05
    {"hc_kv_attention_rows_", "kv_attention_umma"},
    {"hc_kv_attention_", "kv_attention"}, // _{i8,e4m3}_d{64,128,256}_r{1,2}[_any]
};

} // namespace

const char *hcServingImageOf(const char *kernel) {
  for (const auto &f : kFamilies)
    if (std::strncmp(kernel, f.prefix, std::strlen(f.prefix)) == 0)
      return f.image;
  return nullptr;
}

extern "C" {

int hcAddRmsNorm(HcContext c, const void *x, const void *residual, void *summed,
                 const void *gain, void *out, float *scaleOut, long long rows, long long cols,
                 long long xPitch, long long residualPitch, long long summedPitch,
                 long long outPitch, long long scalePitch, long long group, float eps,
                 int dtype, int outDtype) {
  if (!c)
    return 1;
  if (dtype != HC_BF16 && dtype != HC_F32)
    return c->fail("hcAddRmsNorm: unsupported dtype %d", dtype);
  const bool narrow = outDtype == HC_I8 || outDtype == HC_E4M3;
  if (!narrow && outDtype != dtype)
    return c->fail("hcAddRmsNorm: unsupported output dtype %d", outDtype);
  if (rows < 0 || cols < 0 || rows > 0x7fffffffLL || xPitch < cols || outPitch < cols ||
      (residual && residualPitch < cols) || (summed && summedPitch < cols))
    return c->fail("hcAddRmsNorm: invalid shape %lld x %lld", rows, cols);
  if (group < 0 || group > 0x7fffffffLL || (group && !narrow))
    return c->fail("hcAddRmsNorm: invalid group %lld", group);
  if (group >= cols)
    group = 0; // one group is the whole row
  const long long groups = group ? ceilDiv(cols, group) : 1;
  if (narrow && scalePitch < groups)
    return c->fail("hcAddRmsNorm: scale pitch %lld is below the %lld groups of a row",
                   scalePitch, groups);
  if (!(eps >= 0.0f))
    return c->fail("hcAddRmsNorm: eps must not be negative");
  if (rows == 0 || cols == 0)
    return 0;
  if (!x || !gain || !out || (narrow && !scaleOut))
    return c->fail("hcAddRmsNorm: null buffer");
  if (summed && !residual)
    return c->fail("hcAddRmsNorm: a sum to write but no residual");
  NormParams p{x,      residual,     summed,        gain,        out,      scaleOut,  rows, cols,
               xPitch, residualPitch, summedPitch,  outPitch,    scalePitch, eps,     int(group)};
  const char *tname = dtype == HC_BF16 ? "bf16" : "f32";
  const char *oname = outDtype == HC_I8 ? "i8" : outDtype == HC_E4M3 ? "e4m3" : "same";
  // Packets of 8 elements: 16-byte loads (bf16), two of them (f32).  Groups that are
  // not a power of two up to 32 packets cross lanes unevenly: element by element.
  const int step = dtype == HC_BF16 ? 8 : 4; // elements of 16 bytes
  const bool fits = cols % 8 == 0 && cols <= 16384 && xPitch % step == 0 && aligned(x, 16) &&
                    aligned(gain, 16) &&
                    (!residual || (residualPitch % step == 0 && aligned(residual, 16))) &&
                    (!summed || (summedPitch % step == 0 && aligned(summed, 16))) &&
                    (narrow ? outPitch % 8 == 0 && aligned(out, 8)
                            : outPitch % step == 0 && aligned(out, 16)) &&
                    (group == 0 || (group >= 8 && group <= 256 && (group & (group - 1)) == 0));
  char name[64];
  if (!fits) {
    size_t smem = size_t(cols) * 4;
    int cached = 1;
    if (smem > 160 * 1024) { // does not fit: the kernel computes the row's values again
      smem = 0;
      cached = 0;
    }
    std::snprintf(name, sizeof name, "hc_add_rms_norm_%s_%s_generic", tname, oname);
    void *args[] = {&p, &cached};
    return c->launch(name, size_t(rows), 1, 1, 256, args, 2, smem);
  }
  const long long packets = cols / 8;
  // Threads x packets per thread that cover a row.  With few rows a row gets more
  // threads of fewer packets (latency); with many, threads that hold more packets
  // keep more loads in flight per resident CTA.
  const bool few = rows <= 2 * c->smCount;
  int threads = 512, v = 4;
  if (packets <= 64)
    threads = 64, v = 1;
  else if (packets <= 128)
    threads = 128, v = 1;
  else if (packets <= 256)
    threads = few ? 256 : 128, v = few ? 1 : 2;
  else if (packets <= 512)
    threads = few ? 512 : 256, v = few ? 1 : 2;
  else if (packets <= 1024)
    threads = few ? 512 : 256, v = few ? 2 : 4;
  std::snprintf(name, sizeof name, "hc_add_rms_norm_%s_%s_t%d_v%d", tname, oname, threads, v);
  void *args[] = {&p};
  return c->launch(name, size_t(rows), 1, 1, size_t(threads), args, 1, 0);
}

size_t hcGemmW4WorkspaceBytes(long long M, long long N, long long K, long long lda,
                              long long ldw, int aDtype) {
  if (M <= 0 || N <= 0 || K <= 0)
    return 0;
  return w4RowBytes(M, K, aDtype != HC_I8 && lda % 8 == 0) + w4WeightBytes(M, N, K, ldw % 16 == 0);
}

size_t hcGemmW4CallWorkspaceBytes(HcContext c, long long M, long long N, long long K,
                                  long long group, long long lda, long long ldw, int aDtype) {
  if (!c || group <= 0 || w4RunsFew(c, M, K, aDtype == HC_I8, group))
    return 0;
  return hcGemmW4WorkspaceBytes(M, N, K, lda, ldw, aDtype);
}

int hcGemmW4(HcContext c, const void *a, const float *aScale, const void *w, const void *scale,
             const void *zero, void *out, void *workspace, size_t workspaceBytes, long long M,
             long long N, long long K, long long group, long long aGroup, long long lda,
             long long ldas, long long ldw, long long lds, long long ldz, long long ldc,
             int aDtype, int scaleDtype) {
  if (!c)
    return 1;
  if (aDtype != HC_BF16 && aDtype != HC_I8)
    return c->fail("hcGemmW4: unsupported activation dtype %d", aDtype);
  if (scaleDtype != HC_BF16 && scaleDtype != HC_F32)
    return c->fail("hcGemmW4: unsupported scale dtype %d", scaleDtype);
  constexpr long long kMost = 1ll << 30;
  if (M < 0 || N < 0 || K < 0 || M > kMost || N > kMost || K > kMost || lda < K || ldc < N ||
      ldw < ceilDiv(K, 2))
    return c->fail("hcGemmW4: invalid shape M=%lld N=%lld K=%lld (lda %lld ldw %lld ldc %lld)", M,
                   N, K, lda, ldw, ldc);
  if (group <= 0 || group % 32 || group > kMost)
    return c->fail("hcGemmW4: group %lld is not a multiple of 32", group);
  if (aGroup == 0 || aGroup >= K)
    aGroup = std::max<long long>(K, 1);
  else if (aDtype == HC_I8 && (aGroup < 0 || aGroup % group))
    return c->fail("hcGemmW4: the activations' group %lld is not a multiple of the weights' %lld",
                   aGroup, group);
  const long long groups = ceilDiv(K, group);
  if (lds < groups || (zero && ldz < groups) ||
      (aDtype == HC_I8 && ldas < ceilDiv(K, aGroup)))
    return c->fail("hcGemmW4: a pitch is below the %lld groups of a row", groups);
  if (M == 0 || N == 0)
    return 0;
  if (!out || (K > 0 && (!a || !w || !scale || (aDtype == HC_I8 && !aScale))))
    return c->fail("hcGemmW4: null buffer");
  W4Params p{};
  p.a = a;
  p.aScale = aScale;
  p.w = static_cast<const uint8_t *>(w);
  p.scale = scale;
  p.zero = static_cast<const uint8_t *>(zero);
  p.out = out;
  p.lda = lda, p.ldas = ldas, p.ldw = ldw, p.lds = lds, p.ldz = ldz, p.ldc = ldc;
  p.M = int(M), p.N = int(N), p.K = int(K), p.group = int(group), p.aGroup = int(aGroup);
  p.scaleF32 = scaleDtype == HC_F32;
  p.vec = ldw % 16 == 0 && aligned(w, 16);
  const bool narrow = aDtype == HC_I8;
  p.vecA = narrow ? lda % 8 == 0 && aligned(a, 8) : lda % 8 == 0 && aligned(a, 16);
  char name[64];
  const bool coarse = w4Coarse(K, group);
  const bool few = w4RunsFew(c, M, K, narrow, group);
  if (c->w4Variant == 1 && !few)
    return c->fail("hcGemmW4: %lld rows of %lld do not fit the kernel for few rows", M, K);
  if (K == 0) // zeros
    return hcGemmBf16(c, a, w, out, M, N, 0, lda, N, ldc);
  if (few) {
    const W4Few f = w4Few(M, K, narrow, !coarse, group);
    p.warpsK = f.warpsK;
    p.perWarp = f.perWarp;
    const long long teams = 16 / f.warpsK;
    const long long ctas = std::min<long long>(c->smCount, ceilDiv(ceilDiv(N, 16), teams));
    std::snprintf(name, sizeof name, "hc_gemm_w4_%s_%s%s", narrow ? "i8" : "bf16",
                  coarse ? "coarse" : "fine", p.vec && K % 32 == 0 ? "" : "_any");
    void *args[] = {&p};
    return c->launch(name, size_t(ctas), 1, 1, 512, args, 1, f.smem);
  }
  if (c->ccMajor != 10)
    return c->fail("hcGemmW4: this form needs a device with tcgen05");
  const bool tmaRows = !narrow && lda % 8 == 0 && aligned(a, 16);
  const size_t rowBytes = w4RowBytes(M, K, tmaRows);
  const size_t need = rowBytes + w4WeightBytes(M, N, K, p.vec);
  if (need && (!workspace || workspaceBytes < need || !aligned(workspace, 256)))
    return c->fail("hcGemmW4: %lld rows need a 256-byte aligned workspace of %zu bytes, got %zu",
                   M, need, workspaceBytes);
  // The activations as bf16 rows that TMA can read.  A single scale per int8 row stays
  // out of them (the integers are exact in bf16): the products' epilogues apply it.  (That
  // of the CUDA-core product, which "gemm_variant" 3 forces, has none.)
  const bool fused = M <= kW4FusedRows;
  const bool rowScaled = narrow && aGroup >= K && (fused || c->gemmVariant != 3);
  long long pitchA = lda;
  if (!tmaRows) {
    void *rows = workspace;
    pitchA = roundUp(K, 8);
    int scaled = narrow && !rowScaled;
    void *args[] = {&p, &rows, &pitchA, &scaled};
    if (c->launch(narrow ? "hc_repack_a8_bf16" : "hc_repack_a16_bf16", size_t(M),
                  size_t(std::min<long long>(ceilDiv(K, 256), 16)), 1, 256, args, 4, 0))
      return 1;
    a = rows;
  }
  void *const weights = static_cast<char *>(workspace) + rowBytes;
  if (fused) {
    if (!p.vec) {
      const long long bytes = ceilDiv(K, 2);
      if (hcCopy2D(c, w, weights, N, bytes, ldw, roundUp(bytes, 16), 1))
        return 1;
      w = weights;
      ldw = roundUp(bytes, 16);
    }
    W4UmmaParams u{};
    u.scale = scale, u.zero = p.zero, u.out = out;
    u.rowScale = rowScaled ? aScale : nullptr;
    u.rowScaleStride = ldas;
    u.lds = lds, u.ldz = ldz, u.ldc = ldc;
    u.M = p.M, u.N = p.N, u.K = p.K;
    u.group32 = int(group / 32);
    u.inverse = u.group32 == 1 ? 0 : uint32_t((1ull << 32) / unsigned(u.group32));
    u.groups = int(groups);
    u.packed = group == 32 && lds % 4 == 0 && aligned(scale, 8) &&
               (!zero || (ldz % 4 == 0 && aligned(zero, 4)));
    u.tilesM = int(ceilDiv(M, 256));
    u.cols = int(roundUp(ceilDiv(M, u.tilesM), 16));
    u.status = c->statusWord;
    // Up to 64 columns: two CTAs per SM, half of the tensor memory each.
    const bool two = u.cols <= 64;
    u.tmemCols = two ? 256 : 512;
    const long long stageBytes = (long long)u.cols * 256, wBytes = 16 * 1024;
    u.stagesA = int(std::min(6ll, (u.tmemCols - roundUp(u.cols, 32)) / 64));
    const long long room = (two ? 108ll : 224ll) * 1024;
    u.stagesB = int(std::min(6ll, (room - 3 * wBytes) / stageBytes));
    u.stagesW = int(std::min(6ll, (room - u.stagesB * stageBytes) / wBytes));
    const long long tiles = ceilDiv(N, 128) * u.tilesM, pairs = ceilDiv(K, 256);
    // CTAs that share a tile's K: as many as fit the GPU at once, 512 k each at least.
    const long long slots = c->smCount * (two ? 2 : 1);
    const long long splits = std::max<long long>(1, std::min({8ll, slots / tiles, pairs / 2}));
    alignas(64) CUtensorMap mapB, mapW;
    if (olxEncodeTensorMap2D(c->device, &mapB, /*bf16*/ 0, a, size_t(M), size_t(K),
                             size_t(pitchA) * 2, unsigned(u.cols), 64, 128) ||
        olxEncodeTensorMap2D(c->device, &mapW, /*bytes*/ 2, w, size_t(N), size_t(ceilDiv(K, 2)),
                             size_t(ldw), 128, 128, 128))
      return c->fail("tensor map encoding failed: %s", c->lastError.c_str());
    std::snprintf(name, sizeof name, "hc_gemm_w4_umma_%s_%s_%s", two ? "narrow" : "wide",
                  coarse ? "coarse" : "fine", p.scaleF32 ? "f32" : "bf16");
    void *args[] = {&mapB, &mapW, &u};
    return c->launchCluster(name, size_t(tiles), size_t(splits), size_t(splits), two ? 384 : 640,
                            args,
                            size_t(u.stagesB * stageBytes + u.stagesW * wBytes + 1024));
  }
  const long long pitch = roundUp(N, 16);
  long long outPitch = pitch;
  void *converted = weights;
  void *args[] = {&p, &converted, &outPitch};
  if (ceilDiv(K, 128) > 65535)
    return c->fail("hcGemmW4: K=%lld is too large for a conversion", K);
  if (c->launch("hc_dequant_w4_bf16", size_t(ceilDiv(N, 128)), size_t(ceilDiv(K, 128)), 1, 256,
                args, 3, 0))
    return 1;
  if (rowScaled)
    return hcGemmBf16RowScaled(c, a, weights, aScale, ldas, out, M, N, K, pitchA, pitch, ldc);
  return hcGemmBf16(c, a, weights, out, M, N, K, pitchA, pitch, ldc);
}

int hcKvAppend(HcContext c, const HcKvCache *cache, const HcKvPlace *place, const void *k,
               const void *v, long long kTokenStride, long long kHeadStride,
               long long vTokenStride, long long vHeadStride) {
  if (!c)
    return 1;
  AppendParams p{};
  if (checkKv(c, "hcKvAppend", cache, place, p.cache, p.place))
    return 1;
  if (kTokenStride < 0 || kHeadStride < 0 || vTokenStride < 0 || vHeadStride < 0)
    return c->fail("hcKvAppend: negative strides");
  if (p.place.seqs == 0 || p.place.tokens == 0 || p.place.maxNew == 0 || p.place.width == 0 ||
      p.cache.pages == 0)
    return 0;
  if (!k || !v)
    return c->fail("hcKvAppend: null buffer");
  p.k = k, p.v = v;
  p.tokenStride = kTokenStride, p.headStride = kHeadStride;
  p.tokenStrideV = vTokenStride, p.headStrideV = vHeadStride;
  p.touched = hcKvTouchedBlocks(p.place.maxNew, p.cache.block);
  p.vec = kTokenStride % 8 == 0 && kHeadStride % 8 == 0 && vTokenStride % 8 == 0 &&
          vHeadStride % 8 == 0 && aligned(k, 16) && aligned(v, 16);
  const long long blocks = (long long)p.place.seqs * p.touched;
  if (blocks > 0x7fffffffLL)
    return c->fail("hcKvAppend: %d sequences of up to %d new tokens are too many", p.place.seqs,
                   p.place.maxNew);
  // A warp per unit (a block's keys or values of one head) where they are many, or small
  // (four turns of eight elements per lane); else a CTA.
  const long long units = blocks * 2 * p.cache.heads;
  const bool warps = units >= 16 * c->smCount ||
                     (long long)std::min(p.place.maxNew, p.cache.block) * p.cache.dim <= 1024;
  char name[64];
  std::snprintf(name, sizeof name, "hc_kv_append_%s_%s", p.cache.dtype == HC_I8 ? "i8" : "e4m3",
                warps ? "warp" : "cta");
  void *args[] = {&p};
  return c->launch(name, size_t(blocks),
                   size_t(warps ? ceilDiv(2 * p.cache.heads, 4) : 2 * p.cache.heads), 1,
                   warps ? 128 : 256, args, 1, 0);
}

size_t hcKvAttentionWorkspaceBytes(HcContext c) {
  if (!c)
    return 0;
  return HC_KV_COUNTER_BYTES + std::max(attentionSlotBytes(c), rowsSlotBytes(c));
}

int hcKvAttention(HcContext c, const HcKvCache *cache, const HcKvPlace *place, const void *q,
                  void *out, float *lse, int share, float scale, int window,
                  long long qTokenStride, long long qHeadStride, long long outTokenStride,
                  long long outHeadStride, long long lseStride, void *workspace,
                  size_t workspaceBytes) {
  if (!c)
    return 1;
  AttentionParams p{};
  if (checkKv(c, "hcKvAttention", cache, place, p.cache, p.place))
    return 1;
  if (share < 1 || share > 65535 || window < 0 || !std::isfinite(scale))
    return c->fail("hcKvAttention: %d query heads per key/value head, window %d, scale %g", share,
                   window, double(scale));
  if (qTokenStride < 0 || qHeadStride < 0 || outTokenStride < 0 || outHeadStride < 0 ||
      (lse && lseStride < (long long)p.cache.heads * share))
    return c->fail("hcKvAttention: invalid strides");
  if (p.place.seqs == 0 || p.place.tokens == 0)
    return 0;
  if (!q || !out)
    return c->fail("hcKvAttention: null buffer");
  if (!aligned(out, 8) || outTokenStride % 4 || outHeadStride % 4)
    return c->fail("hcKvAttention: the rows of out must be 8-byte aligned");
  if (!workspace || workspaceBytes < hcKvAttentionWorkspaceBytes(c) || !aligned(workspace, 256))
    return c->fail("hcKvAttention: a 256-byte aligned workspace of %zu bytes is needed, got %zu",
                   hcKvAttentionWorkspaceBytes(c), workspaceBytes);
  p.q = q, p.out = out, p.lse = lse;
  p.qTokenStride = qTokenStride, p.qHeadStride = qHeadStride;
  p.outTokenStride = outTokenStride, p.outHeadStride = outHeadStride;
  p.lseStride = lseStride;
  p.scaleLog2 = scale * 1.44269504088896341f;
  p.share = share, p.window = window;
  const long long maxRows = (long long)std::max(p.place.maxNew, 1) * share;
  const int cap = p.cache.dim <= 64 ? 64 : p.cache.dim <= 128 ? 128 : 256;
  // (The kernels divide row numbers by products.)
  if (maxRows * share > 0x7fffffffLL)
    return c->fail("hcKvAttention: up to %lld query rows are too many for one call", maxRows);
  p.stepBlocks = 16 / p.cache.block;
  p.stepRows = 16 % p.cache.block;
  auto inverse = [](unsigned n) { return n == 1 ? 0u : uint32_t((1ull << 32) / n + 1); };
  p.blockInverse = inverse(unsigned(p.cache.block) / 16);
  p.shareInverse = inverse(unsigned(share));
  p.vecQ = aligned(q, 16) && qTokenStride % 8 == 0 && qHeadStride % 8 == 0;
  p.counters = static_cast<unsigned *>(workspace);
  p.partial =
      reinterpret_cast<float *>(static_cast<char *>(workspace) + HC_KV_COUNTER_BYTES);
  char name[64];
  const char *const type = p.cache.dtype == HC_I8 ? "i8" : "e4m3";
  if (c->attentionVariant != 1 && c->ccMajor == 10 &&
      (maxRows >= kManyRows || c->attentionVariant == 2)) {
    KvRowsParams u{};
    u.cache = p.cache, u.place = p.place;
    u.q = p.q, u.out = p.out, u.lse = p.lse;
    u.qTokenStride = qTokenStride, u.qHeadStride = qHeadStride;
    u.outTokenStride = outTokenStride, u.outHeadStride = outHeadStride, u.lseStride = lseStride;
    u.scaleLog2 = p.scaleLog2, u.share = share, u.window = window;
    u.rowTiles = int(ceilDiv(maxRows, 128));
    // Where few sequences have as many rows as the longest: the units that there are.
    long long unitsOfHead = (long long)p.place.seqs * u.rowTiles;
    const long long most = (long long)p.place.tokens * share / 128 + p.place.seqs;
    u.compact = most < unitsOfHead;
    unitsOfHead = std::min(unitsOfHead, most);
    u.blockInverse = p.blockInverse, u.shareInverse = p.shareInverse, u.vecQ = p.vecQ;
    u.vecOut = aligned(out, 16) && outTokenStride % 8 == 0 && outHeadStride % 8 == 0;
    u.counters = p.counters, u.partial = p.partial, u.status = c->statusWord;
    const long long units = unitsOfHead * p.cache.heads;
    if (units > 0x7fffffffLL)
      return c->fail("hcKvAttention: %lld tiles of query rows are too many", units);
    const int step = cap == 256 ? 64 : 128;
    long long reach = (long long)p.place.width * p.cache.block; // tokens that a row can see
    if (window > 0)
      reach = std::min<long long>(reach, window + ceilDiv(128, share));
    u.splits = rowSplits(units, ceilDiv(reach, step), c->smCount,
                         (long long)(rowsSlotBytes(c) / (rowsSlotFloats(cap) * 4)),
                         kCounters);
    std::snprintf(name, sizeof name, "hc_kv_attention_rows_%s_d%d", type, cap);
    void *args[] = {&u};
    return c->launch(name, size_t(units), size_t(u.splits), 1, 544, args, 1,
                     size_t(cap / 64) * 128 * (128 + 4 * step) + 1024);
  }
  // Eight query rows per MMA; sixteen share one reading of the cache where there are as
  // many and the registers allow it.
  const int nt = maxRows > 8 && cap <= 128 ? 2 : 1;
  const long long rowTiles = ceilDiv(maxRows, 8 * nt);
  const long long tiles = (long long)p.place.seqs * p.cache.heads * rowTiles *
                          (ceilDiv((long long)p.place.width * p.cache.block, 16) + 1);
  if (tiles > 0x7fffffffLL) // (the kernel counts them in 31 bits)
    return c->fail("hcKvAttention: %d sequences of up to %lld query rows against %lld tokens are "
                   "too many for one call",
                   p.place.seqs, maxRows, (long long)p.place.width * p.cache.block);
  p.rowTiles = int(rowTiles);
  const int perSm = cap == 64 || (cap == 128 && nt == 1) ? 2 : 1;
  const long long ctas =
      std::max<long long>(1, std::min({ceilDiv(tiles, 8), c->smCount * perSm, kCounters}));
  std::snprintf(name, sizeof name, "hc_kv_attention_%s_d%d_r%d%s", type, cap, nt, p.cache.dim == cap ? "" : "_any");
  void *args[] = {&p};
  return c->launch(name, size_t(ctas), 1, 1, 256, args, 1,
                   size_t(8) * 8 * nt * (2 * (cap + 8) + 8 * cap) +
                       size_t(4) * 8 * nt * std::max<long long>(16, ctas));
}

} // extern "C"
