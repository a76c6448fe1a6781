// Entry points of the serving operators (include/hc_b200_kernels.h): checks of the
// arguments, the choice of a kernel variant, the launch.
#include "context.hpp"

#include <algorithm>
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
  int sliceK;
  int stepK;
  int vec;
  int vecA;
};

long long roundUp(long long a, long long b) { return ceilDiv(a, b) * b; }

// Rows that the weight-streaming kernel of hcGemmW4 takes.
constexpr long long kW4FewRows = 64;

// Which image defines which family of kernels (names start with `prefix`).
const struct {
  const char *prefix, *image;
} kFamilies[] = {
    // hc_add_rms_norm_{bf16,f32}_{same,i8,e4m3}_{t<threads>_v<packets>,generic}
    {"hc_add_rms_norm_", "add_rms_norm"},
    // hc_gemm_w4_{bf16,i8}_{coarse,fine}_m{1,2,4,8}[_any]: activation type, groups that
    // are multiples of 128 or not, eights of activation rows, weight rows that 16-byte
    // loads do not tile; and the conversions
    {"hc_gemm_w4_", "gemm_w4"},
    {"hc_dequant_w4_", "gemm_w4"},
    {"hc_dequant_a8_", "gemm_w4"},
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

long long hcGemmW4FewRows(void) { return kW4FewRows; }

size_t hcGemmW4WorkspaceBytes(long long M, long long N, long long K, int aDtype) {
  if (M <= kW4FewRows || N <= 0 || K <= 0)
    return 0;
  const long long weights = roundUp(N, 16) * K * 2;
  return size_t(weights + (aDtype == HC_I8 ? M * roundUp(K, 8) * 2 : 0));
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
  if (M <= kW4FewRows) {
    const int nt = M <= 8 ? 1 : M <= 16 ? 2 : M <= 32 ? 4 : 8;
    const long long tiles = ceilDiv(N, 128);
    long long splits = c->w4Splits;
    if (splits == 0) {
      splits = 1;
      while (splits < 8 && tiles * splits * 2 <= 4 * c->smCount && K > splits * 2 * 128)
        splits *= 2;
    }
    p.sliceK = int(std::max<long long>(roundUp(ceilDiv(K, splits), 128), 128));
    // A step of K in shared memory: 64 KiB of activations in fragment order at most.
    const int spanBytes = nt * 4 * 32 * (narrow ? 8 : 16);
    p.stepK = int(std::min<long long>(p.sliceK, 128ll * (64 * 1024 / spanBytes)));
    // Groups of 32 bring 4 scales and zero points per 128 weights of each row.
    p.stepK = int(std::min<long long>(p.stepK, std::max<long long>(128, 32 * group / 128 * 128)));
    const size_t maxGroups = size_t(ceilDiv(p.stepK, group) + 1);
    const size_t staged = size_t(p.stepK / 128) * spanBytes + maxGroups * 128 * 8 +
                          maxGroups * 8 * nt * 8;
    const size_t partial = splits > 1 ? size_t(128) * (8 * nt + 1) * 4 : 0;
    std::snprintf(name, sizeof name, "hc_gemm_w4_%s_%s_m%d%s", narrow ? "i8" : "bf16",
                  group % 128 == 0 || group >= K ? "coarse" : "fine", nt,
                  p.vec && K % 32 == 0 ? "" : "_any");
    void *args[] = {&p};
    return c->launchCluster(name, size_t(tiles), size_t(splits), size_t(splits), 256, args,
                            std::max(staged, partial));
  }
  const size_t need = hcGemmW4WorkspaceBytes(M, N, K, aDtype);
  if (K > 0 && (!workspace || workspaceBytes < need || !aligned(workspace, 16)))
    return c->fail("hcGemmW4: %lld rows need a 16-byte aligned workspace of %zu bytes, got %zu",
                   M, need, workspaceBytes);
  const long long pitch = roundUp(N, 16);
  void *weights = workspace;
  if (K > 0) {
    long long outPitch = pitch;
    void *args[] = {&p, &weights, &outPitch};
    if (ceilDiv(K, 128) > 65535)
      return c->fail("hcGemmW4: K=%lld is too large for a conversion", K);
    if (c->launch("hc_dequant_w4_bf16", size_t(ceilDiv(N, 64)), size_t(ceilDiv(K, 128)), 1, 256,
                  args, 3, 0))
      return 1;
  }
  if (narrow && K > 0) {
    void *rows = static_cast<char *>(workspace) + pitch * K * 2;
    long long outPitch = roundUp(K, 8);
    void *args[] = {&p, &rows, &outPitch};
    if (c->launch("hc_dequant_a8_bf16", size_t(M), size_t(std::min<long long>(ceilDiv(K, 256), 16)),
                  1, 256, args, 3, 0))
      return 1;
    return hcGemmBf16(c, rows, weights, out, M, N, K, outPitch, pitch, ldc);
  }
  return hcGemmBf16(c, a, weights, out, M, N, K, lda, pitch, ldc);
}

} // extern "C"
