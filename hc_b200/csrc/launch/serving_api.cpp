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

// Which image defines which family of kernels (names start with `prefix`).
const struct {
  const char *prefix, *image;
} kFamilies[] = {
    // hc_add_rms_norm_{bf16,f32}_{same,i8,e4m3}_{t<threads>_v<packets>,generic}
    {"hc_add_rms_norm_", "add_rms_norm"},
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

} // extern "C"
