// The context behind an HcContext handle, shared by the translation units of
// libhc-b200-kernels.so.
#pragma once

#include "hc_b200_kernels.h"

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <map>
#include <mutex>
#include <string>
#include <vector>

// The last error's text: threads that share a context write it and read copies.
class HcErrorText {
public:
  void operator=(const char *s) {
    std::lock_guard<std::mutex> hold(lock);
    text = s;
  }
  // The calling thread's copy of this context's text, valid until it asks again.
  const char *c_str() const {
    static thread_local std::map<const HcErrorText *, std::string> copies;
    std::lock_guard<std::mutex> hold(lock);
    return (copies[this] = text).c_str();
  }

private:
  mutable std::mutex lock;
  std::string text;
};

// One thread may be inside a host-buffer entry point (Python runs those without its
// interpreter lock) while another launches through the same context: what both reach -
// the tables of loaded images, the error's text, the count of launches - is guarded, and
// which queue a launch goes to is a matter of the thread that launches.
struct HcContextImpl {
  OlErrorCallback callback = nullptr;
  void *callbackCtx = nullptr;
  OlDevice device = nullptr;
  OlQueue ownQueue = nullptr;
  OlQueue chosenQueue = nullptr; // ownQueue, or a borrowed one (hcUseStream)
  // Where the calling thread's launches go: what it pushed last (hcPushStream,
  // HcQueueScope), else chosenQueue.
  OlQueue queue() const;
  // The queue on a caller's stream, or null (with an error).
  OlQueue borrowed(void *stream);
  std::mutex tables; // guards the next three
  std::map<void *, OlQueue> borrowedQueues; // by the caller's stream handle
  std::vector<OlModule> modules; // one slot per image, loaded on first use
  std::map<std::string, OlKernel> kernels;
  int *statusWord = nullptr; // device
  HcErrorText lastError;
  std::atomic<long long> launches{0};
  long long smCount = 0;
  long long ccMajor = 0;
  long long ccMinor = 0;
  long long gemmVariant = 0;
  long long softmaxVariant = 0; // 0 auto, 1 register kernel, 2 bulk-copy pipeline
  long long tiledVariant = 0;
  long long reduceVariant = 0;
  long long mappedStack = 0;
  long long rowVariant = 0;
  long long fusedVariant = 0; // 1: never use the precompiled bodies
  long long gemmBand = 0;     // row tiles per band of the tcgen05 GEMMs' tile order (0: default)
  long long convVariant = 0;  // 1: image operand in shared memory, 2: in tensor memory
  long long convStacked = 0;  // 1: never run a_hi * [b_hi; b_lo] as one MMA of double width
  long long convStages = 0;   // 2..6: pipeline stages of the convolution (0: as many as fit)
  long long pairSlots = 0; // CTA pairs of the tcgen05 kernels resident at once
  int pairSlotsF32 = 0; // the same for the float32 tensor-core kernel
  int pairSlotsBanded = 0; // the same for the dequant GEMM that converts band by band
  int pairSlotsW8 = 0;  // the same for the dequant GEMM that converts in its pipeline
  long long attentionVariant = 0; // hcKvAttention: 1 sixteen rows at a time, 2 tcgen05
  long long w4Variant = 0; // hcGemmW4: 1 the kernel for few rows, 2 never that one
  long long w8Variant = 0; // 1: convert the weights in a pass of its own, 2: never
  // Programs without a precompiled body: 0 interpret them, 1 compile them at their
  // first launch and interpret where that is not possible, 2 fail where it is not.
  long long specialiseMode = 1;
  struct HcSpecialiser *specialiser = nullptr; // specialise.cpp

  int fail(const char *fmt, ...) __attribute__((format(printf, 2, 3))) {
    char text[320];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    lastError = text;
    if (callback)
      callback(callbackCtx, OlSeverity::Error, text);
    return 1;
  }

  // ol* failures arrive here through the loader/backend callback.
  static void onBackendMessage(void *self, OlSeverity sev, const char *desc) {
    auto *c = static_cast<HcContextImpl *>(self);
    if (sev == OlSeverity::Error)
      c->lastError = desc ? desc : "";
    if (c->callback)
      c->callback(c->callbackCtx, sev, desc);
  }

  // The kernel `name` from the embedded images (loaded on first use), or null.
  OlKernel kernel(const char *name);
  // Launches `name` with a one-dimensional block on the context's queue.
  int launch(const char *name, size_t gx, size_t gy, size_t gz, size_t threads, void **args,
             size_t nArgs, size_t smem);
  // The same in clusters of `cluster` CTAs along y (1..8; gy is a multiple of it).
  int launchCluster(const char *name, size_t gx, size_t gy, size_t cluster, size_t threads,
                    void **args, size_t smem);
  // Scratch of the host-buffer entry points (host_api.cpp), released with the context.
  struct HostPipeline *hostPipeline = nullptr;
  std::mutex hostCalls; // one of them at a time
};

// Sends the calling thread's launches through `c` to `q` for the length of the scope,
// whatever other threads choose meanwhile.
class HcQueueScope {
public:
  HcQueueScope(HcContextImpl *c, OlQueue q);
  ~HcQueueScope();
  HcQueueScope(const HcQueueScope &) = delete;
  HcQueueScope &operator=(const HcQueueScope &) = delete;

private:
  HcContextImpl *const context;
};

// Frees what the host-buffer entry points keep in a context (host_api.cpp).
void hcReleaseHostPipeline(HcContextImpl *c);

// hcGemmBf16 on the tensor cores with row m of the product times rowScale[m *
// rowScaleStride] before it is rounded (kernels_api.cpp).  Operands as TMA takes them.
extern "C" int hcGemmBf16RowScaled(HcContextImpl *c, const void *a, const void *b,
                                   const float *rowScale, long long rowScaleStride, void *out,
                                   long long M, long long N, long long K, long long lda,
                                   long long ldb, long long ldc);

// Image of a serving kernel by its name, or null (serving_api.cpp).
const char *hcServingImageOf(const char *kernel);

// Run-time specialisation (specialise.cpp).
struct HcMapProgramDev;
bool hcSpecialisable(const HcMapProgramDev &p, bool row, int dtype);
const char *hcSpecialise(HcContextImpl *c, bool row, int dtype, const HcMapProgramDev &p);
const char *hcSpecialiseItems(HcContextImpl *c, int dtype, const uint32_t *code, int nInstr,
                              bool wide);
const char *hcSpecialiserNote(HcContextImpl *c);
long long hcSpecialiserCount(HcContextImpl *c, int which);
void hcReleaseSpecialiser(HcContextImpl *c);
