/* A stand-in for libcuda.so.1 with one B200-like device that computes nothing and
 * records its launches.
 *
 * TEST INFRASTRUCTURE ONLY.  With it on LD_LIBRARY_PATH a context opens on a host
 * without a GPU, so that the host side of an entry point can be tested there: which
 * calls it refuses, and which kernel, grid, shared memory and stream it chooses for
 * the others.  Device addresses are made up and never dereferenced.  It is never
 * loaded in a process that uses a real GPU.
 */
#include <pthread.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

struct launch {
  char name[96];
  unsigned grid[3], block, smem;
  unsigned long long stream;
};
#define ROOM 65536 /* further launches overwrite the last one */
static struct launch launches[ROOM];
static int count; /* threads may launch at the same time */

int recorded_launches(void) { return count < ROOM ? count : ROOM; }
void recorded_clear(void) { count = 0; }
const struct launch *recorded_launch(int i) { return &launches[i]; }

#define OK(name) int name() { return 0; }
OK(cuInit)
OK(cuDevicePrimaryCtxRelease_v2)
OK(cuCtxPushCurrent_v2)
OK(cuCtxPopCurrent_v2)
OK(cuModuleUnload)
OK(cuFuncSetAttribute)
OK(cuStreamDestroy_v2)
OK(cuStreamSynchronize)
OK(cuMemFree_v2)
OK(cuMemcpyDtoHAsync_v2)
OK(cuMemsetD8Async)
OK(cuTensorMapEncodeTiled)
OK(cuEventDestroy_v2)
OK(cuEventRecord)
OK(cuEventElapsedTime)
OK(cuStreamWaitEvent)
OK(cuMemHostRegister_v2)
OK(cuMemHostUnregister)
/* Uploads: which thread made each. */
static unsigned long uploads[ROOM];
static int uploaded;
int recorded_uploads(void) { return uploaded < ROOM ? uploaded : ROOM; }
unsigned long recorded_upload(int i) { return uploads[i]; }
int cuMemcpyHtoDAsync_v2(unsigned long long dst, const void *src, size_t n, void *stream) {
  int at = __atomic_fetch_add(&uploaded, 1, __ATOMIC_RELAXED);
  uploads[at < ROOM ? at : ROOM - 1] = (unsigned long)pthread_self();
  return 0;
}
int cuGetErrorName(int error, const char **name) {
  *name = "CUDA_ERROR_UNKNOWN";
  return 0;
}
int cuDeviceGet(int *d, int ordinal) { *d = ordinal; return 0; }
int cuDeviceGetCount(int *n) { *n = 1; return 0; }
int cuDeviceGetAttribute(int *v, int what, int dev) {
  switch (what) {
  case 16: *v = 148; break;        /* multiprocessors */
  case 75: *v = 10; break;         /* compute capability */
  case 76: *v = 0; break;
  case 38: *v = 126 << 20; break;  /* L2 */
  case 97: *v = 227 << 10; break;  /* shared memory per CTA, opt-in */
  default: *v = 0;
  }
  return 0;
}
int cuDevicePrimaryCtxRetain(void **c, int dev) { *c = (void *)0x10; return 0; }
int cuModuleLoadData(void **m, const void *image) { *m = (void *)image; return 0; }
int cuModuleGetFunction(void **f, void *m, const char *name) {
  *f = strdup(name); /* kept for the process's life */
  return 0;
}
int cuFuncGetAttribute(int *v, int what, void *f) { *v = 0; return 0; }
int cuStreamCreate(void **s, unsigned flags) {
  static uintptr_t next = 0x7000;
  *s = (void *)(next += 0x10);
  return 0;
}
int cuMemAlloc_v2(unsigned long long *p, size_t n) {
  static unsigned long long next = 0x700000000000ull;
  *p = next;
  next += (n + 4095) & ~4095ull;
  return 0;
}
int cuOccupancyMaxActiveClusters(int *n, void *f, const void *config) { *n = 74; return 0; }
int cuPointerGetAttribute(void *v, int what, unsigned long long p) { *(int *)v = 0; return 0; }
int cuEventCreate(void **e, unsigned flags) { *e = (void *)0x20; return 0; }
int cuLaunchKernel(void *f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned by,
                   unsigned bz, unsigned smem, void *stream, void **params, void **extra) {
  int at = __atomic_fetch_add(&count, 1, __ATOMIC_RELAXED);
  struct launch *l = &launches[at < ROOM ? at : ROOM - 1];
  snprintf(l->name, sizeof l->name, "%s", (const char *)f);
  l->grid[0] = gx, l->grid[1] = gy, l->grid[2] = gz;
  l->block = bx * by * bz, l->smem = smem, l->stream = (unsigned long long)(uintptr_t)stream;
  return 0;
}

/* The head of CUlaunchConfig. */
struct config {
  unsigned grid[3], block[3], smem;
  void *stream;
};
int cuLaunchKernelEx(const struct config *c, void *f, void **params, void **extra) {
  return cuLaunchKernel(f, c->grid[0], c->grid[1], c->grid[2], c->block[0], c->block[1],
                        c->block[2], c->smem, c->stream, params, extra);
}
