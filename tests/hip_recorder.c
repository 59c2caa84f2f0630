/* A HIP runtime without GPUs for tests of the host side: device memory is host memory, kernels do not run, and every call that
 * queues work or waits is recorded with the calling thread's current device.  Loaded with RTLD_GLOBAL before the library. */
#define __HIP_PLATFORM_AMD__
#include <hip/hip_runtime_api.h>
#include <stdlib.h>
#include <string.h>

#define EXPORT __attribute__((visibility("default")))
#define MAX_CALLS 65536

static struct {
  const char *name;
  int device;
  void *stream;
} calls[MAX_CALLS];
static int ncalls, current, capture_status;
static hipStreamCaptureMode thread_mode = hipStreamCaptureModeGlobal;

static void record(const char *name, void *stream) {
  if (ncalls < MAX_CALLS) {
    calls[ncalls].name = name;
    calls[ncalls].device = current;
    calls[ncalls].stream = stream;
    ++ncalls;
  }
}

EXPORT int rec_count(void) { return ncalls; }
EXPORT const char *rec_name(int i) { return calls[i].name; }
EXPORT int rec_device(int i) { return calls[i].device; }
EXPORT void *rec_stream(int i) { return calls[i].stream; }
EXPORT void rec_clear(void) { ncalls = 0; }
EXPORT int rec_thread_mode(void) { return (int)thread_mode; }
EXPORT void rec_capture(int status) { capture_status = status; }

EXPORT hipError_t hipGetDeviceCount(int *n) { *n = 2; return hipSuccess; }
EXPORT hipError_t hipSetDevice(int d) { current = d; return hipSuccess; }
EXPORT hipError_t hipGetDevice(int *d) { *d = current; return hipSuccess; }
EXPORT hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int d) {
  memset(p, 0, sizeof(*p));
  p->multiProcessorCount = 256;
  p->warpSize = 64;
  return hipSuccess;
}
EXPORT hipError_t hipDeviceGetAttribute(int *v, hipDeviceAttribute_t a, int d) { *v = 64; return hipSuccess; }
EXPORT hipError_t hipMalloc(void **p, size_t n) {
  record(thread_mode == hipStreamCaptureModeRelaxed ? "hipMalloc, relaxed" : "hipMalloc", NULL);
  *p = aligned_alloc(256, (n + 255) / 256 * 256 + 256);
  if (!*p) return hipErrorOutOfMemory;
  memset(*p, 0, (n + 255) / 256 * 256 + 256);
  return hipSuccess;
}
EXPORT hipError_t hipFree(void *p) { free(p); return hipSuccess; }
EXPORT hipError_t hipHostMalloc(void **p, size_t n, unsigned flags) { *p = calloc(1, n + 256); return hipSuccess; }
EXPORT hipError_t hipHostFree(void *p) { free(p); return hipSuccess; }
EXPORT hipError_t hipHostGetDevicePointer(void **d, void *h, unsigned flags) { *d = h; return hipSuccess; }
EXPORT hipError_t hipGetSymbolAddress(void **p, const void *s) { static char scratch[1 << 20]; *p = scratch; return hipSuccess; }
EXPORT hipError_t hipMemcpy(void *d, const void *s, size_t n, hipMemcpyKind k) {
  record("hipMemcpy", NULL);
  memcpy(d, s, n);
  return hipSuccess;
}
EXPORT hipError_t hipMemcpyAsync(void *d, const void *s, size_t n, hipMemcpyKind k, hipStream_t st) {
  record("hipMemcpyAsync", st);
  memcpy(d, s, n);
  return hipSuccess;
}
EXPORT hipError_t hipMemcpyWithStream(void *d, const void *s, size_t n, hipMemcpyKind k, hipStream_t st) {
  record("hipMemcpyWithStream", st);
  memcpy(d, s, n);
  return hipSuccess;
}
EXPORT hipError_t hipMemsetAsync(void *d, int v, size_t n, hipStream_t st) {
  record("hipMemsetAsync", st);
  memset(d, v, n);
  return hipSuccess;
}
EXPORT hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned flags) { *s = (hipStream_t)(size_t)0x5000; return hipSuccess; }
EXPORT hipError_t hipStreamDestroy(hipStream_t s) { return hipSuccess; }
EXPORT hipError_t hipStreamSynchronize(hipStream_t s) { record("hipStreamSynchronize", s); return hipSuccess; }
EXPORT hipError_t hipStreamQuery(hipStream_t s) { record("hipStreamQuery", s); return hipSuccess; }
EXPORT hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus *status) {
  *status = (hipStreamCaptureStatus)(capture_status & 3);
  return capture_status & 4 ? hipErrorStreamCaptureImplicit : hipSuccess;
}
EXPORT hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode *mode) {
  const hipStreamCaptureMode before = thread_mode;
  thread_mode = *mode;
  *mode = before;
  return hipSuccess;
}
EXPORT int hipGetStreamDeviceId(hipStream_t s) { return current; }
EXPORT hipError_t hipEventCreate(hipEvent_t *e) { *e = (hipEvent_t)(size_t)0x7000; return hipSuccess; }
EXPORT hipError_t hipEventDestroy(hipEvent_t e) { return hipSuccess; }
EXPORT hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) { record("hipEventRecord", s); return hipSuccess; }
EXPORT hipError_t hipEventElapsedTime(float *ms, hipEvent_t a, hipEvent_t b) { *ms = 1.0f; return hipSuccess; }
EXPORT const char *hipGetErrorString(hipError_t e) { return "error of the recording runtime"; }
EXPORT hipError_t hipGetLastError(void) { return hipSuccess; }
EXPORT hipError_t hipFuncSetAttribute(const void *f, hipFuncAttribute a, int v) { return hipSuccess; }
EXPORT hipError_t hipOccupancyMaxActiveBlocksPerMultiprocessor(int *n, const void *f, int b, size_t lds) { *n = 1; return hipSuccess; }
EXPORT hipError_t hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t lds, hipStream_t s) {
  record("hipLaunchKernel", s);
  return hipSuccess;
}
EXPORT hipError_t hipLaunchCooperativeKernel(const void *f, dim3 g, dim3 b, void **args, unsigned lds, hipStream_t s) {
  record("hipLaunchCooperativeKernel", s);
  return hipSuccess;
}

/* what the compiler's registration and launch code calls */
static dim3 pushed_grid, pushed_block;
static size_t pushed_lds;
static hipStream_t pushed_stream;
EXPORT hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t s) {
  pushed_grid = g, pushed_block = b, pushed_lds = lds, pushed_stream = s;
  return hipSuccess;
}
EXPORT hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *lds, hipStream_t *s) {
  *g = pushed_grid, *b = pushed_block, *lds = pushed_lds, *s = pushed_stream;
  return hipSuccess;
}
EXPORT void **__hipRegisterFatBinary(const void *data) { static void *handle; return &handle; }
EXPORT void __hipUnregisterFatBinary(void **modules) {}
EXPORT void __hipRegisterFunction(void **m, const void *f, char *df, const char *n, unsigned t, void *a, void *b, void *c, void *d, int *w) {}
EXPORT void __hipRegisterVar(void **m, void *v, char *hv, char *dv, int ext, size_t n, int c, int g) {}
