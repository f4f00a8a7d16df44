// A CUDA runtime of two devices that runs nothing: it keeps the current device and each kernel's
// shared-memory limit per device, and refuses a launch or an occupancy query above it, as the real one does.
// The library's objects are linked against it to check their host side without a GPU.
#include <cuda.h>
#include <cuda_runtime_api.h>

#include <cstring>
#include <map>
#include <utility>

namespace {
constexpr int kDevices = 2, kDefaultLimit = 48 * 1024, kMost = 232448;
int current = 0, launches[kDevices], refused = 0, failing_queries = 0;
cudaError_t last = cudaSuccess;
std::map<std::pair<int, const void*>, int> limits;

cudaError_t fail(cudaError_t e) { return last = e; }
int limit(const void* f) {
  auto it = limits.find({current, f});
  return it == limits.end() ? kDefaultLimit : it->second;
}
cudaError_t launch(const void* f, size_t smem) {
  if ((int64_t)smem > limit(f)) {
    ++refused;
    return fail(cudaErrorInvalidValue);
  }
  ++launches[current];
  return cudaSuccess;
}
CUresult encode(...) { return CUDA_SUCCESS; }
struct Call {
  dim3 grid, block;
  size_t smem;
  cudaStream_t stream;
} pushed;
}  // namespace

extern "C" {
int fake_current() { return current; }
int fake_launches(int dev) { return launches[dev]; }
int fake_refused() { return refused; }
void fake_fail_queries(int n) { failing_queries = n; }

cudaError_t cudaGetDevice(int* d) { return *d = current, cudaSuccess; }
cudaError_t cudaSetDevice(int d) {
  if (d < 0 || d >= kDevices) return fail(cudaErrorInvalidDevice);
  current = d;
  return cudaSuccess;
}
cudaError_t cudaGetLastError() {
  const cudaError_t e = last;
  last = cudaSuccess;
  return e;
}
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int d) {
  if (d < 0 || d >= kDevices) return fail(cudaErrorInvalidDevice);
  if (failing_queries > 0) return --failing_queries, fail(cudaErrorUnknown);
  *v = a == cudaDevAttrMultiProcessorCount ? 148 : a == cudaDevAttrMaxSharedMemoryPerBlockOptin ? kMost : 0;
  return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute a, int v) {
  if (a != cudaFuncAttributeMaxDynamicSharedMemorySize || v > kMost) return fail(cudaErrorInvalidValue);
  limits[{current, f}] = v;
  return cudaSuccess;
}
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) {
  memset(a, 0, sizeof(*a));
  a->numRegs = 128;
  return cudaSuccess;
}
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void* f, const cudaLaunchConfig_t* c) {
  if (failing_queries > 0) return --failing_queries, fail(cudaErrorUnknown);
  if ((int64_t)c->dynamicSmemBytes > limit(f)) return fail(cudaErrorInvalidValue);
  return *n = 74, cudaSuccess;
}
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int* n, const void* f, int, size_t smem, unsigned) {
  if ((int64_t)smem > limit(f)) return fail(cudaErrorInvalidValue);
  return *n = 2, cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void* f, dim3, dim3, void**, size_t smem, cudaStream_t) { return launch(f, smem); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) { return launch(f, c->dynamicSmemBytes); }
unsigned __cudaPushCallConfiguration(dim3 g, dim3 b, size_t s, void* st) {
  pushed = {g, b, s, static_cast<cudaStream_t>(st)};
  return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3* g, dim3* b, size_t* s, void* st) {
  *g = pushed.grid, *b = pushed.block, *s = pushed.smem, *static_cast<cudaStream_t*>(st) = pushed.stream;
  return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char*, void** p, unsigned long long, cudaDriverEntryPointQueryResult* q) {
  *p = reinterpret_cast<void*>(&encode);
  if (q) *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}
// registration, and calls that the checks do not reach
void** __cudaRegisterFatBinary(void*) {
  static void* handle;
  return &handle;
}
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
cudaError_t cudaDeviceSynchronize() { return cudaSuccess; }
cudaError_t cudaFree(void*) { return cudaErrorNotSupported; }
cudaError_t cudaGetSymbolAddress(void**, const void*) { return cudaErrorNotSupported; }
cudaError_t cudaIpcCloseMemHandle(void*) { return cudaErrorNotSupported; }
cudaError_t cudaIpcGetMemHandle(cudaIpcMemHandle_t*, void*) { return cudaErrorNotSupported; }
cudaError_t cudaIpcOpenMemHandle(void**, cudaIpcMemHandle_t, unsigned) { return cudaErrorNotSupported; }
cudaError_t cudaMalloc(void**, size_t) { return cudaErrorNotSupported; }
cudaError_t cudaMemcpyAsync(void*, const void*, size_t, cudaMemcpyKind, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaMemset(void*, int, size_t) { return cudaErrorNotSupported; }
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
}
