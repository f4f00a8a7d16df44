// Host-side helpers shared by the entry points: device attributes, the TMA descriptor encoder,
// the current-device guard.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdlib>
#include <map>
#include <mutex>
#include <utility>

namespace qmla {

constexpr int kMaxDynSmem = 232448;  // 227 KB opt-in limit per block on sm_100

struct DevInfo {
  int sms = 0;
  int max_smem = 0;
  bool ok = false;
};

inline DevInfo dev_info(int dev) {
  static std::mutex mu;
  static std::map<int, DevInfo> devs;
  std::lock_guard<std::mutex> lk(mu);
  auto it = devs.find(dev);
  if (it != devs.end()) return it->second;
  DevInfo d;
  if (cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess &&
      cudaDeviceGetAttribute(&d.max_smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) ==
          cudaSuccess) {
    d.ok = true;
    devs[dev] = d;
  } else {
    cudaGetLastError();  // nothing of a failure stays: the next call asks again
  }
  return d;
}

// Lets `kernel` have up to `bytes` of dynamic shared memory on the current device.  The limit belongs to
// the pair of kernel and device: it is set once for each, and a failure is not remembered.
inline bool allow_smem(const void* kernel, int bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> known;
  int dev;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  std::lock_guard<std::mutex> lk(mu);
  auto it = known.find({dev, kernel});
  if (it != known.end() && it->second >= bytes) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();  // the caller's return code says it; it is not the next launch's error
    return false;
  }
  known[{dev, kernel}] = bytes;
  return true;
}
template <typename... A>
bool allow_smem(void (*kernel)(A...), int bytes) {
  return allow_smem(reinterpret_cast<const void*>(kernel), bytes);
}

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// Tiled map over 2-byte (bf16) or 1-byte elements, 128-byte swizzle; dims[0] is dense, strides in
// bytes are those of dims[1..].  False when the driver refuses it.
inline bool encode_tiled(CUtensorMap* m, bool fp8, const void* base, int nd, const cuuint64_t* dims,
                         const cuuint64_t* strides, const cuuint32_t* box) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return fn(m, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, nd, const_cast<void*>(base), dims,
            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How long a wait of the tensor-core operators may last.
inline uint32_t wait_limit_us() {
  if (const char* e = getenv("QMLA_WAIT_US")) return (uint32_t)atoi(e);  // test hook: 0 gives up at once
  return 2000000;
}

// Reads (and clears) a status word in device memory by its symbol, on the current device.
inline int take_status(const void* symbol, bool clear, cudaStream_t st, int32_t* bits) {
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, symbol) != cudaSuccess ||
      cudaMemcpyAsync(bits, p, 4, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
      (clear && cudaMemsetAsync(p, 0, 4, st) != cudaSuccess) || cudaStreamSynchronize(st) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  return 0;
}
int weights_status(bool clear, cudaStream_t st, int32_t* bits);  // the attention weights' word

inline int gcd_int(int a, int b) {
  while (b) {
    int t = a % b;
    a = b;
    b = t;
  }
  return a;
}

inline int64_t align_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// Makes `dev` the current device for the lifetime of the guard and puts the caller's current
// device back on every return path, so an entry point never leaves a thread that drives several
// GPUs pointed at another one.
class DeviceGuard {
 public:
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev_) != cudaSuccess) return;
    if (prev_ == dev) {
      ok_ = true;
      return;
    }
    ok_ = cudaSetDevice(dev) == cudaSuccess;
    switched_ = ok_;
  }
  ~DeviceGuard() {
    if (switched_) cudaSetDevice(prev_);
  }
  bool ok() const { return ok_; }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;

 private:
  int prev_ = -1;
  bool ok_ = false, switched_ = false;
};

}  // namespace qmla
