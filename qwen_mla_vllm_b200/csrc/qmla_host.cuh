// Host-side helpers shared by the entry points: device attributes, the TMA descriptor encoder,
// the current-device guard.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <map>
#include <mutex>

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
          cudaSuccess)
    d.ok = true;
  devs[dev] = d;
  return d;
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
