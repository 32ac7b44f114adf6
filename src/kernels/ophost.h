// Host side shared by the operator entry points: the message of a refusal,
// and the device they run on for the length of a call.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdio>

namespace nb {

inline void op_message(char* err, size_t cap, const char* msg) {
  if (err && cap) std::snprintf(err, cap, "%s", msg);
}

// `code` above 0: a CUDA error, which is reported here and must not come up again as the
// last error of a later launch of the caller's.
inline int op_refuse(char* err, size_t cap, const char* msg, int code = -1) {
  op_message(err, cap, msg);
  if (code > 0) cudaGetLastError();
  return code;
}

// Makes `device` current and restores the caller's device on exit.
class OpDevice {
 public:
  explicit OpDevice(int device) {
    err_ = cudaGetDevice(&before_);
    if (err_ == cudaSuccess && before_ != device) {
      err_ = cudaSetDevice(device);
      switched_ = err_ == cudaSuccess;
    }
    // 0: no SM count known yet. Threads that race store the same number.
    static std::atomic<int> known[64];
    const bool keeps = device >= 0 && device < 64;
    if (err_ == cudaSuccess && keeps) sms_ = known[device].load(std::memory_order_relaxed);
    if (err_ == cudaSuccess && !sms_) {
      err_ = cudaDeviceGetAttribute(&sms_, cudaDevAttrMultiProcessorCount, device);
      if (err_ == cudaSuccess && sms_ < 1) sms_ = 1;
      if (err_ == cudaSuccess && keeps) known[device].store(sms_, std::memory_order_relaxed);
    }
  }
  ~OpDevice() {
    if (err_ != cudaSuccess) cudaGetLastError();  // the call reports it
    if (switched_) cudaSetDevice(before_);
  }
  OpDevice(const OpDevice&) = delete;
  OpDevice& operator=(const OpDevice&) = delete;
  cudaError_t error() const { return err_; }
  int sms() const { return sms_; }

 private:
  cudaError_t err_ = cudaSuccess;
  int before_ = 0, sms_ = 0;
  bool switched_ = false;
};

// Lets `fn` have up to `bytes` of dynamic shared memory on `device` (the current
// one): asked for once, since the call takes about a microsecond.
inline cudaError_t op_allow_smem(const void* fn, int device, int bytes) {
  constexpr int kSlots = 64;
  static std::atomic<const void*> known[64][kSlots];
  const bool keeps = device >= 0 && device < 64;
  int slot = 0;
  if (keeps)
    for (; slot < kSlots; ++slot) {
      const void* k = known[device][slot].load(std::memory_order_acquire);
      if (k == fn) return cudaSuccess;
      if (!k) break;
    }
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && keeps && slot < kSlots) {
    const void* none = nullptr;  // another thread may have taken the slot: then the next call asks again
    known[device][slot].compare_exchange_strong(none, fn, std::memory_order_release);
  }
  return e;
}

// Launches a kernel that begins with op_wait_for_previous(): its blocks may be
// set up while the stream's previous kernel ends.
inline cudaError_t op_launch_after(const void* fn, dim3 grid, dim3 block, void** argv, cudaStream_t stream) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, fn, argv);
}

}  // namespace nb
