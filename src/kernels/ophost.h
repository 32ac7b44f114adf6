// Host side shared by the operator entry points: the message of a refusal,
// and the device they run on for the length of a call.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdio>

namespace nb {

inline void op_message(char* err, size_t cap, const char* msg) {
  if (err && cap) std::snprintf(err, cap, "%s", msg);
}

inline int op_refuse(char* err, size_t cap, const char* msg, int code = -1) {
  op_message(err, cap, msg);
  return code;
}

// Makes `device` current and restores the caller's device on exit.
class OpDevice {
 public:
  explicit OpDevice(int device) : device_(device) {
    err_ = cudaGetDevice(&before_);
    if (err_ == cudaSuccess && before_ != device) {
      err_ = cudaSetDevice(device);
      switched_ = err_ == cudaSuccess;
    }
    if (err_ == cudaSuccess) err_ = cudaDeviceGetAttribute(&sms_, cudaDevAttrMultiProcessorCount, device_);
    if (err_ == cudaSuccess && sms_ < 1) sms_ = 1;
  }
  ~OpDevice() {
    if (switched_) cudaSetDevice(before_);
  }
  OpDevice(const OpDevice&) = delete;
  OpDevice& operator=(const OpDevice&) = delete;
  cudaError_t error() const { return err_; }
  int sms() const { return sms_; }

 private:
  cudaError_t err_ = cudaSuccess;
  int device_ = 0, before_ = 0, sms_ = 0;
  bool switched_ = false;
};

}  // namespace nb
