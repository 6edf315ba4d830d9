// What the operator entry points that work on caller-owned device memory share on the host: error strings, the device check
// and the caller's current device.
#pragma once
#include <cuda_runtime.h>
#include <stdlib.h>
#include <string.h>

#include <atomic>
#include <exception>
#include <string>

#include "common.cuh"

namespace b200lm {

// Makes `device` current for the duration of a call and puts the caller's device back afterwards.
struct DeviceScope {
  int prev = -1;
  explicit DeviceScope(int device) {
    if (cudaGetDevice(&prev) != cudaSuccess) { cudaGetLastError(); prev = -1; }
    if (prev == device) prev = -1;            // already current: nothing to set, nothing to put back
    else B2_CUDA(cudaSetDevice(device));
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

inline int static_fail(char** err, int code, const std::string& msg) {
  if (err) {
    *err = reinterpret_cast<char*>(malloc(msg.size() + 1));
    if (*err) memcpy(*err, msg.c_str(), msg.size() + 1);
  }
  return code;
}

inline void require_device(int device) {
  static std::atomic<int> known{0};           // the count does not change while a process runs
  int ndev = known.load(std::memory_order_relaxed);
  if (ndev <= 0) {
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev <= 0) {
      cudaGetLastError();
      throw Error{kFailedPrecondition, "no CUDA device: this backend has no CPU fallback"};
    }
    known.store(ndev, std::memory_order_relaxed);
  }
  B2_CHECK(device >= 0 && device < ndev, kInvalidArgument, "device ordinal out of range");
}

// Around the body of an entry point: failures become status codes and messages.
#define OP_TRY if (err) *err = nullptr; try {
#define OP_END                                                                                                    \
  return ::b200lm::kOk; }                                                                                         \
  catch (const ::b200lm::Error& e_) { return ::b200lm::static_fail(err, e_.code, e_.msg); }                       \
  catch (const std::exception& e_) { return ::b200lm::static_fail(err, ::b200lm::kInternal, e_.what()); }         \
  catch (...) { return ::b200lm::static_fail(err, ::b200lm::kInternal, "unknown failure"); }

// Multiprocessors of `device`, asked for once.
inline int device_sms(int device) {
  static std::atomic<int> known[64];
  int n = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  B2_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
  if (device < 64) known[device].store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace b200lm
