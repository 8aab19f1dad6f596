// entry.h — what the entry points of the operators (f8.cu, rules.cu) share: the status of a
// C-ABI call from what it throws, and the caller's current device kept.
#pragma once

#include <atomic>
#include <new>

#include "engine.h"

namespace svl {

// Runs f; every exception ends here as a status and a message (none may cross the C ABI).
template <class F>
svl_status entry(F&& f) {
  try {
    f();
    return SVL_OK;
  } catch (const Error& e) {
    set_last_error(e.what());
    return e.code;
  } catch (const std::bad_alloc&) {
    set_last_error("host allocation failed");
    return SVL_ERR_OOM;
  } catch (const std::exception& e) {
    set_last_error(e.what());
    return SVL_ERR_CUDA;
  } catch (...) {
    set_last_error("unknown failure");
    return SVL_ERR_CUDA;
  }
}

inline void require(bool ok, const char* msg, svl_status code = SVL_ERR_INVALID_INPUT) {
  if (!ok) throw Error(code, msg);
}

// Every pointer that is given starts on a multiple of its elements' size.
template <class... P>
void require_aligned(size_t size, P... pointers) {
  require(((reinterpret_cast<uintptr_t>(pointers) % size == 0) && ...), "a pointer is not aligned to its elements");
}

// `device` current for the life of the guard, the caller's device again afterwards: the
// operators work on tensors of any device, whichever is current.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    check_cuda(cudaGetDevice(&before_), "cudaGetDevice");
    if (before_ != device) {
      check_cuda(cudaSetDevice(device), "cudaSetDevice");
      moved_ = true;
    }
  }
  ~OnDevice() {
    if (moved_) cudaSetDevice(before_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int before_ = 0;
  bool moved_ = false;
};

// Raises a kernel's dynamic shared-memory limit, once per device (the attribute is the device's).
template <auto kernel>
void allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  check_cuda(cudaGetDevice(&device), "cudaGetDevice");
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (done.load(std::memory_order_acquire) & bit)) return;
  check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), "shared memory");
  if (device < 64) done.fetch_or(bit, std::memory_order_release);
}

}  // namespace svl
