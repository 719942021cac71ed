// A plan's device or pinned host buffer, grown by doubling as the reference's workspace is
// (flashinfer_plan_run.cu:47-65).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

namespace mi355x {

struct Buffer {
  void* ptr = nullptr;
  size_t capacity = 0;
  bool pinned = false;
  hipError_t reserve(size_t bytes, uint64_t& allocations) {
    if (bytes <= capacity) return hipSuccess;
    size_t grown = std::max(bytes, capacity ? capacity * 2 : size_t(65536));
    void* fresh = nullptr;
    hipError_t st = allocate(&fresh, grown);
    if (st != hipSuccess && grown > bytes) st = allocate(&fresh, grown = bytes);
    if (st != hipSuccess) return st;
    release();
    ptr = fresh;
    capacity = grown;
    ++allocations;
    return hipSuccess;
  }
  hipError_t allocate(void** out, size_t bytes) const {
    const hipError_t st =
        pinned ? hipHostMalloc(out, bytes, hipHostMallocDefault) : hipMalloc(out, bytes);
    if (st != hipSuccess) (void)hipGetLastError();  // answered here, not by the next launch's check
    return st;
  }
  void release() {
    if (ptr) {
      if (pinned)
        (void)hipHostFree(ptr);
      else
        (void)hipFree(ptr);
    }
    ptr = nullptr;
    capacity = 0;
  }
  ~Buffer() { release(); }
};

}  // namespace mi355x
