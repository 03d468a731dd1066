// smem_attr.cuh -- permission for a kernel's launches to use more than 48 KB of dynamic shared memory.
#pragma once
#include <cuda_runtime_api.h>

#include <atomic>
#include <cstddef>

namespace anima {

// Largest dynamic shared memory of a block (sm_100a), for kernels without static shared memory.
constexpr size_t kMaxSmem = 227 * 1024;

// One per kernel.  The attribute is an assignment, not a maximum, and launches of one kernel differ in size:
// it is set to the largest there is, once per device, so that two threads whose first calls meet assign the
// same value.  A launch passes its own size.
struct SmemAttr {
  std::atomic<bool> is_set[64];
  SmemAttr() {
    for (auto& s : is_set) s.store(false);
  }
  bool raise(const void* kern, size_t bytes) {
    int dev = 0;
    if (bytes > kMaxSmem || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (is_set[dev].load(std::memory_order_acquire)) return true;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    is_set[dev].store(true, std::memory_order_release);
    return true;
  }
};

}  // namespace anima
