// A kernel's limit of dynamic shared memory belongs to a device: it is raised at the first launch on each.
#pragma once
#include <cuda_runtime_api.h>

#include <atomic>
#include <cstdint>

inline cudaError_t vb_allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& devices) {
  int d = 0;
  cudaError_t rc = cudaGetDevice(&d);
  if (rc != cudaSuccess) return rc;
  const uint64_t bit = d < 64 ? uint64_t(1) << d : 0;
  if (devices.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (rc == cudaSuccess) devices.fetch_or(bit, std::memory_order_relaxed);
  return rc;
}
