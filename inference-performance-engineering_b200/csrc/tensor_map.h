// Host helpers shared by the TMA-fed kernels: 2-D tensor maps for bf16 [rows, k] matrices and the
// SM count of the current device.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace ipe {

// A K-contiguous bf16 matrix [rows, k] read in boxes of box_k x box_rows with 128-byte swizzle
// (box_k * 2 must be 128). Returns false if the driver entry point is missing or the encode fails.
bool make_map_2d(CUtensorMap* map, const void* ptr, int rows, int k, int box_rows, int box_k);

// Slices of a K-contiguous bf16 array: `slices` matrices of `rows` rows (of k elements), slice s
// starting slice_rows * s rows in; rows >= `rows` of a slice read as zeros (TMA out-of-bounds fill),
// so a slice can stop short of its allocation. Boxes of box_k x box_rows x box_slices, 128-byte swizzle.
bool make_map_3d(CUtensorMap* map, const void* ptr, int k, int rows, int slices, int64_t slice_rows, int box_rows,
                 int box_k, int box_slices = 1);

int sm_count();

// Lets `kernel` use `bytes` of dynamic shared memory on the current device. `done` remembers the devices
// on which that has been said (one word per kernel, zero at first).
template <typename Kernel>
cudaError_t allow_shared_memory(Kernel kernel, size_t bytes, std::atomic<uint64_t>* done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (done->load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess) done->fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace ipe
