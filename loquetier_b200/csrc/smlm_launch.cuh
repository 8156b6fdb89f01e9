// Host side of a launch, shared by the files that define the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <utility>
#include <vector>

#include "../../include/smlm_b200.h"
#include "paged_kv.cuh"

namespace {

using namespace smlm;

constexpr int kNumSMs = 148;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline bool kv_shape_ok(int head_dim, int page_size) {
  return head_dim == kPdDim && (page_size == 8 || page_size == 16 || page_size == 32 || page_size == 64);
}

// The opt-in to more than 48 KB of dynamic shared memory is a property of (kernel, device): it is
// set when a kernel is first launched on a device, or with more shared memory than before, and
// remembered - not repeated per launch.
constexpr int kMaxDevices = 64;
std::mutex g_attr_mutex;
std::vector<std::pair<const void*, int>> g_attr_done[kMaxDevices];

bool ensure_dynamic_smem(const void* kern, int smem_bytes) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    return false;
  }
  {
    std::lock_guard<std::mutex> lock(g_attr_mutex);
    for (const auto& k : g_attr_done[dev])
      if (k.first == kern && k.second >= smem_bytes) return true;
  }
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  std::lock_guard<std::mutex> lock(g_attr_mutex);
  for (auto& k : g_attr_done[dev])
    if (k.first == kern) {
      k.second = std::max(k.second, smem_bytes);
      return true;
    }
  g_attr_done[dev].emplace_back(kern, smem_bytes);
  return true;
}

template <typename Kern, typename... Args>
int launch(Kern kern, dim3 grid, int threads, int cluster_x, int smem_bytes, cudaStream_t stream,
           const Args&... args) {
  if (grid.x == 0 || grid.y == 0) return SMLM_OK;
  // the limit without the opt-in is 48 KB for dynamic and static shared memory TOGETHER, hence the margin
  if (smem_bytes > 40 * 1024 && !ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem_bytes))
    return SMLM_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster_x;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  // every kernel of the library calls pdl_wait() before it touches memory that an earlier kernel
  // of the stream may have written, so it may be scheduled while its predecessor drains
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) {
    cudaGetLastError();
    return SMLM_ERR_CUDA;
  }
  return SMLM_OK;
}

}  // namespace
