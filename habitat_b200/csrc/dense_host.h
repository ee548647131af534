// Host-side helpers of the dense-layer operators: tensor maps, launches, the status word.
#pragma once

#include <cuda.h>

#include <atomic>

#include "hb_common.h"

namespace dense {

// A tensor map of `planes` matrices of `rows` rows of `cols` elements, rows `pitch` and matrices `plane_stride` elements
// apart, in boxes of box_rows rows x 128 bytes, 128-byte swizzle, zeros outside.  elem_bytes 1 (8-bit) or 2 (16-bit).
cudaError_t encode_planes(CUtensorMap* map, const void* base, int elem_bytes, int64_t cols, int64_t rows, int64_t planes,
                          int64_t pitch, int64_t plane_stride, int box_rows);

// The word that kernels on the current GPU write when a bounded wait runs out (page-locked, created on first use), and
// HB_ERR_DEVICE_TIMEOUT (once for each host thread) when an earlier launch has written it.
hb_status begin_call(const char* name, int32_t** word);

hb_status sm_count(int* sms);

// Whether arrays of elements of these sizes can start at these addresses.
inline bool starts_on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0; }
inline int bytes_of(int32_t type) { return type == HB_F32 ? 4 : 2; }

}  // namespace dense

#if defined(__CUDACC__)
namespace dense {
// Launches `clusters` clusters of `cluster` CTAs, overlapped with the end of the launch before (hb_common.h).
template <typename... KArgs, typename... Args>
cudaError_t launch_clusters(void (*kernel)(KArgs...), int clusters, int cluster, int threads, int smem, cudaStream_t stream,
                            Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = hb::overlapped_launch_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// How many clusters of a kernel the current GPU holds at a time; sets the kernel's shared memory size first.  One static
// table per kernel, a word per GPU.
template <typename... KArgs>
hb_status max_clusters(void (*kernel)(KArgs...), int cluster, int threads, int smem, std::atomic<int>* per_gpu, int* out) {
  int dev = 0;
  HB_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) {
    hb::set_error("device ordinal %d out of range", dev);
    return HB_ERR_UNSUPPORTED;
  }
  int n = per_gpu[dev].load();
  if (n == 0) {
    HB_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(cluster));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HB_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    if (n < 1) {
      hb::set_error("the GPU holds no cluster of %d blocks", cluster);
      return HB_ERR_UNSUPPORTED;
    }
    per_gpu[dev].store(n);
  }
  *out = n;
  return HB_OK;
}
}  // namespace dense
#endif
