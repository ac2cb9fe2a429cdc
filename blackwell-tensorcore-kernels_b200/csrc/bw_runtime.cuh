// Host-side runtime shared by the library's translation units: per-thread error text,
// per-device state (SM count, device status word, workspace), TMA descriptor encoding
// through the driver entry point (no link-time dependency on libcuda).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdlib>
#include <string>

#include "../../include/bwgemm.h"

namespace bw {

int set_error(int code, const char* fmt, ...);
int cuda_error(cudaError_t e, const char* what);
#define BW_CUDA(call)                                  \
  do {                                                 \
    cudaError_t e_ = (call);                           \
    if (e_ != cudaSuccess) return cuda_error(e_, #call); \
  } while (0)

struct DeviceState {
  bool ready = false;
  int sms = 0;
  int major = 0, minor = 0;
  int* status = nullptr;         // device status word (kernels' bounded waits report here)
  void* workspace = nullptr;     // small scratch for quantiser reductions
  size_t workspace_bytes = 0;
  struct SplitWs {               // FP32 split-K partial sums for BF16 outputs, one per stream
    void* stream = nullptr;
    float* buf = nullptr;
    size_t bytes = 0;
  };
  static constexpr int kSplitWs = 8;
  SplitWs splitk[kSplitWs];
};

// Ensures the current device is initialised; returns BW_OK or an error status.
int ensure_device(DeviceState** out);
unsigned long long wait_budget_ns();
// FP32 workspace of at least `bytes` private to `stream` on this device (grown on demand, kept
// until bw_shutdown); BW_ERR_UNSUPPORTED when every slot belongs to another stream.
int splitk_workspace(DeviceState& d, cudaStream_t stream, size_t bytes, float** out);
unsigned long long* trace_buffer(int ctas_needed);  // null unless bw_set_trace_buffer armed one

// 2-D row-major tensor map: dims {inner, outer}, box {box_inner, box_outer}, 128B swizzle.
int make_tmap_2d(CUtensorMap* map, CUtensorMapDataType dtype, const void* base, uint64_t inner, uint64_t outer,
                 uint64_t row_stride_bytes, uint32_t box_inner, uint32_t box_outer,
                 CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B);

// 3-D row-major tensor map (dims {inner, mid, outer}, box {box_inner, box_mid, 1}), 128B swizzle.
int make_tmap_3d(CUtensorMap* map, CUtensorMapDataType dtype, const void* base, uint64_t inner, uint64_t mid,
                 uint64_t outer, uint64_t mid_stride_bytes, uint64_t outer_stride_bytes, uint32_t box_inner,
                 uint32_t box_mid);

// [world][M][N/world] -> row-major M x N for 4-byte (FP32) or 2-byte (BF16) elements.
int unshard_elems(const void* src, void* dst, int M, int N, int world, int elem_bytes, cudaStream_t stream);

inline int env_int(const char* name, int dflt) {
  const char* s = getenv(name);
  return s && *s ? atoi(s) : dflt;
}

// Co-resident CTA pairs of a persistent `__cluster_dims__(2,1,1)` kernel (clusters must fit
// inside one GPC, so this can be below sms / 2); falls back to sms / 2 if the query fails.
template <typename Kernel>
int pair_clusters_resident(Kernel kern, int threads, int smem_bytes, const DeviceState& d) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (d.sms / 2), 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem_bytes;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = d.sms / 2;
  }
  return n;
}

// Launches a kernel that waits for the one before it by itself (grid_dependency_wait, bw_ptx.cuh).
template <typename Kernel, typename... Args>
cudaError_t launch_dependent(Kernel kern, dim3 grid, int block, size_t smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace bw
