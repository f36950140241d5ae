// serve.h -- shared pieces of the batched serving operators (host side and
// device helpers): element types, the thread's last error message, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/vtq.h"
#include "vtq_internal.h"

namespace vtq {

// Records `msg` as this thread's vtq_device_last_error and returns `s`.
vtq_status serve_fail(vtq_status s, const char* fmt, ...);
// VTQ_OK, or VTQ_ERR_GPU / VTQ_ERR_OOM with the CUDA error in the message.
vtq_status serve_cuda(cudaError_t e, const char* where);

// Bits of the operators' optional device status word (vtq.h).
enum : unsigned { SERVE_BAD_INDEX = 2u };

inline int serve_elt(int dtype) {  // bytes per element, 0 for a type the operators do not take
  return dtype == VTQ_F32 ? 4 : dtype == VTQ_F16 || dtype == VTQ_BF16 ? 2 : 0;
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The kernel's limit of dynamic shared memory, raised once for each device (the call takes about 1 us).
// `done` is the caller's own static word, a bit a device.
inline cudaError_t allow_smem(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1))) return e;
  int most = 0;
  if ((e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev)) != cudaSuccess) return e;
  cudaFuncAttributes f;
  if ((e = cudaFuncGetAttributes(&f, kernel)) != cudaSuccess) return e;
  if ((size_t)most < bytes + f.sharedSizeBytes) return cudaErrorInvalidConfiguration;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)f.sharedSizeBytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  return e;
}

// A launch that may begin while the kernel before it in the stream ends (programmatic dependent launch):
// the kernel begins with tc5::grid_wait(), which waits for that kernel and, through it, all before.
template <typename... KArgs, typename... Args>
cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, unsigned block, size_t smem, int cluster, cudaStream_t st,
                         Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    n++;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  kernel_launch_count()++;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

}  // namespace vtq
