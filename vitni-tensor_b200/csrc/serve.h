// serve.h -- shared pieces of the batched serving operators (host side and
// device helpers): element types, the thread's last error message, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/vtq.h"

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
