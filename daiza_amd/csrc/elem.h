// elem.h — element types of device arrays (DZ_F32, DZ_F16, DZ_BF16) and the checks of device pointers.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "runtime.h"

namespace dz {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__hip_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half(x); }
template <>
__device__ __forceinline__ __hip_bfloat16 from_f32<__hip_bfloat16>(float x) { return __float2bfloat16(x); }

inline int check_type(int type) {
  if (type == DZ_F32 || type == DZ_F16 || type == DZ_BF16) return DZ_OK;
  return set_error(DZ_ERR_UNSUPPORTED, "element type %d (F32 0, F16 1, BF16 30)", type);
}
template <class F>
int with_type(int type, F&& f) {
  switch (type) {
    case DZ_F32: return f((float*)nullptr);
    case DZ_F16: return f((__half*)nullptr);
    case DZ_BF16: return f((__hip_bfloat16*)nullptr);
    default: return check_type(type);
  }
}

// A kernel that is handed host memory, or another device's, ends the process: such arrays are refused before the launch.
inline int check_array(const void* p, size_t align, int device, const char* what) {
  hipPointerAttribute_t a{};
  const hipError_t e = hipPointerGetAttributes(&a, p);
  if (e != hipSuccess) (void)hipGetLastError();
  if (e != hipSuccess || (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged) || a.device != device)
    return set_error(DZ_ERR_TENSOR, "%s is not in the memory of device %d", what, device);
  if (reinterpret_cast<uintptr_t>(p) % align) return set_error(DZ_ERR_TENSOR, "%s is not aligned to %zu bytes", what, align);
  return DZ_OK;
}
inline size_t type_size(int type) { return type == DZ_F32 ? 4 : 2; }

}  // namespace dz
