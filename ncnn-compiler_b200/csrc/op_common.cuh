// What the stand-alone operators on device arrays share: element types, wide loads and stores, checks of arguments.
#pragma once

#include "../../include/ncnn_b200.h"

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "device_guard.h"

namespace nb {

void set_global_error(const std::string& message);  // c_api.cu

// ------------------------------------------------------------------ elements
// 16-bit elements become fp32 on the way in and are rounded once, to nearest even, on the way out.
template <class T> __device__ __forceinline__ float op_get(T v);
template <> __device__ __forceinline__ float op_get<float>(float v) { return v; }
template <> __device__ __forceinline__ float op_get<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float op_get<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T op_put(float v);
template <> __device__ __forceinline__ float op_put<float>(float v) { return v; }
template <> __device__ __forceinline__ __half op_put<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 op_put<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements at an address that is a multiple of their size together (N elements of at most 16 bytes).
template <class T, int N>
struct alignas(sizeof(T) * N) OpVec {
  T e[N];
};

// ------------------------------------------------------------------ host side
inline int op_elem_bytes(int32_t type) { return type == NCNN_B200_F32 ? 4 : 2; }
inline bool op_type_ok(int32_t type) { return type == NCNN_B200_F32 || type == NCNN_B200_F16 || type == NCNN_B200_BF16; }

inline int op_fail(int status, const std::string& message) {
  set_global_error(message);
  return status;
}

// The device that `p` lives on; negative where it is no memory that a kernel of this process can reach.  (The driver's own
// call: 0.1 us an array less than the runtime's, of some 5.7 that a small call takes on the host.)
inline int op_device_of(const void* p) {
  using AttributesFn = CUresult (*)(unsigned, CUpointer_attribute*, void**, CUdeviceptr);
  static const AttributesFn attributes = [] {
    cudaDriverEntryPointQueryResult query;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuPointerGetAttributes", &f, cudaEnableDefault, &query) != cudaSuccess || query != cudaDriverEntryPointSuccess) f = nullptr;
    return reinterpret_cast<AttributesFn>(f);
  }();
  if (attributes != nullptr) {
    unsigned type = 0;
    int device = -1;
    CUpointer_attribute which[2] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL};
    void* to[2] = {&type, &device};
    if (attributes(2, which, to, reinterpret_cast<CUdeviceptr>(p)) == CUDA_SUCCESS && type == CU_MEMORYTYPE_DEVICE) return device;
  }
  cudaPointerAttributes a{};
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  return a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged ? a.device : -1;
}

// Whether an array starts where its elements can: a kernel would fault on one that does not.
inline bool op_starts(const void* p, int elem_bytes) { return reinterpret_cast<uintptr_t>(p) % elem_bytes == 0; }

// Every array of a call on one device: that device, or a message.
inline int op_common_device(const char* op, std::initializer_list<const void*> arrays, std::string* why) {
  int device = -1;
  for (const void* p : arrays) {
    if (p == nullptr) continue;
    const int d = op_device_of(p);
    if (d < 0) {
      *why = std::string(op) + ": an array is not in device memory";
      return -1;
    }
    if (device >= 0 && d != device) {
      *why = std::string(op) + ": the arrays are on different devices";
      return -1;
    }
    device = d;
  }
  return device;
}

inline int op_sm_count(int device) {
  int n = 148;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
  return n;
}

// The status of a launch: what the launch itself answered.  (cudaGetLastError holds errors of earlier calls, too: a model that
// could not be laid out would make the next operator fail.)
inline int op_launched(const char* op, cudaError_t e) {
  if (e == cudaSuccess) return NCNN_B200_STATUS_SUCCESS;
  cudaGetLastError();  // said here, and not to be met by another call
  return op_fail(NCNN_B200_STATUS_RUNTIME, std::string(op) + ": launch failed: " + cudaGetErrorString(e));
}

// CTAs of `cluster` along x, if any
template <class... P, class... A>
inline cudaError_t op_launch(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t st, int cluster, const A&... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute size{};
  size.id = cudaLaunchAttributeClusterDimension;
  size.val.clusterDim.x = cluster;
  size.val.clusterDim.y = size.val.clusterDim.z = 1;
  c.attrs = &size;
  c.numAttrs = cluster > 0 ? 1 : 0;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

// f(T{}) with the element type that `type` names
template <class F>
inline int op_by_type(int32_t type, F&& f) {
  if (type == NCNN_B200_F32) return f(float{});
  if (type == NCNN_B200_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

// No C++ exception leaves an entry point.
template <class F>
inline int op_guarded(const char* op, F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    try {
      set_global_error(std::string(op) + ": internal error: " + e.what());
    } catch (...) {
    }
    return NCNN_B200_STATUS_RUNTIME;
  } catch (...) {
    return NCNN_B200_STATUS_RUNTIME;
  }
}

}  // namespace nb
