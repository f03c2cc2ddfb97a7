// Helpers shared by the training-step kernels (optim.cu, embed.cu, logprob.cu): errors, the device
// guard of a C entry, element types, 16-byte loads and stores. Not part of the C ABI.
#pragma once
#include "../../include/suika_reshard.h"
#include "internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <exception>
#include <string>
#include <utility>

namespace suika_train {

inline int tfail(int code, const std::string& msg) { return suika_rs::fail(code, msg); }

inline int tcuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return RS_OK;
  return tfail(RS_ERR_CUDA, std::string(what) + ": " + cudaGetErrorName(e) + " (" + cudaGetErrorString(e) + ")");
}

// Makes `device` current for one C entry and puts the caller's device back.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    err = cudaGetDevice(&prev_);
    if (err == cudaSuccess && prev_ != device) {
      err = cudaSetDevice(device);
      switched_ = err == cudaSuccess;
    }
  }
  ~DeviceGuard() {
    if (switched_) cudaSetDevice(prev_);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
  cudaError_t err = cudaSuccess;

 private:
  int prev_ = 0;
  bool switched_ = false;
};

// Multiprocessors of a device (148 on a B200), for grid sizes; asked of the driver on each call.
inline int sm_count(int device) {
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) sms = 148;
  return sms;
}

inline int dtype_bytes(uint32_t dtype) { return dtype == RS_F32 ? 4 : 2; }
inline bool dtype_known(uint32_t dtype) { return dtype <= RS_F16; }

// Whether one of the addresses does not lie at a multiple of `bytes` (NULL does).
template <class... P>
bool misaligned(int bytes, P... p) {
  return (((uint64_t)p % bytes != 0) || ...);
}

// Runs `body` so that no C++ exception leaves a C entry.
template <class F>
int guarded(const char* what, F&& body) {
  try {
    return body();
  } catch (const std::exception& e) {
    return tfail(RS_ERR_ARG, std::string(what) + ": " + e.what());
  } catch (...) {
    return tfail(RS_ERR_ARG, std::string(what) + ": unknown exception");
  }
}

// Launches a kernel that follows another of the same call on the stream: it may be set up while its
// predecessor runs out (programmatic dependent launch), and begins with after_predecessor().
template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, dim3 block, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// ---- device side --------------------------------------------------------------------------

// Waits until the kernel before this one has ended and its stores are visible. Every thread of a kernel
// launched by launch_after calls it first, also one that has nothing to do: the next kernel takes
// the end of this one for the end of both.
__device__ __forceinline__ void after_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next kernel's CTAs be set up as soon as every CTA of this one has begun to end.
__device__ __forceinline__ void let_successor_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// 16 bytes that this launch reads once (no L1 line is kept for them).
__device__ __forceinline__ uint4 ld16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void st16(void* p, uint4 v) {
  asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};" :: "l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// Round to nearest even, the one rounding of a result that was computed in 32 bits.
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float2 bf16x2_f32(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 f16x2_f32(uint32_t w) {
  __half2 h;
  *reinterpret_cast<uint32_t*>(&h) = w;
  return __half22float2(h);
}
__device__ __forceinline__ uint32_t f32_bf16x2(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t f32_f16x2(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// The values of one 16-byte vector of T: 4 fp32 or 8 of 16 bits.
template <class T> struct Vec16 { static constexpr int N = 16 / sizeof(T); };
template <class T> __device__ __forceinline__ void unpack16(uint4 v, float* x);
template <> __device__ __forceinline__ void unpack16<float>(uint4 v, float* x) {
  x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}
template <> __device__ __forceinline__ void unpack16<__nv_bfloat16>(uint4 v, float* x) {
  float2 a = bf16x2_f32(v.x), b = bf16x2_f32(v.y), c = bf16x2_f32(v.z), d = bf16x2_f32(v.w);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}
template <> __device__ __forceinline__ void unpack16<__half>(uint4 v, float* x) {
  float2 a = f16x2_f32(v.x), b = f16x2_f32(v.y), c = f16x2_f32(v.z), d = f16x2_f32(v.w);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}
template <class T> __device__ __forceinline__ uint4 pack16(const float* x);
template <> __device__ __forceinline__ uint4 pack16<float>(const float* x) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
template <> __device__ __forceinline__ uint4 pack16<__nv_bfloat16>(const float* x) {
  return make_uint4(f32_bf16x2(x[0], x[1]), f32_bf16x2(x[2], x[3]), f32_bf16x2(x[4], x[5]), f32_bf16x2(x[6], x[7]));
}
template <> __device__ __forceinline__ uint4 pack16<__half>(const float* x) {
  return make_uint4(f32_f16x2(x[0], x[1]), f32_f16x2(x[2], x[3]), f32_f16x2(x[4], x[5]), f32_f16x2(x[6], x[7]));
}

}  // namespace suika_train
