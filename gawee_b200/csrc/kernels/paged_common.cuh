// Element types and small device helpers of the paged key/value cache kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "paged_kv.h"

namespace gawee {
namespace kern {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void set_status(int* st, int code) {
  if (st) atomicCAS(st, 0, code);
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <class T>
struct TypeCode;
template <>
struct TypeCode<float> { static constexpr int value = DT_F32; };
template <>
struct TypeCode<__half> { static constexpr int value = DT_F16; };
template <>
struct TypeCode<__nv_bfloat16> { static constexpr int value = DT_BF16; };

// Element i of an activation array whose type is only known at run time: the
// few values a block reads once or writes once.
__device__ __forceinline__ float load_act(const void* p, int dt, int64_t i) {
  if (dt == DT_F32) return static_cast<const float*>(p)[i];
  if (dt == DT_F16) return to_f(static_cast<const __half*>(p)[i]);
  return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
}

template <class A>
__device__ __forceinline__ void store4(A* p, float a, float b, float c, float d) {
  p[0] = from_f<A>(a);
  p[1] = from_f<A>(b);
  p[2] = from_f<A>(c);
  p[3] = from_f<A>(d);
}
__device__ __forceinline__ void store_act4(void* p, int dt, int64_t i, float a, float b, float c, float d) {
  if (dt == DT_F32) store4(static_cast<float*>(p) + i, a, b, c, d);
  else if (dt == DT_F16) store4(static_cast<__half*>(p) + i, a, b, c, d);
  else store4(static_cast<__nv_bfloat16*>(p) + i, a, b, c, d);
}

}  // namespace paged
}  // namespace kern
}  // namespace gawee
