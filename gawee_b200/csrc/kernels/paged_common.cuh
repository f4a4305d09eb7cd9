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

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exp(s - m); a maximum of -inf (nothing attended yet) leaves exp(-inf) = 0, and NaN for a NaN score.
__device__ __forceinline__ float exp_from(float s, float m) {
  return exp2_fast((s - (m == -INFINITY ? 0.f : m)) * kLog2e);
}
__device__ __forceinline__ void add_scaled(float4& to, const float4& x, float f) {
  to.x += x.x * f;
  to.y += x.y * f;
  to.z += x.z * f;
  to.w += x.w * f;
}

// Elements d .. d + 3 of a head's result, from the sum of its weights `lt` (relative to their maximum `mt`).
__device__ __forceinline__ void store_result(const KvAttendParams& p, int b, int head, int d, float mt, float lt,
                                             const float4& o) {
  const bool any = lt != 0.f;
  store_act4(p.out, p.dt, b * p.out_stride + (int64_t)head * p.geom.head_dim + d, any ? o.x / lt : 0.f,
             any ? o.y / lt : 0.f, any ? o.z / lt : 0.f, any ? o.w / lt : 0.f);
  if (p.weights_out && d == 0)
    reinterpret_cast<float2*>(p.stats)[(int64_t)b * p.heads + head] = make_float2(mt, lt);
}

}  // namespace paged
}  // namespace kern
}  // namespace gawee
