// What the kernels on rows of scores share (distill.cu, top_logits.cu, balance.cu): element types, sums of exponentials, order.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "clb_common.cuh"

namespace clb {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A set of exponents as (m, l): the largest value and the sum of exp((value - m) / T).  m = -inf, l = 0: none.  NaN is kept in l.
struct ExpSum {
    float m, l;
};
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }
// d * c with c = log2(e) / T: differences from the largest value are taken before anything is scaled, so that a value of the type's lowest stays one
__device__ __forceinline__ float exp_diff(float v, float m, float c) { return exp2f((v - m) * c); }
__device__ __forceinline__ ExpSum single(float v) { return {v != v ? -INFINITY : v, v != v ? v : v == -INFINITY ? 0.f : 1.f}; }
__device__ __forceinline__ ExpSum merge(ExpSum a, ExpSum b, float c)
{
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.l + b.l}; // nothing, or NaN in l
    return {m, a.l * exp_diff(a.m, m, c) + b.l * exp_diff(b.m, m, c)};
}

// Order of scores as unsigned integers: larger is larger, -0 equals +0, NaN above everything; never 0 and never all ones, which stand for "before the
// first" and "after the last" where keys are compared.
__device__ __forceinline__ uint32_t order_key(float v)
{
    if (v != v) return 0xfffffffeu;
    const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

} // namespace clb

namespace clb_host {
// calls f with a value of the element type that dtype names; false for another dtype
template <typename F> inline bool with_score_type(int dtype, F &&f)
{
    if (dtype == CLB_F32) f(0.f);
    else if (dtype == CLB_F16) f(__half());
    else if (dtype == CLB_BF16) f(__nv_bfloat16());
    else return false;
    return true;
}
} // namespace clb_host
