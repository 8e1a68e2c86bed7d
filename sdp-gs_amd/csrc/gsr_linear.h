// gsr_linear.h -- what the product kernels of gsr_linear*.hip share: the arguments of one product,
// element conversions and the activations.
//
// Every product is C(i, j) = sum_r A(i, r) B(j, r) with an epilogue:
//   forward   i = row of x, j = output,  r = input:   y = act(C + bias) + residual
//   dz        the same product again:                 dz = dy * act'(C + bias)
//   dx        i = row of x, j = input,   r = output:  dx = C
//   dw        i = output,   j = input,   r = row of x: partial sums over ranges of r
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/gsr_linear.h"

namespace gsr {

struct ProductArgs {
  const void* a;
  int64_t a_i, a_r;  // element strides of A(i, r)
  const void* b[2];  // gated forward: gate and up weights; dx of a gated pair: its two segments
  int64_t b_j, b_r;
  int64_t I, J, R;
  int segments;     // dx of a gated pair: R is summed over twice, A moving on by a_segment elements
  int64_t a_segment;
  int64_t r_chunk;  // dw: rows of x per partial sum
  const void* bias[2];
  const void* extra;  // forward: residual; dz: dy
  int64_t extra_row;
  void* out;  // gated dz: [I, 2J], gate then up
  int64_t out_row;
  float* part;      // dw: [splits][I][J]
  float* part_sum;  // dw: [splits][I] row sums of A (the bias gradient), or NULL
  int act;
};

enum { EPI_FORWARD, EPI_DZ, EPI_PLAIN, EPI_PARTIAL };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half(v); }
template <> __device__ __forceinline__ __hip_bfloat16 from_f<__hip_bfloat16>(float v) {
  return __float2bfloat16(v);
}

// The normal distribution's integral and exp(-z^2/2): Abramowitz & Stegun 7.1.26 (a rational
// approximation of erf, absolute error below 1.5e-7, a float's own rounding next to 1), which
// shares its exponential with the density that gelu's slope needs.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f));
  e = __expf(-x * x);
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float tail = 0.5f * p * t * e;  // 1 - cdf(|z|)
  return z < 0.0f ? tail : 1.0f - tail;
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == GSR_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays NaN
  if constexpr (ACT == GSR_ACT_GELU) {
    float e;
    return z * normal_cdf(z, e);
  }
  if constexpr (ACT == GSR_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __expf(-z));
  return z;
}

// The activation's value and slope at z.
template <int ACT>
__device__ __forceinline__ float act_both(float z, float& value) {
  if constexpr (ACT == GSR_ACT_GELU) {
    float e;
    const float c = normal_cdf(z, e);
    value = z * c;
    return fmaf(z * 0.39894228040143268f, e, c);
  }
  if constexpr (ACT == GSR_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    value = z * s;
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  value = act_value<ACT>(z);
  if constexpr (ACT == GSR_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  return 1.0f;
}

}  // namespace gsr
