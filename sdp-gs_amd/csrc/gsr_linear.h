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
  void* out;  // gated dz: [I, 2J], gate then up; dw: where there is one range, else NULL
  int64_t out_row;
  float* part;      // dw: [splits][I][J]
  // The bias gradient's partial sums, or NULL.  dw: [splits][I], row sums of A.  dz in 16 bits:
  // [sum_rows][J, gated 2J], sums over a wave's rows of the gradients before they are rounded.
  float* part_sum;
  int64_t* sum_rows;  // dz, on the host: receives their number
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

// gelu(z) = z cdf(z) = max(z, 0) - |z| T(|z|), T(a) = cdf(-a), the normal distribution's tail.
// log2 T is nearly a parabola: a weighted minimax polynomial of degree 8 on [0, 8] (fitted to
// T itself) gives |z| T to 5e-8 with one exponential and no division.  Beyond 8 the term stays what
// it is there, 5e-15.  NaN and -inf give NaN, as 0.5 z (1 + erf(z / sqrt 2)) does.
__device__ __forceinline__ float relu_exact(float z) { return fmaf(0.5f, z, 0.5f * fabsf(z)); }
__device__ __forceinline__ float gelu_value(float z) {
  const float a = fminf(fabsf(z), 8.0f);
  float p = fmaf(-1.9919228e-06f, a, 2.9272256e-05f);
  p = fmaf(p, a, -1.380893e-04f);
  p = fmaf(p, a, -2.5343438e-04f);
  p = fmaf(p, a, 7.2163874e-03f);
  p = fmaf(p, a, -5.2603047e-02f);
  p = fmaf(p, a, -4.5917222e-01f);
  p = fmaf(p, a, -1.1511097f);
  p = fmaf(p, a, -0.9999999f);
  return fmaf(-a, __builtin_amdgcn_exp2f(p), relu_exact(z));
}
// gelu'(z) = 1/2 + sign(z) (1/2 - h(|z|)), h(a) = T(a) - a density(a) = exp(-a^2/2) Q(a): the
// exponential has the steep part, Q is a minimax polynomial of degree 10 on [0, 6] (h to 1.7e-7);
// beyond 6 h stays what it is there, -3.5e-8.
// The value shares both: T(a) = exp(-a^2/2) (Q(a) + a / sqrt(2 pi)).
__device__ __forceinline__ float gelu_both(float z, float& value) {
  const float a = fminf(fabsf(z), 6.0f);
  const float e = __builtin_amdgcn_exp2f(a * a * -0.72134752f);
  float q = fmaf(1.2712853e-06f, a, -2.8994787e-05f);
  q = fmaf(q, a, 2.951621e-04f);
  q = fmaf(q, a, -1.8013967e-03f);
  q = fmaf(q, a, 7.5418255e-03f);
  q = fmaf(q, a, -2.3762807e-02f);
  q = fmaf(q, a, 6.0701676e-02f);
  q = fmaf(q, a, -1.3230555e-01f);
  q = fmaf(q, a, 2.4986956e-01f);
  q = fmaf(q, a, -7.9787475e-01f);
  q = fmaf(q, a, 4.9999988e-01f);
  value = fmaf(-a, e * fmaf(a, 0.39894228f, q), relu_exact(z));
  return fmaf(z, 0.0f, 0.5f) + copysignf(fmaf(-e, q, 0.5f), z);  // z * 0: NaN stays NaN
}

// silu's exponential and reciprocal are the hardware's, each within a few 2^-24 of its value.
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == GSR_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays NaN
  if constexpr (ACT == GSR_ACT_GELU) return gelu_value(z);
  if constexpr (ACT == GSR_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __expf(-z));
  return z;
}

// The activation's slope at z, and its value.
template <int ACT>
__device__ __forceinline__ float act_both(float z, float& value) {
  if constexpr (ACT == GSR_ACT_GELU) return gelu_both(z, value);
  if constexpr (ACT == GSR_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    value = z * s;
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  value = act_value<ACT>(z);
  if constexpr (ACT == GSR_ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;  // 1 at NaN: the gradient goes through
  return 1.0f;
}

}  // namespace gsr
