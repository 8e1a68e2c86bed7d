// gsr_rows.h -- the product of few rows (a handful of points, one token): the weights' bytes are
// the bound, and latency where they are few.
//
// A workgroup takes 16 outputs and up to 64 rows; its 8 waves share the inputs among themselves,
// 64 at a time, and add up their sums through LDS at the end, in a fixed order.  Both operands come
// from memory straight into the matrix instruction's layout: nothing is staged, so every load of a
// wave's next 256 inputs is in flight at once.  A lane reads 32 consecutive bytes of its row (64 in
// 32 bits), four lanes a whole cache line.
#pragma once
#include "gsr_product.h"

namespace gsr {

template <typename T, int EPI, bool GATED, int MI>
__global__ __launch_bounds__(512) void rows_kernel(ProductArgs p) {
  constexpr int kPlanes = Operand<T>::kPlanes, kWaves = 8, G = GATED ? 2 : 1;
  constexpr int kUnroll = sizeof(T) == 4 || MI * G > 2 ? 2 : 4;
  __shared__ f32x4 sums[kWaves][G * MI][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int m = lane & 15, q = lane >> 4;
  const int64_t j0 = (int64_t)blockIdx.x * 16, i0 = (int64_t)blockIdx.y * (16 * MI);
  // a row past the last is the last one again: its results are not stored
  const int64_t j = j0 + m < p.J ? j0 + m : p.J - 1;
  const T* w[G];
#pragma unroll
  for (int g = 0; g < G; g++) w[g] = (const T*)p.b[g] + j * p.b_j;
  const T* x[MI];
#pragma unroll
  for (int u = 0; u < MI; u++) {
    const int64_t i = i0 + u * 16 + m;
    x[u] = (const T*)p.a + (i < p.I ? i : p.I - 1) * p.a_i;
  }
  f32x4 acc[G][MI] = {};
  auto step = [&](auto tail, int64_t k0, auto count) {
    constexpr int N = decltype(count)::value;
    constexpr bool TAIL = decltype(tail)::value;
    Chunk<T> cw[N][2][G], cx[N][2][MI];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        // any order of the inputs will do as long as both operands have it
        const int64_t k = k0 + n * (64 * kWaves) + q * 16 + h * 8;
#pragma unroll
        for (int g = 0; g < G; g++) cw[n][h][g] = TAIL ? load_tail(w[g], k, 1, p.R) : load_whole(w[g] + k);
#pragma unroll
        for (int u = 0; u < MI; u++) cx[n][h][u] = TAIL ? load_tail(x[u], k, 1, p.R) : load_whole(x[u] + k);
      }
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        s16x8 b[G][kPlanes], a[kPlanes];
#pragma unroll
        for (int g = 0; g < G; g++) split_chunk<T>(b[g], cw[n][h][g]);
#pragma unroll
        for (int u = 0; u < MI; u++) {
          split_chunk<T>(a, cx[n][h][u]);
#pragma unroll
          for (int z = 0; z < Parts<kPlanes>::kProducts; z++)
#pragma unroll
            for (int g = 0; g < G; g++)
              acc[g][u] = mfma<T>(b[g][Parts<kPlanes>::kB[z]], a[Parts<kPlanes>::kA[z]], acc[g][u]);
        }
      }
  };
  int64_t k0 = wave * 64;
  for (; k0 + (kUnroll - 1) * (64 * kWaves) + 64 <= p.R; k0 += kUnroll * (64 * kWaves))
    step(Const<0>(), k0, Const<kUnroll>());
  for (; k0 + 64 <= p.R; k0 += 64 * kWaves) step(Const<0>(), k0, Const<1>());
  if (k0 < p.R) step(Const<1>(), k0, Const<1>());

#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int u = 0; u < MI; u++) sums[wave][g * MI + u][lane] = acc[g][u];
  __syncthreads();
  if (wave >= MI) return;  // wave u finishes rows 16 u..
  const int64_t i = i0 + wave * 16 + m, jq = j0 + 4 * q, n = p.J - jq;
  if (i >= p.I || n <= 0) return;
  float v[4], u[4] = {}, e[4] = {}, bias[4] = {}, bias1[4] = {};
  f32x4 total[G] = {};
#pragma unroll
  for (int g = 0; g < G; g++) {
#pragma unroll
    for (int z = 0; z < kWaves; z++) total[g] += sums[z][g * MI + wave][lane];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (jq + k < p.J && !(fabsf(total[g][k]) <= 3.4e38f))
          total[g][k] = exact_sum((const float*)p.a, p.a_i, 1, (const float*)p.b[g], nullptr, p.b_j, 1, 1, 0, i, jq + k, 0, p.R);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int64_t at = k < n ? jq + k : p.J - 1;
    if (p.bias[0]) bias[k] = to_f(((const T*)p.bias[0])[at]);
    if (GATED && p.bias[1]) bias1[k] = to_f(((const T*)p.bias[1])[at]);
    if (p.extra) e[k] = to_f(((const T*)p.extra)[i * p.extra_row + at]);
    v[k] = total[0][k] + bias[k];
    if (GATED) u[k] = total[G - 1][k] + bias1[k];
  }
  with_act<EPI>(p.act, [&](auto act) {
    T* out = (T*)p.out + i * p.out_row + jq;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (k >= n) continue;
      const float a = act_value<decltype(act)::value>(v[k]);
      out[k] = from_f<T>(GATED ? a * u[k] : a + e[k]);
    }
  });
}

template <typename T, int EPI, bool GATED>
int launch_rows(const ProductArgs& p, hipStream_t s) {
  const int64_t tiles = (p.J + 15) / 16;
  if (tiles > 0x7fffffff) return 1;
  if (p.I <= 16)
    hipLaunchKernelGGL((rows_kernel<T, EPI, GATED, 1>), dim3((uint32_t)tiles, 1), dim3(512), 0, s, p);
  else if (p.I <= 32)
    hipLaunchKernelGGL((rows_kernel<T, EPI, GATED, 2>), dim3((uint32_t)tiles, 1), dim3(512), 0, s, p);
  else
    hipLaunchKernelGGL((rows_kernel<T, EPI, GATED, 4>), dim3((uint32_t)tiles, (uint32_t)((p.I + 63) / 64)), dim3(512), 0, s, p);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

// Where this kernel is faster than the tiled one, whole or with its sum cut into ranges: where a wave's
// own part of the sum is short -- R (1 + blocks of 16 rows) elements come in for each workgroup of 16
// outputs, more than 256 workgroups take turns -- or where the weights of a single block of rows
// stream through every CU.  us, these : tiled, bf16 64x1024x1024 7.6 : 9.2, 256x512x512 5.5 : 6.3,
// 1x4096x4096 7.6 : 10.1, gated 16x2048x5504 14.2 : 14.9, but 64x4096x1024 20.6 : 9.1, 32x4096x4096
// 14.1 : 11.7, 128x256x8192 10.5 : 5.2; fp32 64x512x512 8.2 : 11.5, 16x4096x4096 21.3 : 24.7, but
// 64x8192x1024 79.7 : 17.6, 64x1024x6144 24.3 : 18.2.  Of 848 sizes (1 to 256 rows, 256 to 8192
// inputs and outputs) the rule is 0.8 % off the faster one on average, at worst 1.44 times (fp32,
// gated 1x4096x8192 95.5 : 66.1).
inline bool rows_sizes(int64_t I, int64_t J, int64_t R) {
  if (I > 256) return false;
  const int64_t blocks = I > 64 ? 4 : (I + 15) / 16, groups = (J + 15) / 16 * ((I + 63) / 64);
  if (groups >= 256 && blocks == 1) return true;
  if (groups > 256 && I > 64) return false;
  return R * (1 + blocks) * (groups > 256 ? groups : 256) <= 5120 * 256;
}

}  // namespace gsr
