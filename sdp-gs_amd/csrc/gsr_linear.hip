// gsr_linear.hip -- fused linear layer and gated pair, forward and backward (include/gsr_linear.h).
#include "gsr_linear.h"

namespace {

using namespace gsr;

constexpr int kTile = 64, kDepth = 16;

// One 64x64 tile of C per workgroup, 4x4 sums per lane in 32-bit FMAs, both operands staged
// through LDS as floats.  Any strides, any sizes.
template <typename T, int EPI, bool GATED>
__global__ __launch_bounds__(256) void product_kernel(ProductArgs p) {
  constexpr int G = GATED ? 2 : 1;
  __shared__ float sa[kDepth][kTile + 4], sb[G][kDepth][kTile + 4];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t i0 = (int64_t)blockIdx.x * kTile, j0 = (int64_t)blockIdx.y * kTile;
  const T* A = (const T*)p.a;
  float acc[G][4][4] = {}, sum[4] = {};
  int64_t r_begin = 0, r_end = p.R;
  if (EPI == EPI_PARTIAL) {
    r_begin = (int64_t)blockIdx.z * p.r_chunk;
    r_end = r_begin + p.r_chunk < p.R ? r_begin + p.r_chunk : p.R;
  }
  for (int s = 0; s < (EPI == EPI_PLAIN ? p.segments : 1); s++) {
    for (int64_t r0 = r_begin; r0 < r_end; r0 += kDepth) {
      for (int e = threadIdx.x; e < kTile * kDepth; e += 256) {
        const int r = p.a_r == 1 ? e % kDepth : e / kTile, i = p.a_r == 1 ? e / kDepth : e % kTile;
        const bool in = i0 + i < p.I && r0 + r < r_end;
        sa[r][i] = in ? to_f(A[(i0 + i) * p.a_i + (r0 + r) * p.a_r]) : 0.0f;
        const int rb = p.b_r == 1 ? e % kDepth : e / kTile, j = p.b_r == 1 ? e / kDepth : e % kTile;
        const bool inb = j0 + j < p.J && r0 + rb < r_end;
        for (int g = 0; g < G; g++)
          sb[g][rb][j] =
              inb ? to_f(((const T*)p.b[GATED ? g : s])[(j0 + j) * p.b_j + (r0 + rb) * p.b_r])
                  : 0.0f;
      }
      __syncthreads();
      for (int r = 0; r < kDepth; r++) {
        for (int u = 0; u < 4; u++) {
          const float a = sa[r][ty * 4 + u];
          if (EPI == EPI_PARTIAL) sum[u] += a;
          for (int g = 0; g < G; g++)
            for (int v = 0; v < 4; v++) acc[g][u][v] = fmaf(a, sb[g][r][tx * 4 + v], acc[g][u][v]);
        }
      }
      __syncthreads();
    }
    A += p.a_segment;
  }
  for (int u = 0; u < 4; u++) {
    const int64_t i = i0 + ty * 4 + u;
    if (i >= p.I) break;
    if (EPI == EPI_PARTIAL && p.part_sum && blockIdx.y == 0 && tx == 0)
      p.part_sum[(int64_t)blockIdx.z * p.I + i] = sum[u];
    for (int v = 0; v < 4; v++) {
      const int64_t j = j0 + tx * 4 + v;
      if (j >= p.J) break;
      if (EPI == EPI_PARTIAL) {
        p.part[((int64_t)blockIdx.z * p.I + i) * p.J + j] = acc[0][u][v];
        continue;
      }
      T* out = (T*)p.out + i * p.out_row + j;
      if (EPI == EPI_PLAIN) {
        *out = from_f<T>(acc[0][u][v]);
        continue;
      }
      const float z = acc[0][u][v] + (p.bias[0] ? to_f(((const T*)p.bias[0])[j]) : 0.0f);
      const float ex = p.extra ? to_f(((const T*)p.extra)[i * p.extra_row + j]) : 0.0f;
      if (GATED) {
        const float w = acc[G - 1][u][v] + (p.bias[1] ? to_f(((const T*)p.bias[1])[j]) : 0.0f);
        if (EPI == EPI_FORWARD) {
          *out = from_f<T>(act_value(z, p.act) * w);
        } else {
          out[0] = from_f<T>(ex * w * act_slope(z, p.act));
          out[p.J] = from_f<T>(ex * act_value(z, p.act));
        }
      } else {
        *out = from_f<T>(EPI == EPI_FORWARD ? act_value(z, p.act) + ex : ex * act_slope(z, p.act));
      }
    }
  }
}

// out[e] = sum over the splits of part[s][e], in a fixed order; the row sums follow the products.
template <typename T>
__global__ __launch_bounds__(256) void reduce_kernel(const float* part, const float* part_sum,
                                                     int splits, int64_t n, int64_t n_sum, T* dw,
                                                     T* db) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool first = e < n;
  if (!first && e - n >= n_sum) return;
  const float* src = first ? part + e : part_sum + (e - n);
  const int64_t step = first ? n : n_sum;
  float v = 0.0f;
  for (int s = 0; s < splits; s++) v += src[s * step];
  if (first) dw[e] = from_f<T>(v);
  else db[e - n] = from_f<T>(v);
}

template <typename T>
__global__ __launch_bounds__(256) void zero_kernel(T* p, int64_t n) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e < n) p[e] = from_f<T>(0.0f);
}

size_t type_bytes(int dtype) { return dtype == GSR_F32 ? 4 : 2; }
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t tiles(int64_t v) { return (v + kTile - 1) / kTile; }

// Ranges of the summed rows for dw: enough workgroups to fill 256 CUs twice, each with at least
// 64 rows.
int64_t splits_of(int64_t I, int64_t J, int64_t R) {
  const int64_t t = tiles(I) * tiles(J);
  int64_t s = (512 + t - 1) / t;
  const int64_t most = (R + 63) / 64;
  s = s < most ? s : most;
  return s < 1 ? 1 : s;
}

template <typename T, int EPI, bool GATED>
int launch(const ProductArgs& p, int64_t splits, hipStream_t stream) {
  const int64_t gi = tiles(p.I), gj = tiles(p.J);
  if (gi > 0x7fffffff || gj > 65535 || splits > 65535) return 1;
  hipLaunchKernelGGL((product_kernel<T, EPI, GATED>), dim3((uint32_t)gi, (uint32_t)gj, (uint32_t)splits),
                     dim3(256), 0, stream, p);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

bool sizes_ok(int dtype, int64_t M, int64_t K, int64_t N, int act) {
  return dtype >= GSR_F32 && dtype <= GSR_BF16 && act >= GSR_ACT_NONE && act <= GSR_ACT_SILU &&
         M >= 0 && K >= 1 && N >= 1 && K <= (1 << 22) && N <= (1 << 21) && M <= (1LL << 36);
}

bool x_ok(int64_t M, int64_t K, int64_t x_row, int64_t x_col) {
  return (x_col == 1 && (x_row >= K || M <= 1)) || (x_row == 1 && (x_col >= M || K == 1));
}

// The weight gradients: partial products over ranges of x's rows, then their sum.
template <typename T>
int weight_gradients(const void* dz, int64_t dz_row, int64_t M, int64_t K, int64_t I, const void* x,
                     int64_t x_row, int64_t x_col, void* dw, void* db, char* scratch,
                     hipStream_t stream) {
  if (M == 0) {
    if (dw) hipLaunchKernelGGL(zero_kernel<T>, dim3((I * K + 255) / 256), dim3(256), 0, stream, (T*)dw, I * K);
    if (db) hipLaunchKernelGGL(zero_kernel<T>, dim3((I + 255) / 256), dim3(256), 0, stream, (T*)db, I);
    return hipGetLastError() == hipSuccess ? 0 : 2;
  }
  const int64_t splits = splits_of(I, K, M);
  ProductArgs p{};
  p.a = dz; p.a_i = 1; p.a_r = dz_row;
  p.b[0] = x; p.b_j = x_col; p.b_r = x_row;
  p.I = I; p.J = K; p.R = M; p.segments = 1;
  p.r_chunk = (M + splits - 1) / splits;
  p.part = (float*)scratch;
  p.part_sum = db ? p.part + splits * I * K : nullptr;
  if (int rc = launch<T, EPI_PARTIAL, false>(p, splits, stream)) return rc;
  const int64_t n = dw ? I * K : 0, n_sum = db ? I : 0;
  hipLaunchKernelGGL(reduce_kernel<T>, dim3((uint32_t)((n + n_sum + 255) / 256)), dim3(256), 0, stream,
                     p.part, p.part_sum, (int)splits, n, n_sum, (T*)dw, (T*)db);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

size_t partial_bytes(int64_t M, int64_t K, int64_t I) {
  return M == 0 ? 0 : (size_t)splits_of(I, K, M) * I * (K + 1) * 4;
}

template <typename T>
int linear_backward(const ProductArgs& fwd, const void* dy, int64_t dy_row, void* dx, void* dw,
                    void* db, char* scratch, hipStream_t stream) {
  const int64_t M = fwd.I, K = fwd.R, N = fwd.J;
  const void* dz = dy;
  int64_t dz_row = dy_row;
  if (fwd.act != GSR_ACT_NONE && M > 0) {
    ProductArgs p = fwd;
    p.extra = dy; p.extra_row = dy_row;
    p.out = scratch; p.out_row = N;
    if (int rc = launch<T, EPI_DZ, false>(p, 1, stream)) return rc;
    dz = scratch; dz_row = N;
    scratch += up(M * N * sizeof(T), 256);
  }
  if (dx && M > 0) {
    ProductArgs p{};
    p.a = dz; p.a_i = dz_row; p.a_r = 1;
    p.b[0] = fwd.b[0]; p.b_j = 1; p.b_r = fwd.b_j;
    p.I = M; p.J = K; p.R = N; p.segments = 1;
    p.out = dx; p.out_row = K;
    if (int rc = launch<T, EPI_PLAIN, false>(p, 1, stream)) return rc;
  }
  if (!dw && !db) return 0;
  return weight_gradients<T>(dz, dz_row, M, K, N, fwd.a, fwd.a_i, fwd.a_r, dw, db, scratch, stream);
}

template <typename T>
int gated_backward(const ProductArgs& fwd, const void* dh, int64_t dh_row, void* dx, void* dw,
                   void* db, char* scratch, hipStream_t stream) {
  const int64_t M = fwd.I, K = fwd.R, N = fwd.J;
  const void* dz = scratch;
  if (M > 0) {
    ProductArgs p = fwd;
    p.extra = dh; p.extra_row = dh_row;
    p.out = scratch; p.out_row = 2 * N;
    if (int rc = launch<T, EPI_DZ, true>(p, 1, stream)) return rc;
    scratch += up(2 * M * N * sizeof(T), 256);
    if (dx) {
      ProductArgs q{};
      q.a = dz; q.a_i = 2 * N; q.a_r = 1;
      q.b[0] = fwd.b[0]; q.b[1] = fwd.b[1]; q.b_j = 1; q.b_r = fwd.b_j;
      q.I = M; q.J = K; q.R = N; q.segments = 2; q.a_segment = N;
      q.out = dx; q.out_row = K;
      if (int rc = launch<T, EPI_PLAIN, false>(q, 1, stream)) return rc;
    }
  }
  if (!dw && !db) return 0;
  return weight_gradients<T>(dz, 2 * N, M, K, 2 * N, fwd.a, fwd.a_i, 1, dw, db, scratch, stream);
}

ProductArgs forward_args(int64_t M, int64_t K, int64_t N, const void* x, int64_t x_row,
                         int64_t x_col, const void* w, const void* w2, int64_t w_row, const void* b,
                         const void* b2, int act) {
  ProductArgs p{};
  p.a = x; p.a_i = x_row; p.a_r = x_col;
  p.b[0] = w; p.b[1] = w2; p.b_j = w_row; p.b_r = 1;
  p.I = M; p.J = N; p.R = K; p.segments = 1;
  p.bias[0] = b; p.bias[1] = b2;
  p.act = act;
  return p;
}

template <bool GATED>
int forward(int dtype, const ProductArgs& p, hipStream_t s) {
  if (dtype == GSR_F32) return launch<float, EPI_FORWARD, GATED>(p, 1, s);
  if (dtype == GSR_F16) return launch<__half, EPI_FORWARD, GATED>(p, 1, s);
  return launch<__hip_bfloat16, EPI_FORWARD, GATED>(p, 1, s);
}

}  // namespace

extern "C" int gsr_linear(int dtype, int64_t M, int64_t K, int64_t N, const void* x, int64_t x_row,
                          int64_t x_col, const void* w, int64_t w_row, const void* bias,
                          const void* residual, int64_t residual_row, int act, void* y,
                          int64_t y_row, void* stream) {
  if (!sizes_ok(dtype, M, K, N, act) || !x_ok(M, K, x_row, x_col) || w_row < K) return 1;
  if (M == 0) return 0;
  if (!x || !w || !y || y_row < N || (residual && residual_row < N && M > 1)) return 1;
  ProductArgs p = forward_args(M, K, N, x, x_row, x_col, w, nullptr, w_row, bias, nullptr, act);
  p.extra = residual; p.extra_row = residual_row;
  p.out = y; p.out_row = y_row;
  return forward<false>(dtype, p, (hipStream_t)stream);
}

extern "C" size_t gsr_linear_backward_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N,
                                                    int act, int need_dw) {
  if (!sizes_ok(dtype, M, K, N, act)) return 0;
  return (act == GSR_ACT_NONE ? 0 : (size_t)up(M * N * type_bytes(dtype), 256)) +
         (need_dw ? partial_bytes(M, K, N) : 0) + 256;
}

extern "C" int gsr_linear_backward(int dtype, int64_t M, int64_t K, int64_t N, const void* x,
                                   int64_t x_row, int64_t x_col, const void* w, int64_t w_row,
                                   const void* bias, int act, const void* dy, int64_t dy_row,
                                   void* dx, void* dw, void* dbias, void* scratch, void* stream) {
  if (!sizes_ok(dtype, M, K, N, act) || !x_ok(M, K, x_row, x_col) || w_row < K) return 1;
  if (M > 0 && (!x || !w || !dy || !scratch || (dy_row < N && M > 1))) return 1;
  const ProductArgs p = forward_args(M, K, N, x, x_row, x_col, w, nullptr, w_row, bias, nullptr, act);
  hipStream_t s = (hipStream_t)stream;
  char* t = (char*)scratch;
  if (dtype == GSR_F32) return linear_backward<float>(p, dy, dy_row, dx, dw, dbias, t, s);
  if (dtype == GSR_F16) return linear_backward<__half>(p, dy, dy_row, dx, dw, dbias, t, s);
  return linear_backward<__hip_bfloat16>(p, dy, dy_row, dx, dw, dbias, t, s);
}

extern "C" int gsr_gated(int dtype, int64_t M, int64_t K, int64_t N, const void* x, int64_t x_row,
                         const void* wg, const void* wu, int64_t w_row, const void* bg,
                         const void* bu, int act, void* h, int64_t h_row, void* stream) {
  if (!sizes_ok(dtype, M, K, N, act) || !x_ok(M, K, x_row, 1) || w_row < K) return 1;
  if (M == 0) return 0;
  if (!x || !wg || !wu || !h || h_row < N) return 1;
  ProductArgs p = forward_args(M, K, N, x, x_row, 1, wg, wu, w_row, bg, bu, act);
  p.out = h; p.out_row = h_row;
  return forward<true>(dtype, p, (hipStream_t)stream);
}

extern "C" size_t gsr_gated_backward_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N,
                                                   int need_dw) {
  if (!sizes_ok(dtype, M, K, N, GSR_ACT_NONE)) return 0;
  return (size_t)up(2 * M * N * type_bytes(dtype), 256) + (need_dw ? partial_bytes(M, K, 2 * N) : 0) +
         256;
}

extern "C" int gsr_gated_backward(int dtype, int64_t M, int64_t K, int64_t N, const void* x,
                                  int64_t x_row, const void* wg, const void* wu, int64_t w_row,
                                  const void* bg, const void* bu, int act, const void* dh,
                                  int64_t dh_row, void* dx, void* dw, void* db, void* scratch,
                                  void* stream) {
  if (!sizes_ok(dtype, M, K, N, act) || !x_ok(M, K, x_row, 1) || w_row < K) return 1;
  if (M > 0 && (!x || !wg || !wu || !dh || !scratch || (dh_row < N && M > 1))) return 1;
  const ProductArgs p = forward_args(M, K, N, x, x_row, 1, wg, wu, w_row, bg, bu, act);
  hipStream_t s = (hipStream_t)stream;
  char* t = (char*)scratch;
  if (dtype == GSR_F32) return gated_backward<float>(p, dh, dh_row, dx, dw, db, t, s);
  if (dtype == GSR_F16) return gated_backward<__half>(p, dh, dh_row, dx, dw, db, t, s);
  return gated_backward<__hip_bfloat16>(p, dh, dh_row, dx, dw, db, t, s);
}
