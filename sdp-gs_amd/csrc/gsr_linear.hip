// gsr_linear.hip -- fused linear layer and gated pair, forward and backward (include/gsr_linear.h).
#include "gsr_product.h"

namespace {

using namespace gsr;

// out[e] = sum over s of part[s][e] in a fixed order: of `splits` weight gradients, and behind them of
// `sum_splits` bias gradients.  64 outputs to a workgroup, the splits shared by its four waves (a wave
// of few outputs alone would wait for one split after the other: 33 us for 128 splits of 203 x 161,
// against 7).  With `all` rows each blockIdx.y sums `splits` of them, dw[y][e].
template <typename T>
__global__ __launch_bounds__(256) void reduce_kernel(const float* part, const float* part_sum,
                                                     int splits, int sum_splits, int64_t n,
                                                     int64_t n_sum, int64_t all, T* dw, T* db) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t e = (int64_t)blockIdx.x * 64 + lane;
  const bool first = e < n, in = first || e - n < n_sum;
  const float* src = first ? part + e : part_sum + (in ? e - n : 0);
  const int64_t step = first ? n : n_sum;
  if (!first) splits = sum_splits;
  if (all) {
    const int64_t row = (int64_t)blockIdx.y * splits;
    src += row * step;
    dw += (int64_t)blockIdx.y * n;
    splits = all - row < splits ? (int)(all - row) : splits;
  }
  const int each = (splits + 3) / 4, begin = wave * each;
  const int end = begin + each < splits ? begin + each : splits;
  float v = 0.0f;
  if (in) {
    int s = begin;
    for (; s + 8 <= end; s += 8) {
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; k++) w[k] = src[(s + k) * step];
#pragma unroll
      for (int k = 0; k < 8; k++) v += w[k];
    }
    for (; s < end; s++) v += src[s * step];
  }
  sums[wave][lane] = v;
  __syncthreads();
  if (wave || !in) return;
  v = sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane];
  if (first) dw[e] = from_f<T>(v);
  else db[e - n] = from_f<T>(v);
}

template <typename T>
__global__ __launch_bounds__(256) void zero_kernel(T* p, int64_t n) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256)
    p[e] = from_f<T>(0.0f);
}
template <typename T>
void zero(void* p, int64_t n, hipStream_t stream) {
  const int64_t groups = (n + 255) / 256;
  hipLaunchKernelGGL(zero_kernel<T>, dim3((uint32_t)(groups < 65536 ? groups : 65536)), dim3(256), 0, stream, (T*)p, n);
}

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Ranges of the summed rows for dw: enough tiles to fill the 256 CUs, twice with 128 x 128 tiles,
// once with 256 x 256, each with at least 256 rows and a whole number of the kernel's steps.
struct Ranges {
  int64_t rows, count;
};
Ranges ranges_of(int64_t I, int64_t J, int64_t R, bool huge) {
  const int64_t side = huge ? 256 : 128, want = huge ? 256 : 512;
  const int64_t t = (I + side - 1) / side * ((J + side - 1) / side), n = (want + t - 1) / t;
  int64_t rows = up((R + n - 1) / n, 64);  // one workgroup more than there is room for doubles the time
  if (rows < 256) rows = 256;
  return {rows, (R + rows - 1) / rows};
}

bool sizes_ok(int dtype, int64_t M, int64_t K, int64_t N, int act) {
  return dtype >= GSR_F32 && dtype <= GSR_BF16 && act >= GSR_ACT_NONE && act <= GSR_ACT_SILU &&
         M >= 0 && K >= 1 && N >= 1 && K <= (1 << 22) && N <= (1 << 21) && M <= (1LL << 36);
}

bool x_ok(int64_t M, int64_t K, int64_t x_row, int64_t x_col) {
  return (x_col == 1 && (x_row >= K || M <= 1)) || (x_row == 1 && (x_col >= M || K == 1));
}

// The bias gradient's partial sums that a 16-bit dz kernel makes: `rows` of them of `width` at most (a
// wave has 16 rows or more, a workgroup up to 256; four rows where the product is cut, which more than
// 8192 are not).  kSumGroup at a time are summed first, if there
// are more, while the scratch they lie in is still theirs.
constexpr int kSumGroup = 128;
struct ColumnSums {
  int64_t width, rows;
  ColumnSums(int64_t M, int64_t width) : width(width), rows(up(M, 256) / (M <= 8192 ? 4 : 16)) {}
  bool grouped() const { return rows > kSumGroup; }
  int64_t kept_bytes() const { return up((grouped() ? (rows + kSumGroup - 1) / kSumGroup : rows) * width * 4, 256); }
  int64_t bytes() const { return grouped() ? up(rows * width * 4, 256) : 0; }
};

// The gradients before the activation, to `dz`, and if they are 16-bit their sums over the rows, to
// what is returned in `sums`; `scratch` moves on behind what is kept.
// 16-bit gradients are rounded once more here, the results of dx and dw have an error of 2.35e-3 in
// bfloat16 where the one rounding of a result gives 1.66e-3: the matrix instruction takes operands of
// one type, so more bits would be a second operand of remainders, written, read twice and multiplied.
// That is what a pair's backward does with its second half: 2011 us for 762048x256x512 where a
// layer's takes 1163.
template <typename T>
int activation_gradients(ProductArgs p, bool gated, bool need_db, char*& scratch, const float** sums,
                         int64_t* sum_rows, hipStream_t stream) {
  const int64_t width = gated ? 2 * p.J : p.J;
  p.out = scratch; p.out_row = width;
  scratch += up(p.I * width * sizeof(T), 256);
  *sums = nullptr;
  if (sizeof(T) == 4 || !need_db) return product_dz<T>(p, gated, scratch, stream);
  const ColumnSums c(p.I, width);
  float* kept = (float*)scratch;
  scratch += c.kept_bytes();
  p.part_sum = c.grouped() ? (float*)scratch : kept;
  p.sum_rows = sum_rows;
  *sums = kept;
  if (int rc = product_dz<T>(p, gated, scratch + c.bytes(), stream)) return rc;
  if (!c.grouped()) return 0;
  const int64_t all = *sum_rows;
  *sum_rows = (all + kSumGroup - 1) / kSumGroup;
  for (int64_t at = 0; at < *sum_rows; at += 65535) {  // groups are the grid's y
    const int64_t n = *sum_rows - at < 65535 ? *sum_rows - at : 65535, row = at * kSumGroup;
    hipLaunchKernelGGL(reduce_kernel<float>, dim3((uint32_t)((width + 63) / 64), (uint32_t)n), dim3(256), 0, stream,
                       p.part_sum + row * width, nullptr, kSumGroup, 0, width, 0, all - row, kept + at * width,
                       nullptr);
  }
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

// A bias gradient that is summed beside the weight gradients comes, where these are not asked for,
// with those of a few of x's columns: the same ranges, the same bits, without the product's work.
int64_t columns_of(int64_t K, bool dw) { return dw || K < 8 ? K : 8; }

// The weight gradients: partial products over ranges of x's rows, then their sum.  The bias gradient
// is dz's sum beside them, or that of `sum_rows` rows of `sums`.
template <typename T>
int weight_gradients(const void* dz, int64_t dz_row, int64_t M, int64_t K, int64_t I, const void* x,
                     int64_t x_row, int64_t x_col, void* dw, void* db, const float* sums, int64_t sum_rows,
                     char* scratch, hipStream_t stream) {
  if (M == 0) {
    if (dw) zero<T>(dw, I * K, stream);
    if (db) zero<T>(db, I, stream);
    return hipGetLastError() == hipSuccess ? 0 : 2;
  }
  ProductArgs p{};
  if (dw || !sums) {
    p.a = dz; p.a_i = 1; p.a_r = dz_row;
    p.b[0] = x; p.b_j = x_col; p.b_r = x_row;
    p.I = I; p.J = K; p.R = M; p.segments = 1;
    const Ranges ranges = ranges_of(I, K, M, product_dw_huge<T>(p));
    p.J = columns_of(K, dw);
    p.r_chunk = ranges.rows;
    p.part = (float*)scratch;
    const bool direct = dw && ranges.count == 1;  // nothing to add: written as they are
    p.part_sum = !db || sums ? nullptr : direct ? p.part : p.part + ranges.count * I * p.J;
    if (direct) {
      p.out = dw; p.out_row = K;
    }
    if (int rc = product_dw<T>(p, ranges.count, stream)) return rc;
    if (direct && !db) return 0;
    if (!sums) sums = p.part_sum, sum_rows = ranges.count;
    const int64_t n = dw && !direct ? I * K : 0, n_sum = db ? I : 0;
    hipLaunchKernelGGL(reduce_kernel<T>, dim3((uint32_t)((n + n_sum + 63) / 64)), dim3(256), 0, stream, p.part, sums,
                       (int)ranges.count, (int)sum_rows, n, n_sum, 0, (T*)dw, (T*)db);
  } else {
    hipLaunchKernelGGL(reduce_kernel<T>, dim3((uint32_t)((I + 63) / 64)), dim3(256), 0, stream, nullptr, sums, 0,
                       (int)sum_rows, 0, I, 0, nullptr, (T*)db);
  }
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

// What weight_gradients takes; dw: they are asked for, not the bias gradient alone.
size_t partial_bytes(int64_t M, int64_t K, int64_t I, bool dw) {
  if (M == 0) return 0;
  auto of = [&](bool huge) {
    const int64_t n = ranges_of(I, K, M, huge).count;
    return n * (columns_of(K, dw && n > 1) + 1);  // one range is written where it belongs
  };
  const int64_t small = of(false), huge = takes_huge_dw(I, K) ? of(true) : 0;
  return (size_t)(small > huge ? small : huge) * I * 4;
}

// Scratch of a backward, in order: the gradients before the activation, their sums, then what one
// product at a time needs (the weights' images, the partial sums).
template <typename T>
size_t backward_bytes(int64_t M, int64_t K, int64_t N, bool gated, bool has_dz, int need_dw) {
  const int64_t width = gated ? 2 * N : N;
  const bool column_sums = has_dz && need_dw && sizeof(T) == 2;
  const ColumnSums c(M, width);
  size_t most = has_dz ? dz_scratch<T>(M, K, N, gated) : 0;
  if (column_sums) most += c.bytes();
  const size_t dx = dx_scratch<T>(M, K, N, gated ? 2 : 1);
  most = dx > most ? dx : most;
  const size_t dw = need_dw ? partial_bytes(M, K, width, need_dw != GSR_NEED_DB) : 0;
  most = dw > most ? dw : most;
  return (has_dz ? (size_t)up(M * width * sizeof(T), 256) : 0) + (column_sums ? c.kept_bytes() : 0) + most;
}

template <typename T>
int linear_backward(const ProductArgs& fwd, const void* dy, int64_t dy_row, void* dx, void* dw,
                    void* db, char* scratch, hipStream_t stream) {
  const int64_t M = fwd.I, K = fwd.R, N = fwd.J;
  const void* dz = dy;
  int64_t dz_row = dy_row, sum_rows = 0;
  const float* sums = nullptr;
  if (fwd.act != GSR_ACT_NONE && M > 0) {
    ProductArgs p = fwd;
    p.extra = dy; p.extra_row = dy_row;
    dz = scratch; dz_row = N;
    if (int rc = activation_gradients<T>(p, false, db, scratch, &sums, &sum_rows, stream)) return rc;
  }
  if (dx && M > 0) {
    ProductArgs p{};
    p.a = dz; p.a_i = dz_row; p.a_r = 1;
    p.b[0] = fwd.b[0]; p.b_j = 1; p.b_r = fwd.b_j;
    p.I = M; p.J = K; p.R = N; p.segments = 1;
    p.out = dx; p.out_row = K;
    if (int rc = product_dx<T>(p, scratch, stream)) return rc;
  }
  if (!dw && !db) return 0;
  return weight_gradients<T>(dz, dz_row, M, K, N, fwd.a, fwd.a_i, fwd.a_r, dw, db, sums, sum_rows, scratch, stream);
}

template <typename T>
int gated_backward(const ProductArgs& fwd, const void* dh, int64_t dh_row, void* dx, void* dw,
                   void* db, char* scratch, hipStream_t stream) {
  const int64_t M = fwd.I, K = fwd.R, N = fwd.J;
  const void* dz = scratch;
  int64_t sum_rows = 0;
  const float* sums = nullptr;
  if (M > 0) {
    ProductArgs p = fwd;
    p.extra = dh; p.extra_row = dh_row;
    if (int rc = activation_gradients<T>(p, true, db, scratch, &sums, &sum_rows, stream)) return rc;
    if (dx) {
      ProductArgs q{};
      q.a = dz; q.a_i = 2 * N; q.a_r = 1;
      q.b[0] = fwd.b[0]; q.b[1] = fwd.b[1]; q.b_j = 1; q.b_r = fwd.b_j;
      q.I = M; q.J = K; q.R = N; q.segments = 2; q.a_segment = N;
      q.out = dx; q.out_row = K;
      if (int rc = product_dx<T>(q, scratch, stream)) return rc;
    }
  }
  if (!dw && !db) return 0;
  return weight_gradients<T>(dz, 2 * N, M, K, 2 * N, fwd.a, fwd.a_i, 1, dw, db, sums, sum_rows, scratch, stream);
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

// f(a null pointer of the call's type)
template <typename F>
auto with_type(int dtype, F f) {
  if (dtype == GSR_F32) return f((float*)nullptr);
  if (dtype == GSR_F16) return f((__half*)nullptr);
  return f((__hip_bfloat16*)nullptr);
}
template <typename P> struct Pointee;
template <typename T> struct Pointee<T*> { using type = T; };

int forward(int dtype, const ProductArgs& p, bool gated, void* scratch, void* stream) {
  return with_type(dtype, [&](auto t) {
    return product_forward<typename Pointee<decltype(t)>::type>(p, gated, (char*)scratch, (hipStream_t)stream);
  });
}

size_t forward_bytes(int dtype, int64_t M, int64_t K, int64_t N, bool gated) {
  return with_type(dtype, [&](auto t) {
    return forward_scratch<typename Pointee<decltype(t)>::type>(M, K, N, gated);
  });
}

}  // namespace

extern "C" size_t gsr_linear_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N) {
  return sizes_ok(dtype, M, K, N, GSR_ACT_NONE) ? forward_bytes(dtype, M, K, N, false) : 0;
}

extern "C" int gsr_linear(int dtype, int64_t M, int64_t K, int64_t N, const void* x, int64_t x_row,
                          int64_t x_col, const void* w, int64_t w_row, const void* bias,
                          const void* residual, int64_t residual_row, int act, void* y,
                          int64_t y_row, void* scratch, void* stream) {
  if (!sizes_ok(dtype, M, K, N, act) || !x_ok(M, K, x_row, x_col) || w_row < K) return 1;
  if (M == 0) return 0;
  if (!x || !w || !y || y_row < N || (residual && residual_row < N && M > 1)) return 1;
  if (!scratch && forward_bytes(dtype, M, K, N, false)) return 1;
  ProductArgs p = forward_args(M, K, N, x, x_row, x_col, w, nullptr, w_row, bias, nullptr, act);
  p.extra = residual; p.extra_row = residual_row;
  p.out = y; p.out_row = y_row;
  return forward(dtype, p, false, scratch, stream);
}

extern "C" size_t gsr_linear_backward_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N,
                                                    int act, int need_dw) {
  if (!sizes_ok(dtype, M, K, N, act)) return 0;
  return with_type(dtype, [&](auto t) {
    return backward_bytes<typename Pointee<decltype(t)>::type>(M, K, N, false, act != GSR_ACT_NONE, need_dw);
  }) + 256;
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
  return with_type(dtype, [&](auto k) {
    return linear_backward<typename Pointee<decltype(k)>::type>(p, dy, dy_row, dx, dw, dbias, t, s);
  });
}

extern "C" size_t gsr_gated_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N) {
  return sizes_ok(dtype, M, K, N, GSR_ACT_NONE) ? forward_bytes(dtype, M, K, N, true) : 0;
}

extern "C" int gsr_gated(int dtype, int64_t M, int64_t K, int64_t N, const void* x, int64_t x_row,
                         const void* wg, const void* wu, int64_t w_row, const void* bg,
                         const void* bu, int act, void* h, int64_t h_row, void* scratch, void* stream) {
  if (!sizes_ok(dtype, M, K, N, act) || !x_ok(M, K, x_row, 1) || w_row < K) return 1;
  if (M == 0) return 0;
  if (!x || !wg || !wu || !h || h_row < N) return 1;
  if (!scratch && forward_bytes(dtype, M, K, N, true)) return 1;
  ProductArgs p = forward_args(M, K, N, x, x_row, 1, wg, wu, w_row, bg, bu, act);
  p.out = h; p.out_row = h_row;
  return forward(dtype, p, true, scratch, stream);
}

extern "C" size_t gsr_gated_backward_scratch_bytes(int dtype, int64_t M, int64_t K, int64_t N,
                                                   int need_dw) {
  if (!sizes_ok(dtype, M, K, N, GSR_ACT_NONE)) return 0;
  return with_type(dtype, [&](auto t) {
    return backward_bytes<typename Pointee<decltype(t)>::type>(M, K, N, true, true, need_dw);
  }) + 256;
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
  return with_type(dtype, [&](auto k) {
    return gated_backward<typename Pointee<decltype(k)>::type>(p, dh, dh_row, dx, dw, db, t, s);
  });
}
