// gsr_clip.hip -- the global norm of many gradient tensors and clipping by it (include/gsr_optim.h).
//
//   norm  = (sum |g|^p)^(1/p) over every element of every tensor, p = 1, 2 or infinity
//   scale = min(1, max_norm / (norm + 1e-6)),   g <- g * scale
// Both passes stream: the norm reads each gradient once, the scaling reads and writes it once.
// A workgroup takes every G-th chunk of the tensors laid end to end and leaves one partial sum in
// 64 bits, where no square of a float overflows or vanishes and a sum of 10^8 of them keeps more
// digits than the result has (64-bit adds are far from the bound: two per 4 bytes read).  Whoever
// needs the norm adds the at most kGrid partial sums of each launch in their order: no atomics, so
// the same gradients give the same bits.
//
// HBM bounds both: of 62M floats (248 MB) the norm takes 41 us (6.0 TB/s), a call that scales 114
// (read, then read and write: 744 MB, 6.5 TB/s, some of them from the last-level cache), one that
// finds nothing to scale 42.  60 small tensors: the host's call.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/gsr_linear.h"
#include "../../include/gsr_optim.h"

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;  // elements: two batches of a lane in 32 bits, one in 16
constexpr int kGrid = 2048;   // workgroups (and partial sums) of a launch: 8 per CU
constexpr int kTensors = GSR_CLIP_LAUNCH_TENSORS;

struct Tensors {
  int n;
  void* g[kTensors];
  int64_t numel[kTensors];
  uint32_t chunk0[kTensors + 1];  // first chunk of each tensor
  uint8_t dtype[kTensors];
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__hip_bfloat16>(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half(v); }
template <> __device__ __forceinline__ __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

// 16 bytes of elements at any element's address (a gradient may start anywhere).
template <typename T> struct __attribute__((packed, aligned(2))) Vec {
  T e[16 / sizeof(T)];
};
constexpr int kBatch = 4;  // vectors of a lane in flight

template <int NORM>
__device__ __forceinline__ double join(double a, double b) {
  if (NORM != GSR_NORM_INF) return a + b;
  return b > a || b != b ? b : a;  // NaN wins
}
template <int NORM>
__device__ __forceinline__ double term(float g) {
  const double d = g;
  return NORM == GSR_NORM_2 ? d * d : fabs(d);
}

template <int NORM>
__device__ double block_join(double v) {
  __shared__ double part[kThreads / 64];
  for (int o = 32; o; o >>= 1) v = join<NORM>(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
  for (int w = 1; w < kThreads / 64; w++) v = join<NORM>(v, part[w]);
  return v;
}

template <typename T, int NORM>
__device__ __forceinline__ double chunk_sum(const T* g, int n) {
  constexpr int V = 16 / sizeof(T), kStep = kBatch * kThreads * V;
  double v = 0.0;
  int i = 0;
  for (; i + kStep <= n; i += kStep) {
    Vec<T> w[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; u++) w[u] = *(const Vec<T>*)(g + i + (u * kThreads + threadIdx.x) * V);
#pragma unroll
    for (int u = 0; u < kBatch; u++)
#pragma unroll
      for (int e = 0; e < V; e++) v = join<NORM>(v, term<NORM>(to_f(w[u].e[e])));
  }
  for (i += threadIdx.x * V; i < n; i += kThreads * V) {
    if (i + V <= n) {
      const Vec<T> w = *(const Vec<T>*)(g + i);
#pragma unroll
      for (int e = 0; e < V; e++) v = join<NORM>(v, term<NORM>(to_f(w.e[e])));
    } else {
      for (int e = i; e < n; e++) v = join<NORM>(v, term<NORM>(to_f(g[e])));
    }
  }
  return v;
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void norm_kernel(Tensors a, double* part) {
  double v = 0.0;
  int t = 0;
  for (uint32_t c = blockIdx.x; c < a.chunk0[a.n]; c += gridDim.x) {
    while (c >= a.chunk0[t + 1]) t++;
    const int64_t at = (int64_t)(c - a.chunk0[t]) * kChunk;
    const int n = a.numel[t] - at < kChunk ? (int)(a.numel[t] - at) : kChunk;
    if (a.dtype[t] == GSR_F32) v = join<NORM>(v, chunk_sum<float, NORM>((const float*)a.g[t] + at, n));
    else if (a.dtype[t] == GSR_F16) v = join<NORM>(v, chunk_sum<__half, NORM>((const __half*)a.g[t] + at, n));
    else v = join<NORM>(v, chunk_sum<__hip_bfloat16, NORM>((const __hip_bfloat16*)a.g[t] + at, n));
  }
  v = block_join<NORM>(v);
  if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <int NORM>
__device__ float norm_of(const double* part, int n) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) v = join<NORM>(v, part[i]);
  v = block_join<NORM>(v);
  return (float)(NORM == GSR_NORM_2 ? sqrt(v) : v);
}

__device__ __forceinline__ float scale_of(float norm, float max_norm) {
  const float c = max_norm / (norm + 1e-6f);
  return c > 1.0f ? 1.0f : c;  // NaN stays NaN
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void finish_kernel(const double* part, int n, float max_norm,
                                                          float* norm, float* scale) {
  const float v = norm_of<NORM>(part, n);
  if (threadIdx.x == 0) {
    *norm = v;
    if (scale) *scale = scale_of(v, max_norm);
  }
}

template <typename T>
__device__ __forceinline__ void chunk_scale(T* g, int n, float c) {
  constexpr int V = 16 / sizeof(T), kStep = kBatch * kThreads * V;
  int i = 0;
  for (; i + kStep <= n; i += kStep) {
    Vec<T> w[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; u++) w[u] = *(const Vec<T>*)(g + i + (u * kThreads + threadIdx.x) * V);
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
#pragma unroll
      for (int e = 0; e < V; e++) w[u].e[e] = from_f<T>(to_f(w[u].e[e]) * c);
      *(Vec<T>*)(g + i + (u * kThreads + threadIdx.x) * V) = w[u];
    }
  }
  for (i += threadIdx.x * V; i < n; i += kThreads * V)
    for (int e = i; e < n && e < i + V; e++) g[e] = from_f<T>(to_f(g[e]) * c);
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void scale_kernel(Tensors a, const double* part, int n_part,
                                                         float max_norm, float* norm) {
  const float v = norm_of<NORM>(part, n_part);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  const float s = scale_of(v, max_norm);
  if (s == 1.0f) return;  // a product with 1 changes nothing
  int t = 0;
  for (uint32_t c = blockIdx.x; c < a.chunk0[a.n]; c += gridDim.x) {
    while (c >= a.chunk0[t + 1]) t++;
    const int64_t at = (int64_t)(c - a.chunk0[t]) * kChunk;
    const int n = a.numel[t] - at < kChunk ? (int)(a.numel[t] - at) : kChunk;
    if (a.dtype[t] == GSR_F32) chunk_scale((float*)a.g[t] + at, n, s);
    else if (a.dtype[t] == GSR_F16) chunk_scale((__half*)a.g[t] + at, n, s);
    else chunk_scale((__hip_bfloat16*)a.g[t] + at, n, s);
  }
}

// The tensors [first, first + n) of the call as one launch's arguments; false if one is invalid.
bool fill(Tensors& a, int first, int n, void* const* grads, const int64_t* numel, const int* dtype) {
  a.n = n;
  uint64_t chunks = 0;
  for (int t = 0; t < n; t++) {
    const int k = first + t;
    if (numel[k] < 0 || (numel[k] > 0 && !grads[k]) || dtype[k] < GSR_F32 || dtype[k] > GSR_BF16)
      return false;
    a.g[t] = grads[k];
    a.numel[t] = numel[k];
    a.dtype[t] = (uint8_t)dtype[k];
    a.chunk0[t] = (uint32_t)chunks;
    chunks += (uint64_t)((numel[k] + kChunk - 1) / kChunk);
    if (chunks > 0x7fffffffu) return false;
  }
  a.chunk0[n] = (uint32_t)chunks;
  return true;
}

uint32_t grid_of(const Tensors& a) {
  const uint32_t c = a.chunk0[a.n];
  return c < 1 ? 1 : c < kGrid ? c : kGrid;
}

// Partial sums of every tensor; *n_part receives how many there are.
template <int NORM>
int norm_parts(int n_tensors, void* const* grads, const int64_t* numel, const int* dtype,
               double* part, int* n_part, hipStream_t s) {
  int at = 0;
  for (int first = 0; first < n_tensors; first += kTensors) {
    Tensors a;
    if (!fill(a, first, n_tensors - first < kTensors ? n_tensors - first : kTensors, grads, numel, dtype))
      return 1;
    const uint32_t g = grid_of(a);
    hipLaunchKernelGGL(norm_kernel<NORM>, dim3(g), dim3(kThreads), 0, s, a, part + at);
    at += (int)g;
  }
  *n_part = at;
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

template <int NORM>
int norm_call(int n_tensors, void* const* grads, const int64_t* numel, const int* dtype,
              float max_norm, float* norm, float* scale, double* part, hipStream_t s) {
  int n = 0;
  if (int rc = norm_parts<NORM>(n_tensors, grads, numel, dtype, part, &n, s)) return rc;
  hipLaunchKernelGGL(finish_kernel<NORM>, dim3(1), dim3(kThreads), 0, s, part, n, max_norm, norm, scale);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

template <int NORM>
int clip_call(int n_tensors, void* const* grads, const int64_t* numel, const int* dtype,
              float max_norm, float* norm, double* part, hipStream_t s) {
  int n = 0;
  if (int rc = norm_parts<NORM>(n_tensors, grads, numel, dtype, part, &n, s)) return rc;
  for (int first = 0; first < n_tensors; first += kTensors) {
    Tensors a;
    fill(a, first, n_tensors - first < kTensors ? n_tensors - first : kTensors, grads, numel, dtype);
    hipLaunchKernelGGL(scale_kernel<NORM>, dim3(grid_of(a)), dim3(kThreads), 0, s, a, part, n, max_norm, norm);
  }
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

}  // namespace

extern "C" size_t gsr_grad_norm_scratch_bytes(int n_tensors) {
  return n_tensors < 1 ? 256 : (size_t)((n_tensors + kTensors - 1) / kTensors) * kGrid * sizeof(double);
}

extern "C" int gsr_grad_norm(int n_tensors, const void* const* grads, const int64_t* numel,
                             const int* dtype, int norm_type, float max_norm, float* norm,
                             float* scale, void* scratch, void* stream) {
  if (n_tensors < 1 || !grads || !numel || !dtype || !norm || !scratch) return 1;
  if (scale && !(max_norm >= 0.0f)) return 1;  // a negative factor would turn the gradients round
  void* const* g = const_cast<void* const*>(grads);
  hipStream_t s = (hipStream_t)stream;
  double* part = (double*)scratch;
  if (norm_type == GSR_NORM_1) return norm_call<GSR_NORM_1>(n_tensors, g, numel, dtype, max_norm, norm, scale, part, s);
  if (norm_type == GSR_NORM_2) return norm_call<GSR_NORM_2>(n_tensors, g, numel, dtype, max_norm, norm, scale, part, s);
  if (norm_type == GSR_NORM_INF) return norm_call<GSR_NORM_INF>(n_tensors, g, numel, dtype, max_norm, norm, scale, part, s);
  return 1;
}

extern "C" int gsr_clip_grads(int n_tensors, void* const* grads, const int64_t* numel,
                              const int* dtype, int norm_type, float max_norm, float* norm,
                              void* scratch, void* stream) {
  if (n_tensors < 1 || !grads || !numel || !dtype || !norm || !scratch || !(max_norm >= 0.0f)) return 1;
  hipStream_t s = (hipStream_t)stream;
  double* part = (double*)scratch;
  if (norm_type == GSR_NORM_1) return clip_call<GSR_NORM_1>(n_tensors, grads, numel, dtype, max_norm, norm, part, s);
  if (norm_type == GSR_NORM_2) return clip_call<GSR_NORM_2>(n_tensors, grads, numel, dtype, max_norm, norm, part, s);
  if (norm_type == GSR_NORM_INF) return clip_call<GSR_NORM_INF>(n_tensors, grads, numel, dtype, max_norm, norm, part, s);
  return 1;
}
