// gsr_product.h -- the tiled matrix-core product behind gsr_linear*.hip.
//
//   C(i, j) = sum_r A(i, r) B(j, r), one BI x BJ tile of C per workgroup, epilogues in gsr_linear.h.
//
// Matrix instruction: v_mfma_f32_16x16x32 on 16-bit operands, the rows of B (outputs j) as the
// instruction's rows and the rows of A (i) as its columns, so that a lane's four results are four
// consecutive j of one i and leave as 16-byte stores.
//
// 32-bit operands: a float is the exact sum of three bfloat16 parts (8 + 8 + 8 bits, each the
// rounded remainder of the one before) from 2^-110 on; below that the last parts pass the type's
// smallest step, 2^-133, and the float is held to half of it.  Six of the nine products of parts are formed, those of
// 2^-16 or more; the three left out are below 2^-24 of the product together, a float product's own
// rounding.  At 6/16 the rate of the 16-bit instruction that is 2.6x the float instruction's rate.
// Parts of an infinity or a NaN do not sum to it, so a result that is not finite is computed again
// from the operands in plain 32-bit arithmetic (exact_sum).
//
// LDS holds the operands' 16-bit planes.  An operand that is contiguous along r is kept as rows of
// r and read 16 bytes (8 r) at a time; one that is contiguous along its rows is kept as it lies and
// read through ds_read_b64_tr, which hands each lane 4 r of its own row.  16-byte chunks are
// permuted within a row (swizzle) so that the 16 lanes of a read hit 16 different bank groups.
#pragma once
#include "gsr_linear.h"

namespace gsr {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any address: operands may start anywhere (a slice, an odd row length)
struct __attribute__((packed, aligned(1))) Bytes16 { u32x4 v; };

template <int V> struct Const { static constexpr int value = V; };

template <typename T> struct Operand {
  static constexpr int kPlanes = 1, kDepth = 64, kBuffers = 2, kRaw = 1;  // kRaw: 16-byte words per 8 elements
};
template <> struct Operand<float> {
  static constexpr int kPlanes = 3, kDepth = 32, kBuffers = 1, kRaw = 2;
};

template <typename T>
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma<__half>(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t round_pair(f32x2 v) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ f32x2 widen_pair(uint32_t v) {
  return f32x2{__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)};
}

// 8 consecutive elements as they come from memory.
template <typename T> struct Chunk {
  u32x4 w[Operand<T>::kRaw];
};

template <typename T>
__device__ __forceinline__ Chunk<T> load_whole(const T* p) {
  Chunk<T> c;
#pragma unroll
  for (int k = 0; k < Operand<T>::kRaw; k++) c.w[k] = ((const Bytes16*)p)[k].v;
  return c;
}

// Elements k..k+7 of a row of n (n >= 1) that are `step` apart; those past its end are zero.  Every
// load is made, from the last element where there is none: no branch, so all are in flight at once.
template <typename T>
__device__ __forceinline__ Chunk<T> load_tail(const T* row, int64_t k, int64_t step, int64_t n) {
  Chunk<T> c;
#pragma unroll
  for (int e = 0; e < Operand<T>::kRaw; e++) c.w[e] = u32x4{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int64_t at = (k + e < n ? k + e : n - 1) * step;
    if constexpr (sizeof(T) == 4) {
      const uint32_t v = ((const uint32_t*)row)[at];
      c.w[e >> 2][e & 3] = k + e < n ? v : 0u;
    } else {
      const uint32_t v = ((const uint16_t*)row)[at];
      c.w[0][e >> 1] |= (k + e < n ? v : 0u) << (16 * (e & 1));
    }
  }
  return c;
}
// The same from whole words: up to 7 elements past the row's end are read, which has to be memory
// of the tensor (there are rows after it).
template <typename T>
__device__ __forceinline__ Chunk<T> load_masked(const T* row, int64_t k, int64_t n) {
  Chunk<T> c = load_whole(row + (k < n ? k : 0));
  const int64_t left = n - k;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; e++) c.w[e >> 2][e & 3] = e < left ? c.w[e >> 2][e & 3] : 0u;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) c.w[0][e] &= 2 * e + 1 < left ? ~0u : 2 * e < left ? 0xffffu : 0u;
  }
  return c;
}
constexpr int kSpareRows = 8;  // with so many rows after it, a row may be read 7 elements too far

// N words moved down by `off` elements (0..7), zeros from above.
template <typename T, int N>
__device__ __forceinline__ void shift_down(uint32_t (&w)[N], int off) {
  const int words = sizeof(T) == 4 ? off : off >> 1;
#pragma unroll
  for (int bit = 4; bit; bit >>= 1) {
    if (bit >= N) continue;
#pragma unroll
    for (int e = 0; e < N; e++) w[e] = words & bit ? (e + bit < N ? w[e + bit] : 0u) : w[e];
  }
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int e = 0; e < N; e++) {
      const uint32_t next = e + 1 < N ? w[e + 1] : 0u;
      w[e] = off & 1 ? w[e] >> 16 | next << 16 : w[e];
    }
  }
}
// Elements k..k+7 of a row of n; those past its end are zero.  One read of whole words and no
// branch: at the end of the tensor (`end`: past its last element, at least 8 after its first) an
// earlier place is read and moved down.
template <typename T>
__device__ __forceinline__ Chunk<T> load_row_end(const T* row, int64_t k, int64_t n, const T* end) {
  constexpr int N = 4 * Operand<T>::kRaw;
  const T* p = row + (k < n ? k : 0);
  const int off = p + 8 > end ? (int)(p + 8 - end) : 0;
  const Chunk<T> c = load_whole(p - off);
  uint32_t w[N];
#pragma unroll
  for (int e = 0; e < N; e++) w[e] = c.w[e >> 2][e & 3];
  shift_down<T, N>(w, off);
  const int64_t left = n - k;
  Chunk<T> r;
#pragma unroll
  for (int e = 0; e < N; e++) {
    if constexpr (sizeof(T) == 4) r.w[e >> 2][e & 3] = e < left ? w[e] : 0u;
    else r.w[0][e] = w[e] & (2 * e + 1 < left ? ~0u : 2 * e < left ? 0xffffu : 0u);
  }
  return r;
}
// The same for the 16 bytes at element k, anything in the place of those past the row's end.
template <typename T>
__device__ __forceinline__ u32x4 load_words_end(const T* row, int64_t k, int64_t n, const T* end) {
  constexpr int RUN = 16 / sizeof(T);
  const T* p = row + (k < n ? k : 0);
  const int off = p + RUN > end ? (int)(p + RUN - end) : 0;
  const u32x4 c = ((const Bytes16*)(p - off))->v;
  uint32_t w[4] = {c[0], c[1], c[2], c[3]};
  shift_down<T, 4>(w, off);
  return u32x4{w[0], w[1], w[2], w[3]};
}

// Which parts are multiplied: smallest products first.
template <int PLANES> struct Parts {
  static constexpr int kProducts = 1, kA[1] = {0}, kB[1] = {0};
};
template <> struct Parts<3> {
  static constexpr int kProducts = 6, kA[6] = {2, 0, 1, 1, 0, 0}, kB[6] = {0, 2, 1, 0, 1, 0};
};

// Waits for this wave's LDS accesses, then for the other waves; global accesses stay in flight.
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The 8 elements as 16-bit parts.
template <typename T>
__device__ __forceinline__ void split_chunk(s16x8 (&part)[Operand<T>::kPlanes], const Chunk<T>& c) {
  if constexpr (Operand<T>::kPlanes == 1) {
    part[0] = __builtin_bit_cast(s16x8, c.w[0]);
  } else {
    u32x4 w[3];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      f32x2 v = {__uint_as_float(c.w[k >> 1][(k & 1) * 2]), __uint_as_float(c.w[k >> 1][(k & 1) * 2 + 1])};
#pragma unroll
      for (int p = 0; p < 3; p++) {
        w[p][k] = round_pair(v);
        v -= widen_pair(w[p][k]);
      }
    }
#pragma unroll
    for (int p = 0; p < 3; p++) part[p] = __builtin_bit_cast(s16x8, w[p]);
  }
}
template <typename T>
__device__ __forceinline__ void put_chunk(char* to, int plane_bytes, const Chunk<T>& c) {
  s16x8 part[Operand<T>::kPlanes];
  split_chunk<T>(part, c);
#pragma unroll
  for (int p = 0; p < Operand<T>::kPlanes; p++) *(s16x8*)(to + p * plane_bytes) = part[p];
}

// One operand's tile in LDS.  RC: contiguous along r (rows of kDepth), else rows of ROWS.
// PAIRED: the epilogue takes 8 consecutive rows j per lane, so the 16 rows of a read are
// 4 + 4 + 4 + 4 rows, 8 apart.
template <typename T, bool RC, int ROWS, int THREADS, bool PAIRED>
struct Tile {
  static constexpr int kDepth = Operand<T>::kDepth, kPlanes = Operand<T>::kPlanes;
  static constexpr int kPerRow = (RC ? kDepth : ROWS) / 8;   // chunks in a row of LDS
  static constexpr int kChunks = ROWS * kDepth / 8 / THREADS;  // chunks a thread stages
  static constexpr int kPlaneBytes = ROWS * kDepth * 2;
  static constexpr int kBytes = kPlaneBytes * kPlanes;
  static_assert(ROWS * kDepth % (8 * THREADS) == 0, "");

  // Which of a row's chunks is kept where: the rows that one read takes together differ in it.
  static __device__ __forceinline__ int swizzle(int row) {
    if (!RC) {  // rows are r: a read takes 4 of each 8
      if (ROWS == 64) return 2 * (((row >> 1) & 1) | (((row >> 3) & 1) << 1));
      return 2 * ((row & 3) | (((row >> 3) & 1) << 2));
    }
    if (kDepth == 32) return (row >> 2) & 3;
    return PAIRED ? ((row >> 1) & 1) | (((row >> 3) & 3) << 1) : (row >> 1) & 7;
  }

  // Rows [o0, o0 + ROWS) of O, r in [r0, r0 + kDepth) below r_end (zeros from there on) of R.  A row
  // past the last is some other row: its results are not stored.  base1: rows from SPLIT on.
  template <int SPLIT>
  static __device__ __forceinline__ void load(Chunk<T> (&c)[kChunks], const T* base, const T* base1, int64_t ld,
                                              int64_t o0, int64_t O, int64_t r0, int64_t r_end, int64_t R) {
    const bool deep = r0 + kDepth <= r_end;
    const bool spare = (RC ? o0 + (SPLIT ? SPLIT : ROWS) + kSpareRows <= O : r0 + kDepth + kSpareRows <= R);
    auto each = [&](auto kind) {
      constexpr int KIND = decltype(kind)::value;  // 0: all there, 1: whole words, 2: element by element
#pragma unroll
      for (int s = 0; s < kChunks; s++) {
        const int q = s * THREADS + threadIdx.x, row = q / kPerRow, col = q % kPerRow * 8;
        if (RC) {
          const bool second = SPLIT && row >= SPLIT;
          int64_t o = o0 + (second ? row - SPLIT : row);
          o = o < O ? o : O - 1;
          const T* p = (second ? base1 : base) + o * ld;
          if (KIND == 0) c[s] = load_whole(p + r0 + col);
          else if (KIND == 1) c[s] = load_masked(p, r0 + col, r_end);
          else c[s] = load_tail(p, r0 + col, 1, r_end);
        } else {
          if (KIND == 0) {
            c[s] = load_whole(base + (r0 + row) * ld + o0 + col);
          } else if (KIND == 1) {
            c[s] = load_whole(base + (r0 + row) * ld + (o0 + col < O ? o0 + col : o0));
          } else {
            const bool in = r0 + row < r_end;
            c[s] = load_tail(base + (in ? r0 + row : r_end - 1) * ld, o0 + col, 1, O);
#pragma unroll
            for (int k = 0; k < Operand<T>::kRaw; k++) c[s].w[k] = in ? c[s].w[k] : u32x4{0, 0, 0, 0};
          }
        }
      }
    };
    if (deep && (RC || o0 + ROWS <= O)) each(Const<0>());
    else if (spare && (RC || deep)) each(Const<1>());
    else each(Const<2>());
  }

  // Every row and base a multiple of 16 bytes and no chunk across an end (16-bit types): straight
  // into LDS, 1 KB per instruction, each lane fetching the chunk that belongs where it writes.  A
  // chunk past an end is another one instead; where it is past r_end, clear() follows.
  static __device__ __forceinline__ void direct(char* lds, const T* base, const T* base1, int split, int64_t ld,
                                                int64_t o0, int64_t O, int64_t r0, int64_t r_end) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto each = [&](auto whole) {
#pragma unroll
      for (int s = 0; s < kChunks; s++) {
        const int q = s * THREADS + threadIdx.x, row = q / kPerRow, col = (q % kPerRow ^ swizzle(row)) * 8;
        const T* p;
        if (RC) {
          const bool second = split && row >= split;
          int64_t o = o0 + (second ? row - split : row);
          o = o < O ? o : O - 1;
          p = (second ? base1 : base) + o * ld + (decltype(whole)::value || r0 + col < r_end ? r0 + col : 0);
        } else {
          // the lane's own part of the address does not change from step to step
          const int64_t c = o0 + col < O ? o0 + col : 0;
          if (decltype(whole)::value) p = base + r0 * ld + (row * ld + c);
          else p = base + (r0 + row < r_end ? r0 + row : r_end - 1) * ld + c;
        }
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                         (__attribute__((address_space(3))) void*)(lds + (s * THREADS + wave * 64) * 16),
                                         16, 0, 0);
      }
    };
    if (r0 + kDepth <= r_end) each(Const<1>());
    else each(Const<0>());
  }
  // Zeros for the chunks of a last step that are past r_end; each thread those that it fetched.
  static __device__ __forceinline__ void clear(char* lds, int64_t r0, int64_t r_end) {
#pragma unroll
    for (int s = 0; s < kChunks; s++) {
      const int q = s * THREADS + threadIdx.x, row = q / kPerRow, col = (q % kPerRow ^ swizzle(row)) * 8;
      if (r0 + (RC ? col : row) >= r_end) *(u32x4*)(lds + q * 16) = u32x4{0, 0, 0, 0};
    }
  }

  static __device__ __forceinline__ void store(char* lds, const Chunk<T> (&c)[kChunks]) {
#pragma unroll
    for (int s = 0; s < kChunks; s++) {
      const int q = s * THREADS + threadIdx.x, row = q / kPerRow, at = q % kPerRow ^ swizzle(row);
      put_chunk<T>(lds + (row * kPerRow + at) * 16, kPlaneBytes, c[s]);
    }
  }

  // The 16 rows of step t (of 16 rows each) and r in [32 kk, 32 kk + 32) as a matrix operand: lane
  // l holds row l % 16 and r = 8 (l / 16) + 0..7.
  static __device__ __forceinline__ s16x8 read(const char* lds, int t, int kk) {
    const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
    if (RC) {
      const int row = PAIRED ? 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3) : 16 * t + m;
      return *(const s16x8*)(lds + row * (kPerRow * 16) + (((kk * 4 + q) ^ swizzle(row)) * 16));
    }
    const int p = m & 3, r = kk * 32 + 8 * q + (m >> 2);
    const int col = PAIRED ? 32 * (t >> 1) + 8 * p + 4 * (t & 1) : 16 * t + 4 * p;
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds4*)(lds + r * (kPerRow * 16) + (((col >> 3) ^ swizzle(r)) * 16) + ((col >> 2) & 1) * 8));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds4*)(lds + (r + 4) * (kPerRow * 16) + (((col >> 3) ^ swizzle(r + 4)) * 16) + ((col >> 2) & 1) * 8));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// 16 bytes of a row, RUN elements, as floats and back; `n` of them exist.
template <typename T>
__device__ __forceinline__ u32x4 load_words(const T* p, int64_t n) {
  constexpr int RUN = 16 / sizeof(T);
  if (n >= RUN) return ((const Bytes16*)p)->v;
  u32x4 w = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < RUN - 1; k++) {
    if (k >= n) break;
    if constexpr (sizeof(T) == 4) w[k] = ((const uint32_t*)p)[k];
    else w[k >> 1] |= (uint32_t)((const uint16_t*)p)[k] << (16 * (k & 1));
  }
  return w;
}
template <typename T, int RUN>
__device__ __forceinline__ void widen(float (&v)[RUN], u32x4 w) {
#pragma unroll
  for (int k = 0; k < RUN; k++) {
    if constexpr (sizeof(T) == 4) v[k] = __uint_as_float(w[k]);
    else if constexpr (__is_same(T, __half)) v[k] = to_f(__builtin_bit_cast(__half, (uint16_t)(w[k >> 1] >> (16 * (k & 1)))));
    else v[k] = __uint_as_float(k & 1 ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16);
  }
}
template <typename T, int RUN>
__device__ __forceinline__ void load_run(float (&v)[RUN], const T* p, int64_t n) {
  widen<T, RUN>(v, load_words(p, n));
}
// Two floats rounded to nearest even, as one word.
template <typename T>
__device__ __forceinline__ uint32_t narrow_pair(float a, float b) {
  if constexpr (__is_same(T, __half)) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  } else {
    return round_pair(f32x2{a, b});
  }
}

// RUN results (16 bytes of them, or 8), n of which exist.
template <typename T, int RUN>
__device__ __forceinline__ void store_run(T* p, const float (&v)[RUN], int64_t n) {
  if (n >= RUN) {
    if constexpr (sizeof(T) * RUN == 8) {
      struct __attribute__((packed, aligned(1))) Bytes8 { uint32_t a, b; };
      *(Bytes8*)p = Bytes8{narrow_pair<T>(v[0], v[1]), narrow_pair<T>(v[2], v[3])};
      return;
    }
    u32x4 w;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < RUN; k++) w[k] = __float_as_uint(v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < RUN; k += 2) w[k >> 1] = narrow_pair<T>(v[k], v[k + 1]);
    }
    ((Bytes16*)p)->v = w;
    return;
  }
#pragma unroll
  for (int k = 0; k < RUN; k++)
    if (k < n) p[k] = from_f<T>(v[k]);
}

// The epilogue of RUN results v (and w, the up half) of row i at columns j..; n of them exist.
// EXTRA: with ex, the residual or the incoming gradient.
template <typename T, int EPI, bool GATED, bool EXTRA, int ACT, int RUN>
__device__ __forceinline__ void epilogue(const ProductArgs& p, int64_t i, int64_t j, int64_t n,
                                         float (&v)[RUN], float (&w)[RUN], const float (&ex)[RUN]) {
  T* out = (T*)p.out + i * p.out_row + j;
#pragma unroll
  for (int k = 0; k < RUN; k++) {
    if (EPI == EPI_FORWARD) {
      v[k] = act_value<ACT>(v[k]);
      if (GATED) v[k] *= w[k];
      if (EXTRA) v[k] += ex[k];
    } else if (EPI == EPI_DZ) {
      float a;
      const float s = act_both<ACT>(v[k], a);
      v[k] = GATED ? ex[k] * w[k] * s : ex[k] * s;
      if (GATED) w[k] = ex[k] * a;
    }
  }
  store_run<T, RUN>(out, v, n);
  if (EPI == EPI_DZ && GATED) store_run<T, RUN>(out + p.J, w, n);
}

// Whether a dz kernel also makes the bias gradient's partial sums: with 16-bit results, whose
// rounding would be in every sum of them (an error as large as that of the sum's own rounding).  A
// sum of 32-bit results loses nothing, it is made beside the weight gradients.
template <typename T, int EPI> constexpr bool kColumnSums = EPI == EPI_DZ && sizeof(T) == 2;

// v[k] summed over the 16 lanes of a DPP row, n of them stored by the first.
template <int RUN>
__device__ __forceinline__ void store_sums(float* p, int m, int64_t n, float (&v)[RUN]) {
  auto ror = [](auto by, float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + decltype(by)::value, 15, 15, false));
  };
#pragma unroll
  for (int k = 0; k < RUN; k++) {
    v[k] += ror(Const<8>(), v[k]);
    v[k] += ror(Const<4>(), v[k]);
    v[k] += ror(Const<2>(), v[k]);
    v[k] += ror(Const<1>(), v[k]);
  }
  if (m) return;
#pragma unroll
  for (int h = 0; h < RUN; h += 4) store_run<float, 4>(p + h, {v[h], v[h + 1], v[h + 2], v[h + 3]}, n - h);
}

// f(integral constant of the activation): one branch for a whole epilogue.
template <int EPI, typename F>
__device__ __forceinline__ void with_act(int act, F f) {
  if (EPI != EPI_FORWARD && EPI != EPI_DZ) return f(Const<GSR_ACT_NONE>());
  if (act == GSR_ACT_RELU) f(Const<GSR_ACT_RELU>());
  else if (act == GSR_ACT_GELU) f(Const<GSR_ACT_GELU>());
  else if (act == GSR_ACT_SILU) f(Const<GSR_ACT_SILU>());
  else f(Const<GSR_ACT_NONE>());
}

// One result in plain 32-bit arithmetic, r in [r0, r1) of each segment.
__device__ __noinline__ float exact_sum(const float* a, int64_t a_i, int64_t a_r, const float* b0,
                                        const float* b1, int64_t b_j, int64_t b_r, int segments,
                                        int64_t a_segment, int64_t i, int64_t j, int64_t r0, int64_t r1) {
  float v = 0.0f;
  for (int s = 0; s < segments; s++) {
    const float* A = a + s * a_segment + i * a_i;
    const float* B = (s ? b1 : b0) + j * b_j;
    for (int64_t r = r0; r < r1 && v == v; r++) v = fmaf(A[r * a_r], b0 ? B[r * b_r] : 1.0f, v);  // NaN stays
  }
  return v;
}

// The tiles of C, j fastest, then i, then the ranges of r: consecutive tiles share rows of A.
// Workgroups go to the 8 XCDs in turn, so XCD x takes the x-th eighth of them: tiles that share
// operands share an L2.
struct Place {
  int64_t i;  // tile
  uint32_t j, split;
  bool in;
};
__device__ __forceinline__ Place place(uint32_t tiles_i, uint32_t tiles_j, uint32_t splits) {
  const uint32_t total = tiles_i * tiles_j * splits, each = gridDim.x >> 3;
  const uint32_t t = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
  Place p;
  p.in = t < total;
  p.j = t % tiles_j;
  const uint32_t rest = t / tiles_j;
  p.i = rest % tiles_i;
  p.split = rest / tiles_i;
  return p;
}

// WI x WJ waves; a wave has BI / WI rows i and BJ / WJ rows j of the tile.  GATED: the tile's BJ
// rows are BJ / 2 of the gate's weights and the same BJ / 2 of the up weights.
template <typename T, bool RCA, bool RCB, int EPI, bool GATED, bool DIRECT, int BI, int WI, int BJ, int WJ>
__global__ __launch_bounds__(64 * WI * WJ, 2) void product_kernel(ProductArgs p, uint32_t tiles_i,
                                                               uint32_t tiles_j, uint32_t splits) {
  constexpr int NT = 64 * WI * WJ, kDepth = Operand<T>::kDepth, kPlanes = Operand<T>::kPlanes;
  constexpr int kBuffers = Operand<T>::kBuffers;
  constexpr int NI = BI / WI / 16, NJ = BJ / WJ / 16;  // 16x16 tiles of a wave
  constexpr bool kPaired = sizeof(T) == 2 && EPI != EPI_PARTIAL;
  constexpr int RUN = kPaired ? 8 : 4;
  constexpr int kOut = GATED ? BJ / 2 : BJ;  // outputs of the tile
  static_assert(!GATED || (WJ == 1 && RCB), "");
  using TA = Tile<T, RCA, BI, NT, false>;
  using TB = Tile<T, RCB, BJ, NT, kPaired>;
  __shared__ __attribute__((aligned(256))) char lds[kBuffers * (TA::kBytes + TB::kBytes)];

  const Place at = place(tiles_i, tiles_j, splits);
  if (!at.in) return;
  const int wave = threadIdx.x >> 6, wi = wave / WJ, wj = wave % WJ;
  const int64_t i0 = at.i * BI, j0 = (int64_t)at.j * kOut;
  int64_t r_begin = 0, r_end = p.R;
  const T *a0 = (const T*)p.a, *b0 = (const T*)p.b[0];
  if (EPI == EPI_PARTIAL) {
    uint32_t range = at.split;
    if (!GATED && p.segments == 2 && range >= splits / 2) {  // the second segment's ranges
      range -= splits / 2;
      a0 += p.a_segment;
      b0 = (const T*)p.b[1];
    }
    r_begin = (int64_t)range * p.r_chunk;
    r_end = r_begin + p.r_chunk < p.R ? r_begin + p.r_chunk : p.R;
  }
  const int64_t lda = RCA ? p.a_i : p.a_r, ldb = RCB ? p.b_j : p.b_r;
  const uint32_t steps = (uint32_t)((r_end - r_begin + kDepth - 1) / kDepth);
  const uint32_t total = EPI == EPI_PLAIN ? steps * p.segments : steps;

  Chunk<T> ca[TA::kChunks], cb[TB::kChunks];
  constexpr int kSplit = GATED ? BJ / 2 : 0;
  // Where step `it` starts: f(A, B, r0).
  auto at_step = [&](uint32_t it, auto f) {
    const T *a = a0, *b = b0;
    if (EPI == EPI_PLAIN && it >= steps) {  // the second segment
      it -= steps;
      a += p.a_segment;
      b = (const T*)p.b[1];
    }
    f(a, b, r_begin + (int64_t)it * kDepth);
  };
  auto load = [&](uint32_t it) {
    at_step(it, [&](const T* a, const T* b, int64_t r0) {
      TA::template load<0>(ca, a, nullptr, lda, i0, p.I, r0, r_end, p.R);
      TB::template load<kSplit>(cb, b, (const T*)p.b[1], ldb, j0, p.J, r0, r_end, p.R);
    });
  };
  auto store = [&](int buffer) {
    char* s = lds + buffer * (TA::kBytes + TB::kBytes);
    TA::store(s, ca);
    TB::store(s + TA::kBytes, cb);
  };

  f32x4 acc[NI][NJ] = {}, sum[NI] = {};
  const bool sums = EPI == EPI_PARTIAL && p.part_sum && at.j == 0 && wj == 0;
  auto compute = [&](int buffer) {
    const char* sa = lds + buffer * (TA::kBytes + TB::kBytes);
    const char* sb = sa + TA::kBytes;
#pragma unroll
    for (int kk = 0; kk < kDepth / 32; kk++) {
      s16x8 b[NJ][kPlanes];
#pragma unroll
      for (int t = 0; t < NJ; t++)
#pragma unroll
        for (int q = 0; q < kPlanes; q++) b[t][q] = TB::read(sb + q * TB::kPlaneBytes, wj * NJ + t, kk);
#pragma unroll
      for (int u = 0; u < NI; u++) {
        s16x8 a[kPlanes];
#pragma unroll
        for (int q = 0; q < kPlanes; q++) a[q] = TA::read(sa + q * TA::kPlaneBytes, wi * NI + u, kk);
#pragma unroll
        for (int k = 0; k < Parts<kPlanes>::kProducts; k++)  // consecutive ones work on different results
#pragma unroll
          for (int t = 0; t < NJ; t++)
            acc[u][t] = mfma<T>(b[t][Parts<kPlanes>::kB[k]], a[Parts<kPlanes>::kA[k]], acc[u][t]);
        if (EPI == EPI_PARTIAL && sums) {  // the bias gradient: the same rows times ones
          const short one = sizeof(T) == 2 && __is_same(T, __half) ? 0x3c00 : 0x3f80;
          const s16x8 ones = {one, one, one, one, one, one, one, one};
#pragma unroll
          for (int q = kPlanes - 1; q >= 0; q--) sum[u] = mfma<T>(ones, a[q], sum[u]);
        }
      }
    }
  };

  if constexpr (DIRECT) {
    // a step goes straight to LDS while the step before it is worked on
    auto stage = [&](uint32_t it, int buffer) {
      at_step(it, [&](const T* a, const T* b, int64_t r0) {
        char* s = lds + buffer * (TA::kBytes + TB::kBytes);
        TA::direct(s, a, nullptr, 0, lda, i0, p.I, r0, r_end);
        TB::direct(s + TA::kBytes, b, (const T*)p.b[1], kSplit, ldb, j0, p.J, r0, r_end);
      });
    };
    auto arrived = [&](uint32_t it, int buffer) {  // this wave's part of the step is in LDS
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      at_step(it, [&](const T*, const T*, int64_t r0) {
        if (r0 + kDepth <= r_end) return;
        char* s = lds + buffer * (TA::kBytes + TB::kBytes);
        TA::clear(s, r0, r_end);
        TB::clear(s + TA::kBytes, r0, r_end);
      });
    };
    stage(0, 0);
    arrived(0, 0);
    for (uint32_t it = 0; it < total; it++) {
      barrier();  // every wave's part of this step is there, and everyone has left the other buffer
      if (it + 1 < total) stage(it + 1, (it + 1) & 1);
      compute(it & 1);
      if (it + 1 < total) arrived(it + 1, (it + 1) & 1);
    }
  } else if constexpr (kBuffers == 2) {
    load(0);
    store(0);
    for (uint32_t it = 0; it < total; it++) {
      __syncthreads();  // everyone has stored this step and left the other buffer
      if (it + 1 < total) load(it + 1);
      compute(it & 1);
      if (it + 1 < total) store((it + 1) & 1);
    }
  } else {
    load(0);
    for (uint32_t it = 0; it < total; it++) {
      if (it) __syncthreads();  // everyone has left the buffer
      store(0);
      __syncthreads();
      if (it + 1 < total) load(it + 1);
      compute(0);
    }
  }

  const int m = threadIdx.x & 15, q = (threadIdx.x & 63) >> 4;
  if constexpr (sizeof(T) == 4) {
    float odd = 0.0f;  // stays 0 while every result is finite
#pragma unroll
    for (int u = 0; u < NI; u++) {
#pragma unroll
      for (int t = 0; t < NJ; t++)
#pragma unroll
        for (int v = 0; v < 4; v++) odd = fmaf(acc[u][t][v], 0.0f, odd);
      if (sums) odd = fmaf(sum[u][0], 0.0f, odd);
    }
    if (odd != 0.0f) {
#pragma unroll
      for (int u = 0; u < NI; u++) {
        const int64_t i = i0 + (wi * NI + u) * 16 + m;
        if (i >= p.I) continue;
        const int segments = EPI == EPI_PLAIN ? p.segments : 1;
#pragma unroll
        for (int t = 0; t < NJ; t++)
#pragma unroll
          for (int v = 0; v < 4; v++) {
            const int row = (wj * NJ + t) * 16 + 4 * q + v;
            const bool second = GATED && row >= kOut;
            const int64_t j = j0 + (second ? row - kOut : row);
            if (j < p.J && !(fabsf(acc[u][t][v]) <= 3.4e38f))
              acc[u][t][v] = exact_sum((const float*)a0, p.a_i, p.a_r, second ? (const float*)p.b[1] : (const float*)b0,
                                       (const float*)p.b[1], p.b_j, p.b_r, segments, p.a_segment, i, j,
                                       r_begin, r_end);
          }
        if (sums && !(fabsf(sum[u][0]) <= 3.4e38f))
          sum[u][0] = exact_sum((const float*)p.a, p.a_i, p.a_r, nullptr, nullptr, 0, 0, 1, 0, i, 0, r_begin, r_end);
      }
    }
  }

  if (EPI == EPI_PARTIAL && sums && q == 0) {
#pragma unroll
    for (int u = 0; u < NI; u++) {
      const int64_t i = i0 + (wi * NI + u) * 16 + m;
      if (i < p.I) p.part_sum[(int64_t)at.split * p.I + i] = sum[u][0];
    }
  }
  constexpr int kRuns = NJ * 4 / RUN / (GATED ? 2 : 1);
  with_act<EPI>(p.act, [&](auto act) {
#pragma unroll
    for (int s = 0; s < kRuns; s++) {
      const int64_t j = j0 + wj * (NJ * 16) + (kPaired ? 32 * s + 8 * q : 16 * s + 4 * q);
      const int64_t n = p.J - j;
      if (n <= 0) continue;
      float bias[RUN] = {}, bias1[RUN] = {};
      if (EPI == EPI_FORWARD || EPI == EPI_DZ) {
        if (p.bias[0]) load_run<T, RUN>(bias, (const T*)p.bias[0] + j, n);
        if (GATED && p.bias[1]) load_run<T, RUN>(bias1, (const T*)p.bias[1] + j, n);
      }
      float total[RUN] = {}, total1[RUN] = {};
#pragma unroll
      for (int u = 0; u < NI; u++) {
        const int64_t i = i0 + (wi * NI + u) * 16 + m;
        if (i >= p.I) continue;
        float v[RUN], w[RUN], ex[RUN] = {};
#pragma unroll
        for (int k = 0; k < RUN; k++) {
          v[k] = acc[u][s * (RUN / 4) + k / 4][k % 4] + bias[k];
          if (GATED) w[k] = acc[u][NJ / 2 + s * (RUN / 4) + k / 4][k % 4] + bias1[k];
        }
        if constexpr (EPI == EPI_PARTIAL) {
          if (!GATED && p.out) {  // one range: the sum is the result
            store_run<T, RUN>((T*)p.out + i * p.out_row + j, v, n);
            continue;
          }
          float* part = p.part + ((int64_t)at.split * p.I + i) * (GATED ? 2 * p.J : p.J) + j;
          store_run<float, RUN>(part, v, n);
          if (GATED) store_run<float, RUN>(part + p.J, w, n);
        } else {
          if (EPI != EPI_PLAIN && p.extra) load_run<T, RUN>(ex, (const T*)p.extra + i * p.extra_row + j, n);
          epilogue<T, EPI, GATED, true, decltype(act)::value, RUN>(p, i, j, n, v, w, ex);
        }
        if (kColumnSums<T, EPI>) {
#pragma unroll
          for (int k = 0; k < RUN; k++) {
            total[k] += v[k];
            if (GATED) total1[k] += w[k];
          }
        }
      }
      if (kColumnSums<T, EPI> && p.part_sum) {
        float* sums_of = p.part_sum + (at.i * WI + wi) * (GATED ? 2 * p.J : p.J) + j;
        store_sums(sums_of, m, n, total);
        if (GATED) store_sums(sums_of + p.J, m, n, total1);
      }
    }
  });
}

// Whether every 16-byte chunk of the operands is aligned and within an end or past it, so that steps
// can go straight to LDS.
template <typename T, bool RCA, bool RCB>
bool takes_direct(const ProductArgs& p) {
  if ((RCA || RCB) && p.R % 8) return false;
  if ((!RCA && p.I % 8) || (!RCB && p.J % 8)) return false;
  const uint64_t bits = (uint64_t)p.a | (uint64_t)p.b[0] | (uint64_t)p.b[1] |
                        (uint64_t)((RCA ? p.a_i : p.a_r) | (RCB ? p.b_j : p.b_r) | p.a_segment) * sizeof(T);
  return sizeof(T) == 2 && bits % 16 == 0;
}

// A launch of 2^32 threads or more is refused, or begins only as many as are left over that without
// an error.
constexpr int64_t kMostThreads = 0xffffffff;
// So more rows than this are taken in slabs, of 256 threads for 64 rows or more.
constexpr int64_t kSlabRows = 1 << 29;

// f(the product of some of its rows) over slabs of about the same size (of more rows than those that
// choose a kernel or ask for scratch); `width` of the partial column sums, if it makes any.
template <typename T, typename F>
int in_slabs(const ProductArgs& p, int64_t width, F f) {
  if (p.I <= kSlabRows) return f(p);
  const int64_t slabs = (p.I + kSlabRows - 1) / kSlabRows;
  const int64_t each = ((p.I + slabs - 1) / slabs + 255) / 256 * 256;
  int64_t sums = 0;
  for (int64_t at = 0; at < p.I; at += each) {
    ProductArgs q = p;
    int64_t rows = 0;
    q.I = p.I - at < each ? p.I - at : each;
    q.a = (const T*)p.a + at * p.a_i;
    q.extra = p.extra ? (const T*)p.extra + at * p.extra_row : nullptr;
    q.out = (T*)p.out + at * p.out_row;
    q.part_sum = p.part_sum ? p.part_sum + sums * width : nullptr;
    q.sum_rows = &rows;
    if (int rc = f(q)) return rc;
    sums += rows;
  }
  if (p.sum_rows) *p.sum_rows = sums;
  return 0;
}

template <typename T, bool RCA, bool RCB, int EPI, bool GATED, bool DIRECT, int BI, int WI, int BJ, int WJ>
int launch_tiles(const ProductArgs& p, int64_t splits, hipStream_t stream) {
  constexpr int kOut = GATED ? BJ / 2 : BJ;
  const int64_t ti = (p.I + BI - 1) / BI, tj = (p.J + kOut - 1) / kOut;
  if (ti > 0x7fffffff / tj || ti * tj > 0x7ffffff0 / splits) return 1;
  const int64_t total = ti * tj * splits, grid = (total + 7) / 8 * 8;
  if (grid > kMostThreads / (64 * WI * WJ)) return 1;
  if (kColumnSums<T, EPI> && p.part_sum) *p.sum_rows = ti * WI;
  hipLaunchKernelGGL((product_kernel<T, RCA, RCB, EPI, GATED, DIRECT, BI, WI, BJ, WJ>), dim3((uint32_t)grid),
                     dim3(64 * WI * WJ), 0, stream, p, (uint32_t)ti, (uint32_t)tj, (uint32_t)splits);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}
template <typename T, bool RCA, bool RCB, int EPI, bool GATED, int BI, int WI, int BJ, int WJ>
int launch_product(const ProductArgs& p, int64_t splits, hipStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (takes_direct<T, RCA, RCB>(p))
      return launch_tiles<T, RCA, RCB, EPI, GATED, true, BI, WI, BJ, WJ>(p, splits, stream);
  return launch_tiles<T, RCA, RCB, EPI, GATED, false, BI, WI, BJ, WJ>(p, splits, stream);
}

// Whether a 16-bit weight gradient of I x J takes 256 x 256 tiles (if its operands are aligned).
inline bool takes_huge_dw(int64_t I, int64_t J) { return I > 128 && J > 128; }  // 256 x 256 tiles

// The tile by the size of C.  256 x 256 where one a CU keeps it busy and operands go straight to LDS
// (us, these : 128 x 128; bf16 8192x4096x4096 264 : 332, weight gradients of 762048x256x512 290 : 330,
// 100000x1024x1024 272 : 302).  128 x 128 where there is one for each CU, 64 x 64 below that (64 x 64
// : 128 x 128; bf16 512x4096x4096 43 : 52, 2048x512x512 7.1 : 10.4, fp32 17 : 34; at 1024x4096x4096,
// 256 tiles, bf16 55 : 55, fp32 296 : 257).  128 x 64 for up to 64 columns of many rows (fp32
// weight gradient of 762048x64x256 271, with 64 x 64 348; but of 762048x3x64, 64 rows, 128 : 76).
// The 128 x 128 weight gradient in 32 bits keeps 7 registers in scratch memory.
template <typename T, bool RCA, bool RCB, int EPI>
int launch_linear(const ProductArgs& p, int64_t splits, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    const int64_t huge = (p.I + 255) / 256 * ((p.J + 255) / 256) * splits;
    if ((EPI == EPI_PARTIAL ? takes_huge_dw(p.I, p.J) : p.J > 128 && huge >= 256) && takes_direct<T, RCA, RCB>(p))
      return launch_tiles<T, RCA, RCB, EPI, false, true, 256, 4, 256, 2>(p, splits, stream);
  }
  const int64_t large = (p.I + 127) / 128 * ((p.J + 127) / 128) * splits;
  if (p.I > 64 && large >= 256) {
    if (p.J > 64) return launch_product<T, RCA, RCB, EPI, false, 128, 2, 128, 2>(p, splits, stream);
    return launch_product<T, RCA, RCB, EPI, false, 128, 4, 64, 1>(p, splits, stream);
  }
  return launch_product<T, RCA, RCB, EPI, false, 64, 4, 64, 1>(p, splits, stream);
}

template <typename T, int EPI>
int launch_gated(const ProductArgs& p, hipStream_t stream) {
  const int64_t large = (p.I + 127) / 128 * ((p.J + 63) / 64);
  if (large >= 256) return launch_product<T, true, true, EPI, true, 128, 4, 128, 1>(p, 1, stream);
  return launch_product<T, true, true, EPI, true, 64, 4, 128, 1>(p, 1, stream);
}

// Few tiles and a long sum: the sum is cut into ranges, so that there is work for every CU, and a
// second kernel adds the ranges (in their order: the same bits every time) and has the epilogue.
// Ranges per segment for C of I x J, summed over R of each of `segments`; 1: not cut.  us, cut :
// whole, fp32 300x4096x512 24 : 105, 512x1024x1024 21 : 30, 4096x512x128 14.8 : 16.7; bf16
// 300x4096x512 12.8 : 35.7, 128x2048x2048 12.2 : 15.7, but 512x1024x1024 13.8 : 9.7, 4096x512x128
// 10 : 6.9 (a step of 16-bit operands takes less time, the second kernel as long).
template <typename T>
int64_t cuts_of(int64_t I, int64_t J, int64_t R, int64_t segments) {
  const int64_t tiles = (I + 63) / 64 * ((J + 63) / 64) * segments;
  if (tiles < 1 || tiles > 128 || R < (sizeof(T) == 4 ? 512 : 2048)) return 1;  // no rows: no tiles
  const int64_t most = R / 256, want = 512 / tiles;
  return want < most ? want : most;
}
inline int64_t cut_rows(int64_t R, int64_t cuts) { return ((R + cuts - 1) / cuts + 63) / 64 * 64; }
template <typename T>
size_t cut_bytes(int64_t I, int64_t J, int64_t R, int64_t segments, bool gated) {
  const int64_t cuts = cuts_of<T>(I, J, R, segments);
  return cuts > 1 ? (size_t)cuts * segments * I * J * (gated ? 8 : 4) : 0;
}

// A wave has one row of 64 columns, a workgroup four.
template <typename T, int EPI, bool GATED>
__global__ __launch_bounds__(256) void finish_kernel(ProductArgs p, uint32_t splits) {
  __shared__ float rows[GATED ? 2 : 1][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t j = (int64_t)blockIdx.x * 64 + lane, i = (int64_t)blockIdx.y * 4 + wave;
  const bool in = i < p.I && j < p.J;
  const int64_t width = GATED ? 2 * p.J : p.J, step = p.I * width;
  float v = 0.0f, w = 0.0f;
  if (in) {
    const float* part = p.part + i * width + j;
    uint32_t s = 0;
    for (; s + 8 <= splits; s += 8) {
      float x[8], y[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        x[k] = part[(s + k) * step];
        if (GATED) y[k] = part[(s + k) * step + p.J];
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        v += x[k];
        if (GATED) w += y[k];
      }
    }
    for (; s < splits; s++) {
      v += part[s * step];
      if (GATED) w += part[s * step + p.J];
    }
    if (EPI != EPI_PLAIN) {
      if (p.bias[0]) v += to_f(((const T*)p.bias[0])[j]);
      if (GATED && p.bias[1]) w += to_f(((const T*)p.bias[1])[j]);
    }
    const float e = EPI != EPI_PLAIN && p.extra ? to_f(((const T*)p.extra)[i * p.extra_row + j]) : 0.0f;
    with_act<EPI>(p.act, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      if (EPI == EPI_FORWARD) {
        v = act_value<ACT>(v);
        if (GATED) v *= w;
        if (p.extra) v += e;
      } else if (EPI == EPI_DZ) {
        float a;
        const float slope = act_both<ACT>(v, a);
        v = GATED ? e * w * slope : e * slope;
        if (GATED) w = e * a;
      }
    });
    T* out = (T*)p.out + i * p.out_row + j;
    out[0] = from_f<T>(v);
    if (EPI == EPI_DZ && GATED) out[p.J] = from_f<T>(w);
  }
  if (kColumnSums<T, EPI> && p.part_sum) {
    rows[0][wave][lane] = v;
    if (GATED) rows[GATED][wave][lane] = w;
    __syncthreads();
    if (wave || j >= p.J) return;
    float* sums = p.part_sum + blockIdx.y * width + j;
#pragma unroll
    for (int h = 0; h < (GATED ? 2 : 1); h++)
      sums[h * p.J] = rows[h][0][lane] + rows[h][1][lane] + rows[h][2][lane] + rows[h][3][lane];
  }
}

// The product cut into `cuts` ranges per segment, their results in `scratch`.
template <typename T, bool RCB, int EPI, bool GATED>
int launch_cut(ProductArgs p, int64_t cuts, char* scratch, hipStream_t stream) {
  p.r_chunk = cut_rows(p.R, cuts);
  const int64_t splits = (p.R + p.r_chunk - 1) / p.r_chunk * p.segments;
  p.part = (float*)scratch;
  ProductArgs ranges = p;
  ranges.part_sum = nullptr;
  ranges.out = nullptr;
  const int rc = GATED ? launch_product<T, true, RCB, EPI_PARTIAL, GATED, 64, 4, 128, 1>(ranges, splits, stream)
                       : launch_product<T, true, RCB, EPI_PARTIAL, GATED, 64, 4, 64, 1>(ranges, splits, stream);
  if (rc) return rc;
  const int64_t rows = (p.I + 3) / 4;
  if (kColumnSums<T, EPI> && p.part_sum) *p.sum_rows = rows;
  hipLaunchKernelGGL((finish_kernel<T, EPI, GATED>), dim3((uint32_t)((p.J + 63) / 64), (uint32_t)rows), dim3(256), 0,
                     stream, p, (uint32_t)splits);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

// What gsr_linear.hip needs of each type (gsr_linear_f32.hip, _f16.hip, _bf16.hip).
// Scratch of a forward, dz or dx product of these sizes; dx is over `segments`.
template <typename T> size_t forward_scratch(int64_t M, int64_t K, int64_t N, bool gated);
template <typename T> size_t dz_scratch(int64_t M, int64_t K, int64_t N, bool gated);
template <typename T> size_t dx_scratch(int64_t M, int64_t K, int64_t N, int segments);
template <typename T> int product_forward(const ProductArgs& p, bool gated, char* scratch, hipStream_t s);
template <typename T> int product_dz(const ProductArgs& p, bool gated, char* scratch, hipStream_t s);
template <typename T> int product_dx(const ProductArgs& p, char* scratch, hipStream_t s);
template <typename T> int product_dw(const ProductArgs& p, int64_t splits, hipStream_t s);
template <typename T> bool product_dw_huge(const ProductArgs& p);

}  // namespace gsr
