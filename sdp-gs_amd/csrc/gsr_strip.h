// gsr_strip.h -- the product of many rows with few inputs (a head's layers: K <= 256, a view's
// pixels as rows): a wave keeps its rows of x in registers and walks along the outputs.
//
// At these widths a tile of C has only a few steps along K, so a tiled kernel spends its time
// filling and draining pipelines.  Here a wave loads all of its 16 NI rows at once, straight into
// the matrix instruction's operand layout (every byte of x is read once).  The weights are first
// written out once as the images that LDS is to hold (16-bit parts, padded with zeros to whole
// tiles, rows in reading order, biases among them): a tile's image goes to LDS by direct loads
// without passing registers or needing bounds, the next one while this one is worked on, and a
// tile's results leave as soon as they are there.
//
// What bounds it: a view's layer 762048x256x512 in bfloat16 moves 1.17 GB (230 us at a copy's rate)
// and takes 353 us forward, 380 with gelu (a call; its kernel alone 361 and more where x is not in a
// cache); its products and its stores overlap only in part (156 us of the one and 172 us of the other
// and of x's loads when timed alone).  762048x3x64 in 32 bits, channel-major, takes 57 us a call and
// its kernel 49, 204 MB at 4.2 TB/s: each of the 5954 workgroups has a single tile, whose loads,
// image, product and stores follow each other, and only the two others on its CU fill the gaps.
//
// Registers: three forms in 32 bits do not fit theirs and keep some in scratch memory, up to 32
// inputs with a residual (48) or an incoming gradient (32), and 65 to 128 inputs (18 and 12).  It
// shows little: with a residual, 762048x20x64 119 us (3.8 TB/s) and 762048x100x64 170 (4.1), forms
// that fit 762048x60x64 136 (4.2) and 762048x160x64 233 (3.8).
#pragma once
#include "gsr_rows.h"

namespace gsr {

// kRows rows of weights in a tile (128 bytes of a result's row; gated, 64 of each half's), kWaves
// waves of 16 kNI rows of x, for up to 32 KS inputs; kGroups workgroups to a CU, as many as its
// registers and LDS hold.
template <typename T, int KS, bool GATED> struct Strip {
  static constexpr bool kSplit = sizeof(T) == 4, kWide = kSplit && KS > 6;
  static constexpr int kNI = kSplit && KS > 4 ? 1 : 2;  // three parts of x fill the registers
  static constexpr int kWaves = kWide && GATED ? 8 : 4;
  static constexpr int kRows = !kSplit || KS == 1 ? 64 : kWide && !GATED ? 16 : 32;
  static constexpr int kGroups = kWide && GATED ? 1 : kSplit || KS > 2 ? 2 : 3;
  static constexpr int kOut = GATED ? kRows / 2 : kRows;  // outputs of a tile
  // Bytes of a row: the 32 of padding turn it by two of the 16 bank groups, so that the lanes that
  // a 16-byte read takes together (0-3, 12-15, 20-23, 24-27 and so on) hit different ones.  The
  // first rows' padding holds the tile's biases as floats, 8 to a row.
  static constexpr int kRow = KS * 64 + 32;
  static constexpr int kPlane = kRows * kRow;
  static constexpr int kImage = (kPlane * Operand<T>::kPlanes + 1023) / 1024 * 1024;
};

// Chunk `at` (8 weights) of row `row` of a tile's image; the first chunk brings the row's bias.
template <typename T, bool GATED, int KS>
__device__ __forceinline__ void image_chunk(const ProductArgs& p, uint32_t tile, int row, int at, char* image) {
  using S = Strip<T, KS, GATED>;
  const bool second = GATED && row >= S::kOut;
  const int64_t j = (int64_t)tile * S::kOut + (second ? row - S::kOut : row);
  const bool in = j < p.J;
  const T* w = (const T*)p.b[second ? 1 : 0];
  const T* row_of_w = w + (in ? j : 0) * p.b_j;
  const int64_t whole = (p.J - 1) * p.b_j + p.R;  // elements, if rows are contiguous
  Chunk<T> c = p.b_r == 1 && whole >= 8 ? load_row_end(row_of_w, at * 8, p.R, w + whole)
                                        : load_tail(row_of_w, at * 8, p.b_r, p.R);
#pragma unroll
  for (int k = 0; k < Operand<T>::kRaw; k++) c.w[k] = in ? c.w[k] : u32x4{0, 0, 0, 0};
  if (at == 0) {
    const T* bias = (const T*)p.bias[second ? 1 : 0];
    ((float*)(image + row / 8 * S::kRow + KS * 64))[row % 8] = bias && in ? to_f(bias[j]) : 0.0f;
  }
  // 16-bit results leave 8 at a time: the rows of a read are 4 + 4 + 4 + 4, 8 apart
  const int place = sizeof(T) == 2 ? (row & ~31) + 16 * ((row >> 2) & 1) + 4 * ((row >> 3) & 3) + (row & 3) : row;
  put_chunk<T>(image + place * S::kRow + at * 16, S::kPlane, c);
}
template <typename T, bool GATED, int KS>
__global__ __launch_bounds__(256) void image_kernel(ProductArgs p, char* images, uint32_t chunks) {
  using S = Strip<T, KS, GATED>;
  const uint32_t id = blockIdx.x * 256 + threadIdx.x;
  if (id >= chunks) return;
  const uint32_t tile = id / (KS * 4 * S::kRows);
  image_chunk<T, GATED, KS>(p, tile, id / (KS * 4) % S::kRows, id % (KS * 4), images + (size_t)tile * S::kImage);
}

// EXTRA: there is a residual (forward).
template <typename T, bool RCA, int EPI, bool GATED, bool EXTRA, int KS>
__global__ __launch_bounds__((64 * Strip<T, KS, GATED>::kWaves), 2) void strip_kernel(
    ProductArgs p, const char* images, uint32_t strips, uint32_t parts, uint32_t part_tiles) {
  using S = Strip<T, KS, GATED>;
  constexpr int kPlanes = Operand<T>::kPlanes, NI = S::kNI, kWaves = S::kWaves, kOut = S::kOut;
  constexpr bool kPaired = sizeof(T) == 2;
  constexpr int RUN = kPaired ? 8 : 4, NJ = S::kRows / 16, kRuns = kOut / 4 / RUN;
  static_assert(kRuns >= 1 && NJ >= 1, "");
  __shared__ __attribute__((aligned(1024))) char lds[2 * S::kImage];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int m = lane & 15, q = lane >> 4;
  const int K = (int)p.R;
  const uint32_t each = gridDim.x >> 3, id = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
  if (id >= strips * parts) return;
  const int64_t i0 = ((int64_t)(id / parts) * kWaves + wave) * (16 * NI);
  const uint32_t tiles = (uint32_t)((p.J + kOut - 1) / kOut), tile0 = id % parts * part_tiles;
  const uint32_t tile1 = tile0 + part_tiles < tiles ? tile0 + part_tiles : tiles;

  // An image into LDS, 1 KB per instruction; every wave issues as many (the last KB more than once).
  constexpr int kFetches = (S::kImage / 1024 + kWaves - 1) / kWaves;
  auto fetch = [&](uint32_t tile, int buffer) {
    const char* src = images + (size_t)tile * S::kImage + lane * 16;
    char* to = lds + buffer * S::kImage;
#pragma unroll
    for (int u = 0; u < kFetches; u++) {
      const int unit = u * kWaves + wave, at = (unit < S::kImage / 1024 ? unit : S::kImage / 1024 - 1) * 1024;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + at),
                                       (__attribute__((address_space(3))) void*)(to + at), 16, 0, 0);
    }
  };
  auto row_of = [&](int u) {  // a row past the last is the last one again: its results are not stored
    const int64_t i = i0 + u * 16 + m;
    return i < p.I ? i : p.I - 1;
  };
  auto column_of = [&](int s) { return kPaired ? 32 * s + 8 * q : 16 * s + 4 * q; };
  auto load_extra = [&](u32x4 (&ex)[NI][kRuns], uint32_t tile) {
    const int64_t j0 = (int64_t)tile * kOut;
    const bool whole = j0 + kOut <= p.J;
#pragma unroll
    for (int u = 0; u < NI; u++)
#pragma unroll
      for (int s = 0; s < kRuns; s++) {
        const T* e = (const T*)p.extra + row_of(u) * p.extra_row;
        ex[u][s] = whole ? ((const Bytes16*)(e + j0 + column_of(s)))->v
                         : load_words_end(e, j0 + column_of(s), p.J, (const T*)p.extra + (p.I - 1) * p.extra_row + p.J);
      }
  };
  const T* const x_end = (const T*)p.a + (p.I - 1) * p.a_i + K;
  if (images) fetch(tile0, 0);
  s16x8 a[NI][KS][kPlanes];
#pragma unroll
  for (int u = 0; u < NI; u++) {
    const int64_t i = row_of(u);
#pragma unroll
    for (int kk = 0; kk < KS; kk++) {
      const int k = kk * 32 + q * 8;
      Chunk<T> c = {};
      if (RCA) {
        const T* x = (const T*)p.a + i * p.a_i;
        if (kk * 32 + 32 <= K) c = load_whole(x + k);
        else if (kk * 32 < K) c = load_row_end(x, k, K, x_end);
      } else if (kk * 32 < K) {
        c = load_tail((const T*)p.a + i, k, p.a_r, K);
      }
      split_chunk<T>(a[u][kk], c);
    }
  }
  u32x4 ex[NI][kRuns] = {}, ex_next[NI][kRuns] = {};
  if (EXTRA) load_extra(ex, tile0);
  if (!images)  // all outputs are one tile: everyone makes its image
    for (int id = threadIdx.x; id < S::kRows * KS * 4; id += 64 * kWaves)
      image_chunk<T, GATED, KS>(p, 0, id / (KS * 4), id % (KS * 4), lds);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  int buffer = 0;

  with_act<EPI>(p.act, [&](auto act) {
    // One tile.  FULL: it lies within C, so its epilogue has no branch and stores kStores times.
    auto step = [&](auto full, uint32_t tile) {
      constexpr bool FULL = decltype(full)::value;
      // every wave's part of this image is in LDS, and everyone has left the image before it
      barrier();
      const uint32_t next = tile + 1 < tile1 ? tile + 1 : tile;
      if (images) fetch(next, buffer ^ 1);
      if (EXTRA) load_extra(ex_next, next);
      const int64_t j0 = (int64_t)tile * kOut;
      const char* image = lds + buffer * S::kImage;
      // the biases (8 of them to a row's padding) are what the sums start from
      f32x4 acc[NI][NJ];
#pragma unroll
      for (int t = 0; t < NJ; t++) {
        const int row = kPaired ? 32 * (t >> 1) + 8 * q + 4 * (t & 1) : 16 * t + 4 * q;
        f32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
        if (EPI != EPI_PLAIN) bias = *(const f32x4*)(image + row / 8 * S::kRow + KS * 64 + row % 8 * 4);
#pragma unroll
        for (int u = 0; u < NI; u++) acc[u][t] = bias;
      }
      // the operands of kQueue reads are on their way while the products of the one before are formed
      constexpr int kReads = KS * NJ, kQueue = kReads * kPlanes < 8 ? kReads : 8 / kPlanes;
      s16x8 b[kQueue][kPlanes];
      auto read = [&](int n) {
        const int kk = n / NJ, t = n % NJ;
#pragma unroll
        for (int z = 0; z < kPlanes; z++)
          b[n % kQueue][z] = *(const s16x8*)(image + z * S::kPlane + (16 * t + m) * S::kRow + (kk * 4 + q) * 16);
      };
#pragma unroll
      for (int n = 0; n < kQueue; n++) read(n);
      // Two workgroups that are both at their products would stay in step and leave memory idle
      // in between: one of the two gives way to the other.
      if (S::kGroups == 2) {
        if (blockIdx.x >> 8 & 1) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
      }
#pragma unroll
      for (int n = 0; n < kReads; n++) {
        const int kk = n / NJ, t = n % NJ;
#pragma unroll
        for (int k = 0; k < Parts<kPlanes>::kProducts; k++)
#pragma unroll
          for (int u = 0; u < NI; u++)
            acc[u][t] = mfma<T>(b[n % kQueue][Parts<kPlanes>::kB[k]], a[u][kk][Parts<kPlanes>::kA[k]], acc[u][t]);
        if (n + kQueue < kReads) read(n + kQueue);
        __builtin_amdgcn_sched_barrier(0);  // keeps this order
      }
      if (S::kGroups == 2) __builtin_amdgcn_s_setprio(3);
      if constexpr (sizeof(T) == 4) {
        float odd = 0.0f;  // stays 0 while every result is finite
#pragma unroll
        for (int u = 0; u < NI; u++)
#pragma unroll
          for (int t = 0; t < NJ; t++)
#pragma unroll
            for (int v = 0; v < 4; v++) odd = fmaf(acc[u][t][v], 0.0f, odd);
        if (odd != 0.0f) {
#pragma unroll
          for (int u = 0; u < NI; u++)
#pragma unroll
            for (int t = 0; t < NJ; t++)
#pragma unroll
              for (int v = 0; v < 4; v++) {
                const int row = t * 16 + 4 * q + v;
                const bool second = GATED && row >= kOut;
                const int64_t i = i0 + u * 16 + m, j = j0 + (second ? row - kOut : row);
                if (i >= p.I || j >= p.J || fabsf(acc[u][t][v]) <= 3.4e38f) continue;
                const float* bias = (const float*)p.bias[second ? 1 : 0];
                acc[u][t][v] = exact_sum((const float*)p.a, p.a_i, p.a_r, (const float*)p.b[second ? 1 : 0],
                                         nullptr, p.b_j, p.b_r, 1, 0, i, j, 0, K) +
                               (EPI != EPI_PLAIN && bias ? bias[j] : 0.0f);
              }
        }
      }
#pragma unroll
      for (int s = 0; s < kRuns; s++) {
        const int64_t j = j0 + column_of(s), n = FULL ? RUN : p.J - j;
        if (!FULL && n <= 0) continue;
        float total[RUN] = {}, total1[RUN] = {};
#pragma unroll
        for (int u = 0; u < NI; u++) {
          const int64_t i = i0 + u * 16 + m;
          if (!FULL && i >= p.I) continue;
          float v[RUN], w[RUN], e[RUN];
          widen<T, RUN>(e, ex[u][s]);
#pragma unroll
          for (int k = 0; k < RUN; k++) {
            v[k] = acc[u][s * (RUN / 4) + k / 4][k % 4];
            if (GATED) w[k] = acc[u][NJ / 2 + s * (RUN / 4) + k / 4][k % 4];
          }
          epilogue<T, EPI, GATED, EXTRA, decltype(act)::value, RUN>(p, i, j, n, v, w, e);
          if (kColumnSums<T, EPI>) {
#pragma unroll
            for (int k = 0; k < RUN; k++) {
              total[k] += v[k];
              if (GATED) total1[k] += w[k];
            }
          }
        }
        if (kColumnSums<T, EPI> && p.part_sum) {
          float* sums = p.part_sum + ((int64_t)(id / parts) * kWaves + wave) * (GATED ? 2 * p.J : p.J) + j;
          store_sums(sums, m, n, total);
          if (GATED) store_sums(sums + p.J, m, n, total1);
        }
      }
      // This wave's part of the next image has to be there.  It was asked for before the stores of
      // this tile, the last kStores of which may go on.
      constexpr int kStores = NI * kRuns * (EPI == EPI_DZ && GATED ? 2 : 1);
      if (FULL) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kStores) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (EXTRA) {
#pragma unroll
        for (int u = 0; u < NI; u++)
#pragma unroll
          for (int s = 0; s < kRuns; s++) ex[u][s] = ex_next[u][s];
      }
      buffer ^= 1;
    };
    // the tiles that lie within C, then the last ones of a ragged C
    const uint32_t fit = i0 + 16 * NI <= p.I ? (uint32_t)(p.J / kOut) : 0;
    uint32_t tile = tile0;
    for (; tile < tile1 && tile < fit; tile++) step(Const<1>(), tile);
    for (; tile < tile1; tile++) step(Const<0>(), tile);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing arrives in LDS that is another's
  });
}

template <typename T, bool GATED, int KS>
bool needs_images(int64_t J) {
  return KS > 2 || J > Strip<T, KS, GATED>::kOut;
}
template <typename T, bool GATED, int KS>
size_t image_bytes(int64_t J) {
  using S = Strip<T, KS, GATED>;
  return needs_images<T, GATED, KS>(J) ? (size_t)((J + S::kOut - 1) / S::kOut) * S::kImage : 0;
}

template <typename T, bool RCA, int EPI, bool GATED, int KS>
int launch_strip(const ProductArgs& p, char* scratch, hipStream_t stream) {
  using S = Strip<T, KS, GATED>;
  constexpr int kOut = S::kOut, kBlock = S::kWaves * 16 * S::kNI;
  const int64_t strips = (p.I + kBlock - 1) / kBlock, tiles = (p.J + kOut - 1) / kOut;
  const int64_t chunks = tiles * S::kRows * KS * 4, groups = 256 * S::kGroups;
  // fewer strips than workgroups: several share one's outputs
  int64_t parts = strips >= groups ? 1 : (groups + strips - 1) / strips;
  if (parts > tiles) parts = tiles;
  const int64_t part_tiles = (tiles + parts - 1) / parts;
  parts = (tiles + part_tiles - 1) / part_tiles;
  const int64_t items = strips * parts;
  if (items + 7 > kMostThreads / (64 * S::kWaves) || chunks > 0x7fffffff) return 1;
  if (kColumnSums<T, EPI> && p.part_sum) *p.sum_rows = strips * S::kWaves;
  // one small tile of weights is made by every workgroup itself: cheaper than a launch before this
  // one (762048x3x64 in 32 bits: 67 us a call with it, 57 without); not a large one (bf16
  // 762048x256x64: 101 us with it, 142 without)
  const char* images = needs_images<T, GATED, KS>(p.J) ? scratch : nullptr;
  if (images)
    hipLaunchKernelGGL((image_kernel<T, GATED, KS>), dim3((uint32_t)((chunks + 255) / 256)), dim3(256), 0, stream, p,
                       scratch, (uint32_t)chunks);
  auto go = [&](auto extra) {
    hipLaunchKernelGGL((strip_kernel<T, RCA, EPI, GATED, decltype(extra)::value, KS>),
                       dim3((uint32_t)((items + 7) / 8 * 8)), dim3(64 * S::kWaves), 0, stream, p,
                       images, (uint32_t)strips, (uint32_t)parts, (uint32_t)part_tiles);
  };
  if (EPI == EPI_DZ || (EPI == EPI_FORWARD && !GATED && p.extra)) go(Const<EPI != EPI_PLAIN && !(EPI == EPI_FORWARD && GATED)>());
  else go(Const<EPI == EPI_DZ>());
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

// Strips for up to 256 inputs and enough rows that every CU has one of 128: below that the tiled
// kernel, which needs no images, is as fast or faster (us, strips : tiles; bf16 20011x256x512 gated
// 26 : 23, 5000x256x512 11 : 7, fp32 20011x193x333 33 : 30; but bf16 190512x256x512 gated 121 : 213,
// 762048x256x512 345 : 480, fp32 262144x256x256 220 : 246).
inline bool takes_strips(int64_t I, int64_t R) { return R <= 256 && I >= 32768; }

// f(integral constant KS) for R inputs.
template <typename F>
auto with_steps(int64_t R, F f) {
  if (R <= 32) return f(Const<1>());
  if (R <= 64) return f(Const<2>());
  if (R <= 128) return f(Const<4>());
  if (R <= 192) return f(Const<6>());
  return f(Const<8>());
}

template <typename T, bool RCA, int EPI, bool GATED>
int launch_strips(const ProductArgs& p, char* scratch, hipStream_t s) {
  return with_steps(p.R, [&](auto ks) { return launch_strip<T, RCA, EPI, GATED, decltype(ks)::value>(p, scratch, s); });
}

template <typename T>
size_t strips_scratch(int64_t J, int64_t R, bool gated) {
  return with_steps(R, [&](auto ks) {
    constexpr int KS = decltype(ks)::value;
    return gated ? image_bytes<T, true, KS>(J) : image_bytes<T, false, KS>(J);
  });
}

template <typename T, int EPI>
size_t forward_or_dz_scratch(int64_t M, int64_t K, int64_t N, bool gated) {
  if (takes_strips(M, K)) return strips_scratch<T>(N, K, gated);
  return EPI == EPI_FORWARD && rows_sizes(M, N, K) ? 0 : cut_bytes<T>(M, N, K, 1, gated);
}

template <typename T, int EPI>
int forward_or_dz(const ProductArgs& p, bool gated, char* scratch, hipStream_t s) {
  const bool strips = takes_strips(p.I, p.R), few = EPI == EPI_FORWARD && rows_sizes(p.I, p.J, p.R);
  if constexpr (EPI == EPI_FORWARD)
    if (few && p.a_r == 1) return gated ? launch_rows<T, EPI, true>(p, s) : launch_rows<T, EPI, false>(p, s);
  const int64_t cuts = strips || few || p.a_r != 1 ? 1 : cuts_of<T>(p.I, p.J, p.R, 1);
  if (cuts > 1)
    return gated ? launch_cut<T, true, EPI, true>(p, cuts, scratch, s) : launch_cut<T, true, EPI, false>(p, cuts, scratch, s);
  if (gated) return strips ? launch_strips<T, true, EPI, true>(p, scratch, s) : launch_gated<T, EPI>(p, s);
  if (p.a_r == 1)
    return strips ? launch_strips<T, true, EPI, false>(p, scratch, s) : launch_linear<T, true, true, EPI>(p, 1, s);
  return strips ? launch_strips<T, false, EPI, false>(p, scratch, s) : launch_linear<T, false, true, EPI>(p, 1, s);
}

template <typename T>
int dx_product(const ProductArgs& p, char* scratch, hipStream_t s) {
  if (p.segments == 1 && takes_strips(p.I, p.R)) return launch_strips<T, true, EPI_PLAIN, false>(p, scratch, s);
  const int64_t cuts = cuts_of<T>(p.I, p.J, p.R, p.segments);
  if (cuts > 1) return launch_cut<T, false, EPI_PLAIN, false>(p, cuts, scratch, s);
  return launch_linear<T, true, false, EPI_PLAIN>(p, 1, s);
}

#define GSR_PRODUCTS(T)                                                                              \
  template <> size_t forward_scratch<T>(int64_t M, int64_t K, int64_t N, bool gated) {               \
    return forward_or_dz_scratch<T, EPI_FORWARD>(M, K, N, gated);                                    \
  }                                                                                                  \
  template <> size_t dz_scratch<T>(int64_t M, int64_t K, int64_t N, bool gated) {                    \
    return forward_or_dz_scratch<T, EPI_DZ>(M, K, N, gated);                                         \
  }                                                                                                  \
  template <> size_t dx_scratch<T>(int64_t M, int64_t K, int64_t N, int segments) {                  \
    if (segments == 1 && takes_strips(M, N)) return strips_scratch<T>(K, N, false);                  \
    return cut_bytes<T>(M, K, N, segments, false);                                                      \
  }                                                                                                  \
  template <> int product_forward<T>(const ProductArgs& p, bool gated, char* scratch, hipStream_t s) { \
    return in_slabs<T>(p, 0, [&](const ProductArgs& q) {                                             \
      return forward_or_dz<T, EPI_FORWARD>(q, gated, scratch, s);                                    \
    });                                                                                              \
  }                                                                                                  \
  template <> int product_dz<T>(const ProductArgs& p, bool gated, char* scratch, hipStream_t s) {    \
    return in_slabs<T>(p, gated ? 2 * p.J : p.J, [&](const ProductArgs& q) {                         \
      return forward_or_dz<T, EPI_DZ>(q, gated, scratch, s);                                         \
    });                                                                                              \
  }                                                                                                  \
  template <> int product_dx<T>(const ProductArgs& p, char* scratch, hipStream_t s) {                \
    return in_slabs<T>(p, 0, [&](const ProductArgs& q) { return dx_product<T>(q, scratch, s); });    \
  }                                                                                                  \
  template <> bool product_dw_huge<T>(const ProductArgs& p) {                                        \
    return sizeof(T) == 2 && takes_huge_dw(p.I, p.J) &&                                              \
           (p.b_j == 1 ? takes_direct<T, false, false>(p) : takes_direct<T, false, true>(p));        \
  }                                                                                                  \
  template <> int product_dw<T>(const ProductArgs& p, int64_t splits, hipStream_t s) {               \
    return p.b_j == 1 ? launch_linear<T, false, false, EPI_PARTIAL>(p, splits, s)                    \
                      : launch_linear<T, false, true, EPI_PARTIAL>(p, splits, s);                    \
  }

}  // namespace gsr
