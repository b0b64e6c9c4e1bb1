// Newton-Schulz orthogonalisation of updates of phi, and the whole momentum
// update around it.
//
// For a matrix U whose shorter side has R <= 80 rows (the n*n + 2n rows of phi,
// n <= 8; a matrix with more rows than columns is read transposed),
//   X_0 = U / (|U|_F + eps),  X_{k+1} = (a_k I + b_k A + c_k A^2) X_k,  A = X_k X_k^T.
// Every factor is a polynomial of A, so they commute and the whole iteration is
// one R x R matrix applied once:
//   A_0 = U U^T / (|U|_F + eps)^2, |U|_F^2 = trace(U U^T)
//   M_k = a_k I + b_k A_k + c_k A_k^2,  A_{k+1} = A_k M_k^2,  Q_{k+1} = Q_k M_k
//   O = (Q / (|U|_F + eps)) U.
// U is read twice (Gram product, application) and O written once, whatever the
// number of steps; the iteration itself never touches a long row.
//
// The price is precision: A_0 holds the squares of the singular values, and the
// iteration lifts a small one a few hundred times, so what rounding takes from
// a small eigenvalue of A_0 is lifted with it (32-bit sums: up to about a
// percent of a singular value near 1/500 of the norm); and in the application
// the strong directions cancel (32-bit sums: 3e-6 of the result, measured).  So
// all three run in 64 bits, on the double-precision matrix instruction
// (8 x 8 x 4), 18.5 T multiply-adds a second here against 34.5 of the scalar
// 32-bit ones; with few rows memory bounds the two passes over U all the same.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

#undef MHC_FILE_ID
#define MHC_FILE_ID 9   // debug-bounds site ids: 9 * 100000 + line

namespace mhc {
namespace ortho {

constexpr int kMaxRows = 80;
constexpr int kMaxSteps = 16;
#ifdef MHC_DEBUG_BOUNDS
constexpr int kMaxMats = 8;      // matrices of one launch: three buffers each fit the debug table
#else
constexpr int kMaxMats = 64;     // matrices of one launch (their pointers travel as kernel arguments)
#endif
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct Mats {
  const void* grad[kMaxMats];
  float* mom[kMaxMats];      // NULL entries never: absent as a whole (orthogonalise only)
  void* out[kMaxMats];       // the orthogonalised matrix, or the parameter to update
};

struct Params {
  int R, C;                  // short and long side
  int64_t rs, cs;            // element (i, k) of the short x long view is at i * rs + k * cs
  int mats;                  // matrices of this launch
  int chunks;                // column chunks of a matrix in the Gram pass
  int gram_ctas;             // CTAs that share the mats * chunks chunks
  int segments;              // Gram partial sums per matrix at most
  double* part;              // [mats][segments][blocks][64]
  double* q;                 // [mats][P][P], P = 8 * NB
  double* exchange;          // [mats][2][P][P], what the clusters' CTAs pass on
  float momentum, rest;      // the update's coefficients (rest = 1 - mu); unused when only orthogonalising
  int nesterov;
  float lr, decay, scale;
  const float* lr_dev;       // NULL, or the learning rate in device memory
  int steps;
  double eps;
  double coeffs[3 * kMaxSteps];
};

// Equal shares of a list of `total` items for `n` takers: taker i has [share(i), share(i + 1)).
__host__ __device__ __forceinline__ int64_t share(int64_t total, int n, int64_t i) { return total * i / n; }
// The taker of item x: the largest i with share(i) <= x.
__device__ __forceinline__ int taker(int64_t total, int n, int64_t x) { return (int)(((x + 1) * n - 1) / total); }

// 8-row blocks, rounded up to the sizes compiled (n = 1 .. 8 need 1 1 2 3 5 6 8 10).
inline int row_blocks(int R) {
  const int nb = (R + 7) / 8;
  return nb <= 3 ? nb : nb <= 5 ? 5 : nb <= 6 ? 6 : nb <= 8 ? 8 : 10;
}
constexpr int lower_blocks(int NB) { return NB * (NB + 1) / 2; }
// Columns of one staged chunk: about 16 to 24 KB a chunk.
constexpr int chunk_cols(int NB) { return NB <= 2 ? 256 : NB <= 5 ? 128 : 64; }
// CTAs on an SM that the kernels' registers are bounded for.
constexpr int gram_occupancy(int NB) { return NB <= 3 ? 3 : NB <= 6 ? 2 : 1; }
// Warps that share one set of columns: more than 21 blocks of accumulators (84
// registers) are split over two warps by block rows.
constexpr int gram_roles(int NB) { return NB > 6 ? 2 : 1; }
constexpr int role_split(int NB) { return NB == 10 ? 7 : NB == 8 ? 6 : NB; }   // first block row of role 1

// D += A B on 8 x 8 x 4 doubles: lane l holds A[l / 4][l % 4], B[l % 4][l / 4]
// and D[l / 4][2 (l % 4) + {0, 1}].  With B the transpose of a row block, A and
// B fragments are loaded the same way.
__device__ __forceinline__ void dmma(double (&d)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
               : "+d"(d[0]), "+d"(d[1])
               : "d"(a), "d"(b));
}

// Four neighbouring elements of a row of the long side as they lie in memory.
template <class T>
struct Raw4 {
  using V = std::conditional_t<std::is_same_v<T, float>, float4, uint2>;
  V v;
  __device__ __forceinline__ void unpack(float (&f)[4]) const {
    if constexpr (std::is_same_v<T, float>) {
      f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    } else {
      f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xFFFF0000u);
      f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ void pack(const float (&f)[4]) {
    if constexpr (std::is_same_v<T, float>) {
      v = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      v.x = pack_bf16x2(f[0], f[1]);
      v.y = pack_bf16x2(f[2], f[3]);
    }
  }
};
template <class T>
__device__ __forceinline__ float ld1(const T* p) {
  if constexpr (std::is_same_v<T, float>) return MHC_LD(p);
  else return bf16_bits_to_f32(MHC_LD(p));
}
template <class T>
__device__ __forceinline__ void st1(T* p, float v) {
  if constexpr (std::is_same_v<T, float>) MHC_ST(p, v);
  else MHC_ST(p, f32_to_bf16_bits(v));
}
// Elements (r, c + j * gap), j = 0 .. 3; zeros beyond the matrix.  kVec: rows of
// cs = 1 that start on a multiple of four elements and have a multiple of four
// of them, gap 1.  Element by element a wider gap lets neighbouring lanes take
// neighbouring columns.
template <bool kVec, class T>
__device__ __forceinline__ void load4(Raw4<T>& raw, const T* base, const Params& P, int r, int64_t c, int gap = 1) {
  raw.v = {};
  if constexpr (kVec) {
    if (r < P.R && c < P.C) raw.v = MHC_LD(reinterpret_cast<const typename Raw4<T>::V*>(base + r * P.rs + c));
  } else {
    const T* p = base + r * P.rs + c * P.cs;
    const int64_t d = gap * P.cs;
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = r < P.R && c + j * gap < P.C ? ld1(p + j * d) : 0.f;
    raw.pack(f);
  }
}
template <bool kVec, class T>
__device__ __forceinline__ void store4(T* base, const Params& P, int r, int64_t c, const float (&f)[4], int gap = 1) {
  if constexpr (kVec) {
    if (r < P.R && c < P.C) {
      Raw4<T> raw;
      raw.pack(f);
      MHC_ST(reinterpret_cast<typename Raw4<T>::V*>(base + r * P.rs + c), raw.v);
    }
  } else {
    T* p = base + r * P.rs + c * P.cs;
    const int64_t d = gap * P.cs;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (r < P.R && c + j * gap < P.C) st1(p + j * d, f[j]);
  }
}

// momentum and the matrix that is orthogonalised, the same rounding in every
// kernel that forms them: m' = mu m + (1 - mu) g, u = mu m' + (1 - mu) g or m'.
__device__ __forceinline__ float new_momentum(const Params& P, float m, float g) {
  return fmaf(P.momentum, m, P.rest * g);
}
__device__ __forceinline__ float update_of(const Params& P, float m1, float g) {
  return P.nesterov ? fmaf(P.momentum, m1, P.rest * g) : m1;
}

// Accumulates block rows [R0, R1) of the lower triangle of u u^T over one
// warp's columns of a staged chunk.
template <int R0, int R1>
struct Gram {
  static constexpr int kBlocks = lower_blocks(R1) - lower_blocks(R0);
  double acc[kBlocks][2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) acc[i][0] = acc[i][1] = 0.0;
  }
  __device__ __forceinline__ void run(const float* tile, int stride, int cols, int lane) {
    const float* p = tile + (lane >> 2) * stride + (lane & 3);
#pragma unroll 2
    for (int k = 0; k < cols; k += 4) {
      double f[R1];
#pragma unroll
      for (int i = 0; i < R1; ++i) f[i] = (double)p[i * 8 * stride + k];
      int x = 0;
#pragma unroll
      for (int i = R0; i < R1; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j) dmma(acc[x++], f[i], f[j]);
    }
  }
  __device__ __forceinline__ void store(double* dst, int lane) const {   // dst: [lower blocks][64]
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      double* d = dst + (lower_blocks(R0) + i) * 64 + 2 * lane;
      d[0] = acc[i][0];
      d[1] = acc[i][1];
    }
  }
};

template <int NB>
constexpr size_t gram_smem() {
  const size_t tiles = 2 * (size_t)(8 * NB) * (chunk_cols(NB) + 4) * sizeof(float);
  const size_t sums = (size_t)(kWarps / gram_roles(NB)) * lower_blocks(NB) * 64 * sizeof(double);
  return tiles > sums ? tiles : sums;
}

// Partial Gram products.  The matrices' chunks of columns are one list of which
// every CTA takes an equal share; a share that ends inside a matrix leaves a
// partial sum there.  A CTA walks its chunks through two shared-memory tiles:
// the next chunk's loads are in flight while the warps multiply this one, each
// taking its share of a chunk's columns.  With momentum the kernel also forms
// and writes the new momentum; the thread that loads an element writes it.
// 64 x 24 x 16384 with momentum: 53 us, 302 MB at 5.7 TB/s.  8 x 80 x 32768:
// 90 us, 0.92 G multiply-adds, 55% of the matrix pipe's rate.
template <int NB, class T, bool kMom, bool kVec>
__global__ void __launch_bounds__(kThreads, gram_occupancy(NB)) gram_kernel(const __grid_constant__ Params P,
                                                                           const __grid_constant__ Mats M) {
  constexpr int kRows = 8 * NB, KC = chunk_cols(NB), kStride = KC + 4, kB = lower_blocks(NB);
  constexpr int kRoles = gram_roles(NB), kColWarps = kWarps / kRoles, kWarpCols = KC / kColWarps;
  constexpr int kPer = kRows * (KC / 4) / kThreads;   // 4-element pieces of a chunk per thread
  constexpr int kGap = kVec ? 1 : KC / 4;             // columns between a piece's elements
  static_assert(kRows * (KC / 4) % kThreads == 0 && kWarpCols % 4 == 0, "chunk split");
  extern __shared__ __align__(16) unsigned char smem[];
  float* tile = reinterpret_cast<float*>(smem);       // two of [kRows][kStride]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t total = (int64_t)P.mats * P.chunks;
  const int64_t x0 = share(total, P.gram_ctas, blockIdx.x), x1 = share(total, P.gram_ctas, blockIdx.x + 1);

  Raw4<T> g[kPer];
  Raw4<float> m[kPer];
  auto fetch = [&](int64_t x) {
    const int mat = (int)(x / P.chunks);
    const int64_t col = (x - (int64_t)mat * P.chunks) * KC;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = threadIdx.x + i * kThreads, r = e / (KC / 4), c = (e % (KC / 4)) * (kVec ? 4 : 1);
      load4<kVec>(g[i], static_cast<const T*>(M.grad[mat]), P, r, col + c, kGap);
      if (kMom) load4<kVec>(m[i], static_cast<const float*>(M.mom[mat]), P, r, col + c, kGap);
    }
  };
  auto stage = [&](int64_t x, float* dst) {
    const int mat = (int)(x / P.chunks);
    const int64_t col = (x - (int64_t)mat * P.chunks) * KC;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = threadIdx.x + i * kThreads, r = e / (KC / 4), c = (e % (KC / 4)) * (kVec ? 4 : 1);
      float f[4];
      g[i].unpack(f);
      if (kMom) {
        float m1[4];
        m[i].unpack(m1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m1[j] = new_momentum(P, m1[j], f[j]);
          f[j] = update_of(P, m1[j], f[j]);
        }
        store4<kVec>(M.mom[mat], P, r, col + c, m1, kGap);
      }
      if constexpr (kVec) {
        *reinterpret_cast<float4*>(dst + r * kStride + c) = make_float4(f[0], f[1], f[2], f[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[r * kStride + c + j * kGap] = f[j];
      }
    }
  };

  const int cw = warp / kRoles;
  double* sums = reinterpret_cast<double*>(smem) + (size_t)cw * kB * 64;
  // The matrix's sum over this CTA's chunks: the column warps' in warp order.
  auto finish = [&](int mat, auto& gram) {
    __syncthreads();   // the tiles have been read
    gram.store(sums, lane);
    __syncthreads();
    const int first = taker(total, P.gram_ctas, (int64_t)mat * P.chunks);
    double* dst = P.part + ((int64_t)mat * P.segments + (blockIdx.x - first)) * (kB * 64);
    for (int i = threadIdx.x; i < kB * 64; i += kThreads) {
      double v = 0.0;
#pragma unroll
      for (int w = 0; w < kColWarps; ++w) v += reinterpret_cast<const double*>(smem)[w * kB * 64 + i];
      MHC_ST(dst + i, v);
    }
    __syncthreads();
    gram.clear();
  };
  // One role's whole walk, so that a warp holds its own accumulators only; both
  // roles pass the same number of barriers.
  auto walk = [&](auto gram) {
    gram.clear();
    if (x0 < x1) fetch(x0);
    bool staged = false;
    for (int64_t x = x0; x < x1; ++x) {
      float* cur = tile + ((x - x0) & 1) * kRows * kStride;
      float* nxt = tile + ((x - x0 + 1) & 1) * kRows * kStride;
      if (!staged) {
        stage(x, cur);
        __syncthreads();
      }
      const int mat = (int)(x / P.chunks);
      const bool last = x + 1 == x1 || (int)((x + 1) / P.chunks) != mat;
      if (x + 1 < x1) fetch(x + 1);
      gram.run(cur + cw * kWarpCols, kStride, kWarpCols, lane);
      staged = !last;
      if (last) {
        finish(mat, gram);   // the sums lie over the tiles: the next chunk is staged after them
      } else {
        stage(x + 1, nxt);   // last read in the round before, ended by its barrier
        __syncthreads();
      }
    }
  };
  cudaTriggerProgrammaticLaunchCompletion();   // the iteration waits for this kernel's end itself
  if constexpr (kRoles == 1) {
    walk(Gram<0, NB>{});
  } else {
    if ((warp & 1) == 0)
      walk(Gram<0, role_split(NB)>{});
    else
      walk(Gram<role_split(NB), NB>{});
  }
}

// Row stride of an R x R matrix of doubles in shared memory: 4 or 12 modulo 16,
// so that the four rows a half warp's fragment load touches fall into different banks.
constexpr int ns_stride(int NB) { return 8 * NB + 4; }

// One 8 x 8 block of X Y^T over all columns: x, y point at the lane's fragment
// places in X's and Y's row blocks.  Two chains of products, added at the end.
template <int NB>
__device__ __forceinline__ void block_product(const double* x, const double* y, double (&d)[2]) {
  double e[2] = {0.0, 0.0};
  d[0] = d[1] = 0.0;
#pragma unroll
  for (int k = 0; k < 8 * NB; k += 8) {
    dmma(d, x[k], y[k]);
    dmma(e, x[k + 4], y[k + 4]);
  }
  d[0] += e[0];
  d[1] += e[1];
}
// Partial Gram sums of a matrix.
__device__ __forceinline__ const double* partials(const Params& P, int mat, int blocks, int& segments) {
  const int64_t total = (int64_t)P.mats * P.chunks, c0 = (int64_t)mat * P.chunks;
  segments = taker(total, P.gram_ctas, c0 + P.chunks - 1) - taker(total, P.gram_ctas, c0) + 1;
  return P.part + (int64_t)mat * P.segments * (blocks * 64);
}
// 1 / (|U|_F + eps) from the diagonal, by one warp.
__device__ __forceinline__ double inverse_norm(const double* A, int rows, int stride, double eps) {
  double tr = 0.0;
  for (int i = threadIdx.x & 31; i < rows; i += 32) tr += A[i * stride + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tr += __shfl_xor_sync(0xffffffffu, tr, o);
  return 1.0 / (sqrt(tr) + eps);
}

// Block x of the lower triangle, row by row, and the first of a lane's two
// neighbouring results in it.
__host__ __device__ constexpr void block_place(int x, int lane, int& bi, int& bj, int& r, int& c) {
  bi = 0;
  while (lower_blocks(bi + 1) <= x) ++bi;
  bj = x - lower_blocks(bi);
  r = 8 * bi + (lane >> 2);
  c = 8 * bj + 2 * (lane & 3);
}
// A result at (r, c) of the lower triangle's blocks is stored in its place and its
// mirror image's.  In a diagonal block (r, c) and (c, r) are two lanes' results,
// which may differ in their last bits: the one on or below the diagonal is stored,
// in both places, so that every word has one writer and the matrix is symmetric.
__host__ __device__ constexpr bool mirrors(int r, int c) { return r >= c; }
__device__ __forceinline__ void put_mirrored(double* X, int stride, int r, int c, double v) {
  if (!mirrors(r, c)) return;
  X[r * stride + c] = v;
  X[c * stride + r] = v;
}
template <int NB>
constexpr bool one_writer_a_word() {
  int writers[8 * NB][8 * NB] = {};
  for (int x = 0; x < lower_blocks(NB); ++x)
    for (int lane = 0; lane < 32; ++lane) {
      int bi = 0, bj = 0, r = 0, c = 0;
      block_place(x, lane, bi, bj, r, c);
      for (int j = 0; j < 2; ++j)
        if (mirrors(r, c + j)) {
          ++writers[r][c + j];
          if (r != c + j) ++writers[c + j][r];
        }
    }
  for (const auto& row : writers)
    for (int n : row)
      if (n != 1) return false;
  return true;
}

// The iteration on matrices of up to 40 rows, a CTA each: a warp per block of
// the lower triangle (products of commuting symmetric matrices are symmetric;
// Y's rows serve as its columns) and another for the second product of a step.
// What is left is latency: 13 dependent products of at most 10 instructions.
// Five steps: 3.9 us for 8 rows, 7 for 24, 12 for 35.
constexpr int kSmallBlocks = 5;
constexpr int small_warps(int NB) { return 2 * lower_blocks(NB); }
template <int NB>
constexpr size_t small_smem() {
  return (size_t)4 * (8 * NB) * ns_stride(NB) * sizeof(double);
}
// The place of a warp and lane in it; warps past the two sets have none.
template <int NB>
struct SmallPlace {
  static constexpr int kB = lower_blocks(NB), S = ns_stride(NB);
  static_assert(one_writer_a_word<NB>(), "a word of the square with no writer or with two");
  bool first, second;   // this warp has a block of the first or of the second product
  int x, r, c, fx, fy;  // its block, this lane's two results (r, c), (r, c + 1), fragment places
  __device__ __forceinline__ SmallPlace() {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    first = warp < kB;
    second = warp >= kB && warp < 2 * kB;
    x = second ? warp - kB : first ? warp : 0;
    int bi, bj;
    block_place(x, lane, bi, bj, r, c);
    fx = (8 * bi + (lane >> 2)) * S + (lane & 3);
    fy = (8 * bj + (lane >> 2)) * S + (lane & 3);
  }
  __device__ __forceinline__ void put(double* X, double v0, double v1) const {
    put_mirrored(X, S, r, c, v0);
    put_mirrored(X, S, r, c + 1, v1);
  }
};
// From the Gram matrix in A (all of it, behind a barrier) to Q, by a whole CTA;
// returns 1 / (|U|_F + eps), which Q lacks.  Q is behind a barrier.
template <int NB>
__device__ __forceinline__ double iterate_small(const Params& P, const SmallPlace<NB>& pl, double* A, double* Mk,
                                                double* W, double* Q, double* shared_inv) {
  constexpr int kRows = 8 * NB, S = ns_stride(NB);
  if (threadIdx.x < 32) {
    const double v = inverse_norm(A, kRows, S, P.eps);
    if (threadIdx.x == 0) *shared_inv = v;
  }
  __syncthreads();
  const double inv = *shared_inv;
  for (int e = threadIdx.x; e < kRows * kRows; e += blockDim.x) A[e / kRows * S + e % kRows] *= inv * inv;
  __syncthreads();
  double d[2];
  for (int k = 0; k < P.steps; ++k) {
    const double a = P.coeffs[3 * k], b = P.coeffs[3 * k + 1], cc = P.coeffs[3 * k + 2];
    const bool more = k + 1 < P.steps;
    if (pl.first) {
      block_product<NB>(A + pl.fx, A + pl.fy, d);
      const int at = pl.r * S + pl.c;
      const double v0 = (pl.r == pl.c ? a : 0.0) + b * A[at] + cc * d[0];
      const double v1 = (pl.r == pl.c + 1 ? a : 0.0) + b * A[at + 1] + cc * d[1];
      pl.put(Mk, v0, v1);
      if (k == 0) pl.put(Q, v0, v1);
    }
    __syncthreads();
    const bool work = (pl.first && more) || (pl.second && k > 0);
    if (work) block_product<NB>(pl.second ? Q + pl.fx : A + pl.fx, Mk + pl.fy, d);
    __syncthreads();
    if (work) pl.put(pl.second ? Q : W, d[0], d[1]);
    __syncthreads();
    if (more) {
      if (pl.first) {
        block_product<NB>(W + pl.fx, Mk + pl.fy, d);
        pl.put(A, d[0], d[1]);
      }
      __syncthreads();
    }
  }
  return inv;
}
template <int NB>
__global__ void __launch_bounds__(32 * small_warps(NB)) iterate_small_kernel(const __grid_constant__ Params P) {
  constexpr int kRows = 8 * NB, S = ns_stride(NB), kB = lower_blocks(NB), kT = 32 * small_warps(NB);
  extern __shared__ __align__(16) unsigned char smem[];
  double* A = reinterpret_cast<double*>(smem);
  double *Mk = A + kRows * S, *W = Mk + kRows * S, *Q = W + kRows * S;
  __shared__ double shared_inv;
  const SmallPlace<NB> pl;
  const int odd = pl.second ? 1 : 0;   // first warps add the even elements of their block, second ones the odd
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  int segments;
  const double* part = partials(P, blockIdx.x, kB, segments) + pl.x * 64 + 2 * (threadIdx.x & 31) + odd;
  double v = 0.0;
#pragma unroll 16
  for (int s = 0; s < segments; ++s) v += MHC_LD(part + (int64_t)s * (kB * 64));
  put_mirrored(A, S, pl.r, pl.c + odd, v);
  __syncthreads();
  const double inv = iterate_small<NB>(P, pl, A, Mk, W, Q, &shared_inv);
  double* q = P.q + (int64_t)blockIdx.x * kRows * kRows;
  for (int e = threadIdx.x; e < kRows * kRows; e += kT) MHC_ST(q + e, Q[e / kRows * S + e % kRows] * inv);
}

// Small matrices whole in one launch, a CTA each: the matrix stays in shared
// memory between the Gram product, the iteration and the application.  One CTA's
// matrix pipe takes about 4 cycles a product, so the limit is 3,000 of them,
// some 6 us, about what three kernels cost in launches and starts alone.
// 8 x 1024: 7 us against 10 in three kernels, and 10 a call against 15.
constexpr int kFusedBlocks = 3;
constexpr int kFusedThreads = 384;   // 12 warps: 24 rows' iteration needs as many
constexpr int kFusedWarps = kFusedThreads / 32;
__host__ __device__ constexpr int fused_stride(int C) { return (C + 31) / 32 * 32 + 4; }
constexpr size_t kFusedMatrix = 128 * 1024;   // bytes of the matrix at most
inline bool fused_fits(int NB, int C) {
  return NB <= kFusedBlocks && (int64_t)(lower_blocks(NB) + NB * NB) * C <= 4 * 3000 &&
         (int64_t)8 * NB * fused_stride(C) * 4 <= (int64_t)kFusedMatrix;
}
template <int NB>
constexpr size_t fused_fixed_smem() {   // beside the matrix
  return small_smem<NB>() + (size_t)kFusedWarps * lower_blocks(NB) * 64 * sizeof(double);
}
template <int NB>
size_t fused_smem(int C) {
  return fused_fixed_smem<NB>() + (size_t)8 * NB * fused_stride(C) * sizeof(float);
}
template <int NB, class T, class TO, bool kMom, bool kVec>
__global__ void __launch_bounds__(kFusedThreads) fused_kernel(const __grid_constant__ Params P,
                                                              const __grid_constant__ Mats M) {
  constexpr int kRows = 8 * NB, S = ns_stride(NB), kB = lower_blocks(NB);
  extern __shared__ __align__(16) unsigned char smem[];
  double* A = reinterpret_cast<double*>(smem);
  double *Mk = A + kRows * S, *W = Mk + kRows * S, *Q = W + kRows * S;
  double* sums = Q + kRows * S;                                              // [kFusedWarps][kB][64]
  float* U = reinterpret_cast<float*>(sums + kFusedWarps * kB * 64);         // [kRows][stride]
  __shared__ double shared_inv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, stride = fused_stride(P.C), width = stride - 4;
  const T* g = static_cast<const T*>(M.grad[blockIdx.x]);
  float* mom = kMom ? M.mom[blockIdx.x] : nullptr;
  TO* out = static_cast<TO*>(M.out[blockIdx.x]);
  const int quarter = width / 4, gap = kVec ? 1 : quarter;
  for (int e = threadIdx.x; e < kRows * quarter; e += kFusedThreads) {
    const int r = e / quarter, c = (e % quarter) * (kVec ? 4 : 1);
    Raw4<T> raw;
    load4<kVec>(raw, g, P, r, c, gap);
    float f[4];
    raw.unpack(f);
    if constexpr (kMom) {
      Raw4<float> rm;
      load4<kVec>(rm, static_cast<const float*>(mom), P, r, c, gap);
      float m1[4];
      rm.unpack(m1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m1[j] = new_momentum(P, m1[j], f[j]);
        f[j] = update_of(P, m1[j], f[j]);
      }
      store4<kVec>(mom, P, r, c, m1, gap);
    }
    if constexpr (kVec) {
      *reinterpret_cast<float4*>(U + r * stride + c) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) U[r * stride + c + j * gap] = f[j];
    }
  }
  __syncthreads();
  {
    Gram<0, NB> gram;
    gram.clear();
    // every warp eight columns at a time
    for (int c = warp * 8; c < width; c += kFusedWarps * 8) gram.run(U + c, stride, 8, lane);
    gram.store(sums + warp * kB * 64, lane);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kB * 64; e += kFusedThreads) {
    double v = 0.0;
#pragma unroll
    for (int w = 0; w < kFusedWarps; ++w) v += sums[w * kB * 64 + e];
    int bi, bj, r, c;
    block_place(e / 64, (e & 63) >> 1, bi, bj, r, c);
    put_mirrored(A, S, r, c + (e & 1), v);
  }
  __syncthreads();
  const SmallPlace<NB> pl;
  const double inv = iterate_small<NB>(P, pl, A, Mk, W, Q, &shared_inv);
  for (int e = threadIdx.x; e < kRows * kRows; e += kFusedThreads) Q[e / kRows * S + e % kRows] *= inv;
  __syncthreads();
  float keep = 0.f, step = 0.f;
  if (kMom) {
    const float lr = P.lr_dev ? MHC_LDG(P.lr_dev) : P.lr;
    keep = 1.f - lr * P.decay;
    step = -lr * P.scale;
  }
  // a warp eight columns at a time: B fragments are U[4 k + lane % 4][c + lane / 4],
  // results the neighbouring columns c + 2 (lane % 4) and the next of rows lane / 4 + 8 i
  for (int c = warp * 8; c < P.C; c += kFusedWarps * 8) {
    double acc[NB][2];
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i][0] = acc[i][1] = 0.0;
#pragma unroll
    for (int k = 0; k < 2 * NB; ++k) {
      const double f = (double)U[(4 * k + (lane & 3)) * stride + c + (lane >> 2)];
#pragma unroll
      for (int i = 0; i < NB; ++i) dmma(acc[i], Q[(8 * i + (lane >> 2)) * S + 4 * k + (lane & 3)], f);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = 8 * i + (lane >> 2);
        const int64_t oc = c + 2 * (lane & 3) + j;
        if (r < P.R && oc < P.C) {
          TO* o = out + r * P.rs + oc * P.cs;
          const float v = (float)acc[i][j];
          st1(o, kMom ? fmaf(keep, ld1(static_cast<const TO*>(o)), step * v) : v);
        }
      }
  }
}

// The iteration on larger matrices, a cluster each.  One CTA's matrix pipe
// needs 40 us for five steps on 80 rows at its peak (83 measured); the cluster's
// CTAs share the rows, kSP row blocks each.  With A whole in every CTA, a strip
// X of rows stays local under X -> X A, so a step is four of these,
//   B = A_s A, C = B A, D = C A, E = D A:
//   A_s' = a^2 A_s + 2ab B + (b^2 + 2ac) C + 2bc D + c^2 E,
//   Q_s' = a Q_s + b Q_s A + c (Q_s A) A,
// and one exchange of the new strips.  That goes through a copy in global memory
// (the L2): a CTA's stores into the others' shared memory took 320 cycles for
// each of them, 3,200 a step at ten CTAs.  Two warps have a block column,
// one for each chain of products; every lane keeps its two elements of a strip
// in registers.  Five steps on 80 rows: 22 us, about 4 of them a step.
template <int NB, int kSP>
constexpr size_t cluster_smem() {
  return (size_t)(8 * NB + 5 * 8 * kSP) * ns_stride(NB) * sizeof(double);
}
template <int NB, int kSP>
__global__ void __launch_bounds__(64 * NB) iterate_cluster_kernel(const __grid_constant__ Params P) {
  constexpr int kRows = 8 * NB, S = ns_stride(NB), kB = lower_blocks(NB), kCl = NB / kSP, kT = 64 * NB;
  extern __shared__ __align__(16) unsigned char smem[];
  double* A = reinterpret_cast<double*>(smem);       // this step's whole matrix
  double* strips = A + kRows * S;
  double *X0 = strips, *X1 = strips + 8 * kSP * S, *X2 = strips + 16 * kSP * S;   // B, C, D
  double *Qs = strips + 24 * kSP * S, *QA = strips + 32 * kSP * S;
  __shared__ double inv_norm;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool qside = warp >= NB;                     // this warp has the Q chain
  const int col = qside ? warp - NB : warp;          // and this block column
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int rank = (int)cluster.block_rank(), mat = blockIdx.x / kCl;
  const int fr = lane >> 2, fc = lane & 3;           // fragment place in a block
  const int row0 = rank * kSP * 8;                   // the strip's first row
  const int c = 8 * col + 2 * fc;                    // this lane's two columns
  double* shared_a = P.exchange + (int64_t)mat * 2 * kRows * kRows;   // two copies in turn
  auto gather = [&](int which) {                     // the others' strips; never cached in L1
    const double2* src = reinterpret_cast<const double2*>(shared_a + which * kRows * kRows);
    constexpr int kRowPairs = kRows / 2;
#pragma unroll 4
    for (int e = threadIdx.x; e < kRows * kRowPairs; e += kT)
      *reinterpret_cast<double2*>(A + e / kRowPairs * S + 2 * (e % kRowPairs)) = __ldcg(MHC_LDP(src + e, 16));
  };
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  {
    // the Gram partial sums, each block by one warp of the cluster
    int segments;
    const double* part = partials(P, mat, kB, segments);
    for (int x = rank * 2 * NB + warp; x < kB; x += kCl * 2 * NB) {
      double v0 = 0.0, v1 = 0.0;
#pragma unroll 16
      for (int s = 0; s < segments; ++s) {
        const double2 v = MHC_LD(reinterpret_cast<const double2*>(part + (int64_t)s * (kB * 64) + x * 64 + 2 * lane));
        v0 += v.x;
        v1 += v.y;
      }
      int bi = 0;
      while (lower_blocks(bi + 1) <= x) ++bi;
      const int bj = x - lower_blocks(bi), r = 8 * bi + fr, cc = 8 * bj + 2 * fc;
      if (bj < bi) {   // below the diagonal blocks: the mirror image too
        MHC_ST(shared_a + cc * kRows + r, v0);
        MHC_ST(shared_a + (cc + 1) * kRows + r, v1);
      }
      MHC_ST(reinterpret_cast<double2*>(shared_a + r * kRows + cc), make_double2(v0, v1));
    }
  }
  cluster.sync();
  gather(0);
  __syncthreads();
  if (warp == 0) {
    const double v = inverse_norm(A, kRows, S, P.eps);
    if (lane == 0) inv_norm = v;
  }
  __syncthreads();
  const double inv = inv_norm;
  for (int e = threadIdx.x; e < kRows * kRows; e += kT) A[e / kRows * S + e % kRows] *= inv * inv;
  __syncthreads();
  double as[kSP][2], q[kSP][2];   // the lane's elements: as on the A side, q on the Q side
#pragma unroll
  for (int s = 0; s < kSP; ++s)
#pragma unroll
    for (int j = 0; j < 2; ++j) as[s][j] = A[(row0 + 8 * s + fr) * S + c + j];
  // strip rows in X (row stride S) times this warp's block column of A
  auto times = [&](const double* X, double (&d)[kSP][2]) {
#pragma unroll
    for (int s = 0; s < kSP; ++s) block_product<NB>(X + (8 * s + fr) * S + fc, A + (8 * col + fr) * S + fc, d[s]);
  };
  auto put = [&](double* X, const double (&d)[kSP][2]) {
#pragma unroll
    for (int s = 0; s < kSP; ++s)
      *reinterpret_cast<double2*>(X + (8 * s + fr) * S + c) = make_double2(d[s][0], d[s][1]);
  };
  for (int k = 0; k < P.steps; ++k) {
    const double a = P.coeffs[3 * k], b = P.coeffs[3 * k + 1], cc = P.coeffs[3 * k + 2];
    const bool more = k + 1 < P.steps;
    double B[kSP][2], C[kSP][2], D[kSP][2], E[kSP][2];
    if (qside) {
      if (k == 0) {
        // Q = I: the new Q is the step's polynomial itself, B from the A side
      } else {
        times(Qs, B);        // Q A
        put(QA, B);
      }
    } else if (k == 0 || more) {
      times(A + row0 * S, B);
      put(X0, B);
    }
    __syncthreads();
    if (qside) {
      if (k == 0) {
#pragma unroll
        for (int s = 0; s < kSP; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            q[s][j] = (row0 + 8 * s + fr == c + j ? a : 0.0) + b * as[s][j] + cc * X0[(8 * s + fr) * S + c + j];
      } else {
        times(QA, C);
#pragma unroll
        for (int s = 0; s < kSP; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j) q[s][j] = a * q[s][j] + b * B[s][j] + cc * C[s][j];
      }
      put(Qs, q);            // read before the barrier above
    } else if (more) {
      times(X0, C);
      put(X1, C);
    }
    if (!more) break;
    __syncthreads();
    if (!qside) {
      times(X1, D);
      put(X2, D);
    }
    __syncthreads();
    if (!qside) {
      times(X2, E);
      const double ka = a * a, kb = 2 * a * b, kc = b * b + 2 * a * cc, kd = 2 * b * cc, ke = cc * cc;
      double* dst = shared_a + ((k + 1) & 1) * kRows * kRows;
#pragma unroll
      for (int s = 0; s < kSP; ++s) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          as[s][j] = ka * as[s][j] + kb * B[s][j] + kc * C[s][j] + kd * D[s][j] + ke * E[s][j];
        MHC_ST(reinterpret_cast<double2*>(dst + (row0 + 8 * s + fr) * kRows + c), make_double2(as[s][0], as[s][1]));
      }
    }
    // the strips are written and A has been read; a copy is written again two
    // steps later, behind a barrier that its readers have passed
    cluster.sync();
    gather((k + 1) & 1);
    __syncthreads();
  }
  double* out = P.q + (int64_t)mat * kRows * kRows;
  if (qside)
#pragma unroll
    for (int s = 0; s < kSP; ++s)
      MHC_ST(reinterpret_cast<double2*>(out + (row0 + 8 * s + fr) * kRows + c),
             make_double2(q[s][0] * inv, q[s][1] * inv));
}

// O = Q U and what is made of it: the output, or the parameter's update
//   p' = (1 - lr decay) p - lr scale O.
// A warp takes 32 columns at a time.  Lane l loads four neighbouring columns
// 4 (l / 4) .. of row 4 k + l % 4, which are its B fragments of four 8-column
// products whose columns lie four apart; their results leave it eight
// neighbouring columns 8 (l % 4) .. of rows l / 4 + 8 i.  So both ends are whole
// vectors (element by element the columns of a product lie side by side instead,
// for the lanes' sake) and nothing goes through shared memory but Q and the old
// parameters, which are fetched there (cp.async, by the lane that updates them) while the
// products run.  The next columns' first rows are loaded before this step's
// results are stored.  With few rows all of a step's loads are in registers at
// once instead, and other warps' work covers them.
// 64 x 24 x 16384, update: 77 us, 403 MB at 5.2 TB/s.  8 x 80 x 32768: 141 us,
// 1.68 G multiply-adds, 65% of the matrix pipe's rate; taking out the stores, the
// parameters or the loads gains 10 us each, so no single one of them holds it.
// Turns at the pipe for the two warps that share one (288 us a call where this
// took 274) and 16 warps of half the rows each (283) were slower.
constexpr int apply_occupancy(int NB) { return NB <= 3 ? 2 : 1; }
// row loads in flight; element by element they are all that hides their latency
constexpr int apply_ahead(int NB, bool vec) { return NB <= 3 || (!vec && NB == 5) ? 2 * NB : !vec && NB == 6 ? 6 : 4; }
// Old parameters go through shared memory where the registers are full of sums
// (24 rows: 76 us with them loaded behind the products, 82 through shared memory).
constexpr bool apply_stages(int NB, bool mom, bool vec) { return NB > 3 && mom && vec; }
// 16-byte pieces of old parameters a lane fetches: two halves of four columns a row block
template <int NB, class TO>
constexpr int apply_pieces() {
  return NB * 8 * (int)sizeof(TO) / 16;
}
template <int NB, class TO, bool kStage>
constexpr size_t apply_smem(int warps) {
  return (size_t)(8 * NB) * ns_stride(NB) * sizeof(double) +
         (kStage && NB > 3 ? (size_t)warps * apply_pieces<NB, TO>() * 32 * 16 : 0);
}
template <int NB, class T, class TO, bool kMom, bool kVec>
__global__ void __launch_bounds__(kThreads, apply_occupancy(NB)) apply_kernel(const __grid_constant__ Params P,
                                                                             const __grid_constant__ Mats M) {
  constexpr int kRows = 8 * NB, S = ns_stride(NB), kK = 2 * NB, kAhead = apply_ahead(NB, kVec);
  constexpr bool kStage = apply_stages(NB, kMom, kVec);
  constexpr int kGap = kVec ? 1 : 8, kHalf = kVec ? 4 : 1;
  constexpr int kPieces = apply_pieces<NB, TO>(), kPer = 8 * (int)sizeof(TO) / 16;   // pieces of a row block
  extern __shared__ __align__(16) unsigned char smem[];
  double* Q = reinterpret_cast<double*>(smem);   // [kRows][S]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint4* olds = reinterpret_cast<uint4*>(Q + kRows * S) + warp * kPieces * 32 + lane;   // [kPieces][32]
  const int steps = (P.C + 32 * warps - 1) / (32 * warps);
  const int64_t total = (int64_t)P.mats * steps;
  const int64_t x0 = share(total, gridDim.x, blockIdx.x), x1 = share(total, gridDim.x, blockIdx.x + 1);
  float keep = 0.f, step = 0.f;
  if (kMom) {
    const float lr = P.lr_dev ? MHC_LDG(P.lr_dev) : P.lr;
    keep = 1.f - lr * P.decay;
    step = -lr * P.scale;
  }
  Raw4<T> g[kAhead];
  Raw4<float> m[kAhead];
  auto place = [&](int64_t x, int& mat, int64_t& col) {
    mat = (int)(x / steps);
    col = (x - (int64_t)mat * steps) * (32 * warps) + warp * 32;
  };
  auto fetch_grad = [&](int mat, int64_t col, int k) {
    const int64_t c = col + (kVec ? 4 : 1) * (lane >> 2);
    load4<kVec>(g[k % kAhead], static_cast<const T*>(M.grad[mat]), P, 4 * k + (lane & 3), c, kGap);
  };
  auto fetch_mom = [&](int mat, int64_t col, int k) {
    const int64_t c = col + (kVec ? 4 : 1) * (lane >> 2);
    if (kMom) load4<kVec>(m[k % kAhead], static_cast<const float*>(M.mom[mat]), P, 4 * k + (lane & 3), c, kGap);
  };
  // The first rows of a step.  Momenta were written by this call's Gram kernel, so
  // the first read of them is behind the wait: that kernel had ended when this one
  // could start, but what it wrote is promised to be seen only from there on.
  // Gradients, parameters and the learning rate are older than the call.
  auto fetch_first = [&](int mat, int64_t col, bool wait) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch_grad(mat, col, k);
    if (kMom && wait) cudaGridDependencySynchronize();
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch_mom(mat, col, k);
  };
  int loaded = -1, mat;
  int64_t col;
  // from the end: what the Gram pass touched last is the likeliest to be in the L2
  place(x1 - 1, mat, col);
  if (kStage && x0 < x1) fetch_first(mat, col, true);
  for (int64_t x = x1 - 1; x >= x0; --x) {
    place(x, mat, col);
    TO* out = static_cast<TO*>(M.out[mat]);
    // this lane's eight columns of the result: half j at oc + kHalf * j, kGap apart
    const int64_t oc = col + (kVec ? 8 : 2) * (lane & 3);
    if constexpr (!kStage) fetch_first(mat, col, loaded < 0);
    if constexpr (kStage) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int r = 8 * (i / kPer) + (lane >> 2);
        const int64_t pc = oc + (i % kPer) * (16 / (int)sizeof(TO));
        const TO* src = out + r * P.rs + pc;
        // rows end on a multiple of four elements: of eight bf16 the second half may be beyond
        const int bytes = r < P.R && pc < P.C ? (int)min((int64_t)16, (P.C - pc) * (int64_t)sizeof(TO)) : 0;
        const uint32_t d = (uint32_t)__cvta_generic_to_shared(olds + i * 32);
        if constexpr (sizeof(TO) == 4) {
          const int n = bytes && MHC_CHK(src, bytes) ? bytes : 0;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
        } else {   // eight-byte pieces: the rows need not be 16-byte aligned
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n = bytes > 8 * h && MHC_CHK(src + 4 * h, 8) ? 8 : 0;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(d + 8 * h), "l"(src + 4 * h), "r"(n)
                         : "memory");
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if (mat != loaded) {   // the same for the whole CTA
      cudaGridDependencySynchronize();   // Q is ready when the iteration has ended
      __syncthreads();
      const double* q = P.q + (int64_t)mat * kRows * kRows;
      for (int e = threadIdx.x; e < kRows * kRows; e += blockDim.x) Q[e / kRows * S + e % kRows] = MHC_LD(q + e);
      __syncthreads();
      loaded = mat;
    }
    double acc[NB][4][2];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e][0] = acc[i][e][1] = 0.0;
    const double* a = Q + (lane >> 2) * S + (lane & 3);
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      float f[4];
      g[k % kAhead].unpack(f);
      if (kMom) {
        float m1[4];
        m[k % kAhead].unpack(m1);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = update_of(P, m1[j], f[j]);
      }
      if (k + kAhead < kK) {
        fetch_grad(mat, col, k + kAhead);
        fetch_mom(mat, col, k + kAhead);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const double q = a[8 * i * S + 4 * k];
#pragma unroll
        for (int e = 0; e < 4; ++e) dmma(acc[i][e], q, (double)f[e]);
      }
    }
    if constexpr (kStage) {
      if (x > x0) {
        int nmat;
        int64_t ncol;
        place(x - 1, nmat, ncol);
        fetch_first(nmat, ncol, false);
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    constexpr int kBatch = NB <= 3 && kVec ? NB : 1;   // row blocks whose parameters are loaded together
#pragma unroll
    for (int b = 0; b < NB; b += kBatch) {
      Raw4<TO> old[kBatch][2];
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (kStage && sizeof(TO) == 4)
            old[i][j].v = *reinterpret_cast<const float4*>(olds + (2 * (b + i) + j) * 32);
          else if constexpr (kStage)
            old[i][j].v = reinterpret_cast<const uint2*>(olds + (b + i) * 32)[j];
          else if constexpr (kMom)
            load4<kVec>(old[i][j], static_cast<const TO*>(out), P, 8 * (b + i) + (lane >> 2), oc + kHalf * j, kGap);
        }
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float o[4], p[4];
          if constexpr (kMom) old[i][j].unpack(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = (float)acc[b + i][e][j];
            o[e] = kMom ? fmaf(keep, p[e], step * v) : v;
          }
          store4<kVec>(out, P, 8 * (b + i) + (lane >> 2), oc + kHalf * j, o, kGap);
        }
    }
  }
}

}  // namespace ortho
}  // namespace mhc
