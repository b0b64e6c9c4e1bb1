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
// percent of a singular value near 1/500 of the norm).  The Gram product and
// the iteration therefore run in 64 bits, on the double-precision matrix
// instruction (8 x 8 x 4); only the application, which lifts nothing, is in 32.
#pragma once

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
constexpr int kNsThreads = 512;
constexpr int kNsWarps = kNsThreads / 32;

struct Mats {
  const void* grad[kMaxMats];
  float* mom[kMaxMats];      // NULL entries never: absent as a whole (orthogonalise only)
  void* out[kMaxMats];       // the orthogonalised matrix, or the parameter to update
};

struct Params {
  int R, C;                  // short and long side
  int64_t rs, cs;            // element (i, k) of the short x long view is at i * rs + k * cs
  int slices;                // Gram partial sums per matrix
  int chunks_per_slice;
  double* part;              // [L][slices][blocks][64]
  float* q;                  // [L][P][P], P = 8 * NB
  float momentum;            // the update's coefficients; unused when only orthogonalising
  int nesterov;
  float lr, decay, scale;
  const float* lr_dev;       // NULL, or the learning rate in device memory
  int steps;
  double eps;
  double coeffs[3 * kMaxSteps];
};

// 8-row blocks, rounded up to the sizes compiled (n = 1 .. 8 need 1 1 2 3 5 6 8 10).
inline int row_blocks(int R) {
  const int nb = (R + 7) / 8;
  return nb <= 3 ? nb : nb <= 5 ? 5 : nb <= 6 ? 6 : nb <= 8 ? 8 : 10;
}
constexpr int lower_blocks(int NB) { return NB * (NB + 1) / 2; }
// Columns of one staged chunk: about 16 to 24 KB a chunk.
constexpr int chunk_cols(int NB) { return NB <= 2 ? 256 : NB <= 5 ? 128 : 64; }
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

template <class T>
__device__ __forceinline__ float ld1(const T* p) {
  if constexpr (std::is_same_v<T, float>) return MHC_LD(p);
  else return bf16_bits_to_f32(MHC_LD(p));
}
template <class T>
__device__ __forceinline__ void ld4(const T* p, float (&f)[4]) {
  if constexpr (std::is_same_v<T, float>) {
    const float4 v = MHC_LD(reinterpret_cast<const float4*>(p));
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  } else {
    const uint2 v = MHC_LD(reinterpret_cast<const uint2*>(p));
    f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xFFFF0000u);
    f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xFFFF0000u);
  }
}
template <class T>
__device__ __forceinline__ void st1(T* p, float v) {
  if constexpr (std::is_same_v<T, float>) MHC_ST(p, v);
  else MHC_ST(p, f32_to_bf16_bits(v));
}

// momentum and the matrix that is orthogonalised, the same rounding in every
// kernel that forms them: m' = mu m + (1 - mu) g, u = mu m' + (1 - mu) g or m'.
__device__ __forceinline__ float new_momentum(float m, float g, float mu) { return fmaf(mu, m, (1.f - mu) * g); }
__device__ __forceinline__ float update_of(float m1, float g, float mu, int nesterov) {
  return nesterov ? fmaf(mu, m1, (1.f - mu) * g) : m1;
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

// Partial Gram products.  Grid (slices, matrices).  A CTA walks its chunks of
// columns through two shared-memory tiles (the next chunk's loads are in
// registers while the warps multiply this one), each warp taking its share of a
// chunk's columns.  With momentum the kernel also forms and writes the new
// momentum; only this kernel's thread that loads an element writes it.
template <int NB, class T, bool kMom, bool kVec>
__global__ void __launch_bounds__(kThreads) gram_kernel(const __grid_constant__ Params P,
                                                        const __grid_constant__ Mats M) {
  constexpr int kRows = 8 * NB, KC = chunk_cols(NB), kStride = KC + 4;
  constexpr int kRoles = gram_roles(NB), kColWarps = kWarps / kRoles, kWarpCols = KC / kColWarps;
  constexpr int kPer = kRows * (KC / 4) / kThreads;   // 4-element pieces of a chunk per thread
  static_assert(kRows * (KC / 4) % kThreads == 0 && kWarpCols % 4 == 0, "chunk split");
  extern __shared__ __align__(16) unsigned char smem[];
  float* tile = reinterpret_cast<float*>(smem);       // two of [kRows][kStride]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mat = blockIdx.y;
  const T* g = static_cast<const T*>(M.grad[mat]);
  float* mom = kMom ? M.mom[mat] : nullptr;
  const int chunks = (P.C + KC - 1) / KC;
  const int c0 = blockIdx.x * P.chunks_per_slice, c1 = min(c0 + P.chunks_per_slice, chunks);

  float reg[kPer][4];
  auto fetch = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = threadIdx.x + i * kThreads, r = e / (KC / 4), c = chunk * KC + (e % (KC / 4)) * 4;
      if (kVec && r < P.R && c < P.C) {   // C is a multiple of 4 here
        const int64_t o = r * P.rs + c;
        ld4(g + o, reg[i]);
        if (kMom) {
          float m[4];
          ld4(mom + o, m);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            m[j] = new_momentum(m[j], reg[i][j], P.momentum);
            reg[i][j] = update_of(m[j], reg[i][j], P.momentum, P.nesterov);
          }
          MHC_ST(reinterpret_cast<float4*>(mom + o), make_float4(m[0], m[1], m[2], m[3]));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          reg[i][j] = 0.f;
          if (!kVec && r < P.R && c + j < P.C) {
            const int64_t o = r * P.rs + (c + j) * P.cs;
            const float gv = ld1(g + o);
            reg[i][j] = gv;
            if (kMom) {
              const float m1 = new_momentum(MHC_LD(mom + o), gv, P.momentum);
              reg[i][j] = update_of(m1, gv, P.momentum, P.nesterov);
              MHC_ST(mom + o, m1);
            }
          }
        }
      }
    }
  };
  auto stage = [&](float* dst) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = threadIdx.x + i * kThreads, r = e / (KC / 4), c = (e % (KC / 4)) * 4;
      *reinterpret_cast<float4*>(dst + r * kStride + c) = make_float4(reg[i][0], reg[i][1], reg[i][2], reg[i][3]);
    }
  };

  double* sums = reinterpret_cast<double*>(smem) + (size_t)(warp / kRoles) * lower_blocks(NB) * 64;
  // One role's whole walk, so that a warp holds its own accumulators only; both
  // roles pass the same number of barriers.
  auto walk = [&](auto gram) {
    gram.clear();
    const int col0 = (warp / kRoles) * kWarpCols;
    if (c0 < c1) {
      fetch(c0);
      stage(tile);
      __syncthreads();
      for (int c = c0; c < c1; ++c) {
        float* cur = tile + ((c - c0) & 1) * kRows * kStride;
        float* nxt = tile + ((c - c0 + 1) & 1) * kRows * kStride;
        if (c + 1 < c1) fetch(c + 1);
        gram.run(cur + col0, kStride, kWarpCols, lane);
        if (c + 1 < c1) stage(nxt);   // last read in the round before, ended by its barrier
        __syncthreads();
      }
    }
    gram.store(sums, lane);
  };
  if constexpr (kRoles == 1) {
    walk(Gram<0, NB>{});
  } else {
    if ((warp & 1) == 0)
      walk(Gram<0, role_split(NB)>{});
    else
      walk(Gram<role_split(NB), NB>{});
  }
  // sum over the column warps in warp order
  __syncthreads();
  double* dst = P.part + ((int64_t)mat * P.slices + blockIdx.x) * (lower_blocks(NB) * 64);
  for (int i = threadIdx.x; i < lower_blocks(NB) * 64; i += kThreads) {
    double v = 0.0;
#pragma unroll
    for (int w = 0; w < kColWarps; ++w) v += reinterpret_cast<const double*>(smem)[w * lower_blocks(NB) * 64 + i];
    MHC_ST(dst + i, v);
  }
}

// Row stride of an R x R matrix of doubles in shared memory: 4 or 12 modulo 16,
// so that the four rows a half warp's fragment load touches fall into different banks.
constexpr int ns_stride(int NB) { return 8 * NB + 4; }
template <int NB>
constexpr size_t ns_smem() {
  return 4 * (size_t)(8 * NB) * ns_stride(NB) * sizeof(double);
}

// Lower-triangle blocks of X Y for commuting symmetric X, Y (their product is
// symmetric and Y's rows serve as its columns); a warp's blocks in registers.
template <int NB>
struct Product {
  static constexpr int kPerWarp = (lower_blocks(NB) + kNsWarps - 1) / kNsWarps;
  double acc[kPerWarp][2];
  __device__ __forceinline__ static void block(int x, int& i, int& j) {
    i = 0;
    while (lower_blocks(i + 1) <= x) ++i;
    j = x - lower_blocks(i);
  }
  __device__ __forceinline__ void run(const double* X, const double* Y, int warp, int lane) {
    constexpr int S = ns_stride(NB);
#pragma unroll
    for (int t = 0; t < kPerWarp; ++t) {
      const int x = warp + t * kNsWarps;
      acc[t][0] = acc[t][1] = 0.0;
      if (x < lower_blocks(NB)) {
        int i, j;
        block(x, i, j);
        const double* a = X + (8 * i + (lane >> 2)) * S + (lane & 3);
        const double* b = Y + (8 * j + (lane >> 2)) * S + (lane & 3);
#pragma unroll
        for (int k = 0; k < 8 * NB; k += 4) dmma(acc[t], a[k], b[k]);
      }
    }
  }
  // f(row, col, value) for each element of the lower blocks, and its mirror
  template <class F>
  __device__ __forceinline__ void each(int warp, int lane, F f) const {
#pragma unroll
    for (int t = 0; t < kPerWarp; ++t) {
      const int x = warp + t * kNsWarps;
      if (x < lower_blocks(NB)) {
        int i, j;
        block(x, i, j);
        const int r = 8 * i + (lane >> 2), c = 8 * j + 2 * (lane & 3);
        f(r, c, acc[t][0]);
        f(r, c + 1, acc[t][1]);
      }
    }
  }
};

// The iteration on the small matrices, one CTA per matrix.
template <int NB>
__global__ void __launch_bounds__(kNsThreads) iterate_kernel(const __grid_constant__ Params P) {
  constexpr int kRows = 8 * NB, S = ns_stride(NB), kB = lower_blocks(NB);
  extern __shared__ __align__(16) unsigned char smem[];
  double* A = reinterpret_cast<double*>(smem);
  double* Mk = A + kRows * S;
  double* W = Mk + kRows * S;
  double* Q = W + kRows * S;
  __shared__ double inv_norm;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const double* part = P.part + (int64_t)blockIdx.x * P.slices * (kB * 64);
  auto both = [&](double* X, int r, int c, double v) {
    X[r * S + c] = v;
    X[c * S + r] = v;
  };
  for (int e = threadIdx.x; e < kB * 64; e += kNsThreads) {
    double v = 0.0;
    for (int s = 0; s < P.slices; ++s) v += MHC_LD(part + (int64_t)s * (kB * 64) + e);
    int i, j;
    Product<NB>::block(e / 64, i, j);
    const int l = (e & 63) >> 1;
    both(A, 8 * i + (l >> 2), 8 * j + 2 * (l & 3) + (e & 1), v);
  }
  __syncthreads();
  if (warp == 0) {
    double tr = 0.0;
    for (int i = lane; i < kRows; i += 32) tr += A[i * S + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tr += __shfl_xor_sync(0xffffffffu, tr, o);
    if (lane == 0) inv_norm = 1.0 / (sqrt(tr) + P.eps);
  }
  __syncthreads();
  const double inv = inv_norm;
  for (int e = threadIdx.x; e < kRows * kRows; e += kNsThreads) A[(e / kRows) * S + e % kRows] *= inv * inv;
  __syncthreads();
  Product<NB> p, p2;
  for (int k = 0; k < P.steps; ++k) {
    const double a = P.coeffs[3 * k], b = P.coeffs[3 * k + 1], c = P.coeffs[3 * k + 2];
    p.run(A, A, warp, lane);
    p.each(warp, lane, [&](int r, int col, double v) {
      v = (r == col ? a : 0.0) + b * A[r * S + col] + c * v;
      both(Mk, r, col, v);
      if (k == 0) both(Q, r, col, v);
    });
    __syncthreads();
    const bool more = k + 1 < P.steps;
    if (more) p.run(A, Mk, warp, lane);
    if (k > 0) p2.run(Q, Mk, warp, lane);
    __syncthreads();
    if (more) p.each(warp, lane, [&](int r, int col, double v) { both(W, r, col, v); });
    if (k > 0) p2.each(warp, lane, [&](int r, int col, double v) { both(Q, r, col, v); });
    __syncthreads();
    if (more) {
      p.run(W, Mk, warp, lane);
      p.each(warp, lane, [&](int r, int col, double v) { both(A, r, col, v); });
      __syncthreads();
    }
  }
  float* q = P.q + (int64_t)blockIdx.x * kRows * kRows;
  for (int e = threadIdx.x; e < kRows * kRows; e += kNsThreads) {
    const int r = e / kRows, c = e % kRows;
    const bool in = r < P.R && c < P.R;   // beyond the matrix: the a_k on the padded diagonal
    MHC_ST(q + e, in ? (float)(Q[r * S + c] * inv) : 0.f);
  }
}

// O = Q U on two columns per thread (kVec: neighbours, else kThreads apart),
// and what is made of it: the output, or the parameter's update
//   p' = (1 - lr decay) p - lr scale O.
constexpr int apply_threads(int NB) { return NB > 6 ? 128 : 256; }
template <int NB, class T, class TO, bool kMom, bool kVec>
__global__ void __launch_bounds__(apply_threads(NB)) apply_kernel(const __grid_constant__ Params P,
                                                                  const __grid_constant__ Mats M) {
  constexpr int kRows = 8 * NB, kT = apply_threads(NB);
  extern __shared__ __align__(16) unsigned char smem[];
  float2* q = reinterpret_cast<float2*>(smem);   // [kRows][kRows], each value twice (packed products)
  const int mat = blockIdx.y;
  const T* g = static_cast<const T*>(M.grad[mat]);
  const float* mom = kMom ? M.mom[mat] : nullptr;
  TO* out = static_cast<TO*>(M.out[mat]);
  const float* qs = P.q + (int64_t)mat * kRows * kRows;
  const int64_t base = (int64_t)blockIdx.x * (2 * kT);
  const int64_t ca = kVec ? base + 2 * threadIdx.x : base + threadIdx.x, cb = kVec ? ca + 1 : ca + kT;
  float2 u[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    u[r] = make_float2(0.f, 0.f);
    if (r < P.R) {
      float gv[2] = {0.f, 0.f}, m[2] = {0.f, 0.f};
      if constexpr (kVec) {
        if (ca < P.C) {
          const int64_t o = r * P.rs + ca;
          if constexpr (std::is_same_v<T, float>) {
            const float2 v = MHC_LDG(reinterpret_cast<const float2*>(g + o));
            gv[0] = v.x, gv[1] = v.y;
          } else {
            const uint32_t v = MHC_LDG(reinterpret_cast<const uint32_t*>(g + o));
            gv[0] = __uint_as_float(v << 16), gv[1] = __uint_as_float(v & 0xFFFF0000u);
          }
          if (kMom) {
            const float2 v = MHC_LDG(reinterpret_cast<const float2*>(mom + o));
            m[0] = v.x, m[1] = v.y;
          }
        }
      } else {
        const int64_t oa = r * P.rs + ca * P.cs, ob = r * P.rs + cb * P.cs;
        if (ca < P.C) gv[0] = ld1(g + oa);
        if (cb < P.C) gv[1] = ld1(g + ob);
        if (kMom) {
          if (ca < P.C) m[0] = MHC_LD(mom + oa);
          if (cb < P.C) m[1] = MHC_LD(mom + ob);
        }
      }
      u[r] = kMom ? make_float2(update_of(m[0], gv[0], P.momentum, P.nesterov),
                                update_of(m[1], gv[1], P.momentum, P.nesterov))
                  : make_float2(gv[0], gv[1]);
    }
  }
  for (int e = threadIdx.x; e < kRows * kRows; e += kT) {
    const float v = MHC_LDG(qs + e);
    q[e] = make_float2(v, v);
  }
  __syncthreads();
  float keep = 0.f, step = 0.f;
  if (kMom) {
    const float lr = P.lr_dev ? MHC_LDG(P.lr_dev) : P.lr;
    keep = 1.f - lr * P.decay;
    step = -lr * P.scale;
  }
  for (int r = 0; r < P.R; ++r) {
    const float4* qr = reinterpret_cast<const float4*>(q + r * kRows);
    float2 o0 = make_float2(0.f, 0.f), o1 = o0;
#pragma unroll
    for (int k = 0; k < kRows; k += 2) {
      const float4 w = qr[k / 2];
      o0 = __ffma2_rn(make_float2(w.x, w.y), u[k], o0);
      o1 = __ffma2_rn(make_float2(w.z, w.w), u[k + 1], o1);
    }
    float v0 = o0.x + o1.x, v1 = o0.y + o1.y;
    if constexpr (kVec) {
      if (ca < P.C) {
        const int64_t o = r * P.rs + ca;
        if constexpr (std::is_same_v<TO, float>) {
          if (kMom) {
            const float2 p = MHC_LD(reinterpret_cast<const float2*>(out + o));
            v0 = fmaf(keep, p.x, step * v0);
            v1 = fmaf(keep, p.y, step * v1);
          }
          MHC_ST(reinterpret_cast<float2*>(out + o), make_float2(v0, v1));
        } else {
          if (kMom) {
            const uint32_t p = MHC_LD(reinterpret_cast<const uint32_t*>(out + o));
            v0 = fmaf(keep, __uint_as_float(p << 16), step * v0);
            v1 = fmaf(keep, __uint_as_float(p & 0xFFFF0000u), step * v1);
          }
          MHC_ST(reinterpret_cast<uint32_t*>(out + o), pack_bf16x2(v0, v1));
        }
      }
    } else {
      const int64_t oa = r * P.rs + ca * P.cs, ob = r * P.rs + cb * P.cs;
      if (ca < P.C) st1(out + oa, kMom ? fmaf(keep, ld1(out + oa), step * v0) : v0);
      if (cb < P.C) st1(out + ob, kMom ? fmaf(keep, ld1(out + ob), step * v1) : v1);
    }
  }
}

}  // namespace ortho
}  // namespace mhc
