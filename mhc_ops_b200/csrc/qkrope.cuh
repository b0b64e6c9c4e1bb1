// Norms of queries and keys for each head with the rotary position rotation in
// the same pass, forward and backward: what stands between the projection of
// h_in and the attention of a hyper-connection block's sublayer.
//
// Per head row x [d] of token t at position p (s = row_scale[t] or 1, w the
// norm's weight or ones, f = inv_freq [rot/2]):
//   z = s x ; r = (mean z^2 + eps)^-1/2 ; a = r z w ; y = Rot(p f) a
// Rot turns the pairs of the first rot elements ((i, i + rot/2), or
// (2i, 2i + 1) when interleaved) by the angles p f_i; the rest passes.  A value
// row is only scaled: v_out = s v.  With s = h_in_rstd (mhc_fwd_ex) and the
// sublayer norm's weight folded into the projection, RMSNorm(h_in) is never
// written.  Backward, da = Rot^T dy:
//   dw += r z da ; dn = w da ; dx = s r (dn - n m), n = r z, m = mean(dn n)
//   ds = eps r^3 sum(dn x) over the normed heads + sum(v dv_out)
// (sum(x . dz), the direct form of ds, cancels down to the eps term; the line
// above is what is left, without a division by s.)
//
// The angle is p f / 2pi in 64 bits, reduced to half a turn there, then one
// sincospi in 32 bits: exact to 32 bits at any position below 2^31, without a
// table that would have to be as long as the longest sequence.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

#undef MHC_FILE_ID
#define MHC_FILE_ID 8   // debug-bounds site ids: 8 * 100000 + line

namespace mhc {
namespace rope {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxD = 1024;       // widest head
constexpr int kFinCols = 32;      // columns of one finalize CTA

// A [B, S, H, d] tensor with unit stride along d; strides in elements.
struct View {
  const void* p;
  int64_t sb, ss, sh;
};

struct Params {
  View q, k, v;             // inputs (v.p NULL: no values)
  View dq, dk, dv;          // backward: upstream gradients
  View oq, ok, ov;          // outputs (forward) / input gradients (backward); written
  const float* wq;          // [d] or NULL
  const float* wk;
  const float* inv_freq;    // [rot / 2]
  const void* pos;          // NULL: the token's index in its sequence
  const float* row_scale;   // [T] or NULL
  float* d_row_scale;       // backward, [T] or NULL
  float* dw_part;           // backward, [grid][2][d] or NULL
  int64_t pos_sb, pos_ss;
  int64_t T;
  int S;
  int pos64;
  int Hq, Hk, Hv;
  int d, rot;
  int G, gshift;            // vector kernels: lanes per head row, a power of two, and its logarithm
  int parts;                // warps that share a token's heads (1, 2, 4 or 8)
  float eps;
};

__device__ __forceinline__ float to_f32(uint16_t v, __nv_bfloat16*) { return bf16_bits_to_f32(v); }

template <class T>
__device__ __forceinline__ float load1(const T* p) {
  if constexpr (std::is_same_v<T, float>) return MHC_LDG(p);
  if constexpr (std::is_same_v<T, __half>)
    return __half2float(__ushort_as_half(MHC_LDG(reinterpret_cast<const unsigned short*>(p))));
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    return bf16_bits_to_f32(MHC_LDG(reinterpret_cast<const unsigned short*>(p)));
}
template <class T>
__device__ __forceinline__ void store1(T* p, float v) {
  if constexpr (std::is_same_v<T, float>) MHC_ST(p, v);
  if constexpr (std::is_same_v<T, __half>)
    MHC_ST(reinterpret_cast<unsigned short*>(p), __half_as_ushort(__float2half_rn(v)));
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    MHC_ST(reinterpret_cast<unsigned short*>(p), f32_to_bf16_bits(v));
}

// Eight consecutive elements as they lie in memory (one or two 16-byte words).
template <class T>
struct Raw8 {
  static constexpr int kWords = sizeof(T) * 8 / 16;
  uint4 w[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = MHC_LDG(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void unpack(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (std::is_same_v<T, float>) f[4 * i + j] = __uint_as_float(u[j]);
        if constexpr (std::is_same_v<T, __half>) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
          f[2 * j] = v.x;
          f[2 * j + 1] = v.y;
        }
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
          f[2 * j] = __uint_as_float(u[j] << 16);
          f[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
        }
      }
    }
  }
};

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(a, b);
  }
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if constexpr (std::is_same_v<T, float>) {
    MHC_ST(reinterpret_cast<uint4*>(p), make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                                   __float_as_uint(f[3])));
    MHC_ST(reinterpret_cast<uint4*>(p) + 1, make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]),
                                                       __float_as_uint(f[6]), __float_as_uint(f[7])));
  } else {
    MHC_ST(reinterpret_cast<uint4*>(p),
           make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7])));
  }
}

__device__ __forceinline__ int64_t position(const Params& P, int b, int s) {
  if (!P.pos) return s;
  const int64_t i = b * P.pos_sb + s * P.pos_ss;
  if (P.pos64) return MHC_LDG(reinterpret_cast<const long long*>(P.pos) + i);
  return MHC_LDG(reinterpret_cast<const int*>(P.pos) + i);
}

// cos and sin of pos * f; see the head of this file.
__device__ __forceinline__ void turn(int64_t pos, float f, float& c, float& s) {
  double rev = (double)pos * ((double)f * 0.15915494309189533577);
  rev -= rint(rev);
  sincospif(2.0f * (float)rev, &s, &c);
}

// The two 8-element chunks of unit u of a head row (d / 16 units).  Half-split
// pairs: a rotated unit holds 8 elements of either half, so that every pair is
// in one lane; the passing tail and interleaved rows go 16 by 16.  In every
// case the angles a unit needs are 8u .. 8u + 7 (those past rot / 2 are zero).
template <bool kInter>
__device__ __forceinline__ void unit_offsets(int u, int rot, int& a, int& b) {
  if (!kInter && u < rot / 16) {
    a = 8 * u;
    b = rot / 2 + 8 * u;
  } else {
    a = 16 * u;
    b = 16 * u + 8;
  }
}

// Rot (dir = 1) or its transpose (dir = -1: sn holds the negated sines) on a unit.
template <bool kInter>
__device__ __forceinline__ void rotate(float (&a)[8], float (&b)[8], const float (&cs)[8], const float (&sn)[8]) {
  if constexpr (kInter) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a0 = a[2 * j], a1 = a[2 * j + 1], b0 = b[2 * j], b1 = b[2 * j + 1];
      a[2 * j] = a0 * cs[j] - a1 * sn[j];
      a[2 * j + 1] = a0 * sn[j] + a1 * cs[j];
      b[2 * j] = b0 * cs[4 + j] - b1 * sn[4 + j];
      b[2 * j + 1] = b0 * sn[4 + j] + b1 * cs[4 + j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = a[j], y = b[j];
      a[j] = x * cs[j] - y * sn[j];
      b[j] = x * sn[j] + y * cs[j];
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int G) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < G) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <class T>
__device__ __forceinline__ const T* row(const View& v, int b, int s, int h) {
  return static_cast<const T*>(v.p) + (b * v.sb + s * v.ss + h * v.sh);
}

// Forward, 16-byte vectors.  A warp works on 32 / G heads of one token at a
// time, G lanes a head with 16 elements each; its heads are the token's query,
// key and value heads in one list, of which `parts` warps of the CTA take every
// parts-th group.  The token's angles are computed once per warp.
template <class T, bool kInter>
__global__ void __launch_bounds__(kThreads) fwd_vec_kernel(const Params P) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = P.G, u = lane & (G - 1), hsub = lane >> P.gshift, hpw = 32 >> P.gshift;
  const bool act = 16 * u < P.d;
  int oa, ob;
  unit_offsets<kInter>(u, P.rot, oa, ob);
  float wq[2][8], wk[2][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    wq[0][j] = act && P.wq ? MHC_LDG(P.wq + oa + j) : 1.f;
    wq[1][j] = act && P.wq ? MHC_LDG(P.wq + ob + j) : 1.f;
    wk[0][j] = act && P.wk ? MHC_LDG(P.wk + oa + j) : 1.f;
    wk[1][j] = act && P.wk ? MHC_LDG(P.wk + ob + j) : 1.f;
  }
  const int H = P.Hq + P.Hk + P.Hv, Hqk = P.Hq + P.Hk;
  const float inv_d = 1.f / (float)P.d;
  const int part = warp & (P.parts - 1);
  const int tok_per_cta = kWarps / P.parts;
  for (int64_t t = (int64_t)blockIdx.x * tok_per_cta + warp / P.parts; t < P.T;
       t += (int64_t)gridDim.x * tok_per_cta) {
    const int b = (int)((uint32_t)t / (uint32_t)P.S), s = (int)((uint32_t)t - (uint32_t)b * (uint32_t)P.S);
    const float sc = P.row_scale ? MHC_LDG(P.row_scale + t) : 1.f;
    const int64_t pos = position(P, b, s);
    auto locate = [&](int h, const T*& src, T*& dst) {
      const bool isq = h < P.Hq, isk = !isq && h < Hqk;
      const View& in = isq ? P.q : isk ? P.k : P.v;
      const View& out = isq ? P.oq : isk ? P.ok : P.ov;
      const int hh = isq ? h : isk ? h - P.Hq : h - Hqk;
      src = row<T>(in, b, s, hh);
      dst = const_cast<T*>(row<T>(out, b, s, hh));
    };
    Raw8<T> ra, rb;
    const T* src;
    T* dst;
    int h = part * hpw + hsub;
    ra.zero();
    rb.zero();
    if (h < H && act) {
      locate(h, src, dst);
      ra.load(src + oa);
      rb.load(src + ob);
    }
    float cs[8], sn[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      cs[j] = 1.f;
      sn[j] = 0.f;
      if (8 * u + j < P.rot / 2) turn(pos, MHC_LDG(P.inv_freq + 8 * u + j), cs[j], sn[j]);
    }
    for (int h0 = part * hpw; h0 < H; h0 += P.parts * hpw) {
      const int hn = h + P.parts * hpw;
      Raw8<T> na, nb;
      const T* nsrc;
      T* ndst = nullptr;
      na.zero();
      nb.zero();
      if (hn < H && act) {   // the next group's loads run during this one's arithmetic
        locate(hn, nsrc, ndst);
        na.load(nsrc + oa);
        nb.load(nsrc + ob);
      }
      float a[8], c[8];
      ra.unpack(a);
      rb.unpack(c);
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] *= sc;
        c[j] *= sc;
        sq = fmaf(a[j], a[j], sq);
        sq = fmaf(c[j], c[j], sq);
      }
      sq = group_sum(sq, G);
      if (h < Hqk) {
        const float r = __frsqrt_rn(fmaf(sq, inv_d, P.eps));
        const bool isq = h < P.Hq;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a[j] = a[j] * r * (isq ? wq[0][j] : wk[0][j]);
          c[j] = c[j] * r * (isq ? wq[1][j] : wk[1][j]);
        }
        rotate<kInter>(a, c, cs, sn);
      }
      if (h < H && act) {
        store8(dst + oa, a);
        store8(dst + ob, c);
      }
      ra = na;
      rb = nb;
      dst = ndst;
      h = hn;
    }
  }
}

// Sums of one warp's lanes of equal unit, over the head groups of the warp.
__device__ __forceinline__ float across_heads(float v, int G) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o >= G) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Backward, 16-byte vectors, the forward's split.  Each lane keeps the weight
// gradients of its 16 elements for queries and keys over all its tokens; the
// CTA's warps are added in warp order and the CTA's row written for the
// finalize kernel, so repeated calls give the same bits.
template <class T, bool kInter>
__global__ void __launch_bounds__(kThreads) bwd_vec_kernel(const Params P) {
  __shared__ float sds[kWarps];
  __shared__ float sdw[kWarps][2][512];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = P.G, u = lane & (G - 1), hsub = lane >> P.gshift, hpw = 32 >> P.gshift;
  const bool act = 16 * u < P.d;
  int oa, ob;
  unit_offsets<kInter>(u, P.rot, oa, ob);
  float wq[2][8], wk[2][8], gq[2][8], gk[2][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    wq[0][j] = act && P.wq ? MHC_LDG(P.wq + oa + j) : 1.f;
    wq[1][j] = act && P.wq ? MHC_LDG(P.wq + ob + j) : 1.f;
    wk[0][j] = act && P.wk ? MHC_LDG(P.wk + oa + j) : 1.f;
    wk[1][j] = act && P.wk ? MHC_LDG(P.wk + ob + j) : 1.f;
    gq[0][j] = gq[1][j] = gk[0][j] = gk[1][j] = 0.f;
  }
  const int H = P.Hq + P.Hk + P.Hv, Hqk = P.Hq + P.Hk;
  const float inv_d = 1.f / (float)P.d;
  const int part = warp & (P.parts - 1);
  const int tok_per_cta = kWarps / P.parts;
  // every warp makes the same number of rounds: the row factor's sum over a
  // token's warps needs a barrier per round
  for (int64_t t0 = (int64_t)blockIdx.x * tok_per_cta; t0 < P.T; t0 += (int64_t)gridDim.x * tok_per_cta) {
    const int64_t t = t0 + warp / P.parts;
    float ds = 0.f;
    if (t < P.T) {
      const int b = (int)((uint32_t)t / (uint32_t)P.S), s = (int)((uint32_t)t - (uint32_t)b * (uint32_t)P.S);
      const float sc = P.row_scale ? MHC_LDG(P.row_scale + t) : 1.f;
      const int64_t pos = position(P, b, s);
      Raw8<T> xa, xb, ya, yb;
      auto fetch = [&](int h, Raw8<T>& xa, Raw8<T>& xb, Raw8<T>& ya, Raw8<T>& yb) {
        xa.zero();
        xb.zero();
        ya.zero();
        yb.zero();
        if (h < H && act) {
          const bool isq = h < P.Hq, isk = !isq && h < Hqk;
          const int hh = isq ? h : isk ? h - P.Hq : h - Hqk;
          const T* x = row<T>(isq ? P.q : isk ? P.k : P.v, b, s, hh);
          const T* y = row<T>(isq ? P.dq : isk ? P.dk : P.dv, b, s, hh);
          xa.load(x + oa);
          xb.load(x + ob);
          ya.load(y + oa);
          yb.load(y + ob);
        }
      };
      int h = part * hpw + hsub;
      fetch(h, xa, xb, ya, yb);
      float cs[8], sn[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs[j] = 1.f;
        sn[j] = 0.f;
        if (8 * u + j < P.rot / 2) {
          turn(pos, MHC_LDG(P.inv_freq + 8 * u + j), cs[j], sn[j]);
          sn[j] = -sn[j];   // the transpose
        }
      }
      for (int h0 = part * hpw; h0 < H; h0 += P.parts * hpw) {
        Raw8<T> nxa, nxb, nya, nyb;
        const int hn = h + P.parts * hpw;
        fetch(hn, nxa, nxb, nya, nyb);
        float x0[8], x1[8], y0[8], y1[8];
        xa.unpack(x0);
        xb.unpack(x1);
        ya.unpack(y0);
        yb.unpack(y1);
        const bool isq = h < P.Hq, isk = !isq && h < Hqk;
        if (isq || isk) rotate<kInter>(y0, y1, cs, sn);   // da
        float sq = 0.f, dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float za = x0[j] * sc, zb = x1[j] * sc;
          sq = fmaf(za, za, sq);
          sq = fmaf(zb, zb, sq);
          const float wa = isq ? wq[0][j] : isk ? wk[0][j] : 1.f, wb = isq ? wq[1][j] : isk ? wk[1][j] : 1.f;
          dot = fmaf(y0[j] * wa, x0[j], dot);
          dot = fmaf(y1[j] * wb, x1[j], dot);
        }
        sq = group_sum(sq, G);
        dot = group_sum(dot, G);   // sum(dn x); sum(v dv_out) on value rows
        float o0[8], o1[8];
        if (isq || isk) {
          const float r = __frsqrt_rn(fmaf(sq, inv_d, P.eps));
          const float sr = sc * r;
          const float m = sr * dot * inv_d;
          if (u == 0) ds += P.eps * r * r * r * dot;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float n0 = x0[j] * sr, n1 = x1[j] * sr;
            if (isq) {
              gq[0][j] = fmaf(n0, y0[j], gq[0][j]);
              gq[1][j] = fmaf(n1, y1[j], gq[1][j]);
            } else {
              gk[0][j] = fmaf(n0, y0[j], gk[0][j]);
              gk[1][j] = fmaf(n1, y1[j], gk[1][j]);
            }
            o0[j] = sr * (y0[j] * (isq ? wq[0][j] : wk[0][j]) - n0 * m);
            o1[j] = sr * (y1[j] * (isq ? wq[1][j] : wk[1][j]) - n1 * m);
          }
        } else {
          if (u == 0) ds += dot;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            o0[j] = sc * y0[j];
            o1[j] = sc * y1[j];
          }
        }
        if (h < H && act) {
          const int hh = isq ? h : isk ? h - P.Hq : h - Hqk;
          T* dst = const_cast<T*>(row<T>(isq ? P.oq : isk ? P.ok : P.ov, b, s, hh));
          store8(dst + oa, o0);
          store8(dst + ob, o1);
        }
        xa = nxa;
        xb = nxb;
        ya = nya;
        yb = nyb;
        h = hn;
      }
    }
    if (P.d_row_scale) {
      ds = warp_sum(ds);
      if (P.parts == 1) {
        if (lane == 0 && t < P.T) MHC_ST(P.d_row_scale + t, ds);
      } else {
        if (lane == 0) sds[warp] = ds;
        __syncthreads();
        if (part == 0 && lane == 0 && t < P.T) {
          float sum = 0.f;
          for (int i = 0; i < P.parts; ++i) sum += sds[warp + i];
          MHC_ST(P.d_row_scale + t, sum);
        }
        __syncthreads();
      }
    }
  }
  if (P.dw_part) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v[4] = {across_heads(gq[0][j], G), across_heads(gq[1][j], G), across_heads(gk[0][j], G),
                          across_heads(gk[1][j], G)};
      if (hsub == 0 && act) {
        sdw[warp][0][oa + j] = v[0];
        sdw[warp][0][ob + j] = v[1];
        sdw[warp][1][oa + j] = v[2];
        sdw[warp][1][ob + j] = v[3];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * P.d; i += kThreads) {
      const int side = i >= P.d, col = i - side * P.d;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += sdw[w][side][col];
      MHC_ST(P.dw_part + (int64_t)blockIdx.x * 2 * P.d + i, sum);
    }
  }
}

// Any head width, stride and alignment: a warp per head row, lane l the pairs
// l, l + 32, ... and the passing elements likewise.  Dynamic shared memory per
// warp: the token's cos and sin [rot/2] and, in the backward, the weight
// gradients [2][d] of the warp (a lane only ever touches its own columns).
template <class T, bool kInter>
__global__ void __launch_bounds__(kThreads) fwd_any_kernel(const Params P) {
  extern __shared__ float dyn[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = P.rot / 2;
  float* cs = dyn + warp * P.rot;
  float* sn = cs + half;
  const int H = P.Hq + P.Hk + P.Hv, Hqk = P.Hq + P.Hk;
  const float inv_d = 1.f / (float)P.d;
  const int part = warp & (P.parts - 1);
  const int tok_per_cta = kWarps / P.parts;
  for (int64_t t = (int64_t)blockIdx.x * tok_per_cta + warp / P.parts; t < P.T;
       t += (int64_t)gridDim.x * tok_per_cta) {
    const int b = (int)((uint32_t)t / (uint32_t)P.S), s = (int)((uint32_t)t - (uint32_t)b * (uint32_t)P.S);
    const float sc = P.row_scale ? MHC_LDG(P.row_scale + t) : 1.f;
    const int64_t pos = position(P, b, s);
    for (int i = lane; i < half; i += 32) turn(pos, MHC_LDG(P.inv_freq + i), cs[i], sn[i]);   // own lane's slots
    for (int h = part; h < H; h += P.parts) {
      const bool isq = h < P.Hq, isk = !isq && h < Hqk;
      const int hh = isq ? h : isk ? h - P.Hq : h - Hqk;
      const T* x = row<T>(isq ? P.q : isk ? P.k : P.v, b, s, hh);
      T* y = const_cast<T*>(row<T>(isq ? P.oq : isk ? P.ok : P.ov, b, s, hh));
      if (!isq && !isk) {
        for (int i = lane; i < P.d; i += 32) store1(y + i, load1(x + i) * sc);
        continue;
      }
      float sq = 0.f;
      for (int i = lane; i < P.d; i += 32) {
        const float z = load1(x + i) * sc;
        sq = fmaf(z, z, sq);
      }
      sq = warp_sum(sq);
      const float r = __frsqrt_rn(fmaf(sq, inv_d, P.eps));
      const float* w = isq ? P.wq : P.wk;
      for (int i = lane; i < half; i += 32) {
        const int ia = kInter ? 2 * i : i, ib = kInter ? 2 * i + 1 : i + half;
        const float a = load1(x + ia) * sc * r * (w ? MHC_LDG(w + ia) : 1.f);
        const float c = load1(x + ib) * sc * r * (w ? MHC_LDG(w + ib) : 1.f);
        store1(y + ia, a * cs[i] - c * sn[i]);
        store1(y + ib, a * sn[i] + c * cs[i]);
      }
      for (int i = P.rot + lane; i < P.d; i += 32)
        store1(y + i, load1(x + i) * sc * r * (w ? MHC_LDG(w + i) : 1.f));
    }
  }
}

template <class T, bool kInter>
__global__ void __launch_bounds__(kThreads) bwd_any_kernel(const Params P) {
  extern __shared__ float dyn[];
  __shared__ float sds[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = P.rot / 2;
  float* cs = dyn + warp * (P.rot + 2 * P.d);
  float* sn = cs + half;
  float* gw = dyn + warp * (P.rot + 2 * P.d) + P.rot;   // [2][d]
  for (int i = lane; i < 2 * P.d; i += 32) gw[i] = 0.f;
  __syncwarp();
  const int H = P.Hq + P.Hk + P.Hv, Hqk = P.Hq + P.Hk;
  const float inv_d = 1.f / (float)P.d;
  const int part = warp & (P.parts - 1);
  const int tok_per_cta = kWarps / P.parts;
  for (int64_t t0 = (int64_t)blockIdx.x * tok_per_cta; t0 < P.T; t0 += (int64_t)gridDim.x * tok_per_cta) {
    const int64_t t = t0 + warp / P.parts;
    float ds = 0.f;
    if (t < P.T) {
      const int b = (int)((uint32_t)t / (uint32_t)P.S), s = (int)((uint32_t)t - (uint32_t)b * (uint32_t)P.S);
      const float sc = P.row_scale ? MHC_LDG(P.row_scale + t) : 1.f;
      const int64_t pos = position(P, b, s);
      for (int i = lane; i < half; i += 32) turn(pos, MHC_LDG(P.inv_freq + i), cs[i], sn[i]);
      for (int h = part; h < H; h += P.parts) {
        const bool isq = h < P.Hq, isk = !isq && h < Hqk;
        const int hh = isq ? h : isk ? h - P.Hq : h - Hqk;
        const T* x = row<T>(isq ? P.q : isk ? P.k : P.v, b, s, hh);
        const T* dy = row<T>(isq ? P.dq : isk ? P.dk : P.dv, b, s, hh);
        T* dx = const_cast<T*>(row<T>(isq ? P.oq : isk ? P.ok : P.ov, b, s, hh));
        if (!isq && !isk) {
          for (int i = lane; i < P.d; i += 32) {
            const float g = load1(dy + i);
            ds = fmaf(load1(x + i), g, ds);
            store1(dx + i, g * sc);
          }
          continue;
        }
        const float* w = isq ? P.wq : P.wk;
        float* g = gw + (isq ? 0 : P.d);
        float sq = 0.f, dot = 0.f;
        for (int i = lane; i < P.d; i += 32) {
          const float z = load1(x + i) * sc;
          sq = fmaf(z, z, sq);
        }
        // da of a pair, dn = w da
        for (int i = lane; i < half; i += 32) {
          const int ia = kInter ? 2 * i : i, ib = kInter ? 2 * i + 1 : i + half;
          const float ya = load1(dy + ia), yb = load1(dy + ib);
          const float da = ya * cs[i] + yb * sn[i], db = yb * cs[i] - ya * sn[i];
          dot = fmaf(da * (w ? MHC_LDG(w + ia) : 1.f), load1(x + ia), dot);
          dot = fmaf(db * (w ? MHC_LDG(w + ib) : 1.f), load1(x + ib), dot);
        }
        for (int i = P.rot + lane; i < P.d; i += 32)
          dot = fmaf(load1(dy + i) * (w ? MHC_LDG(w + i) : 1.f), load1(x + i), dot);
        sq = warp_sum(sq);
        dot = warp_sum(dot);
        const float r = __frsqrt_rn(fmaf(sq, inv_d, P.eps));
        const float sr = sc * r;
        const float m = sr * dot * inv_d;
        if (lane == 0) ds += P.eps * r * r * r * dot;
        for (int i = lane; i < half; i += 32) {
          const int ia = kInter ? 2 * i : i, ib = kInter ? 2 * i + 1 : i + half;
          const float ya = load1(dy + ia), yb = load1(dy + ib);
          const float da = ya * cs[i] + yb * sn[i], db = yb * cs[i] - ya * sn[i];
          const float na = load1(x + ia) * sr, nb = load1(x + ib) * sr;
          g[ia] = fmaf(na, da, g[ia]);
          g[ib] = fmaf(nb, db, g[ib]);
          store1(dx + ia, sr * (da * (w ? MHC_LDG(w + ia) : 1.f) - na * m));
          store1(dx + ib, sr * (db * (w ? MHC_LDG(w + ib) : 1.f) - nb * m));
        }
        for (int i = P.rot + lane; i < P.d; i += 32) {
          const float da = load1(dy + i), n = load1(x + i) * sr;
          g[i] = fmaf(n, da, g[i]);
          store1(dx + i, sr * (da * (w ? MHC_LDG(w + i) : 1.f) - n * m));
        }
      }
    }
    if (P.d_row_scale) {
      ds = warp_sum(ds);
      if (lane == 0) sds[warp] = ds;
      __syncthreads();
      if (part == 0 && lane == 0 && t < P.T) {
        float sum = 0.f;
        for (int i = 0; i < P.parts; ++i) sum += sds[warp + i];
        MHC_ST(P.d_row_scale + t, sum);
      }
      __syncthreads();
    }
  }
  __syncthreads();
  if (P.dw_part)
    for (int i = threadIdx.x; i < 2 * P.d; i += kThreads) {
      float sum = 0.f;
      for (int w = 0; w < kWarps; ++w) sum += dyn[w * (P.rot + 2 * P.d) + P.rot + i];
      MHC_ST(P.dw_part + (int64_t)blockIdx.x * 2 * P.d + i, sum);
    }
}

// Weight gradients: the CTAs' rows [parts][2 d] added in a fixed order, 32
// columns a CTA, every warp an eighth of the rows.
__global__ void __launch_bounds__(kThreads) bwd_weights_kernel(const float* __restrict__ part, int rows, int d,
                                                               float* __restrict__ dwq, float* __restrict__ dwk) {
  __shared__ float acc[kWarps][kFinCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * kFinCols + lane;
  float sum = 0.f;
  if (col < 2 * d)
    for (int r = warp; r < rows; r += kWarps) sum += MHC_LDG(part + (int64_t)r * 2 * d + col);
  acc[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && col < 2 * d) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += acc[w][lane];
    if (col < d) {
      if (dwq) MHC_ST(dwq + col, v);
    } else if (dwk) {
      MHC_ST(dwk + col - d, v);
    }
  }
}

}  // namespace rope
}  // namespace mhc
