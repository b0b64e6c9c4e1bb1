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
  __device__ __forceinline__ void unpack(float2 (&f)[4]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
      if constexpr (std::is_same_v<T, float>) {
        f[2 * i] = make_float2(__uint_as_float(u[0]), __uint_as_float(u[1]));
        f[2 * i + 1] = make_float2(__uint_as_float(u[2]), __uint_as_float(u[3]));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (std::is_same_v<T, __half>)
            f[j] = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
          else
            f[j] = make_float2(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xFFFF0000u));
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
__device__ __forceinline__ void store8(T* p, const float2 (&f)[4]) {
  if constexpr (std::is_same_v<T, float>) {
    MHC_ST(reinterpret_cast<float4*>(p), make_float4(f[0].x, f[0].y, f[1].x, f[1].y));
    MHC_ST(reinterpret_cast<float4*>(p) + 1, make_float4(f[2].x, f[2].y, f[3].x, f[3].y));
  } else {
    MHC_ST(reinterpret_cast<uint4*>(p), make_uint4(pack2<T>(f[0].x, f[0].y), pack2<T>(f[1].x, f[1].y),
                                                   pack2<T>(f[2].x, f[2].y), pack2<T>(f[3].x, f[3].y)));
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

// Two fp32 operations an instruction; each half rounds as the scalar one does.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 swapped(float2 v) { return make_float2(v.y, v.x); }

// A turn of the pairs of a unit as x -> P x + Q x', x' the other element of
// the pair: half-split pairs lie in the two chunks, interleaved ones side by side.
struct Turn {
  float2 pa[4], qa[4], pb[4], qb[4];
};
template <bool kInter>
__device__ __forceinline__ void apply_turn(const Turn& t, const float2 (&a)[4], const float2 (&b)[4], float2 (&ya)[4],
                                           float2 (&yb)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (kInter) {
      ya[j] = fma2(swapped(a[j]), t.qa[j], mul2(a[j], t.pa[j]));
      yb[j] = fma2(swapped(b[j]), t.qb[j], mul2(b[j], t.pb[j]));
    } else {
      ya[j] = fma2(b[j], t.qa[j], mul2(a[j], t.pa[j]));
      yb[j] = fma2(a[j], t.qb[j], mul2(b[j], t.pb[j]));
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

// What a lane of the vector kernels works on: G lanes a head row with 16
// elements each, 32 / G head rows of one token and one side (queries, keys or
// values) at a time.
struct Lane {
  int G, u, hsub, hpw, oa, ob;
  bool act;
  int ng[3];   // head groups of each side
};
template <bool kInter>
__device__ __forceinline__ Lane lane_of(const Params& P) {
  Lane l;
  const int lane = threadIdx.x & 31;
  l.G = P.G;
  l.u = lane & (P.G - 1);
  l.hsub = lane >> P.gshift;
  l.hpw = 32 >> P.gshift;
  l.act = 16 * l.u < P.d;
  unit_offsets<kInter>(l.u, P.rot, l.oa, l.ob);
  l.ng[0] = (P.Hq + l.hpw - 1) / l.hpw;
  l.ng[1] = (P.Hk + l.hpw - 1) / l.hpw;
  l.ng[2] = (P.Hv + l.hpw - 1) / l.hpw;
  return l;
}
// Head group g of the token's list: its side and this lane's head.
__device__ __forceinline__ int group_side(const Params& P, const Lane& l, int g, int& h, bool& in) {
  const int side = g < l.ng[0] ? 0 : g < l.ng[0] + l.ng[1] ? 1 : 2;
  const int g0 = side == 0 ? 0 : side == 1 ? l.ng[0] : l.ng[0] + l.ng[1];
  h = (g - g0) * l.hpw + l.hsub;
  in = l.act && h < (side == 0 ? P.Hq : side == 1 ? P.Hk : P.Hv);
  return side;
}

// cos and sin of a token's rot / 2 angles into the warp's slots (ang[0] cos,
// ang[1] sin; 1 and 0 up to the lanes' 8 per unit), each computed once a warp.
__device__ __forceinline__ void token_angles(const Params& P, const Lane& l, int64_t pos, float (*ang)[256]) {
  const int lane = threadIdx.x & 31;
  __syncwarp();   // the token before has been read
  for (int i = lane; i < P.d / 2; i += 32) {
    float c = 1.f, s = 0.f;
    if (i < P.rot / 2) turn(pos, MHC_LDG(P.inv_freq + i), c, s);
    ang[0][i] = c;
    ang[1][i] = s;
  }
  __syncwarp();
}
__device__ __forceinline__ void unit_angles(const float (*ang)[256], const Lane& l, float (&cs)[8], float (&sn)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    cs[j] = l.act ? ang[0][8 * l.u + j] : 1.f;
    sn[j] = l.act ? ang[1][8 * l.u + j] : 0.f;
  }
}

// The unit's weights of a side from shared memory (ones without a weight).
__device__ __forceinline__ void unit_weights(const float* sw, const Lane& l, float2 (&wa)[4], float2 (&wb)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    wa[j] = l.act ? *reinterpret_cast<const float2*>(sw + l.oa + 2 * j) : both(1.f);
    wb[j] = l.act ? *reinterpret_cast<const float2*>(sw + l.ob + 2 * j) : both(1.f);
  }
}
__device__ __forceinline__ void load_weights(const Params& P, float (*sw)[512]) {
  for (int i = threadIdx.x; i < P.d; i += kThreads) {
    sw[0][i] = P.wq ? MHC_LDG(P.wq + i) : 1.f;
    sw[1][i] = P.wk ? MHC_LDG(P.wk + i) : 1.f;
  }
  __syncthreads();
}

// Forward, 16-byte vectors.  A warp takes a token's head groups (all of them,
// or every parts-th), the next group's loads running during this one's
// arithmetic.  The side's weights are folded into the turn's coefficients once
// per token and side, so that a pair costs three packed instructions each way.
template <class T, bool kInter>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : 3) fwd_vec_kernel(const Params P) {
  __shared__ __align__(16) float sw[2][512];
  __shared__ __align__(16) float angles[kWarps][2][256];
  load_weights(P, sw);
  const Lane l = lane_of<kInter>(P);
  const int warp = threadIdx.x >> 5;
  const int groups = l.ng[0] + l.ng[1] + l.ng[2];
  const float inv_d = 1.f / (float)P.d;
  const int part = warp & (P.parts - 1);
  const int tok_per_cta = kWarps / P.parts;
  for (int64_t t = (int64_t)blockIdx.x * tok_per_cta + warp / P.parts; t < P.T;
       t += (int64_t)gridDim.x * tok_per_cta) {
    const int b = (int)((uint32_t)t / (uint32_t)P.S), s = (int)((uint32_t)t - (uint32_t)b * (uint32_t)P.S);
    auto fetch = [&](int g, Raw8<T>& ra, Raw8<T>& rb) {
      int h;
      bool in;
      const int side = group_side(P, l, g, h, in);
      ra.zero();
      rb.zero();
      if (g < groups && in) {
        const T* src = row<T>(side == 0 ? P.q : side == 1 ? P.k : P.v, b, s, h);
        ra.load(src + l.oa);
        rb.load(src + l.ob);
      }
    };
    Raw8<T> ra, rb;
    fetch(part, ra, rb);
    const float sc = P.row_scale ? MHC_LDG(P.row_scale + t) : 1.f;
    token_angles(P, l, position(P, b, s), angles[warp]);
    Turn tn;
    int cur = -1;
    for (int g = part; g < groups; g += P.parts) {
      Raw8<T> na, nb;
      fetch(g + P.parts, na, nb);
      int h;
      bool in;
      const int side = group_side(P, l, g, h, in);
      if (side != cur && side < 2) {   // the same for the whole warp
        cur = side;
        float2 wa[4], wb[4];
        float cs[8], sn[8];
        unit_weights(sw[side], l, wa, wb);
        unit_angles(angles[warp], l, cs, sn);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kInter) {
            tn.pa[j] = mul2(wa[j], both(cs[j]));
            tn.qa[j] = mul2(swapped(wa[j]), make_float2(-sn[j], sn[j]));
            tn.pb[j] = mul2(wb[j], both(cs[4 + j]));
            tn.qb[j] = mul2(swapped(wb[j]), make_float2(-sn[4 + j], sn[4 + j]));
          } else {
            const float2 c2 = make_float2(cs[2 * j], cs[2 * j + 1]), s2 = make_float2(sn[2 * j], sn[2 * j + 1]);
            tn.pa[j] = mul2(wa[j], c2);
            tn.qa[j] = mul2(wb[j], make_float2(-s2.x, -s2.y));
            tn.pb[j] = mul2(wb[j], c2);
            tn.qb[j] = mul2(wa[j], s2);
          }
        }
      }
      float2 a[4], c[4], ya[4], yc[4];
      ra.unpack(a);
      rb.unpack(c);
      float f = sc;
      if (side < 2) {
        float2 sq = mul2(a[0], a[0]);
#pragma unroll
        for (int j = 1; j < 4; ++j) sq = fma2(a[j], a[j], sq);
#pragma unroll
        for (int j = 0; j < 4; ++j) sq = fma2(c[j], c[j], sq);
        const float ms = group_sum(sq.x + sq.y, l.G) * inv_d;
        f = sc * __frsqrt_rn(fmaf(ms * sc, sc, P.eps));
        apply_turn<kInter>(tn, a, c, ya, yc);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) ya[j] = a[j], yc[j] = c[j];
      }
      if (in) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ya[j] = mul2(ya[j], both(f));
          yc[j] = mul2(yc[j], both(f));
        }
        T* dst = const_cast<T*>(row<T>(side == 0 ? P.oq : side == 1 ? P.ok : P.ov, b, s, h));
        store8(dst + l.oa, ya);
        store8(dst + l.ob, yc);
      }
      ra = na;
      rb = nb;
    }
  }
}

// Backward, 16-byte vectors, the forward's split.  Each lane keeps the weight
// gradients of its 16 elements: in registers over a side's head groups, in its
// own shared-memory slots over tokens.  The CTA's warps are added in warp order
// and the CTA's row written for the finalize kernel, so repeated calls give the
// same bits.
template <class T, bool kInter>
__global__ void __launch_bounds__(kThreads, 2) bwd_vec_kernel(const Params P) {
  __shared__ __align__(16) float sw[2][512];
  __shared__ __align__(16) float angles[kWarps][2][256];
  __shared__ float sds[kWarps];
  extern __shared__ __align__(16) float dyn[];   // [kWarps][2][16][32] weight gradients, with dw_part only
  load_weights(P, sw);
  const Lane l = lane_of<kInter>(P);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* gacc = dyn + warp * 1024 + lane;
  if (P.dw_part)
    for (int i = 0; i < 32; ++i) gacc[i * 32] = 0.f;
  const int groups = l.ng[0] + l.ng[1] + l.ng[2];
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
      auto fetch = [&](int g, Raw8<T>& xa, Raw8<T>& xb, Raw8<T>& ya, Raw8<T>& yb) {
        int h;
        bool in;
        const int side = group_side(P, l, g, h, in);
        xa.zero();
        xb.zero();
        ya.zero();
        yb.zero();
        if (g < groups && in) {
          const T* x = row<T>(side == 0 ? P.q : side == 1 ? P.k : P.v, b, s, h);
          const T* y = row<T>(side == 0 ? P.dq : side == 1 ? P.dk : P.dv, b, s, h);
          xa.load(x + l.oa);
          xb.load(x + l.ob);
          ya.load(y + l.oa);
          yb.load(y + l.ob);
        }
      };
      Raw8<T> xa, xb, ya, yb;
      fetch(part, xa, xb, ya, yb);
      const float sc = P.row_scale ? MHC_LDG(P.row_scale + t) : 1.f;
      float cs[8], sn[8];
      token_angles(P, l, position(P, b, s), angles[warp]);
      unit_angles(angles[warp], l, cs, sn);
      float2 wa[4], wb[4], ga[4], gb[4];
      int cur = -1;
      auto flush = [&]() {   // the side's sums into the lane's slots
        if (P.dw_part && cur >= 0) {
          float* g = gacc + cur * 512;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            g[(2 * j) * 32] += ga[j].x;
            g[(2 * j + 1) * 32] += ga[j].y;
            g[(8 + 2 * j) * 32] += gb[j].x;
            g[(8 + 2 * j + 1) * 32] += gb[j].y;
          }
        }
      };
      for (int g = part; g < groups; g += P.parts) {
        Raw8<T> nxa, nxb, nya, nyb;
        fetch(g + P.parts, nxa, nxb, nya, nyb);
        int h;
        bool in;
        const int side = group_side(P, l, g, h, in);
        float2 x0[4], x1[4], y0[4], y1[4], o0[4], o1[4];
        xa.unpack(x0);
        xb.unpack(x1);
        ya.unpack(y0);
        yb.unpack(y1);
        if (side < 2) {
          if (side != cur) {
            flush();
            cur = side;
            unit_weights(sw[side], l, wa, wb);
#pragma unroll
            for (int j = 0; j < 4; ++j) ga[j] = gb[j] = both(0.f);
          }
          float2 d0[4], d1[4];   // da = Rot^T dy
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (kInter) {
              d0[j] = fma2(swapped(y0[j]), make_float2(sn[j], -sn[j]), mul2(y0[j], both(cs[j])));
              d1[j] = fma2(swapped(y1[j]), make_float2(sn[4 + j], -sn[4 + j]), mul2(y1[j], both(cs[4 + j])));
            } else {
              const float2 c2 = make_float2(cs[2 * j], cs[2 * j + 1]), s2 = make_float2(sn[2 * j], sn[2 * j + 1]);
              d0[j] = fma2(y1[j], s2, mul2(y0[j], c2));
              d1[j] = fma2(y0[j], make_float2(-s2.x, -s2.y), mul2(y1[j], c2));
            }
          }
          float2 sq = both(0.f), dt = both(0.f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sq = fma2(x0[j], x0[j], sq);
            sq = fma2(x1[j], x1[j], sq);
            y0[j] = mul2(d0[j], x0[j]);   // da x
            y1[j] = mul2(d1[j], x1[j]);
            dt = fma2(y0[j], wa[j], dt);
            dt = fma2(y1[j], wb[j], dt);
          }
          const float ms = group_sum(sq.x + sq.y, l.G) * inv_d;
          const float dot = group_sum(dt.x + dt.y, l.G);   // sum(dn x)
          // a lane without a row adds nothing, whatever eps
          const float r = in ? __frsqrt_rn(fmaf(ms * sc, sc, P.eps)) : 0.f;
          const float sr = sc * r;
          const float m2 = -sr * (sr * dot * inv_d);   // -s r m
          if (l.u == 0) ds += P.eps * r * r * r * dot;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ga[j] = fma2(y0[j], both(sr), ga[j]);
            gb[j] = fma2(y1[j], both(sr), gb[j]);
            o0[j] = mul2(both(sr), fma2(both(m2), x0[j], mul2(d0[j], wa[j])));
            o1[j] = mul2(both(sr), fma2(both(m2), x1[j], mul2(d1[j], wb[j])));
          }
        } else {
          float2 dt = both(0.f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            dt = fma2(x0[j], y0[j], dt);
            dt = fma2(x1[j], y1[j], dt);
            o0[j] = mul2(both(sc), y0[j]);
            o1[j] = mul2(both(sc), y1[j]);
          }
          ds += dt.x + dt.y;
        }
        if (in) {
          T* dst = const_cast<T*>(row<T>(side == 0 ? P.oq : side == 1 ? P.ok : P.ov, b, s, h));
          store8(dst + l.oa, o0);
          store8(dst + l.ob, o1);
        }
        xa = nxa;
        xb = nxb;
        ya = nya;
        yb = nyb;
      }
      flush();
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
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * P.d; i += kThreads) {
      const int side = i >= P.d, col = i - side * P.d;
      // the unit and the place in it that hold this column
      int u, e;
      if (!kInter && col < P.rot) {
        const int half = P.rot / 2, c = col < half ? col : col - half;
        u = c / 8;
        e = (col < half ? 0 : 8) + c % 8;
      } else {
        u = col / 16;
        e = col % 16;
      }
      float sum = 0.f;
      for (int w = 0; w < kWarps; ++w)
        for (int k = 0; k < l.hpw; ++k) sum += dyn[w * 1024 + side * 512 + e * 32 + (k << P.gshift) + u];
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
