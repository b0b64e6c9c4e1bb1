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
// The angle is p f / 2pi in 64 bits with what its products round off carried
// along, reduced to half a turn there, then one sincospi in 32 bits turned on by
// what rounding the angle lost: right to 32 bits at any position below 2^31,
// without a table that would have to be as long as the longest sequence.
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

// Sides: 0 queries, 1 keys, 2 values (no head where there are none).
struct Params {
  View x[3];                // inputs
  View dy[3];               // backward: upstream gradients
  View out[3];              // outputs (forward) / input gradients (backward); written
  const float* w[2];        // [d] or NULL
  const float* inv_freq;    // [rot / 2]
  const void* pos;          // NULL: the token's index in its sequence
  const float* row_scale;   // [T] or NULL
  float* d_row_scale;       // backward, [T] or NULL
  float* dw_part;           // backward, [grid][2][d] or NULL
  int64_t pos_sb, pos_ss;
  int64_t T;
  int S;
  int pos64;
  int heads[3];
  int d, rot;
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

// cos and sin of pos * f; see the head of this file.  Without the products' low
// parts the angle is off by up to 8 * 2^-24 at positions near 2^31; without the
// last step by up to 1.6 * 2^-24 at any, where cos and sin round by 2^-25.
__device__ __forceinline__ void turn(int64_t pos, float f, float& c, float& s) {
  constexpr double kHi = 0x1.45f306dc9c883p-3, kLo = -0x1.6b01ec5417056p-57;   // 1 / 2pi
  // products rounded by themselves: contracted into a sum, h's low part would count twice
  const double p = __dmul_rn((double)pos, (double)f), e = fma((double)pos, (double)f, -p);
  const double h = __dmul_rn(p, kHi);
  const double rev = (h - rint(h)) + fma(e, kHi, fma(p, kLo, fma(p, kHi, -h)));
  const float r = 2.0f * (float)rev;
  const float rest = (float)(2.0 * rev - (double)r) * 3.14159265358979f;
  sincospif(r, &s, &c);
  const float s0 = s;
  s = fmaf(c, rest, s);
  c = fmaf(-s0, rest, c);
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

// Sum over the 2^kGS lanes of a head row.
template <int kGS>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = 1; o < (1 << kGS); o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <class T>
__device__ __forceinline__ const T* row(const View& v, int b, int s, int h) {
  return static_cast<const T*>(v.p) + (b * v.sb + s * v.ss + h * v.sh);
}

// ------------------------------------------------------------ vector kernels
// 2^kGS lanes take a head row, 16 elements each, so a warp has 32 >> kGS head
// rows of one token and one side (queries, keys or values) at a time: a head
// group.  Its groups are every parts-th of the list of its tokens' groups, queries
// first, tokens `stride` apart.  Loads go through a ring in shared memory,
// kDepth groups ahead and across tokens, that only the lane itself writes
// (cp.async) and reads: depth without registers, no barrier.  With the next
// group's loads in registers instead (one ahead) the forward took 91 us at
// B=4, S=4096, 32+8+8 heads of 128, bf16, where a copy of the same rows takes 65.
//
// A cursor walks the groups with the lane's addresses in kN tensors.
template <class T, int kGS, int kN>
struct Cursor {
  static constexpr int kHpw = 32 >> kGS;
  const View* views[kN];   // [3] by side
  const T* p[kN];
  int64_t step[kN];
  int64_t t, stride;
  int part, hsub;
  int side, left, h;       // left: groups of this side from here on, the other warps' among them

  __device__ __forceinline__ bool more(const Params& P) const { return t < P.T; }
  __device__ __forceinline__ bool in(const Params& P) const { return h < P.heads[side]; }
  // to group `skip` from the start of `side`, of a later side or of the next token
  __device__ __forceinline__ void enter(const Params& P, int skip) {
    for (;;) {
      if (side == 3) {
        t += stride;
        side = 0;
        skip = part;
      }
      if (t >= P.T) return;
      const int ng = (P.heads[side] + kHpw - 1) / kHpw;
      if (skip < ng) {
        left = ng - skip;
        break;
      }
      skip -= ng;
      ++side;
    }
    const int b = (int)((uint32_t)t / (uint32_t)P.S), s = (int)((uint32_t)t - (uint32_t)b * (uint32_t)P.S);
    h = skip * kHpw + hsub;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      p[i] = row<T>(views[i][side], b, s, h);
      step[i] = (int64_t)(P.parts * kHpw) * views[i][side].sh;
    }
  }
  __device__ __forceinline__ void start(const Params& P, int64_t t0, int64_t stride_, int part_, int hsub_) {
    t = t0;
    stride = stride_;
    part = part_;
    hsub = hsub_;
    side = 0;
    enter(P, part);
  }
  __device__ __forceinline__ void advance(const Params& P) {
    left -= P.parts;
    if (left > 0) {
      h += P.parts * kHpw;
#pragma unroll
      for (int i = 0; i < kN; ++i) p[i] += step[i];
    } else {
      ++side;
      enter(P, -left);
    }
  }
};

// 16 bytes to the lane's own slot, zeros when there is nothing to load.
__device__ __forceinline__ void async16(uint4* dst, const void* src, bool in) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  const int bytes = in && MHC_CHK(src, 16) ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// Groups in flight per warp and 16-byte words a lane has in each, for kN tensors.
template <class T, int kN>
struct Ring {
  static constexpr int kWords = 2 * kN * Raw8<T>::kWords;
  static constexpr int kDepth = kWords <= 2 ? 5 : kWords <= 4 ? 3 : 2;
  static constexpr size_t kBytes = (size_t)kWarps * kDepth * kWords * 32 * 16;
};

// cos and sin of a token's rot / 2 angles into the warp's slots (ang[0] cos,
// ang[1] sin; 1 and 0 for the pairs that do not turn), each computed once a warp.
__device__ __forceinline__ void token_angles(const Params& P, int64_t pos, float (*ang)[256]) {
  __syncwarp();   // the token before has been read
  for (int i = threadIdx.x & 31; i < P.d / 2; i += 32) {
    float c = 1.f, s = 0.f;
    if (i < P.rot / 2) turn(pos, MHC_LDG(P.inv_freq + i), c, s);
    ang[0][i] = c;
    ang[1][i] = s;
  }
  __syncwarp();
}
// The unit's 8 values at [8 u] of a warp's angles.
__device__ __forceinline__ void unit_angles(const float (*ang)[256], int u, float2 (&cs)[4], float2 (&sn)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    cs[j] = *reinterpret_cast<const float2*>(&ang[0][8 * u + 2 * j]);
    sn[j] = *reinterpret_cast<const float2*>(&ang[1][8 * u + 2 * j]);
  }
}
__device__ __forceinline__ void load_weights(const Params& P, float (*sw)[512]) {
  for (int i = threadIdx.x; i < P.d; i += kThreads) {
    sw[0][i] = P.w[0] ? MHC_LDG(P.w[0] + i) : 1.f;
    sw[1][i] = P.w[1] ? MHC_LDG(P.w[1] + i) : 1.f;
  }
  __syncthreads();
}
__device__ __forceinline__ void unit_weights(const float* sw, int oa, int ob, float2 (&wa)[4], float2 (&wb)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    wa[j] = *reinterpret_cast<const float2*>(sw + oa + 2 * j);
    wb[j] = *reinterpret_cast<const float2*>(sw + ob + 2 * j);
  }
}

// Lanes beyond a row of d elements work on unit 0's coefficients and on zeros.
template <bool kInter, int kGS>
__device__ __forceinline__ bool lane_unit(const Params& P, int lane, int& u, int& oa, int& ob) {
  u = lane & ((1 << kGS) - 1);
  const bool act = 16 * u < P.d;
  if (!act) u = 0;
  unit_offsets<kInter>(u, P.rot, oa, ob);
  return act;
}

// Forward.  The side's weights are folded into the turn's coefficients once per
// token and side, so that a pair costs three packed instructions each way.
// Memory bounds it: 72 us at B=4, S=4096, 32+8+8 heads of 128, bf16, 403 MB at
// 5.6 TB/s (a copy of the same rows: 65 us).  A few tokens are bound by the
// launch: 5.0 us for one.
template <class T, bool kInter, int kGS>
__global__ void __launch_bounds__(kThreads, 2) fwd_vec_kernel(const __grid_constant__ Params P) {
  __shared__ __align__(16) float sw[2][512];
  __shared__ __align__(16) float angles[kWarps][2][256];
  extern __shared__ __align__(16) uint4 ring[];   // [kWarps][kDepth][kWords][32]
  using R = Ring<T, 1>;
  constexpr int kW = Raw8<T>::kWords;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int u, oa, ob;
  const bool act = lane_unit<kInter, kGS>(P, lane, u, oa, ob);
  uint4* slots = ring + (warp * R::kDepth * R::kWords) * 32 + lane;
  const float inv_d = 1.f / (float)P.d;
  const int tok_per_cta = kWarps / P.parts, part = warp & (P.parts - 1);
  const int64_t t0 = (int64_t)blockIdx.x * tok_per_cta + warp / P.parts, stride = (int64_t)gridDim.x * tok_per_cta;
  Cursor<T, kGS, 1> f, c;
  f.views[0] = P.x;
  c.views[0] = P.out;
  f.start(P, t0, stride, part, lane >> kGS);
  c.start(P, t0, stride, part, lane >> kGS);
  auto issue = [&](int slot) {
    uint4* dst = slots + slot * R::kWords * 32;
    if (f.more(P)) {
      const bool in = act && f.in(P);
#pragma unroll
      for (int i = 0; i < kW; ++i) {
        async16(dst + i * 32, reinterpret_cast<const uint4*>(f.p[0] + oa) + i, in);
        async16(dst + (kW + i) * 32, reinterpret_cast<const uint4*>(f.p[0] + ob) + i, in);
      }
      f.advance(P);
    }
    async_commit();
  };
#pragma unroll
  for (int i = 0; i < R::kDepth; ++i) issue(i);
  load_weights(P, sw);
  int64_t token = -1;
  int cur = -1, slot = 0;
  float sc = 1.f;
  Turn tn;
  while (c.more(P)) {
    const int side = c.side;
    if (c.t != token) {
      token = c.t;
      cur = -1;
      const int b = (int)((uint32_t)token / (uint32_t)P.S), s = (int)((uint32_t)token - (uint32_t)b * (uint32_t)P.S);
      if (P.row_scale) sc = MHC_LDG(P.row_scale + token);
      token_angles(P, position(P, b, s), angles[warp]);
    }
    if (side != cur && side < 2) {   // the same for the whole warp
      cur = side;
      float2 wa[4], wb[4], cs[4], sn[4];
      unit_weights(sw[side], oa, ob, wa, wb);
      unit_angles(angles[warp], u, cs, sn);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kInter) {
          const float c0 = j & 1 ? cs[j / 2].y : cs[j / 2].x, s0 = j & 1 ? sn[j / 2].y : sn[j / 2].x;
          const float c1 = j & 1 ? cs[2 + j / 2].y : cs[2 + j / 2].x, s1 = j & 1 ? sn[2 + j / 2].y : sn[2 + j / 2].x;
          tn.pa[j] = mul2(wa[j], both(c0));
          tn.qa[j] = mul2(swapped(wa[j]), make_float2(-s0, s0));
          tn.pb[j] = mul2(wb[j], both(c1));
          tn.qb[j] = mul2(swapped(wb[j]), make_float2(-s1, s1));
        } else {
          tn.pa[j] = mul2(wa[j], cs[j]);
          tn.qa[j] = mul2(wb[j], make_float2(-sn[j].x, -sn[j].y));
          tn.pb[j] = mul2(wb[j], cs[j]);
          tn.qb[j] = mul2(wa[j], sn[j]);
        }
      }
    }
    async_wait<R::kDepth - 1>();
    const uint4* src = slots + slot * R::kWords * 32;
    Raw8<T> ra, rb;
#pragma unroll
    for (int i = 0; i < kW; ++i) ra.w[i] = src[i * 32], rb.w[i] = src[(kW + i) * 32];
    float2 x0[4], x1[4], y0[4], y1[4];
    ra.unpack(x0);
    rb.unpack(x1);
    float fct = sc;
    if (side < 2) {
      float2 sq = mul2(x0[0], x0[0]), sq1 = mul2(x1[0], x1[0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) {
        sq = fma2(x0[j], x0[j], sq);
        sq1 = fma2(x1[j], x1[j], sq1);
      }
      const float ms = group_sum<kGS>((sq.x + sq.y) + (sq1.x + sq1.y)) * inv_d;
      fct = sc * rsqrtf(fmaf(ms * sc, sc, P.eps));
      apply_turn<kInter>(tn, x0, x1, y0, y1);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) y0[j] = x0[j], y1[j] = x1[j];
    }
    issue(slot);
    slot = slot + 1 == R::kDepth ? 0 : slot + 1;
    if (act && c.in(P)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y0[j] = mul2(y0[j], both(fct));
        y1[j] = mul2(y1[j], both(fct));
      }
      T* dst = const_cast<T*>(c.p[0]);
      store8(dst + oa, y0);
      store8(dst + ob, y1);
    }
    c.advance(P);
  }
}

// Backward.  Each lane keeps the weight gradients of its 16 elements: in
// registers over a side's head groups, in its own shared-memory slots over
// tokens.  The CTA's warps are added in warp order, in 64 bits, and the CTA's row
// written for the finalize kernel, so repeated calls give the same bits.  113 us
// for the forward's tokens, 604 MB at 5.3 TB/s (119 to 124 a call with the
// finalize kernel); its sums, angles and weights fill 128 registers, and of 16
// warps an SM 57% of the issue slots are used.  Wide heads, few to a token, wait
// instead: 67 us for 8191 tokens of 16+2 heads of 256, 226 MB at 3.4 TB/s, 44% of
// the slots, three tenths of the stalls on shared memory and conversions (the angles
// and sums of every token, which 18 heads share) and a quarter on the
// instruction before.
template <class T, bool kInter, int kGS>
__global__ void __launch_bounds__(kThreads, 2) bwd_vec_kernel(const __grid_constant__ Params P) {
  __shared__ __align__(16) float sw[2][512];
  __shared__ __align__(16) float angles[kWarps][2][256];
  __shared__ float sds[kWarps];
  extern __shared__ __align__(16) uint4 ring[];   // [kWarps][kDepth][kWords][32], then the gradients
  using R = Ring<T, 2>;
  constexpr int kW = Raw8<T>::kWords;
  float* dyn = reinterpret_cast<float*>(ring + R::kBytes / 16);   // [kWarps][2][16][32], with dw_part only
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int u, oa, ob;
  const bool act = lane_unit<kInter, kGS>(P, lane, u, oa, ob);
  uint4* slots = ring + (warp * R::kDepth * R::kWords) * 32 + lane;
  float* gacc = dyn + warp * 1024 + lane;
  const float inv_d = 1.f / (float)P.d;
  const int tok_per_cta = kWarps / P.parts, part = warp & (P.parts - 1);
  const int64_t t0 = (int64_t)blockIdx.x * tok_per_cta + warp / P.parts, stride = (int64_t)gridDim.x * tok_per_cta;
  Cursor<T, kGS, 2> f;
  Cursor<T, kGS, 1> c;
  f.views[0] = P.x;
  f.views[1] = P.dy;
  c.views[0] = P.out;
  f.start(P, t0, stride, part, lane >> kGS);
  c.start(P, t0, stride, part, lane >> kGS);
  auto issue = [&](int slot) {
    uint4* dst = slots + slot * R::kWords * 32;
    if (f.more(P)) {
      const bool in = act && f.in(P);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < kW; ++i) {
          async16(dst + (2 * n * kW + i) * 32, reinterpret_cast<const uint4*>(f.p[n] + oa) + i, in);
          async16(dst + ((2 * n + 1) * kW + i) * 32, reinterpret_cast<const uint4*>(f.p[n] + ob) + i, in);
        }
      f.advance(P);
    }
    async_commit();
  };
#pragma unroll
  for (int i = 0; i < R::kDepth; ++i) issue(i);
  if (P.dw_part)
    for (int i = 0; i < 32; ++i) gacc[i * 32] = 0.f;
  load_weights(P, sw);
  float2 cs[4], sn[4], wa[4], wb[4], ga[4], gb[4];
  int64_t token = -1;
  int cur = -1, slot = 0;
  float sc = 1.f, ds = 0.f;
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
  while (c.more(P)) {
    const int side = c.side;
    if (c.t != token) {
      token = c.t;
      cur = -1;
      ds = 0.f;
      const int b = (int)((uint32_t)token / (uint32_t)P.S), s = (int)((uint32_t)token - (uint32_t)b * (uint32_t)P.S);
      if (P.row_scale) sc = MHC_LDG(P.row_scale + token);
      token_angles(P, position(P, b, s), angles[warp]);
      unit_angles(angles[warp], u, cs, sn);
    }
    if (side != cur && side < 2) {
      flush();
      cur = side;
      unit_weights(sw[side], oa, ob, wa, wb);
#pragma unroll
      for (int j = 0; j < 4; ++j) ga[j] = gb[j] = both(0.f);
    }
    async_wait<R::kDepth - 1>();
    const uint4* src = slots + slot * R::kWords * 32;
    Raw8<T> ra, rb;
    float2 x0[4], x1[4], y0[4], y1[4];
#pragma unroll
    for (int i = 0; i < kW; ++i) ra.w[i] = src[i * 32], rb.w[i] = src[(kW + i) * 32];
    ra.unpack(x0);
    rb.unpack(x1);
#pragma unroll
    for (int i = 0; i < kW; ++i) ra.w[i] = src[(2 * kW + i) * 32], rb.w[i] = src[(3 * kW + i) * 32];
    ra.unpack(y0);
    rb.unpack(y1);
    const bool in = act && c.in(P);
    if (side < 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {   // da = Rot^T dy, in place
        const float2 g0 = y0[j], g1 = y1[j];
        if constexpr (kInter) {
          const float c0 = j & 1 ? cs[j / 2].y : cs[j / 2].x, s0 = j & 1 ? sn[j / 2].y : sn[j / 2].x;
          const float c1 = j & 1 ? cs[2 + j / 2].y : cs[2 + j / 2].x, s1 = j & 1 ? sn[2 + j / 2].y : sn[2 + j / 2].x;
          y0[j] = fma2(swapped(g0), make_float2(s0, -s0), mul2(g0, both(c0)));
          y1[j] = fma2(swapped(g1), make_float2(s1, -s1), mul2(g1, both(c1)));
        } else {
          y0[j] = fma2(g1, sn[j], mul2(g0, cs[j]));
          y1[j] = fma2(g0, make_float2(-sn[j].x, -sn[j].y), mul2(g1, cs[j]));
        }
      }
      float2 sq = both(0.f), dt = both(0.f), sq1 = both(0.f), dt1 = both(0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sq = fma2(x0[j], x0[j], sq);
        sq1 = fma2(x1[j], x1[j], sq1);
        dt = fma2(mul2(y0[j], x0[j]), wa[j], dt);
        dt1 = fma2(mul2(y1[j], x1[j]), wb[j], dt1);
      }
      const float ms = group_sum<kGS>((sq.x + sq.y) + (sq1.x + sq1.y)) * inv_d;
      const float dot = group_sum<kGS>((dt.x + dt.y) + (dt1.x + dt1.y));   // sum(dn x)
      issue(slot);
      // a lane without a row adds nothing, whatever eps
      const float r = in ? rsqrtf(fmaf(ms * sc, sc, P.eps)) : 0.f;
      const float sr = sc * r;
      const float m2 = -sr * (sr * dot * inv_d);   // -s r m
      if ((lane & ((1 << kGS) - 1)) == 0) ds += P.eps * r * r * r * dot;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 n0 = mul2(both(sr), x0[j]), n1 = mul2(both(sr), x1[j]);
        ga[j] = fma2(y0[j], n0, ga[j]);
        gb[j] = fma2(y1[j], n1, gb[j]);
        y0[j] = mul2(both(sr), fma2(both(m2), x0[j], mul2(y0[j], wa[j])));
        y1[j] = mul2(both(sr), fma2(both(m2), x1[j], mul2(y1[j], wb[j])));
      }
    } else {
      float2 dt = both(0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        dt = fma2(x0[j], y0[j], dt);
        dt = fma2(x1[j], y1[j], dt);
        y0[j] = mul2(both(sc), y0[j]);
        y1[j] = mul2(both(sc), y1[j]);
      }
      ds += dt.x + dt.y;
      issue(slot);
    }
    slot = slot + 1 == R::kDepth ? 0 : slot + 1;
    if (in) {
      T* dst = const_cast<T*>(c.p[0]);
      store8(dst + oa, y0);
      store8(dst + ob, y1);
    }
    c.advance(P);
    if (c.t != token) {   // the token's last group of this warp
      flush();
      if (P.d_row_scale) {
        ds = warp_sum(ds);
        if (P.parts == 1) {
          if (lane == 0) MHC_ST(P.d_row_scale + token, ds);
        } else {
          // the token's warps walk the same tokens: one named barrier for each set of them
          const int id = 1 + warp / P.parts, count = P.parts * 32;
          if (lane == 0) sds[warp] = ds;
          asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(count) : "memory");
          if (part == 0 && lane == 0) {
            float sum = 0.f;
            for (int i = 0; i < P.parts; ++i) sum += sds[warp + i];
            MHC_ST(P.d_row_scale + token, sum);
          }
          asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(count) : "memory");
        }
      }
    }
  }
  async_wait<0>();
  if (P.dw_part) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * P.d; i += kThreads) {
      const int side = i >= P.d, col = i - side * P.d;
      // the unit and the place in it that hold this column
      int unit, e;
      if (!kInter && col < P.rot) {
        const int half = P.rot / 2, cc = col < half ? col : col - half;
        unit = cc / 8;
        e = (col < half ? 0 : 8) + cc % 8;
      } else {
        unit = col / 16;
        e = col % 16;
      }
      double sum = 0.0;   // 64 lanes' sums one behind the other: in 32 bits half of the gradient's error
      for (int w = 0; w < kWarps; ++w)
        for (int k = 0; k < (32 >> kGS); ++k) sum += (double)dyn[w * 1024 + side * 512 + e * 32 + (k << kGS) + unit];
      MHC_ST(P.dw_part + (int64_t)blockIdx.x * 2 * P.d + i, (float)sum);
    }
  }
}

// ------------------------------------------------------------ any width, stride, alignment
// A warp per head row, lane l the pairs l, l + 32, ..: the rotated ones, then
// the passing elements two by two (the last of an odd number alone).  A row is
// read once, into registers, kP pairs a lane (2 up to d = 128, 4 up to 256, else 16).
// Dynamic shared memory per warp: the token's cos and sin [rot/2] and, in the
// backward, the weight gradients [2][d] of the warp (a lane only ever touches its
// own columns).
template <bool kInter>
__device__ __forceinline__ bool pair_places(const Params& P, int p, int& ia, int& ib) {
  const int half = P.rot / 2;
  if (p < half) {
    ia = kInter ? 2 * p : p;
    ib = kInter ? 2 * p + 1 : p + half;
    return true;
  }
  ia = 2 * p;   // rot + 2 (p - half)
  ib = 2 * p + 1;
  return false;
}
__device__ __forceinline__ void head_side(const Params& P, int h, int& side, int& hh) {
  side = h < P.heads[0] ? 0 : h < P.heads[0] + P.heads[1] ? 1 : 2;
  hh = h - (side > 0 ? P.heads[0] : 0) - (side > 1 ? P.heads[1] : 0);
}

template <class T, bool kInter, int kP>
__global__ void __launch_bounds__(kThreads) fwd_any_kernel(const __grid_constant__ Params P) {
  extern __shared__ float dyn[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = P.rot / 2;
  float* cs = dyn + warp * P.rot;
  float* sn = cs + half;
  const int H = P.heads[0] + P.heads[1] + P.heads[2];
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
      int side, hh;
      head_side(P, h, side, hh);
      const T* x = row<T>(P.x[side], b, s, hh);
      T* y = const_cast<T*>(row<T>(P.out[side], b, s, hh));
      const float* w = side < 2 ? P.w[side] : nullptr;
      float xa[kP], xb[kP], sq = 0.f;
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        int ia, ib;
        pair_places<kInter>(P, lane + 32 * i, ia, ib);
        xa[i] = ia < P.d ? load1(x + ia) * sc : 0.f;
        xb[i] = ib < P.d ? load1(x + ib) * sc : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        sq = fmaf(xa[i], xa[i], sq);
        sq = fmaf(xb[i], xb[i], sq);
      }
      const float r = side == 2 ? 1.f : rsqrtf(fmaf(warp_sum(sq), inv_d, P.eps));
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        int ia, ib;
        const bool turned = pair_places<kInter>(P, lane + 32 * i, ia, ib) && side != 2;
        if (ia < P.d) {
          float a = xa[i] * r, c = xb[i] * r;
          if (w) {
            a *= MHC_LDG(w + ia);
            if (ib < P.d) c *= MHC_LDG(w + ib);
          }
          if (turned) {
            const float cc = cs[lane + 32 * i], ss = sn[lane + 32 * i], a0 = a;
            a = a0 * cc - c * ss;
            c = a0 * ss + c * cc;
          }
          store1(y + ia, a);
          if (ib < P.d) store1(y + ib, c);
        }
      }
    }
  }
}

template <class T, bool kInter, int kP>
__global__ void __launch_bounds__(kThreads) bwd_any_kernel(const __grid_constant__ Params P) {
  extern __shared__ float dyn[];
  __shared__ float sds[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = P.rot / 2;
  float* cs = dyn + warp * (P.rot + 2 * P.d);
  float* sn = cs + half;
  float* gw = dyn + warp * (P.rot + 2 * P.d) + P.rot;   // [2][d]
  for (int i = lane; i < 2 * P.d; i += 32) gw[i] = 0.f;
  __syncwarp();
  const int H = P.heads[0] + P.heads[1] + P.heads[2];
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
        int side, hh;
        head_side(P, h, side, hh);
        const T* x = row<T>(P.x[side], b, s, hh);
        const T* dy = row<T>(P.dy[side], b, s, hh);
        T* dx = const_cast<T*>(row<T>(P.out[side], b, s, hh));
        const float* w = side < 2 ? P.w[side] : nullptr;
        float xa[kP], xb[kP], ga[kP], gb[kP];   // x; da = Rot^T dy
#pragma unroll
        for (int i = 0; i < kP; ++i) {
          int ia, ib;
          pair_places<kInter>(P, lane + 32 * i, ia, ib);
          xa[i] = ia < P.d ? load1(x + ia) : 0.f;
          xb[i] = ib < P.d ? load1(x + ib) : 0.f;
          ga[i] = ia < P.d ? load1(dy + ia) : 0.f;
          gb[i] = ib < P.d ? load1(dy + ib) : 0.f;
        }
        float sq = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < kP; ++i) {
          int ia, ib;
          const bool turned = pair_places<kInter>(P, lane + 32 * i, ia, ib) && side != 2;
          if (turned) {
            const float cc = cs[lane + 32 * i], ss = sn[lane + 32 * i], g0 = ga[i];
            ga[i] = g0 * cc + gb[i] * ss;
            gb[i] = gb[i] * cc - g0 * ss;
          }
          const float za = xa[i] * sc, zb = xb[i] * sc;
          sq = fmaf(za, za, sq);
          sq = fmaf(zb, zb, sq);
          dot = fmaf(w && ia < P.d ? ga[i] * MHC_LDG(w + ia) : ga[i], xa[i], dot);
          dot = fmaf(w && ib < P.d ? gb[i] * MHC_LDG(w + ib) : gb[i], xb[i], dot);
        }
        dot = warp_sum(dot);   // sum(dn x); sum(v dv_out) on value rows
        float sr = sc, m = 0.f;
        if (side == 2) {
          if (lane == 0) ds += dot;
        } else {
          const float r = rsqrtf(fmaf(warp_sum(sq), inv_d, P.eps));
          sr = sc * r;
          m = sr * dot * inv_d;
          if (lane == 0) ds += P.eps * r * r * r * dot;
        }
        float* g = gw + (side == 0 ? 0 : P.d);
#pragma unroll
        for (int i = 0; i < kP; ++i) {
          int ia, ib;
          pair_places<kInter>(P, lane + 32 * i, ia, ib);
          if (ia < P.d) {
            const float na = xa[i] * sr;
            if (side != 2) g[ia] = fmaf(na, ga[i], g[ia]);
            const float dn = w ? ga[i] * MHC_LDG(w + ia) : ga[i];
            store1(dx + ia, sr * (side == 2 ? dn : dn - na * m));
          }
          if (ib < P.d) {
            const float nb = xb[i] * sr;
            if (side != 2) g[ib] = fmaf(nb, gb[i], g[ib]);
            const float dn = w ? gb[i] * MHC_LDG(w + ib) : gb[i];
            store1(dx + ib, sr * (side == 2 ? dn : dn - nb * m));
          }
        }
      }
    }
    if (P.d_row_scale) {
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

// Weight gradients: the CTAs' rows [parts][2 d] added in 64 bits in a fixed
// order, 32 columns a CTA, every warp an eighth of the rows.
__global__ void __launch_bounds__(kThreads) bwd_weights_kernel(const float* __restrict__ part, int rows, int d,
                                                               float* __restrict__ dwq, float* __restrict__ dwk) {
  __shared__ double acc[kWarps][kFinCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * kFinCols + lane;
  double sum = 0.0;
  if (col < 2 * d)
    for (int r = warp; r < rows; r += kWarps) sum += (double)MHC_LDG(part + (int64_t)r * 2 * d + col);
  acc[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && col < 2 * d) {
    double sums = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sums += acc[w][lane];
    const float v = (float)sums;
    if (col < d) {
      if (dwq) MHC_ST(dwq + col, v);
    } else if (dwk) {
      MHC_ST(dwk + col - d, v);
    }
  }
}

}  // namespace rope
}  // namespace mhc
