// Activation between the two products of an MLP layer, with its input kept in 8 bits for the backward pass.
//
//   x = (g | u), F columns each, or x = g.      h = act(g) u,  or act(g)
//   kept, per block of 128 columns of a row:     s = max|.| / 127,  q = sign(.) floor(127 |.| / max|.| + 1/2)
//   backward, with g^ = s q and u^ likewise:     dg = dh u^ act'(g^),  du = dh act(g^)      (or dg = dh act'(g^))
//
// Both passes are bound by HBM, and nearly by the issue of instructions.  Forward, eight lanes own a block, sixteen values of g
// and of u per lane in two groups of eight (16-byte loads), so that what a block costs besides its values is spread over many
// of them (sixteen lanes took 1.19 times as long); the two maxima travel together as one packed pair through three shuffles, and
// everything else stays in registers.  Backward there is no such cost, and sixteen lanes with eight values each, whose rows leave
// 256 bytes at a time, are faster (eight lanes: 1.2 times as long).
// 8192 x 14336 gated silu, bf16: forward 138 us, backward 137, each 0.95 GB (6.9 TB/s; the issue slots 70 to 74 % taken); gelu
// 157 and 153.  2051 x 5003 gelu, fp16, rows on any 2-byte boundary, in L2: 19 and 21 us, bound by the instructions (78 and 83 %).
// h is computed from x itself, not from what is kept.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "int8_kernel.cuh"

namespace bsg {

constexpr int kActBlock = 128;        // columns per scale
constexpr int kActThreads = 256;
constexpr int kActForwardLanes = 8, kActBackwardLanes = 16;      // threads per block of columns

struct ActParams {
  const uint16_t* X;      // forward: input
  const uint16_t* G;      // backward: gradient of h
  uint16_t* Y;            // forward: h; backward: gradient of x
  int8_t* Q;              // [rows][parts][pitch]
  float* scale;           // [rows][parts][blocks]
  int64_t ldx, ldg, ldy;  // elements
  int32_t F, blocks, pitch;
  uint32_t items;         // rows * blocks
  uint32_t div_mul, div_shift;      // item / blocks == umulhi(item, div_mul) >> div_shift  (blocks > 1)
};

template <bool FP16>
__device__ __forceinline__ void act_unpack(const uint4& v, float (&x)[8]) {
  i8_unpack2<FP16>(v.x, x[0], x[1]);
  i8_unpack2<FP16>(v.y, x[2], x[3]);
  i8_unpack2<FP16>(v.z, x[4], x[5]);
  i8_unpack2<FP16>(v.w, x[6], x[7]);
}
template <bool FP16>
__device__ __forceinline__ uint4 act_pack(const float (&x)[8]) {
  if constexpr (FP16) return make_uint4(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(x[4], x[5]), pack_f16x2(x[6], x[7]));
  else return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

// Stores eight values of a row.  Rows that do not start on 16 bytes leave as aligned 16-byte words all the same, each made of
// a lane's values and the eight in front of them; the two ends of the block go value by value.
// `left`: the eight values in front of them, where `has_left`; `last`: no other lane of the block takes this lane's last values.
template <bool WIDE>
__device__ __forceinline__ void act_store8(uint16_t* row, int32_t k, int32_t K, const uint4& v, const uint4& left, bool has_left, bool last, bool live) {
  if (!live) return;
  if constexpr (WIDE) {
    *reinterpret_cast<uint4*>(row + k) = v;       // K is a multiple of 8
  } else {
    const uint32_t skip = uint32_t(reinterpret_cast<uintptr_t>(row + k)) & 15u;      // bytes from the boundary to this lane's values
    const int32_t moved = int32_t(skip >> 1);                                          // values of the left neighbour in this lane's word
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if (has_left && k + 8 - moved <= K) {
      *reinterpret_cast<uint4*>(row + k - moved) = skip ? i8_shift16(left, v, 16u - skip) : v;
    } else {
      const uint32_t l[4] = {left.x, left.y, left.z, left.w};
      if (has_left) {
#pragma unroll
        for (int j = 1; j < 8; ++j) {
          if (j >= 8 - moved) row[k - 8 + j] = uint16_t(l[j >> 1] >> (16 * (j & 1)));
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < 8 - moved && k + j < K) row[k + j] = uint16_t(w[j >> 1] >> (16 * (j & 1)));
      }
    }
    if (last || k + 8 >= K) {
#pragma unroll
      for (int j = 1; j < 8; ++j) {
        if (j >= 8 - moved && k + j < K) row[k + j] = uint16_t(w[j >> 1] >> (16 * (j & 1)));
      }
    }
  }
}

// exp(x) and 1 / x of the special-function unit, off by about 2^-22 (the exponential by |x| 2^-24 more); results below 2^-126 are 0.
// All that they feed is rounded to 16 bits (2^-9 or 2^-12 of it), and 1 / x is only taken of 1 and more.
__device__ __forceinline__ float act_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float act_exp(float x) { return act_exp2(x * 1.4426950408889634f); }
__device__ __forceinline__ float act_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// act(x), and its slope.
// gelu: with y = |x| the lower tail of the normal distribution is P(-y) = exp(-y^2 / 2) Q(t), t = 1 / (1 + 0.255 y), whose
// exponential is also that of the slope.  Q is a polynomial of degree 7 without a constant term, fitted by linear programming to
// exp(y^2 / 2) P(-y) over y in [0, 13.4] (below -13.2 the exponential is 0, gelu under 2^-126): off by at most 5.3e-6 of it, and
// in all by 1.4e-8 below y = 2.8, where 1 - P(-y) counts too; at -8 a 16-bit result is then as near as its rounding allows, where
// a formula with a small absolute error (1.5e-7) was off by 1 %.  With CUDA's erfc the forward pass of 8192 x 14336 gated values
// took 1.5 times as long.
// silu: x below -87.3 gives -0 (the exact value is smaller than 2^-119).
__device__ __forceinline__ void act_normal(float x, float& cdf, float& gauss) {      // P(x), exp(-x^2 / 2)
  gauss = act_exp2(x * (x * -0.72134752044448170f));      // log2(e) / 2
  const float t = act_rcp(1.0f + 0.255f * fabsf(x));
  const float q = t * (0.10130616f + t * (0.10814349f + t * (0.05562561f + t * (0.21009077f + t * (-0.17184716f + t * (0.2778888f + t * -0.08120767f))))));
  const float tail = q * gauss;
  cdf = x < 0.0f ? tail : 1.0f - tail;
}
template <int ACT>
__device__ __forceinline__ float act_value(float x) {
  if constexpr (ACT == kActRelu) return x != x ? x : fmaxf(x, 0.0f);
  else if constexpr (ACT == kActSilu) return x * act_rcp(1.0f + act_exp(-x));
  else if constexpr (ACT == kActGelu) {
    float cdf, gauss;
    act_normal(x, cdf, gauss);
    return x * cdf;
  } else return x;
}
template <int ACT>
__device__ __forceinline__ void act_value_slope(float x, float& value, float& slope) {
  if constexpr (ACT == kActRelu) {
    value = x != x ? x : fmaxf(x, 0.0f);
    slope = x != x ? x : (x > 0.0f ? 1.0f : 0.0f);
  } else if constexpr (ACT == kActSilu) {
    const float s = act_rcp(1.0f + act_exp(-x));
    value = x * s;
    slope = s * (1.0f + x * (1.0f - s));
  } else if constexpr (ACT == kActGelu) {
    float phi, gauss;
    act_normal(x, phi, gauss);
    value = x * phi;
    slope = phi + x * 0.39894228040143267794f * gauss;
  } else {
    value = x;
    slope = 1.0f;
  }
}

// max(|.|) of 8 magnitudes of g in the low half, of u in the high half (sign bits are not meaningful).
template <bool FP16>
__device__ __forceinline__ uint32_t act_max_of(const uint4& v) {
  const uint32_t m = i8_maxabs2<FP16>(i8_maxabs2<FP16>(v.x, v.y), i8_maxabs2<FP16>(v.z, v.w));
  return i8_maxabs2<FP16>(m, m >> 16);
}

// The two groups of a lane: columns 8 sub ... and 64 + 8 sub ... of its block.
template <bool WIDE>
__device__ __forceinline__ void act_store16(uint16_t* row, int32_t k, int32_t K, const uint4 (&v)[2], int sub, bool ok) {
  uint4 left[2] = {v[0], v[1]};
  if constexpr (!WIDE) {
    auto up = [](const uint4& a) {
      return make_uint4(__shfl_up_sync(0xffffffffu, a.x, 1, 8), __shfl_up_sync(0xffffffffu, a.y, 1, 8), __shfl_up_sync(0xffffffffu, a.z, 1, 8), __shfl_up_sync(0xffffffffu, a.w, 1, 8));
    };
    // in front of the first lane's second group lies the last lane's first one
    const uint4 end = make_uint4(__shfl_sync(0xffffffffu, v[0].x, 7, 8), __shfl_sync(0xffffffffu, v[0].y, 7, 8), __shfl_sync(0xffffffffu, v[0].z, 7, 8), __shfl_sync(0xffffffffu, v[0].w, 7, 8));
    left[0] = up(v[0]);
    left[1] = up(v[1]);
    if (sub == 0) left[1] = end;
  }
  act_store8<WIDE>(row, k, K, v[0], left[0], sub > 0, false, ok && k < K);
  act_store8<WIDE>(row, k + 64, K, v[1], left[1], true, sub == 7, ok && k + 64 < K);
}

template <bool WIDE>
__device__ __forceinline__ void act_store16lanes(uint16_t* row, int32_t k, int32_t K, const uint4& v, int sub, bool live) {
  uint4 left = v;
  if constexpr (!WIDE)
    left = make_uint4(__shfl_up_sync(0xffffffffu, v.x, 1, 16), __shfl_up_sync(0xffffffffu, v.y, 1, 16), __shfl_up_sync(0xffffffffu, v.z, 1, 16), __shfl_up_sync(0xffffffffu, v.w, 1, 16));
  act_store8<WIDE>(row, k, K, v, left, sub > 0, sub == 15, live);
}

// LANES threads own a block.
template <int LANES>
struct ActItem {
  uint32_t row;
  int32_t block, k;      // k: first column of the lane's first group
  bool ok;
};
template <int LANES>
__device__ __forceinline__ ActItem<LANES> act_item(const ActParams& p) {
  ActItem<LANES> it;
  const uint32_t item = blockIdx.x * (kActThreads / LANES) + threadIdx.x / LANES;
  it.ok = item < p.items;
  it.row = !it.ok ? 0u : p.blocks == 1 ? item : __umulhi(item, p.div_mul) >> p.div_shift;
  it.block = it.ok ? int32_t(item - it.row * uint32_t(p.blocks)) : 0;
  it.k = it.block * kActBlock + int(threadIdx.x % LANES) * 8;
  return it;
}

template <int ACT, bool GATED, bool FP16, bool WIDE>
__global__ void __launch_bounds__(kActThreads) bsg_act_forward_kernel(const ActParams p) {
  constexpr int kParts = GATED ? 2 : 1;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const ActItem<kActForwardLanes> it = act_item<kActForwardLanes>(p);
  const int sub = threadIdx.x % kActForwardLanes;
  const int32_t F = it.ok ? p.F : 0;
  const uint16_t* x = p.X + int64_t(it.row) * p.ldx;
  uint4 gv[2], uv[2];
  {
    I8Raw rg[2], ru[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      rg[c] = i8_raw8<WIDE>(x, it.k + 64 * c, F);
      if constexpr (GATED) ru[c] = i8_raw8<WIDE>(x + p.F, it.k + 64 * c, F);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      gv[c] = i8_fix8<WIDE>(rg[c], x, it.k + 64 * c, F);
      uv[c] = make_uint4(0, 0, 0, 0);
      if constexpr (GATED) uv[c] = i8_fix8<WIDE>(ru[c], x + p.F, it.k + 64 * c, F);
    }
  }
  uint32_t m = i8_maxabs2<FP16>(act_max_of<FP16>(gv[0]), act_max_of<FP16>(gv[1])) & 0xFFFFu;
  if constexpr (GATED) m |= i8_maxabs2<FP16>(act_max_of<FP16>(uv[0]), act_max_of<FP16>(uv[1])) << 16;
#pragma unroll
  for (int o = 4; o >= 1; o >>= 1) m = i8_maxabs2<FP16>(m, __shfl_xor_sync(0xffffffffu, m, o));
  m &= 0x7FFF7FFFu;
  const float mg = i8_unpack(m & 0xFFFFu, FP16), mu = i8_unpack(m >> 16, FP16);
  // the first lane stores the scale of g, the second that of u
  const float step = i8_step(GATED && sub == 1 ? mu : mg);
  if (it.ok && sub < kParts) p.scale[(int64_t(it.row) * kParts + sub) * p.blocks + it.block] = step;
  int8_t* q = p.Q + int64_t(it.row) * kParts * p.pitch + it.k;
  const I8Scale sg = i8_scale(mg), su = i8_scale(mu);
  uint4 out[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (it.k + 64 * c < F) {      // kept rows are padded to 16 values: a group of 8 is stored whole
      *reinterpret_cast<uint2*>(q + 64 * c) = i8_levels8<FP16>(gv[c], sg);
      if constexpr (GATED) *reinterpret_cast<uint2*>(q + p.pitch + 64 * c) = i8_levels8<FP16>(uv[c], su);
    }
    float g[8], h[8];
    act_unpack<FP16>(gv[c], g);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = act_value<ACT>(g[j]);
    if constexpr (GATED) {
      float u[8];
      act_unpack<FP16>(uv[c], u);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] *= u[j];
    }
    out[c] = act_pack<FP16>(h);
  }
  act_store16<WIDE>(p.Y + int64_t(it.row) * p.ldy, it.k, p.F, out, sub, it.ok);
}

// s * q for four levels: a byte becomes fp32 as the last byte of 2^23 (exact), without the conversion unit.
__device__ __forceinline__ void act_dequant4(uint32_t q, float s, float* x) {
  const uint32_t b = q ^ 0x80808080u;       // level + 128
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = s * (__uint_as_float(__byte_perm(b, 0x4B000000u, 0x7540 + j)) - 8388736.0f);
}

template <int ACT, bool GATED, bool FP16, bool WIDE>
__global__ void __launch_bounds__(kActThreads) bsg_act_backward_kernel(const ActParams p) {
  constexpr int kParts = GATED ? 2 : 1;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const ActItem<kActBackwardLanes> it = act_item<kActBackwardLanes>(p);
  const int sub = threadIdx.x % kActBackwardLanes;
  const bool live = it.ok && it.k < p.F;
  if (WIDE && !live) return;
  const int32_t k = live ? it.k : 0;
  const uint16_t* grad = p.G + int64_t(it.row) * p.ldg;
  const I8Raw rd = i8_raw8<WIDE>(grad, k, live ? p.F : 0);
  const int8_t* q = p.Q + int64_t(it.row) * kParts * p.pitch + k;
  const float* scale = p.scale + int64_t(it.row) * kParts * p.blocks + it.block;
  const uint2 qg = *reinterpret_cast<const uint2*>(q);
  const float sg = *scale;
  uint2 qu = make_uint2(0, 0);
  float su = 0.0f;
  if constexpr (GATED) {
    qu = *reinterpret_cast<const uint2*>(q + p.pitch);
    su = scale[p.blocks];
  }
  float d[8], g[8], u[8], dg[8], du[8];
  act_unpack<FP16>(i8_fix8<WIDE>(rd, grad, k, live ? p.F : 0), d);
  act_dequant4(qg.x, sg, g);
  act_dequant4(qg.y, sg, g + 4);
  if constexpr (GATED) {
    act_dequant4(qu.x, su, u);
    act_dequant4(qu.y, su, u + 4);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float value, slope;
    act_value_slope<ACT>(g[j], value, slope);
    dg[j] = GATED ? d[j] * u[j] * slope : d[j] * slope;
    du[j] = d[j] * value;
  }
  uint16_t* y = p.Y + int64_t(it.row) * p.ldy;
  act_store16lanes<WIDE>(y, k, p.F, act_pack<FP16>(dg), sub, live);
  if constexpr (GATED) act_store16lanes<WIDE>(y + p.F, k, p.F, act_pack<FP16>(du), sub, live);
}

}  // namespace bsg
