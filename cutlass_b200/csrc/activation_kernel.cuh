// Activation between the two products of an MLP layer, with its input kept in 8 bits for the backward pass.
//
//   x = (g | u), F columns each, or x = g.      h = act(g) u,  or act(g)
//   kept, per block of 128 columns of a row:     s = max|.| / 127,  q = sign(.) floor(127 |.| / max|.| + 1/2)
//   backward, with g^ = s q and u^ likewise:     dg = dh u^ act'(g^),  du = dh act(g^)      (or dg = dh act'(g^))
//
// Both passes are bound by HBM.  Sixteen lanes own a block: eight consecutive values of g and of u per lane (16-byte loads),
// so the two maxima travel together as one packed pair through four shuffles, and everything else stays in registers.
// h is computed from x itself, not from what is kept.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "int8_kernel.cuh"

namespace bsg {

constexpr int kActBlock = 128;        // columns per scale
constexpr int kActThreads = 256;

struct ActParams {
  const uint16_t* X;      // forward: input
  const uint16_t* G;      // backward: gradient of h
  uint16_t* Y;            // forward: h; backward: gradient of x
  int8_t* Q;              // [rows][parts][pitch]
  float* scale;           // [rows][parts][blocks]
  int64_t ldx, ldg, ldy;  // elements
  int32_t F, blocks, pitch;
  uint32_t items;         // rows * blocks
  int32_t act;
  int32_t wide_in, wide_out;   // every 8-value group of the input / output starts on a 16-byte boundary
};

template <bool FP16>
__device__ __forceinline__ void act_unpack(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (FP16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      x[2 * j] = f.x; x[2 * j + 1] = f.y;
    } else {
      x[2 * j] = __uint_as_float(w[j] << 16); x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
}
template <bool FP16>
__device__ __forceinline__ uint4 act_pack(const float (&x)[8]) {
  if constexpr (FP16) return make_uint4(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(x[4], x[5]), pack_f16x2(x[6], x[7]));
  else return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ void act_store8(uint16_t* row, int32_t k, int32_t K, const uint4& v, bool wide) {
  if (wide && k + 8 <= K) {
    *reinterpret_cast<uint4*>(row + k) = v;
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (k + j < K) row[k + j] = uint16_t(w[j >> 1] >> (16 * (j & 1)));
  }
}

// act(x), and its slope.  The results are rounded to 16 bits, so the fast exponential and quotient (errors near 2^-21) do.
template <int ACT>
__device__ __forceinline__ float act_value(float x) {
  if constexpr (ACT == kActRelu) return x != x ? x : fmaxf(x, 0.0f);
  else if constexpr (ACT == kActSilu) return __fdividef(x, 1.0f + __expf(-x));
  else if constexpr (ACT == kActGelu) return 0.5f * x * erfcf(x * -0.70710678118654752440f);
  else return x;
}
template <int ACT>
__device__ __forceinline__ void act_value_slope(float x, float& value, float& slope) {
  if constexpr (ACT == kActRelu) {
    value = x != x ? x : fmaxf(x, 0.0f);
    slope = x != x ? x : (x > 0.0f ? 1.0f : 0.0f);
  } else if constexpr (ACT == kActSilu) {
    const float s = __fdividef(1.0f, 1.0f + __expf(-x));
    value = x * s;
    slope = s * (1.0f + x * (1.0f - s));
  } else if constexpr (ACT == kActGelu) {
    const float phi = 0.5f * erfcf(x * -0.70710678118654752440f);
    value = x * phi;
    slope = phi + x * 0.39894228040143267794f * __expf(-0.5f * x * x);
  } else {
    value = x;
    slope = 1.0f;
  }
}

template <bool FP16>
__device__ __forceinline__ uint32_t act_max_of(const uint4& v) {        // max of 8 magnitudes, in the low half
  uint32_t m = i8_maxabs2<FP16>(i8_maxabs2<FP16>(v.x, v.y), i8_maxabs2<FP16>(v.z, v.w)) & 0x7FFF7FFFu;
  return i8_maxabs2<FP16>(m, m >> 16) & 0x7FFFu;
}

template <int ACT, bool GATED, bool FP16>
__global__ void __launch_bounds__(kActThreads) bsg_act_forward_kernel(const ActParams p) {
  const uint32_t item = blockIdx.x * (kActThreads / 16) + threadIdx.x / 16;
  const int sub = threadIdx.x & 15;
  const bool ok = item < p.items;
  const uint32_t row = ok ? item / uint32_t(p.blocks) : 0u;
  const int32_t block = ok ? int32_t(item - row * uint32_t(p.blocks)) : 0;
  const int32_t k = block * kActBlock + sub * 8;
  const int32_t F = ok ? p.F : 0;
  const uint16_t* x = p.X + int64_t(row) * p.ldx;
  const bool wide = p.wide_in != 0;
  const uint4 gv = i8_load8(x, k, F, wide);
  uint4 uv = make_uint4(0, 0, 0, 0);
  if constexpr (GATED) uv = i8_load8(x + p.F, k, F, wide);
  uint32_t m = act_max_of<FP16>(gv);
  if constexpr (GATED) m |= act_max_of<FP16>(uv) << 16;
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) m = i8_maxabs2<FP16>(m, __shfl_xor_sync(0xffffffffu, m, o)) & 0x7FFF7FFFu;
  if (!ok || k >= p.F) return;
  constexpr int kParts = GATED ? 2 : 1;
  const I8Scale sg = i8_scale(i8_unpack(m & 0xFFFFu, FP16));
  int8_t* q = p.Q + int64_t(row) * kParts * p.pitch + k;
  float* scale = p.scale + int64_t(row) * kParts * p.blocks + block;
  // the kept rows are padded to 16 values, so a group of 8 is always stored whole
  *reinterpret_cast<uint2*>(q) = i8_levels8<FP16>(gv, sg);
  if (sub == 0) scale[0] = sg.scale;
  float g[8], h[8];
  act_unpack<FP16>(gv, g);
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = act_value<ACT>(g[j]);
  if constexpr (GATED) {
    const I8Scale su = i8_scale(i8_unpack(m >> 16, FP16));
    *reinterpret_cast<uint2*>(q + p.pitch) = i8_levels8<FP16>(uv, su);
    if (sub == 0) scale[p.blocks] = su.scale;
    float u[8];
    act_unpack<FP16>(uv, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] *= u[j];
  }
  act_store8(p.Y + int64_t(row) * p.ldy, k, p.F, act_pack<FP16>(h), p.wide_out != 0);
}

__device__ __forceinline__ void act_dequant8(const uint2& q, float s, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = s * float(int8_t((j < 4 ? q.x : q.y) >> (8 * (j & 3))));
}

template <int ACT, bool GATED, bool FP16>
__global__ void __launch_bounds__(kActThreads) bsg_act_backward_kernel(const ActParams p) {
  const uint32_t item = blockIdx.x * (kActThreads / 16) + threadIdx.x / 16;
  const int sub = threadIdx.x & 15;
  if (item >= p.items) return;
  const uint32_t row = item / uint32_t(p.blocks);
  const int32_t block = int32_t(item - row * uint32_t(p.blocks));
  const int32_t k = block * kActBlock + sub * 8;
  if (k >= p.F) return;
  constexpr int kParts = GATED ? 2 : 1;
  const uint4 dv = i8_load8(p.G + int64_t(row) * p.ldg, k, p.F, p.wide_in != 0);
  const int8_t* q = p.Q + int64_t(row) * kParts * p.pitch + k;
  const float* scale = p.scale + int64_t(row) * kParts * p.blocks + block;
  const uint2 qg = __ldg(reinterpret_cast<const uint2*>(q));
  const float sg = __ldg(scale);
  uint2 qu = make_uint2(0, 0);
  float su = 0.0f;
  if constexpr (GATED) {
    qu = __ldg(reinterpret_cast<const uint2*>(q + p.pitch));
    su = __ldg(scale + p.blocks);
  }
  float d[8], g[8], u[8], dg[8], du[8];
  act_unpack<FP16>(dv, d);
  act_dequant8(qg, sg, g);
  if constexpr (GATED) act_dequant8(qu, su, u);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float value, slope;
    act_value_slope<ACT>(g[j], value, slope);
    dg[j] = GATED ? d[j] * u[j] * slope : d[j] * slope;
    du[j] = d[j] * value;
  }
  uint16_t* y = p.Y + int64_t(row) * p.ldy;
  act_store8(y, k, p.F, act_pack<FP16>(dg), p.wide_out != 0);
  if constexpr (GATED) act_store8(y + p.F, k, p.F, act_pack<FP16>(du), p.wide_out != 0);
}

}  // namespace bsg
