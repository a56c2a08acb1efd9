// Router of a layer of experts: probabilities, the k best experts of every token, per-expert counts, the end rows and the row
// order that the grouped products take, and the balance loss; and the gradient of the logits.
//
//   p = softmax(l);  the k largest logits are chosen, ties to the lower index, -inf never;  w_j = p_j / sum of the chosen, or p_j
//   f_e = counts_e / (n k),  P_e = (1/n) sum_t p_te,  loss = E sum_e f_e P_e        (n tokens that count)
//   dl_i = c p_i (f_i - sum_e f_e p_e) + ...,  c = dloss E / n;   normalised: + w_i (dw_i - sum_j w_j dw_j) on the chosen;
//   not normalised: + p_i (dw_i [chosen] - sum_j p_j dw_j)
//
// Bound by reading the logits (and, backward, writing their gradient); below a few thousand tokens by launches and latency.
// A warp owns a token: its lanes hold E / 32 logits each in registers, so one read serves the maximum, the choice and the sum.
// A lane owns the same experts in every token, so the sums of p over tokens are kept in registers too and leave once per warp;
// they are added in a fixed order (warp, then block), so results do not change from run to run.
// The row order is a stable counting sort: blocks own consecutive tokens; (1) counts per block and expert, (2) prefix over
// blocks, (3) positions, with ranks inside a block from __match_any_sync over 32 slots at a time.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "ptx.cuh"

namespace bsg {

constexpr int kRouteThreads = 256;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 32;

struct RouteParams {
  const void* logits;
  int64_t ld;               // elements
  const uint8_t* mask;      // [tokens] 0: does not count; or null
  int32_t tokens, experts, k;
  int32_t normalize;
  int32_t wide;             // rows of the logits start on 16-byte boundaries
  int32_t blocks, per_block;      // blocks of the token kernel, tokens per block
  int32_t* chosen;          // [tokens][k]
  float* weights;           // [tokens][k]
  int32_t* counts;          // [experts]
  int32_t* offsets;         // [experts]
  int32_t* rows;            // [tokens * k]
  int32_t* positions;       // [tokens][k]
  float* loss;              // [1]
  int32_t* live;            // [1]: tokens that count
  // scratch
  int32_t* block_counts;    // [blocks][experts + 1]; the last entry: tokens that count
  float* block_sums;        // [blocks][experts]
  float* sums;              // [experts]
  // backward
  const float* grad_weights;    // [tokens][k] or null
  const float* grad_loss;       // [1] or null
  void* grad_logits;
  int64_t ld_grad;
  int32_t wide_grad;
};

enum { kRouteBf16 = 0, kRouteF16 = 1, kRouteF32 = 2 };
template <int TYPE> struct RouteType { using T = uint16_t; };
template <> struct RouteType<kRouteF32> { using T = float; };

template <int TYPE>
__device__ __forceinline__ float route_value(typename RouteType<TYPE>::T v) {
  if constexpr (TYPE == kRouteF32) return v;
  else if constexpr (TYPE == kRouteF16) return __half2float(__ushort_as_half(v));
  else return __uint_as_float(uint32_t(v) << 16);
}

// The V values of a lane: groups of C = min(V, 8) consecutive experts, a group every 32 C.
template <int V> struct RouteMap {
  static constexpr int C = V < 8 ? V : 8;
  __device__ static __forceinline__ int expert(int lane, int v) { return (v / C) * 32 * C + lane * C + v % C; }
};

// Values of one row; experts that do not exist read as -inf.
template <int TYPE, int V>
__device__ __forceinline__ void route_load(float (&x)[V], const void* base, int64_t row_off, int lane, int E, bool wide) {
  using T = typename RouteType<TYPE>::T;
  constexpr int C = RouteMap<V>::C;
  constexpr int kPer = 16 / int(sizeof(T));          // values of a 16-byte load
  const T* row = static_cast<const T*>(base) + row_off;
#pragma unroll
  for (int g = 0; g < V / C; ++g) {
    const int e0 = g * 32 * C + lane * C;
    if constexpr (C >= kPer) {
      if (wide && e0 + C <= E) {
#pragma unroll
        for (int h = 0; h < C / kPer; ++h) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + e0) + h);
          const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
          for (int j = 0; j < kPer; ++j) x[g * C + h * kPer + j] = route_value<TYPE>(t[j]);
        }
        continue;
      }
    }
#pragma unroll
    for (int j = 0; j < C; ++j) x[g * C + j] = e0 + j < E ? route_value<TYPE>(__ldg(row + e0 + j)) : -INFINITY;
  }
}

// Order-preserving key of a logit: larger key, larger logit; NaN above all, -inf 0 (never chosen).
__device__ __forceinline__ uint32_t route_key(float x) {
  const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));       // -0 and +0 are one value
  if (x != x) return 0xFFFFFFFFu;
  if (u == 0xFF800000u) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float route_unkey(uint32_t key) {
  if (key == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  if (key == 0u) return -INFINITY;
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ float route_sum(float v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Probabilities of a row whose largest logit is `top` (0 everywhere for a row that does not count).  Returns nothing but p.
template <int V>
__device__ __forceinline__ void route_softmax(float (&p)[V], const float (&x)[V], float top) {
  float sum = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    p[v] = expf(x[v] - top);
    sum += p[v];
  }
  sum = route_sum(sum);
  const float inv = __fdiv_rn(1.0f, sum);
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] *= inv;
}

// (1) one warp per token: choice, weights, counts and sums of p per block.
template <int TYPE, int V>
__global__ void __launch_bounds__(kRouteThreads) bsg_route_tokens_kernel(const RouteParams p) {
  extern __shared__ uint32_t s_route[];
  int32_t* s_count = reinterpret_cast<int32_t*>(s_route);                 // [experts + 1]
  float* s_sum = reinterpret_cast<float*>(s_route + p.experts + 1);       // [warps][experts]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = p.experts, K = p.k;
  for (int e = threadIdx.x; e <= E; e += kRouteThreads) s_count[e] = 0;
  __syncthreads();
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  const int t0 = blockIdx.x * p.per_block, t1 = min(t0 + p.per_block, p.tokens);
  for (int t = t0 + warp; t < t1; t += kRouteWarps) {
    float x[V];
    route_load<TYPE, V>(x, p.logits, int64_t(t) * p.ld, lane, E, p.wide != 0);
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = route_key(x[v]);
    const bool counted = !p.mask || p.mask[t] != 0;
    // k rounds: largest key of the warp, then the lowest expert that has it
    int32_t my_expert = -1;
    float my_logit = -INFINITY, top = -INFINITY;
    for (int j = 0; j < K; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) best = max(best, key[v]);
      best = __reduce_max_sync(0xffffffffu, best);
      if (best == 0u || !counted) break;
      uint32_t e = 0xFFFFFFFFu;
#pragma unroll
      for (int v = V - 1; v >= 0; --v) {
        if (key[v] == best) e = uint32_t(RouteMap<V>::expert(lane, v));
      }
      e = __reduce_min_sync(0xffffffffu, e);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (uint32_t(RouteMap<V>::expert(lane, v)) == e) key[v] = 0u;
      }
      const float value = route_unkey(best);
      if (j == 0) top = value;
      if (lane == j) { my_expert = int32_t(e); my_logit = value; }
    }
    const bool live = __shfl_sync(0xffffffffu, my_expert, 0) >= 0;
    float w = 0.0f;
    if (live) {
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = expf(x[v] - top);
        sum += x[v];
      }
      sum = route_sum(sum);
      const float inv = __fdiv_rn(1.0f, sum);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += x[v] * inv;
      w = my_expert >= 0 ? expf(my_logit - top) : 0.0f;
      w = p.normalize ? __fdiv_rn(w, route_sum(w)) : w * inv;
      if (lane < K && my_expert < 0) w = 0.0f;
      if (lane == 0) atomicAdd(s_count + E, 1);
      if (my_expert >= 0) atomicAdd(s_count + my_expert, 1);
    }
    if (lane < K) {
      p.chosen[int64_t(t) * K + lane] = my_expert;
      p.weights[int64_t(t) * K + lane] = w;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = RouteMap<V>::expert(lane, v);
    if (e < E) s_sum[warp * E + e] = acc[v];
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += kRouteThreads) p.block_counts[int64_t(blockIdx.x) * (E + 1) + e] = s_count[e];
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {
    float s = 0.0f;
    for (int w = 0; w < kRouteWarps; ++w) s += s_sum[w * E + e];
    p.block_sums[int64_t(blockIdx.x) * E + e] = s;
  }
}

// (2) one warp per expert (and one for the number of tokens): counts per block become counts of the blocks before.
static __global__ void __launch_bounds__(kRouteThreads) bsg_route_scan_kernel(const RouteParams p) {
  const int e = blockIdx.x * kRouteWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int E = p.experts;
  if (e > E) return;
  int32_t total = 0;
  float sum = 0.0f;
  for (int b0 = 0; b0 < p.blocks; b0 += 32) {
    const int b = b0 + lane;
    const bool in = b < p.blocks;
    const int32_t c = in ? p.block_counts[int64_t(b) * (E + 1) + e] : 0;
    int32_t upto = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    if (in) p.block_counts[int64_t(b) * (E + 1) + e] = total + upto - c;
    total += __shfl_sync(0xffffffffu, upto, 31);
    if (e < E && in) sum += p.block_sums[int64_t(b) * E + e];
  }
  sum = route_sum(sum);
  if (lane == 0) {
    if (e < E) { p.counts[e] = total; p.sums[e] = sum; }
    else *p.live = total;
  }
}

// (3) end rows, positions, row order, loss.
static __global__ void __launch_bounds__(kRouteThreads) bsg_route_order_kernel(const RouteParams p) {
  extern __shared__ int32_t s_order[];
  const int E = p.experts, K = p.k;
  int32_t* s_base = s_order;                 // [experts]: first row of the expert plus the rows of the blocks before
  int32_t* s_next = s_order + E;             // [warps][experts]
  __shared__ int32_t s_warp[kRouteWarps];
  __shared__ float s_loss[kRouteWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t slots = int64_t(p.tokens) * K;
  // exclusive prefix of the counts over the experts
  int32_t carry = 0;
  for (int e0 = 0; e0 < E; e0 += kRouteThreads) {
    const int e = e0 + int(threadIdx.x);
    const int32_t c = e < E ? p.counts[e] : 0;
    int32_t upto = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    int32_t before = carry, all = carry;
    for (int w = 0; w < kRouteWarps; ++w) {
      if (w < warp) before += s_warp[w];
      all += s_warp[w];
    }
    if (e < E) {
      s_base[e] = before + upto - c + p.block_counts[int64_t(blockIdx.x) * (E + 1) + e];
      if (blockIdx.x == 0) p.offsets[e] = before + upto;
    }
    carry = all;
    __syncthreads();
  }
  const int32_t total = carry;
  if (blockIdx.x == 0) {
    float part = 0.0f;
    for (int e = threadIdx.x; e < E; e += kRouteThreads) part += float(p.counts[e]) * p.sums[e];
    part = route_sum(part);
    if (lane == 0) s_loss[warp] = part;
    __syncthreads();
    if (threadIdx.x == 0) {
      float s = 0.0f;
      for (int w = 0; w < kRouteWarps; ++w) s += s_loss[w];
      const float n = float(max(*p.live, 1));
      *p.loss = __fdiv_rn(__fdiv_rn(s * float(E), n), n * float(K));
    }
  }
  // slots of this block in token order, a consecutive run per warp
  const int64_t i0 = min(int64_t(blockIdx.x) * p.per_block * K, slots), i1 = min(i0 + int64_t(p.per_block) * K, slots);
  const int64_t per_warp = ((i1 - i0 + kRouteWarps - 1) / kRouteWarps + 31) / 32 * 32;
  const int64_t a = min(i0 + warp * per_warp, i1), b = min(a + per_warp, i1);
  for (int e = threadIdx.x; e < kRouteWarps * E; e += kRouteThreads) s_next[e] = 0;
  __syncthreads();
  for (int64_t i = a + lane; i < b; i += 32) {
    const int32_t e = p.chosen[i];
    if (e >= 0) atomicAdd(s_next + warp * E + e, 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {
    int32_t at = s_base[e];
    for (int w = 0; w < kRouteWarps; ++w) {
      const int32_t c = s_next[w * E + e];
      s_next[w * E + e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int64_t i = a; i < b; i += 32) {
    const int64_t s = i + lane;
    const int32_t e = s < b ? p.chosen[s] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    int32_t row = -1;
    if (e >= 0) row = s_next[warp * E + e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0 && (same >> lane) == 1u) s_next[warp * E + e] = row + 1;       // the last lane of the expert
    __syncwarp();
    if (s < b) p.positions[s] = row;
    if (row >= 0) p.rows[row] = int32_t(s / K);
  }
  // rows behind the last one belong to nobody
  for (int64_t r = total + int64_t(blockIdx.x) * kRouteThreads + threadIdx.x; r < slots; r += int64_t(gridDim.x) * kRouteThreads) p.rows[r] = -1;
}

// Gradient of the logits; one warp per token.
template <int TYPE, int V>
__global__ void __launch_bounds__(kRouteThreads) bsg_route_backward_kernel(const RouteParams p) {
  extern __shared__ float s_part[];                  // [warps][experts rounded up to 4]
  using T = typename RouteType<TYPE>::T;
  constexpr int C = RouteMap<V>::C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = p.experts, K = p.k;
  const int pitch = 32 * V;
  float* part = s_part + warp * pitch;
  for (int e = lane; e < pitch; e += 32) part[e] = 0.0f;
  __syncwarp();
  const float n = float(max(*p.live, 1));
  const float c = p.grad_loss ? *p.grad_loss * (float(E) / n) : 0.0f;
  float f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = RouteMap<V>::expert(lane, v);
    f[v] = e < E ? float(p.counts[e]) / (n * float(K)) : 0.0f;
  }
  for (int t = blockIdx.x * kRouteWarps + warp; t < p.tokens; t += gridDim.x * kRouteWarps) {
    float x[V];
    route_load<TYPE, V>(x, p.logits, int64_t(t) * p.ld, lane, E, p.wide != 0);
    const int32_t e = lane < K ? p.chosen[int64_t(t) * K + lane] : -1;
    const float w = e >= 0 ? p.weights[int64_t(t) * K + lane] : 0.0f;
    const float gw = e >= 0 && p.grad_weights ? p.grad_weights[int64_t(t) * K + lane] : 0.0f;
    const bool live = __shfl_sync(0xffffffffu, e, 0) >= 0;
    T* out = static_cast<T*>(p.grad_logits) + int64_t(t) * p.ld_grad;
    float d[V];
#pragma unroll
    for (int v = 0; v < V; ++v) d[v] = 0.0f;
    if (live) {
      float top = -INFINITY;
      bool nan = false;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        nan |= x[v] != x[v];
        top = fmaxf(top, x[v]);
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (__any_sync(0xffffffffu, nan)) top = __uint_as_float(0x7FC00000u);
      route_softmax<V>(d, x, top);
      const float s2 = route_sum(w * gw);
      float s1 = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) s1 += f[v] * d[v];
      s1 = route_sum(s1);
      if (e >= 0) part[e] = p.normalize ? w * (gw - s2) : w * gw;
      __syncwarp();
      const float s0 = p.normalize ? 0.0f : s2;
#pragma unroll
      for (int v = 0; v < V; ++v) d[v] = d[v] * (c * (f[v] - s1) - s0) + part[RouteMap<V>::expert(lane, v)];
      __syncwarp();
      if (e >= 0) part[e] = 0.0f;
    }
#pragma unroll
    for (int g = 0; g < V / C; ++g) {
      const int e0 = g * 32 * C + lane * C;
      constexpr int kPer = 16 / int(sizeof(T));
      if constexpr (C >= kPer) {
        if (p.wide_grad && e0 + C <= E) {
#pragma unroll
          for (int h = 0; h < C / kPer; ++h) {
            const float* y = d + g * C + h * kPer;
            uint4 u;
            if constexpr (TYPE == kRouteF32) u = make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
            else if constexpr (TYPE == kRouteF16) u = make_uint4(pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3]), pack_f16x2(y[4], y[5]), pack_f16x2(y[6], y[7]));
            else u = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
            *(reinterpret_cast<uint4*>(out + e0) + h) = u;
          }
          continue;
        }
      }
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if (e0 + j < E) {
          if constexpr (TYPE == kRouteF32) out[e0 + j] = d[g * C + j];
          else if constexpr (TYPE == kRouteF16) out[e0 + j] = __half_as_ushort(__float2half_rn(d[g * C + j]));
          else out[e0 + j] = __bfloat16_as_ushort(__float2bfloat16_rn(d[g * C + j]));
        }
      }
    }
  }
}

}  // namespace bsg
