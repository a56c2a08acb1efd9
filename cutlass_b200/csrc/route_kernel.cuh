// Router of a layer of experts: probabilities, the k best experts of every token, per-expert counts, the end rows and the row
// order that the grouped products take, and the balance loss; and the gradient of the logits.
//
//   p = softmax(l);  the k largest logits are chosen, ties to the lower index, -inf never;  w_j = p_j / sum of the chosen, or p_j
//   f_e = counts_e / (n k),  P_e = (1/n) sum_t p_te,  loss = E sum_e f_e P_e        (n tokens that count)
//   dl_i = c p_i (f_i - sum_e f_e p_e) + ...,  c = dloss E / n;   normalised: + w_i (dw_i - sum_j w_j dw_j) on the chosen;
//   not normalised: + p_i (dw_i [chosen] - sum_j p_j dw_j)
//
// Bound by reading the logits (and, backward, writing their gradient) and by the instructions that choose; below a few thousand
// tokens by launches and latency.  A warp owns a token: its lanes hold E / 32 logits each in registers, so one read serves the
// maximum, the choice and the sum.  A lane owns the same experts in every token, so the sums of p over tokens are kept in
// registers too and leave once per warp; they are added in a fixed order (warp, then block), so results do not change from run
// to run.  The row order is a stable counting sort: blocks, and warps inside them, own consecutive tokens, and the k experts of
// a token differ, so a warp counts its rows per expert without atomics and knows the rank of each at once; (1) ranks inside a
// block and counts per block and expert, (2) prefix over blocks, (3) rows.  Up to 16 tokens are one block and up
// to 512 a cluster of eight, which do all three in one launch: a token to a warp, or four, since a token's latency (1 us with 256
// experts) is what counts there.  128 tokens, 256 experts, k = 8: 8.2 us a call, 16.4 in one block; 512 tokens: 12.3, 14 in three
// launches; 1024 tokens: 19.4 and 14.
// 65536 tokens, 256 experts, k = 8, bf16: (1) 32 us (bound by issue; 34 MB are read, 5 us), (2) and (3), which start while it ends,
// 9 more; the gradient 23 us (67 MB, 10 us).  16 tokens, 64 experts: 3.6 and 2.5 us.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "ptx.cuh"

namespace bsg {

constexpr int kRouteThreads = 256;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteOneWarps = 16;           // warps of the block that does a small batch alone
constexpr int kRouteOneTokens = 16;          // one to a warp
constexpr int kRouteClusterCtas = 8;         // such blocks, in one cluster, that do a batch together
constexpr int kRouteClusterTokens = 512;
constexpr int kRouteBlocksMax = 740;         // five blocks for each of 148 SMs
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
  float2* softmax;          // [tokens]: largest logit, 1 / sum of exp(l - largest)
  // scratch
  int32_t* block_counts;    // [experts + 1][pitch]; the last row: tokens that count
  float* block_sums;        // [experts][pitch]
  float* sums;              // [experts]
  int32_t pitch;            // blocks rounded up to 4
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

// One row as it lies in memory, 32 bits at a time (a lone value of 16 bits in the low half): a lane's V values; experts that do
// not exist read as -inf.
template <int TYPE, int V> struct RouteRow {
  static constexpr bool k16 = TYPE != kRouteF32;
  static constexpr int kWords = k16 ? (V + 1) / 2 : V;
  uint32_t w[kWords];
};
template <int TYPE, int V>
__device__ __forceinline__ void route_load(RouteRow<TYPE, V>& r, const void* base, int64_t row_off, int lane, int E, bool wide) {
  using T = typename RouteType<TYPE>::T;
  constexpr int C = RouteMap<V>::C;
  constexpr int kPer = 16 / int(sizeof(T));          // values of a 16-byte load
  constexpr uint32_t kNone = TYPE == kRouteF32 ? 0xFF800000u : TYPE == kRouteF16 ? 0xFC00u : 0xFF80u;      // -inf
  const T* row = static_cast<const T*>(base) + row_off;
#pragma unroll
  for (int g = 0; g < V / C; ++g) {
    const int e0 = g * 32 * C + lane * C;
    if constexpr (C >= kPer) {
      if (wide && e0 + C <= E) {
#pragma unroll
        for (int h = 0; h < C / kPer; ++h) {
          const uint4 u = reinterpret_cast<const uint4*>(row + e0)[h];
          uint32_t* to = r.w + (g * C + h * kPer) * int(sizeof(T)) / 4;
          to[0] = u.x; to[1] = u.y; to[2] = u.z; to[3] = u.w;
        }
        continue;
      }
    }
    uint32_t bits[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      bits[j] = kNone;
      if (e0 + j < E) {
        if constexpr (TYPE == kRouteF32) bits[j] = __float_as_uint(row[e0 + j]);
        else bits[j] = row[e0 + j];
      }
    }
    if constexpr (TYPE == kRouteF32) {
#pragma unroll
      for (int j = 0; j < C; ++j) r.w[g * C + j] = bits[j];
    } else if constexpr (C == 1) {
      r.w[g] = bits[0] | (kNone << 16);
    } else {
#pragma unroll
      for (int j = 0; j < C / 2; ++j) r.w[g * C / 2 + j] = bits[2 * j] | (bits[2 * j + 1] << 16);
    }
  }
}
template <int TYPE, int V>
__device__ __forceinline__ void route_unpack(float (&x)[V], const RouteRow<TYPE, V>& r) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if constexpr (TYPE == kRouteF32) x[v] = __uint_as_float(r.w[v]);
    else if constexpr (TYPE == kRouteF16) x[v] = __half2float(__ushort_as_half(static_cast<unsigned short>(v & 1 ? r.w[v / 2] >> 16 : r.w[v / 2] & 0xFFFFu)));
    else x[v] = __uint_as_float(v & 1 ? r.w[v / 2] & 0xFFFF0000u : r.w[v / 2] << 16);
  }
}

// Order-preserving keys: larger key, larger logit.  The bits of a positive value get the sign bit, those of a negative one are
// inverted.  Adding +0 first makes -0 +0, and every NaN the positive one, which is above all.  -inf and what is below it are never
// chosen.
__device__ __forceinline__ uint32_t route_sign16(uint32_t w) {      // the sign of either half, all over that half
  uint32_t m;
  asm("prmt.b32 %0, %1, 0, 0xBB99;" : "=r"(m) : "r"(w));
  return m;
}
template <int TYPE>
__device__ __forceinline__ uint32_t route_key2(uint32_t w) {        // two values of 16 bits
  if constexpr (TYPE == kRouteF16) {
    const __half2 z = __hadd2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0)));
    w = *reinterpret_cast<const uint32_t*>(&z);
  } else {
    asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(0u));
  }
  return w ^ (route_sign16(w) | 0x80008000u);
}
__device__ __forceinline__ uint32_t route_key(float x) {
  const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
template <int TYPE>
__device__ __forceinline__ constexpr uint32_t route_lowest() {      // the key of -inf (16-bit types: in the upper half, with any expert)
  return TYPE == kRouteF32 ? 0x007FFFFFu : TYPE == kRouteF16 ? 0x03FFFFFFu : 0x007FFFFFu;
}
template <int TYPE>
__device__ __forceinline__ float route_value_of(uint32_t key) {
  if constexpr (TYPE == kRouteF32) return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
  const uint32_t h = key >> 16, bits = h & 0x8000u ? h & 0x7FFFu : ~h & 0xFFFFu;
  if constexpr (TYPE == kRouteF16) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  return __uint_as_float(bits << 16);
}

__device__ __forceinline__ float route_sum(float v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// exp(x - top) for x <= top, off by about 2^-22 + |x - top| 2^-24; below 2^-126 it is 0.
__device__ __forceinline__ float route_exp(float x, float top) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((x - top) * 1.4426950408889634f));
  return y;
}

// Sorting networks, descending (Batcher's odd-even merge sort).
template <int N, class F>
__device__ __forceinline__ void route_network(F exchange) {
#pragma unroll
  for (int p = 1; p < N; p *= 2) {
#pragma unroll
    for (int k = p; k >= 1; k /= 2) {
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k) {
#pragma unroll
        for (int i = 0; i < k; ++i) {
          if (j + i + k < N && (j + i) / (2 * p) == (j + i + k) / (2 * p)) exchange(j + i, j + i + k);
        }
      }
    }
  }
}
template <int N>
__device__ __forceinline__ void route_sort(uint32_t (&key)[N]) {
  route_network<N>([&](int a, int b) {
    const uint32_t hi = max(key[a], key[b]), lo = min(key[a], key[b]);
    key[a] = hi;
    key[b] = lo;
  });
}
template <int N>
__device__ __forceinline__ void route_sort_pairs(uint32_t (&key)[N], uint32_t (&at)[N]) {      // equal keys: lower `at` first
  route_network<N>([&](int a, int b) {
    const bool swap = key[a] < key[b] || (key[a] == key[b] && at[a] > at[b]);
    const uint32_t ka = key[a], kb = key[b], ia = at[a], ib = at[b];
    key[a] = swap ? kb : ka; key[b] = swap ? ka : kb;
    at[a] = swap ? ib : ia; at[b] = swap ? ia : ib;
  });
}

// The k largest of a warp's values, one per round: lane j gets the j-th largest (its value and the lowest expert that has it;
// expert -1 where there is nothing above -inf left).  Up to eight values a lane are sorted first: a lane then shows its largest
// only, and where that is taken the others move up; more of them are searched in every round.
// 16-bit logits: the upper half of a 32-bit word takes the key and the lower half the expert (the lower one larger), so that one
// warp maximum gives both; fp32 logits take a second one, for the expert.  ROUNDS: 2, 4 or 8, at least k, or 0 for k of them;
// known, the rounds are free of branches, and in each only as many values move up as can still be taken.  The integer unit, which
// compares and selects, is what bounds all of this: 65536 tokens, 256 experts, k = 8: 87 us for the kernel when every round
// searched, took two reductions and turned its result back into a value; 72 with packed keys of fp32 width; 42 sorted, with both
// halves of a word made at a time; 32 with known rounds.
template <int TYPE, int V, int ROUNDS>
__device__ __forceinline__ void route_choose(const RouteRow<TYPE, V>& r, int lane, int K, int32_t& my_expert, float& my_logit) {
  constexpr bool kSorted = V <= 8;
  uint32_t won = 0, won_at = 0;
  auto rounds = [&](auto body) {
    if constexpr (ROUNDS > 0) {
#pragma unroll
      for (int j = 0; j < ROUNDS; ++j) body(j, ROUNDS - 1 - j);
    } else {
#pragma unroll 2
      for (int j = 0; j < K; ++j) body(j, V);
    }
  };
  if constexpr (TYPE != kRouteF32) {
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      const uint32_t two = route_key2<TYPE>(r.w[v / 2]);
      key[v] = (two << 16) | uint32_t(kRouteMaxExperts - 1 - RouteMap<V>::expert(lane, v));
      if (v + 1 < V) key[v + 1] = (two & 0xFFFF0000u) | uint32_t(kRouteMaxExperts - 1 - RouteMap<V>::expert(lane, v + 1 < V ? v + 1 : v));
    }
    if constexpr (kSorted) route_sort<V>(key);
    rounds([&](int j, int left) {      // `left` rounds follow
      uint32_t m = key[0];
      if constexpr (!kSorted) {
#pragma unroll
        for (int v = 1; v < V; ++v) m = max(m, key[v]);
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if (lane == j) won = m;
      if constexpr (kSorted) {
        if (key[0] == m) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            if (v < left) key[v] = v + 1 < V ? key[v + 1 < V ? v + 1 : v] : 0u;
          }
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = key[v] == m ? 0u : key[v];
      }
    });
    if ((won | 0xFFFFu) <= route_lowest<TYPE>()) won = 0u;
    won_at = kRouteMaxExperts - 1 - (won & 0xFFFFu);
  } else {
    uint32_t key[V], at[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      key[v] = route_key(__uint_as_float(r.w[v]));
      at[v] = uint32_t(RouteMap<V>::expert(lane, v));
    }
    if constexpr (kSorted) route_sort_pairs<V>(key, at);
    rounds([&](int j, int left) {
      uint32_t m = key[0];
      if constexpr (!kSorted) {
#pragma unroll
        for (int v = 1; v < V; ++v) m = max(m, key[v]);
      }
      m = __reduce_max_sync(0xffffffffu, m);
      uint32_t e = 0xFFFFFFFFu;
      if constexpr (kSorted) {
        e = __reduce_min_sync(0xffffffffu, key[0] == m ? at[0] : e);
        if (key[0] == m && at[0] == e) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            if (v < left) {
              key[v] = v + 1 < V ? key[v + 1 < V ? v + 1 : v] : 0u;
              at[v] = at[v + 1 < V ? v + 1 : v];
            }
          }
        }
      } else {
#pragma unroll
        for (int v = V - 1; v >= 0; --v) e = key[v] == m ? at[v] : e;
        e = __reduce_min_sync(0xffffffffu, e);
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = at[v] == e ? 0u : key[v];
      }
      if (lane == j) {
        won = m;
        won_at = e;
      }
    });
    if (won <= route_lowest<TYPE>()) won = 0u;
  }
  if (ROUNDS > 0 && lane >= K) won = 0u;
  my_expert = won ? int32_t(won_at) : -1;
  my_logit = won ? route_value_of<TYPE>(won) : -INFINITY;
}

// Exclusive prefix of count(e) over the experts, into `base`, by the whole block; returns the sum.
template <int WARPS, class F>
__device__ __forceinline__ int32_t route_prefix(int32_t* base, int32_t* s_warp, int E, F count) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int32_t carry = 0;
  for (int e0 = 0; e0 < E; e0 += WARPS * 32) {
    const int e = e0 + int(threadIdx.x);
    const int32_t c = e < E ? count(e) : 0;
    int32_t upto = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    int32_t before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int32_t n = s_warp[w];
      before += w < warp ? n : 0;
      all += n;
    }
    if (e < E) base[e] = before + upto - c;
    carry = all;
    __syncthreads();
  }
  return carry;
}

// E sum_e (counts_e / (n k)) (sums_e / n) by the whole block; the result is thread 0's.
template <int WARPS, class F>
__device__ __forceinline__ float route_loss(float* s_part, int E, int K, int32_t live, F product) {
  float part = 0.0f;
  for (int e = threadIdx.x; e < E; e += WARPS * 32) part += product(e);
  part = route_sum(part);
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = part;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) s += s_part[w];
  const float n = float(max(live, 1));
  return __fdiv_rn(__fdiv_rn(s * float(E), n), n * float(K));
}

// (1) one warp per token: choice, weights, rank of every row among those of its expert in the block, counts and sums of p per
// block.  CTAS: 0, or that many blocks, one cluster, are all there is and finish everything; they see one another's counts and sums
// through distributed shared memory.
template <int TYPE, int V, int WARPS, int CTAS, int ROUNDS>
__global__ void __launch_bounds__(WARPS * 32) bsg_route_tokens_kernel(const RouteParams p) {
  constexpr bool ONE = CTAS > 0;
  extern __shared__ uint32_t s_route[];
  const int E = p.experts, K = p.k;
  int32_t* s_count = reinterpret_cast<int32_t*>(s_route);                 // [warps][experts]: rows so far, then rows of the warps before
  float* s_sum = reinterpret_cast<float*>(s_route + WARPS * E);           // [warps][experts]
  int32_t* s_base = reinterpret_cast<int32_t*>(s_sum);                    // ONE, once the sums are added up: [experts] first rows,
  int32_t* s_all = s_base + E;                                            // ... rows over all blocks,
  int32_t* s_mine = s_base + 2 * E;                                       // ... this block's rows
  float* s_mine_sum = s_sum + 3 * E;                                      // ... and sums of p
  static_assert(WARPS >= 4, "four arrays in the place of the warps' sums");
  __shared__ int32_t s_live[WARPS];
  __shared__ float s_part[WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < WARPS * E; e += WARPS * 32) s_count[e] = 0;
  __syncthreads();
  ptx::grid_dependency_wait();
  int32_t* my_count = s_count + warp * E;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  // (sums of token numbers, of which there may be 2^31 - 1, are unsigned)
  const uint32_t all = p.tokens, t0 = min(blockIdx.x * uint32_t(p.per_block), all), t1 = min(t0 + p.per_block, all);
  const uint32_t per_warp = (t1 - t0 + WARPS - 1) / WARPS;
  const int a = min(t0 + warp * per_warp, t1), b = min(a + per_warp, t1);
  constexpr bool kAhead = V <= 8;             // the next token's logits are asked for before this one's are used
  int k_lanes = ROUNDS > 0 ? ROUNDS : 1;       // a power of two, at least k
  if constexpr (ROUNDS == 0) {
    while (k_lanes < K) k_lanes <<= 1;
  }
  RouteRow<TYPE, V> raw, next;
  int32_t live_tokens = 0;
  if (a < b) route_load<TYPE, V>(raw, p.logits, int64_t(a) * p.ld, lane, E, p.wide != 0);
  for (int t = a; t < b; ++t) {
    if constexpr (kAhead) {
      if (t + 1 < b) route_load<TYPE, V>(next, p.logits, int64_t(t + 1) * p.ld, lane, E, p.wide != 0);
    }
    int32_t my_expert = -1;
    float my_logit = -INFINITY;
    if (!p.mask || p.mask[t] != 0) route_choose<TYPE, V, ROUNDS>(raw, lane, K, my_expert, my_logit);
    const float top = __shfl_sync(0xffffffffu, my_logit, 0);
    const bool live = __shfl_sync(0xffffffffu, my_expert, 0) >= 0;
    float x[V];
    route_unpack<TYPE, V>(x, raw);
    float w = 0.0f, inv = 0.0f;
    if (live) {
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = route_exp(x[v], top);
        sum += x[v];
      }
      sum = route_sum(sum);
      inv = __fdividef(1.0f, sum);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += x[v] * inv;
      w = my_expert >= 0 ? route_exp(my_logit, top) : 0.0f;
      float chosen = w;
      for (int o = k_lanes >> 1; o >= 1; o >>= 1) chosen += __shfl_xor_sync(0xffffffffu, chosen, o);      // lanes below k hold the slots
      w = p.normalize ? __fdividef(w, chosen) : w * inv;
      if (my_expert < 0) w = 0.0f;
      ++live_tokens;
    }
    if (lane < K) {
      int32_t rank = -1;
      if (my_expert >= 0) {      // the experts of a token differ: no two lanes meet
        rank = my_count[my_expert];
        my_count[my_expert] = rank + 1;
      }
      p.chosen[int64_t(t) * K + lane] = my_expert;
      p.weights[int64_t(t) * K + lane] = w;
      p.positions[int64_t(t) * K + lane] = rank;
    }
    if (lane == 0) p.softmax[t] = make_float2(top, inv);
    __syncwarp();
    if constexpr (kAhead) {
      raw = next;
    } else {
      if (t + 1 < b) route_load<TYPE, V>(raw, p.logits, int64_t(t + 1) * p.ld, lane, E, p.wide != 0);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = RouteMap<V>::expert(lane, v);
    if (e < E) s_sum[warp * E + e] = acc[v];
  }
  if (lane == 0) s_live[warp] = live_tokens;
  ptx::grid_launch_dependents();
  __syncthreads();
  constexpr int kMine = ONE ? (kRouteMaxExperts + WARPS * 32 - 1) / (WARPS * 32) : 1;      // experts of a thread
  int32_t mine[kMine];
  float mine_sum[kMine];
#pragma unroll 1
  for (int e0 = threadIdx.x, n = 0; e0 < E; e0 += WARPS * 32, ++n) {
    int32_t count = 0;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int32_t c = s_count[w * E + e0];
      s_count[w * E + e0] = count;
      count += c;
      sum += s_sum[w * E + e0];
    }
    if constexpr (ONE) {
#pragma unroll
      for (int u = 0; u < kMine; ++u) {
        if (u == n) {
          mine[u] = count;
          mine_sum[u] = sum;
        }
      }
    } else {
      p.block_counts[int64_t(e0) * p.pitch + blockIdx.x] = count;
      p.block_sums[int64_t(e0) * p.pitch + blockIdx.x] = sum;
    }
  }
  int32_t live_all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) live_all += s_live[w];
  if constexpr (!ONE) {
    if (threadIdx.x == 0) p.block_counts[int64_t(E) * p.pitch + blockIdx.x] = live_all;
  }
  __syncthreads();
  int32_t total = 0;
  if constexpr (ONE) {
    __shared__ int32_t s_scan[WARPS];
    __shared__ int32_t s_live_mine;
    const bool first = CTAS == 1 || blockIdx.x == 0;
    int32_t before[kMine] = {};      // rows of an expert in the blocks before this one
    float my_product = 0.0f;         // counts_e sums_e of this thread's experts
    if constexpr (CTAS > 1) {
#pragma unroll
      for (int u = 0; u < kMine; ++u) {
        const int e = u * WARPS * 32 + threadIdx.x;
        if (e < E) {
          s_mine[e] = mine[u];
          s_mine_sum[e] = mine_sum[u];
        }
      }
      if (threadIdx.x == 0) s_live_mine = live_all;
      __syncwarp();      // (the barrier's instructions want a whole warp at once, also below)
      ptx::cluster_arrive();
      ptx::cluster_wait();
      live_all = 0;
#pragma unroll
      for (uint32_t c = 0; c < uint32_t(CTAS); ++c) live_all += int32_t(ptx::ld_shared_cluster_u32(ptx::mapa(ptx::smem_u32(&s_live_mine), c)));
#pragma unroll
      for (int u = 0; u < kMine; ++u) {
        const int e = u * WARPS * 32 + threadIdx.x;
        if (e < E) {
          int32_t count[CTAS];
          float sum[CTAS];
#pragma unroll
          for (uint32_t c = 0; c < uint32_t(CTAS); ++c) {
            count[c] = int32_t(ptx::ld_shared_cluster_u32(ptx::mapa(ptx::smem_u32(s_mine + e), c)));
            sum[c] = __uint_as_float(ptx::ld_shared_cluster_u32(ptx::mapa(ptx::smem_u32(s_mine_sum + e), c)));
          }
          mine[u] = 0;
          mine_sum[u] = 0.0f;
#pragma unroll
          for (int c = 0; c < CTAS; ++c) {
            if (c < int(blockIdx.x)) before[u] += count[c];
            mine[u] += count[c];
            mine_sum[u] += sum[c];
          }
        }
      }
      __syncwarp();
      ptx::cluster_arrive();      // what this block needed of the others it has; it leaves when they have theirs
    }
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      const int e = u * WARPS * 32 + threadIdx.x;
      if (e < E) {
        s_all[e] = mine[u];
        my_product += float(mine[u]) * mine_sum[u];
      }
    }
    total = route_prefix<WARPS>(s_base, s_scan, E, [&](int e) { return s_all[e]; });      // (this thread's own writes)
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      const int e = u * WARPS * 32 + threadIdx.x;
      if (e < E) {
        if (first) {
          p.counts[e] = mine[u];
          p.offsets[e] = s_base[e] + mine[u];
        }
        s_base[e] += before[u];
      }
    }
    my_product = route_sum(my_product);
    if (lane == 0) s_part[warp] = my_product;
    __syncthreads();
    if (first && threadIdx.x == 0) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s += s_part[w];
      const float n = float(max(live_all, 1));
      *p.loss = __fdiv_rn(__fdiv_rn(s * float(E), n), n * float(K));
      *p.live = live_all;
    }
  }
  // this warp's slots: rank in the block, or, where this launch is all, the row
  for (int64_t i = int64_t(a) * K + lane; i < int64_t(b) * K; i += 32) {
    const int32_t e = p.chosen[i];
    if (e >= 0) {
      const int32_t at = p.positions[i] + my_count[e] + (ONE ? s_base[e] : 0);
      p.positions[i] = at;
      if constexpr (ONE) p.rows[at] = int32_t(i / K);
    }
  }
  if constexpr (ONE) {
    for (int64_t r = total + int64_t(blockIdx.x) * WARPS * 32 + threadIdx.x; r < int64_t(p.tokens) * K; r += CTAS * WARPS * 32) p.rows[r] = -1;
    if constexpr (CTAS > 1) {
      __syncwarp();
      ptx::cluster_wait();
    }
  }
}

// (2) one warp per expert (and one for the number of tokens): counts per block become counts of the blocks before.
static __global__ void __launch_bounds__(128) bsg_route_scan_kernel(const RouteParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int e = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int E = p.experts;
  if (e > E) return;
  constexpr int kPieces = (kRouteBlocksMax + 127) / 128;      // of 128 blocks: four per lane; all loads before the first use
  int4 c[kPieces];
  float4 f[kPieces];
  int32_t* counts = p.block_counts + int64_t(e) * p.pitch;
  const float* sums = p.block_sums + int64_t(e) * p.pitch;
  auto piece = [&](int i) { return i * 128 + lane * 4; };
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const bool in = piece(i) < p.pitch;
    c[i] = in ? *reinterpret_cast<const int4*>(counts + piece(i)) : make_int4(0, 0, 0, 0);
    f[i] = in && e < E ? *reinterpret_cast<const float4*>(sums + piece(i)) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  int32_t total = 0;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int left = p.blocks - piece(i);      // what lies behind the last block is not initialised
    const int32_t c0 = left > 0 ? c[i].x : 0, c1 = left > 1 ? c[i].y : 0, c2 = left > 2 ? c[i].z : 0, c3 = left > 3 ? c[i].w : 0;
    sum += (left > 0 ? f[i].x : 0.f) + (left > 1 ? f[i].y : 0.f) + (left > 2 ? f[i].z : 0.f) + (left > 3 ? f[i].w : 0.f);
    const int32_t mine = c0 + c1 + c2 + c3;
    int32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    const int32_t at = total + upto - mine;
    if (piece(i) < p.pitch) *reinterpret_cast<int4*>(counts + piece(i)) = make_int4(at, at + c0, at + c0 + c1, at + c0 + c1 + c2);
    total += __shfl_sync(0xffffffffu, upto, 31);
  }
  sum = route_sum(sum);
  if (lane == 0) {
    if (e < E) { p.counts[e] = total; p.sums[e] = sum; }
    else *p.live = total;
  }
}

// (3) end rows, rows of the slots, loss.
static __global__ void __launch_bounds__(kRouteThreads) bsg_route_order_kernel(const RouteParams p) {
  __shared__ int32_t s_base[kRouteMaxExperts];      // first row of the expert plus the rows of the blocks before
  __shared__ int32_t s_scan[kRouteWarps];
  __shared__ float s_part[kRouteWarps];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int E = p.experts, K = p.k;
  const int64_t slots = int64_t(p.tokens) * K;
  const int64_t i0 = min(int64_t(blockIdx.x) * p.per_block * K, slots), i1 = min(i0 + int64_t(p.per_block) * K, slots);
  constexpr int kAhead = 4;      // slots of a thread whose expert and rank are asked for before the prefix over the experts
  int32_t expert[kAhead], rank[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const int64_t i = i0 + u * kRouteThreads + threadIdx.x;
    expert[u] = i < i1 ? __ldcg(p.chosen + i) : -1;
    rank[u] = i < i1 ? __ldcg(p.positions + i) : 0;
  }
  const int32_t total = route_prefix<kRouteWarps>(s_base, s_scan, E, [&](int e) { return __ldcg(p.counts + e); });
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {      // (the entries this thread has written)
    if (blockIdx.x == 0) p.offsets[e] = s_base[e] + __ldcg(p.counts + e);
    s_base[e] += __ldcg(p.block_counts + int64_t(e) * p.pitch + blockIdx.x);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    const float loss = route_loss<kRouteWarps>(s_part, E, K, __ldcg(p.live), [&](int e) { return float(__ldcg(p.counts + e)) * __ldcg(p.sums + e); });
    if (threadIdx.x == 0) *p.loss = loss;
  }
  auto place = [&](int64_t i, int32_t e, int32_t r) {
    if (e >= 0) {
      const int32_t row = s_base[e] + r;
      p.positions[i] = row;
      p.rows[row] = int32_t(uint32_t(i) / uint32_t(K));
    }
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) place(i0 + u * kRouteThreads + threadIdx.x, expert[u], rank[u]);
  for (int64_t i = i0 + kAhead * kRouteThreads + threadIdx.x; i < i1; i += kRouteThreads) place(i, __ldcg(p.chosen + i), __ldcg(p.positions + i));
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
  int k_lanes = 1;
  while (k_lanes < K) k_lanes <<= 1;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const float n = float(max(*p.live, 1));
  const float c = p.grad_loss ? *p.grad_loss * (float(E) / n) : 0.0f;
  float f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = RouteMap<V>::expert(lane, v);
    f[v] = e < E ? float(p.counts[e]) / (n * float(K)) : 0.0f;
  }
  // what a token needs, asked for one token ahead
  struct Slot { int32_t e; float w, gw; float2 soft; };
  auto slot_of = [&](uint32_t t) {
    Slot s;
    s.e = lane < K ? p.chosen[int64_t(t) * K + lane] : -1;
    s.w = lane < K ? p.weights[int64_t(t) * K + lane] : 0.0f;
    s.gw = lane < K && p.grad_weights ? p.grad_weights[int64_t(t) * K + lane] : 0.0f;
    s.soft = p.softmax[t];
    return s;
  };
  constexpr bool kAhead = V <= 8;
  const uint32_t tokens = p.tokens, step = gridDim.x * kRouteWarps;      // (t + step may pass 2^31)
  uint32_t t = blockIdx.x * kRouteWarps + warp;
  RouteRow<TYPE, V> raw, next;
  Slot slot{}, next_slot{};
  if (t < tokens) {
    route_load<TYPE, V>(raw, p.logits, int64_t(t) * p.ld, lane, E, p.wide != 0);
    slot = slot_of(t);
  }
  for (; t < tokens; t += step) {
    if constexpr (kAhead) {
      if (t + step < tokens) {
        route_load<TYPE, V>(next, p.logits, int64_t(t + step) * p.ld, lane, E, p.wide != 0);
        next_slot = slot_of(t + step);
      }
    }
    const int32_t e = slot.e < E ? slot.e : -1;      // (none behind the experts that the forward pass writes: `part` ends there)
    const float w = e >= 0 ? slot.w : 0.0f, gw = e >= 0 ? slot.gw : 0.0f;
    const float2 soft = slot.soft;
    const bool live = __shfl_sync(0xffffffffu, e, 0) >= 0;
    T* out = static_cast<T*>(p.grad_logits) + int64_t(t) * p.ld_grad;
    float x[V];
    route_unpack<TYPE, V>(x, raw);
    float d[V];
#pragma unroll
    for (int v = 0; v < V; ++v) d[v] = 0.0f;
    if (live) {
#pragma unroll
      for (int v = 0; v < V; ++v) d[v] = route_exp(x[v], soft.x) * soft.y;
      float s2 = w * gw;
      for (int o = k_lanes >> 1; o >= 1; o >>= 1) s2 += __shfl_xor_sync(0xffffffffu, s2, o);      // lanes below k hold the slots
      s2 = __shfl_sync(0xffffffffu, s2, 0);
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
    if constexpr (kAhead) {
      raw = next;
      slot = next_slot;
    } else if (t + step < tokens) {
      route_load<TYPE, V>(raw, p.logits, int64_t(t + step) * p.ld, lane, E, p.wide != 0);
      slot = slot_of(t + step);
    }
  }
}

}  // namespace bsg
