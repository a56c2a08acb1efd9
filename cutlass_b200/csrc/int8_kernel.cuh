// Matrix product in 8-bit integers with one scale per token (row of A) and one per output channel (row of B):
//
//   q[m,k] = sign(x) floor(127 |x[m,k]| / a_m + 1/2),  a_m = max_k |x[m,k]|,  sa[m] = a_m / 127
//   D[m,n] = act(sa[m] * sb[n] * sum_k q[m,k] w[n,k] + bias[n])
//
// The sum is a 32-bit integer and exact (K <= 131071: 127 * 128 * K < 2^31), so neither the order of the additions nor
// a split of K changes a result.  The kernels:
//
//   bsg_i8_quant_kernel   tokens -> 8 bits; bound by HBM (8192 x 8192: 34 us, 5.9 TB/s)
//   bsg_i8_rows_kernel    many rows: tokens are the M side of the MMA; bound by the tensor pipe (8192^3: 316 us)
//   bsg_i8_few_kernel     few rows: the output channels are the M side of the MMA and the tokens its N side, so that the
//                         tile carries no padding rows; bound by reading the weights (32 rows in 64 experts, 7168 x 2048:
//                         61 us, 6.1 TB/s), for one dense tile per CTA by latency (17 x 14336 x 4096: 14 us, 4.2 TB/s)
//   bsg_i8_token_kernel   up to four tokens, quantised on the way; bound by reading the weights and by latency (one token,
//                         4096 x 4096: 4.9 us a call, 3.4 TB/s)
//
// The two products are dense (one group of rows) or grouped (ragged rows per group, end rows on the device).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "gemm_kernel.cuh"
#include "ptx.cuh"

namespace bsg {

constexpr int kI8MaxK = 131071;

// ------------------------------------------------------------------------------------------------ quantiser
struct I8QuantParams {
  const uint16_t* X;         // bf16 or fp16 bits
  const int32_t* index;      // row r of Q is made from row index[r] of X; null: from row r
  int8_t* Q;
  float* scale;
  int64_t ldx, ldq;          // elements
  int32_t rows, tokens, K;
};

__device__ __forceinline__ float i8_unpack(uint32_t bits16, bool fp16) {
  return fp16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(bits16))) : __uint_as_float(bits16 << 16);
}

// max(|a|, |b|) of two packed pairs; a NaN operand gives NaN.  (The sign bits of the result are not meaningful.)
template <bool FP16>
__device__ __forceinline__ uint32_t i8_maxabs2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (FP16) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a & 0x7FFF7FFFu), "r"(b & 0x7FFF7FFFu));
  else asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Levels.  `inv` is 127 / amax, enlarged by 2^-21: the distance of 127 |x| / amax from the next half k + 1/2 is 0 or, for 16-bit
// x and amax, at least 2^-19 of its size (254 |x| - (2k + 1) amax is a multiple of the smaller operand's last place), so the
// enlarged ratio, in which `inv` is off by at most 2^-22, lies above every half that the exact ratio reaches and below every
// half that it does not: rounding to nearest gives floor(127 |x| / amax + 1/2) without a division per value.  The rounding is
// that of one fused multiply-add with 1.5 * 2^23, whose last byte is then the level in two's complement.
struct I8Scale {
  float inv;       // 127 / (amax * pre), enlarged; 0 for a row of zeros
  float pre;       // 2^64 for rows so small that 127 / amax leaves fp32's range, 2^-64 for rows so large that 1 / amax may be
                   // subnormal, which has fewer bits, else 1
  uint32_t keep;   // all ones; 0 for a row that holds a NaN or an infinity, whose levels are 0
};
__device__ __forceinline__ float i8_rcp(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));      // off by at most 2^-23 where the result is normal (x up to 2^126)
  return r;
}
__device__ __forceinline__ I8Scale i8_scale(float amax) {
  I8Scale s;
  const bool finite = amax < __uint_as_float(0x7F800000u);
  s.keep = finite ? 0xFFFFFFFFu : 0u;
  s.pre = amax < 0x1p-64f ? 0x1p64f : amax > 0x1p64f ? 0x1p-64f : 1.0f;
  s.inv = amax > 0.0f && finite ? __fmul_rn(i8_rcp(__fmul_rn(amax, s.pre)), 127.0f * (1.0f + 0x1p-21f)) : 0.0f;
  return s;
}
// amax / 127; NaN for a row that holds a NaN or an infinity.
__device__ __forceinline__ float i8_step(float amax) {
  return amax < __uint_as_float(0x7F800000u) ? __fdiv_rn(amax, 127.0f) : __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ uint32_t i8_level_bits(float x, float inv) { return __float_as_uint(__fmaf_rn(x, inv, 12582912.0f)); }

// 32 bytes that start on a 16-byte boundary -> the 16 of them that start `skip` bytes in (skip even, below 16).
__device__ __forceinline__ uint4 i8_shift16(const uint4& lo, const uint4& hi, uint32_t skip) {
  uint32_t w[7] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z}, last = hi.w;
  const bool two = skip & 8u, one = skip & 4u;
  uint32_t v[6];
#pragma unroll
  for (int j = 0; j < 5; ++j) v[j] = two ? w[j + 2] : w[j];
  v[5] = two ? last : w[5];
  uint32_t u[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) u[j] = one ? v[j + 1] : v[j];
  const uint32_t bits = (skip & 2u) * 8u;
  return make_uint4(__funnelshift_r(u[0], u[1], bits), __funnelshift_r(u[1], u[2], bits), __funnelshift_r(u[2], u[3], bits), __funnelshift_r(u[3], u[4], bits));
}

// Eight consecutive values of a row, zeros past its end, in two steps, so that many loads are under way before the first is
// looked at.  WIDE: rows start on 16 bytes and K is a multiple of 8 where it ends inside a group.  Otherwise the one or two
// aligned 16-byte words that hold the values are read whole: a word with at least one value of the row lies in the row's
// allocation (and on its page), whose bounds are multiples of 16.
// (Ordinary loads: what a kernel reads may be written by the one before it until it has waited for that one.)
struct I8Raw { uint4 lo, hi; };
template <bool WIDE>
__device__ __forceinline__ I8Raw i8_raw8(const uint16_t* row, int32_t k, int32_t K) {
  I8Raw r;
  r.lo = r.hi = make_uint4(0, 0, 0, 0);
  if constexpr (WIDE) {
    if (k < K) r.lo = *reinterpret_cast<const uint4*>(row + k);
  } else {
    const uintptr_t a = reinterpret_cast<uintptr_t>(row + k);
    const uint4* at = reinterpret_cast<const uint4*>(a & ~uintptr_t(15));
    if (k < K) r.lo = *at;
    if (k < K && reinterpret_cast<const uint16_t*>(at + 1) < row + K) r.hi = at[1];
  }
  return r;
}
template <bool WIDE>
__device__ __forceinline__ uint4 i8_fix8(const I8Raw& r, const uint16_t* row, int32_t k, int32_t K) {
  if constexpr (WIDE) return r.lo;
  uint4 v = i8_shift16(r.lo, r.hi, uint32_t(reinterpret_cast<uintptr_t>(row + k)) & 15u);
  if (k + 8 > K) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] &= (k + 2 * j < K ? 0xFFFFu : 0u) | (k + 2 * j + 1 < K ? 0xFFFF0000u : 0u);
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
template <bool WIDE>
__device__ __forceinline__ uint4 i8_load8(const uint16_t* row, int32_t k, int32_t K) { return i8_fix8<WIDE>(i8_raw8<WIDE>(row, k, K), row, k, K); }

// Two packed 16-bit values to fp32.
template <bool FP16>
__device__ __forceinline__ void i8_unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (FP16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x; hi = f.y;
  } else {
    lo = __uint_as_float(w << 16); hi = __uint_as_float(w & 0xFFFF0000u);
  }
}
template <bool FP16>
__device__ __forceinline__ uint2 i8_levels8(const uint4& v, const I8Scale& s) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) i8_unpack2<FP16>(w[j], x[2 * j], x[2 * j + 1]);
  if (!FP16 && s.pre != 1.0f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(x[j], s.pre);
  }
  uint32_t q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = i8_level_bits(x[j], s.inv);
  const uint32_t lo = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  const uint32_t hi = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
  return make_uint2(lo & s.keep, hi & s.keep);
}

// TPR threads own a row; a thread holds kI8Chunks groups of 8 values in registers between the maximum and the rounding, so
// a row of up to TPR * 64 values is read once.  Longer rows are read a second time (from L2).
constexpr int kI8Chunks = 8;
constexpr int kI8QuantThreads = 256;
template <int TPR, bool FP16, bool WIDE>
__global__ void __launch_bounds__(TPR > kI8QuantThreads ? TPR : kI8QuantThreads) bsg_i8_quant_kernel(const I8QuantParams p) {
  constexpr int kThreads = TPR > kI8QuantThreads ? TPR : kI8QuantThreads;
  constexpr int kRows = kThreads / TPR;
  const int t = threadIdx.x % TPR;
  const int32_t r = blockIdx.x * kRows + threadIdx.x / TPR;
  __shared__ float s_max[kThreads / 32];
  // The product behind may start its set-up now (and fetch weights: what it reads besides this kernel's results is older, and
  // complete, since this kernel has waited first).
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const bool row_ok = r < p.rows;
  int32_t src = r;
  if (row_ok && p.index) src = p.index[r];
  const bool src_ok = row_ok && src >= 0 && src < p.tokens;
  const uint16_t* row = p.X + (src_ok ? int64_t(src) * p.ldx : 0);
  const int32_t K = src_ok ? p.K : 0;
  uint4 v[kI8Chunks];
  uint32_t m = 0;
  {
    I8Raw raw[kI8Chunks];
#pragma unroll
    for (int c = 0; c < kI8Chunks; ++c) raw[c] = i8_raw8<WIDE>(row, (c * TPR + t) * 8, K);
#pragma unroll
    for (int c = 0; c < kI8Chunks; ++c) v[c] = i8_fix8<WIDE>(raw[c], row, (c * TPR + t) * 8, K);
  }
#pragma unroll
  for (int c = 0; c < kI8Chunks; ++c) {
    if (c * TPR * 8 < K) m = i8_maxabs2<FP16>(m, i8_maxabs2<FP16>(i8_maxabs2<FP16>(v[c].x, v[c].y), i8_maxabs2<FP16>(v[c].z, v[c].w)));
  }
  for (int32_t k = (kI8Chunks * TPR + t) * 8; k < K; k += TPR * 8) {
    const uint4 u = i8_load8<WIDE>(row, k, K);
    m = i8_maxabs2<FP16>(m, i8_maxabs2<FP16>(i8_maxabs2<FP16>(u.x, u.y), i8_maxabs2<FP16>(u.z, u.w)));
  }
  m &= 0x7FFF7FFFu;
  float amax = ptx::fmax_nan(i8_unpack(m & 0xFFFFu, FP16), i8_unpack(m >> 16, FP16));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) amax = ptx::fmax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
    __syncthreads();
    const int w0 = (threadIdx.x / TPR) * (TPR / 32);
    amax = s_max[w0];
#pragma unroll
    for (int w = 1; w < TPR / 32; ++w) amax = ptx::fmax_nan(amax, s_max[w0 + w]);
  }
  if (!row_ok) return;
  const I8Scale s = i8_scale(amax);
  // a row whose index names no token: zeros with a NaN scale, so that a product that uses it shows it
  if (t == 0) p.scale[r] = src_ok ? i8_step(amax) : __uint_as_float(0x7FC00000u);
  int8_t* out = p.Q + int64_t(r) * p.ldq;
  auto store = [&](int32_t k, const uint4& u) {
    const uint2 q = i8_levels8<FP16>(u, s);
    if (k + 8 <= p.K) {      // (rows of Q start on 16 bytes)
      *reinterpret_cast<uint2*>(out + k) = q;
    } else {
      for (int j = 0; j < 8 && k + j < p.K; ++j) out[k + j] = int8_t((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
    }
  };
#pragma unroll
  for (int c = 0; c < kI8Chunks; ++c) {
    const int32_t k = (c * TPR + t) * 8;
    if (k < p.K) store(k, v[c]);
  }
  for (int32_t k = (kI8Chunks * TPR + t) * 8; k < p.K; k += TPR * 8) store(k, i8_load8<WIDE>(row, k, K));
}

// Rows of quantised tokens, and their scales, copied into the order of an index: one warp per row, so that a token that
// several rows use is quantised once.  Entries that name no token: zeros with the scale NaN.
struct I8CopyParams {
  const int8_t* Q;
  const float* scale;
  const int32_t* index;
  int8_t* out;
  float* out_scale;
  int32_t rows, tokens, pitch, words;      // bytes between rows, a multiple of 16; 16-byte words of a row
};
static __global__ void __launch_bounds__(256) bsg_i8_copy_rows_kernel(const I8CopyParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int32_t r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= p.rows) return;
  const int32_t at = p.index[r];
  const bool ok = at >= 0 && at < p.tokens;
  const uint4* src = reinterpret_cast<const uint4*>(p.Q + (ok ? int64_t(at) * p.pitch : 0));
  uint4* dst = reinterpret_cast<uint4*>(p.out + int64_t(r) * p.pitch);
  const int32_t n = p.words;
  for (int32_t i0 = 0; i0 < n; i0 += 32 * 8) {
    uint4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int32_t i = i0 + u * 32 + lane;
      v[u] = ok && i < n ? __ldcg(src + i) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int32_t i = i0 + u * 32 + lane;
      if (i < n) dst[i] = v[u];
    }
  }
  if (lane == 0) p.out_scale[r] = ok ? __ldcg(p.scale + at) : __uint_as_float(0x7FC00000u);
}

// ------------------------------------------------------------------------------------------------ products
// Barriers and loads of tensor memory are instructions of whole warps (.aligned): a __syncwarp stands before each.
struct I8GemmParams {
  int32_t num_groups;         // 1 for a dense product
  int32_t total_rows, N, K;
  const int32_t* offsets;     // grouped: end row of each group (device); null: one group with all rows
  int32_t tiles_n, band;
  int32_t out_kind;           // kOutBf16, kOutF16 or kOutF32
  int32_t activation;
  int32_t tma_out;            // rows kernel: D's address and pitch allow TMA stores
  int32_t tma_edge;           // ... and a row is whole 16-byte pieces: a store that crosses the last column writes up to the next
                              // 16-byte boundary, so otherwise the last columns are copied
  const float* sa;            // [total_rows]
  const float* sb;            // [num_groups][N]
  const float* bias;          // [num_groups][N] or null
  void* D;
  int64_t ldd;                // elements
  uint32_t* status;
};

struct alignas(16) I8Ctl {
  uint64_t full[8];
  uint64_t empty[8];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint32_t tmem_base;
  volatile uint32_t abort;
  int32_t total_tiles;
  int32_t pad;
  int32_t tile_start[kMaxGroups + 1];
  int32_t end[kMaxGroups];
  uint16_t order[kMaxGroups];      // sorted walk: the group at every place
};
constexpr int kI8CtlBytes = (int(sizeof(I8Ctl)) + 127) / 128 * 128;

static __device__ __noinline__ uint32_t i8_slow_wait(uint32_t bar, uint32_t parity, I8Ctl* ctl) {
  const long long t0 = clock64();
  while (true) {
    if (ptx::mbar_spin(bar, parity, 64)) return 1;
    if (clock64() - t0 > (ctl->abort ? 40000ll : 4000000000ll)) break;      // ~20 us once aborting, else ~2 s
  }
  ctl->abort = 1;
  return 0;
}
// Bounded wait; `dead` makes later waits of this thread short once one has run out.
__device__ __forceinline__ void i8_wait(uint32_t bar, uint32_t parity, I8Ctl* ctl, uint32_t& dead) {
  uint32_t ok = ptx::mbar_spin(bar, parity, dead ? 16u : 100000u);
  if (!ok) {
    ok = dead ? 0u : i8_slow_wait(bar, parity, ctl);
    if (!ok) dead = 1;
  }
}

// kind::i8: signed 8-bit operands, 32-bit integer accumulator, K = 32 per instruction.
template <int CG>
__device__ __forceinline__ void i8_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__host__ __device__ constexpr uint32_t i8_idesc(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);      // D s32, A s8, B s8, both K-major
}
__device__ __forceinline__ void i8_tmem_ld_x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

// Group table, built by one whole warp: end row and first tile of every group.  End rows that fall, or that leave
// [0, total_rows], are clamped and reported.
__device__ __forceinline__ void i8_build_groups(I8Ctl* ctl, const I8GemmParams& p, int32_t tile_rows) {
  const int lane = threadIdx.x & 31;
  int32_t prev_end = 0, tiles = 0;
  bool bad = false;
  for (int base = 0; base < p.num_groups; base += 32) {
    const int g = base + lane;
    const bool in = g < p.num_groups;
    const int32_t raw = !in ? 0 : p.offsets ? __ldg(p.offsets + g) : p.total_rows;
    int32_t end = min(max(raw, 0), p.total_rows);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t up = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end = max(end, up);
    }
    end = max(end, prev_end);
    if (in && end != raw) bad = true;
    int32_t begin = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) begin = prev_end;
    const int32_t mine = in ? ((end - begin + tile_rows - 1) / tile_rows) * p.tiles_n : 0;
    int32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    if (in) {
      ctl->end[g] = end;
      ctl->tile_start[g] = tiles + upto - mine;
    }
    tiles += __shfl_sync(0xffffffffu, upto, 31);
    prev_end = __shfl_sync(0xffffffffu, end, 31);
  }
  if (lane == 0) {
    ctl->tile_start[p.num_groups] = tiles;
    ctl->total_tiles = tiles;
  }
  if (bad) atomicOr(p.status, kStBadOffsets);
}

struct I8Tile {
  int32_t g, tm, tn, row0, row_end;
};

// Tokens of a tile of a group with r rows, when tiles take any multiple of 32 tokens up to 256: its tiles are of one height.
__device__ __forceinline__ int32_t i8_height(int32_t r) {
  if (r <= 0) return 0;
  const int32_t m = (r + 255) / 256;
  return ((r + m - 1) / m + 31) & ~31;
}
// The group table of a walk over the groups by falling height of their tiles: a walk in steps of the number of CTA pairs then
// gives every pair the same sum of heights, but for one tile.  i8_build_groups has left the end rows.  One whole warp.
__device__ __forceinline__ void i8_sort_groups(I8Ctl* ctl, const I8GemmParams& p) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  int32_t place = 0, tiles = 0;
  for (int32_t height = 256; height >= 0; height -= 32) {
    for (int base = 0; base < p.num_groups; base += 32) {
      const int g = base + lane;
      const int32_t r = g < p.num_groups ? ctl->end[g] - (g ? ctl->end[g - 1] : 0) : 0;
      const bool mine = g < p.num_groups && i8_height(r) == height;
      const uint32_t all = __ballot_sync(0xffffffffu, mine);
      if (all == 0) continue;
      const int32_t n = mine && height ? (r + height - 1) / height * p.tiles_n : 0;
      int32_t upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      if (mine) {
        const int32_t at = place + __popc(all & ((1u << lane) - 1u));
        ctl->order[at] = uint16_t(g);
        ctl->tile_start[at] = tiles + upto - n;
      }
      place += __popc(all);
      tiles += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  if (lane == 0) {
    ctl->tile_start[p.num_groups] = tiles;
    ctl->total_tiles = tiles;
  }
}
// Tile t of that walk; `height` is its number of MMA columns.
__device__ __forceinline__ I8Tile i8_decode_sorted(const I8Ctl* ctl, const I8GemmParams& p, const WorkItem& wi, int32_t* height) {
  int lo = 0, hi = p.num_groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (ctl->tile_start[mid] <= wi.t) lo = mid; else hi = mid;
  }
  I8Tile ti;
  ti.g = ctl->order[lo];
  const int32_t begin = ti.g ? ctl->end[ti.g - 1] : 0, end = ctl->end[ti.g];
  const int32_t h = i8_height(end - begin);
  const int32_t local = wi.t - ctl->tile_start[lo];
  const int32_t tiles_m = (end - begin + h - 1) / h;
  const int32_t per_band = p.band * p.tiles_n;
  const int32_t b = local / per_band, rem = local - b * per_band;
  const int32_t bh = min(p.band, tiles_m - b * p.band);
  ti.tm = b * p.band + rem % bh;
  ti.tn = rem / bh;
  ti.row0 = begin + ti.tm * h;
  ti.row_end = min(ti.row0 + h, end);
  *height = h;
  if (wi.split) {      // a half of the tokens; of 32 all are in the first half
    const int32_t first = ((h >> 1) + 31) & ~31;
    if (wi.half) ti.row0 += first; else ti.row_end = min(ti.row_end, ti.row0 + first);
    *height = wi.half ? max(h - first, 32) : first;
  }
  return ti;
}
// Tile t of the walk: groups in order; inside a group bands of `band` row tiles, rows fastest.
__device__ __forceinline__ I8Tile i8_decode(const I8Ctl* ctl, const I8GemmParams& p, int32_t t, int32_t tile_rows) {
  int lo = 0, hi = p.num_groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (ctl->tile_start[mid] <= t) lo = mid; else hi = mid;
  }
  I8Tile ti;
  ti.g = lo;
  const int32_t begin = lo ? ctl->end[lo - 1] : 0;
  ti.row_end = ctl->end[lo];
  const int32_t local = t - ctl->tile_start[lo];
  const int32_t tiles_m = (ti.row_end - begin + tile_rows - 1) / tile_rows;
  const int32_t per_band = p.band * p.tiles_n;
  const int32_t b = local / per_band, rem = local - b * per_band;
  const int32_t bh = min(p.band, tiles_m - b * p.band);
  ti.tm = b * p.band + rem % bh;
  ti.tn = rem / bh;
  ti.row0 = begin + ti.tm * tile_rows;
  return ti;
}

// The bias is 0 where there is none: adding it then changes nothing (a sum of -0 becomes +0).
__device__ __forceinline__ float i8_finish(uint32_t acc, float sa, float sb, float bias) {
  return __fmaf_rn(__fmul_rn(__int2float_rn(int32_t(acc)), sa), sb, bias);
}
// Activation of a register tile, behind one branch and in a loop that is not unrolled: inlined at every value, its code was
// larger than the instruction caches and a 256-column epilogue took 28 us instead of 2.
template <int N>
__device__ __forceinline__ void i8_activate(float (&x)[N], int act) {
  if (act == kActIdentity) return;
  if (act == kActRelu) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = apply_activation(x[j], kActRelu);
  } else if (act == kActGelu) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = apply_activation(x[j], kActGelu);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = apply_activation(x[j], kActSilu);
  }
}

// Columns (tokens) of one channel, finished and stored; consecutive lanes hold consecutive channels.
template <int N>
__device__ __forceinline__ void i8_put(const I8GemmParams& p, const uint32_t (&v)[N], const float* sa, int n_here, float sb, float bias, int64_t at) {
  float x[N];
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = i8_finish(v[j], sa[j], sb, bias);
  i8_activate(x, p.activation);
  if (p.out_kind == kOutBf16) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j < n_here) reinterpret_cast<__nv_bfloat16*>(p.D)[at + j * p.ldd] = __float2bfloat16_rn(x[j]);
    }
  } else if (p.out_kind == kOutF16) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j < n_here) reinterpret_cast<__half*>(p.D)[at + j * p.ldd] = __float2half_rn(x[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j < n_here) reinterpret_cast<float*>(p.D)[at + j * p.ldd] = x[j];
    }
  }
}

// ---- many rows: D tile = (128 * CG rows) x BN columns, persistent, two accumulators of BN columns in tensor memory.
// Bound by the tensor cores (8192^3: 316 us, 3.5 P op/s, the pipe 92 % active) and, in a long run, by the power that they take.
// Eight epilogue warps, two for every quarter of the rows with half of the columns each: with four, a tile took 6 us to finish
// (latencies of tensor-memory loads, conversions and staged stores, one after the other), more than its products up to K = 2500.
// The staging of eight warps leaves room for five stages of 256 columns: 2 % slower than six at K = 4096, 8 % faster at K = 512
// than six with half of the staging.
// TURN, for groups: the weights are the MMA's rows and the tokens its columns, of which there may be any multiple of 32; the
// tiles of a group then carry at most 31 tokens too many each, where tiles of 256 rows are on average half empty at a group's
// end.  A lane of the epilogue holds a channel, and 32 of them a 64-byte piece of a result row, which goes to memory as it is: no
// staging, and a stage more.  32768 rows in 64 groups of uneven size, 2048 x 7168: 380 us, 397 with five stages, 406 with tiles of
// 256 rows (what is left to bound it is power: 327 us on weights and tokens of zeros, 390 in tiles of 256 rows).  Asking L2 for weights ahead of their copies made it
// slower (16 k-tiles ahead 402, 32 ahead 440).
constexpr int kI8EpiWarps = 8;
constexpr int kI8RowsThreads = 32 * (2 + kI8EpiWarps);      // warps 0-3 and 6-9 epilogue, 4 MMA, 5 TMA
template <int CG, int BN, bool TURN>
struct I8RowsCfg {
  static constexpr int kTileM = 128 * CG;
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBRows = BN / CG;
  static constexpr int kBBytes = kBRows * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kEpiBytes = TURN ? 0 : kI8EpiWarps * 4096;    // per warp 32 rows of 128 bytes
  static constexpr int kColBytes = 2 * 2 * BN * 4;        // scale and bias of the tile's columns, two tiles
  static constexpr int kStagesRaw = (232448 - 1024 - kI8CtlBytes - kEpiBytes - kColBytes) / kStageBytes;
  static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;
  static constexpr int kSmemBytes = kStages * kStageBytes + kEpiBytes + kColBytes + kI8CtlBytes + 1024;
  static constexpr int kTmemCols = 2 * BN;
  static_assert(kTmemCols == 64 || kTmemCols == 128 || kTmemCols == 256 || kTmemCols == 512, "tensor-memory columns");
};

template <int CG, int BN, bool TURN>
__global__ void __launch_bounds__(kI8RowsThreads, 1)
bsg_i8_rows_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmD, const I8GemmParams p) {
  using C = I8RowsCfg<CG, BN, TURN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + C::kStages * C::kABytes;
  uint8_t* sEpi = sB + C::kStages * C::kBBytes;
  float* sCol = reinterpret_cast<float*>(sEpi + C::kEpiBytes);
  I8Ctl* ctl = reinterpret_cast<I8Ctl*>(sEpi + C::kEpiBytes + C::kColBytes);

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t cta_rank = CG == 2 ? ptx::cluster_ctarank() : 0u;
  const bool is_leader = cta_rank == 0;
  const int32_t cluster_idx = CG == 2 ? int32_t(ptx::cluster_id_x()) : int32_t(blockIdx.x);
  const int32_t num_clusters = CG == 2 ? int32_t(ptx::num_clusters_x()) : int32_t(gridDim.x);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&ctl->full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctl->empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(ptx::smem_u32(&ctl->tmem_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctl->tmem_empty[s]), kI8EpiWarps * CG);
    }
    ctl->abort = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async();
  }
  if (warp == 5 && lane == 0) {
    ptx::prefetch_tmap(&tmA);
    ptx::prefetch_tmap(&tmB);
    ptx::prefetch_tmap(&tmD);
  }
  if (warp == 4) {
    ptx::tmem_alloc<CG>(ptx::smem_u32(&ctl->tmem_base), C::kTmemCols);
    ptx::tmem_relinquish<CG>();
  }
  // Launched behind the quantiser with programmatic stream serialisation: from here on its results are read.
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (warp == 0) {
    i8_build_groups(ctl, p, C::kTileM);
    if constexpr (TURN) i8_sort_groups(ctl, p);
  }
  __syncwarp();
  ptx::tc_fence_before();
  if constexpr (CG == 2) { ptx::cluster_arrive(); ptx::cluster_wait(); } else { __syncthreads(); }
  ptx::tc_fence_after();

  const uint32_t tmem_base = bcast(ctl->tmem_base);
  const int32_t total_tiles = bcast(ctl->total_tiles);
  const int32_t k_tiles = (p.K + 127) / 128;
  uint32_t dead = 0;
  // The tiles of a last wave that is at most half full are computed as two halves of their columns each, by twice as many pairs.
  int32_t split_from = total_tiles;
  if (BN == 256 && total_tiles > num_clusters) {
    const int32_t tail = total_tiles % num_clusters;
    if (2 * tail <= num_clusters) split_from = total_tiles - tail;
  }
  const int32_t total_work = split_from + 2 * (total_tiles - split_from);

  if (warp == 5) {
    // ---------------------------------------------------------------- TMA producer
    const uint32_t elected = ptx::elect_one_sync();
    const uint32_t sA0 = ptx::smem_u32(sA), sB0 = ptx::smem_u32(sB);
    const uint32_t full0 = ptx::smem_u32(&ctl->full[0]), empty0 = ptx::smem_u32(&ctl->empty[0]);
    const uint32_t full0_leader = CG == 2 ? ptx::mapa(full0, 0) : full0;
    int stage = 0;
    uint32_t phase = 0;
    for (int32_t t = cluster_idx; t < total_work; t += num_clusters) {
      const WorkItem wi = decode_work(t, split_from);
      int32_t a_row, b_row, g;
      // (boxes always bring kBRows rows of B, of which the MMA may read fewer)
      if constexpr (TURN) {
        int32_t height;
        const I8Tile ti = i8_decode_sorted(ctl, p, wi, &height);
        a_row = bcast(ti.tn * 256 + int32_t(cta_rank) * 128);
        b_row = bcast(ti.row0 + int32_t(cta_rank) * (height >> 1));
        g = bcast(ti.g);
      } else {
        const I8Tile ti = i8_decode(ctl, p, wi.t, C::kTileM);
        a_row = bcast(ti.row0 + int32_t(cta_rank) * 128);
        b_row = bcast(ti.tn * BN + (wi.split ? wi.half * (BN / 2) + int32_t(cta_rank) * (C::kBRows / 2) : int32_t(cta_rank) * C::kBRows));
        g = bcast(ti.g);
      }
      for (int32_t kt = 0; kt < k_tiles; ++kt) {
        i8_wait(empty0 + stage * 8, phase ^ 1u, ctl, dead);
        if (elected && !dead) {
          if (is_leader) ptx::mbar_arrive_expect_tx(full0 + stage * 8, uint32_t(C::kStageBytes) * CG);
          const uint32_t bar = full0_leader + stage * 8;
          ptx::tma_load_3d<CG>(sA0 + stage * C::kABytes, TURN ? &tmB : &tmA, bar, kt * 128, a_row, TURN ? g : 0);
          ptx::tma_load_3d<CG>(sB0 + stage * C::kBBytes, TURN ? &tmA : &tmB, bar, kt * 128, b_row, TURN ? 0 : g);
        }
        if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
      }
    }
    // Every stage must have been released before this CTA leaves: no commit is then in flight towards it.
    for (int s = 0; s < C::kStages; ++s) {
      i8_wait(empty0 + stage * 8, phase ^ 1u, ctl, dead);
      if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
    }
    if (dead) atomicOr(p.status, kStTimeoutEmpty);
  } else if (warp == 4) {
    // ---------------------------------------------------------------- MMA issue
    if (is_leader) {
      constexpr uint32_t idesc_full = i8_idesc(C::kTileM, BN), idesc_half = i8_idesc(C::kTileM, BN / 2);
      const uint32_t elected = ptx::elect_one_sync();
      const uint32_t sA0 = ptx::smem_u32(sA), sB0 = ptx::smem_u32(sB);
      const uint32_t full0 = ptx::smem_u32(&ctl->full[0]), empty0 = ptx::smem_u32(&ctl->empty[0]);
      const uint32_t tfull0 = ptx::smem_u32(&ctl->tmem_full[0]), tempty0 = ptx::smem_u32(&ctl->tmem_empty[0]);
      int stage = 0;
      uint32_t phase = 0, ready = 0;
      int32_t it = 0;
      for (int32_t t = cluster_idx; t < total_work; t += num_clusters, ++it) {
        uint32_t idesc = t >= split_from ? idesc_half : idesc_full;
        if constexpr (TURN) {
          int32_t height;
          i8_decode_sorted(ctl, p, decode_work(t, split_from), &height);
          idesc = i8_idesc(256, uint32_t(bcast(height)));
        }
        const int acc = it & 1;
        const uint32_t d_tmem = tmem_base + uint32_t(acc) * BN;
        i8_wait(tempty0 + acc * 8, (uint32_t(it >> 1) & 1u) ^ 1u, ctl, dead);
        ptx::tc_fence_after();
        for (int32_t kt = 0; kt < k_tiles; ++kt) {
          if (!ready) i8_wait(full0 + stage * 8, phase, ctl, dead);
          int next_stage = stage + 1;
          uint32_t next_phase = phase;
          if (next_stage == C::kStages) { next_stage = 0; next_phase ^= 1u; }
          ready = ptx::mbar_spin_test(full0 + next_stage * 8, next_phase, 1);
          ptx::tc_fence_after();
          const uint64_t a_desc = make_desc_sw128(sA0 + stage * C::kABytes);
          const uint64_t b_desc = make_desc_sw128(sB0 + stage * C::kBBytes);
          if (elected && !dead) {
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) i8_mma<CG>(d_tmem, a_desc + 2 * kb, b_desc + 2 * kb, idesc, kb > 0 || kt > 0);
            ptx::umma_commit<CG>(empty0 + stage * 8);
          }
          stage = next_stage;
          phase = next_phase;
        }
        if (elected && !dead) ptx::umma_commit<CG>(tfull0 + acc * 8);
      }
      if (dead) atomicOr(p.status, kStTimeoutFull | kStTimeoutTmemEmpty);
    }
  } else if constexpr (TURN) {
    // ---------------------------------------------------------------- epilogue: a lane is an output channel
    const int quarter = warp & 3, half = warp >= 6 ? 1 : 0;      // every second step of 32 tokens
    const int epi = half * 4 + quarter;
    const uint32_t tfull0 = ptx::smem_u32(&ctl->tmem_full[0]), tempty0 = ptx::smem_u32(&ctl->tmem_empty[0]);
    const bool has_bias = p.bias != nullptr;
    struct Need { int32_t n, row0, rows, height; float sb, bias, sa; };
    auto need_of = [&](int32_t t) {
      Need d;
      const I8Tile ti = i8_decode_sorted(ctl, p, decode_work(t, split_from), &d.height);
      d.n = ti.tn * 256 + int32_t(cta_rank) * 128 + quarter * 32 + lane;
      d.row0 = ti.row0;
      d.rows = ti.row_end - ti.row0;
      const int64_t at = int64_t(ti.g) * p.N + d.n;
      d.sb = d.n < p.N ? __ldg(p.sb + at) : 0.0f;
      d.bias = d.n < p.N && has_bias ? __ldg(p.bias + at) : 0.0f;
      d.sa = epi * 32 + lane < d.rows ? __ldcg(p.sa + ti.row0 + epi * 32 + lane) : 0.0f;
      return d;
    };
    int32_t it = 0;
    Need need{};
    if (cluster_idx < total_work) need = need_of(cluster_idx);
    for (int32_t t = cluster_idx; t < total_work; t += num_clusters, ++it) {
      const int acc = it & 1;
      const Need d = need;
      float* sa = sCol + acc * 256;
      sa[epi * 32 + lane] = d.sa;
      if (t + num_clusters < total_work) need = need_of(t + num_clusters);
      __syncwarp();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      i8_wait(tfull0 + acc * 8, uint32_t(it >> 1) & 1u, ctl, dead);
      __syncwarp();
      ptx::tc_fence_after();
      const uint32_t lane_addr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(acc) * BN;
#pragma unroll 1
      for (int c0 = half * 32; c0 < d.height; c0 += 64) {
        uint32_t v[32];
        __syncwarp();
        ptx::tmem_ld_32x32b_x32(lane_addr + c0, v);
        ptx::tmem_ld_wait();
        if (d.n < p.N && c0 < d.rows) i8_put(p, v, sa + c0, min(32, d.rows - c0), d.sb, d.bias, int64_t(d.row0 + c0) * p.ldd + d.n);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_remote_relaxed(ptx::mapa(tempty0 + acc * 8, 0));
    }
    if (dead) atomicOr(p.status, kStTimeoutTmemFull);
  } else {
    // ---------------------------------------------------------------- epilogue
    const int quarter = warp & 3, half = warp >= 6 ? 1 : 0;      // (a warp reaches the tensor-memory lanes of its number mod 4)
    const int epi = half * 4 + quarter;
    const uint32_t tfull0 = ptx::smem_u32(&ctl->tmem_full[0]), tempty0 = ptx::smem_u32(&ctl->tmem_empty[0]);
    uint8_t* stage_buf = sEpi + epi * 4096;
    const int out_kind = p.out_kind, act = p.activation;
    const bool f32 = out_kind == kOutF32, has_bias = p.bias != nullptr;
    // What a tile needs besides its sums: its place, the scale and the bias of one of its columns per thread, the scale of this
    // lane's row.  Asked for one tile ahead.
    struct Need { int32_t g, col0, cols, row0, rows; float sb, bias, sa; };
    auto need_of = [&](int32_t t) {
      const WorkItem wi = decode_work(t, split_from);
      const I8Tile ti = i8_decode(ctl, p, wi.t, C::kTileM);
      Need n;
      n.g = ti.g;
      n.col0 = ti.tn * BN + wi.half * (BN / 2);
      n.cols = wi.split ? BN / 2 : BN;
      n.row0 = ti.row0 + int32_t(cta_rank) * 128 + quarter * 32;
      n.rows = min(32, ti.row_end - n.row0);
      const int32_t c = n.col0 + epi * 32 + lane;
      const bool in = epi * 32 + lane < n.cols && c < p.N;
      n.sb = in ? __ldg(p.sb + int64_t(n.g) * p.N + c) : 0.0f;
      n.bias = in && has_bias ? __ldg(p.bias + int64_t(n.g) * p.N + c) : 0.0f;
      n.sa = lane < n.rows ? __ldcg(p.sa + n.row0 + lane) : 0.0f;
      return n;
    };
    static_assert(BN <= 32 * kI8EpiWarps, "one column per thread");
    int32_t it = 0;
    Need need{};
    if (cluster_idx < total_work) need = need_of(cluster_idx);
    for (int32_t t = cluster_idx; t < total_work; t += num_clusters, ++it) {
      const int acc = it & 1;
      const int32_t col0 = need.col0, cols = need.cols, warp_row0 = need.row0, rows_here = need.rows;
      const float sa = need.sa;
      float* cs = sCol + acc * 2 * BN;
      if (epi * 32 + lane < cols) {
        cs[epi * 32 + lane] = need.sb;
        cs[BN + epi * 32 + lane] = need.bias;
      }
      if (t + num_clusters < total_work) need = need_of(t + num_clusters);
      __syncwarp();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      i8_wait(tfull0 + acc * 8, uint32_t(it >> 1) & 1u, ctl, dead);
      __syncwarp();
      ptx::tc_fence_after();
      const uint32_t lane_addr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(acc) * BN;
      // Whole warps of rows leave by TMA; the warp that holds a group's last rows, and outputs whose rows do not start
      // on 16 bytes, are copied row by row from the same staging tile.
      const bool tma = p.tma_out != 0 && rows_here == 32;
      const int32_t c_end = (half + 1) * (cols / 2);
#pragma unroll 1
      for (int c0 = half * (cols / 2); c0 < c_end; c0 += 32) {
        uint32_t v[32];
        __syncwarp();
        ptx::tmem_ld_32x32b_x32(lane_addr + c0, v);
        ptx::tmem_ld_wait();
        if (c0 + 32 == c_end) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) {       // relaxed: what is handed back is tensor memory, whose reads have completed
            if constexpr (CG == 2) ptx::mbar_arrive_remote_relaxed(ptx::mapa(tempty0 + acc * 8, 0));
            else ptx::mbar_arrive_relaxed(tempty0 + acc * 8);
          }
        }
        if (rows_here <= 0 || col0 + c0 >= p.N) continue;
        float x[32];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 s4 = *reinterpret_cast<const float4*>(cs + c0 + j);
          const float4 b4 = *reinterpret_cast<const float4*>(cs + BN + c0 + j);
          x[j + 0] = i8_finish(v[j + 0], sa, s4.x, b4.x);
          x[j + 1] = i8_finish(v[j + 1], sa, s4.y, b4.y);
          x[j + 2] = i8_finish(v[j + 2], sa, s4.z, b4.z);
          x[j + 3] = i8_finish(v[j + 3], sa, s4.w, b4.w);
        }
        i8_activate(x, act);
        // 128 bytes of a row at a time: 32 columns of 32 bits, or two steps of 32 columns of 16 bits (TMA moves a row of a box in
        // about seven cycles, whatever its length).  Staging: 16-byte piece c of row r at piece c ^ (r & 7).  Before it is written
        // again the last copy out of it has to have read it, whatever way this tile goes: the copy may be the tile before's.
        const int second = f32 ? 0 : (c0 >> 5) & 1;
        if (second == 0) {
          if (lane == 0) ptx::bulk_wait_group_read<0>();
          __syncwarp();
        }
        if (f32) {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(stage_buf + lane * 128 + ((q ^ (lane & 7)) * 16)) = make_float4(x[q * 4], x[q * 4 + 1], x[q * 4 + 2], x[q * 4 + 3]);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 o;
            if (out_kind == kOutBf16)
              o = make_uint4(pack_bf16x2(x[q * 8], x[q * 8 + 1]), pack_bf16x2(x[q * 8 + 2], x[q * 8 + 3]), pack_bf16x2(x[q * 8 + 4], x[q * 8 + 5]), pack_bf16x2(x[q * 8 + 6], x[q * 8 + 7]));
            else
              o = make_uint4(pack_f16x2(x[q * 8], x[q * 8 + 1]), pack_f16x2(x[q * 8 + 2], x[q * 8 + 3]), pack_f16x2(x[q * 8 + 4], x[q * 8 + 5]), pack_f16x2(x[q * 8 + 6], x[q * 8 + 7]));
            *reinterpret_cast<uint4*>(stage_buf + lane * 128 + (((second * 4 + q) ^ (lane & 7)) * 16)) = o;
          }
        }
        if (!f32 && second == 0 && col0 + c0 + 32 < p.N) continue;      // the tile fills up in the next step
        const int32_t out_col = col0 + c0 - 32 * second, width = f32 ? 32 : 64;
        if (tma && (p.tma_edge || out_col + width <= p.N)) {
          ptx::fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            ptx::tma_store_3d(&tmD, ptx::smem_u32(stage_buf), out_col, warp_row0, 0);
            ptx::bulk_commit_group();
          }
        } else {
          __syncwarp();
          const int32_t left = min(width, p.N - out_col);
          for (int c = lane; c < left; c += 32) {
            if (f32) {
#pragma unroll 4
              for (int r = 0; r < rows_here; ++r)
                reinterpret_cast<float*>(p.D)[int64_t(warp_row0 + r) * p.ldd + out_col + c] =
                    *reinterpret_cast<const float*>(stage_buf + r * 128 + (((c >> 2) ^ (r & 7)) * 16) + (c & 3) * 4);
            } else {      // (32-bit words, shifted for rows that start on an odd column, took 1.7 times as long)
#pragma unroll 4
              for (int r = 0; r < rows_here; ++r)
                reinterpret_cast<uint16_t*>(p.D)[int64_t(warp_row0 + r) * p.ldd + out_col + c] =
                    *reinterpret_cast<const uint16_t*>(stage_buf + r * 128 + (((c >> 3) ^ (r & 7)) * 16) + (c & 7) * 2);
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) ptx::bulk_wait_group<0>();
    if (dead) atomicOr(p.status, kStTimeoutTmemFull);
  }

  if (ctl->abort) {      // copies and MMAs that may still be in flight land before the memory is handed back
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000ll) __nanosleep(1000);
  }
  __syncwarp();
  ptx::tc_fence_before();
  if constexpr (CG == 2) { ptx::cluster_arrive(); ptx::cluster_wait(); } else { __syncthreads(); }
  if (warp == 4) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<CG>(tmem_base, C::kTmemCols);
  }
}

// ---- few rows: D^T tile = 128 channels x BT tokens.  The CTAs of a cluster (SPLIT of them) take consecutive parts of K of
// one tile; each sends the columns that another one finishes into that CTA's shared memory, and each finishes BT / SPLIT.
template <int BT, int SPLIT>
struct I8FewCfg {
  static_assert(SPLIT == 1 || BT <= 64, "wide tiles do not split");
  static constexpr int kWBytes = 128 * 128;
  static constexpr int kTBytes = BT * 128;
  static constexpr int kStageBytes = kWBytes + kTBytes;
  static constexpr int kRedBytes = SPLIT > 1 ? BT * 512 : 0;          // [SPLIT][BT / SPLIT][128] int32
  static constexpr int kSaBytes = 2 * BT * 4;                         // token scales of two tiles
  static constexpr int kStagesRaw = (115712 - 1024 - kI8CtlBytes - kRedBytes - kSaBytes) / kStageBytes;     // two CTAs per SM
  static constexpr int kStages = kStagesRaw > 6 ? 6 : kStagesRaw;
  static constexpr int kSmemBytes = kStages * kStageBytes + kRedBytes + kSaBytes + kI8CtlBytes + 1024;
  static constexpr int kTmemCols = 2 * BT;
  static_assert(kStages >= 3, "stages");
};

template <int BT, int SPLIT>
__global__ void __launch_bounds__(192, 2)
bsg_i8_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const I8GemmParams p) {
  using C = I8FewCfg<BT, SPLIT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sT = sW + C::kStages * C::kWBytes;
  uint8_t* sRed = sT + C::kStages * C::kTBytes;
  float* sSa = reinterpret_cast<float*>(sRed + C::kRedBytes);
  I8Ctl* ctl = reinterpret_cast<I8Ctl*>(sRed + C::kRedBytes + C::kSaBytes);

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int32_t rank = SPLIT > 1 ? int32_t(ptx::cluster_ctarank()) : 0;
  const int32_t worker = int32_t(blockIdx.x) / SPLIT, workers = int32_t(gridDim.x) / SPLIT;
  const int32_t k_all = (p.K + 127) / 128;
  const int32_t kt0 = k_all * rank / SPLIT, kt1 = k_all * (rank + 1) / SPLIT;
  const int32_t early_tiles = min(kt1 - kt0, C::kStages);
  const bool dense = p.offsets == nullptr;

  // The weights do not depend on the quantiser in front of this kernel: those of the first stages are asked for before
  // anything else (dense: the first tile is known without the group table), and before its results are waited for.
  auto fetch_early = [&](int32_t tn, int32_t g) {
    const uint32_t full0 = ptx::smem_u32(&ctl->full[0]), sW0 = ptx::smem_u32(sW);
    for (int32_t i = 0; i < early_tiles; ++i) {
      ptx::mbar_arrive_expect_tx(full0 + i * 8, C::kStageBytes);
      ptx::tma_load_3d<1>(sW0 + i * C::kWBytes, &tmW, full0 + i * 8, (kt0 + i) * 128, tn * 128, g);
    }
  };
  const int32_t dense_tiles_m = (p.total_rows + BT - 1) / BT;
  if (warp == 5) {
    if (ptx::elect_one_sync()) {
      for (int s = 0; s < C::kStages; ++s) {
        ptx::mbar_init(ptx::smem_u32(&ctl->full[s]), 1);
        ptx::mbar_init(ptx::smem_u32(&ctl->empty[s]), 1);
      }
      for (int s = 0; s < 2; ++s) {
        ptx::mbar_init(ptx::smem_u32(&ctl->tmem_full[s]), 1);
        ptx::mbar_init(ptx::smem_u32(&ctl->tmem_empty[s]), 4);
      }
      ctl->abort = 0;
      ptx::fence_mbar_init();
      ptx::fence_proxy_async();
      if (dense) fetch_early(worker / dense_tiles_m, 0);       // one band: the token tiles of a channel tile follow one another
      ptx::prefetch_tmap(&tmX);
    }
    __syncwarp();
  } else if (warp == 4) {
    ptx::tmem_alloc<1>(ptx::smem_u32(&ctl->tmem_base), C::kTmemCols);
    ptx::tmem_relinquish<1>();
  } else if (warp == 0) {
    // needs the end rows only, which are older than the quantiser this kernel may overlap with
    i8_build_groups(ctl, p, BT);
  }
  __syncwarp();
  ptx::tc_fence_before();
  if constexpr (SPLIT > 1) { ptx::cluster_arrive(); ptx::cluster_wait(); } else { __syncthreads(); }
  ptx::tc_fence_after();

  const uint32_t tmem_base = bcast(ctl->tmem_base);
  const int32_t total_tiles = bcast(ctl->total_tiles);
  uint32_t dead = 0;

  if (warp == 5) {
    // ---------------------------------------------------------------- TMA producer
    const uint32_t elected = ptx::elect_one_sync();
    const uint32_t sW0 = ptx::smem_u32(sW), sT0 = ptx::smem_u32(sT);
    const uint32_t full0 = ptx::smem_u32(&ctl->full[0]), empty0 = ptx::smem_u32(&ctl->empty[0]);
    int stage = 0;
    uint32_t phase = 0;
    int32_t early = 0;
    if (worker < total_tiles) {
      early = early_tiles;
      if (!dense) {
        const I8Tile ti = i8_decode(ctl, p, worker, BT);
        if (elected) fetch_early(ti.tn, ti.g);
      }
    }
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    for (int32_t t = worker; t < total_tiles; t += workers) {
      const I8Tile ti = i8_decode(ctl, p, t, BT);
      const int32_t w_row = bcast(ti.tn * 128), t_row = bcast(ti.row0), g = bcast(ti.g);
      for (int32_t kt = kt0; kt < kt1; ++kt) {
        const bool first = early > 0;
        if (first) --early;
        else i8_wait(empty0 + stage * 8, phase ^ 1u, ctl, dead);
        if (elected && !dead) {
          const uint32_t bar = full0 + stage * 8;
          if (!first) {
            ptx::mbar_arrive_expect_tx(bar, C::kStageBytes);
            ptx::tma_load_3d<1>(sW0 + stage * C::kWBytes, &tmW, bar, kt * 128, w_row, g);
          }
          ptx::tma_load_3d<1>(sT0 + stage * C::kTBytes, &tmX, bar, kt * 128, t_row, 0);
        }
        if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
      }
    }
    for (int s = 0; s < C::kStages; ++s) {
      i8_wait(empty0 + stage * 8, phase ^ 1u, ctl, dead);
      if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
    }
    if (dead) atomicOr(p.status, kStTimeoutEmpty);
  } else if (warp == 4) {
    // ---------------------------------------------------------------- MMA issue
    constexpr uint32_t idesc = i8_idesc(128, BT);
    const uint32_t elected = ptx::elect_one_sync();
    const uint32_t sW0 = ptx::smem_u32(sW), sT0 = ptx::smem_u32(sT);
    const uint32_t full0 = ptx::smem_u32(&ctl->full[0]), empty0 = ptx::smem_u32(&ctl->empty[0]);
    const uint32_t tfull0 = ptx::smem_u32(&ctl->tmem_full[0]), tempty0 = ptx::smem_u32(&ctl->tmem_empty[0]);
    int stage = 0;
    uint32_t phase = 0;
    int32_t it = 0;
    for (int32_t t = worker; t < total_tiles; t += workers, ++it) {
      const int acc = it & 1;
      const uint32_t d_tmem = tmem_base + uint32_t(acc) * BT;
      i8_wait(tempty0 + acc * 8, (uint32_t(it >> 1) & 1u) ^ 1u, ctl, dead);
      ptx::tc_fence_after();
      for (int32_t kt = kt0; kt < kt1; ++kt) {
        i8_wait(full0 + stage * 8, phase, ctl, dead);
        ptx::tc_fence_after();
        const uint64_t a_desc = make_desc_sw128(sW0 + stage * C::kWBytes);
        const uint64_t b_desc = make_desc_sw128(sT0 + stage * C::kTBytes);
        if (elected && !dead) {
#pragma unroll
          for (int kb = 0; kb < 4; ++kb) i8_mma<1>(d_tmem, a_desc + 2 * kb, b_desc + 2 * kb, idesc, kb > 0 || kt > kt0);
          ptx::umma_commit<1>(empty0 + stage * 8);
        }
        if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
      }
      if (elected && !dead) ptx::umma_commit<1>(tfull0 + acc * 8);
    }
    if (dead) atomicOr(p.status, kStTimeoutFull | kStTimeoutTmemEmpty);
  } else {
    // ---------------------------------------------------------------- epilogue: a lane is an output channel
    constexpr int kPer = BT / SPLIT;             // columns that this CTA finishes
    constexpr int kChunk = BT < 32 ? BT : 32;
    const uint32_t tfull0 = ptx::smem_u32(&ctl->tmem_full[0]), tempty0 = ptx::smem_u32(&ctl->tmem_empty[0]);
    const bool has_bias = p.bias != nullptr;
    ptx::grid_dependency_wait();          // the token scales come from the quantiser, and D may still be read by what ran before
    int32_t it = 0;
    for (int32_t t = worker; t < total_tiles; t += workers, ++it) {
      const I8Tile ti = i8_decode(ctl, p, t, BT);
      const int acc = it & 1;
      const int32_t n = ti.tn * 128 + warp * 32 + lane;
      const bool n_ok = n < p.N;
      const int64_t at = int64_t(ti.g) * p.N + n;
      const float sb = n_ok ? __ldg(p.sb + at) : 0.0f;
      const float bias = n_ok && has_bias ? __ldg(p.bias + at) : 0.0f;
      const int32_t cols = min(BT, ti.row_end - ti.row0);
      float* sa = sSa + acc * BT;
      if (threadIdx.x < BT) sa[threadIdx.x] = int32_t(threadIdx.x) < cols ? __ldcg(p.sa + ti.row0 + threadIdx.x) : 0.0f;
      __syncwarp();
      asm volatile("bar.sync 1, 128;" ::: "memory");
      i8_wait(tfull0 + acc * 8, uint32_t(it >> 1) & 1u, ctl, dead);
      __syncwarp();
      ptx::tc_fence_after();
      const uint32_t lane_addr = tmem_base + (uint32_t(warp * 32) << 16) + uint32_t(acc) * BT;
#pragma unroll 1
      for (int c0 = 0; c0 < BT; c0 += kChunk) {
        uint32_t v[kChunk];
        __syncwarp();
        if constexpr (kChunk == 32) ptx::tmem_ld_32x32b_x32(lane_addr + c0, v);
        else i8_tmem_ld_x16(lane_addr + c0, v);
        ptx::tmem_ld_wait();
        if (c0 + kChunk == BT) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_relaxed(tempty0 + acc * 8);
        }
        if constexpr (SPLIT == 1) {
          if (n_ok && c0 < cols) i8_put(p, v, sa + c0, min(kChunk, cols - c0), sb, bias, int64_t(ti.row0 + c0) * p.ldd + n);
        } else {
          const uint32_t mine = ptx::smem_u32(sRed) + uint32_t((rank * kPer * 128 + warp * 32 + lane) * 4);
#pragma unroll
          for (int j = 0; j < kChunk; ++j) {
            const int c = c0 + j;
            if (c < cols) ptx::st_shared_cluster_u32(ptx::mapa(mine + uint32_t((c % kPer) * 512), uint32_t(c / kPer)), v[j]);
          }
        }
      }
    }
    if (dead) atomicOr(p.status, kStTimeoutTmemFull);
  }

  if constexpr (SPLIT > 1) {
    // One tile per cluster: every part of it has been sent once all CTAs are here.
    __syncwarp();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (warp < 4) {
      constexpr int kPer = BT / SPLIT, kStep = kPer < 8 ? kPer : 8;
      const I8Tile ti = i8_decode(ctl, p, worker, BT);
      const int32_t n = ti.tn * 128 + warp * 32 + lane;
      const int32_t left = ti.row_end - (ti.row0 + rank * kPer);
      if (n < p.N) {
        const float sb = __ldg(p.sb + n), bias = p.bias ? __ldg(p.bias + n) : 0.0f;
        const int32_t* red = reinterpret_cast<const int32_t*>(sRed) + warp * 32 + lane;
#pragma unroll 1
        for (int c0 = 0; c0 < kPer && c0 < left; c0 += kStep) {
          uint32_t v[kStep];
#pragma unroll
          for (int j = 0; j < kStep; ++j) {      // columns behind the last token hold nothing and are not stored
            int32_t sum = 0;
#pragma unroll
            for (int s = 0; s < SPLIT; ++s) sum += red[(s * kPer + c0 + j) * 128];
            v[j] = uint32_t(sum);
          }
          i8_put(p, v, sSa + rank * kPer + c0, min(kStep, left - c0), sb, bias, int64_t(ti.row0 + rank * kPer + c0) * p.ldd + n);
        }
      }
    }
  }
  if (ctl->abort) {
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000ll) __nanosleep(1000);
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem_base, C::kTmemCols);
  }
}

// ---- up to four tokens, quantised in the kernel itself: one launch, no tensor memory, no tensor maps.
// Every CTA quantises the tokens into its shared memory (they are few and come from L2) while its first weights are already on
// their way.  A warp owns two channels, or, where there are few channels, `parts` warps share two and take every parts-th
// piece of K; lanes stride over K with 16-byte loads and __dp4a, and one integer warp reduction per sum ends it.
constexpr int kI8TokenThreads = 256;
constexpr int kI8TokenMost = 4;
constexpr int kI8TokenShared = 65536;         // bytes of tokens in shared memory, at most
struct I8TokenParams {
  const uint16_t* X;
  const int8_t* W;
  const float* sb;
  const float* bias;
  void* D;
  int64_t ldx, ldw, ldd;
  int32_t M, N, K;
  int32_t out_kind, activation;
  int32_t parts;            // 1, 2, 4 or 8
};

// Sixteen weights of a row, zeros past its end (nothing past K is read).
__device__ __forceinline__ uint4 i8_weights16(const int8_t* row, int32_t k, int32_t K) {
  if (k + 16 <= K) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + k));
    return v;
  }
  uint32_t w[4] = {0, 0, 0, 0};
  for (int j = 0; j < 16 && k + j < K; ++j) w[j >> 2] |= uint32_t(uint8_t(row[k + j])) << (8 * (j & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int MT, bool FP16, bool WIDE>
__global__ void __launch_bounds__(kI8TokenThreads, 2) bsg_i8_token_kernel(const I8TokenParams p) {
  constexpr int kWarps = kI8TokenThreads / 32, kChan = 2, kUnroll = 4;
  constexpr int kPerToken = kI8TokenThreads / MT;            // threads that quantise one token: whole warps
  extern __shared__ __align__(16) uint8_t s_tok[];           // [MT][K rounded up to 16]
  __shared__ float s_max[kWarps], s_scale[MT];
  __shared__ int32_t s_part[2][kWarps][kChan * MT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t pitch = (p.K + 15) & ~15;
  const int32_t k_first = (warp % p.parts) * 512 + lane * 16, k_step = p.parts * 512;
  const int32_t batches = (pitch + kUnroll * k_step - 1) / (kUnroll * k_step);       // per group, the same for every warp
  const int32_t per_group = kChan * (kWarps / p.parts);                               // channels of a CTA's group
  const int32_t groups = (p.N + per_group - 1) / per_group;
  const int32_t n_warp = (warp / p.parts) * kChan;

  uint4 w[kUnroll][kChan], ahead[kUnroll][kChan];
  auto fetch = [&](uint4 (&to)[kUnroll][kChan], int32_t grp, int32_t batch) {
    const int32_t n0 = grp * per_group + n_warp, k0 = k_first + batch * kUnroll * k_step;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int c = 0; c < kChan; ++c) {
        const int32_t k = k0 + u * k_step;
        to[u][c] = n0 + c < p.N && k < p.K ? i8_weights16(p.W + int64_t(n0 + c) * p.ldw, k, p.K) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  fetch(w, blockIdx.x, 0);

  {
    const int m = threadIdx.x / kPerToken, t = threadIdx.x % kPerToken;
    const uint16_t* row = p.X + int64_t(m < p.M ? m : 0) * p.ldx;
    uint32_t mx = 0;
    for (int32_t k = t * 8; k < p.K; k += kPerToken * 8) {
      const uint4 u = i8_load8<WIDE>(row, k, p.K);
      mx = i8_maxabs2<FP16>(mx, i8_maxabs2<FP16>(i8_maxabs2<FP16>(u.x, u.y), i8_maxabs2<FP16>(u.z, u.w)));
    }
    mx &= 0x7FFF7FFFu;
    float amax = ptx::fmax_nan(i8_unpack(mx & 0xFFFFu, FP16), i8_unpack(mx >> 16, FP16));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) amax = ptx::fmax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) s_max[warp] = amax;
    __syncthreads();
    const int w0 = m * (kPerToken / 32);
    amax = s_max[w0];
#pragma unroll
    for (int i = 1; i < kPerToken / 32; ++i) amax = ptx::fmax_nan(amax, s_max[w0 + i]);
    const I8Scale s = i8_scale(amax);
    if (t == 0) s_scale[m] = i8_step(amax);
    for (int32_t k = t * 8; k < pitch; k += kPerToken * 8)
      *reinterpret_cast<uint2*>(s_tok + m * pitch + k) = i8_levels8<FP16>(i8_load8<WIDE>(row, k, p.K), s);
    __syncthreads();
  }

  int32_t acc[kChan][MT];
#pragma unroll
  for (int c = 0; c < kChan; ++c) {
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[c][m] = 0;
  }
  int32_t grp = blockIdx.x, batch = 0, turn = 0;
  while (grp < groups) {
    // the next batch, of this group or the CTA's next one, is fetched while this one is multiplied
    const bool last = batch + 1 == batches;
    const int32_t next_grp = last ? grp + int32_t(gridDim.x) : grp, next_batch = last ? 0 : batch + 1;
    if (next_grp < groups) fetch(ahead, next_grp, next_batch);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int32_t k = k_first + (batch * kUnroll + u) * k_step;
      if (k < pitch) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int4 x = *reinterpret_cast<const int4*>(s_tok + m * pitch + k);
#pragma unroll
          for (int c = 0; c < kChan; ++c) {
            acc[c][m] = __dp4a(x.x, int(w[u][c].x), acc[c][m]);
            acc[c][m] = __dp4a(x.y, int(w[u][c].y), acc[c][m]);
            acc[c][m] = __dp4a(x.z, int(w[u][c].z), acc[c][m]);
            acc[c][m] = __dp4a(x.w, int(w[u][c].w), acc[c][m]);
          }
        }
      }
    }
    if (last) {
      // lane m of the warp holds token m of the first channel, lane MT + m that of the second
      int32_t mine = 0;
#pragma unroll
      for (int c = 0; c < kChan; ++c) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int32_t sum = __reduce_add_sync(0xffffffffu, acc[c][m]);
          if (lane == c * MT + m) mine = sum;
          acc[c][m] = 0;
        }
      }
      bool finish = lane < kChan * MT;
      if (p.parts > 1) {
        if (finish) s_part[turn][warp][lane] = mine;
        __syncthreads();      // two turns of s_part: a warp is at most one group ahead of another
        finish = finish && warp % p.parts == 0;
        if (finish) {
          for (int i = 1; i < p.parts; ++i) mine += s_part[turn][warp + i][lane];
        }
        turn ^= 1;
      }
      const int32_t n = grp * per_group + n_warp + lane / MT, m = lane % MT;
      if (finish && n < p.N && m < p.M) {
        float x[1] = {i8_finish(uint32_t(mine), s_scale[m], p.sb[n], p.bias ? p.bias[n] : 0.0f)};
        i8_activate(x, p.activation);
        const int64_t at = int64_t(m) * p.ldd + n;
        if (p.out_kind == kOutBf16) reinterpret_cast<__nv_bfloat16*>(p.D)[at] = __float2bfloat16_rn(x[0]);
        else if (p.out_kind == kOutF16) reinterpret_cast<__half*>(p.D)[at] = __float2half_rn(x[0]);
        else reinterpret_cast<float*>(p.D)[at] = x[0];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int c = 0; c < kChan; ++c) w[u][c] = ahead[u][c];
    }
    grp = next_grp;
    batch = next_batch;
  }
}

}  // namespace bsg
