// Host side of the 8-bit integer product (bsg_int8_*): argument checks, choice of kernel and tile, launch.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>
#include <mutex>

#include "../../include/bsgemm.h"
#include "host.h"
#include "int8_kernel.cuh"

namespace {

using bsg::host_aligned;
using bsg::host_fail;

// `own_q`: Q and q_scale are the caller's (false for the kernel that quantises on the way and has none).
int32_t check_quantise(const bsg_int8_args& a, bool own_q) {
  if (a.in_kind != BSG_OUT_BF16 && a.in_kind != BSG_OUT_F16) return host_fail(BSG_ERR_NOT_SUPPORTED, "X must be bf16 or fp16 (kind %d)", a.in_kind);
  if (a.rows < 0 || a.tokens < 0 || a.K < 1) return host_fail(BSG_ERR_INVALID_PROBLEM, "extents must be positive (rows=%lld tokens=%lld K=%lld)", (long long)a.rows, (long long)a.tokens, (long long)a.K);
  if (a.rows > 0x3FFFFFFF || a.tokens > 0x3FFFFFFF || a.K > 0x3FFFFFFF) return host_fail(BSG_ERR_INVALID_PROBLEM, "extent exceeds 2^30");
  if (!a.index && a.rows != a.tokens) return host_fail(BSG_ERR_INVALID_PROBLEM, "without an index the %lld rows must be the %lld tokens", (long long)a.rows, (long long)a.tokens);
  if (a.rows == 0) return BSG_OK;
  if ((own_q && (!a.Q || !a.q_scale)) || (!a.X && a.tokens > 0)) return host_fail(BSG_ERR_INVALID_PROBLEM, "X, Q and q_scale must not be null");
  if (!host_aligned(a.X, 2) || !host_aligned(a.q_scale, 4)) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "X and q_scale must be aligned to their elements");
  if (a.ldx < a.K && a.tokens > 1) return host_fail(BSG_ERR_INVALID_PROBLEM, "ldx=%lld is smaller than K", (long long)a.ldx);
  if (own_q && (a.ldq < a.K || a.ldq % 16 != 0 || !host_aligned(a.Q, 16))) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "rows of Q must start on 16-byte boundaries (ldq=%lld, at least K)", (long long)a.ldq);
  return BSG_OK;
}

struct I8Plan {
  bool few;        // bsg_i8_few_kernel
  int32_t tile;    // few: tokens per tile; rows: columns per tile
  int32_t split;   // few: CTAs of a cluster that share one tile's K
};

// Kernel, tile and split, by a model of the time.  A CTA (or pair) streams its part of K through a pipeline that is bound by the
// latency of a TMA round trip, so a k-tile of 128 values takes a time that depends on the tile alone, and a tile takes at least
// as long as its epilogue; two CTAs of the kernel for few rows are resident on an SM, one pair of the other kernel on two SMs; a
// grid runs in whole waves.  The constants were fitted to 80 problems from 16 x 512 x 512 to 5000 x 14336 x 8192 (rows x N x K).
// Both sides of some choices: 777 x 5000 x 8192: 128-token tiles 34.3 us, 256 x 256 40.4, 64-token tiles 43.9; 2000 x 5000 x
// 8192: 256 x 256 60.3, 256 x 128 68.8, 128-token tiles 78.8; 777 x 512 x 512: 32-token tiles 4.6, 16 4.9, 64 6.2, 128 8.1.  Over
// 85 other problems, drawn at random, the choice took 1.04 times the time of the best variant in the geometric mean, 1.21 at most.
// Grouped, reading the weights and the rest are added as squares: small tiles read them several times (900 rows in 30 groups,
// 3001 x 1000: 32-token tiles 17.1 us, 16-token tiles 20.5), which over 36 problems brings the choice from 1.057 to 1.018 times the
// best.  Results whose rows are no whole 16-byte pieces leave row by row and take the kernel of many rows twice as long (9000 rows
// in 5 groups, 1500 x 700: 256 x 128 33.4 us, 128-token tiles 22.7).
struct Variant {
  bool few;
  int32_t tile;
  double per_k_tile, least, fixed;      // microseconds: of a k-tile, of a tile's epilogue, of the launch
};
constexpr Variant kVariants[] = {{true, 16, 0.20, 1.3, 3.6}, {true, 32, 0.24, 1.6, 3.8}, {true, 64, 0.31, 2.8, 4.6}, {true, 128, 0.45, 5.0, 6.0},
                                 {false, 128, 0.225, 2.2, 5.5}, {false, 256, 0.33, 3.3, 6.8}};
// Grouped, 256 channels: tiles of 256 channels by up to 256 tokens, whose results leave by plain stores.  13818 rows in 16 groups,
// 7168 x 512: 147 us, in tiles of 256 rows x 128 columns 110; 7971 rows in 16 groups, 7168 x 4096: 198 and 250.
constexpr Variant kTurned = {false, 256, 0.40, 6.0, 6.8};
constexpr double kHbmBytesPerUs = 6.5e6;

int32_t choose(const bsg_int8_args& a, I8Plan* plan) {
  const int64_t k_tiles = (a.K + 127) / 128;
  const int64_t active = a.rows < a.num_groups ? a.rows : a.num_groups;      // groups that can have rows
  const double weights = double(a.N) * double(a.K) * double(active > 0 ? active : 1) / kHbmBytesPerUs;
  const int64_t esz = a.out_kind == BSG_OUT_F32 ? 4 : 2;
  const bool whole_rows = host_aligned(a.D, 16) && a.ldd * esz % 16 == 0;      // results leave by TMA
  double best = 1e300;
  bool found = false;
  for (const Variant& of : kVariants) {
    const Variant& v = a.offsets && !of.few && of.tile == 256 ? kTurned : of;
    if ((a.kernel == 1 && !v.few) || (a.kernel == 2 && v.few) || (a.tile && a.tile != v.tile)) continue;
    const int64_t tile_m = v.few ? v.tile : 256, tile_n = v.few ? 128 : v.tile;
    // row tiles: grouped, half of a group's last tile is empty on average
    double tiles_m = double((a.rows + tile_m - 1) / tile_m);
    if (a.offsets) {
      tiles_m = double(a.rows) / double(tile_m) + 0.5 * double(active);
      if (tiles_m < double(active)) tiles_m = double(active);
    }
    const double tiles = tiles_m * double((a.N + tile_n - 1) / tile_n);
    for (int split = 1; split <= 8; split *= 2) {
      if (split > 1 && (!v.few || v.tile > 64 || a.offsets || split > k_tiles)) break;
      if (a.split ? a.split != split : split > 1 && (tiles * split > 296 || k_tiles < split)) continue;
      const double slots = v.few ? 296.0 : 74.0;
      double waves = double(int64_t(tiles * split / slots));
      const double tail = tiles * split - waves * slots;
      if (tail > 0.0) waves += !v.few && v.tile == 256 && waves > 0.0 && 2.0 * tail <= slots ? 0.6 : 1.0;      // a thin last wave is split
      double tile_time = double((k_tiles + split - 1) / split) * v.per_k_tile;
      const double least = v.few || &v == &kTurned || whole_rows ? v.least : 2.0 * v.least;
      if (waves > 1.0 && tile_time < least) tile_time = least;      // (the first tile's epilogue is in `fixed`)
      double t = waves * tile_time;
      if (a.offsets) t = sqrt(t * t + weights * weights);
      else if (t < weights) t = weights;
      t += v.fixed + (split > 1 ? 0.8 + 0.02 * v.tile : 0.0);      // the cluster's barrier and the exchange of partial sums
      if (t < best) {
        best = t;
        found = true;
        plan->few = v.few;
        plan->tile = v.tile;
        plan->split = split;
      }
    }
  }
  if (!found)
    return host_fail(BSG_ERR_NOT_SUPPORTED, "no variant with kernel %d, tile %d and split %d (few rows: 16, 32, 64 or 128 tokens, up to 64 of them "
                     "with a split of 2, 4 or 8, dense, over at least as many 128-value pieces of K; many rows: 128 or 256 columns)", a.kernel, a.tile, a.split);
  return BSG_OK;
}

int32_t check_product(const bsg_int8_args& a, bool own_q, I8Plan* plan) {
  if (a.out_kind != BSG_OUT_BF16 && a.out_kind != BSG_OUT_F16 && a.out_kind != BSG_OUT_F32)
    return host_fail(BSG_ERR_NOT_SUPPORTED, "the 8-bit integer product writes bf16, fp16 or fp32 (output kind %d)", a.out_kind);
  if (a.num_groups < 1 || a.num_groups > BSG_MAX_GROUPS) return host_fail(BSG_ERR_INVALID_PROBLEM, "group count %d outside [1, %d]", a.num_groups, BSG_MAX_GROUPS);
  if (!a.offsets && a.num_groups != 1) return host_fail(BSG_ERR_INVALID_PROBLEM, "%d groups need offsets", a.num_groups);
  if (a.rows < 0 || a.N < 1 || a.K < 1) return host_fail(BSG_ERR_INVALID_PROBLEM, "extents must be positive (rows=%lld N=%lld K=%lld)", (long long)a.rows, (long long)a.N, (long long)a.K);
  if (a.K > bsg::kI8MaxK) return host_fail(BSG_ERR_INVALID_PROBLEM, "K=%lld exceeds %d (32-bit sums)", (long long)a.K, bsg::kI8MaxK);
  if (a.rows > 0x3FFFFFFF || a.N > 0x3FFFFFFF) return host_fail(BSG_ERR_INVALID_PROBLEM, "extent exceeds 2^30");
  if (a.activation < BSG_ACT_IDENTITY || a.activation > BSG_ACT_SILU) return host_fail(BSG_ERR_NOT_SUPPORTED, "unknown activation %d", a.activation);
  if (a.kernel < 0 || a.kernel > 2) return host_fail(BSG_ERR_NOT_SUPPORTED, "unknown kernel %d", a.kernel);
  if (!a.W || !a.w_scale) return host_fail(BSG_ERR_INVALID_PROBLEM, "W and w_scale must not be null");
  if (a.rows > 0 && (!a.D || (own_q && (!a.Q || !a.q_scale)))) return host_fail(BSG_ERR_INVALID_PROBLEM, "Q, q_scale and D must not be null");
  if (!host_aligned(a.W, 16) || a.ldw % 16 != 0 || (own_q && (!host_aligned(a.Q, 16) || a.ldq % 16 != 0)))
    return host_fail(BSG_ERR_MISALIGNED_OPERAND, "rows of Q and W must start on 16-byte boundaries (ldq=%lld, ldw=%lld)", (long long)a.ldq, (long long)a.ldw);
  if (a.ldw < a.K || (own_q && a.ldq < a.K) || a.ldd < a.N) return host_fail(BSG_ERR_INVALID_PROBLEM, "ldq, ldw or ldd is smaller than a row");
  if (a.num_groups > 1 && a.group_stride_w % 16 != 0) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "group_stride_w must be a multiple of 16");
  if (a.num_groups > 1 && a.group_stride_w < a.K) return host_fail(BSG_ERR_INVALID_PROBLEM, "the groups of W overlap (group_stride_w=%lld)", (long long)a.group_stride_w);
  const int esz = a.out_kind == BSG_OUT_F32 ? 4 : 2;
  if (!host_aligned(a.D, esz) || !host_aligned(a.w_scale, 4) || !host_aligned(a.q_scale, 4) || !host_aligned(a.bias, 4) || !host_aligned(a.offsets, 4))
    return host_fail(BSG_ERR_MISALIGNED_OPERAND, "tensors must be aligned to their elements");
  return choose(a, plan);
}

// Raises the dynamic shared-memory limit of a kernel once per device.
struct SmemOnce {
  std::mutex mu;
  bool done[64] = {};
  int32_t set(const void* kernel, int bytes, int dev) {
    if (dev < 0 || dev >= 64) return host_fail(BSG_ERR_NOT_SUPPORTED, "device ordinal %d is outside [0, 64)", dev);
    std::lock_guard<std::mutex> lock(mu);
    if (done[dev]) return BSG_OK;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done[dev] = true;
    return BSG_OK;
  }
};

template <bool FP16, bool WIDE>
int32_t launch_quantise(const bsg::I8QuantParams& p, cudaStream_t s) {
  // A thread keeps up to 64 values, so these rows are read once; one warp per row needs no shared memory.
  cudaError_t e;
  if (p.K <= 32 * 64) e = bsg::host_launch(bsg::bsg_i8_quant_kernel<32, FP16, WIDE>, unsigned(p.rows + 7) / 8, 256, 0, s, p);
  else if (p.K <= 64 * 64) e = bsg::host_launch(bsg::bsg_i8_quant_kernel<64, FP16, WIDE>, unsigned(p.rows + 3) / 4, 256, 0, s, p);
  else if (p.K <= 128 * 64) e = bsg::host_launch(bsg::bsg_i8_quant_kernel<128, FP16, WIDE>, unsigned(p.rows + 1) / 2, 256, 0, s, p);
  else e = bsg::host_launch(bsg::bsg_i8_quant_kernel<512, FP16, WIDE>, unsigned(p.rows), 512, 0, s, p);
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "quantiser launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}

// Whether rows of 16-bit values can be read in groups of eight with single 16-byte loads.
bool wide_rows(const bsg_int8_args& a) { return host_aligned(a.X, 16) && a.K % 8 == 0 && (a.ldx % 8 == 0 || a.tokens <= 1); }

int32_t quantise(const bsg_int8_args& a, cudaStream_t s) {
  if (a.rows == 0) return BSG_OK;
  bsg::I8QuantParams p;
  p.X = static_cast<const uint16_t*>(a.X); p.index = a.index; p.Q = static_cast<int8_t*>(a.Q); p.scale = a.q_scale;
  p.ldx = a.ldx; p.ldq = a.ldq; p.rows = int32_t(a.rows); p.tokens = int32_t(a.tokens); p.K = int32_t(a.K);
  if (wide_rows(a)) return a.in_kind == BSG_OUT_F16 ? launch_quantise<true, true>(p, s) : launch_quantise<false, true>(p, s);
  return a.in_kind == BSG_OUT_F16 ? launch_quantise<true, false>(p, s) : launch_quantise<false, false>(p, s);
}

// Where tokens are used by several rows each, and there is enough of them to pay for one more kernel, they are quantised once
// and copied into order (32768 rows of 4096 tokens x 7168: 60 us instead of 117).
bool copies_rows(const bsg_int8_args& a) { return a.index && a.rows >= 2 * a.tokens && a.rows * a.K >= (int64_t(1) << 24); }

int32_t copy_rows(const bsg_int8_args& a, const void* q, const float* scale, cudaStream_t s) {
  bsg::I8CopyParams p;
  p.Q = static_cast<const int8_t*>(q); p.scale = scale; p.index = a.index; p.out = static_cast<int8_t*>(a.Q); p.out_scale = a.q_scale;
  p.rows = int32_t(a.rows); p.tokens = int32_t(a.tokens); p.pitch = int32_t(a.ldq); p.words = int32_t((a.K + 15) / 16);
  cudaError_t e = bsg::host_launch(bsg::bsg_i8_copy_rows_kernel, unsigned((a.rows + 7) / 8), 256, 0, s, p);
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}

int32_t launch_ex(cudaLaunchConfig_t& cfg, int clusters, bool pdl, cudaLaunchAttribute* attr) {
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(clusters); attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  return BSG_OK;
}

template <int CG, int BN, bool TURN>
int32_t launch_rows(const bsg_int8_args& a, bsg::I8GemmParams& p, cudaStream_t s, int sms, int dev, bool pdl) {
  using C = bsg::I8RowsCfg<CG, BN, TURN>;
  static SmemOnce once;
  auto kernel = bsg::bsg_i8_rows_kernel<CG, BN, TURN>;
  int32_t rc = once.set(reinterpret_cast<const void*>(kernel), C::kSmemBytes, dev);
  if (rc != BSG_OK) return rc;
  CUtensorMap tmA, tmB, tmD;
  if ((rc = bsg::host_operand_map(&tmA, a.Q, a.K, a.rows, 1, a.ldq, a.rows * a.ldq, 128)) != BSG_OK) return rc;
  if ((rc = bsg::host_operand_map(&tmB, a.W, a.K, a.N, a.num_groups, a.ldw, a.num_groups > 1 ? a.group_stride_w : a.N * a.ldw, C::kBRows)) != BSG_OK) return rc;
  const int esz = a.out_kind == BSG_OUT_F32 ? 4 : 2;
  p.tma_out = host_aligned(a.D, 16) && (a.ldd * esz) % 16 == 0;
  p.tma_edge = (a.N * esz) % 16 == 0;
  tmD = tmA;
  if (p.tma_out && (rc = bsg::host_out_map(&tmD, a.D, a.out_kind, a.N, a.rows, a.ldd)) != BSG_OK) return rc;
  p.tiles_n = int32_t((a.N + BN - 1) / BN);
  p.band = 16;
  if (a.rows / C::kTileM + a.num_groups > 0x3FFFFFFF / p.tiles_n) return host_fail(BSG_ERR_INVALID_PROBLEM, "too many tiles for one launch");
  int64_t clusters = sms / CG;
  if (!a.offsets) {
    const int64_t tiles = ((a.rows + C::kTileM - 1) / C::kTileM) * p.tiles_n;
    if (tiles < clusters) clusters = tiles;
  }
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(unsigned(clusters * CG), 1, 1);
  cfg.blockDim = dim3(bsg::kI8RowsThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  launch_ex(cfg, CG, pdl, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tmA, tmB, tmD, p);
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}

template <int BT, int SPLIT>
int32_t launch_few(const bsg_int8_args& a, bsg::I8GemmParams& p, cudaStream_t s, int sms, int dev, bool pdl) {
  using C = bsg::I8FewCfg<BT, SPLIT>;
  constexpr int split = SPLIT;
  static SmemOnce once;
  auto kernel = bsg::bsg_i8_few_kernel<BT, SPLIT>;
  int32_t rc = once.set(reinterpret_cast<const void*>(kernel), C::kSmemBytes, dev);
  if (rc != BSG_OK) return rc;
  CUtensorMap tmW, tmX;
  if ((rc = bsg::host_operand_map(&tmW, a.W, a.K, a.N, a.num_groups, a.ldw, a.num_groups > 1 ? a.group_stride_w : a.N * a.ldw, 128)) != BSG_OK) return rc;
  if ((rc = bsg::host_operand_map(&tmX, a.Q, a.K, a.rows, 1, a.ldq, a.rows * a.ldq, BT)) != BSG_OK) return rc;
  p.tiles_n = int32_t((a.N + 127) / 128);
  p.band = int32_t((a.rows + BT - 1) / BT);      // all token tiles of a channel tile in a row: its weights are then in L2
  if (a.rows / BT + a.num_groups > 0x3FFFFFFF / split / p.tiles_n) return host_fail(BSG_ERR_INVALID_PROBLEM, "too many tiles for one launch");
  p.tma_out = 0;
  int64_t workers = int64_t(2) * sms;
  const int64_t tiles = a.offsets ? (a.rows / BT + a.num_groups) * p.tiles_n : ((a.rows + BT - 1) / BT) * p.tiles_n;
  if (split > 1 || tiles < workers) workers = tiles;      // a split tile is its cluster's only one
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(unsigned(workers * split), 1, 1);
  cfg.blockDim = dim3(192, 1, 1);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  launch_ex(cfg, split, pdl, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tmW, tmX, p);
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}

template <int BT>
int32_t launch_few_split(const bsg_int8_args& a, bsg::I8GemmParams& p, int split, cudaStream_t s, int sms, int dev, bool pdl) {
  switch (split) {
    case 1: return launch_few<BT, 1>(a, p, s, sms, dev, pdl);
    case 2: return launch_few<BT, 2>(a, p, s, sms, dev, pdl);
    case 4: return launch_few<BT, 4>(a, p, s, sms, dev, pdl);
    default: return launch_few<BT, 8>(a, p, s, sms, dev, pdl);
  }
}

// Up to four dense tokens of at most 64 KB in 8 bits: the kernel that quantises on the way.
bool fits_token_kernel(const bsg_int8_args& a) {
  return !a.offsets && !a.index && a.num_groups == 1 && a.rows >= 1 && a.rows <= bsg::kI8TokenMost &&
         int64_t(a.rows <= 1 ? 1 : a.rows <= 2 ? 2 : 4) * ((a.K + 15) / 16 * 16) <= bsg::kI8TokenShared;
}

template <int MT, bool FP16, bool WIDE>
int32_t launch_token(const bsg::I8TokenParams& p, cudaStream_t s, int sms, int dev) {
  static SmemOnce once;
  auto kernel = bsg::bsg_i8_token_kernel<MT, FP16, WIDE>;
  int32_t rc = once.set(reinterpret_cast<const void*>(kernel), bsg::kI8TokenShared, dev);
  if (rc != BSG_OK) return rc;
  const int groups = int((int64_t(p.N) * p.parts + 15) / 16), grid = groups < 2 * sms ? groups : 2 * sms;      // two CTAs fit an SM
  cudaError_t e = bsg::host_launch(kernel, unsigned(grid), bsg::kI8TokenThreads, size_t(MT) * ((p.K + 15) / 16 * 16), s, p);
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}
template <bool FP16, bool WIDE>
int32_t pick_token(const bsg::I8TokenParams& p, cudaStream_t s, int sms, int dev) {
  if (p.M <= 1) return launch_token<1, FP16, WIDE>(p, s, sms, dev);
  if (p.M <= 2) return launch_token<2, FP16, WIDE>(p, s, sms, dev);
  return launch_token<4, FP16, WIDE>(p, s, sms, dev);
}
int32_t token_product(const bsg_int8_args& a, cudaStream_t s, int sms, int dev) {
  bsg::I8TokenParams p;
  p.X = static_cast<const uint16_t*>(a.X); p.W = static_cast<const int8_t*>(a.W); p.sb = a.w_scale; p.bias = a.bias; p.D = a.D;
  p.ldx = a.ldx; p.ldw = a.ldw; p.ldd = a.ldd; p.M = int32_t(a.rows); p.N = int32_t(a.N); p.K = int32_t(a.K);
  p.out_kind = a.out_kind; p.activation = a.activation;
  // Warps share two channels where there would be fewer CTAs than SMs otherwise (every CTA quantises the tokens for itself, so
  // more of them than that cost more than they bring: one token, 4096 x 4096: 6.4 us unshared, 8.5 shared by two; 512 x 16384:
  // 14.3 unshared, 7.0 shared by eight).
  p.parts = 1;
  while (p.parts < 8 && a.N * p.parts < 16 * int64_t(sms) && a.K > p.parts * 512) p.parts *= 2;
  if (wide_rows(a)) return a.in_kind == BSG_OUT_F16 ? pick_token<true, true>(p, s, sms, dev) : pick_token<false, true>(p, s, sms, dev);
  return a.in_kind == BSG_OUT_F16 ? pick_token<true, false>(p, s, sms, dev) : pick_token<false, false>(p, s, sms, dev);
}

int32_t product(const bsg_int8_args& a, const I8Plan& plan, void* workspace, cudaStream_t s, int sms, int dev, bool pdl) {
  bsg::I8GemmParams p;
  memset(&p, 0, sizeof(p));
  p.num_groups = a.num_groups; p.total_rows = int32_t(a.rows); p.N = int32_t(a.N); p.K = int32_t(a.K);
  p.offsets = a.offsets; p.out_kind = a.out_kind; p.activation = a.activation;
  p.sa = a.q_scale; p.sb = a.w_scale; p.bias = a.bias; p.D = a.D; p.ldd = a.ldd;
  p.status = static_cast<uint32_t*>(workspace);
  if (plan.few) {
    switch (plan.tile) {
      case 16: return launch_few_split<16>(a, p, plan.split, s, sms, dev, pdl);
      case 32: return launch_few_split<32>(a, p, plan.split, s, sms, dev, pdl);
      case 64: return launch_few_split<64>(a, p, plan.split, s, sms, dev, pdl);
      default: return launch_few<128, 1>(a, p, s, sms, dev, pdl);
    }
  }
  if (plan.tile == 128) return launch_rows<2, 128, false>(a, p, s, sms, dev, pdl);
  return a.offsets ? launch_rows<2, 256, true>(a, p, s, sms, dev, pdl) : launch_rows<2, 256, false>(a, p, s, sms, dev, pdl);
}

int32_t check_workspace(const void* workspace, size_t bytes) {
  if (!workspace || bytes < 16) return host_fail(BSG_ERR_WORKSPACE_NULL, "a workspace of at least 16 bytes is needed");
  if (!host_aligned(workspace, 4)) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "workspace must be 4-byte aligned");
  return BSG_OK;
}

}  // namespace

extern "C" {

int32_t bsg_int8_query(const bsg_int8_args* args, bsg_caps* caps) {
  if (!args) return host_fail(BSG_ERR_INVALID_PROBLEM, "args is null");
  I8Plan plan;
  int32_t rc = check_product(*args, true, &plan);
  if (rc != BSG_OK) return rc;
  if (caps) {
    memset(caps, 0, sizeof(*caps));
    caps->tile_m = plan.few ? plan.tile : 256;
    caps->tile_n = plan.few ? 128 : plan.tile;
    caps->tile_k = 128;
    caps->cta_group = plan.few ? 1 : 2;
    caps->num_tiles = args->offsets ? -1 : ((args->rows + caps->tile_m - 1) / caps->tile_m) * ((args->N + caps->tile_n - 1) / caps->tile_n);
  }
  return BSG_OK;
}

int32_t bsg_int8_quantize(const bsg_int8_args* args, void* cuda_stream) {
  if (!args) return host_fail(BSG_ERR_INVALID_PROBLEM, "args is null");
  int32_t rc = check_quantise(*args, true);
  int dev = 0, sms = 0;
  if (rc == BSG_OK && args->rows > 0) rc = bsg::host_device(BSG_ERR_ARCH_MISMATCH, BSG_ERR_CUDA, &dev, &sms);
  return rc != BSG_OK ? rc : quantise(*args, static_cast<cudaStream_t>(cuda_stream));
}

int32_t bsg_int8_gemm_run(const bsg_int8_args* args, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  if (!args) return host_fail(BSG_ERR_INVALID_PROBLEM, "args is null");
  I8Plan plan;
  int dev = 0, sms = 0;
  int32_t rc = check_product(*args, true, &plan);
  if (rc == BSG_OK) rc = check_workspace(workspace, workspace_bytes);
  if (rc != BSG_OK || args->rows == 0) return rc;
  if ((rc = bsg::host_device(BSG_ERR_ARCH_MISMATCH, BSG_ERR_CUDA, &dev, &sms)) != BSG_OK) return rc;
  return product(*args, plan, workspace, static_cast<cudaStream_t>(cuda_stream), sms, dev, false);
}

int32_t bsg_int8_linear_run(const bsg_int8_args* args, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  if (!args) return host_fail(BSG_ERR_INVALID_PROBLEM, "args is null");
  I8Plan plan;
  int dev = 0, sms = 0;
  const bool token = !args->Q && !args->q_scale && args->kernel == 0 && fits_token_kernel(*args);
  int32_t rc = check_quantise(*args, !token);
  if (rc == BSG_OK) rc = check_product(*args, !token, &plan);
  if (rc == BSG_OK) rc = check_workspace(workspace, workspace_bytes);
  if (rc != BSG_OK || args->rows == 0) return rc;
  if ((rc = bsg::host_device(BSG_ERR_ARCH_MISMATCH, BSG_ERR_CUDA, &dev, &sms)) != BSG_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  if (token) return token_product(*args, s, sms, dev);
  if (copies_rows(*args)) {
    // the tokens' 8-bit rows and scales lie behind those of the product's rows, with the same pitch
    bsg_int8_args t = *args;
    t.index = nullptr;
    t.rows = args->tokens;
    t.Q = static_cast<int8_t*>(args->Q) + args->rows * args->ldq;
    t.q_scale = args->q_scale + args->rows;
    if ((rc = quantise(t, s)) != BSG_OK || (rc = copy_rows(*args, t.Q, t.q_scale, s)) != BSG_OK) return rc;
  } else if ((rc = quantise(*args, s)) != BSG_OK) {
    return rc;
  }
  return product(*args, plan, workspace, s, sms, dev, true);
}

int32_t bsg_int8_scratch_rows(const bsg_int8_args* args, int64_t* rows) {
  if (!args || !rows) return host_fail(BSG_ERR_INVALID_PROBLEM, "args and rows must not be null");
  *rows = args->rows + (copies_rows(*args) ? args->tokens : 0);
  return BSG_OK;
}

}  // extern "C"
