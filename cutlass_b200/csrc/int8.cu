// Host side of the 8-bit integer product (bsg_int8_*): argument checks, choice of kernel and tile, launch.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstring>
#include <mutex>

#include "../../include/bsgemm.h"
#include "host.h"
#include "int8_kernel.cuh"

namespace {

using bsg::host_aligned;
using bsg::host_fail;

int32_t check_quantise(const bsg_int8_args& a) {
  if (a.in_kind != BSG_OUT_BF16 && a.in_kind != BSG_OUT_F16) return host_fail(BSG_ERR_NOT_SUPPORTED, "X must be bf16 or fp16 (kind %d)", a.in_kind);
  if (a.rows < 0 || a.tokens < 0 || a.K < 1) return host_fail(BSG_ERR_INVALID_PROBLEM, "extents must be positive (rows=%lld tokens=%lld K=%lld)", (long long)a.rows, (long long)a.tokens, (long long)a.K);
  if (a.rows > 0x3FFFFFFF || a.tokens > 0x3FFFFFFF || a.K > 0x3FFFFFFF) return host_fail(BSG_ERR_INVALID_PROBLEM, "extent exceeds 2^30");
  if (!a.index && a.rows != a.tokens) return host_fail(BSG_ERR_INVALID_PROBLEM, "without an index the %lld rows must be the %lld tokens", (long long)a.rows, (long long)a.tokens);
  if (a.rows == 0) return BSG_OK;
  if (!a.Q || !a.q_scale || (!a.X && a.tokens > 0)) return host_fail(BSG_ERR_INVALID_PROBLEM, "X, Q and q_scale must not be null");
  if (!host_aligned(a.X, 2) || !host_aligned(a.q_scale, 4)) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "X and q_scale must be aligned to their elements");
  if (a.ldx < a.K && a.tokens > 1) return host_fail(BSG_ERR_INVALID_PROBLEM, "ldx=%lld is smaller than K", (long long)a.ldx);
  if (a.ldq < a.K || a.ldq % 16 != 0 || !host_aligned(a.Q, 16)) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "rows of Q must start on 16-byte boundaries (ldq=%lld, at least K)", (long long)a.ldq);
  return BSG_OK;
}

struct I8Plan {
  bool few;        // bsg_i8_few_kernel
  int32_t tile;    // few: tokens per tile; rows: columns per tile
  int32_t split;   // few: CTAs of a cluster that share one tile's K
};

int32_t check_product(const bsg_int8_args& a, I8Plan* plan) {
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
  if (a.rows > 0 && (!a.Q || !a.q_scale || !a.D)) return host_fail(BSG_ERR_INVALID_PROBLEM, "Q, q_scale and D must not be null");
  if (!host_aligned(a.W, 16) || a.ldw % 16 != 0 || !host_aligned(a.Q, 16) || a.ldq % 16 != 0)
    return host_fail(BSG_ERR_MISALIGNED_OPERAND, "rows of Q and W must start on 16-byte boundaries (ldq=%lld, ldw=%lld)", (long long)a.ldq, (long long)a.ldw);
  if (a.ldw < a.K || a.ldq < a.K || a.ldd < a.N) return host_fail(BSG_ERR_INVALID_PROBLEM, "ldq, ldw or ldd is smaller than a row");
  if (a.num_groups > 1 && (a.group_stride_w % 16 != 0 || a.group_stride_w < 0)) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "group_stride_w must be a multiple of 16");
  const int esz = a.out_kind == BSG_OUT_F32 ? 4 : 2;
  if (!host_aligned(a.D, esz) || !host_aligned(a.w_scale, 4) || !host_aligned(a.q_scale, 4) || !host_aligned(a.bias, 4) || !host_aligned(a.offsets, 4))
    return host_fail(BSG_ERR_MISALIGNED_OPERAND, "tensors must be aligned to their elements");
  // Tiles.  Grouped: the ragged rows per group live on the device; the mean is what the host knows.
  const int64_t mean = (a.rows + a.num_groups - 1) / a.num_groups;
  plan->few = a.kernel ? a.kernel == 1 : mean <= 128;
  if (plan->few) {
    plan->tile = a.tile ? a.tile : mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : 128;
    if (plan->tile != 16 && plan->tile != 32 && plan->tile != 64 && plan->tile != 128) return host_fail(BSG_ERR_NOT_SUPPORTED, "token tile %d: 16, 32, 64 or 128", plan->tile);
    plan->split = 1;
    if (!a.offsets && plan->tile <= 64) {
      const int64_t tiles = ((a.N + 127) / 128) * ((a.rows + plan->tile - 1) / plan->tile), k_tiles = (a.K + 127) / 128;
      while (plan->split < 8 && tiles * plan->split * 2 <= 296 && k_tiles >= plan->split * 4) plan->split *= 2;
    }
    if (a.split > 1) {
      if (a.offsets || plan->tile > 64 || (a.split != 2 && a.split != 4 && a.split != 8) || a.split > (a.K + 127) / 128)
        return host_fail(BSG_ERR_NOT_SUPPORTED, "split %d: 2, 4 or 8 parts of at least 128 values, dense, token tile up to 64", a.split);
      plan->split = a.split;
    }
  } else {
    plan->tile = a.tile ? a.tile : a.N <= 128 ? 128 : 256;
    plan->split = 1;
    if (plan->tile != 128 && plan->tile != 256) return host_fail(BSG_ERR_NOT_SUPPORTED, "column tile %d: 128 or 256", plan->tile);
    if (a.split > 1) return host_fail(BSG_ERR_NOT_SUPPORTED, "only the kernel for few rows splits K");
  }
  return BSG_OK;
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

template <bool FP16>
int32_t launch_quantise(const bsg::I8QuantParams& p, cudaStream_t s) {
  // A thread keeps up to 64 values, so these rows are read once; one warp per row needs no shared memory.
  if (p.K <= 32 * 64) bsg::bsg_i8_quant_kernel<32, FP16><<<(p.rows + 7) / 8, 256, 0, s>>>(p);
  else if (p.K <= 128 * 64) bsg::bsg_i8_quant_kernel<128, FP16><<<(p.rows + 1) / 2, 256, 0, s>>>(p);
  else bsg::bsg_i8_quant_kernel<512, FP16><<<p.rows, 512, 0, s>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "quantiser launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}

int32_t quantise(const bsg_int8_args& a, cudaStream_t s) {
  if (a.rows == 0) return BSG_OK;
  bsg::I8QuantParams p;
  p.X = static_cast<const uint16_t*>(a.X); p.index = a.index; p.Q = static_cast<int8_t*>(a.Q); p.scale = a.q_scale;
  p.ldx = a.ldx; p.ldq = a.ldq; p.rows = int32_t(a.rows); p.tokens = int32_t(a.tokens); p.K = int32_t(a.K);
  p.fp16 = a.in_kind == BSG_OUT_F16;
  p.wide = host_aligned(a.X, 16) && a.ldx % 8 == 0;
  return p.fp16 ? launch_quantise<true>(p, s) : launch_quantise<false>(p, s);
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

template <int CG, int BN>
int32_t launch_rows(const bsg_int8_args& a, bsg::I8GemmParams& p, cudaStream_t s, int sms, int dev, bool pdl) {
  using C = bsg::I8RowsCfg<CG, BN>;
  static SmemOnce once;
  auto kernel = bsg::bsg_i8_rows_kernel<CG, BN>;
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
  int64_t clusters = sms / CG;
  if (!a.offsets) {
    const int64_t tiles = ((a.rows + C::kTileM - 1) / C::kTileM) * p.tiles_n;
    if (tiles < clusters) clusters = tiles;
  }
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(unsigned(clusters * CG), 1, 1);
  cfg.blockDim = dim3(192, 1, 1);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  launch_ex(cfg, CG, pdl, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tmA, tmB, tmD, p);
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}

template <int BT>
int32_t launch_few(const bsg_int8_args& a, bsg::I8GemmParams& p, int split, cudaStream_t s, int sms, int dev, bool pdl) {
  using C = bsg::I8FewCfg<BT>;
  static SmemOnce once;
  auto kernel = bsg::bsg_i8_few_kernel<BT>;
  int32_t rc = once.set(reinterpret_cast<const void*>(kernel), C::kSmemBytes, dev);
  if (rc != BSG_OK) return rc;
  CUtensorMap tmW, tmX;
  if ((rc = bsg::host_operand_map(&tmW, a.W, a.K, a.N, a.num_groups, a.ldw, a.num_groups > 1 ? a.group_stride_w : a.N * a.ldw, 128)) != BSG_OK) return rc;
  if ((rc = bsg::host_operand_map(&tmX, a.Q, a.K, a.rows, 1, a.ldq, a.rows * a.ldq, BT)) != BSG_OK) return rc;
  p.tiles_n = int32_t((a.N + 127) / 128);
  p.band = 0x3FFFFF / p.tiles_n + 1;      // all token tiles of a channel tile in a row: its weights are then in L2
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
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tmW, tmX, p, int32_t(split));
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return BSG_OK;
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
      case 16: return launch_few<16>(a, p, plan.split, s, sms, dev, pdl);
      case 32: return launch_few<32>(a, p, plan.split, s, sms, dev, pdl);
      case 64: return launch_few<64>(a, p, plan.split, s, sms, dev, pdl);
      default: return launch_few<128>(a, p, plan.split, s, sms, dev, pdl);
    }
  }
  return plan.tile == 128 ? launch_rows<2, 128>(a, p, s, sms, dev, pdl) : launch_rows<2, 256>(a, p, s, sms, dev, pdl);
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
  int32_t rc = check_product(*args, &plan);
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
  int32_t rc = check_quantise(*args);
  int dev = 0, sms = 0;
  if (rc == BSG_OK && args->rows > 0) rc = bsg::host_device(BSG_ERR_ARCH_MISMATCH, BSG_ERR_CUDA, &dev, &sms);
  return rc != BSG_OK ? rc : quantise(*args, static_cast<cudaStream_t>(cuda_stream));
}

int32_t bsg_int8_gemm_run(const bsg_int8_args* args, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  if (!args) return host_fail(BSG_ERR_INVALID_PROBLEM, "args is null");
  I8Plan plan;
  int dev = 0, sms = 0;
  int32_t rc = check_product(*args, &plan);
  if (rc == BSG_OK) rc = check_workspace(workspace, workspace_bytes);
  if (rc != BSG_OK || args->rows == 0) return rc;
  if ((rc = bsg::host_device(BSG_ERR_ARCH_MISMATCH, BSG_ERR_CUDA, &dev, &sms)) != BSG_OK) return rc;
  return product(*args, plan, workspace, static_cast<cudaStream_t>(cuda_stream), sms, dev, false);
}

int32_t bsg_int8_linear_run(const bsg_int8_args* args, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  if (!args) return host_fail(BSG_ERR_INVALID_PROBLEM, "args is null");
  I8Plan plan;
  int dev = 0, sms = 0;
  int32_t rc = check_quantise(*args);
  if (rc == BSG_OK) rc = check_product(*args, &plan);
  if (rc == BSG_OK) rc = check_workspace(workspace, workspace_bytes);
  if (rc != BSG_OK || args->rows == 0) return rc;
  if ((rc = bsg::host_device(BSG_ERR_ARCH_MISMATCH, BSG_ERR_CUDA, &dev, &sms)) != BSG_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  if ((rc = quantise(*args, s)) != BSG_OK) return rc;
  return product(*args, plan, workspace, s, sms, dev, true);
}

}  // extern "C"
