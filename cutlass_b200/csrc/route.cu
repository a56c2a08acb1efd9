// Host side of the router (bsg_route_*): argument checks and launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>
#include <mutex>

#include "../../include/bsgemm.h"
#include "gemm_kernel.cuh"
#include "host.h"
#include "route_kernel.cuh"

namespace {

using bsg::host_aligned;
using bsg::host_fail;

int64_t route_blocks(int64_t tokens) {
  if (tokens <= bsg::kRouteOneTokens) return 1;
  if (tokens <= bsg::kRouteClusterTokens) return bsg::kRouteClusterCtas;
  const int64_t b = (tokens + 15) / 16;      // at least two tokens a warp
  return b > bsg::kRouteBlocksMax ? bsg::kRouteBlocksMax : b;
}
int64_t route_pitch(int64_t tokens) { return (route_blocks(tokens) + 3) / 4 * 4; }

int32_t check(const bsg_route_args* a, bool forward) {
  if (!a) return host_fail(BSG_ERR_INVALID_PROBLEM, "args is null");
  if (a->type != BSG_OUT_BF16 && a->type != BSG_OUT_F16 && a->type != BSG_OUT_F32) return host_fail(BSG_ERR_NOT_SUPPORTED, "logits must be bf16, fp16 or fp32 (type %d)", a->type);
  if (a->experts < 1 || a->experts > bsg::kRouteMaxExperts) return host_fail(BSG_ERR_INVALID_PROBLEM, "expert count %d outside [1, %d]", a->experts, bsg::kRouteMaxExperts);
  if (a->k < 1 || a->k > bsg::kRouteMaxK || a->k > a->experts) return host_fail(BSG_ERR_INVALID_PROBLEM, "k = %d outside [1, min(%d, %d experts)]", a->k, bsg::kRouteMaxK, a->experts);
  if (a->tokens < 0 || a->tokens * a->k > 0x7FFFFFFFll) return host_fail(BSG_ERR_INVALID_PROBLEM, "%lld tokens with %d choices exceed 2^31 rows", (long long)a->tokens, a->k);
  if (a->normalize != 0 && a->normalize != 1) return host_fail(BSG_ERR_INVALID_PROBLEM, "normalize must be 0 or 1");
  if (!a->counts || !a->live || (forward && (!a->offsets || !a->loss))) return host_fail(BSG_ERR_INVALID_PROBLEM, "per-expert tensors and the loss must not be null");
  if (a->tokens > 0) {
    if (!a->logits || !a->chosen || !a->weights || !a->softmax) return host_fail(BSG_ERR_INVALID_PROBLEM, "logits, chosen, weights and softmax must not be null");
    if (!host_aligned(a->softmax, 8)) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "softmax must be 8-byte aligned");
    if (forward && (!a->rows || !a->positions)) return host_fail(BSG_ERR_INVALID_PROBLEM, "rows and positions must not be null");
    if (!forward && !a->grad_logits) return host_fail(BSG_ERR_INVALID_PROBLEM, "grad_logits must not be null");
    if (a->ld < a->experts || (!forward && a->ld_grad < a->experts)) return host_fail(BSG_ERR_INVALID_PROBLEM, "a row pitch is smaller than the %d experts", a->experts);
    const int esz = a->type == BSG_OUT_F32 ? 4 : 2;
    if (!host_aligned(a->logits, esz) || !host_aligned(a->grad_logits, esz)) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "tensors must be aligned to their elements");
  }
  return BSG_OK;
}

int64_t scratch_words(const bsg_route_args* a) {
  if (a->tokens <= bsg::kRouteClusterTokens) return 0;
  return route_pitch(a->tokens) * (2 * a->experts + 1) + a->experts;
}

bsg::RouteParams params(const bsg_route_args* a, void* scratch) {
  bsg::RouteParams p;
  memset(&p, 0, sizeof(p));
  const int esz = a->type == BSG_OUT_F32 ? 4 : 2;
  p.logits = a->logits; p.ld = a->ld; p.mask = a->mask; p.tokens = int32_t(a->tokens); p.experts = a->experts; p.k = a->k;
  p.normalize = a->normalize; p.wide = host_aligned(a->logits, 16) && (a->ld * esz) % 16 == 0;
  p.chosen = a->chosen; p.weights = a->weights; p.counts = a->counts; p.offsets = a->offsets; p.rows = a->rows;
  p.positions = a->positions; p.loss = a->loss; p.live = a->live;
  p.grad_weights = a->grad_weights; p.grad_loss = a->grad_loss; p.grad_logits = a->grad_logits; p.ld_grad = a->ld_grad;
  p.wide_grad = host_aligned(a->grad_logits, 16) && (a->ld_grad * esz) % 16 == 0;
  const int64_t b = route_blocks(a->tokens);
  p.per_block = int32_t((a->tokens + b - 1) / b);
  p.blocks = int32_t(p.per_block > 0 ? (a->tokens + p.per_block - 1) / p.per_block : 1);
  if (p.blocks < 1) p.blocks = 1;
  int32_t* w = static_cast<int32_t*>(scratch);
  p.pitch = int32_t(route_pitch(a->tokens));
  p.block_counts = w;
  p.block_sums = reinterpret_cast<float*>(w + int64_t(p.pitch) * (a->experts + 1));
  p.sums = p.block_sums + int64_t(p.pitch) * a->experts;
  p.softmax = reinterpret_cast<float2*>(a->softmax);
  return p;
}

// Kernels that use more than 48 KB of shared memory, their few hundred static bytes included, are allowed to once per device.
struct SmemOnce {
  std::mutex mu;
  bool done[64] = {};
  int32_t set(const void* kernel, int bytes, int dev) {
    if (bytes <= 48 * 1024 - kStaticMost) return BSG_OK;
    if (dev < 0 || dev >= 64) return host_fail(BSG_ERR_NOT_SUPPORTED, "device ordinal %d is outside [0, 64)", dev);
    std::lock_guard<std::mutex> lock(mu);
    if (done[dev]) return BSG_OK;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * bsg::kRouteOneWarps * bsg::kRouteMaxExperts * 4);
    if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done[dev] = true;
    return BSG_OK;
  }
  static constexpr int kStaticMost = 1024;      // the arrays of one entry per warp take up to 208
};

template <int TYPE, int V, int ROUNDS>
int32_t forward_v(const bsg::RouteParams& p, int dev, cudaStream_t s) {
  cudaError_t e;
  if (p.tokens <= bsg::kRouteOneTokens) {
    static SmemOnce once;
    auto kernel = bsg::bsg_route_tokens_kernel<TYPE, V, bsg::kRouteOneWarps, 1, ROUNDS>;
    const int shared = 2 * bsg::kRouteOneWarps * p.experts * 4;
    int32_t rc = once.set(reinterpret_cast<const void*>(kernel), shared, dev);
    if (rc != BSG_OK) return rc;
    e = bsg::host_launch(kernel, 1, bsg::kRouteOneWarps * 32, size_t(shared), s, p);
  } else if (p.tokens <= bsg::kRouteClusterTokens) {
    static SmemOnce once;
    auto kernel = bsg::bsg_route_tokens_kernel<TYPE, V, bsg::kRouteOneWarps, bsg::kRouteClusterCtas, ROUNDS>;
    const int shared = 2 * bsg::kRouteOneWarps * p.experts * 4;
    int32_t rc = once.set(reinterpret_cast<const void*>(kernel), shared, dev);
    if (rc != BSG_OK) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(bsg::kRouteClusterCtas, 1, 1);
    cfg.blockDim = dim3(bsg::kRouteOneWarps * 32, 1, 1);
    cfg.dynamicSmemBytes = size_t(shared);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = bsg::kRouteClusterCtas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kernel, p);
  } else {
    static SmemOnce once;
    auto kernel = bsg::bsg_route_tokens_kernel<TYPE, V, bsg::kRouteWarps, 0, ROUNDS>;
    const int shared = 2 * bsg::kRouteWarps * p.experts * 4;
    int32_t rc = once.set(reinterpret_cast<const void*>(kernel), shared, dev);
    if (rc != BSG_OK) return rc;
    e = bsg::host_launch(kernel, unsigned(p.blocks), bsg::kRouteThreads, size_t(shared), s, p);
    if (e == cudaSuccess) e = bsg::host_launch(bsg::bsg_route_scan_kernel, unsigned(p.experts + 1 + 3) / 4, 128, 0, s, p);
    if (e == cudaSuccess) e = bsg::host_launch(bsg::bsg_route_order_kernel, unsigned(p.blocks), bsg::kRouteThreads, 0, s, p);
  }
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "router launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}
// Up to 256 experts (sorted lanes) and k = 8 the rounds are unrolled.
template <int TYPE, int V>
int32_t forward_k(const bsg::RouteParams& p, int dev, cudaStream_t s) {
  if constexpr (V <= 8) {
    if (p.k <= 2) return forward_v<TYPE, V, 2>(p, dev, s);
    if (p.k <= 4) return forward_v<TYPE, V, 4>(p, dev, s);
    if (p.k <= 8) return forward_v<TYPE, V, 8>(p, dev, s);
  }
  return forward_v<TYPE, V, 0>(p, dev, s);
}
template <int TYPE, int V>
int32_t backward_v(const bsg::RouteParams& p, int sms, cudaStream_t s) {
  // one wave of what fits the SMs: a block goes on to its next tokens with their data already asked for
  static std::atomic<int> per_sm{0};      // the same for every device of this architecture
  auto kernel = bsg::bsg_route_backward_kernel<TYPE, V>;
  const size_t shared = size_t(bsg::kRouteWarps) * 32 * V * 4;
  int n = per_sm.load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, bsg::kRouteThreads, shared) != cudaSuccess || n < 1) n = 4;
    per_sm.store(n, std::memory_order_relaxed);
  }
  const int64_t want = (int64_t(p.tokens) + bsg::kRouteWarps - 1) / bsg::kRouteWarps, most = int64_t(n) * sms;
  cudaError_t e = bsg::host_launch(kernel, unsigned(want < most ? want : most), bsg::kRouteThreads, shared, s, p);
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "router launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}
template <int TYPE>
int32_t pick(const bsg::RouteParams& p, bool forward, int dev, int sms, cudaStream_t s) {
#define BSG_ROUTE_V(V) return forward ? forward_k<TYPE, V>(p, dev, s) : backward_v<TYPE, V>(p, sms, s)
  if (p.experts <= 32) BSG_ROUTE_V(1);
  if (p.experts <= 64) BSG_ROUTE_V(2);
  if (p.experts <= 128) BSG_ROUTE_V(4);
  if (p.experts <= 256) BSG_ROUTE_V(8);
  if (p.experts <= 512) BSG_ROUTE_V(16);
  BSG_ROUTE_V(32);
#undef BSG_ROUTE_V
}
int32_t run(const bsg::RouteParams& p, int32_t type, bool forward, int dev, int sms, cudaStream_t s) {
  if (type == BSG_OUT_BF16) return pick<bsg::kRouteBf16>(p, forward, dev, sms, s);
  if (type == BSG_OUT_F16) return pick<bsg::kRouteF16>(p, forward, dev, sms, s);
  return pick<bsg::kRouteF32>(p, forward, dev, sms, s);
}

}  // namespace

extern "C" {

int32_t bsg_route_scratch_size(const bsg_route_args* args, size_t* bytes) {
  if (!args || !bytes) return host_fail(BSG_ERR_INVALID_PROBLEM, "args and bytes must not be null");
  if (args->tokens < 0 || args->experts < 1 || args->experts > bsg::kRouteMaxExperts) return host_fail(BSG_ERR_INVALID_PROBLEM, "extents out of range");
  *bytes = size_t(scratch_words(args)) * 4;
  return BSG_OK;
}

int32_t bsg_route_forward(const bsg_route_args* args, void* scratch, size_t scratch_bytes, void* cuda_stream) {
  int32_t rc = check(args, true);
  if (rc != BSG_OK) return rc;
  if (scratch_words(args) > 0 && (!scratch || scratch_bytes < size_t(scratch_words(args)) * 4)) return host_fail(BSG_ERR_WORKSPACE_NULL, "the router needs %lld bytes of scratch", (long long)scratch_words(args) * 4);
  if (!host_aligned(scratch, 16)) return host_fail(BSG_ERR_MISALIGNED_OPERAND, "scratch must be 16-byte aligned");
  int dev = 0, sms = 0;
  if ((rc = bsg::host_device(BSG_ERR_ARCH_MISMATCH, BSG_ERR_CUDA, &dev, &sms)) != BSG_OK) return rc;
  return run(params(args, scratch), args->type, true, dev, sms, static_cast<cudaStream_t>(cuda_stream));
}

int32_t bsg_route_backward(const bsg_route_args* args, void* cuda_stream) {
  int32_t rc = check(args, false);
  if (rc != BSG_OK || args->tokens == 0) return rc;
  int dev = 0, sms = 0;
  if ((rc = bsg::host_device(BSG_ERR_ARCH_MISMATCH, BSG_ERR_CUDA, &dev, &sms)) != BSG_OK) return rc;
  return run(params(args, nullptr), args->type, false, dev, sms, static_cast<cudaStream_t>(cuda_stream));
}

}  // extern "C"
