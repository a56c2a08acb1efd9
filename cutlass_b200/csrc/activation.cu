// Host side of the checkpointed activation (bsg_act_*): argument checks and launch.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstring>

#include "../../include/bsgemm.h"
#include "activation_kernel.cuh"
#include "host.h"

namespace {

using bsg::host_aligned;
using bsg::host_fail;

int32_t check(const bsg_act_args* a, bool forward) {
  if (!a) return host_fail(BSG_ERR_INVALID_PROBLEM, "args is null");
  if (a->type != BSG_OUT_BF16 && a->type != BSG_OUT_F16) return host_fail(BSG_ERR_NOT_SUPPORTED, "the checkpointed activation takes bf16 or fp16 (type %d)", a->type);
  if (a->activation < BSG_ACT_IDENTITY || a->activation > BSG_ACT_SILU) return host_fail(BSG_ERR_NOT_SUPPORTED, "unknown activation %d", a->activation);
  if (a->gated != 0 && a->gated != 1) return host_fail(BSG_ERR_INVALID_PROBLEM, "gated must be 0 or 1");
  if (a->rows < 0 || a->width < 1 || a->rows > 0x3FFFFFFF || a->width > 0x1FFFFFFF) return host_fail(BSG_ERR_INVALID_PROBLEM, "extents out of range (rows=%lld width=%lld)", (long long)a->rows, (long long)a->width);
  const int64_t blocks = (a->width + bsg::kActBlock - 1) / bsg::kActBlock;
  if (a->rows * blocks > 0x7FFFFFFFll) return host_fail(BSG_ERR_INVALID_PROBLEM, "more than 2^31 blocks of 128 values");
  if (a->rows == 0) return BSG_OK;
  if (!a->in || !a->out || !a->kept || !a->kept_scale) return host_fail(BSG_ERR_INVALID_PROBLEM, "tensors must not be null");
  const int64_t x_cols = a->width * (a->gated ? 2 : 1);
  if (a->ld_in < (forward ? x_cols : a->width) || a->ld_out < (forward ? a->width : x_cols)) return host_fail(BSG_ERR_INVALID_PROBLEM, "a row pitch is smaller than a row");
  if (!host_aligned(a->in, 2) || !host_aligned(a->out, 2) || !host_aligned(a->kept, 16) || !host_aligned(a->kept_scale, 4))
    return host_fail(BSG_ERR_MISALIGNED_OPERAND, "tensors must be aligned to their elements, the kept values to 16 bytes");
  return BSG_OK;
}

template <int ACT, bool GATED, bool FP16, bool WIDE>
cudaError_t launch(const bsg::ActParams& p, bool forward, cudaStream_t s) {
  const unsigned per_cta = bsg::kActThreads / (forward ? bsg::kActForwardLanes : bsg::kActBackwardLanes);
  const unsigned grid = (p.items + per_cta - 1) / per_cta;
  return bsg::host_launch(forward ? bsg::bsg_act_forward_kernel<ACT, GATED, FP16, WIDE> : bsg::bsg_act_backward_kernel<ACT, GATED, FP16, WIDE>, grid,
                          bsg::kActThreads, 0, s, p);
}
template <int ACT, bool GATED, bool FP16>
cudaError_t pick_wide(const bsg::ActParams& p, bool wide, bool forward, cudaStream_t s) {
  return wide ? launch<ACT, GATED, FP16, true>(p, forward, s) : launch<ACT, GATED, FP16, false>(p, forward, s);
}
template <int ACT>
cudaError_t pick(const bsg::ActParams& p, bool gated, bool fp16, bool wide, bool forward, cudaStream_t s) {
  if (gated) return fp16 ? pick_wide<ACT, true, true>(p, wide, forward, s) : pick_wide<ACT, true, false>(p, wide, forward, s);
  return fp16 ? pick_wide<ACT, false, true>(p, wide, forward, s) : pick_wide<ACT, false, false>(p, wide, forward, s);
}

int32_t run(const bsg_act_args* a, bool forward, void* stream) {
  int32_t rc = check(a, forward);
  if (rc != BSG_OK || a->rows == 0) return rc;
  int dev = 0, sms = 0;
  if ((rc = bsg::host_device(BSG_ERR_ARCH_MISMATCH, BSG_ERR_CUDA, &dev, &sms)) != BSG_OK) return rc;
  bsg::ActParams p;
  memset(&p, 0, sizeof(p));
  p.F = int32_t(a->width);
  p.blocks = int32_t((a->width + bsg::kActBlock - 1) / bsg::kActBlock);
  p.pitch = int32_t((a->width + 15) / 16 * 16);
  p.items = uint32_t(a->rows * p.blocks);
  // division of items below 2^31 by the number of blocks d: with l = ceil(log2 d), floor(2^(31 + l) / d) + 1 fits 32 bits and
  // (item * that) >> (31 + l) is exact
  if (p.blocks > 1) {
    int l = 0;
    while ((int64_t(1) << l) < p.blocks) ++l;
    p.div_mul = uint32_t((uint64_t(1) << (31 + l)) / uint64_t(p.blocks) + 1);
    p.div_shift = uint32_t(l - 1);
  }
  p.Q = static_cast<int8_t*>(a->kept); p.scale = a->kept_scale;
  p.Y = static_cast<uint16_t*>(a->out); p.ldy = a->ld_out;
  if (forward) { p.X = static_cast<const uint16_t*>(a->in); p.ldx = a->ld_in; }
  else { p.G = static_cast<const uint16_t*>(a->in); p.ldg = a->ld_in; }
  // every group of 8 values of the input and of the output starts on a 16-byte boundary
  const bool wide = a->width % 8 == 0 && host_aligned(a->in, 16) && a->ld_in % 8 == 0 && host_aligned(a->out, 16) && a->ld_out % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool fp16 = a->type == BSG_OUT_F16;
  cudaError_t e;
  switch (a->activation) {
    case BSG_ACT_RELU: e = pick<bsg::kActRelu>(p, a->gated, fp16, wide, forward, s); break;
    case BSG_ACT_GELU: e = pick<bsg::kActGelu>(p, a->gated, fp16, wide, forward, s); break;
    case BSG_ACT_SILU: e = pick<bsg::kActSilu>(p, a->gated, fp16, wide, forward, s); break;
    default: e = pick<bsg::kActIdentity>(p, a->gated, fp16, wide, forward, s); break;
  }
  if (e != cudaSuccess) return host_fail(BSG_ERR_CUDA, "activation launch: %s", cudaGetErrorString(e));
  return BSG_OK;
}

}  // namespace

extern "C" {
int32_t bsg_act_forward(const bsg_act_args* args, void* cuda_stream) { return run(args, true, cuda_stream); }
int32_t bsg_act_backward(const bsg_act_args* args, void* cuda_stream) { return run(args, false, cuda_stream); }
}
