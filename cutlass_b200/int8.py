"""Matrix product in 8-bit integers with one scale per token and one per output channel.

    W = quantize_int8(w)                                          # (N, K) weights, once
    y = int8_linear(x, W.quantized.tensor, W.scale.tensor, bias)  # (M, K) bf16 / fp16 tokens -> (M, N)

``int8_linear`` quantises the tokens and multiplies; with ``offsets`` (and ``rows``) it is the product of a layer of
experts.  Operands that are already quantised go through ``GemmArguments`` / ``GroupedGemmArguments`` and
``get_operators`` like the block-scaled ones (``accumulator_type=torch.int32``).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import lib as L
from .arguments import ACTIVATIONS, ScaledOperand, ScaleSwizzleMode
from .operator import MAX_INT8_K, _default_workspace, to_cuda_stream

_IN_KINDS = {torch.bfloat16: L.OUT_BF16, torch.float16: L.OUT_F16}
_OUT_KINDS = {torch.bfloat16: L.OUT_BF16, torch.float16: L.OUT_F16, torch.float32: L.OUT_F32}


def _on_stream(device, stream, run, *made):
    """Calls ``run(handle)`` with ``device`` current and the raw handle of ``stream`` (None: torch's current stream of that
    device).  ``made`` are tensors this module allocated on the current stream: another stream's use of them is recorded."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _on_stream(device, stream, run, *made)
    handle = torch.cuda.current_stream().cuda_stream
    if stream is not None and to_cuda_stream(stream) != handle:
        handle = to_cuda_stream(stream)
        other = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
        for t in made:
            t.record_stream(other)
    return run(handle)


def _no_gradient(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad() or detach its inputs")


def _check_tokens(x) -> None:
    if x.dim() != 2 or x.dtype not in _IN_KINDS or not x.is_cuda or (x.stride(1) != 1 and x.shape[1] > 1):
        raise ValueError("x must be a 2-D bf16 or fp16 CUDA tensor with unit stride along K")
    if x.shape[1] < 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        raise ValueError("x must have at least one column and rows that do not overlap")


def _check_vector(name, t, dtype, shape, device) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {device}")


def quantize_int8(x, *, rows=None, out=None, scale_out=None, stream=None) -> ScaledOperand:
    """Quantise every row of ``x`` (M, K) bf16 / fp16 to 8 bits: ``scale = max|x| / 127`` (fp32) and
    ``quantized = sign(x) floor(127 |x| / max|x| + 1/2)``.  A row with a NaN or an infinity gets scale NaN and zeros.

    ``rows`` (int32, R entries): row r of the result is made from ``x[rows[r]]`` (an entry outside ``x`` gives zeros with
    scale NaN), as a grouped product wants its tokens.  The result's rows start on 16-byte boundaries, whatever K is.
    ``out`` (R, K) int8 with such rows and ``scale_out`` (R,) fp32 may be given.  Asynchronous on ``stream`` (None: torch's
    current stream)."""
    _check_tokens(x)
    _no_gradient("quantize_int8", x)
    M, K = x.shape
    if rows is not None and (rows.dim() != 1 or rows.dtype != torch.int32 or not rows.is_contiguous() or rows.device != x.device):
        raise ValueError("rows must be a contiguous 1-D int32 tensor on the device of x")
    R = M if rows is None else rows.shape[0]
    made = []
    if out is None:
        made.append(torch.empty((R, -(-K // 16) * 16), dtype=torch.int8, device=x.device))
        out = made[-1][:, :K]
    elif tuple(out.shape) != (R, K) or out.dtype != torch.int8 or out.device != x.device or (K > 1 and out.stride(1) != 1) \
            or (R > 1 and (out.stride(0) < K or out.stride(0) % 16 != 0)) or out.data_ptr() % 16 != 0:
        raise ValueError(f"out must be an int8 tensor of shape {(R, K)} on {x.device} whose rows start on 16-byte boundaries")
    if scale_out is None:
        scale_out = torch.empty(R, dtype=torch.float32, device=x.device)
        made.append(scale_out)
    _check_vector("scale_out", scale_out, torch.float32, (R,), x.device)
    a = L.Int8Args()
    a.in_kind, a.rows, a.tokens, a.K = _IN_KINDS[x.dtype], R, M, K
    a.X, a.ldx = x.data_ptr(), x.stride(0) if M > 1 else K
    a.index = rows.data_ptr() if rows is not None else None
    a.Q, a.ldq, a.q_scale = out.data_ptr(), out.stride(0) if R > 1 else -(-K // 16) * 16, scale_out.data_ptr()
    _on_stream(x.device, stream, lambda s: L.check(L.load().bsg_int8_quantize(C.byref(a), s)), *made)
    return ScaledOperand(out, scale_out, (1, 1, K), ScaleSwizzleMode.SwizzleNone)


def int8_linear(x, weight, weight_scale, bias=None, *, activation="identity", offsets=None, rows=None, out=None,
                out_dtype=None, stream=None) -> torch.Tensor:
    """``act(x @ (weight_scale * weight)^T + bias)`` with ``x`` (M, K) bf16 / fp16 quantised per row on the way (see
    ``quantize_int8``) and exact integer sums; ``weight`` (N, K) int8 with rows on 16-byte boundaries (what
    ``quantize_int8`` returns), ``weight_scale`` and ``bias`` (N,) fp32.  ``out_dtype``: bf16, fp16 or fp32 (default: that
    of ``x``).  ``activation``: "identity", "relu", "gelu" (erf form) or "silu".  K is at most 131071.

    Experts: with ``offsets`` (E,) int32, the cumulative end rows of a grouped product, ``weight`` is (E, N, K),
    ``weight_scale`` and ``bias`` are (E, N).  ``rows`` (R,) int32 names the token of every row, so that tokens need not be
    copied into expert order first (``route_tokens`` makes both).  Rows of the result at or behind the last end row are not
    written.  Offsets that fall or leave the rows are clamped and reported by ``check_device_status`` of an operator.

    No gradient is kept.  Asynchronous on ``stream`` (None: torch's current stream)."""
    _check_tokens(x)
    _no_gradient("int8_linear", x, weight_scale, bias)
    M, K = x.shape
    device = x.device
    grouped = offsets is not None
    if weight.dim() != (3 if grouped else 2) or weight.dtype != torch.int8 or weight.device != device or weight.shape[-1] != K:
        raise ValueError(f"weight must be an int8 tensor of shape {'(experts, N, K)' if grouped else '(N, K)'} with K = {K} on {device}")
    N = weight.shape[-2]
    strides = weight.stride()
    if N < 1 or (K > 1 and strides[-1] != 1) or (N > 1 and (strides[-2] < K or strides[-2] % 16 != 0)) or weight.data_ptr() % 16 != 0 \
            or (grouped and weight.shape[0] > 1 and strides[0] % 16 != 0):
        raise ValueError("the rows of weight must have unit stride along K and start on 16-byte boundaries (quantize_int8 lays them out so)")
    per_channel = (weight.shape[0], N) if grouped else (N,)
    _check_vector("weight_scale", weight_scale, torch.float32, per_channel, device)
    if bias is not None:
        _check_vector("bias", bias, torch.float32, per_channel, device)
    if grouped:
        if not 1 <= weight.shape[0] <= L.MAX_GROUPS:
            raise ValueError(f"between 1 and {L.MAX_GROUPS} experts are supported, got {weight.shape[0]}")
        _check_vector("offsets", offsets, torch.int32, (weight.shape[0],), device)
    if rows is not None and (not grouped or rows.dim() != 1 or rows.dtype != torch.int32 or not rows.is_contiguous() or rows.device != device):
        raise ValueError("rows must be a contiguous 1-D int32 tensor on the device of x, and goes with offsets")
    if K > MAX_INT8_K:
        raise ValueError(f"K={K} exceeds {MAX_INT8_K} (32-bit sums)")
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: one of {sorted(ACTIVATIONS)}")
    R = M if rows is None else rows.shape[0]
    pitch = -(-K // 16) * 16
    scratch = torch.empty(R * (pitch + 4), dtype=torch.int8, device=device)        # 8-bit tokens, then their scales
    made = [scratch]
    if out is None:
        out = torch.empty((R, N), dtype=out_dtype or x.dtype, device=device)
        made.append(out)
    elif tuple(out.shape) != (R, N) or out.device != device or (out_dtype is not None and out.dtype != out_dtype) \
            or (N > 1 and out.stride(1) != 1) or (R > 1 and out.stride(0) < N):
        raise ValueError(f"out must be a row-major {out_dtype or 'bf16, fp16 or fp32'} tensor of shape {(R, N)} on {device}")
    if out.dtype not in _OUT_KINDS:
        raise ValueError(f"out dtype {out.dtype} is not supported (bf16, fp16 or fp32)")
    if R == 0:
        return out
    q = scratch.data_ptr()
    a = L.Int8Args(
        _IN_KINDS[x.dtype], _OUT_KINDS[out.dtype], weight.shape[0] if grouped else 1, ACTIVATIONS[activation], R, M, N, K,
        x.data_ptr(), x.stride(0) if M > 1 else K, rows.data_ptr() if rows is not None else None, q, pitch, q + R * pitch,
        weight.data_ptr(), strides[-2] if N > 1 else pitch, strides[0] if grouped and weight.shape[0] > 1 else 0,
        weight_scale.data_ptr(), bias.data_ptr() if bias is not None else None, offsets.data_ptr() if grouped else None,
        out.data_ptr(), out.stride(0) if R > 1 else N)
    ws = _default_workspace(device)
    _on_stream(device, stream, lambda s: L.check(L.load().bsg_int8_linear_run(C.byref(a), ws.data_ptr(), 16, s)), *made)
    return out
