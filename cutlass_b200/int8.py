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
from torch.autograd import forward_ad

from . import lib as L
from .arguments import ACTIVATIONS, ScaledOperand, ScaleSwizzleMode
from .operator import MAX_INT8_K, _default_workspace, _default_workspaces, to_cuda_stream

_IN_KINDS = {torch.bfloat16: L.OUT_BF16, torch.float16: L.OUT_F16}
_OUT_KINDS = {torch.bfloat16: L.OUT_BF16, torch.float16: L.OUT_F16, torch.float32: L.OUT_F32}
_POWER = (1, 1, 2, 4, 4)       # number of tokens -> the next power of two
_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _launch(device: int, call, *args) -> None:
    """``call(*args, handle)`` with ``device`` current and the raw handle of torch's current stream of that device."""
    if device != _current_device():
        with torch.cuda.device(device):
            return _launch(device, call, *args)
    code = call(*args, _current_stream(device))
    if code:
        L.check(code)


def _other_stream(x, stream):
    """``stream`` as a torch stream, where it is another one than torch's current stream of the device of ``x``; else None."""
    device = x.get_device()
    if stream is None or device < 0:
        return None
    handle = to_cuda_stream(stream)
    if handle == _current_stream(device):
        return None
    return torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)


def _elsewhere(other, call, *args, out=None, **more):
    """``call`` with ``other`` as torch's current stream, so that what it allocates is memory of that stream: a block that the
    current stream has given back may still be in use by work queued there, for which ``other`` does not wait.  What is returned
    is not reused before the work that the stream of the caller has queued by the time it is freed."""
    here = torch.cuda.current_stream(other.device)
    with torch.cuda.stream(other):
        made = call(*args, **more) if out is None else call(*args, out=out, **more)

    def keep(t):
        if isinstance(t, ScaledOperand):
            t = (t.quantized.tensor, t.scale.tensor)
        if isinstance(t, tuple):
            for part in t:
                keep(part)
        elif isinstance(t, torch.Tensor) and t is not out:
            t.record_stream(here)
    keep(made)
    return made


def _pitch(K: int) -> int:
    """Bytes between 8-bit rows.  Rows on 128-byte boundaries, where they are longer: a copy of 128 of a row's bytes by TMA then
    takes one line of L2 instead of two (777 x 5000 x 2050, tokens and weights: 15.0 us, on 16-byte boundaries 20.2; only the
    tokens 17.4)."""
    return (K + 15) & ~15 if K <= 128 else (K + 127) & ~127


def _no_tangent(name, *tensors) -> None:
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has no forward-mode derivative: its inputs must not carry tangents")


def _no_gradient(name, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no gradient: call it under torch.no_grad() or detach its inputs")
    _no_tangent(name, *tensors)


def _no_lazy_sign(name, t) -> None:
    if t.is_neg():
        raise ValueError(f"{name} is a view with its sign turned, which its memory does not show: pass {name}.resolve_neg()")


def _matrix(name, t, kinds):
    """(kind, device index, rows, columns, row pitch) of a row-major CUDA matrix; columns that do not overlap."""
    shape, kind, device = t.shape, kinds.get(t.dtype), t.get_device()
    if len(shape) != 2 or kind is None or device < 0:
        raise ValueError(f"{name} must be a 2-D CUDA tensor of type {', '.join(str(k) for k in kinds)}, got {t.dtype} {tuple(shape)} on {t.device}")
    _no_lazy_sign(name, t)
    rows, cols = shape
    pitch, step = t.stride()
    if cols < 1 or (step != 1 and cols > 1 and rows > 0) or (rows > 1 and pitch < cols):
        raise ValueError(f"{name} must have at least one column, unit stride along its columns and rows that do not overlap")
    return kind, device, rows, cols, (pitch if rows > 1 else cols)


def _share_memory(a, b) -> bool:
    """Whether two row-major matrices have a byte in common (or may have: pitches that differ)."""
    spans = []
    for t in (a, b):
        size = t.element_size()
        pitch = (t.stride(0) if t.shape[0] > 1 else t.shape[1]) * size
        spans.append((t.data_ptr(), pitch, t.shape[1] * size, (t.shape[0] - 1) * pitch + t.shape[1] * size if t.numel() else 0))
    (p, p_pitch, p_row, p_all), (q, q_pitch, q_row, q_all) = spans
    if p + p_all <= q or q + q_all <= p or not p_all or not q_all:
        return False
    if a.shape[0] > 1 and b.shape[0] > 1 and p_pitch == q_pitch:
        behind = (q - p) % p_pitch      # columns of one buffer, side by side
        return behind < p_row or behind + q_row > p_pitch
    return True


def _check_array(name, t, dtype, shape, device) -> None:
    if t.dtype != dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on CUDA device {device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    _no_lazy_sign(name, t)


def _check_rows(rows, device) -> int:
    if rows.dtype != torch.int32 or rows.dim() != 1 or rows.get_device() != device or not rows.is_contiguous():
        raise ValueError("rows must be a contiguous 1-D int32 tensor on the device of x")
    return rows.shape[0]


def quantize_int8(x, *, rows=None, out=None, scale_out=None, stream=None) -> ScaledOperand:
    """Quantise every row of ``x`` (M, K) bf16 / fp16 to 8 bits: ``scale = max|x| / 127`` (fp32) and
    ``quantized = sign(x) floor(127 |x| / max|x| + 1/2)``.  A row with a NaN or an infinity gets scale NaN and zeros.

    ``rows`` (int32, R entries): row r of the result is made from ``x[rows[r]]`` (an entry outside ``x`` gives zeros with
    scale NaN), as a grouped product wants its tokens.  The result's rows start on 128-byte boundaries (up to K = 128: 16-byte).
    ``out`` (R, K) int8 with rows on 16-byte boundaries and ``scale_out`` (R,) fp32 may be given.  Asynchronous on ``stream`` (None: torch's
    current stream)."""
    other = _other_stream(x, stream)
    if other is not None:
        return _elsewhere(other, quantize_int8, x, rows=rows, out=out, scale_out=scale_out)
    kind, device, M, K, ldx = _matrix("x", x, _IN_KINDS)
    _no_gradient("quantize_int8", x)
    R = M if rows is None else _check_rows(rows, device)
    if out is None:
        out = torch.empty((R, _pitch(K)), dtype=torch.int8, device=x.device)[:, :K]
    elif tuple(out.shape) != (R, K) or out.dtype != torch.int8 or out.device != x.device or (K > 1 and out.stride(1) != 1) \
            or (R > 1 and (out.stride(0) < K or out.stride(0) % 16 != 0)) or out.data_ptr() % 16 != 0:
        raise ValueError(f"out must be an int8 tensor of shape {(R, K)} on {x.device} whose rows start on 16-byte boundaries")
    if scale_out is None:
        scale_out = torch.empty(R, dtype=torch.float32, device=x.device)
    _check_array("scale_out", scale_out, torch.float32, (R,), device)
    pack, call = L.direct("bsg_int8_quantize", L.INT8_LAYOUT)
    args = pack(kind, 0, 1, 0, R, M, 1, K, x.data_ptr(), ldx, 0 if rows is None else rows.data_ptr(), out.data_ptr(),
                out.stride(0) if R > 1 else _pitch(K), scale_out.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    _launch(device, call, args)
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

    ``out`` may share memory with ``x``.  No gradient is kept.  Asynchronous on ``stream`` (None: torch's current stream)."""
    if out is None and stream is None and x.is_cuda:
        y = L.binding().int8_linear(x, weight, weight_scale, bias, activation, offsets, rows, out_dtype)
        if y is not None:
            return y
    other = _other_stream(x, stream)
    if other is not None:
        return _elsewhere(other, int8_linear, x, weight, weight_scale, bias, activation=activation, offsets=offsets, rows=rows, out=out, out_dtype=out_dtype)
    in_kind, device, M, K, ldx = _matrix("x", x, _IN_KINDS)
    _no_gradient("int8_linear", x, weight_scale, bias)
    shape, strides, w = weight.shape, weight.stride(), weight.data_ptr()
    if offsets is None:
        if rows is not None:
            raise ValueError("rows goes with offsets")
        if len(shape) != 2:
            raise ValueError(f"weight must be (N, K), or (experts, N, K) with offsets; got {tuple(shape)}")
        experts, group_stride, R, per_channel = 1, 0, M, shape[:1]
    else:
        if len(shape) != 3 or not 1 <= shape[0] <= L.MAX_GROUPS:
            raise ValueError(f"with offsets, weight must be (experts, N, K) with 1 to {L.MAX_GROUPS} experts; got {tuple(shape)}")
        experts, per_channel = shape[0], shape[:2]
        group_stride = strides[0] if experts > 1 else 0
        _check_array("offsets", offsets, torch.int32, shape[:1], device)
        R = M if rows is None else _check_rows(rows, device)
    N, whole, pitch = shape[-2], (K + 15) & ~15, _pitch(K)
    ldw = strides[-2] if N > 1 else whole
    if weight.dtype != torch.int8 or weight.get_device() != device or shape[-1] != K or N < 1:
        raise ValueError(f"weight must be an int8 tensor on CUDA device {device} whose last extent is K = {K}, got {weight.dtype} {tuple(shape)} on {weight.device}")
    if (strides[-1] != 1 and K > 1) or ldw < K or ldw & 15 or w & 15 or group_stride & 15 or (experts > 1 and group_stride < K):
        raise ValueError("the rows of weight must have unit stride along K, start on 16-byte boundaries (quantize_int8 lays them out so) and not overlap")
    _check_array("weight_scale", weight_scale, torch.float32, per_channel, device)
    if bias is not None:
        _check_array("bias", bias, torch.float32, per_channel, device)
    if K > MAX_INT8_K:
        raise ValueError(f"K={K} exceeds {MAX_INT8_K} (32-bit sums)")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}: one of {sorted(ACTIVATIONS)}")
    if out is None:
        out, ldd = x.new_empty((R, N), dtype=out_dtype), N
        out_kind = _OUT_KINDS.get(out.dtype)
    else:
        out_kind, out_device, out_rows, out_cols, ldd = _matrix("out", out, _OUT_KINDS)
        if (out_rows, out_cols, out_device) != (R, N, device) or (out_dtype is not None and out.dtype != out_dtype):
            raise ValueError(f"out must be a {out_dtype or ''} tensor of shape {(R, N)} on CUDA device {device}")
    if out_kind is None:
        raise ValueError(f"out dtype {out.dtype} is not supported (bf16, fp16 or fp32)")
    if R == 0:
        return out
    if offsets is None and R <= 4 and _POWER[R] * whole <= 65536 and not _share_memory(x, out):
        q = q_scale = 0      # quantised inside the product's kernel, whose blocks read x while others already write
    else:
        held = R
        if rows is not None:      # tokens that several rows use may be held twice: as they come, and in the order of the rows
            count = C.c_int64()
            L.check(L.load().bsg_int8_scratch_rows(C.byref(L.Int8Args(rows=R, tokens=M, K=K, index=rows.data_ptr())), C.byref(count)))
            held = count.value
        scratch = x.new_empty(held * (pitch + 4), dtype=torch.int8)       # 8-bit tokens, then their scales
        q = scratch.data_ptr()
        q_scale = q + held * pitch
    status = _default_workspaces.get(device)
    if status is None:
        status = _default_workspace(x.device)
    pack, call = L.direct("bsg_int8_linear_run", L.INT8_LAYOUT)
    args = pack(in_kind, out_kind, experts, act, R, M, N, K, x.data_ptr(), ldx, 0 if rows is None else rows.data_ptr(), q, pitch,
                q_scale, w, ldw, group_stride, weight_scale.data_ptr(), 0 if bias is None else bias.data_ptr(),
                0 if offsets is None else offsets.data_ptr(), out.data_ptr(), ldd, 0, 0, 0, 0)
    _launch(device, call, args, status.data_ptr(), 16)
    return out
