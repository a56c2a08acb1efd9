"""Activation between the two products of an MLP layer, with its input kept in 8 bits for the backward pass.

    h, kept = checkpoint_activation(x, "silu")            # x (T, 2F) = (gate | up) -> h (T, F) = silu(gate) * up
    dx = checkpoint_activation_backward(dh, kept)         # (T, 2F)
    h = checkpointed_activation(x, "silu")                # the same through torch's autograd

What is kept is one byte per value of ``x`` and one fp32 scale per 128 of them, instead of ``x`` itself.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import lib as L
from .arguments import ACTIVATIONS
from .int8 import _IN_KINDS, _no_gradient, _on_stream

BLOCK = 128      # columns of a row that share one scale


@dataclass
class ActivationCheckpoint:
    """Input of an activation in 8 bits: ``quantized`` (T, parts, F rounded up to 16) int8 and ``scale`` (T, parts, F / 128
    rounded up) fp32, with parts = 2 (gate, up) when ``gated``, else 1; its value is ``scale * quantized`` per block."""

    quantized: torch.Tensor
    scale: torch.Tensor
    activation: str
    gated: bool
    width: int
    dtype: torch.dtype

    def nbytes(self) -> int:
        return self.quantized.numel() + 4 * self.scale.numel()


def _check_matrix(name, t, cols, dtype=None, rows=None, device=None) -> None:
    if t.dim() != 2 or t.dtype not in _IN_KINDS or not t.is_cuda or (t.shape[1] > 1 and t.stride(1) != 1) \
            or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} must be a 2-D row-major bf16 or fp16 CUDA tensor")
    if t.shape[1] < 1 or (cols is not None and t.shape[1] != cols) or (rows is not None and t.shape[0] != rows) \
            or (dtype is not None and t.dtype != dtype) or (device is not None and t.device != device):
        raise ValueError(f"{name} must be a {dtype} tensor of shape {(rows, cols)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def checkpoint_activation(x, activation: str = "silu", *, gated: bool = True, out=None, stream=None):
    """``(h, kept)``: ``h = act(x[:, :F]) * x[:, F:]`` for ``gated`` (x has 2F columns), else ``act(x)``, computed from ``x``
    itself, and the ``ActivationCheckpoint`` that ``checkpoint_activation_backward`` takes.  ``x`` is (T, 2F) or (T, F) bf16 /
    fp16; ``activation``: "identity", "relu", "gelu" (erf form) or "silu"; ``out`` (T, F) may be given.  A block of 128 values
    with a NaN or an infinity is kept as NaN.  Asynchronous on ``stream`` (None: torch's current stream)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: one of {sorted(ACTIVATIONS)}")
    _check_matrix("x", x, None)
    _no_gradient("checkpoint_activation", x)
    T, cols = x.shape
    if gated and cols % 2 != 0:
        raise ValueError(f"a gated activation needs an even number of columns (gate | up), got {cols}")
    parts = 2 if gated else 1
    F = cols // parts
    device = x.device
    made = [torch.empty((T, parts, -(-F // 16) * 16), dtype=torch.int8, device=device),
            torch.empty((T, parts, -(-F // BLOCK)), dtype=torch.float32, device=device)]
    kept = ActivationCheckpoint(made[0], made[1], activation, bool(gated), F, x.dtype)
    if out is None:
        out = torch.empty((T, F), dtype=x.dtype, device=device)
        made.append(out)
    else:
        _check_matrix("out", out, F, x.dtype, T, device)
    a = L.ActArgs(_IN_KINDS[x.dtype], ACTIVATIONS[activation], parts - 1, 0, T, F, x.data_ptr(), x.stride(0) if T > 1 else cols,
                  out.data_ptr(), out.stride(0) if T > 1 else F, made[0].data_ptr(), made[1].data_ptr())
    _on_stream(device, stream, lambda s: L.check(L.load().bsg_act_forward(C.byref(a), s)), *made)
    return out, kept


def checkpoint_activation_backward(grad, kept: ActivationCheckpoint, *, out=None, stream=None) -> torch.Tensor:
    """Gradient of ``x`` for the gradient ``grad`` (T, F) of ``h``, from what ``checkpoint_activation`` kept: (T, 2F) or (T, F)
    in the type of ``x``.  ``out`` may be given.  Asynchronous on ``stream`` (None: torch's current stream)."""
    T, parts, F = kept.quantized.shape[0], 2 if kept.gated else 1, kept.width
    device = kept.quantized.device
    _check_matrix("grad", grad, F, kept.dtype, T, device)
    _no_gradient("checkpoint_activation_backward", grad)
    made = []
    if out is None:
        out = torch.empty((T, parts * F), dtype=kept.dtype, device=device)
        made.append(out)
    else:
        _check_matrix("out", out, parts * F, kept.dtype, T, device)
    a = L.ActArgs(_IN_KINDS[kept.dtype], ACTIVATIONS[kept.activation], parts - 1, 0, T, F, grad.data_ptr(), grad.stride(0) if T > 1 else F,
                  out.data_ptr(), out.stride(0) if T > 1 else parts * F, kept.quantized.data_ptr(), kept.scale.data_ptr())
    _on_stream(device, stream, lambda s: L.check(L.load().bsg_act_backward(C.byref(a), s)), *made)
    return out


class _CheckpointedActivation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, activation, gated):
        h, kept = checkpoint_activation(x, activation, gated=gated)
        ctx.save_for_backward(kept.quantized, kept.scale)
        ctx.how = (activation, kept.gated, kept.width, kept.dtype)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        kept = ActivationCheckpoint(*ctx.saved_tensors, *ctx.how)
        if grad.stride(1) != 1 or (grad.shape[0] > 1 and grad.stride(0) < grad.shape[1]):      # e.g. an expanded gradient
            grad = grad.contiguous()
        return checkpoint_activation_backward(grad, kept), None, None


def checkpointed_activation(x, activation: str = "silu", *, gated: bool = True) -> torch.Tensor:
    """``checkpoint_activation`` under autograd: only the 8-bit checkpoint is kept for the backward pass, not ``x``.  Runs on
    torch's current stream."""
    return _CheckpointedActivation.apply(x, activation, gated)
