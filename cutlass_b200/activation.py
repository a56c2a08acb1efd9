"""Activation between the two products of an MLP layer, with its input kept in 8 bits for the backward pass.

    h, kept = checkpoint_activation(x, "silu")            # x (T, 2F) = (gate | up) -> h (T, F) = silu(gate) * up
    dx = checkpoint_activation_backward(dh, kept)         # (T, 2F)
    h = checkpointed_activation(x, "silu")                # the same through torch's autograd

What is kept is one byte per value of ``x`` and one fp32 scale per 128 of them, instead of ``x`` itself.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import lib as L
from .arguments import ACTIVATIONS
from .int8 import _IN_KINDS, _check_array, _elsewhere, _launch, _matrix, _no_gradient, _other_stream, _share_memory

BLOCK = 128      # columns of a row that share one scale


class ActivationCheckpoint(NamedTuple):
    """Input of an activation in 8 bits: ``quantized`` (T, parts, F rounded up to 16) int8 and ``scale`` (T, parts, F / 128
    rounded up) fp32, with parts = 2 (gate, up) when ``gated``, else 1; its value is ``scale * quantized`` per block.  Both lie
    in one buffer, ``data``."""

    data: torch.Tensor
    activation: str
    gated: bool
    rows: int
    width: int
    dtype: torch.dtype

    def _split(self) -> int:
        return self.rows * (2 if self.gated else 1) * ((self.width + 15) & ~15)

    @property
    def quantized(self) -> torch.Tensor:
        return self.data[:self._split()].view(self.rows, 2 if self.gated else 1, (self.width + 15) & ~15)

    @property
    def scale(self) -> torch.Tensor:
        return self.data[self._split():].view(torch.float32).view(self.rows, 2 if self.gated else 1, -(-self.width // BLOCK))

    def nbytes(self) -> int:
        return self.data.numel()


def _given(name, t, kind, device, rows, cols) -> int:
    """Row pitch of a matrix of the caller's that has to have this type, place and shape."""
    k, d, r, c, pitch = _matrix(name, t, _IN_KINDS)
    if (k, d, r, c) != (kind, device, rows, cols):
        raise ValueError(f"{name} must have the type of x, on CUDA device {device}, and shape {(rows, cols)}; got {t.dtype} {(r, c)} on {t.device}")
    return pitch


def _check_place(out, inp, ld_out, ld_in) -> None:
    """A result may lie where its input lies, value on value (every value is read before its place is written), or elsewhere."""
    if _share_memory(out, inp) and (out.data_ptr() != inp.data_ptr() or (ld_out != ld_in and out.shape[0] > 1)):
        raise ValueError("out must begin where the input begins, with the same distance between rows, or share no memory with it")


def checkpoint_activation(x, activation: str = "silu", *, gated: bool = True, out=None, stream=None):
    """``(h, kept)``: ``h = act(x[:, :F]) * x[:, F:]`` for ``gated`` (x has 2F columns), else ``act(x)``, computed from ``x``
    itself, and the ``ActivationCheckpoint`` that ``checkpoint_activation_backward`` takes.  ``x`` is (T, 2F) or (T, F) bf16 /
    fp16; ``activation``: "identity", "relu", "gelu" (erf form) or "silu"; ``out`` (T, F) may be given, also the columns of ``x`` that it begins with.  A block of 128 values
    with a NaN or an infinity is kept as NaN.  Asynchronous on ``stream`` (None: torch's current stream)."""
    if out is None and stream is None and x.is_cuda:
        done = L.binding().act_forward(x, activation, gated)
        if done is not None:
            return done
    other = _other_stream(x, stream)
    if other is not None:
        return _elsewhere(other, checkpoint_activation, x, activation, gated=gated, out=out)
    gated = bool(gated)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}: one of {sorted(ACTIVATIONS)}")
    kind, device, T, cols, ldx = _matrix("x", x, _IN_KINDS)
    _no_gradient("checkpoint_activation", x)
    if gated and cols % 2 != 0:
        raise ValueError(f"a gated activation needs an even number of columns (gate | up), got {cols}")
    parts, F = (2, cols // 2) if gated else (1, cols)
    split = T * parts * ((F + 15) & ~15)
    data = x.new_empty(split + 4 * T * parts * ((F + BLOCK - 1) // BLOCK), dtype=torch.int8)
    if out is None:
        out, ldh = x.new_empty((T, F)), F
    else:
        ldh = _given("out", out, kind, device, T, F)
        _check_place(out, x, ldh, ldx)
    q = data.data_ptr()
    pack, call = L.direct("bsg_act_forward", L.ACT_LAYOUT)
    _launch(device, call, pack(kind, act, parts - 1, 0, T, F, x.data_ptr(), ldx, out.data_ptr(), ldh, q, q + split))
    return out, ActivationCheckpoint(data, activation, gated, T, F, x.dtype)


def checkpoint_activation_backward(grad, kept: ActivationCheckpoint, *, out=None, stream=None) -> torch.Tensor:
    """Gradient of ``x`` for the gradient ``grad`` (T, F) of ``h``, from what ``checkpoint_activation`` kept: (T, 2F) or (T, F)
    in the type of ``x``.  ``out`` may be given.  Asynchronous on ``stream`` (None: torch's current stream)."""
    if out is None and stream is None and grad.is_cuda:
        dx = L.binding().act_backward(grad, kept)
        if dx is not None:
            return dx
    other = _other_stream(grad, stream)
    if other is not None:
        return _elsewhere(other, checkpoint_activation_backward, grad, kept, out=out)
    data, T, F, parts = kept.data, kept.rows, kept.width, 2 if kept.gated else 1
    kind, act, device = _IN_KINDS.get(kept.dtype), ACTIVATIONS.get(kept.activation), data.get_device()
    if kind is None or act is None or type(T) is not int or type(F) is not int or T < 0 or F < 1:
        raise ValueError(f"kept is no checkpoint: activation {kept.activation!r}, {T!r} rows of {F!r} values of {kept.dtype}")
    _check_array("kept.data", data, torch.int8, (kept._split() + 4 * T * parts * -(-F // BLOCK),), device)
    q = data.data_ptr()
    ldg = _given("grad", grad, kind, device, T, F)
    _no_gradient("checkpoint_activation_backward", grad)
    if out is None:
        out, ldx = grad.new_empty((T, parts * F)), parts * F
    else:
        ldx = _given("out", out, kind, device, T, parts * F)
        _check_place(out, grad, ldx, ldg)
    pack, call = L.direct("bsg_act_backward", L.ACT_LAYOUT)
    _launch(device, call, pack(kind, act, parts - 1, 0, T, F, grad.data_ptr(), ldg, out.data_ptr(), ldx,
                               q, q + kept._split()))
    return out


class _CheckpointedActivation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, activation, gated):
        h, kept = checkpoint_activation(x, activation, gated=gated)
        ctx.save_for_backward(kept.data)
        ctx.how = (activation, kept.gated, kept.rows, kept.width, kept.dtype)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        kept = ActivationCheckpoint(*ctx.saved_tensors, *ctx.how)
        grad = grad.resolve_neg()
        if grad.stride(1) != 1 or (grad.shape[0] > 1 and grad.stride(0) < grad.shape[1]):      # e.g. an expanded gradient
            grad = grad.contiguous()
        return checkpoint_activation_backward(grad, kept), None, None


def checkpointed_activation(x, activation: str = "silu", *, gated: bool = True) -> torch.Tensor:
    """``checkpoint_activation`` under autograd: only the 8-bit checkpoint is kept for the backward pass, not ``x``.  Runs on
    torch's current stream."""
    return _CheckpointedActivation.apply(x, activation, gated)
