"""Router in front of a layer of experts.

    r = route_tokens(logits, top_k)                       # logits (T, E)
    y = int8_linear(x, W, W_scale, offsets=r.offsets, rows=r.rows)      # (T * top_k, N), rows sorted by expert
    loss = task_loss + 0.01 * r.balance_loss

``r.offsets`` are the end rows that ``GroupedGemmArguments`` and ``int8_linear`` take.  ``r.weights`` and ``r.balance_loss``
carry gradients to the logits when those require them.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import lib as L
from .int8 import _OUT_KINDS as _KINDS
from .int8 import _check_array, _elsewhere, _launch, _matrix, _no_lazy_sign, _no_tangent, _other_stream

MAX_EXPERTS, MAX_TOP_K = 1024, 32


class Routing(NamedTuple):
    """What ``route_tokens`` returns.  A slot that chose nothing (a token that does not count, or fewer than k logits above
    -inf) has expert -1, weight 0 and position -1, which is no row: what is taken at positions has to be masked there (the rows of
    a grouped product behind the last end row are not written and may hold anything, also NaN).  Rows at or behind
    ``offsets[-1]`` name token -1.

    Without gradients the tensors are parts of one buffer: keeping any of them keeps the memory of all."""

    experts: torch.Tensor         # (T, k) int32, largest logit first
    weights: torch.Tensor         # (T, k) fp32
    counts: torch.Tensor          # (E,) int32: rows of every expert
    offsets: torch.Tensor         # (E,) int32: cumulative end rows
    rows: torch.Tensor            # (T * k,) int32: token of every row, rows sorted by expert, stable in (token, slot)
    positions: torch.Tensor       # (T, k) int32: row of every slot
    balance_loss: torch.Tensor    # () fp32
    num_tokens: torch.Tensor      # (1,) int32: tokens that count
    softmax: torch.Tensor         # (2 T,) bits of fp32, for the backward pass: largest logit, 1 / sum of exp(logit - largest)
    normalize: bool


def _scratch_words(T: int, E: int) -> int:      # what bsg_route_scratch_size says
    if T <= 512:
        return 0
    return ((min((T + 15) // 16, 740) + 3) & ~3) * (2 * E + 1) + E


def _check_logits(logits, top_k):
    kind, device, T, E, ld = _matrix("logits", logits, _KINDS)
    if E > MAX_EXPERTS:
        raise ValueError(f"between 1 and {MAX_EXPERTS} experts are supported, got {E}")
    if type(top_k) is not int or not 1 <= top_k <= min(MAX_TOP_K, E):
        raise ValueError(f"top_k must be an int between 1 and min({MAX_TOP_K}, {E}), got {top_k!r}")
    if T * top_k > 0x7FFFFFFF:
        raise ValueError(f"{T} tokens with {top_k} choices exceed 2^31 rows")
    return kind, device, T, E, ld


def _forward(logits, top_k, token_mask, normalize, stream) -> Routing:
    if stream is None and logits.is_cuda:
        r = L.binding().route_forward(logits, top_k, token_mask, bool(normalize))
        if r is not None:
            return r
    kind, device, T, E, ld = _check_logits(logits, top_k)
    if token_mask is not None:
        _check_array("token_mask", token_mask, torch.bool, (T,), device)
    normalize = bool(normalize)
    n = T * top_k
    # What carries no gradient comes from one allocation (int32: softmax, as bits, first, since it is read eight bytes at a time);
    # the two results that carry one are tensors of their own.
    whole = logits.new_empty(2 * T + 3 * n + 2 * E + 1, dtype=torch.int32)
    weights = logits.new_empty((T, top_k), dtype=torch.float32)
    loss = logits.new_empty((), dtype=torch.float32)
    soft = whole.data_ptr()
    w = soft + 8 * T
    pack, call = L.direct("bsg_route_forward", L.ROUTE_LAYOUT)
    args = pack(kind, E, top_k, normalize, T, logits.data_ptr(), ld, 0 if token_mask is None else token_mask.data_ptr(),
                w, weights.data_ptr(), w + 12 * n, w + 12 * n + 8 * E, soft, w + 12 * n + 4 * E, w + 4 * n, w + 8 * n, loss.data_ptr(), 0, 0, 0, 0)
    words = _scratch_words(T, E)
    if words:
        scratch = logits.new_empty(words, dtype=torch.int32)
        _launch(device, call, args, scratch.data_ptr(), 4 * words)
    else:
        _launch(device, call, args, 0, 0)
    softmax, experts, rows, positions, counts, offsets, live = whole.split_with_sizes((2 * T, n, n, n, E, E, 1))
    return Routing(experts.view(T, top_k), weights, counts, offsets, rows, positions.view(T, top_k), loss, live, softmax, normalize)


def route_tokens_backward(logits, routing: Routing, grad_weights=None, grad_balance_loss=None, *, stream=None) -> torch.Tensor:
    """Gradient of ``logits`` (in their type) for the gradients of ``routing.weights`` (T, k) fp32 and ``routing.balance_loss``
    () fp32, either of which may be None (zero).  The counts are constants.  Asynchronous on ``stream`` (None: torch's current
    stream)."""
    if stream is None and logits.is_cuda:
        d = L.binding().route_backward(logits, routing, grad_weights, grad_balance_loss)
        if d is not None:
            return d
    other = _other_stream(logits, stream)
    if other is not None:
        return _elsewhere(other, route_tokens_backward, logits, routing, grad_weights, grad_balance_loss)
    _no_tangent("route_tokens_backward", logits, routing.weights, grad_weights, grad_balance_loss)
    experts, counts = routing.experts, routing.counts
    if experts.dim() != 2:
        raise ValueError(f"routing.experts must be (tokens, k), got {tuple(experts.shape)}")
    k = experts.shape[1]
    kind, device, T, E, ld = _check_logits(logits, k)
    for name, dtype, shape in (("experts", torch.int32, (T, k)), ("weights", torch.float32, (T, k)), ("counts", torch.int32, (E,)),
                               ("num_tokens", torch.int32, (1,)), ("softmax", torch.int32, (2 * T,))):
        _check_array("routing." + name, getattr(routing, name), dtype, shape, device)
    if grad_weights is not None:
        _check_array("grad_weights", grad_weights, torch.float32, experts.shape, device)
    if grad_balance_loss is not None and (grad_balance_loss.dtype != torch.float32 or grad_balance_loss.numel() != 1
                                          or grad_balance_loss.get_device() != device):
        raise ValueError(f"grad_balance_loss must be a one-element fp32 tensor on CUDA device {device}")
    if grad_balance_loss is not None:
        _no_lazy_sign("grad_balance_loss", grad_balance_loss)
    out = logits.new_empty((T, E))
    pack, call = L.direct("bsg_route_backward", L.ROUTE_LAYOUT)
    args = pack(kind, E, k, routing.normalize, T, logits.data_ptr(), ld, 0, experts.data_ptr(), routing.weights.data_ptr(),
                counts.data_ptr(), routing.num_tokens.data_ptr(), routing.softmax.data_ptr(), 0, 0, 0, 0, 0 if grad_weights is None else grad_weights.data_ptr(),
                0 if grad_balance_loss is None else grad_balance_loss.data_ptr(), out.data_ptr(), E)
    _launch(device, call, args)
    return out


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, token_mask, normalize, stream):
        r = _forward(logits, top_k, token_mask, normalize, stream)
        ctx.save_for_backward(logits, r.experts, r.weights, r.counts, r.num_tokens, r.softmax)
        ctx.normalize = r.normalize
        whole = (r.experts, r.counts, r.offsets, r.rows, r.positions, r.num_tokens, r.softmax)
        ctx.mark_non_differentiable(*whole)
        ctx.set_materialize_grads(False)
        return (r.weights, r.balance_loss) + whole

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_weights, grad_loss, *_):
        logits, experts, weights, counts, live, softmax = ctx.saved_tensors
        if grad_weights is None and grad_loss is None:
            return None, None, None, None, None
        r = Routing(experts, weights, counts, None, None, None, None, live, softmax, ctx.normalize)
        grad = route_tokens_backward(logits, r, None if grad_weights is None else grad_weights.resolve_neg().contiguous(), None if grad_loss is None else grad_loss.resolve_neg())
        return grad, None, None, None, None


def route_tokens(logits, top_k: int, *, token_mask=None, normalize: bool = True, stream=None) -> Routing:
    """Choose ``top_k`` experts for every token of ``logits`` (T, E) bf16 / fp16 / fp32.

    The probabilities are ``softmax(logits)`` in fp32.  The k largest logits are chosen, ties to the lower index; -inf is never
    chosen (a masked expert), NaN ranks above all.  ``weights`` are the chosen probabilities, divided by their sum when
    ``normalize``.  ``token_mask`` (T,) bool: False marks padding, which is not routed and does not count; neither does a token
    whose logits are all -inf.  ``balance_loss = E * sum_e f_e P_e`` with f_e the share of the n * k choices that fell on expert
    e and P_e the mean probability over the n tokens that count: 1 when balanced, 0 when n = 0.

    E is at most 1024 and k at most 32.  Results do not depend on the order in which anything runs.  Asynchronous on ``stream``
    (None: torch's current stream); autograd runs the backward pass on the same one."""
    if stream is None and logits.is_cuda:      # (None for logits that want a gradient, too)
        r = L.binding().route_forward(logits, top_k, token_mask, normalize)
        if r is not None:
            return r
    other = _other_stream(logits, stream)
    if other is not None:
        return _elsewhere(other, route_tokens, logits, top_k, token_mask=token_mask, normalize=normalize)
    _no_tangent("route_tokens", logits)
    if not (torch.is_grad_enabled() and logits.requires_grad):
        return _forward(logits, top_k, token_mask, normalize, stream)
    weights, loss, experts, counts, offsets, rows, positions, live, softmax = _Route.apply(logits, top_k, token_mask, normalize, stream)
    return Routing(experts, weights, counts, offsets, rows, positions, loss, live, softmax, bool(normalize))
