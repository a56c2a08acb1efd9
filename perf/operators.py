"""Cases of the operators around an 8-bit expert (or plain) MLP layer: the integer product with scales per token and
channel, the router with its balance loss, and the activation that keeps its input in 8 bits for the backward pass.

``run`` computes a case in its plain form (elementary torch operations in 32 bits) or, where ``own`` is true, with the
library's calls; ``exact`` restates the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BLOCK = 128      # columns of a checkpointed row that share one scale


def listed():
    return [
        # one token of a sequence being generated: the weights are read once, everything else is latency
        dict(name="linear_decode_1", op="linear", tokens=1, inputs=4096, outputs=4096, dtype="bfloat16", out="bfloat16", bias=False),
        # a small batch of sequences being generated, wide projection with a bias
        dict(name="linear_batch_17", op="linear", tokens=17, inputs=4096, outputs=14336, dtype="bfloat16", out="bfloat16", bias=True),
        # a short prompt, no extent a multiple of anything
        dict(name="linear_ragged_777", op="linear", tokens=777, inputs=2050, outputs=5003, dtype="float16", out="float32", bias=True),
        # the library's headline problem size: a long prompt or a training step of a wide layer
        dict(name="linear_8192", op="linear", tokens=8192, inputs=8192, outputs=8192, dtype="bfloat16", out="bfloat16", bias=False),
        # a few tokens of generation through many experts: most experts see no row, some see one or two
        dict(name="experts_decode_16", op="experts", tokens=16, experts=64, top=2, inputs=2048, outputs=7168, skew=0.0, dtype="bfloat16"),
        # a prompt through the 64 experts of the grouped benchmark, unevenly loaded
        dict(name="experts_prompt_4096", op="experts", tokens=4096, experts=64, top=8, inputs=7168, outputs=2048, skew=1.0, dtype="bfloat16"),
        # the router of one generation step
        dict(name="route_decode_16", op="route", tokens=16, experts=64, top=2, dtype="bfloat16", normalize=True, padding=0.0, masked=0.0),
        # a padded batch with some experts switched off per token, logits in fp32, weights not normalised
        dict(name="route_padded_4099", op="route", tokens=4099, experts=160, top=6, dtype="float32", normalize=False, padding=0.2, masked=0.1),
        # the router of a training step over a long batch
        dict(name="route_train_65536", op="route", tokens=65536, experts=256, top=8, dtype="bfloat16", normalize=True, padding=0.0, masked=0.0),
        # a handful of rows: latency of the forward and the backward pass
        dict(name="activation_33", op="activation", tokens=33, width=4096, dtype="bfloat16", activation="silu", gated=True),
        # odd width, plain (not gated) gelu, fp16
        dict(name="activation_gelu_2051", op="activation", tokens=2051, width=5003, dtype="float16", activation="gelu", gated=False),
        # the MLP activation of a training step
        dict(name="activation_train_8192", op="activation", tokens=8192, width=14336, dtype="bfloat16", activation="silu", gated=True),
    ]


def draw(rng):
    def size(lo, hi):       # spread over the logarithm; half of them multiples of 16, the others as they fall
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(16, n // 16 * 16) if n >= 16 and rng.random() < 0.5 else max(lo, min(hi, n))

    op = rng.choice(["linear", "experts", "route", "activation"])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "linear":
        k, n = size(64, 16384), size(64, 16384)
        return dict(op=op, tokens=size(1, min(8192, 8192 ** 3 // (k * n))), inputs=k, outputs=n, dtype=dtype,
                    out=rng.choice([dtype, "float32"]), bias=rng.random() < 0.5)
    if op == "experts":
        e, k, n = size(2, 128), size(64, 7168), size(64, 7168)
        while e * k * n > 64 * 7168 * 2048:
            k, n = max(64, k // 2), max(64, n // 2)
        return dict(op=op, tokens=size(1, 4096), experts=e, top=rng.randint(1, min(8, e)), inputs=k, outputs=n,
                    skew=round(rng.uniform(0.0, 1.0), 3), dtype=dtype)
    if op == "route":
        e = size(4, 256)
        return dict(op=op, tokens=size(1, 65536), experts=e, top=rng.randint(1, min(8, e)), dtype=rng.choice([dtype, "float32"]),
                    normalize=rng.random() < 0.5, padding=round(rng.choice([0.0, rng.uniform(0.0, 0.5)]), 3),
                    masked=round(rng.choice([0.0, rng.uniform(0.0, 0.3)]), 3))
    return dict(op=op, tokens=size(1, 8192), width=size(16, 14336), dtype=dtype, activation=rng.choice(["silu", "gelu", "relu"]),
                gated=rng.random() < 0.7)


def _weights(gen, shape, inputs):
    """int8 weights with a scale per output channel; rows start on 16-byte boundaries, as the quantiser lays them out."""
    pitch = -(-inputs // 16) * 16
    buf = torch.empty(shape + (pitch,), dtype=torch.int8, device="cuda")
    buf.random_(-127, 128, generator=gen)
    scale = (0.5 + torch.rand(shape, device="cuda", generator=gen)) / (73.0 * math.sqrt(inputs))
    return buf[..., :inputs], scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    s = {"case": case}
    if op in ("linear", "experts"):
        t, k, n = case["tokens"], case["inputs"], case["outputs"]
        # activations: some channels are far larger than the others
        loud = 1.0 + 15.0 * (torch.rand(k, device="cuda", generator=gen) < 0.01)
        s["x"] = (normal(t, k) * loud).to(dtype)
        if op == "linear":
            s["w"], s["ws"] = _weights(gen, (n,), k)
            s["bias"] = normal(n) if case["bias"] else None
        else:
            e = case["experts"]
            s["w"], s["ws"] = _weights(gen, (e, n), k)
            liking = case["skew"] * normal(e)
            chosen = (normal(t, e) + liking).topk(case["top"], dim=1).indices.reshape(-1)
            order = chosen.sort(stable=True).indices
            counts = torch.zeros(e, dtype=torch.int64, device="cuda").scatter_add_(0, chosen, torch.ones_like(chosen))
            s["rows"] = (order // case["top"]).to(torch.int32)
            s["offsets"] = counts.cumsum(0).to(torch.int32)
            s["most"] = int(counts.max())
    elif op == "route":
        t, e = case["tokens"], case["experts"]
        s["logits"] = (2.0 * normal(t, e) + normal(e)).to(dtype)
        if case["masked"] > 0:
            s["logits"][torch.rand((t, e), device="cuda", generator=gen) < case["masked"]] = float("-inf")
        s["mask"] = torch.rand(t, device="cuda", generator=gen) >= case["padding"] if case["padding"] > 0 else None
        s["grad_weights"] = normal(t, case["top"])
        s["grad_loss"] = torch.full((), 0.01, device="cuda")
    else:
        t, f = case["tokens"], case["width"]
        s["x"] = (2.0 * normal(t, 2 * f if case["gated"] else f)).to(dtype)
        s["grad"] = normal(t, f).to(dtype)
    return s


# ---------------------------------------------------------------------------------------------- plain forms, 32 bits
def _eight_bits(x, dim=-1):
    """x (fp32) -> whole numbers of magnitude up to 127 and their scale, halves rounded away from zero."""
    amax = x.abs().amax(dim, keepdim=True)
    q = torch.sign(x) * torch.floor(127.0 * x.abs() / amax.clamp_min(torch.finfo(torch.float32).tiny) + 0.5)
    return q, amax / 127.0


def _plain_linear(s):
    q, sx = _eight_bits(s["x"].float())
    y = q @ s["w"].float().t() * sx * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(DTYPES[s["case"]["out"]])


def _plain_experts(s):
    q, sx = _eight_bits(s["x"].float())
    rows, ends = s["rows"].long(), s["offsets"].long()
    at = torch.arange(rows.numel(), device="cuda")
    e = torch.searchsorted(ends, at, right=True)
    place = at - (ends - torch.diff(ends, prepend=ends.new_zeros(1)))[e]
    a = torch.zeros((ends.numel(), s["most"], q.shape[1]), device="cuda")
    a[e, place] = q[rows]
    y = torch.bmm(a, s["w"].float().transpose(1, 2))[e, place]
    return (y * sx[rows] * s["ws"][e]).to(s["x"].dtype)


def _plain_route(s):
    case, logits = s["case"], s["logits"]
    (t, e), k = logits.shape, case["top"]
    ninf = float("-inf")
    l = logits.float()
    real = (l != ninf).any(1)
    if s["mask"] is not None:
        real = real & s["mask"]
    top = l.amax(1, keepdim=True)
    z = torch.exp(l - torch.where(top == ninf, torch.zeros_like(top), top))
    p = torch.where(real[:, None], z / z.sum(1, keepdim=True), torch.zeros_like(z))
    value, index = torch.sort(l, dim=1, descending=True, stable=True)
    index, live = index[:, :k], (value[:, :k] != ninf) & real[:, None]
    chosen = torch.where(live, p.gather(1, index), torch.zeros_like(p[:, :k]))
    total = chosen.sum(1, keepdim=True)
    weights = torch.where(live, chosen / total, chosen) if case["normalize"] else chosen
    flat = torch.where(live, index, torch.full_like(index, e)).reshape(-1)
    counts = torch.zeros(e + 1, dtype=torch.int64, device="cuda").scatter_add_(0, flat, torch.ones_like(flat))[:e]
    offsets = counts.cumsum(0)
    order = torch.sort(flat, stable=True).indices
    at = torch.arange(t * k, device="cuda")
    none = torch.full_like(at, -1)
    rows = torch.where(at < offsets[-1], order // k, none)
    positions = torch.where(live.reshape(-1), torch.empty_like(at).scatter_(0, order, at), none).reshape(t, k)
    n = real.sum().clamp_min(1).float()
    f = counts.float() / (n * k)
    loss = e * (f * (p.sum(0) / n)).sum()
    # gradients of the logits, given those of the weights and of the loss
    gw = torch.where(live, s["grad_weights"], torch.zeros_like(chosen))
    d = s["grad_loss"] * (e / n) * p * (f - (p * f).sum(1, keepdim=True))
    if case["normalize"]:
        part = weights * (gw - (weights * gw).sum(1, keepdim=True))
    else:
        part = chosen * gw
        d = d - p * part.sum(1, keepdim=True)
    d = d.scatter_add(1, index, part)
    whole = [torch.where(live, index, torch.full_like(index, -1)), counts, offsets, rows, positions]
    return [weights, loss, d.to(logits.dtype)] + [v.to(torch.int32) for v in whole]


def _blocks(x):
    """(rows, width) -> the values that the 8-bit blocks of 128 columns stand for."""
    width = x.shape[1]
    padded = torch.nn.functional.pad(x, (0, -width % BLOCK)).reshape(x.shape[0], -1, BLOCK)
    q, scale = _eight_bits(padded)
    return (q * scale).reshape(x.shape[0], -1)[:, :width]


def _value_and_slope(x, name):
    if name == "relu":
        return x.clamp_min(0.0), (x > 0).float()
    if name == "silu":
        g = 1.0 / (1.0 + torch.exp(-x))
        return x * g, g * (1.0 + x * (1.0 - g))
    phi = 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5)))
    return x * phi, phi + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_activation(s):
    case, width = s["case"], s["grad"].shape[1]
    x, dy = s["x"].float(), s["grad"].float()
    h = _value_and_slope(x[:, :width], case["activation"])[0]
    value, slope = _value_and_slope(_blocks(x[:, :width]), case["activation"])
    if case["gated"]:
        h = h * x[:, width:]
        dx = torch.cat([dy * _blocks(x[:, width:]) * slope, dy * value], 1)
    else:
        dx = dy * slope
    return [h.to(s["x"].dtype), dx.to(s["x"].dtype)]


# ---------------------------------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        import cutlass_b200 as ops
        if op == "linear":
            return ops.int8_linear(s["x"], s["w"], s["ws"], s["bias"], out_dtype=DTYPES[case["out"]])
        if op == "experts":
            return ops.int8_linear(s["x"], s["w"], s["ws"], offsets=s["offsets"], rows=s["rows"])
        if op == "route":
            r = ops.route_tokens(s["logits"], case["top"], token_mask=s["mask"], normalize=case["normalize"])
            d = ops.route_tokens_backward(s["logits"], r, s["grad_weights"], s["grad_loss"])
            return [r.weights, r.balance_loss, d, r.experts, r.counts, r.offsets, r.rows, r.positions]
        h, saved = ops.checkpoint_activation(s["x"], case["activation"], gated=case["gated"])
        return [h, ops.checkpoint_activation_backward(s["grad"], saved)]
    return {"linear": _plain_linear, "experts": _plain_experts, "route": _plain_route, "activation": _plain_activation}[op](s)


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "float32" else 2
    if op in ("linear", "experts"):
        t, k, n = case["tokens"], case["inputs"], case["outputs"]
        if op == "linear":
            out = 4 if case["out"] == "float32" else 2
            return {"bytes": n * k + 4 * n * (2 if case["bias"] else 1) + t * k * size + t * n * out, "flops": 2 * t * n * k}
        e, r = case["experts"], t * case["top"]
        met = e * (1.0 - (1.0 - case["top"] / e) ** t)        # experts that a token is expected to reach
        return {"bytes": met * n * (k + 4) + t * k * size + 4 * r + r * n * size, "flops": 2 * r * n * k}
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["top"]
        # logits in, their gradient out; experts, weights, rows, positions out; gradients of the weights in
        return {"bytes": 2 * t * e * size + 20 * t * k + 8 * e, "flops": 12 * t * e}
    t, f, parts = case["tokens"], case["width"], 2 if case["gated"] else 1
    kept = parts * t * (f + 4 * -(-f // BLOCK))
    # the input in, the result out, the checkpoint out and in again, the gradient in, the input's gradient out
    return {"bytes": 2 * parts * t * f * size + 2 * t * f * size + 2 * kept, "flops": 30 * t * f}


# ------------------------------------------------------------------------------------------- definitions, 64 bits
def _to_levels(v):
    """v -> (levels, step): the nearest of 255 evenly spaced levels, halves outwards; one step size per row of the last axis."""
    v = v.double()
    peak = v.abs().max(dim=-1, keepdim=True).values
    ratio = torch.where(peak > 0, v.abs() * 127.0 / peak, torch.zeros_like(v))
    return torch.copysign((ratio + 0.5).floor(), v), peak / 127.0


def _exact_product(s):
    case = s["case"]
    if case["op"] == "linear":
        levels, step = _to_levels(s["x"])
        y = torch.einsum("tk,nk->tn", levels, s["w"].double()) * step * s["ws"].double()
        return y if s["bias"] is None else y + s["bias"].double()
    y = torch.zeros((s["rows"].numel(), case["outputs"]), dtype=torch.float64, device="cuda")
    levels, step = _to_levels(s["x"])
    begin = 0
    for e, end in enumerate(s["offsets"].tolist()):
        if end > begin:
            who = s["rows"][begin:end].long()
            y[begin:end] = (levels[who] * step[who]) @ (s["w"][e].double() * s["ws"][e].double()[:, None]).t()
        begin = end
    return y


def _exact_route(s):
    case, (t, e), k = s["case"], s["logits"].shape, s["case"]["top"]
    l = s["logits"].double()
    counted = ~torch.isneginf(l).all(1) & (s["mask"] if s["mask"] is not None else torch.ones(t, dtype=torch.bool, device="cuda"))
    p = torch.zeros_like(l)
    p[counted] = torch.softmax(l[counted], 1)
    # a larger logit wins; between equal ones the lower index: rank = number of experts that come first
    picks, left = torch.full((t, k), -1, dtype=torch.int64, device="cuda"), l.clone()
    left[~counted] = float("-inf")
    for j in range(k):
        best = left.max(1, keepdim=True).values
        first = (left == best).to(torch.int8).argmax(1)
        ok = ~torch.isneginf(best[:, 0])
        picks[ok, j] = first[ok]
        left[torch.arange(t, device="cuda"), first] = float("-inf")
    live = picks >= 0
    onehot = torch.zeros((t, e + 1), dtype=torch.float64, device="cuda").scatter_(1, torch.where(live, picks, e), 1.0)[:, :e]
    counts = onehot.sum(0).to(torch.int64)
    ends = counts.cumsum(0)
    # rank of a (token, expert) pair among the tokens of that expert
    before = onehot.cumsum(0) - onehot
    base = (ends - counts).double() + before
    positions = torch.where(live, base.gather(1, picks.clamp_min(0)).long(), -1)
    rows = torch.full((t * k,), -1, dtype=torch.int64, device="cuda")
    token = torch.arange(t, device="cuda")[:, None].expand(t, k)
    rows[positions[live]] = token[live]
    n = max(int(counted.sum()), 1)
    w = p.gather(1, picks.clamp_min(0)) * live
    scale = w.sum(1, keepdim=True).clamp_min(1e-300) if case["normalize"] else 1.0
    share = counts.double() / (n * k)
    loss = e * torch.dot(share, p.mean(0) * (t / n))
    gw = torch.zeros((t, e), dtype=torch.float64, device="cuda")
    gw.scatter_add_(1, picks.clamp_min(0), s["grad_weights"].double() * live)
    # through the softmax: dl = p (g - <p, g>), g the gradient of the probabilities
    g = s["grad_loss"].double() * (e / n) * share.expand(t, e)
    if case["normalize"]:
        mean = (gw * onehot * p).sum(1, keepdim=True) / scale
        g = g + onehot * (gw - mean) / scale
    else:
        g = g + gw
    d = p * (g - (p * g).sum(1, keepdim=True))
    return [w / scale, loss, d, None, None, None, None, None] if t * e > 1 << 24 else [w / scale, loss, d, picks, counts, ends, rows, positions]


def _exact_activation(s):
    case, f = s["case"], s["grad"].shape[1]
    x, dy = s["x"].double(), s["grad"].double()

    def kept(v):
        parts = [v[:, i:i + BLOCK] for i in range(0, f, BLOCK)]
        return torch.cat([torch.mul(*_to_levels(b)) for b in parts], 1)

    def act(v):
        if case["activation"] == "relu":
            return torch.where(v > 0, v, torch.zeros_like(v)), torch.where(v > 0, 1.0, 0.0).double()
        if case["activation"] == "silu":
            g = torch.sigmoid(v)
            return v * g, g + v * g * (1.0 - g)
        return 0.5 * v * torch.erfc(-v / math.sqrt(2.0)), 0.5 * torch.erfc(-v / math.sqrt(2.0)) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)

    a, up = act(x[:, :f])[0], x[:, f:]
    ka, slope = act(kept(x[:, :f]))
    if not case["gated"]:
        return [a, dy * slope]
    return [a * up, torch.cat([dy * kept(up) * slope, dy * ka], 1)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("linear", "experts"):
        return _exact_product(s)
    return _exact_route(s) if case["op"] == "route" else _exact_activation(s)
