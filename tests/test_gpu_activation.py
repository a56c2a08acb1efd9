"""The activation with an 8-bit checkpoint on the GPU against its definition in 64 bits."""
import math
from types import SimpleNamespace

import pytest
import torch

import cutlass_b200 as ops

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def kept64(x):
    """(whole numbers, scales per block, values) of the 128-column blocks of every row."""
    x = x.double()
    T, F = x.shape
    b = torch.nn.functional.pad(x, (0, -F % 128)).reshape(T, -1, 128)
    amax = b.abs().amax(2, keepdim=True)
    bad = ~torch.isfinite(amax)
    safe = torch.where(bad | (amax == 0), torch.ones_like(amax), amax)
    q = torch.where(bad | (amax == 0), torch.zeros_like(b), torch.sign(b) * torch.floor(127.0 * b.abs() / safe + 0.5))
    s = torch.where(bad, torch.full_like(amax, math.nan), amax / 127.0)
    return q.reshape(T, -1)[:, :F], s[..., 0], (q * s).reshape(T, -1)[:, :F]


def act64(x, name):
    """value and slope"""
    if name == "identity":
        return x, torch.ones_like(x)
    if name == "relu":
        return torch.where(x > 0, x, torch.where(x != x, x, 0.0)), torch.where(x != x, x, (x > 0).double())
    if name == "silu":
        s = torch.sigmoid(x)
        return x * s, s * (1 + x * (1 - s))
    phi = 0.5 * torch.erfc(-x / math.sqrt(2.0))
    return x * phi, phi + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


def make(T, F, dtype, gated, seed, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cols = 2 * F if gated else F
    buf = torch.zeros((T, cols + pad), dtype=dtype, device="cuda")
    buf[:, :cols] = (3 * torch.randn((T, cols), device="cuda", generator=g)).to(dtype)
    dbuf = torch.zeros((T, F + pad), dtype=dtype, device="cuda")
    dbuf[:, :F] = torch.randn((T, F), device="cuda", generator=g).to(dtype)
    return buf[:, :cols], dbuf[:, :F]


def close(got, want, inner):
    """Half a step of the output type on top of ``inner``, the error before the rounding (and half the smallest step)."""
    info = torch.finfo(got.dtype)
    tol = inner + info.eps / 2 * (want.abs() + inner) + info.smallest_normal * info.eps
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got.double()), nan)
    err = torch.where(nan, torch.zeros_like(tol), (got.double() - want).abs() - tol)
    assert float(err.max()) <= 0, f"{int((err > 0).sum())} of {err.numel()} values off, worst by {float(err.max())}"


def check(x, dh, activation, gated, h, dx, kept):
    """Errors before the last rounding.  The fast exponential is off by 2 + 1.16 |x| units of 2^-24 (|x| < 45 here: under
    2^-18.2), its effect on a sigmoid s is s (1 - s) times that and, with the quotient (2 units) and products, a value is off by
    less than 2^-17 of |x| + 1 and a slope by less than 2^-17 (1 + |x|); scales carry half a unit (2^-24)."""
    F = dh.shape[1]
    parts = [x[:, :F], x[:, F:]] if gated else [x]
    vals = []
    for i, part in enumerate(parts):
        q, s, v = kept64(part)
        assert torch.equal(kept.quantized[:, i, :F].double(), q)
        assert torch.equal(torch.nan_to_num(kept.scale[:, i], 5.0), torch.nan_to_num(s.float(), 5.0))
        vals.append(v)
    e = 2.0 ** -17
    a, _ = act64(x[:, :F].double(), activation)
    u = x[:, F:].double() if gated else torch.ones_like(a)
    close(h, a * u, e * (x[:, :F].double().abs() + 1) * u.abs() * (activation not in ("identity", "relu")) + 2.0 ** -23 * (a * u).abs())
    v, slope = act64(vals[0], activation)
    d = dh.double()
    ub = vals[1] if gated else torch.ones_like(v)
    fuzz = e * (1 + vals[0].abs()) * (activation not in ("identity", "relu"))
    close(dx[:, :F], d * ub * slope, (fuzz + 2.0 ** -22 * slope.abs()) * (d * ub).abs())
    if gated:
        close(dx[:, F:], d * v, (fuzz + 2.0 ** -22 * v.abs()) * d.abs())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("activation", ["silu", "gelu", "relu", "identity"])
@pytest.mark.parametrize("T,F,pad", [(1, 1, 0), (1, 128, 0), (3, 127, 0), (5, 136, 0), (2, 1000, 8), (17, 515, 3), (4, 4096, 0), (33, 264, 1)])
def test_forward_and_backward(cuda_lib, T, F, pad, activation, gated, dtype):
    x, dh = make(T, F, dtype, gated, seed=T * 7 + F, pad=pad)
    h, kept = ops.checkpoint_activation(x, activation, gated=gated)
    dx = ops.checkpoint_activation_backward(dh, kept)
    check(x, dh, activation, gated, h, dx, kept)


@pytest.mark.parametrize("activation", ["silu", "gelu", "relu"])
def test_extreme_blocks(cuda_lib, activation):
    """Zeros, the type's largest and smallest values, a NaN and infinities: they stay in their block of 128."""
    T, F = 6, 300
    x, dh = make(T, F, BF16, True, seed=1)
    x = x.clone()
    x[0] = 0
    x[1, 130], x[2, 5], x[2, 290], x[3, 310] = math.nan, math.inf, 2.0 ** -120, -math.inf
    x[4, :128] = 2.0 ** -133
    x[5, 0], x[5, 299] = 40.0, -40.0
    h, kept = ops.checkpoint_activation(x, activation)
    dx = ops.checkpoint_activation_backward(dh, kept)
    finite = torch.isfinite(x).all(1)
    only = SimpleNamespace(quantized=kept.quantized[finite], scale=kept.scale[finite])
    check(x[finite], dh[finite], activation, True, h[finite], dx[finite], only)
    bad = ~torch.isfinite(dx)
    want = torch.zeros_like(bad)
    for r, lo, hi, part in ((1, 128, 256, 0), (2, 0, 128, 0), (3, 0, 128, 1)):
        if part == 0:
            want[r, lo:hi] = want[r, F + lo:F + hi] = True
        else:
            want[r, lo:hi] = True
    assert torch.equal(bad, want)
    ok = torch.isfinite(h)
    assert not bool(ok[1, 130]) and not bool(ok[3, 10]) and int((~ok).sum()) <= 3


def test_outputs_given_as_views_are_all_that_is_written(cuda_lib):
    T, F = 9, 77
    x, dh = make(T, F, F16, True, seed=2)
    hb, xb = torch.full((T, F + 5), 7.0, dtype=F16, device="cuda"), torch.full((T, 2 * F + 5), 7.0, dtype=F16, device="cuda")
    h, kept = ops.checkpoint_activation(x, "gelu", out=hb[:, 2:2 + F])
    dx = ops.checkpoint_activation_backward(dh, kept, out=xb[:, 3:3 + 2 * F])
    check(x, dh, "gelu", True, h, dx, kept)
    assert bool((hb[:, :2] == 7).all()) and bool((hb[:, 2 + F:] == 7).all()) and bool((xb[:, :3] == 7).all()) and bool((xb[:, 3 + 2 * F:] == 7).all())


@pytest.mark.parametrize("gated", [True, False])
def test_autograd_and_differences(cuda_lib, gated):
    """Under autograd the gradient is the functional one; and it is the slope of h up to what 8 bits lose: with |x - x^| <= s / 2
    per value, silu'' <= 1/2, |silu'| <= 1.1 and |act(g) - act(g^)| <= 1.1 s / 2 bound the difference to the slope in 64 bits."""
    T, F = 7, 200
    x, dh = make(T, F, BF16, gated, seed=4)
    leaf = x.clone().requires_grad_()
    h = ops.checkpointed_activation(leaf, "silu", gated=gated)
    h.backward(dh)
    want, kept = ops.checkpoint_activation(x, "silu", gated=gated)
    assert torch.equal(h.detach(), want) and torch.equal(leaf.grad, ops.checkpoint_activation_backward(dh, kept))
    # central differences of the definition, in 64 bits
    eps, x64, d = 1e-5, x.double(), dh.double()
    f = lambda v: act64(v[:, :F], "silu")[0] * (v[:, F:] if gated else 1.0)  # noqa: E731
    num = torch.zeros_like(x64)
    lo, hi = x64.clone(), x64.clone()
    lo[:, :F] -= eps
    hi[:, :F] += eps
    num[:, :F] = d * (f(hi) - f(lo)) / (2 * eps)
    half = kept.scale.double().repeat_interleave(128, dim=2)[..., :F] / 2
    g, u = x64[:, :F], x64[:, F:] if gated else torch.ones_like(x64)
    bound = d.abs() * (0.5 * half[:, 0] * u.abs() + (1.1 * half[:, 1] + 0.25 * half[:, 0] * half[:, 1] if gated else 0.0))
    if gated:
        lo, hi = x64.clone(), x64.clone()
        lo[:, F:] -= eps
        hi[:, F:] += eps
        num[:, F:] = d * (f(hi) - f(lo)) / (2 * eps)
        bound = torch.cat([bound, d.abs() * 1.1 * half[:, 0]], 1)
    err = (leaf.grad.double() - num).abs()
    assert bool((err <= bound * 1.001 + 2.0 ** -8 * num.abs() + 2.0 ** -8 * bound + 1e-6).all())
    leaf.grad = None
    ops.checkpointed_activation(leaf, "silu", gated=gated).sum().backward()      # an expanded gradient
    assert torch.equal(leaf.grad, ops.checkpoint_activation_backward(torch.ones_like(dh), kept))


def test_streams_and_graphs(cuda_lib):
    x, dh = make(40, 500, BF16, True, seed=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    h, kept = ops.checkpoint_activation(x, stream=side)
    dx = ops.checkpoint_activation_backward(dh, kept, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    check(x, dh, "silu", True, h, dx, kept)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h, kept = ops.checkpoint_activation(x)
        dx = ops.checkpoint_activation_backward(dh, kept)
    for seed in (9, 10):
        nx, nd = make(40, 500, BF16, True, seed=seed)
        x.copy_(nx)
        dh.copy_(nd)
        g.replay()
        check(x, dh, "silu", True, h, dx, kept)


def test_empty(cuda_lib):
    h, kept = ops.checkpoint_activation(torch.empty((0, 32), dtype=BF16, device="cuda"))
    assert h.shape == (0, 16)
    assert ops.checkpoint_activation_backward(torch.empty((0, 16), dtype=BF16, device="cuda"), kept).shape == (0, 32)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_the_tail_of_gelu_keeps_its_relative_precision(cuda_lib, dtype):
    """Every value of the type between 2^-6 and 13 in magnitude, a block of 128 of each.  With y = |x| the lower tail P(-y) is
    exp(-y^2 / 2) times a polynomial of t = 1 / (1 + c y): off by 2^-17 (the fit, 5.3e-6), by y^2 / 2 times 2.5 * 2^-24 (argument of
    the exponential: the square, its product with log2 e, that constant) and by 48 * 2^-24 for the rest (exponential 4, the
    reciprocal 2, seven steps of the polynomial whose terms add up to twice its value, two products).  gelu(x) = x P(x) takes two
    roundings more, its slope P(x) + x p(x) those of p as well; the kept value is off by the roundings of its scale and of
    their product, 2 * 2^-24 of it, which its function passes on by its slope.  Last half a step of the type."""
    bits = torch.arange(1, 1 << 15, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    pos = bits[(bits >= 2.0 ** -6) & (bits <= 13)]
    v = torch.cat([-pos, pos])
    x = v[:, None].expand(-1, 128).contiguous()
    z = v.double()
    y = z.abs()
    tail, p = 0.5 * torch.erfc(y / math.sqrt(2)), torch.exp(-y * y / 2) / math.sqrt(2 * math.pi)
    exponent = y * y / 2 * 2.5 * 2.0 ** -24
    off = 2.0 ** -17 + exponent + 48 * 2.0 ** -24
    one = torch.ones_like(x)

    def near(got, want, inner):
        info = torch.finfo(dtype)
        tol = inner + info.eps / 2 * (want.abs() + inner) + info.smallest_normal * info.eps
        err = (got.double() - want[:, None]).abs() - tol[:, None]
        worst = int(err.amax(1).argmax())
        assert float(err.max()) <= 0, f"at {float(v[worst])}: {float(got[worst, 0])} instead of {float(want[worst])}"

    value, slope = act64(z, "gelu")
    value_off = y * tail * off + 2.0 ** -22 * value.abs()
    h, kept = ops.checkpoint_activation(x, "gelu", gated=False)
    near(h, value, value_off)
    kept_off = 2.0 ** -23 * y
    slope_off = tail * off + y * p * (exponent + 8 * 2.0 ** -24) + 2.0 ** -22 * (tail + y * p) + 2.0 ** -23 * (z > 0) + p * (2 - y * y).abs() * kept_off
    near(ops.checkpoint_activation_backward(one, kept), slope, slope_off)
    h, kept = ops.checkpoint_activation(torch.cat([x, one], 1), "gelu")
    near(h, value, value_off)
    dx = ops.checkpoint_activation_backward(one, kept)
    near(dx[:, :128], slope, slope_off + 2.0 ** -22 * slope.abs())
    near(dx[:, 128:], value, value_off + (tail + y * p) * kept_off * (z < 0) + 1.13 * kept_off * (z > 0))


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("T,F,pad", [(1, 300, 0), (40, 1024, 0), (33, 515, 3), (600, 136, 8)])
def test_results_in_the_place_of_the_input(cuda_lib, T, F, pad, gated):
    """h over the first columns of x and the gradient of x over that of h, value on value; any other overlap is refused."""
    x, dh = make(T, F, BF16, gated, seed=1, pad=pad)
    h, kept = ops.checkpoint_activation(x, "gelu", gated=gated)
    dx = ops.checkpoint_activation_backward(dh, kept)
    buf = x.new_zeros((T, 2 * F + pad + 1))
    cols = x.shape[1]
    buf[:, :cols] = x
    _, again = ops.checkpoint_activation(buf[:, :cols], "gelu", gated=gated, out=buf[:, :F])
    assert torch.equal(buf[:, :F], h) and torch.equal(again.scale, kept.scale) and torch.equal(again.quantized[..., :F], kept.quantized[..., :F])
    buf[:, :F] = dh
    ops.checkpoint_activation_backward(buf[:, :F], kept, out=buf[:, :cols])
    assert torch.equal(buf[:, :cols], dx)
    with pytest.raises(ValueError):
        ops.checkpoint_activation(buf[:, :cols], "gelu", gated=gated, out=buf[:, 1:1 + F])
    with pytest.raises(ValueError):
        ops.checkpoint_activation_backward(buf[:, 1:1 + F], kept, out=buf[:, :cols])
    wide = x.new_zeros((T, cols + F))
    wide[:, :cols] = x
    assert torch.equal(ops.checkpoint_activation(wide[:, :cols], "gelu", gated=gated, out=wide[:, cols:])[0], h)      # columns side by side
