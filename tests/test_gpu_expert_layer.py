"""Router, 8-bit products and the activation with an 8-bit checkpoint together: a layer of experts, forward and backward; and
tensors of more than 2^31 elements."""
import pytest
import torch

import cutlass_b200 as ops
import test_gpu_activation as activation_tests
import test_gpu_int8 as product_tests
import test_gpu_routing as routing_tests

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Layer:
    """Tokens of D columns, E experts with F hidden columns, k of them per token."""

    def __init__(self, T, D, F, E, k, dtype, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.k, self.x = k, torch.randn((T, D), device="cuda", generator=g).to(dtype)
        self.mask = torch.rand(T, device="cuda", generator=g) >= 0.2
        self.logits = (2 * torch.randn((T, E), device="cuda", generator=g)).to(dtype)
        self.logits[:, E // 2] = -float("inf")           # an expert that nobody may choose
        made = [ops.quantize_int8(torch.randn((E * n, c), device="cuda", generator=g).to(dtype)) for n, c in ((2 * F, D), (D, F))]
        (self.w1, self.s1), (self.w2, self.s2) = [(W.quantized.tensor.unflatten(0, (E, -1)), W.scale.tensor.view(E, -1)) for W in made]
        self.up = torch.zeros((T * k, 2 * F), dtype=dtype, device="cuda")      # rows behind the last end row stay zero
        self.down = torch.zeros((T * k, D), dtype=dtype, device="cuda")
        self.grad = torch.randn((T, D), device="cuda", generator=g)
        self.grad_h = torch.randn((T * k, F), device="cuda", generator=g).to(dtype)

    def run(self):
        """Everything on the way, and the gradients of the logits and of the first product's result."""
        logits = self.logits.detach().requires_grad_(True)
        r = ops.route_tokens(logits, self.k, token_mask=self.mask)
        up = ops.int8_linear(self.x, self.w1, self.s1, offsets=r.offsets, rows=r.rows, out=self.up).detach().requires_grad_(True)
        h = ops.checkpointed_activation(up, "silu")
        down = ops.int8_linear(h.detach(), self.w2, self.s2, offsets=r.offsets, out=self.down)
        mine = down[r.positions.clamp_min(0).long()].float() * (r.positions >= 0)[..., None]      # (T, k, D)
        y = (r.weights[..., None] * mine).sum(1)
        ((y * self.grad).sum() + 0.01 * r.balance_loss).backward()
        h.backward(self.grad_h)
        return r, up, h, down, y, logits.grad, up.grad, (mine * self.grad[:, None]).sum(2)

    def check(self, result):
        r, up, h, down, y, d_logits, d_up, d_weights = [t.detach() if torch.is_tensor(t) else t for t in result]
        want = routing_tests.check(self.logits, self.k, self.mask, True, type(r)(*[t.detach() if torch.is_tensor(t) else t for t in r]))
        total, begin = int(r.offsets[-1]), 0
        assert total == int(self.mask.sum()) * self.k
        for e, end in enumerate(r.offsets.tolist()):
            if end > begin:
                token = r.rows[begin:end].long()
                product_tests.check(up[begin:end], self.x[token], self.w1[e], self.s1[e])
                product_tests.check(down[begin:end], h[begin:end], self.w2[e], self.s2[e])
                begin = end
        assert bool((up[total:] == 0).all()) and bool((down[total:] == 0).all())
        kept = ops.checkpoint_activation(up, "silu")[1]
        activation_tests.check(up, self.grad_h, "silu", True, h, d_up, kept)
        # the weighted sum is torch's, in fp32: k products and k - 1 sums
        parts = r.weights.double()[..., None] * down.double()[r.positions.clamp_min(0).long()] * (r.positions >= 0)[..., None]
        assert bool(((y.double() - parts.sum(1)).abs() <= (self.k + 1) * 2.0 ** -24 * parts.abs().sum(1)).all())
        routing_tests.check_grad(d_logits, want, self.k, True, d_weights, 0.01, self.logits.dtype)


@pytest.mark.parametrize("T,D,F,E,k,dtype", [(1, 64, 32, 4, 1, BF16), (16, 200, 136, 8, 2, F16), (77, 256, 130, 5, 4, BF16), (300, 136, 264, 16, 2, BF16)])
def test_a_layer_forward_and_backward(cuda_lib, T, D, F, E, k, dtype):
    layer = Layer(T, D, F, E, k, dtype, seed=T)
    layer.mask[0] = True
    layer.check(layer.run())
    product_tests.status_ok()


def test_a_layer_whose_tokens_are_all_padding(cuda_lib):
    layer = Layer(40, 64, 32, 4, 2, BF16, seed=1)
    layer.mask.zero_()
    r, up, h, down, y, d_logits, d_up, _ = layer.run()
    assert int(r.offsets[-1]) == 0 and bool((r.rows == -1).all()) and float(r.balance_loss.detach()) == 0.0
    for t in (up, h, down, y, d_logits, d_up):
        assert not bool(t.detach().any())


def test_a_captured_layer_follows_its_inputs(cuda_lib):
    """Forward and backward in one graph; replays with other tokens, logits and masks, on the stream of the replay."""
    layer, other = Layer(50, 128, 72, 8, 2, BF16, seed=3), Layer(50, 128, 72, 8, 2, BF16, seed=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = layer.run()
    for source in (other, Layer(50, 128, 72, 8, 2, BF16, seed=5)):
        for name in ("x", "mask", "logits", "grad", "grad_h"):
            getattr(layer, name).copy_(getattr(source, name))
        layer.up.zero_()
        layer.down.zero_()
        graph.replay()
        layer.check(result)


# ------------------------------------------------------------------------------------------------ more than 2^31 elements
def test_a_product_with_more_outputs_than_31_bits(cuda_lib):
    M, N, K = 66000, 33000, 32
    x = product_tests.tokens(M, K, BF16, seed=1)
    w, ws = product_tests.weights((N,), K, seed=2)
    y = ops.int8_linear(x, w, ws)
    for part in (slice(0, 300), slice(31000, 31300), slice(M - 300, M)):
        product_tests.check(y[part], x[part], w, ws)


def test_tokens_with_more_values_than_31_bits(cuda_lib):
    M, N, K = 70000, 24, 32768
    x = torch.zeros((M, K), dtype=F16, device="cuda")
    x[-200:] = product_tests.tokens(200, K, F16, seed=3)
    x[:200] = x[-200:].flip(0)
    w, ws = product_tests.weights((N,), K, seed=4)
    y = ops.int8_linear(x, w, ws)
    assert not bool(y[200:-200].any())
    product_tests.check(y[-200:], x[-200:], w, ws)
    product_tests.check(y[:200], x[:200], w, ws)
    rows = torch.arange(M - 1, M - 201, -1, dtype=torch.int32, device="cuda")
    assert torch.equal(ops.int8_linear(x, w[None], ws[None], offsets=torch.tensor([200], dtype=torch.int32, device="cuda"), rows=rows), y[-200:].flip(0))


def test_experts_with_more_weights_than_31_bits(cuda_lib):
    E, N, K = 136, 4096, 4096
    w = torch.zeros((E, N, K), dtype=torch.int8, device="cuda")
    last, ws = product_tests.weights((N,), K, seed=5)
    w[-1], w[0] = last, last
    x = product_tests.tokens(9, K, BF16, seed=6)
    offsets = torch.full((E,), 4, dtype=torch.int32, device="cuda")
    offsets[-1] = 9
    y = ops.int8_linear(x, w, ws.expand(E, N).contiguous(), offsets=offsets)
    product_tests.check(y, x, last, ws)


@pytest.mark.parametrize("gated", [True, False])
def test_an_activation_of_more_values_than_31_bits(cuda_lib, gated):
    T, F = 140000, 16000 if not gated else 8000
    x = torch.zeros((T, 16000), dtype=BF16, device="cuda")
    some, dh_some = activation_tests.make(300, F, BF16, gated, seed=7)
    dh = torch.zeros((T, F), dtype=BF16, device="cuda")
    x[-300:], dh[-300:] = some, dh_some
    h, kept = ops.checkpoint_activation(x, "silu", gated=gated)
    dx = ops.checkpoint_activation_backward(dh, kept)
    assert not bool(h[:-300].any()) and not bool(dx[:-300].any())

    class Last:
        quantized, scale = kept.quantized[-300:], kept.scale[-300:]
    activation_tests.check(some, dh_some, "silu", gated, h[-300:], dx[-300:], Last)


def test_logits_of_more_values_than_31_bits(cuda_lib):
    """All tokens but the last 300 are padding, so the definition is that of the last ones, with their numbers shifted."""
    T, E, k, n = 2_200_000, 1024, 4, 300
    logits = torch.zeros((T, E), dtype=BF16, device="cuda")
    logits[-n:], _ = routing_tests.make(n, E, BF16, seed=8)
    mask = torch.zeros(T, dtype=torch.bool, device="cuda")
    mask[-n:] = True
    r = ops.route_tokens(logits, k, token_mask=mask)
    assert bool((r.experts[:-n] == -1).all()) and not bool(r.weights[:-n].any()) and bool((r.positions[:-n] == -1).all()) and bool((r.rows[n * k:] == -1).all())
    part = r._replace(experts=r.experts[-n:], weights=r.weights[-n:], positions=r.positions[-n:], rows=r.rows[:n * k] - (T - n))
    want = routing_tests.check(logits[-n:], k, None, True, part)
    gw, gl = torch.zeros((T, k), device="cuda"), torch.tensor(0.3, device="cuda")
    gw[-n:] = torch.randn((n, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    d = ops.route_tokens_backward(logits, r, gw, gl)
    assert not bool(d[:-n].any())
    routing_tests.check_grad(d[-n:], want, k, True, gw[-n:], 0.3, BF16)


# --------------------------------------------------------------------------------------------------- refusals of CUDA tensors
def test_refusals(cuda_lib):
    x = torch.zeros((6, 40), dtype=BF16, device="cuda")
    w, ws = product_tests.weights((24,), 40, seed=1)
    end = torch.tensor([3, 6], dtype=torch.int32, device="cuda")
    w2, ws2 = product_tests.weights((2, 24), 40, seed=1)
    linear = [
        dict(x=x.t()), dict(x=x[0]), dict(x=x.float()), dict(x=x[:1].expand(6, 40)), dict(x=x.cpu()), dict(weight=w.float()), dict(weight=w[:, :32]), dict(weight=w.contiguous()),
        dict(weight=w.cpu()), dict(weight=w[:1].expand(24, 40)), dict(weight=w[0]), dict(weight_scale=ws[:5]), dict(weight_scale=ws.double()), dict(weight_scale=ws.cpu()),
        dict(bias=ws[:1]), dict(bias=ws.half()), dict(activation="tanh"), dict(rows=end), dict(out=torch.empty((6, 23), dtype=BF16, device="cuda")),
        dict(out=torch.empty((24, 6), dtype=BF16, device="cuda").t()), dict(out=torch.empty((6, 24), dtype=torch.float64, device="cuda")), dict(out_dtype=torch.int32),
        dict(out=torch.empty((6, 24), dtype=BF16, device="cuda"), out_dtype=F32), dict(out=torch.empty((1, 24), dtype=BF16, device="cuda").expand(6, 24)), dict(offsets=end),
        dict(x=x.detach().requires_grad_()), dict(bias=torch.zeros(24, device="cuda", requires_grad=True))]
    grouped = [dict(weight=w), dict(offsets=end.long()), dict(offsets=end[:1]), dict(offsets=end.cpu()), dict(weight_scale=ws), dict(bias=ws), dict(rows=end.long()), dict(rows=end[None]),
               dict(rows=end.cpu()), dict(weight=w2[:1].expand(2, 24, 40))]
    for base, cases in ((dict(x=x, weight=w, weight_scale=ws), linear), (dict(x=x, weight=w2, weight_scale=ws2, offsets=end), grouped)):
        ops.int8_linear(**base)
        for case in cases:
            with pytest.raises(ValueError):
                ops.int8_linear(**{**base, **case})
    long = torch.zeros((1, 131072), dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="131071"):
        ops.int8_linear(long, torch.zeros((4, 131072), dtype=torch.int8, device="cuda"), ws[:4].contiguous())
    for case in (dict(x=x.float()), dict(x=x, out=torch.empty((6, 40), dtype=torch.int8, device="cuda")), dict(x=x, scale_out=ws), dict(x=x, rows=end.long()),
                 dict(x=x.detach().requires_grad_())):
        with pytest.raises(ValueError):
            ops.quantize_int8(**case)

    for case in (dict(x=x.float()), dict(x=x[:, :39]), dict(x=x, activation="tanh"), dict(x=x.t()), dict(x=x, out=x), dict(x=x, out=torch.empty((6, 20), dtype=F16, device="cuda")),
                 dict(x=x.detach().requires_grad_()), dict(x=x[:1].expand(6, 40))):
        with pytest.raises(ValueError):
            ops.checkpoint_activation(**case)
    h, kept = ops.checkpoint_activation(x)
    for case in (dict(grad=x), dict(grad=h.half()), dict(grad=h[:5]), dict(grad=h.cpu()), dict(grad=h, out=h), dict(grad=h[:1].expand(6, 20)), dict(grad=h.detach().requires_grad_())):
        with pytest.raises(ValueError):
            ops.checkpoint_activation_backward(kept=kept, **case)

    logits = torch.zeros((6, 8), device="cuda")
    for case in (dict(top_k=0), dict(top_k=9), dict(top_k=2.0), dict(logits=logits.double()), dict(logits=logits.t()), dict(logits=logits[0]), dict(logits=torch.zeros((2, 1025), device="cuda")),
                 dict(logits=torch.zeros((2, 64), device="cuda"), top_k=33), dict(token_mask=torch.ones(5, dtype=torch.bool, device="cuda")), dict(token_mask=torch.ones(6, device="cuda")),
                 dict(token_mask=torch.ones(6, dtype=torch.bool))):
        with pytest.raises(ValueError):
            ops.route_tokens(**{**dict(logits=logits, top_k=2), **case})
    r = ops.route_tokens(logits, 2)
    for case in (dict(logits=logits[:5]), dict(logits=logits[:, :7]), dict(grad_weights=torch.zeros((6, 3), device="cuda")), dict(grad_weights=torch.zeros((6, 2), device="cuda").half()),
                 dict(grad_balance_loss=torch.zeros(2, device="cuda")), dict(grad_balance_loss=torch.zeros(()))):
        with pytest.raises(ValueError):
            ops.route_tokens_backward(**{**dict(logits=logits, routing=r, grad_weights=None, grad_balance_loss=None), **case})


# ------------------------------------------------------------------------------------- calls that the documentation allows
def test_no_tokens_at_all(cuda_lib):
    logits = torch.empty((0, 8), device="cuda", requires_grad=True)
    r = ops.route_tokens(logits, 2)
    assert r.experts.shape == (0, 2) and not bool(r.counts.any()) and not bool(r.offsets.any()) and int(r.num_tokens) == 0 and float(r.balance_loss.detach()) == 0.0
    (r.weights.sum() + r.balance_loss).backward()
    assert logits.grad.shape == (0, 8)
    w, ws = product_tests.weights((3, 24), 40, seed=1)
    end = torch.zeros(3, dtype=torch.int32, device="cuda")
    none = torch.empty((0, 40), dtype=BF16, device="cuda")
    assert ops.int8_linear(none, w, ws, offsets=end, rows=torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 24)
    x = torch.empty((0, 48), dtype=BF16, device="cuda", requires_grad=True)
    ops.checkpointed_activation(x).sum().backward()
    assert x.grad.shape == (0, 48)


def test_rows_of_tokens_that_do_not_exist_are_not_numbers(cuda_lib):
    w, ws = product_tests.weights((2, 24), 40, seed=1)
    end = torch.tensor([1, 3], dtype=torch.int32, device="cuda")
    index = torch.tensor([0, 5, -1], dtype=torch.int32, device="cuda")
    for tokens in (0, 1):
        x = product_tests.tokens(1, 40, BF16, seed=2)[:tokens]
        y = ops.int8_linear(x, w, ws, offsets=end, rows=index)
        assert bool(torch.isnan(y[tokens:]).all())
        if tokens:
            product_tests.check(y[:1], x, w[0], ws[0])


def test_the_lowest_weight_and_one_channel(cuda_lib):
    for M in (1, 40, 600):
        x = torch.full((M, 131071), -3.0, dtype=BF16, device="cuda")
        w = torch.full((1, 131072), -128, dtype=torch.int8, device="cuda")[:, :131071]
        y = ops.int8_linear(x, w, torch.ones(1, device="cuda"), out_dtype=F32)
        product_tests.check(y, x, w, torch.ones(1, device="cuda"))


def test_in_inference_mode_and_with_results_as_leaves(cuda_lib):
    layer = Layer(30, 64, 32, 4, 2, BF16, seed=6)
    with torch.inference_mode():
        r = ops.route_tokens(layer.logits, 2, token_mask=layer.mask)
        up = ops.int8_linear(layer.x, layer.w1, layer.s1, offsets=r.offsets, rows=r.rows)
        h, kept = ops.checkpoint_activation(up)
        down = ops.int8_linear(h, layer.w2, layer.s2, offsets=r.offsets)
    live = int(r.offsets[-1])
    again = ops.route_tokens(layer.logits, 2, token_mask=layer.mask)
    assert torch.equal(r.experts, again.experts) and torch.equal(r.weights, again.weights)
    up2 = ops.int8_linear(layer.x, layer.w1, layer.s1, offsets=again.offsets, rows=again.rows)
    assert torch.equal(up[:live], up2[:live])
    leaf = up2[:live].requires_grad_(True)
    h2 = ops.checkpointed_activation(leaf)
    assert torch.equal(h[:live], h2.detach())
    h2.sum().backward()
    assert bool(torch.isfinite(leaf.grad).all())
    assert torch.equal(down[:live], ops.int8_linear(h2.detach(), layer.w2, layer.s2, offsets=again.offsets)[:live])


def test_two_streams_at_once(cuda_lib):
    """The same layer on two streams, many times without waiting: the shared status words are all that they share."""
    layers = [Layer(200, 128, 72, 8, 2, BF16, seed=s) for s in (7, 8)]
    want = [[t.clone() for t in layer.run()[1:5]] for layer in layers]
    streams = [torch.cuda.Stream() for _ in layers]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for _ in range(10):
        for i, (s, layer) in enumerate(zip(streams, layers)):
            with torch.cuda.stream(s):
                got[i] = layer.run()[1:5]
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.parametrize("T,D,F", [(400, 512, 264), (300, 200, 130), (3, 256, 128)])
def test_each_call_sees_what_the_call_before_it_wrote(cuda_lib, T, D, F):
    """A long row of calls into the same buffers, each of which reads what the one in front of it has just written, against the
    same calls with a wait after each: kernels are set up while the ones before them end."""
    g = torch.Generator(device="cuda").manual_seed(T)
    E, k, steps = 16, 2, 12
    wide = torch.randn((steps, T, 2 * F), device="cuda", generator=g).to(BF16)
    w, ws = product_tests.weights((D,), F, seed=1)
    w2, ws2 = product_tests.weights((E,), D, seed=2)
    w3, ws3 = product_tests.weights((E, 2 * F), D, seed=3)
    x, h, y, logits, dx = (torch.zeros(s, dtype=BF16, device="cuda") for s in ((T, 2 * F), (T, F), (T, D), (T, E), (T, 2 * F)))
    up = torch.zeros((T * k, 2 * F), dtype=BF16, device="cuda")

    def run(wait):
        made = []
        done = torch.cuda.synchronize if wait else lambda: None
        for i in range(steps):
            x.copy_(wide[i])
            _, kept = ops.checkpoint_activation(x, "gelu", out=h)
            done()
            dx_ = ops.checkpoint_activation_backward(h, kept, out=dx)
            done()
            q = ops.quantize_int8(h)
            done()
            ops.int8_linear(h, w, ws * 0.01, out=y)
            done()
            ops.int8_linear(y, w2, ws2, out=logits)
            done()
            r = ops.route_tokens(logits, k)
            done()
            d = ops.route_tokens_backward(logits, r, r.weights, r.balance_loss)
            done()
            ops.int8_linear(y, w3, ws3, offsets=r.offsets, rows=r.rows, out=up)
            done()
            h2, _ = ops.checkpoint_activation(up, "silu")
            x.zero_()
            made.append([t.clone() for t in (h, dx_, q.quantized.tensor, q.scale.tensor, y, logits, r.experts, r.rows, r.balance_loss, d, up, h2)])
        torch.cuda.synchronize()
        return made
    for a, b in zip(run(True), run(False)):
        for s, t in zip(a, b):
            assert torch.equal(torch.nan_to_num(s.float()), torch.nan_to_num(t.float()))


def test_an_event_of_another_stream_is_waited_for(cuda_lib):
    """The stream's last call is ours, then comes a wait for another stream that is still busy making the input."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(2)
    inputs = torch.randn((8, 64, 512), device="cuda", generator=g).to(BF16)
    want = [(ops.quantize_int8(x).quantized.tensor.clone(), ops.checkpoint_activation(x)[0].clone(), ops.route_tokens(x[:, :64], 3).experts.clone()) for x in inputs]
    big = torch.randn((4096, 4096), device="cuda", generator=g)
    x, other = torch.zeros((64, 512), dtype=BF16, device="cuda"), inputs[0].clone()
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        with torch.cuda.stream(a):
            a.wait_stream(b)
            x.zero_()
            for _ in range(3):
                big @ big
            x.copy_(inputs[i])
            made = a.record_event()
        with torch.cuda.stream(b):
            b.wait_stream(a) if i == 0 else None
            for call in (lambda t: ops.quantize_int8(t).quantized.tensor, lambda t: ops.checkpoint_activation(t)[0], lambda t: ops.route_tokens(t[:, :64], 3).experts):
                call(other)
                b.wait_event(made)
                got.append(call(x).clone())
    torch.cuda.synchronize()
    for y, z in zip(got, [t for w in want for t in w]):
        assert torch.equal(y, z)


# ------------------------------------------------------------------------------------------------------ memory of two streams
def _calls(seed):
    """Every operator once, as functions of the stream; inputs of their own."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((600, 512), device="cuda", generator=g).to(BF16)
    w, ws = product_tests.weights((256,), 512, seed=1)
    w3, ws3 = product_tests.weights((2, 256), 512, seed=2)
    ends = torch.tensor([250, 600], dtype=torch.int32, device="cuda")
    index = torch.randperm(600, device="cuda", generator=g).to(torch.int32)
    logits = torch.randn((600, 64), device="cuda", generator=g)
    _, kept = ops.checkpoint_activation(x)
    r = ops.route_tokens(logits, 4)
    return [lambda s: [ops.quantize_int8(x, stream=s).quantized.tensor], lambda s: [ops.int8_linear(x, w, ws, stream=s)],
            lambda s: [ops.int8_linear(x, w3, ws3, offsets=ends, rows=index, stream=s)],
            lambda s: list(ops.checkpoint_activation(x, stream=s)[:1]), lambda s: [ops.checkpoint_activation_backward(x[:, :256], kept, stream=s)],
            lambda s: list(ops.route_tokens(logits, 4, stream=s)[:7]), lambda s: [ops.route_tokens_backward(logits, r, r.weights, None, stream=s)]]


def test_a_given_stream_gets_memory_of_its_own(cuda_lib):
    """A block that the current stream has just given back may still be in use by work queued there: a call on another stream,
    which does not wait for that work, gets none of it."""
    side = torch.cuda.Stream()
    for call in _calls(3):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        sizes = sorted({t.untyped_storage().nbytes() for t in call(None)})
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        held = [torch.empty(n, dtype=torch.int8, device="cuda") for n in sizes for _ in range(12)]
        given_back = [(t.data_ptr(), t.data_ptr() + t.numel()) for t in held]
        del held
        for t in call(side):
            at = t.untyped_storage().data_ptr()
            assert not any(a <= at < b for a, b in given_back)
        side.synchronize()


def test_calls_on_two_streams_by_turns(cuda_lib):
    """Calls of the same sizes on the current stream and, by argument, on another one, many of them without waiting, and their
    temporaries given back at once."""
    side = torch.cuda.Stream()
    here, there = _calls(4), _calls(5)
    want = [[[t.clone() for t in call(None)] for call in calls] for calls in (here, there)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [[], []]
        for a, b in zip(here, there):
            got[0].append(a(None))
            got[1].append(b(side))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            for s, t in zip(w, g):
                for y, z in zip(s, t):
                    assert torch.equal(y, z)


def test_the_gradient_of_a_routing_on_a_given_stream(cuda_lib):
    logits = torch.randn((700, 32), device="cuda")
    a, b = logits.clone().requires_grad_(), logits.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    r, s = ops.route_tokens(a, 3, stream=side), ops.route_tokens(b, 3)
    torch.cuda.current_stream().wait_stream(side)
    for q in (r, s):
        (q.weights.square().sum() + q.balance_loss).backward()
    torch.cuda.synchronize()
    assert torch.equal(r.weights, s.weights) and torch.equal(a.grad, b.grad)


def test_refusals_of_a_checkpoint_that_does_not_fit(cuda_lib):
    """The checkpoint is looked at field by field, whichever way the call goes (a stream or an output given, or neither)."""
    x = torch.randn((6, 400), device="cuda").to(BF16)
    h, kept = ops.checkpoint_activation(x)
    stream, out = torch.cuda.current_stream(), torch.empty_like(x)
    bad = [dict(data=kept.data[:-16]), dict(data=kept.data[:0]), dict(data=torch.cat([kept.data, kept.data])), dict(data=kept.data.view(torch.uint8)), dict(data=kept.data[None]),
           dict(data=kept.data.cpu()), dict(data=torch.zeros(2 * kept.data.numel(), dtype=torch.int8, device="cuda")[::2]), dict(rows=7), dict(width=201), dict(rows=6.0), dict(rows=-1),
           dict(gated=False), dict(activation="tanh"), dict(dtype=F32), dict(dtype=F16)]
    for change in bad:
        for how in (dict(), dict(stream=stream), dict(out=out)):
            with pytest.raises(ValueError):
                ops.checkpoint_activation_backward(h, kept._replace(**change), **how)


def test_refusals_of_a_routing_that_does_not_fit(cuda_lib):
    stream = torch.cuda.current_stream()
    logits = torch.randn((6, 8), device="cuda")
    r = ops.route_tokens(logits, 2)
    for change in (dict(experts=r.experts[:, :1]), dict(experts=r.experts.t().contiguous().t()), dict(experts=r.experts.long()), dict(experts=r.experts.reshape(-1)), dict(weights=r.weights[:5]),
                   dict(weights=r.weights.half()), dict(weights=r.weights.cpu()), dict(weights=torch.zeros((6, 4), device="cuda")[:, ::2]), dict(counts=r.counts[:7]), dict(counts=r.counts.float()),
                   dict(num_tokens=r.num_tokens[:0]), dict(num_tokens=r.num_tokens.long()), dict(softmax=r.softmax[:-1]), dict(softmax=r.softmax.view(F32)), dict(softmax=r.softmax.view(6, 2)),
                   dict(softmax=r.softmax.cpu())):
        for how in (dict(), dict(stream=stream)):
            with pytest.raises(ValueError):
                ops.route_tokens_backward(logits, r._replace(**change), torch.ones((6, r.weights.shape[1]), device="cuda"), None, **how)


def test_choices_that_are_no_experts_have_no_gradient(cuda_lib):
    """A choice outside the experts reads and writes nothing: the slot counts as one that chose nothing."""
    logits = torch.randn((50, 8), device="cuda")
    r = ops.route_tokens(logits, 3)
    gw = torch.randn((50, 3), device="cuda")
    none, outside = r.experts.clone(), r.experts.clone()
    none[::3, 1:], outside[::3, 1:] = -1, 1 << 20
    none[1, 2], outside[1, 2] = -1, 8
    gl = torch.ones((), device="cuda")
    assert torch.equal(ops.route_tokens_backward(logits, r._replace(experts=outside), gw, gl), ops.route_tokens_backward(logits, r._replace(experts=none), gw, gl))


def test_tangents_are_refused(cuda_lib):
    """Forward-mode derivatives exist nowhere here: a tensor that carries a tangent is refused, not stripped of it."""
    fa = torch.autograd.forward_ad
    x, logits = torch.randn((6, 64), device="cuda").to(BF16), torch.randn((6, 8), device="cuda")
    w, ws = product_tests.weights((24,), 64, seed=1)
    bias = torch.zeros(24, device="cuda")
    h, kept = ops.checkpoint_activation(x)
    r = ops.route_tokens(logits, 2)
    gl = torch.ones((), device="cuda")
    stream = torch.cuda.current_stream()
    with fa.dual_level():
        dual = lambda t: fa.make_dual(t, torch.ones_like(t))  # noqa: E731
        for how in (dict(), dict(stream=stream)):
            for call in (lambda: ops.quantize_int8(dual(x), **how), lambda: ops.int8_linear(dual(x), w, ws, **how), lambda: ops.int8_linear(x, w, dual(ws), **how),
                         lambda: ops.int8_linear(x, w, ws, dual(bias), **how), lambda: ops.checkpoint_activation(dual(x), **how),
                         lambda: ops.checkpoint_activation_backward(dual(h), kept, **how), lambda: ops.route_tokens(dual(logits), 2, **how),
                         lambda: ops.route_tokens_backward(dual(logits), r, r.weights, gl, **how), lambda: ops.route_tokens_backward(logits, r, dual(r.weights), gl, **how),
                         lambda: ops.route_tokens_backward(logits, r, None, dual(gl), **how)):
                with pytest.raises(ValueError, match="forward-mode"):
                    call()
                with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                    call()
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.checkpointed_activation(dual(x))
        ops.int8_linear(x, w, ws)      # others go on
    for call in (lambda t: ops.route_tokens(t, 2).weights, lambda t: ops.int8_linear(t.to(BF16), w[:, :8].contiguous(), ws)):
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(call, (logits,), (logits,))
        with pytest.raises((ValueError, RuntimeError)):
            torch.vmap(call)(logits.expand(3, 6, 8))


def test_captured_calls_on_a_given_stream(cuda_lib):
    """Calls on another stream that has joined a capture: their memory belongs to the graph, replays follow their inputs, and
    eager calls of the same sizes between the replays change nothing."""
    side = torch.cuda.Stream()
    x = torch.randn((600, 512), device="cuda").to(BF16)
    logits = torch.randn((600, 64), device="cuda")
    w, ws = product_tests.weights((256,), 512, seed=1)

    def calls(s):
        h, kept = ops.checkpoint_activation(x, stream=s)
        r = ops.route_tokens(logits, 4, stream=s)
        return [ops.int8_linear(x, w, ws, stream=s), h, kept.scale, ops.checkpoint_activation_backward(h, kept, stream=s), r.rows, r.weights,
                ops.route_tokens_backward(logits, r, r.weights, None, stream=s)]
    calls(None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        got = calls(side)
        torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x.copy_(torch.randn((600, 512), device="cuda", generator=g))
        logits.copy_(torch.randn((600, 64), device="cuda", generator=g))
        want = calls(None)
        graph.replay()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_views_with_their_sign_turned(cuda_lib):
    """torch may keep a sign beside a tensor instead of in its memory: such a view is refused as an argument and heeded as a gradient."""
    neg = torch._neg_view
    x, logits = torch.randn((6, 64), device="cuda").to(BF16), torch.randn((6, 8), device="cuda")
    w, ws = product_tests.weights((24,), 64, seed=1)
    h, kept = ops.checkpoint_activation(x)
    r = ops.route_tokens(logits, 2)
    gl = torch.ones((), device="cuda")
    for call in (lambda: ops.quantize_int8(neg(x)), lambda: ops.int8_linear(neg(x), w, ws), lambda: ops.int8_linear(x, w, neg(ws)), lambda: ops.checkpoint_activation(neg(x)),
                 lambda: ops.checkpoint_activation_backward(neg(h), kept), lambda: ops.route_tokens(neg(logits), 2), lambda: ops.route_tokens_backward(neg(logits), r, r.weights, gl),
                 lambda: ops.route_tokens_backward(logits, r, neg(r.weights), gl), lambda: ops.route_tokens_backward(logits, r, r.weights, neg(gl))):
        with pytest.raises(ValueError, match="sign"):
            call()
    up, leaf = x.clone().requires_grad_(), logits.clone().requires_grad_()
    ops.checkpointed_activation(up).backward(neg(h))
    assert torch.equal(up.grad, ops.checkpoint_activation_backward(-h, kept))
    q = ops.route_tokens(leaf, 2)
    torch.autograd.backward([q.weights, q.balance_loss], [neg(r.weights), neg(gl)])
    assert torch.equal(leaf.grad, ops.route_tokens_backward(logits, r, -r.weights, -gl))
