"""The binding of the short calls: what is not its plain case it leaves to the Python around it, which says what is wrong; and
the sizes that both sides compute are the library's."""
import ctypes as C

import pytest
import torch

import cutlass_b200 as ops
from cutlass_b200 import lib as L
from cutlass_b200.routing import _scratch_words


def test_anything_but_cuda_tensors_is_left_alone():
    b = L.binding()
    x = torch.zeros((4, 32), dtype=torch.bfloat16)
    assert b.int8_linear(x, x, x, None, "relu", None, None, None) is None
    assert b.act_forward(x, "relu", True) is None
    assert b.act_backward(x, ops.ActivationCheckpoint(x, "relu", True, 4, 16, torch.bfloat16)) is None
    assert b.route_forward(x, 2, None, True) is None
    assert b.route_backward(x, ops.Routing(x, x, x, x, x, x, x, x, x, True), None, None) is None
    assert b.act_forward(3, 3, True) is None and b.act_forward(x) is None


def test_scratch_of_the_router_is_what_the_library_asks_for():
    for T in (0, 1, 128, 16, 17, 512, 513, 520, 1024, 592 * 16, 740 * 16, 740 * 16 + 1, 100000, 1 << 20):
        for E in (1, 7, 256, 1024):
            a, size = L.RouteArgs(experts=E, k=1, tokens=T), C.c_size_t()
            L.check(L.load().bsg_route_scratch_size(C.byref(a), C.byref(size)))
            assert size.value == 4 * _scratch_words(T, E)


def test_the_bound_entry_points_exist():
    assert set(L.BOUND) <= set(L.SYMBOLS)


@pytest.mark.gpu
def test_both_ways_give_the_same_bits(cuda_lib):
    """A call with its stream or output given goes through Python; without, through the binding."""
    stream = torch.cuda.current_stream()
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((50, 130), device="cuda", generator=g).to(torch.bfloat16)
    w = ops.quantize_int8(torch.randn((70, 130), device="cuda", generator=g).to(torch.bfloat16))
    W, S = w.quantized.tensor, w.scale.tensor
    for rows in (50, 3):
        assert torch.equal(ops.int8_linear(x[:rows], W, S, out_dtype=torch.float32), ops.int8_linear(x[:rows], W, S, out_dtype=torch.float32, stream=stream))
    index = torch.randint(0, 50, (90,), device="cuda", generator=g, dtype=torch.int32)
    ends = torch.tensor([30, 90], dtype=torch.int32, device="cuda")
    W2, S2 = torch.zeros((2, 70, 144), dtype=torch.int8, device="cuda")[..., :130], S.expand(2, 70).contiguous()
    W2.copy_(W)
    assert torch.equal(ops.int8_linear(x, W2, S2, offsets=ends, rows=index), ops.int8_linear(x, W2, S2, offsets=ends, rows=index, stream=stream))
    (h, kept), (h2, kept2) = ops.checkpoint_activation(x), ops.checkpoint_activation(x, stream=stream)
    assert torch.equal(h, h2) and torch.equal(kept.quantized[..., :65], kept2.quantized[..., :65]) and torch.equal(kept.scale, kept2.scale)
    assert torch.equal(ops.checkpoint_activation_backward(h, kept), ops.checkpoint_activation_backward(h, kept2, stream=stream))
    for T in (50, 300):
        l = torch.randn((T, 33), device="cuda", generator=g)
        r, r2 = ops.route_tokens(l, 4), ops.route_tokens(l, 4, stream=stream)
        for a, b in zip(r, r2):
            assert a is b or torch.equal(a, b)
        gl = torch.ones((), device="cuda")
        assert torch.equal(ops.route_tokens_backward(l, r, r.weights, gl), ops.route_tokens_backward(l, r2, r.weights, gl, stream=stream))


@pytest.mark.gpu
def test_results_are_tensors_of_their_own(cuda_lib):
    """The router's results lie in one buffer: changing one in place neither changes another nor what the backward pass reads."""
    l = torch.randn((9, 8), device="cuda", requires_grad=True)
    r = ops.route_tokens(l, 2)
    keep = [t.clone() for t in (r.experts, r.weights, r.rows, r.positions)]
    r.offsets.zero_()
    r.rows.fill_(7)
    with torch.no_grad():
        r.balance_loss.add_(1)
    assert torch.equal(r.experts, keep[0]) and torch.equal(r.weights, keep[1]) and torch.equal(r.positions, keep[3])
    (r.weights.sum() + r.balance_loss).backward()
    again = ops.route_tokens(l.detach(), 2)
    want = ops.route_tokens_backward(l.detach(), again, torch.ones_like(again.weights), torch.ones((), device="cuda"))
    assert torch.equal(l.grad, want)


@pytest.fixture
def unloaded(monkeypatch):
    monkeypatch.setattr(L, "_binding", None)
    return monkeypatch


def test_without_the_binding_python_makes_the_calls(unloaded, tmp_path):
    """Missing, not loadable, or made for another torch: a warning, and every call is left to the Python around it."""
    import cutlass_b200.build as B
    broken = tmp_path / "_binding.so"
    broken.write_bytes(b"no library")
    for change in (lambda m: m.setattr(L, "BINDING_PATH", str(tmp_path / "nothing.so")), lambda m: m.setattr(L, "BINDING_PATH", str(broken)),
                   lambda m: m.setattr(B, "_binding_for", lambda: "python 3.0 torch 0.1")):
        with unloaded.context() as m:
            m.setattr(L, "_binding", None)
            change(m)
            with pytest.warns(RuntimeWarning, match="binding"):
                b = L.binding()
            assert L.binding() is b
            assert b.int8_linear(1, 2, 3) is None and b.route_forward(None, 2, None, True) is None and b.act_backward(None, None) is None
    unloaded.setattr(L, "_binding", None)
    assert L.binding().made_for == B._binding_for()


def test_a_binding_that_cannot_be_built_is_a_warning(monkeypatch, tmp_path):
    """A host without a C++ compiler builds the library; a binding made for another torch is made again."""
    import cutlass_b200.build as B
    made = []
    monkeypatch.setattr(B, "BINDING", str(tmp_path / "_binding.so"))
    monkeypatch.setattr(B, "BINDING_STAMP", str(tmp_path / "binding.for"))
    with monkeypatch.context() as m:
        m.setenv("CXX", str(tmp_path / "no-such-compiler"))
        with pytest.warns(RuntimeWarning, match="not built"):
            assert B.build() == B.OUT
    monkeypatch.setattr(B, "_compile_binding", lambda: (made.append(1), open(B.BINDING, "w").close()))
    for _ in range(2):
        B._build_binding(False)
    assert len(made) == 1
    monkeypatch.setattr(B, "_binding_for", lambda: "python 3.0 torch 0.1")
    B._build_binding(False)
    assert len(made) == 2


@pytest.mark.gpu
def test_the_calls_work_without_the_binding(cuda_lib, unloaded):
    x = torch.randn((50, 128), device="cuda").to(torch.bfloat16)
    w = ops.quantize_int8(torch.randn((64, 128), device="cuda").to(torch.bfloat16))
    logits = torch.randn((50, 16), device="cuda")

    def calls():
        h, kept = ops.checkpoint_activation(x)
        leaf, up = logits.clone().requires_grad_(), x.clone().requires_grad_()
        r = ops.route_tokens(leaf, 2)
        (r.weights.square().sum() + r.balance_loss).backward()
        ops.checkpointed_activation(up).square().sum().backward()
        r2 = ops.route_tokens(logits, 2)
        return [ops.int8_linear(x, w.quantized.tensor, w.scale.tensor), ops.int8_linear(x[:2], w.quantized.tensor, w.scale.tensor), h, kept.scale,
                ops.checkpoint_activation_backward(h, kept), leaf.grad, up.grad, r2.rows, r2.weights, ops.route_tokens_backward(logits, r2, r2.weights, r2.balance_loss)]
    want = calls()
    unloaded.setattr(L, "_binding", None)
    unloaded.setattr(L, "BINDING_PATH", "nothing.so")
    with pytest.warns(RuntimeWarning):
        got = calls()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_other_threads_run_while_a_call_waits(cuda_lib):
    """A launch waits where the queue of the device is full; another Python thread goes on meanwhile."""
    import threading
    import time
    x = torch.randn((40, 128), device="cuda").to(torch.bfloat16)
    w = ops.quantize_int8(torch.randn((64, 128), device="cuda").to(torch.bfloat16))
    logits = torch.randn((8, 16), device="cuda")
    h, kept = ops.checkpoint_activation(x)
    r = ops.route_tokens(logits, 2)
    gl = torch.ones((), device="cuda")
    for call in (lambda: ops.int8_linear(x, w.quantized.tensor, w.scale.tensor), lambda: ops.checkpoint_activation(x), lambda: ops.checkpoint_activation_backward(h, kept),
                 lambda: ops.route_tokens(logits, 2), lambda: ops.route_tokens_backward(logits, r, r.weights, gl)):
        for _ in range(3):
            call()
        torch.cuda.synchronize()
        torch.cuda._sleep(2_500_000_000)      # more than a second
        took = []

        def queue():
            start = time.perf_counter()
            for _ in range(3000):
                call()
            took.append(time.perf_counter() - start)
        worker = threading.Thread(target=queue)
        worker.start()
        longest, last = 0.0, time.perf_counter()
        while worker.is_alive():
            time.sleep(0.002)
            now = time.perf_counter()
            longest, last = max(longest, now - last), now
        worker.join()
        torch.cuda.synchronize()
        assert took[0] > 0.8, "the queue did not fill"
        assert longest < 0.6, f"another thread stood still for {longest:.2f} s"
