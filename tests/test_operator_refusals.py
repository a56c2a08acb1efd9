"""What the 8-bit product, the checkpointed activation and the router refuse, at the C entry points and in Python (no GPU)."""
import ctypes as C

import pytest
import torch

import cutlass_b200 as ops
from cutlass_b200 import lib as L

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    from cutlass_b200 import build as B
    B.build()
    return L.load()


def int8_args(**kw):
    a = L.Int8Args()
    a.in_kind, a.out_kind, a.num_groups = L.OUT_BF16, L.OUT_BF16, 1
    a.rows = a.tokens = 40
    a.N, a.K = 96, 64
    a.X, a.ldx, a.Q, a.ldq, a.q_scale = 0x10000, 64, 0x20000, 64, 0x30000
    a.W, a.ldw, a.w_scale, a.D, a.ldd = 0x40000, 64, 0x50000, 0x60000, 96
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(out_kind=L.OUT_E4M3), 3), (dict(activation=4), 3), (dict(activation=-1), 3), (dict(num_groups=0), 2), (dict(num_groups=257, offsets=0x100), 2),
    (dict(num_groups=2), 2), (dict(N=0), 2), (dict(K=0), 2), (dict(K=131072, ldw=131072, ldq=131072), 2), (dict(rows=-1), 2), (dict(W=None), 2), (dict(w_scale=None), 2),
    (dict(D=None), 2), (dict(Q=None), 2), (dict(W=0x40008), 1), (dict(ldw=72), 1), (dict(ldq=72), 1), (dict(Q=0x20004), 1), (dict(ldw=48), 2), (dict(ldd=95), 2),
    (dict(D=0x60001), 1), (dict(out_kind=L.OUT_F32, D=0x60002), 1), (dict(bias=0x70002), 1), (dict(kernel=3), 3), (dict(tile=48), 3), (dict(kernel=2, tile=64), 3),
    (dict(kernel=2, tile=256, split=2), 3), (dict(kernel=1, tile=128, split=2), 3), (dict(kernel=1, tile=16, split=3), 3), (dict(kernel=1, tile=16, split=4), 3),
    (dict(num_groups=2, offsets=0x100, group_stride_w=1000), 1), (dict(num_groups=2, offsets=0x100), 2), (dict(num_groups=2, offsets=0x100, group_stride_w=48), 2),
    (dict(rows=1 << 31), 2)])
def test_the_product_refuses(lib, kw, code):
    assert lib.bsg_int8_query(C.byref(int8_args(**kw)), None) == code
    assert lib.bsg_int8_gemm_run(C.byref(int8_args(**kw)), 0x100, 16, None) == code
    assert L.last_error()


def test_the_product_accepts_and_wants_a_workspace(lib):
    caps = L.Caps()
    for kw in (dict(), dict(rows=0, tokens=0, Q=None, D=None, q_scale=None), dict(N=1, ldd=1), dict(K=1), dict(out_kind=L.OUT_F32, D=0x60004), dict(D=0x60002),
               dict(offsets=0x100), dict(num_groups=256, offsets=0x100, group_stride_w=96 * 64), dict(kernel=1, tile=16, split=1), dict(kernel=2, tile=256)):
        assert lib.bsg_int8_query(C.byref(int8_args(**kw)), C.byref(caps)) == 0, L.last_error()
        assert caps.tile_k == 128
    for ws, size in ((None, 16), (0x100, 8)):
        assert lib.bsg_int8_gemm_run(C.byref(int8_args()), ws, size, None) == 4
        assert lib.bsg_int8_linear_run(C.byref(int8_args()), ws, size, None) == 4
    assert lib.bsg_int8_gemm_run(C.byref(int8_args()), 0x102, 16, None) == 1
    assert lib.bsg_int8_query(None, None) == 2 and lib.bsg_int8_linear_run(None, None, 0, None) == 2


@pytest.mark.parametrize("kw,code", [(dict(in_kind=L.OUT_F32), 3), (dict(rows=41), 2), (dict(K=0), 2), (dict(X=None), 2), (dict(q_scale=None), 2), (dict(ldx=63), 2),
                                     (dict(ldq=63), 1), (dict(ldq=72), 1), (dict(Q=0x20008), 1), (dict(X=0x10001), 1), (dict(tokens=-1), 2)])
def test_the_quantiser_refuses(lib, kw, code):
    assert lib.bsg_int8_quantize(C.byref(int8_args(**kw)), None) == code
    assert lib.bsg_int8_linear_run(C.byref(int8_args(**kw)), 0x100, 16, None) == code


def test_only_a_few_tokens_may_leave_out_the_scratch(lib):
    """Without Q the tokens are quantised inside the product: at most four rows of at most 64 KB, dense, no index."""
    for kw in (dict(rows=5, tokens=5), dict(rows=2, tokens=2, K=40000, ldx=40000, ldw=40000), dict(rows=2, tokens=2, offsets=0x100), dict(rows=2, tokens=9, index=0x100),
               dict(rows=1, tokens=1, kernel=1)):
        assert lib.bsg_int8_linear_run(C.byref(int8_args(Q=None, q_scale=None, **kw)), 0x100, 16, None) == 2


def test_scratch_rows(lib):
    n = C.c_int64()
    for rows, tokens, K, index, want in ((100, 100, 4096, None, 100), (100, 50, 64, 0x100, 100), (8192, 4096, 4096, 0x100, 8192 + 4096), (8191, 4096, 4096, 0x100, 8191)):
        assert lib.bsg_int8_scratch_rows(C.byref(L.Int8Args(rows=rows, tokens=tokens, K=K, index=index)), C.byref(n)) == 0
        assert n.value == want


def act_args(**kw):
    a = L.ActArgs(L.OUT_BF16, 3, 1, 0, 8, 100, 0x1000, 200, 0x2000, 200, 0x3000, 0x4000)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [(dict(type=L.OUT_F32), 3), (dict(activation=9), 3), (dict(gated=2), 2), (dict(rows=-1), 2), (dict(width=0), 2), (dict(in_=None), 2),
                                     (dict(out=None), 2), (dict(kept=None), 2), (dict(kept_scale=None), 2), (dict(ld_in=99), 2), (dict(ld_out=99), 2), (dict(in_=0x1001), 1),
                                     (dict(kept=0x3008), 1), (dict(kept_scale=0x4002), 1), (dict(rows=1 << 29, width=1 << 20, ld_in=1 << 22, ld_out=1 << 22), 2)])
def test_the_activation_refuses(lib, kw, code):
    assert lib.bsg_act_forward(C.byref(act_args(**kw)), None) == code
    assert lib.bsg_act_backward(C.byref(act_args(**kw)), None) == code


def test_the_activation_knows_which_side_is_wide(lib):
    assert lib.bsg_act_forward(C.byref(act_args(ld_in=199)), None) == 2 and lib.bsg_act_backward(C.byref(act_args(ld_out=199)), None) == 2
    assert lib.bsg_act_forward(C.byref(act_args(rows=0, in_=None)), None) == 0 and lib.bsg_act_forward(None, None) == 2


def route_args(**kw):
    a = L.RouteArgs(L.OUT_BF16, 16, 2, 1, 10, 0x1000, 16, None, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000, 0x8000, 0x9000, 0xa000, None, None, 0xb000, 16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [(dict(type=L.OUT_MXFP8), 3), (dict(experts=0), 2), (dict(experts=1025, ld=1025), 2), (dict(k=0), 2), (dict(k=17), 2), (dict(experts=64, k=33, ld=64), 2),
                                     (dict(tokens=-1), 2), (dict(tokens=1 << 31), 2), (dict(normalize=2), 2), (dict(counts=None), 2), (dict(live=None), 2), (dict(logits=None), 2),
                                     (dict(chosen=None), 2), (dict(weights=None), 2), (dict(softmax=None), 2), (dict(softmax=0x6004), 1), (dict(ld=15), 2), (dict(logits=0x1001), 1)])
def test_the_router_refuses(lib, kw, code):
    assert lib.bsg_route_forward(C.byref(route_args(**kw)), 0x100, 1 << 20, None) == code
    assert lib.bsg_route_backward(C.byref(route_args(**kw)), None) == code


def test_the_router_refuses_one_way(lib):
    for kw, code in ((dict(offsets=None), 2), (dict(loss=None), 2), (dict(rows=None), 2), (dict(positions=None), 2)):
        assert lib.bsg_route_forward(C.byref(route_args(**kw)), None, 0, None) == code
    assert lib.bsg_route_backward(C.byref(route_args(grad_logits=None)), None) == 2 and lib.bsg_route_backward(C.byref(route_args(ld_grad=15)), None) == 2
    assert lib.bsg_route_forward(C.byref(route_args(tokens=2000)), None, 0, None) == 4 and lib.bsg_route_forward(C.byref(route_args(tokens=2000)), 0x100, 16, None) == 4
    assert lib.bsg_route_forward(C.byref(route_args(tokens=2000)), 0x104, 1 << 20, None) == 1


# --------------------------------------------------------------------------------------------------------- Python
def test_python_says_what_is_wrong():
    x = torch.zeros((4, 32), dtype=BF16)
    w, ws = torch.zeros((8, 32), dtype=torch.int8), torch.ones(8)
    for call in (lambda: ops.int8_linear(x, w, ws), lambda: ops.quantize_int8(x), lambda: ops.checkpoint_activation(x), lambda: ops.route_tokens(x, 2)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for bad in (x.float(), x[0], torch.zeros((4, 32), dtype=torch.int8)):
        with pytest.raises(ValueError, match="2-D CUDA tensor"):
            ops.int8_linear(bad, w, ws)


def test_operators_are_found_by_their_operands():
    def operand(rows, K, transpose=False, dtype=torch.int8):
        q = torch.zeros((rows, -(-K // 16) * 16), dtype=dtype)[:, :K]
        return ops.ScaledOperand(q.t() if transpose else q, torch.ones(rows), (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone)
    M, N, K = 6, 10, 40
    out = torch.zeros((M, N), dtype=BF16)
    good = ops.GemmArguments(operand(M, K), operand(N, K, True), out, torch.int32)
    found = ops.get_operators(good)
    assert [o.metadata.kind for o in found] == [L.KIND_INT8] and not found[0].metadata.grouped and found[0].supports(good, "100a")
    assert len(ops.get_operators()) == len(ops.all_operators()) + 2
    wrong = [ops.GemmArguments(operand(M, K), operand(N, K, True), out, torch.float32),
             ops.GemmArguments(operand(M, K), operand(N, K, True), out.to(torch.float8_e4m3fn), torch.int32),
             ops.GemmArguments(operand(M, K, dtype=torch.uint8), operand(N, K, True), out, torch.int32),
             ops.GemmArguments(operand(M, K), operand(N, K, True), out, torch.int32, ops.EpilogueDescriptor(alpha=2.0)),
             ops.GemmArguments(operand(M, K), operand(N, K, True), out, torch.int32, ops.EpilogueDescriptor(bias=torch.zeros(N + 1))),
             ops.GemmArguments(operand(M, K), operand(N, K, True), out, torch.int32, ops.EpilogueDescriptor(activation="tanh")),
             ops.GemmArguments(operand(M, K), operand(N, K, True), torch.zeros((N, M), dtype=BF16).t(), torch.int32),
             ops.GemmArguments(torch.zeros((M, K), dtype=torch.int8), torch.zeros((N, K), dtype=torch.int8).t(), out, torch.int32)]
    contiguous = torch.zeros((N, K), dtype=torch.int8)      # rows of 40 bytes
    wrong.append(ops.GemmArguments(operand(M, K), ops.ScaledOperand(contiguous.t(), torch.ones(N), (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone), out, torch.int32))
    wrong.append(ops.GemmArguments(operand(M, K), ops.ScaledOperand(operand(N, K, True).quantized, torch.ones(N, 2), (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone), out, torch.int32))
    wrong.append(ops.GemmArguments(operand(M, K), ops.ScaledOperand(operand(N, K, True).quantized, torch.ones(N), (1, 1, 16), ops.ScaleSwizzleMode.SwizzleNone), out, torch.int32))
    for args in wrong:
        assert ops.get_operators(args) == []
        with pytest.raises(ValueError):
            found[0].run(args)
    E = 3
    q = torch.zeros((E, N, 48), dtype=torch.int8)[..., :K]
    grouped = ops.GroupedGemmArguments(operand(M, K), ops.ScaledOperand(q.transpose(1, 2), torch.ones((E, N)), (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone), out, torch.int32,
                                       offsets=torch.zeros(E, dtype=torch.int32))
    assert [o.metadata.grouped for o in ops.get_operators(grouped)] == [True]


def _int8_arguments(device, **moved):
    """Dense and grouped arguments on ``device``; ``moved``: names of tensors -> the device they are on instead."""
    at = lambda name: moved.get(name, device)  # noqa: E731
    M, N, K, E = 6, 16, 48, 3
    A = ops.ScaledOperand(torch.zeros((M, K), dtype=torch.int8, device=at("a")), torch.ones(M, device=at("a_scale")), (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone)
    made = []
    for shape in ((N,), (E, N)):
        q = torch.zeros(shape + (K,), dtype=torch.int8, device=at("b")).transpose(-1, -2)
        B = ops.ScaledOperand(q, torch.ones(shape, device=at("b_scale")), (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone)
        out = torch.zeros((M, N), dtype=BF16, device=at("out"))
        epilogue = ops.EpilogueDescriptor(bias=torch.zeros(shape, device=at("bias")))
        made.append(ops.GroupedGemmArguments(A, B, out, torch.int32, offsets=torch.full((E,), M, dtype=torch.int32, device=at("offsets")), epilogue=epilogue) if len(shape) == 2
                    else ops.GemmArguments(A, B, out, torch.int32, epilogue))
    return made


def test_operators_run_on_cuda_tensors_only():
    for args in _int8_arguments("cpu"):
        with pytest.raises(ValueError, match="CUDA device"):
            ops.get_operators(args)[0].run(args)


@pytest.mark.gpu
def test_operators_want_all_tensors_on_one_device(cuda_lib):
    for args in _int8_arguments("cuda"):
        ops.get_operators(args)[0].run(args)
    for name in ("a", "a_scale", "b", "b_scale", "out", "bias", "offsets"):
        dense, grouped = _int8_arguments("cuda", **{name: "cpu"})
        for args in [grouped] if name == "offsets" else [dense, grouped]:
            with pytest.raises(ValueError, match="CUDA device"):
                ops.get_operators(args)[0].run(args)
    torch.cuda.synchronize()
