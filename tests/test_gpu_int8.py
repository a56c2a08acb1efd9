"""The 8-bit integer product and its quantiser on the GPU against the definition in 64 bits."""
import math

import pytest
import torch

import cutlass_b200 as ops
from cutlass_b200 import lib as L
from cutlass_b200.operator import _default_workspace

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def levels(x):
    """(whole numbers, scale) of every row, in 64 bits; rows with a NaN or an infinity: zeros, NaN."""
    x = x.double()
    amax = x.abs().amax(1)
    bad = ~torch.isfinite(amax)
    safe = torch.where(bad | (amax == 0), torch.ones_like(amax), amax)[:, None]
    q = torch.sign(x) * torch.floor(127.0 * x.abs() / safe + 0.5)
    q = torch.where((bad | (amax == 0))[:, None], torch.zeros_like(q), q)
    return q, torch.where(bad, torch.full_like(amax, math.nan), amax / 127.0)


def tokens(M, K, dtype, seed, pitch=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((M, K), device="cuda", generator=g) * torch.exp2(torch.randint(-6, 7, (M, 1), device="cuda", generator=g).float())
    buf = torch.full((M, pitch or K), 7.0, device="cuda", dtype=dtype)
    buf[:, :K] = x.to(dtype)
    return buf[:, :K]


def weights(shape, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.full(shape + (-(-K // 16) * 16,), 99, dtype=torch.int8, device="cuda")      # 99 behind the row: must not be used
    buf[..., :K] = torch.randint(-127, 128, shape + (K,), device="cuda", generator=g, dtype=torch.int8)
    return buf[..., :K], torch.rand(shape, device="cuda", generator=g) * 0.01 + 0.001


def act64(x, name):
    if name == "relu":
        return torch.where(x > 0, x, torch.where(torch.isnan(x), x, torch.zeros_like(x)))
    if name == "gelu":
        return 0.5 * x * torch.erfc(-x / math.sqrt(2.0))
    return x * torch.sigmoid(x) if name == "silu" else x


def check(got, x, w, ws, bias=None, activation="identity"):
    """Per element: the sum is exact; it, the token scale and the two products with the scales are rounded to 24 bits
    (4 * 2^-24 of the product), then the sum with the bias; an activation has a slope of at most 1.13 and its own rounding
    (exponential and error function: 2 units, product and quotient: 1 each, under 2^-20 in all); last the output's half step."""
    q, s = levels(x)
    p = (q @ w.double().t()) * s[:, None] * ws.double()
    b = torch.zeros_like(p) if bias is None else bias.double().expand_as(p)
    want = act64(p + b, activation)
    inner = 6 * 2.0 ** -24 * (p.abs() + b.abs())
    if activation != "identity":
        inner = 1.13 * inner + 2.0 ** -20 * (p + b).abs()
    tol = inner + torch.finfo(got.dtype).eps / 2 * (want.abs() + inner) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got.double()), nan)
    err = torch.where(nan, torch.zeros_like(tol), (got.double() - want).abs() - tol)
    assert float(err.max()) <= 0.0, f"{int((err > 0).sum())} of {err.numel()} values off, worst {float(err.max())}"


def status_ok():
    L.check(L.load().bsg_read_device_status(_default_workspace(torch.device("cuda", torch.cuda.current_device())).data_ptr(),
                                            torch.cuda.current_stream().cuda_stream))


# ---------------------------------------------------------------------------------------------------- quantiser
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,K,pitch", [(1, 1, None), (3, 17, None), (9, 16, 24), (5, 2048, None), (4, 2049, None), (7, 2056, 2058), (2, 8192, None),
                                       (3, 8193, 8200), (2, 33000, None), (300, 129, None)])
def test_quantised_rows_equal_the_definition(cuda_lib, dtype, M, K, pitch):
    x = tokens(M, K, dtype, seed=M * 31 + K, pitch=pitch)
    r = ops.quantize_int8(x)
    q, s = levels(x)
    assert r.quantized.tensor.stride(0) % 16 == 0 or M == 1
    assert torch.equal(r.quantized.tensor.double(), q)
    assert torch.equal(r.scale.tensor, s.float())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_halves_round_outwards_for_every_maximum(cuda_lib, dtype):
    """Every mantissa of the maximum against values on, just under and just above each half k + 1/2 of its levels."""
    mant = torch.arange(128, 256, device="cuda") if dtype == BF16 else torch.arange(1024, 2048, 3, device="cuda")
    amax = mant.to(dtype)
    half = (torch.arange(127, device="cuda").double() + 0.5)[None] * amax.double()[:, None] / 127.0
    near = half.to(dtype)
    bits = near.view(torch.int16)
    x = torch.cat([amax[:, None], near, (bits - 1).view(dtype), -(bits + 1).view(dtype), -near], 1).clamp(-amax[:, None], amax[:, None])
    r = ops.quantize_int8(x.contiguous())
    assert torch.equal(r.quantized.tensor.double(), levels(x)[0])


def test_rows_of_extreme_values(cuda_lib):
    big, tiny = torch.finfo(BF16).max, 2.0 ** -133
    rows = torch.zeros((8, 40), dtype=BF16, device="cuda")
    rows[1] = tiny
    rows[1, 3] = 3 * tiny
    rows[2, ::2], rows[2, 1] = big, -big / 2
    rows[3, 5] = math.nan
    rows[4, 0], rows[4, 39] = math.inf, 1.0
    rows[5, 7], rows[5, 8] = -math.inf, math.nan
    rows[6] = 2.0 ** -64
    rows[6, 1] = 2.0 ** -65
    rows[7] = 1e-30
    r = ops.quantize_int8(rows)
    q, s = levels(rows)
    assert torch.equal(r.quantized.tensor.double(), q)
    got = r.scale.tensor
    assert torch.equal(torch.isnan(got), torch.isnan(s)) and torch.equal(got[~torch.isnan(s)], s.float()[~torch.isnan(s)])


def test_rows_by_index_and_untouched_surroundings(cuda_lib):
    x = tokens(6, 50, BF16, seed=1)
    buf = torch.full((5, 80), 77, dtype=torch.int8, device="cuda")
    scale = torch.full((5,), -1.0, device="cuda")
    rows = torch.tensor([5, 0, -1, 6, 0], dtype=torch.int32, device="cuda")
    ops.quantize_int8(x, rows=rows, out=buf[:, :50], scale_out=scale)
    q, s = levels(x)
    for i, r in enumerate(rows.tolist()):
        if 0 <= r < 6:
            assert torch.equal(buf[i, :50].double(), q[r]) and float(scale[i]) == float(s.float()[r])
        else:
            assert not buf[i, :50].any() and math.isnan(float(scale[i]))
    assert bool((buf[:, 50:] == 77).all())


# ------------------------------------------------------------------------------------------------------- products
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 16), (1, 4096, 4096), (2, 1000, 300), (7, 333, 129), (16, 256, 2048), (17, 257, 1040),
                                   (33, 1003, 515), (64, 512, 1024), (65, 130, 700), (128, 640, 384), (129, 127, 257), (200, 1024, 128),
                                   (300, 1003, 2050), (513, 520, 1000), (1000, 72, 64)])
def test_dense_product(cuda_lib, M, N, K, out_dtype):
    x = tokens(M, K, F16 if out_dtype == F16 else BF16, seed=M + N + K)
    w, ws = weights((N,), K, seed=K)
    if out_dtype == F16:
        ws = ws * (0.05 / math.sqrt(K))
        x = (x / 64).contiguous()
    check(ops.int8_linear(x, w, ws, out_dtype=out_dtype), x, w, ws)
    status_ok()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,N,K,pitch", [(1, 33, 8192, None), (2, 17, 515, 517), (3, 100, 16384, None), (4, 16, 2064, None), (3, 50, 1000, 1001), (4, 5000, 512, None), (5, 64, 512, None),
                                         (4, 40, 16384, None), (4, 40, 16385, None), (1, 9, 65536, None), (1, 9, 65537, None)])
def test_a_few_tokens(cuda_lib, M, N, K, pitch, dtype):
    """Around the limits of the kernel that quantises on the way; its bits are those of the two-step form."""
    x = tokens(M, K, dtype, seed=M + N, pitch=pitch)
    w, ws = weights((N,), K, seed=N)
    bias = torch.randn(N, device="cuda")
    got = ops.int8_linear(x, w, ws, bias, activation="silu", out_dtype=F32)
    check(got, x, w, ws, bias, "silu")
    one = torch.tensor([M], dtype=torch.int32, device="cuda")
    assert torch.equal(got, ops.int8_linear(x, w[None], ws[None], bias[None], activation="silu", out_dtype=F32, offsets=one))


@pytest.mark.parametrize("M,N,K", [(5, 200, 2000), (40, 1030, 1024), (130, 264, 256), (260, 515, 130)])
@pytest.mark.parametrize("activation", ["identity", "relu", "gelu", "silu"])
def test_bias_and_activation(cuda_lib, M, N, K, activation):
    x = tokens(M, K, BF16, seed=3)
    w, ws = weights((N,), K, seed=4)
    ws = ws / math.sqrt(K)
    bias = torch.randn(N, device="cuda")
    check(ops.int8_linear(x, w, ws, bias, activation=activation, out_dtype=F32), x, w, ws, bias, activation)
    check(ops.int8_linear(x, w, ws, bias, activation=activation), x, w, ws, bias, activation)


@pytest.mark.parametrize("kernel,tile,split", [(1, 16, 1), (1, 16, 2), (1, 16, 4), (1, 16, 8), (1, 32, 1), (1, 32, 8), (1, 64, 1), (1, 64, 4),
                                               (1, 128, 1), (2, 128, 0), (2, 256, 0)])
@pytest.mark.parametrize("M,N,K", [(1, 200, 1024), (61, 520, 2100), (300, 400, 1500)])
def test_every_kernel_gives_the_same_bits(cuda_lib, kernel, tile, split, M, N, K):
    """The sums are exact, so kernel, tile and split change nothing."""
    import ctypes as C
    x = tokens(M, K, BF16, seed=9)
    w, ws = weights((N,), K, seed=10)
    A = ops.quantize_int8(x)
    want = ops.int8_linear(x, w, ws, out_dtype=F32)
    out = torch.full((M, N), math.nan, device="cuda")
    B = ops.ScaledOperand(w.t(), ws, (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone)
    args = ops.GemmArguments(A, B, out, torch.int32)
    op = ops.get_operators(args)[0]
    a = op.build_args(args)
    a.kernel, a.tile, a.split = kernel, tile, split
    workspace = torch.zeros(16, dtype=torch.uint8, device="cuda")
    L.check(L.load().bsg_int8_gemm_run(C.byref(a), workspace.data_ptr(), 16, None))
    L.check(L.load().bsg_read_device_status(workspace.data_ptr(), None))
    assert torch.equal(out, want)
    check(out, x, w, ws)


@pytest.mark.parametrize("M,N,dtype", [(2560, 2048, BF16), (2560, 1928, F32), (2300, 2051, F16)])
def test_more_tiles_than_pairs_of_sms(cuda_lib, M, N, dtype):
    """80 tiles of 256 x 256: a whole wave and a thin one, whose tiles are computed in halves, on any number of SMs up to 158."""
    import ctypes as C
    K = 200
    x = tokens(M, K, BF16, seed=1)
    w, ws = weights((N,), K, seed=2)
    ws = ws * 0.001
    A = ops.quantize_int8(x)
    out = torch.full((M, N), math.nan, dtype=dtype, device="cuda")
    op = ops.Int8GemmOperator(ops.get_operators(metadata_filter=lambda m: m.kind == L.KIND_INT8)[0].metadata)
    a = op.build_args(ops.GemmArguments(A, ops.ScaledOperand(w.t(), ws, (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone), out, torch.int32))
    a.kernel, a.tile = 2, 256
    workspace = torch.zeros(16, dtype=torch.uint8, device="cuda")
    L.check(L.load().bsg_int8_gemm_run(C.byref(a), workspace.data_ptr(), 16, None))
    L.check(L.load().bsg_read_device_status(workspace.data_ptr(), None))
    check(out, x, w, ws)


@pytest.mark.parametrize("sizes,N,tile,dtype", [((4099,), 2048, 256, BF16), ((4220,), 2048, 256, F32), ((4099,), 2048, 128, BF16), ((4220,), 2048, 128, F16), ((3920,), 11968, 256, BF16),
                                                ((1000, 517, 0, 333, 2050, 77, 1500), 1024, 128, BF16), ((1000, 517, 0, 333, 2050, 77, 1500), 1024, 128, F32)])
def test_a_groups_last_rows_behind_whole_tiles(cuda_lib, sizes, N, tile, dtype):
    """A pair of SMs goes from a tile whose rows leave by asynchronous copies to one that holds a matrix' or a group's last rows,
    which are stored by threads, with so little to add up that the second tile is ready at once: every value equals that of the
    kernel for few rows, whose results leave another way."""
    import ctypes as C
    M, E, K = sum(sizes), len(sizes), 64
    x = tokens(M, K, BF16, seed=1)
    w, ws = weights((E, N), K, seed=2)
    ws = ws * 0.001
    A = ops.quantize_int8(x)
    ends = torch.tensor(sizes, device="cuda").cumsum(0).to(torch.int32)
    out = torch.full((M, N), math.nan, dtype=dtype, device="cuda")
    if E > 1:
        args = ops.GroupedGemmArguments(A, ops.ScaledOperand(w.transpose(1, 2), ws, (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone), out, torch.int32, offsets=ends)
    else:
        args = ops.GemmArguments(A, ops.ScaledOperand(w[0].t(), ws[0], (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone), out, torch.int32)
    a = ops.get_operators(args)[0].build_args(args)
    workspace = torch.zeros(16, dtype=torch.uint8, device="cuda")

    def product(kernel, tile):
        out.fill_(math.nan)
        a.kernel, a.tile = kernel, tile
        L.check(L.load().bsg_int8_gemm_run(C.byref(a), workspace.data_ptr(), 16, torch.cuda.current_stream().cuda_stream))
        return out.clone()
    want = product(1, 64)
    for _ in range(8):
        assert torch.equal(product(2, tile), want)
    L.check(L.load().bsg_read_device_status(workspace.data_ptr(), torch.cuda.current_stream().cuda_stream))
    begin = 0
    for e, n in enumerate(sizes):
        if n:
            check(want[begin:begin + n], x[begin:begin + n], w[e], ws[e])
        begin += n


def test_the_longest_sum_is_exact(cuda_lib):
    """All products 127 * 127 at the largest K: the sum comes within 2^-9 of the 32-bit range."""
    K = 131071
    x = torch.ones((1, K), dtype=BF16, device="cuda")
    w = torch.full((3, -(-K // 16) * 16), 127, dtype=torch.int8, device="cuda")[:, :K]
    w[1] = -127
    w[2, :5] = -127
    ws = torch.ones(3, device="cuda")
    got = ops.int8_linear(x, w, ws, out_dtype=F32)
    check(got, x, w, ws)


def test_rows_that_cannot_be_quantised_and_views(cuda_lib):
    """NaN and infinity stay in their rows; x, out and bias as unaligned views; nothing outside the view is written."""
    M, N, K = 21, 77, 90
    x = tokens(M, K, BF16, seed=5, pitch=K + 1)
    x[4, 3], x[9, 0], x[20, 89] = math.nan, math.inf, -math.inf
    x[7] = 0
    w, ws = weights((N,), K, seed=6)
    bias = torch.randn(N + 1, device="cuda")[1:]
    for m, dtype in ((M, F32), (M, BF16)):
        buf = torch.full((m, N + 3), 5.0, dtype=dtype, device="cuda")
        ops.int8_linear(x, w, ws, bias, out=buf[:, 1:1 + N])
        check(buf[:, 1:1 + N], x, w, ws, bias)
        assert bool((buf[:, 0] == 5).all()) and bool((buf[:, 1 + N:] == 5).all())
    big = torch.cat([x] * 20)
    buf = torch.full((20 * M, N + 3), 5.0, dtype=BF16, device="cuda")
    ops.int8_linear(big, w, ws, bias, out=buf[:, 1:1 + N])
    check(buf[:, 1:1 + N], big, w, ws, bias)
    assert bool((buf[:, 0] == 5).all()) and bool((buf[:, 1 + N:] == 5).all())


# -------------------------------------------------------------------------------------------------------- experts
@pytest.mark.parametrize("sizes,N,K", [([1], 64, 32), ([0, 3, 0, 0, 5, 1], 130, 200), ([16, 0, 17, 1], 256, 512), ([100, 0, 1, 63, 200], 200, 320),
                                       ([300, 0, 257, 1, 256, 31], 515, 200), ([0, 0, 0], 64, 64), ([2] * 256, 48, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_grouped_product(cuda_lib, sizes, N, K, dtype):
    E, T = len(sizes), 37
    total, spare = sum(sizes), 5
    x = tokens(T, K, dtype, seed=E + N)
    w, ws = weights((E, N), K, seed=E)
    ws = ws * 0.02
    bias = torch.randn((E, N), device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    rows = torch.cat([torch.randint(0, T, (total,), device="cuda", generator=g, dtype=torch.int32),
                      torch.full((spare,), -1, dtype=torch.int32, device="cuda")])
    offsets = torch.tensor(sizes, device="cuda").cumsum(0).to(torch.int32)
    for pitch in (N, -(-N // 8) * 8 + 8):
        buf = torch.full((total + spare, pitch), 3.0, dtype=dtype, device="cuda")
        out = ops.int8_linear(x, w, ws, bias, offsets=offsets, rows=rows, out=buf[:, :N])
        begin = 0
        for e, n in enumerate(sizes):
            if n:
                check(out[begin:begin + n], x[rows[begin:begin + n].long()], w[e], ws[e], bias[e])
            begin += n
        assert bool((buf[total:] == 3).all()) and bool((buf[:, N:] == 3).all()), "written behind the last row or beside the matrix"
    status_ok()


@pytest.mark.parametrize("kernel,tile", [(1, 16), (1, 32), (1, 64), (1, 128), (2, 128), (2, 256), (0, 0)])
@pytest.mark.parametrize("sizes,N,K", [([3, 0, 130, 257, 1], 264, 400), ([700, 0, 300], 515, 130), ([0, 0], 64, 64)])
def test_every_kernel_takes_an_index(cuda_lib, kernel, tile, sizes, N, K):
    """Quantise + product with indexed rows, in each kernel.  Entries that name no token give NaN rows; unused rows are left
    alone."""
    import ctypes as C
    E, T, total = len(sizes), 41, sum(sizes)
    x = tokens(T, K, BF16, seed=1)
    w, ws = weights((E, N), K, seed=2)
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = torch.randint(0, T, (total + 9,), device="cuda", generator=g, dtype=torch.int32)
    if total:
        rows[2], rows[total - 1] = T, -1
    offsets = torch.tensor(sizes, device="cuda").cumsum(0).to(torch.int32)
    out = torch.full((total + 9, N), 3.0, dtype=torch.float32, device="cuda")
    pitch = -(-K // 16) * 16
    a = L.Int8Args(L.OUT_BF16, L.OUT_F32, E, 0, total + 9, T, N, K, x.data_ptr(), x.stride(0), rows.data_ptr(), None, pitch, None, w.data_ptr(),
                   w.stride(1), w.stride(0), ws.data_ptr(), None, offsets.data_ptr(), out.data_ptr(), N, kernel, tile)
    held = C.c_int64()
    L.check(L.load().bsg_int8_scratch_rows(C.byref(a), C.byref(held)))
    assert held.value == total + 9
    q, s = torch.empty((held.value, pitch), dtype=torch.int8, device="cuda"), torch.empty(held.value, device="cuda")
    a.Q, a.q_scale = q.data_ptr(), s.data_ptr()
    workspace = torch.zeros(16, dtype=torch.uint8, device="cuda")
    L.check(L.load().bsg_int8_linear_run(C.byref(a), workspace.data_ptr(), 16, torch.cuda.current_stream().cuda_stream))
    L.check(L.load().bsg_read_device_status(workspace.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert bool((out[total:] == 3).all())
    if not total:
        return
    for bad in (2, total - 1):
        assert bool(torch.isnan(out[bad]).all())
    out[2] = out[total - 1] = 0
    begin = 0
    for e, n in enumerate(sizes):
        part = [i for i in range(begin, begin + n) if i not in (2, total - 1)]
        if part:
            check(out[part], x[rows[part].long()], w[e], ws[e])
        begin += n


def test_tokens_that_many_rows_use(cuda_lib):
    """Enough rows per token that they are quantised once and copied; the result is that of rows given one by one."""
    E, T, N, K, per = 5, 600, 72, 3001, 11
    x = tokens(T, K, F16, seed=1)
    w, ws = weights((E, N), K, seed=2)
    ws = ws * 0.01
    total = T * per
    rows = torch.randperm(total, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).to(torch.int32) % T
    rows[7], rows[total - 3] = -5, T
    offsets = torch.tensor([1000, 1000, 4000, 6100, total - 20], dtype=torch.int32, device="cuda")
    buf = torch.full((total, N), 3.0, dtype=F16, device="cuda")
    out = ops.int8_linear(x, w, ws, offsets=offsets, rows=rows, out=buf)
    safe = rows.long().clamp(0, T - 1)
    want = ops.int8_linear(x[safe], w, ws, offsets=offsets)
    used = torch.arange(total, device="cuda") < total - 20
    assert bool(torch.isnan(out[7]).all()) and bool((out[~used] == 3).all())
    used[7] = False
    assert torch.equal(out[used], want[used])
    check(out[6100:6400], x[safe[6100:6400]], w[4], ws[4])
    status_ok()


def test_grouped_without_an_index_and_through_the_operator(cuda_lib):
    sizes, N, K = [5, 0, 130, 9], 264, 144
    x = tokens(sum(sizes), K, BF16, seed=2)
    w, ws = weights((4, N), K, seed=3)
    offsets = torch.tensor(sizes, device="cuda").cumsum(0).to(torch.int32)
    out = ops.int8_linear(x, w, ws, offsets=offsets)
    A = ops.quantize_int8(x)
    B = ops.ScaledOperand(w.transpose(1, 2), ws, (1, 1, K), ops.ScaleSwizzleMode.SwizzleNone)
    again = torch.empty_like(out)
    args = ops.GroupedGemmArguments(A, B, again, torch.int32, offsets=offsets)
    op = ops.get_operators(args)[0]
    assert op.metadata.grouped
    op.run(args)
    op.check_device_status()
    assert torch.equal(out, again)
    begin = 0
    for e, n in enumerate(sizes):
        if n:
            check(out[begin:begin + n], x[begin:begin + n], w[e], ws[e])
        begin += n


def test_bad_end_rows_are_reported_and_stay_inside(cuda_lib):
    x = tokens(20, 64, BF16, seed=2)
    w, ws = weights((3, 32), 64, seed=3)
    buf = torch.full((30, 32), 9.0, dtype=BF16, device="cuda")
    for bad in ([5, 3, 20], [5, 9, 25], [-4, 3, 20]):
        ops.int8_linear(x, w, ws, offsets=torch.tensor(bad, dtype=torch.int32, device="cuda"), out=buf[:20])
        with pytest.raises(L.BsgError):
            status_ok()
    assert bool((buf[20:] == 9).all())


# --------------------------------------------------------------------------------------------- streams, graphs, devices
def test_other_stream_and_captured_calls(cuda_lib):
    """Two captured graphs and an eager call between them; replays follow their inputs; scratch is not shared."""
    M, N, K = 6, 300, 500
    w, ws = weights((N,), K, seed=1)
    xs = [tokens(M, K, BF16, seed=i) for i in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = ops.int8_linear(xs[0], w, ws, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    check(y, xs[0], w, ws)
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.int8_linear(xs[i], w, ws))
        graphs.append(g)
    for rnd in range(2):
        for i in range(2):
            xs[i].copy_(tokens(M, K, BF16, seed=10 + 2 * rnd + i))
        graphs[0].replay()
        check(ops.int8_linear(xs[1], w, ws), xs[1], w, ws)
        graphs[1].replay()
        for i in range(2):
            check(outs[i], xs[i], w, ws)


def test_empty_inputs(cuda_lib):
    w, ws = weights((8,), 16, seed=0)
    assert ops.int8_linear(torch.empty((0, 16), dtype=BF16, device="cuda"), w, ws).shape == (0, 8)
    assert ops.quantize_int8(torch.empty((0, 16), dtype=BF16, device="cuda")).quantized.tensor.shape == (0, 16)


@pytest.mark.parametrize("exponent", [-126, -110, -72, -71, -70, 56, 57, 58, 100, 117, 118, 119, 120])
def test_halves_round_outwards_at_the_ends_of_the_range(cuda_lib, exponent):
    """Every mantissa of the maximum, the rows scaled to where a reciprocal or a level factor leaves fp32's normal range or a row is
    scaled on its way, against values on and next to each half."""
    amax = (torch.arange(128, 256, device="cuda").double() * 2.0 ** exponent).to(BF16)
    half = (torch.arange(127, device="cuda").double() + 0.5)[None] * amax.double()[:, None] / 127.0
    near = half.to(BF16)
    bits = near.view(torch.int16)
    x = torch.cat([amax[:, None], near, (bits - 1).view(BF16), -(bits + 1).view(BF16), -near, amax[:, None] / 2], 1).clamp(-amax[:, None], amax[:, None]).contiguous()
    q, s = levels(x)
    r = ops.quantize_int8(x)
    assert torch.equal(r.quantized.tensor.double(), q) and torch.equal(r.scale.tensor, s.float())
    for rows in (1, 3):
        for i in range(0, 128, 17):
            few = x[i:i + rows].contiguous()
            eye = torch.zeros((16, 512), dtype=torch.int8, device="cuda")[:, :few.shape[1]]
            eye[torch.arange(16), torch.arange(16) * 31] = 1
            got = ops.int8_linear(few, eye, torch.full((16,), 2.0 ** 100 if exponent < 0 else 2.0 ** -100, device="cuda"), out_dtype=F32)
            n = few.shape[0]
            want = q[i:i + n, torch.arange(16, device="cuda") * 31] * s[i:i + n].float().double()[:, None]
            tol = 3 * 2.0 ** -24 * want.abs() + 2.0 ** -149 * 0.5
            assert bool(((got.double() * (2.0 ** -100 if exponent < 0 else 2.0 ** 100) - want).abs() <= tol).all())


@pytest.mark.parametrize("M", [1, 2, 4, 5, 300])
def test_results_in_the_place_of_the_tokens(cuda_lib, M):
    """``out`` is ``x`` itself, or its columns further on; columns beside those of x in one buffer are no overlap."""
    K = 2048
    w, ws = weights((K,), K, seed=1)
    ws = ws / math.sqrt(K)
    x = tokens(M, K, BF16, seed=M)
    want = ops.int8_linear(x, w, ws)
    for _ in range(5):
        for shift in (0, 3, 8, K):
            buf = torch.zeros((M, 2 * K), dtype=BF16, device="cuda")
            buf[:, :K] = x
            ops.int8_linear(buf[:, :K], w, ws, out=buf[:, shift:shift + K])
            assert torch.equal(buf[:, shift:shift + K], want)
            if shift == K:
                assert torch.equal(buf[:, :K], x)
