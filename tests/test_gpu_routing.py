"""The router on the GPU against its definition in 64 bits."""
import math

import pytest
import torch

import cutlass_b200 as ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def route64(logits, k, mask, normalize):
    """Everything ``route_tokens`` returns, in 64 bits on the CPU, by loops over tokens where the order matters."""
    l = logits.double().cpu()
    T, E = l.shape
    counted = [bool((l[t] != -math.inf).any()) and (mask is None or bool(mask[t])) for t in range(T)]
    experts = torch.full((T, k), -1, dtype=torch.int64)
    p = torch.zeros((T, E), dtype=torch.float64)
    for t in range(T):
        if not counted[t]:
            continue
        row = l[t].tolist()
        p[t] = torch.softmax(l[t], 0)
        order = sorted(range(E), key=lambda e: (0 if row[e] != row[e] else 1, 0.0 if row[e] != row[e] else -row[e], e))
        chosen = [e for e in order if row[e] != -math.inf][:k]
        experts[t, :len(chosen)] = torch.tensor(chosen)
    live = experts >= 0
    w = torch.where(live, p.gather(1, experts.clamp_min(0)), 0.0)
    if normalize:
        w = torch.where(live, w / torch.where(live.any(1, keepdim=True), w.sum(1, keepdim=True), 1.0), 0.0)
    counts = torch.bincount(experts[live], minlength=E)
    offsets = counts.cumsum(0)
    at = (offsets - counts).tolist()
    rows = torch.full((T * k,), -1, dtype=torch.int64)
    positions = torch.full((T, k), -1, dtype=torch.int64)
    for t in range(T):
        for j in range(k):
            e = int(experts[t, j])
            if e >= 0:
                positions[t, j] = at[e]
                rows[at[e]] = t
                at[e] += 1
    n = max(sum(counted), 1)
    loss = E * ((counts.double() / (n * k)) * p.sum(0) / n).sum()
    return dict(experts=experts, weights=w, counts=counts, offsets=offsets, rows=rows, positions=positions, loss=loss, p=p, n=sum(counted), live=live)


def grad64(r, k, normalize, gw, gl):
    p, live, E = r["p"], r["live"], r["p"].shape[1]
    n = max(r["n"], 1)
    f = r["counts"].double() / (n * k)
    gw = torch.where(live, gw.double().cpu(), 0.0)
    d = float(gl) * E / n * p * (f - (p * f).sum(1, keepdim=True))
    w = r["weights"]
    part = w * (gw - (w * gw).sum(1, keepdim=True)) if normalize else w * gw
    if not normalize:
        d = d - p * part.sum(1, keepdim=True)
    return d.scatter_add(1, r["experts"].clamp_min(0), torch.where(live, part, 0.0)), gw


def make(T, E, dtype, seed, masked=0.0, padded=0.0, pitch=None, coarse=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = 2 * torch.randn((T, E), device="cuda", generator=g)
    if coarse:
        l = torch.round(l)              # many equal logits: ties
    l[torch.rand((T, E), device="cuda", generator=g) < masked] = -math.inf
    buf = torch.zeros((T, pitch or E), dtype=dtype, device="cuda")
    buf[:, :E] = l.to(dtype)
    mask = torch.rand(T, device="cuda", generator=g) >= padded if padded else None
    return buf[:, :E], mask


def check(logits, k, mask, normalize, r):
    """Whole numbers are equal.  A probability: the difference l - max is exact or rounded (2^-24 of at most 40 here: 2^-18.6
    relative after exp), exp 2 units, the sum of at most 1024 positive terms 2^-23 more by pairs of 5 + V steps, quotient and
    product one unit each: under 2^-18 in all, twice for a normalised weight.  The loss adds sums over tokens: 2^-16."""
    want = route64(logits, k, mask, normalize)
    assert torch.equal(r.experts.cpu().long(), want["experts"])
    for name in ("counts", "offsets", "rows", "positions"):
        assert torch.equal(getattr(r, name).cpu().long(), want[name]), name
    assert int(r.num_tokens) == want["n"]
    nan = torch.isnan(want["weights"])
    got = r.weights.cpu().double()
    assert torch.equal(torch.isnan(got), nan)
    err = (got - want["weights"]).abs() - 2.0 ** -17 * want["weights"]
    assert float(torch.where(nan, 0.0, err).max() if err.numel() else 0.0) <= 1e-37
    if math.isnan(float(want["loss"])):
        assert math.isnan(float(r.balance_loss))
    else:
        assert abs(float(r.balance_loss) - float(want["loss"])) <= 2.0 ** -16 * float(want["loss"])
    return want


def check_grad(got, want, k, normalize, gw, gl, dtype):
    """Every term of the gradient is a product of at most four factors off by 2^-17 each; what is subtracted is bounded by the
    sums of the magnitudes; then half a step of the type."""
    ref, gwl = grad64(want, k, normalize, gw, gl)
    p, w, E = want["p"], want["weights"], want["p"].shape[1]
    n = max(want["n"], 1)
    f = want["counts"].double() / (n * k)
    size = abs(float(gl)) * E / n * p * (f + (p * f).sum(1, keepdim=True))
    s2 = (w * gwl.abs()).sum(1, keepdim=True)
    part = w * (gwl.abs() + s2) if normalize else w * gwl.abs()
    size = size + (0 if normalize else p * s2)
    size = size.scatter_add(1, want["experts"].clamp_min(0), torch.where(want["live"], part, 0.0))
    tol = 4 * 2.0 ** -17 * size
    info = torch.finfo(dtype)
    tol = tol + info.eps / 2 * (ref.abs() + tol) + info.smallest_normal * info.eps
    nan = torch.isnan(ref)
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), nan)
    err = torch.where(nan, -torch.ones_like(ref), (got - ref).abs() - tol)
    assert float(err.max()) <= 0, f"{int((err > 0).sum())} of {err.numel()} gradients off, worst by {float(err.max())}"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,E,k,masked,padded,pitch", [
    (1, 1, 1, 0, 0, None), (1, 8, 2, 0, 0, None), (5, 3, 3, 0.3, 0, None), (16, 64, 2, 0, 0, None), (33, 32, 32, 0.5, 0.2, None),
    (70, 33, 4, 0, 0.5, 40), (257, 160, 6, 0.1, 0.2, None), (300, 256, 8, 0, 0, 264), (129, 257, 3, 0.9, 0, None), (64, 513, 8, 0, 0, None),
    (40, 1024, 8, 0.97, 0, None), (1000, 60, 8, 0.05, 0.1, 61), (2500, 17, 2, 0, 0.3, None),
    (512, 16, 4, 0, 0, None), (513, 513, 8, 0.2, 0.1, None), (1100, 160, 6, 0.1, 0.2, 168), (540, 257, 32, 0.5, 0, None), (136, 1000, 2, 0, 0.1, None),
    (16, 300, 5, 0.1, 0.2, None), (17, 300, 5, 0.1, 0.2, None),
    (60, 200, 12, 0.1, 0, None), (700, 128, 7, 0.9, 0.1, None), (90, 256, 32, 0.8, 0, None)])
def test_routing_and_its_gradient(cuda_lib, T, E, k, masked, padded, pitch, normalize, dtype):
    logits, mask = make(T, E, dtype, seed=T + E, masked=masked, padded=padded, pitch=pitch)
    r = ops.route_tokens(logits, k, token_mask=mask, normalize=normalize)
    want = check(logits, k, mask, normalize, r)
    gw, gl = torch.randn((T, k), device="cuda"), torch.tensor(0.7, device="cuda")
    check_grad(ops.route_tokens_backward(logits, r, gw, gl), want, k, normalize, gw, gl, dtype)
    check_grad(ops.route_tokens_backward(logits, r, gw, None), want, k, normalize, gw, 0.0, dtype)
    check_grad(ops.route_tokens_backward(logits, r, None, gl), want, k, normalize, torch.zeros_like(gw), gl, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_ties_go_to_the_lower_index(cuda_lib, dtype):
    logits, _ = make(500, 100, dtype, seed=1, coarse=True)
    logits[0] = 0
    logits[1, ::2] = -0.0
    logits[1, 1::2] = 0.0
    logits[2] = torch.finfo(dtype).min
    logits[3] = torch.finfo(dtype).max
    check(logits, 8, None, True, ops.route_tokens(logits, 8))


@pytest.mark.parametrize("normalize", [True, False])
def test_rows_without_anything_to_choose_and_values_that_are_not_numbers(cuda_lib, normalize):
    logits, mask = make(40, 20, F32, seed=2, masked=0.2, padded=0.2)
    logits[3] = -math.inf
    logits[4, 1:] = -math.inf
    mask[3] = mask[4] = True
    r = ops.route_tokens(logits, 4, token_mask=mask, normalize=normalize)
    want = check(logits, 4, mask, normalize, r)
    gw, gl = torch.randn((40, 4), device="cuda"), torch.tensor(1.0, device="cuda")
    check_grad(ops.route_tokens_backward(logits, r, gw, gl), want, 4, normalize, gw, gl, F32)
    logits[7, 5] = math.nan
    logits[8, 2], logits[8, 9] = math.inf, math.nan
    mask[7] = mask[8] = True
    r = ops.route_tokens(logits, 4, token_mask=mask, normalize=normalize)
    check(logits, 4, mask, normalize, r)
    assert r.experts[7, 0] == 5 and r.experts[8, 0] == 9 and r.experts[8, 1] == 2
    d = ops.route_tokens_backward(logits, r, gw, None)
    finite = [t for t in range(40) if t not in (7, 8)]
    assert bool(torch.isfinite(d[finite]).all()) and bool(torch.isnan(d[7]).any()) and bool(torch.isnan(d[8]).any())


def test_nobody_counts(cuda_lib):
    logits, _ = make(10, 6, BF16, seed=3)
    none = torch.zeros(10, dtype=torch.bool, device="cuda")
    for l, m in ((logits, none), (logits[:0], None), (torch.full_like(logits, -math.inf), None)):
        r = ops.route_tokens(l, 2, token_mask=m)
        assert int(r.num_tokens) == 0 and float(r.balance_loss) == 0.0 and not r.counts.any() and not r.offsets.any()
        assert bool((r.experts == -1).all()) and bool((r.rows == -1).all()) and bool((r.positions == -1).all()) and not r.weights.any()
        d = ops.route_tokens_backward(l, r, torch.ones_like(r.weights), torch.tensor(1.0, device="cuda"))
        assert d.shape == l.shape and not d.any()


@pytest.mark.parametrize("normalize", [True, False])
def test_autograd_and_differences(cuda_lib, normalize):
    """Autograd gives the functional gradient; both agree with central differences of the definition in 64 bits (the choice and
    the counts held fixed), whose own error is below 1e-7 here."""
    T, E, k = 12, 9, 3
    logits, mask = make(T, E, F32, seed=5, padded=0.2)
    leaf = logits.clone().requires_grad_()
    r = ops.route_tokens(leaf, k, token_mask=mask, normalize=normalize)
    gw = torch.randn((T, k), device="cuda")
    ((r.weights * gw).sum() + 3 * r.balance_loss).backward()
    plain = ops.route_tokens(logits, k, token_mask=mask, normalize=normalize)
    assert torch.equal(leaf.grad, ops.route_tokens_backward(logits, plain, gw, torch.tensor(3.0, device="cuda")))
    assert not plain.weights.requires_grad and not r.counts.requires_grad
    w64 = route64(logits, k, mask, normalize)
    n, f = w64["n"], w64["counts"].double() / (w64["n"] * k)
    keep = w64["live"].any(1)

    def value(l):
        p = torch.softmax(l, 1) * keep[:, None]
        w = torch.where(w64["live"], p.gather(1, w64["experts"].clamp_min(0)), 0.0)
        if normalize:
            w = torch.where(w64["live"], w / w.sum(1, keepdim=True), 0.0)
        return (w * gw.double().cpu()).sum() + 3 * E * (f * p.sum(0) / n).sum()

    l64, eps = logits.double().cpu(), 1e-5
    for t in range(T):
        for e in range(E):
            up, down = l64.clone(), l64.clone()
            up[t, e] += eps
            down[t, e] -= eps
            assert abs(float((value(up) - value(down)) / (2 * eps)) - float(leaf.grad[t, e])) < 1e-4 * (1 + abs(float(leaf.grad[t, e])))
    # one of the two results alone; and a loss that is changed in place
    leaf.grad = None
    loss = ops.route_tokens(leaf, k, token_mask=mask, normalize=normalize).balance_loss
    loss += 1
    loss.backward()
    assert torch.equal(leaf.grad, ops.route_tokens_backward(logits, plain, None, torch.tensor(1.0, device="cuda")))


def test_runs_are_equal_and_large_batches_are_in_order(cuda_lib):
    """65 537 tokens over all blocks of the grid: rows sorted by expert and stable, positions their inverse; twice the same bits."""
    T, E, k = 65537, 256, 8
    logits, mask = make(T, E, BF16, seed=6, padded=0.1)
    a, b = (ops.route_tokens(logits, k, token_mask=mask) for _ in range(2))
    for x, y in zip(a[:8], b[:8]):
        assert torch.equal(x, y)
    ref = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(a.experts[mask].long(), ref[mask]) and bool((a.experts[~mask] == -1).all())
    flat = torch.where(mask[:, None], ref, E).reshape(-1)
    order = torch.sort(flat, stable=True).indices
    total = int(a.offsets[-1])
    assert total == int(mask.sum()) * k
    assert torch.equal(a.rows[:total].long(), order[:total] // k) and bool((a.rows[total:] == -1).all())
    pos = torch.empty_like(order).scatter_(0, order, torch.arange(T * k, device="cuda"))
    assert torch.equal(a.positions.reshape(-1)[flat < E].long(), pos[flat < E])
    p = torch.softmax(logits.double(), 1) * mask[:, None]
    n = int(mask.sum())
    loss = E * ((a.counts.double() / (n * k)) * p.sum(0) / n).sum()
    assert abs(float(a.balance_loss) - float(loss)) <= 2.0 ** -16 * float(loss)
    gw = torch.randn((T, k), device="cuda")
    gl = torch.tensor(0.5, device="cuda")
    x, y = (ops.route_tokens_backward(logits, a, gw, gl) for _ in range(2))
    assert torch.equal(x, y)


def test_streams_and_graphs(cuda_lib):
    logits, mask = make(100, 64, BF16, seed=7, padded=0.2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    r = ops.route_tokens(logits, 4, token_mask=mask, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    check(logits, 4, mask, True, r)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            q = ops.route_tokens(logits, 4 + i, token_mask=mask)
            d = ops.route_tokens_backward(logits, q, None, q.balance_loss)
        graphs.append((g, q, d, 4 + i))
    for seed in (8, 9):
        nl, nm = make(100, 64, BF16, seed=seed, padded=0.3)
        logits.copy_(nl)
        mask.copy_(nm)
        for g, *_ in graphs:
            g.replay()
        for _, q, d, k in graphs:
            want = check(logits, k, mask, True, q)
            check_grad(d, want, k, True, torch.zeros_like(q.weights), float(q.balance_loss), BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("E", [383, 384, 385, 767, 768, 769])
@pytest.mark.parametrize("T", [9, 100, 600])
def test_expert_counts_around_48_kilobytes_of_shared_memory(cuda_lib, T, E, dtype):
    """Static and dynamic shared memory count together: one block, a cluster and many blocks, on both sides of what needs no
    permission."""
    logits, mask = make(T, E, dtype, seed=E, masked=0.1, padded=0.1)
    r = ops.route_tokens(logits, 8, token_mask=mask)
    want = check(logits, 8, mask, True, r)
    gw, gl = torch.randn((T, 8), device="cuda"), torch.tensor(0.7, device="cuda")
    check_grad(ops.route_tokens_backward(logits, r, gw, gl), want, 8, True, gw, gl, dtype)


def test_as_many_tokens_as_31_bits_count(cuda_lib):
    """2^31 - 1 tokens, the largest number that is taken: all but the last 300 have equal logits and choose the first expert."""
    T, n = (1 << 31) - 1, 300
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 110 << 30:
        pytest.skip("needs 110 GiB of device memory")
    logits = torch.zeros((T, 2), dtype=BF16, device="cuda")
    logits[-n:], _ = make(n, 2, BF16, seed=11)
    tail = logits[-n:].double().cpu()
    pick = (tail[:, 1] > tail[:, 0]).long()
    r = ops.route_tokens(logits, 1, normalize=False)
    second = int(pick.sum())
    assert r.counts.tolist() == [T - second, second] and r.offsets.tolist() == [T - second, T] and int(r.num_tokens) == T
    step = 1 << 28
    for lo in range(0, T - n, step):
        hi = min(lo + step, T - n)
        at = torch.arange(lo, hi, dtype=torch.int32, device="cuda")
        assert not bool(r.experts[lo:hi].any()) and bool((r.weights[lo:hi] == 0.5).all())
        assert torch.equal(r.rows[lo:hi], at) and torch.equal(r.positions[lo:hi, 0], at)
    token = torch.arange(T - n, T)
    assert torch.equal(r.experts[-n:, 0].cpu().long(), pick)
    assert torch.equal(r.rows[T - n:].cpu().long(), torch.cat([token[pick == 0], token[pick == 1]]))
    place = torch.where(pick == 0, T - n + (pick == 0).long().cumsum(0) - 1, T - second + pick.cumsum(0) - 1)
    assert torch.equal(r.positions[-n:, 0].cpu().long(), place)
    p = torch.softmax(tail, 1)
    w = p.gather(1, pick[:, None])
    assert bool(((r.weights[-n:].cpu().double() - w).abs() <= 2.0 ** -17 * w).all())
    want = 2 * ((T - second) / T * (0.5 * (T - n) + float(p[:, 0].sum())) / T + second / T * (0.5 * (T - n) + float(p[:, 1].sum())) / T)
    assert abs(float(r.balance_loss) - want) <= 2.0 ** -16 * want
    gw = torch.zeros((T, 1), device="cuda")
    gw[-n:] = torch.randn((n, 1), device="cuda")
    d = ops.route_tokens_backward(logits, r, gw, None)
    for lo in range(0, T - n, step):
        assert not bool(d[lo:min(lo + step, T - n)].any())
    part = w * gw[-n:].cpu().double()
    ref = torch.zeros_like(p).scatter_(1, pick[:, None], part) - p * part
    size = torch.zeros_like(p).scatter_(1, pick[:, None], part.abs()) + p * part.abs()
    tol = 4 * 2.0 ** -17 * size
    tol = tol + torch.finfo(BF16).eps / 2 * (ref.abs() + tol)
    assert bool(((d[-n:].cpu().double() - ref).abs() <= tol).all())
    del logits, r, gw, d
    torch.cuda.empty_cache()
