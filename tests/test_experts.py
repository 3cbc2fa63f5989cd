"""The experts' operators: the sort equal to a stable sort, gather exact, sums and products within the
bounds that 32-bit arithmetic and one rounding to the output's type allow (those of test_mxfp4 for the
products; a combine adds top terms in 32 bits, each fused product-sum off by at most 2^-23 of the sum
of magnitudes)."""

import numpy as np
import pytest
import torch

import xpu_kernels as xk
from oracle import convrot_oracle as O
from oracle import mxfp4_oracle as X

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALL = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}


def rand(shape, seed, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def f64(t):
    return t.detach().cpu().double().numpy()


def turned(x):
    return torch.from_numpy(O.rotate_groups(x.float().numpy())).to(x.dtype)


def routing(tokens, top, experts, seed, dropped=0.0, used=None):
    """ids [tokens, top], a token's experts different, some slots of no expert; only the experts in `used`."""
    rng = np.random.default_rng(seed)
    pool = np.arange(experts) if used is None else np.asarray(used)
    ids = np.stack([rng.permutation(pool)[:top] for _ in range(tokens)]) if tokens else np.zeros((0, top))
    ids = ids.astype(np.int64)
    bad = rng.random(ids.shape) < dropped
    ids[bad] = rng.choice([-1, experts, -5, 2 ** 31 - 1], bad.sum()) if bad.any() else 0
    return ids


def check(got, ref, spread, terms, dtype, extra=0.0):
    bound = terms * 2.0 ** -23 * spread + ROUND[dtype] * (np.abs(ref) + spread * 2.0 ** -20) + SMALL[dtype] + extra
    off = np.abs(f64(got) - ref) - bound
    assert off.shape == ref.shape
    assert (off <= 0).all(), f"{(off > 0).sum()} of {off.size} past the bound, by {off.max()}"


@pytest.fixture(scope="module")
def gpu():
    from xpu_kernels.int8 import _lib as L
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device")
    if not xk.available():
        pytest.fail(f"libxpuint8 did not load: {L._ERR}")
    yield
    torch.cuda.synchronize()
    assert L.load().xpuint8_fault_status(1) == 0


# -------------------------------------------------------------------------------------------- sort

@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,top,experts,dropped", [
    (1, 1, 1, 0), (1, 8, 64, 0), (3, 2, 5, 0.5), (100, 3, 7, 0), (1000, 4, 1024, 0.1), (1024, 4, 16, 0),
    (1025, 4, 16, 0.05), (4097, 1, 3, 0.2), (20000, 8, 128, 0.05), (70000, 2, 300, 0), (50, 2, 4, 1.0)])
def test_sort(gpu, tokens, top, experts, dropped, kind):
    ids = routing(tokens, top, experts, tokens + top, dropped)
    plan = xk.expert_sort(torch.from_numpy(ids).to(kind).to(DEV), experts)
    order, positions, offsets, scale_rows, tiles = X.sort(ids, experts)
    for got, want in ((plan.order, order), (plan.positions, positions), (plan.offsets, offsets),
                      (plan.scale_rows, scale_rows), (plan.tiles, tiles)):
        assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), want)
    assert plan.tokens == tokens and plan.top == top and plan.rows == tokens * top
    assert tiles[-1] <= plan.max_tiles


@pytest.mark.gpu
def test_sort_of_ids_past_32_bits_and_of_none(gpu):
    ids = np.array([[2 ** 40, 1], [-2 ** 40, 0], [1, 2 ** 32]], dtype=np.int64)  # 2^32 is not expert 0
    plan = xk.expert_sort(torch.from_numpy(ids).to(DEV), 2)
    assert plan.offsets.tolist() == [0, 1, 3] and plan.order.tolist() == [3, 1, 4, 0, 2, 5]
    none = xk.expert_sort(torch.zeros((0, 2), dtype=torch.int64, device=DEV), 3)
    assert none.offsets.tolist() == [0] * 4 and none.tiles.tolist() == [0] * 4 and none.rows == 0
    one = xk.expert_sort(torch.tensor([1, 0, 1], device=DEV), 2)
    assert one.positions.tolist() == [[1], [0], [2]]


# --------------------------------------------------------------------------------- gather, combine

MOVES = [(1, 1, 1, 1, 0), (1, 8, 64, 4096, 0), (5, 2, 3, 33, 0.3), (300, 3, 7, 136, 0.1), (2000, 9, 40, 250, 0.05), (64, 2, 4, 2056, 1.0),
         (200, 3, 7, 300, 0.1), (33, 2, 4, 1028, 0.2), (50, 5, 9, 2050, 0.1), (50, 10, 12, 4097, 0.1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top,experts,width,dropped", MOVES)
def test_gather_and_combine(gpu, tokens, top, experts, width, dropped, dtype):
    ids = routing(tokens, top, experts, 3, dropped)
    plan = xk.expert_sort(torch.from_numpy(ids).to(DEV), experts)
    x, y = rand((tokens, width), 1, dtype), rand((tokens * top, width), 2, dtype)
    w = torch.softmax(rand((tokens, top), 4, torch.float32), -1)
    dx, dy = rand((tokens * top, width), 5, dtype), rand((tokens, width), 6, dtype)
    xd, yd, wd = (v.to(DEV).requires_grad_() for v in (x, y, w))
    rows, out = xk.expert_gather(xd, plan), xk.expert_combine(yd, wd, plan)
    assert np.array_equal(f64(rows), X.gather(f64(x), ids, experts))
    check(out, X.combine(f64(y), f64(w), ids, experts), X.combine(np.abs(f64(y)), f64(w), ids, experts), top + 1, dtype)
    gx, gy, gw = torch.autograd.grad((rows, out), (xd, yd, wd), (dx.to(DEV), dy.to(DEV)))
    ones = np.ones((tokens, top))
    check(gx, X.combine(f64(dx), ones, ids, experts), X.combine(np.abs(f64(dx)), ones, ids, experts), top + 1, dtype)
    want_y, want_w = X.combine_grad(f64(dy), f64(y), f64(w), ids, experts)
    check(gy, want_y, np.abs(want_y), 1, dtype)
    _, spread = X.combine_grad(np.abs(f64(dy)), np.abs(f64(y)), f64(w), ids, experts)
    check(gw, want_w, spread, width, torch.float32)


@pytest.mark.gpu
def test_gradients_against_differences(gpu):
    """Gather and combine are linear in each argument: a difference quotient with whole numbers is
    exact."""
    ids = routing(30, 3, 5, 1, 0.2)
    plan = xk.expert_sort(torch.from_numpy(ids).to(DEV), 5)
    g = torch.Generator().manual_seed(2)
    draw = lambda *s: torch.randint(-4, 5, s, generator=g).float().to(DEV)  # noqa: E731
    x, y, w, dx, dy = draw(30, 16), draw(90, 16), draw(30, 3), draw(90, 16), draw(30, 16)
    for v in (x, y, w):
        v.requires_grad_()
    gx, gy, gw = torch.autograd.grad((xk.expert_gather(x, plan), xk.expert_combine(y, w, plan)), (x, y, w), (dx, dy))
    gather = lambda x: float((xk.expert_gather(x.detach(), plan) * dx).sum())  # noqa: E731
    combine = lambda y, w: float((xk.expert_combine(y.detach(), w.detach(), plan) * dy).sum())  # noqa: E731
    u, v, t = draw(30, 16), draw(90, 16), draw(30, 3)
    assert (gather(x + u) - gather(x - u)) / 2 == float((gx * u).sum())
    assert (combine(y + v, w) - combine(y - v, w)) / 2 == float((gy * v).sum())
    assert (combine(y, w + t) - combine(y, w - t)) / 2 == float((gw * t).sum())


@pytest.mark.gpu
def test_rows_of_no_expert_are_not_read(gpu):
    ids = torch.tensor([[0, -1], [1, 9]], device=DEV)
    plan = xk.expert_sort(ids, 2)
    y = torch.ones((4, 64), device=DEV)
    y[2:] = float("nan")
    y.requires_grad_()
    w = torch.full((2, 2), 0.5, device=DEV, requires_grad=True)
    out = xk.expert_combine(y, w, plan)
    gy, gw = torch.autograd.grad(out, (y, w), torch.ones_like(out))
    assert torch.equal(out, torch.full_like(out, 0.5))
    assert torch.equal(gy[2:], torch.zeros_like(gy[2:])) and gw[:, 1].tolist() == [0, 0] and gw[:, 0].tolist() == [64, 64]
    x = torch.full((2, 64), float("inf"), device=DEV)
    assert torch.equal(xk.expert_gather(x, plan)[2:], torch.zeros((2, 64), device=DEV))


@pytest.mark.gpu
def test_strides_types_of_weights_and_alignments(gpu):
    ids = routing(40, 2, 6, 1, 0.1)
    plan = xk.expert_sort(torch.from_numpy(ids).to(DEV), 6)
    base, rows = rand((40, 300), 1).to(DEV), rand((80, 300), 2).to(DEV)
    w = torch.softmax(rand((40, 2), 3, torch.float32), -1).to(DEV)
    for cut in (slice(0, 256), slice(1, 257), slice(8, 200), slice(0, 300, 2)):
        x, y = base[:, cut], rows[:, cut]
        assert torch.equal(xk.expert_gather(x, plan), xk.expert_gather(x.contiguous(), plan))
        assert torch.equal(xk.expert_combine(y, w, plan), xk.expert_combine(y.contiguous(), w, plan))
    wide = torch.zeros((40, 4), device=DEV)
    wide[:, ::2] = w
    assert torch.equal(xk.expert_combine(rows, wide[:, ::2], plan), xk.expert_combine(rows, w, plan))
    half = w.to(torch.bfloat16).requires_grad_()
    out = xk.expert_combine(rows, half, plan)
    assert torch.equal(out, xk.expert_combine(rows, half.detach().float(), plan))
    out.sum().backward()
    assert half.grad.dtype == torch.bfloat16


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    tokens, width = 9, 256 * 1024 * 1024  # 2.4e9 values
    x = torch.empty((tokens, width), dtype=torch.bfloat16, device=DEV)
    for t in range(tokens):
        x[t] = t + 1
    plan = xk.expert_sort(torch.arange(tokens - 1, -1, -1, device=DEV), tokens)
    rows = xk.expert_gather(x, plan)
    assert rows[:, 0].tolist() == list(range(tokens, 0, -1)) and rows[:, -1].tolist() == list(range(tokens, 0, -1))
    back = xk.expert_combine(rows, torch.ones((tokens, 1), device=DEV), plan)
    assert back[:, -1].tolist() == list(range(1, tokens + 1))


@pytest.mark.gpu
def test_weights_are_by_token_and_choice(gpu):
    plan = xk.expert_sort(torch.zeros((4, 2), dtype=torch.int32, device=DEV), 4)
    y, w = rand((8, 64), 1).to(DEV), rand((4, 2), 2, torch.float32).to(DEV)
    want = xk.expert_combine(y, w, plan)
    assert torch.equal(xk.expert_combine(y, w.reshape(8), plan), want)  # a value a slot
    for wrong in (w.T, w.T.contiguous(), w.reshape(1, 8), w.reshape(8, 1), w.reshape(2, 2, 2)):
        with pytest.raises(ValueError, match=r"weights must be \[4, 2\]"):
            xk.expert_combine(y, wrong, plan)
    one = xk.expert_sort(torch.zeros(8, dtype=torch.int32, device=DEV), 4)
    assert torch.equal(xk.expert_combine(y, w.reshape(8), one), xk.expert_combine(y, w.reshape(8, 1), one))


# --------------------------------------------------------------------------- the experts' product

#: tokens, top, experts, N, K, dropped, the experts that are chosen from (None: all)
PRODUCTS = [(1, 1, 1, 1, 1, 0, None), (1, 2, 4, 128, 256, 0, None), (7, 3, 9, 77, 100, 0.2, None), (16, 4, 64, 256, 512, 0, None),
            (300, 2, 3, 130, 333, 0.1, None), (600, 1, 4, 272, 256, 0, [2]), (1000, 2, 5, 520, 300, 0.05, [0, 1, 4]), (64, 2, 4, 96, 64, 1.0, None)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("in_order", [False, True])
@pytest.mark.parametrize("tokens,top,experts,n,k,dropped,used", PRODUCTS)
def test_expert_product(gpu, tokens, top, experts, n, k, dropped, used, in_order, dtype):
    top = min(top, len(used)) if used else top
    ids = routing(tokens, top, experts, 7, dropped, used)
    plan = xk.expert_sort(torch.from_numpy(ids).to(DEV), experts)
    order, _, offsets, _, _ = X.sort(ids, experts)
    x = rand((tokens * top if in_order else tokens, k), 1, dtype)
    w = rand((experts, n, k), 2, dtype)
    rotate = k % 256 == 0
    got = xk.expert_linear_mxfp4(x.to(DEV), xk.prepare_weight_mxfp4(w.to(DEV), rotate=rotate), plan, rotate=rotate, sorted=in_order)
    t = turned if rotate else (lambda v: v)
    xq = X.rounded(f64(t(x)))
    xq = xq if in_order else xq[order // top]
    ref, spread = np.zeros((tokens * top, n)), np.zeros((tokens * top, n))
    for e in range(experts):
        rows = slice(offsets[e], offsets[e + 1])
        ref[rows], spread[rows] = X.product(xq[rows], X.rounded(f64(t(w[e]))))
    assert got.dtype == dtype
    check(got, ref, spread, k / 64 + 10, dtype)
    assert not f64(got)[offsets[-1]:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("in_order", [False, True])
@pytest.mark.parametrize("tokens,top,experts,n,k,dropped,used", PRODUCTS)
def test_expert_gradients(gpu, tokens, top, experts, n, k, dropped, used, in_order, dtype):
    top = min(top, len(used)) if used else top
    ids = routing(tokens, top, experts, 8, dropped, used)
    plan = xk.expert_sort(torch.from_numpy(ids).to(DEV), experts)
    order, _, offsets, _, _ = X.sort(ids, experts)
    rows_in = tokens * top if in_order else tokens
    x, w, dy = rand((rows_in, k), 1, dtype), rand((experts, n, k), 2, dtype), rand((tokens * top, n), 3, dtype)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = xk.mxfp4_expert_linear(xd, wd, plan, rotate=False, sorted=in_order)
    assert torch.equal(y, xk.expert_linear_mxfp4(xd, xk.prepare_weight_mxfp4(wd, rotate=False), plan, rotate=False, sorted=in_order))
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.to(DEV))
    assert dx.dtype == dw.dtype == dtype
    xs = f64(x) if in_order else f64(x)[order // top]
    d = f64(dy)
    gx, sx = np.zeros((tokens * top, k)), np.zeros((tokens * top, k))
    for e in range(experts):
        r = slice(offsets[e], offsets[e + 1])
        we = f64(w[e])
        gx[r], sx[r] = X.product(X.rounded(d[r]), X.rounded(we.T))
        if offsets[e] == offsets[e + 1]:
            assert not f64(dw[e]).any()
            continue
        ref, spread = X.product(X.rounded(d[r].T), X.rounded(xs[r].T))
        check(dw[e], ref, spread, (offsets[e + 1] - offsets[e]) / 64 + 10, dtype)
    if in_order:
        check(dx, gx, sx, n / 64 + 10, dtype)
    else:  # each row is rounded to the type, then a token's rows are added
        one = np.ones((tokens, top))
        extra = ROUND[dtype] * X.combine(np.abs(gx), one, ids, experts) + top * SMALL[dtype]
        check(dx, X.combine(gx, one, ids, experts), X.combine(sx, one, ids, experts), n / 64 + 10 + top, dtype, extra)


@pytest.mark.gpu
@pytest.mark.parametrize("in_order", [False, True])
def test_rotated_expert_gradients_are_the_plain_ones_turned(gpu, in_order):
    ids = routing(200, 2, 3, 8, 0.1)
    plan = xk.expert_sort(torch.from_numpy(ids).to(DEV), 3)
    x, w, dy = rand((400 if in_order else 200, 512), 1, torch.float32), rand((3, 96, 512), 2, torch.float32), rand((400, 96), 3, torch.float32)

    def grads(x, w, rotate):
        x, w = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        y = xk.mxfp4_expert_linear(x, w, plan, rotate=rotate, sorted=in_order)
        return (y, *torch.autograd.grad(y, (x, w), dy.to(DEV)))

    y, dx, dw = grads(x, w, True)
    py, pdx, pdw = grads(turned(x), turned(w), False)
    assert torch.equal(y, py)
    for got, plain in ((dx, pdx), (dw, pdw)):
        assert np.array_equal(f64(got), f64(turned(plain.cpu())))


@pytest.mark.gpu
@pytest.mark.parametrize("rotate", [False, True])
def test_one_gradient_alone_is_the_same(gpu, rotate):
    plan = xk.expert_sort(torch.from_numpy(routing(200, 2, 3, 8, 0.1)).to(DEV), 3)
    x, w, dy = rand((200, 256), 1).to(DEV), rand((3, 96, 256), 2).to(DEV), rand((400, 96), 3).to(DEV)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = xk.mxfp4_expert_linear(xg, wg, plan, rotate=rotate)
    dx, dw = torch.autograd.grad(y, (xg, wg), dy)
    assert torch.equal(torch.autograd.grad(xk.mxfp4_expert_linear(xg, w, plan, rotate=rotate), xg, dy)[0], dx)
    assert torch.equal(torch.autograd.grad(xk.mxfp4_expert_linear(x, wg, plan, rotate=rotate), wg, dy)[0], dw)
    with torch.no_grad():
        assert torch.equal(xk.mxfp4_expert_linear(xg, wg, plan, rotate=rotate), y)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,top", [(1, 1), (1, 4), (30, 4), (32, 4), (33, 4), (128, 1), (300, 2)])
def test_rows_quantised_in_the_product_are_the_quantiser_s(gpu, tokens, top):
    """Up to 128 rows are quantised inside the product, others before it: each row is its token's times
    its expert's weight, whichever it is."""
    ids = routing(tokens, top, 5, 3)
    plan = xk.expert_sort(torch.from_numpy(ids).to(DEV), 5)
    order, _, offsets, _, _ = X.sort(ids, 5)
    x, w = rand((tokens, 512), 1).to(DEV), rand((5, 140, 512), 2).to(DEV)
    wq = xk.prepare_weight_mxfp4(w)
    got = xk.expert_linear_mxfp4(x, wq, plan)
    sorted_rows = xk.expert_gather(x, plan)
    assert torch.equal(got, xk.expert_linear_mxfp4(sorted_rows, wq, plan, sorted=True))
    for e in range(5):
        rows = slice(int(offsets[e]), int(offsets[e + 1]))
        if rows.start < rows.stop:
            one = xk.MXFP4(wq.codes[e], wq.scales[e], (140, 512))
            assert torch.equal(got[rows], xk.linear_mxfp4(sorted_rows[rows], one))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [30, 60])
def test_one_or_two_rows_an_expert_over_a_long_contraction(gpu, tokens):
    """More k-blocks a CTA than its ring of stages takes in two turns: each is made once, in its turn."""
    ids = (torch.arange(tokens, dtype=torch.int32, device=DEV) % 30).reshape(-1, 1)
    plan = xk.expert_sort(ids, 30)
    x = torch.randn((tokens, 4104), device=DEV).to(torch.bfloat16)
    wq = xk.prepare_weight_mxfp4((torch.randn((30, 1280, 4096), device=DEV) * 0.02).to(torch.bfloat16))
    aligned, other = x[:, :4096].contiguous(), torch.empty(tokens * 4097, dtype=torch.bfloat16, device=DEV)
    odd = other.as_strided((tokens, 4096), (4097, 1))  # rows that are quantised before the product
    odd.copy_(aligned)
    want = xk.expert_linear_mxfp4(odd, wq, plan)
    for _ in range(3):
        assert torch.equal(xk.expert_linear_mxfp4(aligned, wq, plan), want)


@pytest.mark.gpu
def test_the_network(gpu):
    """The whole path against the same steps in 64 bits between its 4-bit roundings, within what
    codes that move at bf16 roundings of the intermediate can change (a step is at most a third of a
    value; measured against the output's norm)."""
    tokens, top, experts, k, f = 150, 2, 4, 256, 512
    ids = routing(tokens, top, experts, 5)
    x, weights = rand((tokens, k), 1), torch.softmax(rand((tokens, top), 2, torch.float32), -1)
    up, down = rand((experts, 2 * f, k), 3, scale=0.05), rand((experts, k, f), 4, scale=0.05)
    got = xk.expert_ffn_mxfp4(x.to(DEV), torch.from_numpy(ids).to(DEV), weights.to(DEV), xk.prepare_weight_mxfp4(up.to(DEV)), xk.prepare_weight_mxfp4(down.to(DEV)))
    order, _, offsets, _, _ = X.sort(ids, experts)
    xq = X.rounded(f64(turned(x)))[order // top]
    y = np.zeros((tokens * top, k))
    for e in range(experts):
        r = slice(offsets[e], offsets[e + 1])
        h = torch.from_numpy(xq[r] @ X.rounded(f64(turned(up[e]))).T).to(torch.bfloat16).double().numpy()
        g, v = h[:, :f], h[:, f:]
        h = torch.from_numpy(g / (1 + np.exp(-g)) * v).to(torch.bfloat16)
        y[r] = X.rounded(f64(turned(h))) @ X.rounded(f64(turned(down[e]))).T
    ref = X.combine(y, f64(weights), ids, experts)
    assert np.linalg.norm(f64(got) - ref) < 3e-2 * np.linalg.norm(ref)


@pytest.mark.gpu
def test_a_captured_network_replays(gpu):
    ids = torch.from_numpy(routing(20, 2, 4, 5)).to(DEV)
    x, weights = rand((20, 256), 1).to(DEV), torch.softmax(rand((20, 2), 2, torch.float32), -1).to(DEV)
    up = xk.prepare_weight_mxfp4(rand((4, 512, 256), 3, scale=0.05).to(DEV))
    down = xk.prepare_weight_mxfp4(rand((4, 256, 256), 4, scale=0.05).to(DEV))
    xk.expert_ffn_mxfp4(x, ids, weights, up, down)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = xk.expert_ffn_mxfp4(x, ids, weights, up, down)
    x.copy_(rand((20, 256), 9).to(DEV))
    ids.copy_(torch.from_numpy(routing(20, 2, 4, 6, 0.2)).to(DEV))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, xk.expert_ffn_mxfp4(x, ids, weights, up, down))


@pytest.mark.gpu
def test_no_tokens(gpu):
    plan = xk.expert_sort(torch.zeros((0, 2), dtype=torch.int32, device=DEV), 3)
    x = torch.zeros((0, 64), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w = rand((3, 32, 64), 1).to(DEV).requires_grad_()
    assert xk.expert_gather(x, plan).shape == (0, 64)
    assert xk.expert_linear_mxfp4(x, xk.prepare_weight_mxfp4(w, rotate=False), plan, rotate=False).shape == (0, 32)
    y = xk.mxfp4_expert_linear(x, w, plan, rotate=False)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == x.shape and not dw.any()
    assert xk.expert_combine(y, torch.zeros((0, 2), device=DEV), plan).shape == (0, 32)


# ----------------------------------------------------------------------------- many tiles a CTA pair

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,in_order,n,k,rotate", [(8192, False, 2816, 2048, True), (4500, True, 2816, 2048, True), (8192, True, 2305, 2000, False),
                                                        (4500, False, 2820, 1999, False)])
def test_products_of_many_tiles(gpu, tokens, in_order, n, k, rotate, dtype):
    """More tiles a CTA pair than it has accumulators, two experts without rows among the others, several
    k-blocks an expert in dw, and operands of two and four 32-row steps a CTA of the kernel that
    quantises along both axes.  Against 64-bit products of operands quantised one axis at a time."""
    experts, top = 8, 2
    rows = tokens * top
    ids = torch.from_numpy(routing(tokens, top, experts, 8, 0.05, used=[0, 1, 3, 4, 6, 7])).to(DEV)
    plan = xk.expert_sort(ids, experts)
    offsets = plan.offsets.tolist()
    x, w, dy = rand((rows if in_order else tokens, k), 1, dtype), rand((experts, n, k), 2, dtype, 0.1), rand((rows, n), 3, dtype, 0.1).to(DEV)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = xk.mxfp4_expert_linear(xd, wd, plan, rotate=rotate, sorted=in_order)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy)
    assert torch.equal(y, xk.mxfp4_expert_linear(xd, wd, plan, rotate=rotate, sorted=in_order))
    xr, wr = (turned(v).to(DEV) if rotate else v.to(DEV) for v in (x, w))
    xs = xr if in_order else xr[plan.order.long() // top]
    h = torch.from_numpy(O.hadamard_matrix()).to(DEV).double()

    def held(v, transpose=False):
        return xk.dequantize_mxfp4(xk.quantize_mxfp4(v, transpose=transpose), dtype=torch.float32).double()

    def groups(v, m):
        return (v.reshape(-1, 256) @ m).reshape(v.shape)

    def within(got, ref, lost):
        """`lost`: what 32 bits lose before the rotation back, if there is one, and the one rounding."""
        if rotate and got is not y:
            ref, lost = groups(ref, h), groups(lost, h.abs()) + 16 * 2.0 ** -24 * groups(ref.abs() + lost, h.abs())
        off = (got.double() - ref).abs() - lost * (1 + ROUND[dtype]) - ROUND[dtype] * ref.abs() - SMALL[dtype]
        assert bool((off <= 0).all()), f"{int((off > 0).sum())} past the bound, by {float(off.max())}"

    def product(a, b, terms):
        ref = a @ b.T
        return ref, (terms / 64 + 10) * 2.0 ** -23 * (a.abs() @ b.abs().T) + 2.0 ** -24 * ref.abs()

    want, lost = (torch.zeros((rows, n), dtype=torch.float64, device=DEV) for _ in range(2))
    gx, lost_x = (torch.zeros((rows, k), dtype=torch.float64, device=DEV) for _ in range(2))
    for e in range(experts):
        r = slice(offsets[e], offsets[e + 1])
        if r.start == r.stop:
            assert not dw[e].any()
            continue
        want[r], lost[r] = product(held(xs[r]), held(wr[e]), k)
        gx[r], lost_x[r] = product(held(dy[r]), held(wr[e], True), n)
        within(dw[e], *product(held(dy[r], True), held(xs[r], True), r.stop - r.start))
    within(y, want, lost)
    if not in_order:
        taken = torch.arange(rows, device=DEV) < offsets[-1]
        token = plan.order.long()[taken] // top
        gx, lost_x, size = (torch.zeros((tokens, k), dtype=torch.float64, device=DEV).index_add_(0, token, v[taken]) for v in (gx, lost_x, gx.abs() + lost_x))
        lost_x = lost_x + top * 2.0 ** -24 * size
    within(dx, gx, lost_x)


# ------------------------------------------------------------------ the experts' gradients, rounded once

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("in_order", [False, True])
@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("tokens,top,experts,n,k,dropped", [(7, 3, 9, 80, 256, 0.2), (300, 2, 3, 130, 512, 0.1), (150, 4, 4, 272, 256, 0)])
def test_expert_gradients_are_rounded_once(gpu, tokens, top, experts, n, k, dropped, rotate, in_order, dtype):
    """Against the formulas with one rounding to the type: the products' rows stay in fp32 up to a
    token's sum and the rotation back."""
    ids = routing(tokens, top, experts, 8, dropped)
    plan = xk.expert_sort(torch.from_numpy(ids).to(DEV), experts)
    order, _, offsets, _, _ = X.sort(ids, experts)
    x, w = rand((tokens * top if in_order else tokens, k), 1, dtype), rand((experts, n, k), 2, dtype, 0.1)
    dy = rand((tokens * top, n), 3, dtype, 0.1)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = xk.mxfp4_expert_linear(xd, wd, plan, rotate=rotate, sorted=in_order)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.to(DEV))
    t = turned if rotate else (lambda v: v)
    xs = f64(t(x)) if in_order else f64(t(x))[order // top]
    d = f64(dy)
    h = np.abs(O.hadamard_matrix().astype(np.float64))
    groups = lambda v: (v.reshape(-1, 256) @ h).reshape(v.shape)  # noqa: E731

    def one_rounding(got, ref, inner):
        """`inner`: what is lost in 32 bits before the rotation (at most ten additions one after
        another, sixteen allowed, each off by 2^-24 of a group's sum)."""
        if rotate:
            ref, inner = O.rotate_groups_dense_f64(ref), groups(inner) + 16 * 2.0 ** -24 * groups(np.abs(ref) + inner)
        check(got, ref, 0 * ref, 0, dtype, inner * (1 + ROUND[dtype]))

    gx, lost = np.zeros((tokens * top, k)), np.zeros((tokens * top, k))
    for e in range(experts):
        r = slice(offsets[e], offsets[e + 1])
        we = f64(t(w[e]))
        gx[r], spread = X.product(X.rounded(d[r]), X.rounded(we.T))
        lost[r] = (n / 64 + 10) * 2.0 ** -23 * spread + 2.0 ** -24 * np.abs(gx[r])
        if offsets[e] == offsets[e + 1]:
            assert not f64(dw[e]).any()
            continue
        ref, spread = X.product(X.rounded(d[r].T), X.rounded(xs[r].T))
        one_rounding(dw[e], ref, ((offsets[e + 1] - offsets[e]) / 64 + 10) * 2.0 ** -23 * spread + 2.0 ** -24 * np.abs(ref))
    if in_order:
        one_rounding(dx, gx, lost)
    else:
        one = np.ones((tokens, top))
        total = X.combine(np.abs(gx) + lost, one, ids, experts)
        one_rounding(dx, X.combine(gx, one, ids, experts), X.combine(lost, one, ids, experts) + top * 2.0 ** -24 * total)


@pytest.mark.gpu
def test_a_rotated_expert_gradient_keeps_fp16_s_range(gpu):
    """A group of dw whose values are all 6144 is one value of 98304 before the rotation back, which
    fp16 does not hold."""
    sign = torch.from_numpy(O.hadamard_matrix()[37] * 16)
    plan = xk.expert_sort(torch.tensor([[1]], device=DEV), 2)
    x = (sign * 1024).to(torch.float16).reshape(1, 256).to(DEV)  # 16384 at place 37 of its rotation
    w = torch.zeros((2, 3, 256), dtype=torch.float16, device=DEV, requires_grad=True)
    dw, = torch.autograd.grad(xk.mxfp4_expert_linear(x, w, plan), w, torch.full((1, 3), 6.0, dtype=torch.float16, device=DEV))
    assert torch.equal(dw[1].cpu(), (sign * 6144).to(torch.float16).expand(3, 256)) and not dw[0].any()


@pytest.mark.gpu
def test_tokens_without_a_choice(gpu):
    plan = xk.expert_sort(torch.zeros((5, 0), dtype=torch.int64, device=DEV), 3)
    x, w = rand((5, 64), 1).to(DEV).requires_grad_(), rand((3, 32, 64), 2).to(DEV).requires_grad_()
    for rows, in_order in ((x, False), (x[:0], True)):
        y = xk.mxfp4_expert_linear(rows, w, plan, rotate=False, sorted=in_order)
        assert y.shape == (0, 32) and y.dtype == x.dtype
        dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert dx.shape == x.shape and dw.shape == w.shape and not dx.any() and not dw.any()
    assert xk.expert_linear_mxfp4(x.detach(), xk.quantize_mxfp4(w), plan, rotate=False).shape == (0, 32)
    out = xk.expert_combine(xk.expert_gather(x, plan), torch.zeros((5, 0), device=DEV), plan)
    assert out.shape == (5, 64) and not out.any() and not torch.autograd.grad(out.sum(), x)[0].any()


# --------------------------------------------------------------------- what has no gradient says so

@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [5, 200])
def test_frozen_experts_have_no_backward_and_say_so(gpu, tokens):
    ids = torch.from_numpy(routing(tokens, 2, 4, 5, 0.1)).to(DEV)
    plan = xk.expert_sort(ids, 4)
    x, weights = rand((tokens, 256), 1).to(DEV), torch.softmax(rand((tokens, 2), 2, torch.float32), -1).to(DEV)
    up = xk.prepare_weight_mxfp4(rand((4, 512, 256), 3, scale=0.05).to(DEV))
    down = xk.prepare_weight_mxfp4(rand((4, 256, 256), 4, scale=0.05).to(DEV))
    want = xk.expert_linear_mxfp4(x, up, plan)
    xg = x.clone().requires_grad_()
    y = xk.expert_linear_mxfp4(xg, up, plan)
    assert torch.equal(y, want) and y.requires_grad and not want.requires_grad
    for loss in (y.sum(), xk.expert_linear_mxfp4(xg, up, plan).sum() + xg.sum()):
        with pytest.raises(RuntimeError, match="mxfp4_expert_linear"):
            torch.autograd.grad(loss, xg)
    with torch.no_grad():
        assert not xk.expert_linear_mxfp4(xg, up, plan).requires_grad
    # the network: the router's gradient is there, a token's is refused
    wg = weights.clone().requires_grad_()
    out = xk.expert_ffn_mxfp4(x, ids, wg, up, down)
    assert torch.equal(out, xk.expert_ffn_mxfp4(x, ids, weights, up, down))
    gw, = torch.autograd.grad(out, wg, torch.ones_like(out))
    h = xk.expert_linear_mxfp4(x, up, plan).chunk(2, dim=1)
    y = xk.expert_linear_mxfp4(torch.nn.functional.silu(h[0]) * h[1], down, plan, sorted=True)
    again = weights.clone().requires_grad_()
    assert torch.equal(gw, torch.autograd.grad(xk.expert_combine(y, again, plan), again, torch.ones_like(out))[0])
    out = xk.expert_ffn_mxfp4(xg, ids, wg, up, down)
    assert torch.equal(torch.autograd.grad(out.sum(), wg, retain_graph=True)[0], gw)
    with pytest.raises(RuntimeError, match="mxfp4_expert_linear"):
        (out + xg).sum().backward()


@pytest.mark.gpu
def test_forward_mode_is_refused(gpu):
    from torch.autograd import forward_ad as fw
    plan = xk.expert_sort(torch.zeros((4, 2), dtype=torch.int32, device=DEV), 2)
    x, y, weights = rand((4, 64), 1).to(DEV), rand((8, 64), 2).to(DEV), torch.ones((4, 2), device=DEV)
    w = xk.quantize_mxfp4(rand((2, 32, 64), 3).to(DEV))
    with fw.dual_level():
        dual = lambda v: fw.make_dual(v, torch.ones_like(v))  # noqa: E731
        for call in (lambda: xk.expert_gather(dual(x), plan), lambda: xk.expert_combine(dual(y), weights, plan),
                     lambda: xk.expert_combine(y, dual(weights), plan), lambda: xk.expert_linear_mxfp4(dual(x), w, plan, rotate=False),
                     lambda: xk.mxfp4_expert_linear(dual(x), torch.ones((2, 32, 64), device=DEV), plan, rotate=False)):
            with pytest.raises(RuntimeError, match="jvp|forward AD"):
                call()


@pytest.mark.gpu
def test_the_experts_weights_are_read_where_their_tensors_are(gpu):
    plan = xk.expert_sort(torch.from_numpy(routing(9, 2, 3, 5)).to(DEV), 3)
    x = rand((9, 256), 1).to(DEV)
    q, other = (xk.prepare_weight_mxfp4(rand((3, 96, 256), seed).to(DEV)) for seed in (2, 3))
    want = xk.expert_linear_mxfp4(x, other, plan)
    q.codes.data, q.scales.data = other.codes.clone(), other.scales.clone()
    assert torch.equal(xk.expert_linear_mxfp4(x, q, plan), want)
    q.codes.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="codes"):
        xk.expert_linear_mxfp4(x, q, plan)
    q.codes.data = other.codes[:2]
    with pytest.raises(ValueError, match="codes"):
        xk.expert_linear_mxfp4(x, q, plan)


# ---------------------------------------------------------------------------------------- refusals

def test_ids_are_checked_before_the_device():
    with pytest.raises(TypeError, match="int32 or int64"):
        xk.expert_sort(torch.zeros((2, 2)), 4)
    with pytest.raises(TypeError, match="CUDA"):
        xk.expert_sort(torch.zeros((2, 2), dtype=torch.int32), 4)


@pytest.mark.gpu
def test_arguments_are_checked(gpu):
    from xpu_kernels.int8 import _lib as L
    ids = torch.zeros((4, 2), dtype=torch.int32, device=DEV)
    for n in (0, 1025):
        with pytest.raises(ValueError, match="num_experts"):
            xk.expert_sort(ids, n)
    with pytest.raises(ValueError, match="T, k"):
        xk.expert_sort(ids[None], 4)
    plan = xk.expert_sort(ids, 4)
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=DEV)
    w = xk.quantize_mxfp4(torch.zeros((4, 32, 64), device=DEV))
    with pytest.raises(ValueError, match="4, W"):
        xk.expert_gather(x[:3], plan)
    with pytest.raises(ValueError, match="on cpu"):
        xk.expert_gather(x.cpu(), plan)
    with pytest.raises(ValueError, match="8, W"):
        xk.expert_combine(x, torch.zeros((4, 2), device=DEV), plan)
    y = torch.zeros((8, 64), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="weights"):
        xk.expert_combine(y, torch.zeros((4, 3), device=DEV), plan)
    with pytest.raises(TypeError, match="floating"):
        xk.expert_combine(y, ids, plan)
    with pytest.raises(TypeError, match="bfloat16"):
        xk.expert_gather(x.double(), plan)
    with pytest.raises(ValueError, match="tokens"):
        xk.expert_linear_mxfp4(y, w, plan, rotate=False)
    with pytest.raises(ValueError, match="sorted rows"):
        xk.expert_linear_mxfp4(x, w, plan, rotate=False, sorted=True)
    with pytest.raises(ValueError, match="do not fit"):
        xk.expert_linear_mxfp4(x[:, :32], w, plan, rotate=False)
    with pytest.raises(ValueError, match="256"):
        xk.expert_linear_mxfp4(x, w, plan)
    with pytest.raises(ValueError, match="do not fit"):
        xk.mxfp4_expert_linear(x, torch.zeros((3, 32, 64), device=DEV), plan)
    lib = L.load()
    p = plan.order.data_ptr()
    assert lib.xpuint8_expert_sort_workspace_bytes(8, 1025) == -1
    assert lib.xpuint8_expert_sort_stream(None, p, 3, 8, 4, p, p, p, p, p, None) == 2
    assert lib.xpuint8_expert_sort_stream(None, p, 4, 8, 4, None, p, p, p, p, None) == 2
    assert lib.xpuint8_expert_sort_stream(None, p, 4, 5000, 4, p, p, p, p, p, None) == 2
    assert b"expert_sort" in lib.xpuint8_last_error()
    assert lib.xpuint8_expert_gather_stream(None, x.data_ptr(), 0, 63, y.data_ptr(), p, p, 4, 2, 64) == 2
    assert lib.xpuint8_expert_combine_stream(None, y.data_ptr(), 0, 64, None, None, p, p, 4, 2, 64) == 2
    assert lib.xpuint8_mxfp4_expert_mm_stream(None, w.codes.data_ptr(), w.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(),
                                              y.data_ptr(), 0, None, p, 8, 1, 32, 64, 4) == 2
    assert lib.xpuint8_mxfp4_expert_dw_stream(None, w.codes.data_ptr(), w.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(),
                                              y.data_ptr(), 0, None, 1, 32, 64, 4) == 2
