"""MXFP4: quantisation bit for bit against the definition in 64 bits, products and linears within the
bound that 32-bit sums and one rounding to the output's type allow.

The bound of a product: the codes' and scales' products are exact, so only the running sums round.
An MMA adds 64 products to a 32-bit sum; with every one of these K / 64 additions, and those of a
split contraction's eight parts and the bias, off by at most 2^-23 of the sum of magnitudes (twice
round-to-nearest's), |error| <= (K / 64 + 10) 2^-23 sum|a||b|, and the result is rounded once to the
output's type (2^-8 of it for bf16, 2^-11 for fp16, 2^-24 for fp32, with 2^-24 below fp16's normal
range).  A rotated gradient is rounded to its type before and after the rotation.
"""

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
    x = torch.randn(*shape, generator=g) * scale
    if shape[-1] >= 64:
        x[..., torch.randperm(shape[-1], generator=g)[: shape[-1] // 64]] *= 20
    return x.to(dtype)


def f64(t):
    return t.detach().cpu().double().numpy()


def turned(x):
    """The rotation of a CPU tensor, 32 bits in the framework's order, rounded to its type."""
    y = O.rotate_groups(x.float().numpy())
    return torch.from_numpy(y).to(x.dtype)


def check_bits(q, x):
    """The stored codes and scales of q against the definition's of x [R, K] (64 bits)."""
    code, e = X.unpack(q.codes.cpu().numpy(), q.scales.cpu().numpy(), q.shape[-2])
    want_code, want_e = X.quantize(x)
    assert np.array_equal(e, want_e)
    fine = (want_e != 255)[..., None]
    # zero has two codes: a value of either sign that rounds to it keeps its sign
    assert np.array_equal(np.where(fine, code & 7, 0), np.where(fine, want_code & 7, 0))
    assert np.array_equal(np.where(fine & (code & 7 != 0), code, 0), np.where(fine & (want_code & 7 != 0), want_code, 0))


def check(got, ref, spread, k, dtype, extra=0.0):
    got = f64(got)
    bound = ((k / 64 + 10) * 2.0 ** -23) * spread + ROUND[dtype] * (np.abs(ref) + spread * 2.0 ** -20) + SMALL[dtype] + extra
    off = np.abs(got - ref) - bound
    assert got.shape == ref.shape
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


# ------------------------------------------------------------------------------- quantisation

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 255), (7, 256), (129, 257), (33, 1000), (300, 512), (1, 16384)])
def test_rows(gpu, rows, k, dtype):
    x = rand((rows, k), rows * 7 + k, dtype)
    q = xk.quantize_mxfp4(x.to(DEV))
    assert q.shape == (rows, k)
    check_bits(q, f64(x))
    for out in TYPES:
        back = xk.dequantize_mxfp4(q, dtype=out)
        assert back.dtype == out and np.array_equal(f64(back), f64(torch.from_numpy(X.rounded(f64(x))).to(out)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 256), (3, 512), (130, 768), (17, 4096)])
def test_rows_behind_the_rotation(gpu, rows, k, dtype):
    x = rand((rows, k), rows + k, dtype)
    check_bits(xk.quantize_mxfp4(x.to(DEV), rotate=True), f64(turned(x)))
    if dtype == torch.bfloat16:  # and of what rotate() gives
        check_bits(xk.quantize_mxfp4(x.to(DEV), rotate=True), f64(xk.rotate(x.to(DEV))))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 70), (31, 3), (32, 64), (33, 65), (127, 130), (128, 64), (129, 1), (300, 333)])
def test_columns(gpu, rows, cols, dtype):
    x = rand((rows, cols), rows * 3 + cols, dtype)
    q = xk.quantize_mxfp4(x.to(DEV), transpose=True)
    assert q.shape == (cols, rows)
    check_bits(q, f64(x).T)


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
def test_stacks(gpu, transpose):
    x = rand((3, 130, 96), 5)
    q = xk.quantize_mxfp4(x.to(DEV), transpose=transpose)
    for i in range(3):
        one = xk.MXFP4(q.codes[i], q.scales[i], q.shape[1:])
        check_bits(one, f64(x[i]).T if transpose else f64(x[i]))


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_where_it_can_go_wrong(gpu, dtype, transpose):
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    rows = [[0.0] * 32, [-0.0] * 32, [top] * 32, [-top, 1.0] + [0.0] * 30,
            [tiny] * 32, [tiny / 4] * 32, [tiny / 64, -tiny / 128] * 16,
            [float("nan")] + [1.0] * 31, [1.0] * 31 + [float("inf")], [-float("inf")] * 32,
            # ties of every step, the largest 4 (scale 1): to the even code
            [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5] + [0.0] * 19,
            # above 6 to 6, and the tie between 4 and 6
            [7.5, 5.0, -5.0, 6.5, 7.0, -7.5] + [0.0] * 26,
            [2.0 ** -i for i in range(32)] if dtype != torch.float16 else [2.0 ** -(i % 14) for i in range(32)]]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    if transpose:
        q = xk.quantize_mxfp4(x.T.contiguous().to(DEV), transpose=True)
    else:
        q = xk.quantize_mxfp4(x.to(DEV))
    check_bits(q, f64(x))
    back = f64(xk.dequantize_mxfp4(q, dtype=torch.float32))
    assert np.isnan(back[7:10]).all() and np.isfinite(np.delete(back, [7, 8, 9], axis=0)).all()


@pytest.mark.gpu
def test_strides_and_alignments(gpu):
    base = rand((40, 600), 9).to(DEV)
    for x in (base[:, 8:520], base[:, 1:301], base[::2, :256], base.T[:256], base[:, ::2]):
        check_bits(xk.quantize_mxfp4(x), f64(x))
        check_bits(xk.quantize_mxfp4(x, transpose=True), f64(x).T)


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    rows, k = 70000, 32768  # 2.3e9 values
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device=DEV)
    tail = rand((3, k), 3).to(DEV)
    x[-3:] = tail
    q = xk.quantize_mxfp4(x)
    assert torch.equal(xk.dequantize_mxfp4(q)[-3:], xk.dequantize_mxfp4(xk.quantize_mxfp4(tail)))


@pytest.mark.gpu
def test_rows_of_codes_whose_steps_pass_32_bits(gpu):
    """32 rows of codes are 2^32 bytes: the second 32-row step of the kernel that quantises along both axes."""
    k = 2 ** 28
    x, w = torch.zeros((1, k), dtype=torch.bfloat16, device=DEV), torch.zeros((33, k), dtype=torch.bfloat16, device=DEV)
    x[0, 5], x[0, 7], w[0, 5], w[32, 7] = 2, 3, 1, 1
    y = xk.mxfp4_linear(x.requires_grad_(), w, rotate=False)
    want = torch.zeros(33)
    want[0], want[32] = 2, 3
    assert torch.equal(y[0].float().cpu(), want)
    del x, w, y
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------- products

PRODUCTS = [(1, 1, 1), (1, 128, 256), (1, 300, 4096), (2, 77, 100), (16, 128, 32), (17, 129, 288), (33, 64, 544),
            (64, 200, 2048), (65, 1000, 320), (128, 130, 64), (129, 16, 96), (200, 300, 1000), (256, 256, 256),
            (257, 512, 257), (300, 77, 5000), (1000, 640, 768), (513, 1283, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(gpu, m, n, k, dtype):
    a, b = rand((m, k), m + k, torch.float32), rand((n, k), n * 3 + k, torch.float32)
    bias = rand((n,), n, torch.float32) if (m + n) % 2 else None
    y = xk.mxfp4_mm(xk.quantize_mxfp4(a.to(DEV)), xk.quantize_mxfp4(b.to(DEV)), None if bias is None else bias.to(DEV), dtype=dtype)
    ref, spread = X.product(X.rounded(f64(a)), X.rounded(f64(b)), None if bias is None else f64(bias))
    check(y, ref, spread, k, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 100, 300])
def test_a_nan_block_reaches_its_row_and_column_only(gpu, m):
    a, b = rand((m, 512), 1), rand((260, 512), 2)
    a[m // 2, 40] = float("nan")
    b[7, 300] = float("inf")
    y = f64(xk.mxfp4_mm(xk.quantize_mxfp4(a.to(DEV)), xk.quantize_mxfp4(b.to(DEV))))
    want = np.zeros((m, 260), dtype=bool)
    want[m // 2] = True
    want[:, 7] = True
    assert np.array_equal(np.isnan(y), want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 300])
def test_the_same_call_gives_the_same_bits(gpu, m):
    a, b = xk.quantize_mxfp4(rand((m, 4096), 1).to(DEV)), xk.quantize_mxfp4(rand((700, 4096), 2).to(DEV))
    first = xk.mxfp4_mm(a, b, dtype=torch.float32)
    for _ in range(20):
        assert torch.equal(first, xk.mxfp4_mm(a, b, dtype=torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,n,rotate", [((1, 512), 256, True), ((3, 256), 100, True), ((2, 5, 333), 48, False), ((200, 768), 96, True), ((0, 256), 16, True)])
def test_linear(gpu, shape, n, rotate, dtype):
    k = shape[-1]
    x, w = rand(shape, 1, dtype), rand((n, k), 2, dtype, 0.02)
    bias = rand((n,), 3, torch.float32)
    y = xk.linear_mxfp4(x.to(DEV), xk.prepare_weight_mxfp4(w.to(DEV), rotate=rotate), bias.to(DEV), rotate=rotate)
    assert y.shape == (*shape[:-1], n) and y.dtype == dtype
    t = turned if rotate else (lambda v: v)
    ref, spread = X.product(X.rounded(f64(t(x.reshape(-1, k)))), X.rounded(f64(t(w))), f64(bias))
    check(y.reshape(-1, n), ref, spread, k, dtype)


@pytest.mark.gpu
def test_modules_and_leading_shapes(gpu):
    lin = torch.nn.Linear(512, 96, device=DEV, dtype=torch.bfloat16)
    x = rand((2, 7, 512), 4).to(DEV)
    want = xk.linear_mxfp4(x, xk.prepare_weight_mxfp4(lin.weight), lin.bias)
    serve, train = xk.Mxfp4Linear.from_linear(lin), xk.TrainableMxfp4Linear.from_linear(lin)
    assert torch.equal(serve(x), want) and torch.equal(train(x), want)
    again = xk.Mxfp4Linear.from_linear(torch.nn.Linear(512, 96, device=DEV, dtype=torch.bfloat16))
    again.load_state_dict(serve.state_dict())
    assert torch.equal(again(x), want)
    train(x).sum().backward()
    assert train.weight.grad.shape == train.weight.shape and train.bias.grad.shape == train.bias.shape


# ------------------------------------------------------------------------------------- gradients

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,rotate", [(1, 16, 256, True), (5, 100, 64, False), (130, 77, 333, False), (300, 272, 512, True), (513, 96, 256, True)])
def test_gradients(gpu, m, n, k, rotate, dtype):
    x, w, dy = rand((m, k), 1, dtype), rand((n, k), 2, dtype, 0.02), rand((m, n), 3, dtype, 0.1)
    bias = torch.zeros(n)
    args = [v.to(DEV).requires_grad_() for v in (x, w, bias)]
    y = xk.mxfp4_linear(*args, rotate=rotate)
    dx, dw, db = torch.autograd.grad(y, args, dy.to(DEV))
    assert dx.dtype == dw.dtype == dtype and db.dtype == torch.float32
    xr, wr = (f64(turned(v)) if rotate else f64(v) for v in (x, w))
    d = f64(dy)
    h = np.abs(O.hadamard_matrix().astype(np.float64))

    def back(ref, spread, contraction):
        if not rotate:
            return ref, spread, 0.0
        inner = (contraction / 64 + 10) * 2.0 ** -23 * spread + ROUND[dtype] * np.abs(ref) + SMALL[dtype]
        groups = lambda v, m: (v.reshape(-1, 256) @ m).reshape(v.shape)  # noqa: E731
        # the rotation itself: 8 additions in 32 bits of 256 values
        extra = groups(inner, h) + 16 * 2.0 ** -24 * groups(np.abs(ref), h)
        return O.rotate_groups_dense_f64(ref), groups(spread, h), extra

    ref, spread = X.product(X.rounded(xr), X.rounded(wr))
    check(y, ref, spread, k, dtype)
    ref, spread, extra = back(*X.product(X.rounded(d), X.rounded(wr.T)), n)
    check(dx, ref, spread if not rotate else 0 * spread, n, dtype, extra)
    ref, spread, extra = back(*X.product(X.rounded(d.T), X.rounded(xr.T)), m)
    check(dw, ref, spread if not rotate else 0 * spread, m, dtype, extra)
    assert np.allclose(f64(db), d.sum(0), rtol=1e-6, atol=1e-6 * np.abs(d).sum(0).max())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 5, 32), (140, 33, 96)])
def test_gradients_against_differences(gpu, m, n, k):
    """Whole numbers up to 4 are MXFP4 values in every block, so on them the linear is its own plain
    form and the difference quotient along a direction of whole numbers is exact."""
    g = torch.Generator().manual_seed(m)
    draw = lambda *s: torch.randint(-3, 4, s, generator=g).float()  # noqa: E731
    step = lambda *s: torch.randint(-1, 2, s, generator=g).float().to(DEV)  # noqa: E731
    x, w, dy = (draw(*s).to(DEV) for s in ((m, k), (n, k), (m, n)))
    x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(xk.mxfp4_linear(x, w, rotate=False), (x, w), dy)
    loss = lambda x, w: float((xk.mxfp4_linear(x.detach(), w.detach(), rotate=False).double() * dy).sum())  # noqa: E731
    for _ in range(4):
        u, v = step(m, k), step(n, k)
        assert (loss(x + u, w) - loss(x - u, w)) / 2 == float((dx.double() * u).sum())
        assert (loss(x, w + v) - loss(x, w - v)) / 2 == float((dw.double() * v).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("rotate", [False, True])
def test_one_gradient_alone_is_the_same(gpu, rotate):
    x, w, dy = rand((140, 256), 1).to(DEV), rand((96, 256), 2).to(DEV), rand((140, 96), 3).to(DEV)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = xk.mxfp4_linear(xg, wg, rotate=rotate)
    dx, dw = torch.autograd.grad(y, (xg, wg), dy)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(xk.mxfp4_linear(xg, w, rotate=rotate), xg, dy)[0], dx)
    assert torch.equal(torch.autograd.grad(xk.mxfp4_linear(x, wg, rotate=rotate), wg, dy)[0], dw)
    both = xk.mxfp4_linear(xg, wg, rotate=rotate)
    assert torch.equal(torch.autograd.grad(both, wg, dy, retain_graph=True)[0], dw)
    assert torch.equal(torch.autograd.grad(both, xg, dy)[0], dx)
    with torch.no_grad():
        assert torch.equal(xk.mxfp4_linear(xg, wg, rotate=rotate), y)


@pytest.mark.gpu
def test_a_second_derivative_is_refused(gpu):
    x, w = rand((4, 32), 1, torch.float32).to(DEV).requires_grad_(), rand((8, 32), 2, torch.float32).to(DEV)
    dx, = torch.autograd.grad(xk.mxfp4_linear(x, w, rotate=False).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 3, 8, 9, 130])
@pytest.mark.parametrize("rotate", [False, True])
def test_a_nan_in_x_reaches_its_row_only(gpu, m, rotate):
    x, w = rand((m, 512), 1), rand((300, 512), 2)
    x[m // 2, 7] = float("nan")
    y = f64(xk.linear_mxfp4(x.to(DEV), xk.prepare_weight_mxfp4(w.to(DEV), rotate=rotate), rotate=rotate))
    want = np.zeros((m, 300), dtype=bool)
    want[m // 2] = True
    assert np.array_equal(np.isnan(y), want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 5, 8])
def test_tokens_quantised_in_the_product_are_the_quantiser_s(gpu, m):
    for dtype in TYPES:
        for k, rotate in ((512, True), (100, False), (2816, True)):
            x, w = rand((m, k), m, dtype).to(DEV), rand((140, k), 2, dtype).to(DEV)
            wq = xk.prepare_weight_mxfp4(w, rotate=rotate)
            want = xk.mxfp4_mm(xk.quantize_mxfp4(x, rotate=rotate), wq, dtype=dtype)
            assert torch.equal(xk.linear_mxfp4(x, wq, rotate=rotate), want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 8])
@pytest.mark.parametrize("n,k,rotate", [(19200, 4096, True), (7790, 12160, False), (19200, 2100, False)])
def test_tokens_over_a_contraction_of_several_turns(gpu, m, n, k, rotate):
    """More k-blocks a CTA than its ring of stages takes in two turns: each is made once, in its turn."""
    for dtype in TYPES:
        x, w = rand((m, k), m, dtype).to(DEV), (torch.randn((n, k), device=DEV) * 0.02).to(dtype)
        wq = xk.prepare_weight_mxfp4(w, rotate=rotate)
        want = xk.mxfp4_mm(xk.quantize_mxfp4(x, rotate=rotate), wq, dtype=dtype)
        for _ in range(3):
            assert torch.equal(xk.linear_mxfp4(x, wq, rotate=rotate), want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(4, 0), (0, 6), (0, 0)])
def test_empty_sizes_have_gradients(gpu, m, n):
    x, w, bias = (torch.zeros(s, device=DEV, requires_grad=True) for s in ((2, m, 256), (n, 256), (n,)))
    y = xk.mxfp4_linear(x, w, bias)
    assert y.shape == (2, m, n)
    grads = torch.autograd.grad(y, (x, w, bias), torch.zeros_like(y))
    for g, v in zip(grads, (x, w, bias)):
        assert g.shape == v.shape and not g.any()


@pytest.mark.gpu
def test_a_bias_s_gradient_is_the_bias_s_own(gpu):
    """Of its shape, its type and its device: any bias that the forward call takes."""
    x, w, dy = rand((7, 64), 1).to(DEV), rand((48, 64), 2).to(DEV), rand((7, 48), 3).to(DEV)
    want = dy.float().sum(0)
    for bias in (torch.zeros(48), torch.zeros((1, 48), device=DEV), torch.zeros((48, 1), device=DEV, dtype=torch.float16)):
        bias.requires_grad_()
        y = xk.mxfp4_linear(x, w, bias, rotate=False)
        g, = torch.autograd.grad(y, bias, dy)
        assert g.shape == bias.shape and g.dtype == bias.dtype and g.device == bias.device
        assert torch.equal(g.reshape(-1), want.to(device=bias.device, dtype=bias.dtype))


# ----------------------------------------------------------------------------- many tiles a CTA pair

def held(q):
    """What q stands for, in 64 bits on the GPU."""
    return xk.dequantize_mxfp4(q, dtype=torch.float32).double()


def check_gpu(got, ref, spread, k, dtype):
    bound = ((k / 64 + 10) * 2.0 ** -23) * spread + ROUND[dtype] * (ref.abs() + spread * 2.0 ** -20) + SMALL[dtype]
    off = (got.double() - ref).abs() - bound
    assert got.shape == ref.shape and bool((off <= 0).all()), f"{int((off > 0).sum())} past the bound, by {float(off.max())}"


#: 17 x 20 (21) tiles of 256 x 256, 15 x 9 of 256 x 128 and 149 of 256 x 128 on 74 pairs, with fewer k-blocks a tile
#: than stages, as many, and more; N across the columns that both accumulators use; odd rows of the output
MANY_TILES = [(4097, 5120, 64, True), (4097, 5121, 288, False), (4097, 5120, 1280, True), (4097, 5121, 1280, True), (4097, 5118, 2560, False),
              (3840, 1152, 1280, True), (38017, 120, 320, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,with_bias", MANY_TILES)
def test_products_of_many_tiles(gpu, m, n, k, with_bias):
    g = torch.Generator(device=DEV).manual_seed(m + n + k)
    a, b = (xk.quantize_mxfp4(torch.randn((r, k), generator=g, device=DEV)) for r in (m, n))
    bias = torch.randn(n, generator=g, device=DEV) if with_bias else None
    va, vb = held(a), held(b)
    ref, spread = va @ vb.T, va.abs() @ vb.abs().T
    if with_bias:
        ref, spread = ref + bias.double(), spread + bias.double().abs()
    for dtype in TYPES:
        y = xk.mxfp4_mm(a, b, bias, dtype=dtype)
        check_gpu(y, ref, spread, k, dtype)
        for _ in range(5):
            assert torch.equal(xk.mxfp4_mm(a, b, bias, dtype=dtype), y)


# ------------------------------------------------------------------ operands quantised along both axes

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,rotate", [(4097, 200, 5120, True), (4100, 200, 5100, False), (8200, 130, 4096, True), (8129, 130, 4095, False),
                                          (130, 4097, 5120, True), (130, 8200, 4099, False)])
def test_large_operands_are_the_single_quantisers_(gpu, m, n, k, rotate, dtype):
    """x and w large enough for two and four 32-row steps a CTA of the kernel that quantises along both
    axes: the products' bits are those of operands quantised one axis at a time."""
    x, w, dy = rand((m, k), 1, dtype), rand((n, k), 2, dtype, 0.02), rand((m, n), 3, dtype, 0.1).to(DEV)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = xk.mxfp4_linear(xd, wd, rotate=rotate)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy)
    xr, wr = (turned(v).to(DEV) if rotate else v.to(DEV) for v in (x, w))
    quant = xk.quantize_mxfp4
    assert torch.equal(y, xk.mxfp4_mm(quant(xr), quant(wr), dtype=dtype))
    want_dx = xk.mxfp4_mm(quant(dy), quant(wr, transpose=True), dtype=torch.float32 if rotate else dtype)
    want_dw = xk.mxfp4_mm(quant(dy, transpose=True), quant(xr, transpose=True), dtype=torch.float32 if rotate else dtype)
    for got, want in ((dx, want_dx), (dw, want_dw)):
        assert torch.equal(got.cpu(), turned(want.cpu()).to(dtype) if rotate else want.cpu())


# ---------------------------------------------------------------------- gradients turned back

def turned_back(ref, spread, terms):
    """A product turned back by the rotation, and what 32 bits lose before the one rounding to the
    gradient's type: the running sums, the product's rounding to fp32, and the rotation's additions (at
    most ten one after another, sixteen allowed, each off by 2^-24 of a group's sum)."""
    h = np.abs(O.hadamard_matrix().astype(np.float64))
    groups = lambda v: (v.reshape(-1, 256) @ h).reshape(v.shape)  # noqa: E731
    inner = terms * 2.0 ** -23 * spread + 2.0 ** -24 * np.abs(ref)
    return O.rotate_groups_dense_f64(ref), groups(inner) + 16 * 2.0 ** -24 * groups(np.abs(ref) + inner)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 16, 256), (300, 272, 512), (513, 96, 768)])
def test_a_rotated_gradient_is_rounded_once(gpu, m, n, k, dtype):
    x, w, dy = rand((m, k), 1, dtype), rand((n, k), 2, dtype, 0.02), rand((m, n), 3, dtype, 0.1)
    args = [v.to(DEV).requires_grad_() for v in (x, w)]
    dx, dw = torch.autograd.grad(xk.mxfp4_linear(*args), args, dy.to(DEV))
    xr, wr, d = f64(turned(x)), f64(turned(w)), f64(dy)
    for got, product, contraction in ((dx, X.product(X.rounded(d), X.rounded(wr.T)), n), (dw, X.product(X.rounded(d.T), X.rounded(xr.T)), m)):
        ref, extra = turned_back(*product, contraction / 64 + 10)
        check(got, ref, 0 * ref, contraction, dtype, extra * (1 + ROUND[dtype]))


@pytest.mark.gpu
def test_a_rotated_gradient_keeps_fp16_s_range(gpu):
    """A group of dw whose values are all 6144 is one value of 98304 before the rotation back, which
    fp16 does not hold."""
    sign = torch.from_numpy(O.hadamard_matrix()[37] * 16)
    x = (sign * 1024).to(torch.float16).reshape(1, 256)  # 16384 at place 37 of its rotation
    w = torch.zeros((3, 256), dtype=torch.float16)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    dw, = torch.autograd.grad(xk.mxfp4_linear(xd, wd), wd, torch.full((1, 3), 6.0, dtype=torch.float16, device=DEV))
    assert torch.equal(dw.cpu(), (sign * 6144).to(torch.float16).expand(3, 256))


# --------------------------------------------------------------------- what has no gradient says so

@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40])
def test_a_frozen_weight_s_linear_has_no_backward_and_says_so(gpu, m):
    x, bias = rand((m, 256), 1).to(DEV), rand((96,), 3, torch.float32).to(DEV)
    w = xk.prepare_weight_mxfp4(rand((96, 256), 2).to(DEV))
    want = xk.linear_mxfp4(x, w, bias)
    assert not want.requires_grad
    for xg, bg in ((x.clone().requires_grad_(), bias), (x, bias.clone().requires_grad_()), (x.clone().requires_grad_(), None)):
        at = xg if xg.requires_grad else bg
        y = xk.linear_mxfp4(xg, w, bg)
        assert y.requires_grad and (bg is None or torch.equal(y, want))
        with pytest.raises(RuntimeError, match="mxfp4_linear"):
            torch.autograd.grad(y.sum(), at, retain_graph=True)
        with pytest.raises(RuntimeError, match="mxfp4_linear"):  # beside another way to the same tensor
            torch.autograd.grad(y.sum() + at.sum(), at)
        with torch.no_grad():
            assert not xk.linear_mxfp4(xg, w, bg).requires_grad
    module = xk.Mxfp4Linear(w, bias)
    with pytest.raises(RuntimeError, match="mxfp4_linear"):
        module(x.clone().requires_grad_()).sum().backward()
    assert torch.equal(module(x), want)


@pytest.mark.gpu
def test_forward_mode_is_refused(gpu):
    from torch.autograd import forward_ad as fw
    x, w = rand((4, 64), 1).to(DEV), xk.quantize_mxfp4(rand((32, 64), 2).to(DEV))
    bias = torch.zeros(32, device=DEV)
    with fw.dual_level():
        dual = lambda v: fw.make_dual(v, torch.ones_like(v))  # noqa: E731
        for call in (lambda: xk.linear_mxfp4(dual(x), w, rotate=False), lambda: xk.linear_mxfp4(x, w, dual(bias), rotate=False),
                     lambda: xk.mxfp4_linear(dual(x), torch.ones_like(x), rotate=False)):
            with pytest.raises(RuntimeError, match="jvp|forward AD"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp|forward AD"):
                call()


# ------------------------------------------------------------------------- matrices whose memory changes

@pytest.mark.gpu
@pytest.mark.parametrize("made", ["by the quantiser", "from tensors"])
def test_a_matrix_is_read_where_its_tensors_are(gpu, made):
    x = rand((5, 256), 1).to(DEV)
    first, other = (xk.prepare_weight_mxfp4(rand((96, 256), seed).to(DEV)) for seed in (2, 3))
    want, values = xk.linear_mxfp4(x, other), xk.dequantize_mxfp4(other)
    product = xk.mxfp4_mm(other, other)
    q = first if made == "by the quantiser" else xk.MXFP4(first.codes.clone(), first.scales.clone(), first.shape)
    q.codes.data = other.codes.clone()
    q.scales.set_(other.scales.clone())
    assert torch.equal(xk.linear_mxfp4(x, q), want) and torch.equal(xk.dequantize_mxfp4(q), values)
    assert torch.equal(xk.mxfp4_mm(q, q), product)
    calls = (lambda: xk.linear_mxfp4(x, q), lambda: xk.dequantize_mxfp4(q), lambda: xk.mxfp4_mm(q, other), lambda: xk.mxfp4_mm(other, q))
    codes = q.codes.clone()

    def refused():
        for call in calls:
            with pytest.raises(ValueError, match="codes|is on|are on"):
                call()

    q.codes.untyped_storage().resize_(0)
    refused()
    for wrong in (codes[:95], codes.to(torch.int16), codes.T, torch.zeros((97, 128), dtype=torch.uint8, device=DEV)):
        q.codes.data = wrong
        refused()
    q.codes.data = codes.cpu()
    with pytest.raises((ValueError, TypeError)):
        xk.linear_mxfp4(x, q)
    q.codes.data = codes
    assert torch.equal(xk.linear_mxfp4(x, q), want)


@pytest.mark.gpu
def test_copies_of_a_matrix_are_their_own(gpu):
    import copy
    import io
    x, q = rand((5, 256), 1).to(DEV), xk.prepare_weight_mxfp4(rand((96, 256), 2).to(DEV))
    want = xk.linear_mxfp4(x, q)
    file = io.BytesIO()
    torch.save(q, file)
    copies = [copy.deepcopy(q), torch.load(io.BytesIO(file.getvalue()), weights_only=False)]
    q.codes, q.scales
    copies.append(copy.deepcopy(q))
    q.codes.zero_()
    q.scales.zero_()
    for c in copies:
        assert c.shape == q.shape and torch.equal(xk.linear_mxfp4(x, c), want)


# ------------------------------------------------------------------------------ a wait that gives up

@pytest.mark.gpu
def test_products_after_a_fault_are_refused_until_it_is_cleared(gpu):
    """One wait of the products' own runs out on a barrier that nothing arrives on; what would be left
    unwritten since then is an error, not a result."""
    from xpu_kernels.int8 import _lib as L
    lib = L.load()
    x, w, dy = rand((40, 256), 1).to(DEV), rand((96, 256), 2).to(DEV), rand((40, 96), 3).to(DEV)
    q, ids = xk.prepare_weight_mxfp4(w), torch.zeros((40, 1), dtype=torch.int32, device=DEV)
    stack, plan = xk.prepare_weight_mxfp4(w[None]), xk.expert_sort(ids, 1)
    xg = x.clone().requires_grad_()
    y = xk.mxfp4_linear(xg, w)
    calls = [lambda: xk.linear_mxfp4(x, q), lambda: xk.linear_mxfp4(x[:1], q), lambda: xk.mxfp4_mm(q, q), lambda: xk.expert_linear_mxfp4(x, stack, plan),
             lambda: xk.mxfp4_expert_linear(x, w[None], plan), lambda: torch.autograd.grad(y, xg, dy, retain_graph=True)[0]]
    want = [call() for call in calls]
    assert lib.xpuint8_mxfp4_wait_probe(200_000, 0) == 2
    assert lib.xpuint8_mxfp4_wait_probe(200_000, 77) == 0
    for call in calls:
        with pytest.raises(RuntimeError, match=r"gave up a wait on the device \(site 77\)"):
            call()
    xk.dequantize_mxfp4(q)  # no product
    assert lib.xpuint8_fault_status(0) == 77 and lib.xpuint8_fault_status(1) == 77 and lib.xpuint8_fault_status(0) == 0
    for call, value in zip(calls, want):
        assert torch.equal(call(), value)


@pytest.mark.gpu
def test_the_first_product_may_be_a_captured_one(gpu):
    """Its preparations on the host are no part of the graph."""
    import os
    import subprocess
    import sys
    code = """
import torch, xpu_kernels as xk
x = torch.ones((3, 256), device="cuda", dtype=torch.bfloat16)
w = xk.prepare_weight_mxfp4(torch.ones((32, 256), device="cuda", dtype=torch.bfloat16))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = xk.linear_mxfp4(x, w)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, xk.linear_mxfp4(x, w)) and y[0, 0] == 256
"""
    path = os.pathsep.join([os.path.dirname(os.path.dirname(xk.__file__)), os.environ.get("PYTHONPATH", "")])
    done = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


# ------------------------------------------------------------------------------ streams and graphs

@pytest.mark.gpu
def test_the_current_stream_is_used(gpu):
    w = xk.prepare_weight_mxfp4(rand((256, 512), 1).to(DEV))
    x = rand((300, 512), 2).to(DEV)
    want = xk.linear_mxfp4(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        later = x * 1
        got = xk.linear_mxfp4(later, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 300])
def test_a_captured_linear_replays(gpu, m):
    w = xk.prepare_weight_mxfp4(rand((256, 512), 1).to(DEV))
    x = rand((m, 512), 2).to(DEV)
    xk.linear_mxfp4(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = xk.linear_mxfp4(x, w)
    other = rand((m, 512), 3).to(DEV)
    x.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, xk.linear_mxfp4(other, w))


# ---------------------------------------------------------------------------------------- refusals

def test_the_binding_takes_entries_that_the_library_has():
    from xpu_kernels import _native
    from xpu_kernels.int8 import _lib as L
    assert {"xpuint8_" + name for name in _native.names()} - {"xpuint8_last_error"} <= set(L._signatures())
    for call in (_native.quantize, _native.linear, _native.sort):
        with pytest.raises(ValueError, match="arguments"):
            call(1)


def test_the_binding_formats_its_errors():
    """By streams, which crash in a module that is linked with a C++ runtime of its own."""
    from xpu_kernels import _native
    with pytest.raises(ValueError, match="expected 3 arguments, got 1"):
        _native.quantize(1)
    with pytest.raises(ValueError, match="expected 2 arguments, got 0"):
        _native.sort()


def test_a_matrix_checks_its_buffers():
    codes, scales = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 1, 32, 16), dtype=torch.uint8)
    assert xk.MXFP4(codes, scales, (4, 64)).shape == (4, 64)
    with pytest.raises(ValueError, match="codes"):
        xk.MXFP4(codes, scales, (4, 96))
    with pytest.raises(ValueError, match="scales"):
        xk.MXFP4(codes, scales[0], (4, 64))
    with pytest.raises(TypeError, match="uint8"):
        xk.MXFP4(codes.to(torch.int8), scales, (4, 64))
    with pytest.raises(ValueError, match="shape"):
        xk.MXFP4(codes, scales, (64,))
    with pytest.raises(ValueError, match="contiguous"):
        xk.MXFP4(torch.zeros((32, 4), dtype=torch.uint8).T, scales, (4, 64))


def test_arguments_are_checked_before_the_device():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    w = xk.MXFP4(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 1, 32, 16), dtype=torch.uint8), (4, 64))
    with pytest.raises(ValueError, match="256"):
        xk.quantize_mxfp4(x, rotate=True)
    with pytest.raises(ValueError, match="transpose"):
        xk.quantize_mxfp4(x, rotate=True, transpose=True)
    with pytest.raises(ValueError, match="R, K"):
        xk.quantize_mxfp4(x[0])
    with pytest.raises(TypeError, match="CUDA"):
        xk.quantize_mxfp4(x)
    with pytest.raises(TypeError, match="bfloat16"):
        xk.quantize_mxfp4(x.double())
    with pytest.raises(TypeError, match="dtype"):
        xk.dequantize_mxfp4(w, dtype=torch.float64)
    with pytest.raises(TypeError, match="CUDA"):
        xk.dequantize_mxfp4(w)
    with pytest.raises(TypeError, match="CUDA"):
        xk.mxfp4_mm(w, w)
    with pytest.raises(ValueError, match="columns"):
        xk.linear_mxfp4(x[:, :32], w, rotate=False)
    with pytest.raises(ValueError, match="256"):
        xk.linear_mxfp4(x, w)
    with pytest.raises(ValueError, match="M, K"):
        xk.mxfp4_mm(w, xk.MXFP4(torch.zeros((4, 16), dtype=torch.uint8), w.scales, (4, 32)))
    with pytest.raises(ValueError, match="columns"):
        xk.mxfp4_linear(x, torch.zeros((4, 32)))
    with pytest.raises(TypeError, match="MXFP4"):
        xk.Mxfp4Linear(x)
    with pytest.raises(TypeError, match="N, K"):
        xk.TrainableMxfp4Linear(x[0])


@pytest.mark.gpu
def test_the_entries_refuse(gpu):
    from xpu_kernels.int8 import _lib as L
    lib = L.load()
    x = torch.zeros((4, 256), dtype=torch.bfloat16, device=DEV)
    q = xk.quantize_mxfp4(x)
    c, s, p = q.codes.data_ptr(), q.scales.data_ptr(), x.data_ptr()
    quant = lib.xpuint8_mxfp4_quantize_stream
    assert quant(None, p, 3, 256, c, s, None, 4, 256, 4, 0) == 2
    assert quant(None, p, 0, 255, c, s, None, 4, 256, 4, 0) == 2
    assert quant(None, p, 0, 256, c + 1, s, None, 4, 256, 4, 0) == 2
    assert quant(None, p, 0, 256, None, None, None, 4, 256, 4, 0) == 2
    assert quant(None, p, 0, 256, c, s, None, 4, 256, 3, 0) == 2
    assert quant(None, p, 0, 256, c, s, None, 0, 256, 4, 0) == 2
    assert quant(None, p, 0, 256, c, s, None, 4, 200, 4, 1) == 3
    assert quant(None, p, 0, 256, c, s, p, 4, 256, 4, 0) == 2
    assert b"mxfp4" in lib.xpuint8_last_error()
    mm = lib.xpuint8_mxfp4_mm_stream
    out = torch.zeros((4, 4), dtype=torch.float32, device=DEV)
    o = out.data_ptr()
    assert mm(None, c, s, c, s, None, o, 2, 3, 4, 4, 256) == 2
    assert mm(None, c, s, c, s, None, o + 2, 2, 4, 4, 4, 256) == 2
    assert mm(None, c, s, c, None, None, o, 2, 4, 4, 4, 256) == 2
    assert mm(None, c, s, c, s, o + 4, o, 2, 4, 4, 4, 256) == 2
    assert mm(None, c, s, c, s, None, o, 2, 4, 4, 4, 0) == 2
    assert lib.xpuint8_mxfp4_quantize_columns_stream(None, p, 0, 256, c, s, 4, 256, 0, None, None, 0, 0) == 2
    assert lib.xpuint8_mxfp4_quantize_columns_stream(None, p, 0, 256, c, s, 4, 256, 1, c, None, 1, 1) == 2
    assert lib.xpuint8_mxfp4_dequantize_stream(None, c, s, o, 5, 4, 256, 4) == 2
    with pytest.raises(ValueError, match="bias"):
        xk.mxfp4_mm(q, q, torch.zeros(3, device=DEV))
    with pytest.raises(ValueError, match="weight on"):
        xk.linear_mxfp4(x.cpu(), q)
