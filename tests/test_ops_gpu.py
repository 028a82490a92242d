"""Row operators on the GPU against their definitions in 64 bits.

Tolerances, derived before the first run.  u = 2^-24 is half a step of float32, e half a step of the
rows' type.  A result is off by its final rounding, e |result| (subnormal results by a tiny absolute
amount), and by float32 roundings on the way, each u relative to what it rounds.
"""
import pytest
import torch

import ops_formulas as f

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
# (rows, dim): one row, lane groups of every width, several chunks a lane, whole blocks, odd lengths
SHAPES = [(1, 1), (3, 5), (70, 8), (33, 17), (257, 64), (19, 100), (65, 128), (300, 256), (41, 301), (12, 602), (9, 1024), (7, 1031),
          (5, 2048), (3, 4099), (2, 16384)]


@pytest.fixture(scope="module")
def ops():
    from aethergraph_b200 import ops

    return ops


def rand(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def near(got, want, tol, what=""):
    got, want = got.detach().to(torch.float64).cpu(), want.detach().to(torch.float64).cpu()
    off = (got - want).abs() - tol.cpu()
    worst = float(off.max()) if off.numel() else 0.0
    assert got.shape == want.shape and worst <= 0, f"{what}: {worst} over the bound at {int(off.argmax())} of {tuple(got.shape)}"


# ----------------------------------------------------------------- dropout --
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_dropout(ops, rows, dim, dtype):
    x = rand(1, rows, dim, dtype=dtype)
    for p, seed, offset in ((0.5, 1, 0), (0.1, 2 ** 64 - 1, 2 ** 40 + 3), (0.0, 3, 1), (1.0, 4, 2), (2.0 ** -17, 5, 3)):
        m = f.mask(rows, dim, p, seed, offset)
        y = ops.dropout(x, p, seed, offset)
        want = x.to(torch.float64).cpu() * m
        # the scale (u), its product (u) and the result's rounding
        near(y, want, (f.STEP[dtype] + 2 * U) * want.abs() + LEAST[dtype], f"p {p}")
        assert torch.equal(y.cpu() == 0, (want == 0) | (y.cpu() == 0)) and not bool((y.cpu()[m == 0] != 0).any())


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_gradient_is_the_same_mask(ops, dtype):
    x = rand(1, 37, 44, dtype=dtype).requires_grad_()
    dy = rand(2, 37, 44, dtype=dtype)
    y = ops.dropout(x, 0.3, 9, 4)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx, ops.dropout(dy, 0.3, 9, 4))
    assert torch.equal(y, ops.dropout(x.detach(), 0.3, 9, 4))


def test_dropout_layouts(ops):
    """A mask depends on row and column alone: pitch, alignment and leading dimensions change nothing."""
    x = rand(1, 50, 40)
    want = ops.dropout(x, 0.4, 8, 1)
    wide = torch.zeros(50, 61, device="cuda")
    wide[:, 3:43] = x
    assert torch.equal(ops.dropout(wide[:, 3:43], 0.4, 8, 1), want)
    assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.4, 8, 1), want)
    assert torch.equal(ops.dropout(x.view(5, 10, 40), 0.4, 8, 1), want.view(5, 10, 40))
    assert torch.equal(ops.dropout(x[:1].expand(50, 40), 0.4, 8, 1), ops.dropout(x[:1].repeat(50, 1), 0.4, 8, 1))
    assert torch.equal(ops.dropout(x[0], 0.4, 8, 1), ops.dropout(x[:1], 0.4, 8, 1)[0])
    assert ops.dropout(x[:0], 0.4, 8, 1).shape == (0, 40)
    inplace = wide[:, 3:43]
    assert ops.dropout_(inplace, 0.4, 8, 1) is inplace
    assert torch.equal(wide[:, 3:43], want) and not bool(wide[:, :3].any()) and not bool(wide[:, 43:].any())


@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_pitches(ops, dtype, p):
    """Aligned rows with a ragged end, rows that are one row, rows two gigabytes apart."""
    x = rand(1, 30, 44, dtype=dtype)
    want = x.double().cpu() * f.mask(30, 44, p, 8, 1)
    wide = torch.zeros(30, 64, dtype=dtype, device="cuda")
    wide[:, :44] = x
    tol = (f.STEP[dtype] + 2 * U) * want.abs() + LEAST[dtype]
    near(ops.dropout(wide[:, :44], p, 8, 1), want, tol)
    ops.dropout_(wide[:, :44], p, 8, 1)
    near(wide[:, :44], want, tol)
    assert not bool(wide[:, 44:].any())
    one = x[:1].expand(30, 44)
    assert torch.equal(ops.dropout(one, p, 8, 1), ops.dropout(one.contiguous(), p, 8, 1))
    far = torch.empty((3 << 30) // x.element_size(), dtype=dtype, device="cuda").as_strided((2, 44), ((3 << 29) // x.element_size(), 1))
    far.copy_(x[:2])
    assert torch.equal(ops.dropout(far, p, 8, 1), ops.dropout(x[:2], p, 8, 1))


def test_changes_in_place_are_seen_by_autograd(ops):
    x, w = rand(1, 8, 16), rand(2, 8, 16).requires_grad_()
    y = x * w  # saves x
    ops.dropout_(x, 0.5, 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        ops.dropout_(rand(1, 8, 16), 0.5, 1)


def test_differentiable_once(ops):
    x = rand(1, 8, 16).requires_grad_()
    for out in (ops.dropout(x, 0.5, 1), ops.add_rms_norm(x)[0]):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_dropped_infinities_and_nan_are_zero(ops):
    x = torch.full((8, 64), float("inf"), device="cuda")
    x[::2] = float("nan")
    m = f.mask(8, 64, 0.5, 3, 0)
    y = ops.dropout(x, 0.5, 3).cpu()
    assert bool((y[m == 0] == 0).all()) and not bool(torch.isfinite(y[m > 0]).any())


def test_rows_far_apart(ops):
    """Element offsets beyond 2^32."""
    big = torch.empty(5 << 30, dtype=torch.bfloat16, device="cuda")
    rows = big.as_strided((5, 24), (1 << 30, 1))
    rows.copy_(rand(1, 5, 24, dtype=torch.bfloat16))
    assert torch.equal(ops.dropout(rows, 0.5, 1), ops.dropout(rows.contiguous(), 0.5, 1))
    y, _ = ops.add_rms_norm(rows)
    assert torch.equal(y, ops.add_rms_norm(rows.contiguous())[0])
    ops.dropout_(rows, 0.5, 1)
    assert torch.equal(rows[4], ops.dropout(rand(1, 5, 24, dtype=torch.bfloat16), 0.5, 1)[4])


def test_rows_beyond_32_bit_elements(ops):
    """More than 2^32 elements in all; the last rows are checked."""
    rows, dim = (1 << 29) + 5, 8
    x = torch.ones(rows, dim, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout_(x, 0.5, 6, 2)
    assert torch.equal(y[-7:].cpu().double(), f.mask(7, dim, 0.5, 6, 2, first_row=rows - 7))


# -------------------------------------------------------------------- norm --
def norm_case(rows, dim, dtype, p, with_res, weight):
    x = rand(1, rows, dim, dtype=dtype, scale=2.0)
    res = rand(2, rows, dim, dtype=dtype) if with_res else None
    w = None if weight is None else (1 + 0.3 * rand(3, dim)).to(weight)
    if rows > 2:
        x[1] = 0
        if with_res:
            res[1] = 0  # a vertex without features: h = 0
    m = f.mask(rows, dim, p, 11, 5) if p else None
    return x, w, res, m


def wide(t):
    return None if t is None else t.detach().to(torch.float64).cpu()


def norm_bounds(x, w, res, m, dtype, eps):
    """Bounds of |y - y*| and |h - h*|."""
    y, h = f.norm(wide(x), wide(w), wide(res), eps, m)
    # h in float32: the scaled x is off by 2u, the sum by u
    dh32 = 2 * U * (wide(x).abs() * (1 if m is None else m)) + U * h.abs()
    r = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    # mean of squares: at most 32 additions in a thread and 14 across threads, each u relative to a sum of
    # positive terms, the squares u and 2 dh32 each (norm-wise no more than the largest ratio's 3u + 2u); half of
    # that in the root; rsqrtf 2 steps (4u), division and two products 3u: 40u in all
    rw = r if w is None else r * wide(w).abs()
    ty = f.STEP[dtype] * y.abs() * (1 + 2 ** -8) + 40 * U * y.abs() + rw * dh32 + LEAST[dtype]
    ss = (dh32 * h.abs()).sum(1, keepdim=True) / (h * h).sum(1, keepdim=True).clamp_min(1e-300)
    ty = ty + y.abs() * ss
    return y, h, ty, f.STEP[dtype] * h.abs() * (1 + 2 ** -8) + dh32 + LEAST[dtype], r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_norm_forward(ops, rows, dim, dtype):
    for p, with_res, weight in ((0.0, True, dtype), (0.25, True, torch.float32), (0.0, False, None), (0.5, False, dtype)):
        x, w, res, m = norm_case(rows, dim, dtype, p, with_res, weight)
        y, h = ops.add_rms_norm(x, w, res, eps=1e-5, p=p, seed=11, offset=5)
        wy, wh, ty, th, _ = norm_bounds(x, w, res, m, dtype, float(torch.tensor(1e-5)))
        near(y, wy, ty, f"y p {p}")
        near(h, wh, th, f"h p {p}")
        if not p and not with_res:
            assert h is x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", SHAPES + [(40_000, 24)])
def test_norm_gradients(ops, rows, dim, dtype):
    for p, with_res, weight, use in ((0.0, True, dtype, "yh"), (0.25, True, torch.float32, "yh"), (0.0, False, None, "y"),
                                     (0.5, False, dtype, "h"), (0.25, True, dtype, "y")):
        x, w, res, m = norm_case(rows, dim, dtype, p, with_res, weight)
        leaves = [t for t in (x, w, res) if t is not None]
        for t in leaves:
            t.requires_grad_()
        y, h = ops.add_rms_norm(x, w, res, eps=1e-5, p=p, seed=11, offset=5)
        dy, dh = rand(4, rows, dim, dtype=dtype), rand(5, rows, dim, dtype=dtype)
        outs, gs = zip(*[(o, g) for o, g, n in ((y, dy, "y"), (h, dh, "h")) if n in use])
        got = dict(zip(("x", "w", "res") if w is not None and res is not None else ("x", "w") if w is not None else ("x", "res") if
                       res is not None else ("x",), torch.autograd.grad(outs, leaves, gs, allow_unused=True)))
        eps = float(torch.tensor(1e-5))
        _, h64, _, th, r = norm_bounds(x, w, res, m, dtype, eps)
        zero = torch.zeros_like(h64)
        dy64, dh64 = (wide(dy) if "y" in use else zero), (wide(dh) if "h" in use else zero)
        g = dy64 if w is None else dy64 * wide(w)
        s = (g * h64).sum(1, keepdim=True)
        t = dh64 + r * g - h64 * r ** 3 / dim * s
        # h comes back rounded to its type (th); sums as in the forward pass; r is off by 50u
        mag = (g.abs() * h64.abs()).sum(1, keepdim=True)
        off_s = (g.abs() * th).sum(1, keepdim=True) + 50 * U * mag
        bound = (60 * U * (r * g.abs() + h64.abs() * r ** 3 / dim * mag + dh64.abs()) +
                 r ** 3 / dim * (th * s.abs() + (h64.abs() + th) * off_s))
        step = f.STEP[dtype] * (1 + 2 ** -7)
        if res is not None:
            near(got["res"], t, bound + step * t.abs() + LEAST[dtype], f"res p {p}")
        mm = 1.0 if m is None else m
        near(got["x"], t * mm, (bound + (step + 3 * U) * t.abs()) * mm + LEAST[dtype], f"x p {p}")
        if w is not None:
            if "y" not in use:
                assert got["w"].shape == w.shape and not bool(got["w"].any())
                continue
            dw = (dy64 * h64 * r).sum(0)
            mags = (dy64.abs() * h64.abs() * r).sum(0)
            off = (dy64.abs() * th * r).sum(0) + (60 + rows / 8) * U * mags  # a thread adds at most rows / 8 in a row
            near(got["w"], dw, off + f.STEP[weight] * (1 + 2 ** -7) * (dw.abs() + off) + LEAST[weight], f"w p {p}")


def test_norm_gradient_against_differences(ops):
    """d loss along a random direction against central differences of the 64-bit formula."""
    x, w, res, m = norm_case(13, 77, torch.float32, 0.25, True, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, res)]
    y, h = ops.add_rms_norm(x, w, res, p=0.25, seed=11, offset=5)
    dy, dh = rand(4, 13, 77), rand(5, 13, 77)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))

    def loss(*at):
        y, h = f.norm(at[0], at[1], at[2], 1e-6, m)
        return float((y * wide(dy)).sum() + (h * wide(dh)).sum())

    at = [wide(t) for t in leaves]
    at[0][1] += 0.5  # a zero row turns too sharply for differences: eps is its whole norm
    x2 = at[0].float().cuda().requires_grad_()
    grads = torch.autograd.grad(ops.add_rms_norm(x2, w, res, p=0.25, seed=11, offset=5), (x2, w, res), (dy, dh))
    for i, g in enumerate(grads):
        d = wide(rand(20 + i, *g.shape))
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - 1e-5 * d, at[i] + 1e-5 * d
        want, got = (loss(*hi) - loss(*lo)) / 2e-5, float((wide(g) * d).sum())
        # differences: 1e-10 of a third derivative of about 1e3, rounding 1e-13 / 1e-5; gradients: 1e-5 of the terms
        assert abs(want - got) < 1e-5 * float((wide(g) * d).abs().sum()) + 1e-6


@pytest.mark.parametrize("dim,left,pitch", [(301, 7, 333), (100, 6, 134), (96, 8, 128)])
def test_norm_bits_repeat_and_layouts(ops, dim, left, pitch):
    x, w, res, _ = norm_case(3000, dim, torch.bfloat16, 0.1, True, torch.bfloat16)
    dy = rand(6, 3000, dim, dtype=torch.bfloat16)

    def all_of(x, res, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, res)]
        y, h = ops.add_rms_norm(*leaves, p=0.1, seed=3)
        return (y, h, *torch.autograd.grad((y, h), leaves, (dy, dy)))

    first = all_of(x, res, dy)
    pad = torch.zeros(3, 3000, pitch, dtype=torch.bfloat16, device="cuda")
    for i, t in enumerate((x, res, dy)):
        pad[i, :, left:left + dim] = t
    for again in (all_of(x, res, dy), all_of(*(pad[i, :, left:left + dim] for i in range(3))),
                  all_of(*(t.t().contiguous().t() for t in (x, res, dy)))):
        for a, b in zip(first, again):
            assert torch.equal(a, b)


def test_norm_partial_gradients(ops):
    """Each leaf alone, and dy expanded from one value."""
    x, w, res, _ = norm_case(20, 48, torch.float32, 0.5, True, torch.float32)
    full = [t.detach().requires_grad_() for t in (x, w, res)]
    y, h = ops.add_rms_norm(*full, p=0.5, seed=2)
    want = torch.autograd.grad(y.sum() + h.sum() * 2, full)
    for i in range(3):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, res))]
        y, h = ops.add_rms_norm(*leaves, p=0.5, seed=2)
        (got,) = torch.autograd.grad(y.sum() + h.sum() * 2, leaves[i])
        assert torch.equal(got, want[i])
    same = x.detach().requires_grad_()  # branch and residual are one tensor
    y, h = ops.add_rms_norm(same, None, same)
    (got,) = torch.autograd.grad(h.sum(), same)
    assert torch.equal(got, torch.full_like(got, 2.0))


def test_norm_of_no_rows_and_extremes(ops):
    y, h = ops.add_rms_norm(torch.empty(0, 32, device="cuda").requires_grad_(), torch.ones(32, device="cuda").requires_grad_())
    assert y.shape == (0, 32)
    w = torch.ones(32, device="cuda").requires_grad_()
    y, _ = ops.add_rms_norm(torch.empty(0, 32, device="cuda"), w)
    assert not bool(torch.autograd.grad(y.sum(), w)[0].any())
    x = torch.zeros(4, 40, device="cuda")
    x[1, 7], x[2, 3] = float("nan"), float("inf")
    x[3] = 2.0 ** -130  # subnormal: the mean of squares is 0, eps alone is left
    y, _ = ops.add_rms_norm(x)
    assert bool((y[0] == 0).all()) and bool(y[1].isnan().all()) and bool(y[2, 3].isnan()) and bool(y[3].isfinite().all())


# ------------------------------------------------------------- 8-bit rows --
def check_f8(codes, scales, want, tol, rows_of=1):
    """codes * scales against `want`, known to `tol` before its encoding."""
    rows, dim = want.shape
    peak = f.block_peaks(want, rows_of)
    loose = f.block_peaks(tol, rows_of)
    s = scales.to(torch.float64).cpu()
    near(s, (peak / f.E4M3_MAX).clamp_min(f.TINY), loose / f.E4M3_MAX + 4 * U * peak / f.E4M3_MAX + 2.0 ** -149, "scales")
    per = s.repeat_interleave(rows_of, 0).repeat_interleave(128, 1)[:rows, :dim]
    got = codes.to(torch.float64).cpu() * per
    # half a step of e4m3: 2^-4 of a normal value, 2^-10 of the scale below; reciprocal and product 3u
    near(got, want, tol + (2.0 ** -4 + 2.0 ** -20) * (want.abs() + tol) + 2.0 ** -10 * per, "values")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_norm_f8(ops, rows, dim, dtype):
    for with_res, weight in ((True, dtype), (False, None)):
        x, w, res, _ = norm_case(rows, dim, dtype, 0.0, with_res, weight)
        codes, scales, h = ops.add_rms_norm_f8(x, w, res, eps=1e-5)
        wy, wh, ty, th, _ = norm_bounds(x, w, res, None, torch.float32, float(torch.tensor(1e-5)))
        check_f8(codes, scales, wy, ty)
        near(h, wh, th + f.STEP[dtype] * wh.abs() * 2 + LEAST[dtype], "h")
        assert codes.stride(0) % 16 == 0 and codes.dtype == torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_encode(ops, rows, dim, dtype):
    x = rand(7, rows, dim, dtype=dtype, scale=30.0)
    if rows > 2:
        x[2] = 0
    codes, scales = ops.encode_f8(x)
    check_f8(codes, scales, wide(x), torch.zeros(rows, dim, dtype=torch.float64))
    codes, scales = ops.encode_weight_f8(x)
    check_f8(codes, scales, wide(x), torch.zeros(rows, dim, dtype=torch.float64), 128)


def test_encode_values_that_are_not_finite(ops):
    x = rand(7, 6, 300)
    x[1, 130], x[2, 299], x[3, 0] = float("inf"), float("nan"), 3e38
    x[4], x[5] = 1e-42, 0
    got = ops.decode_f8(*ops.encode_f8(x))
    nan = got.isnan()
    assert bool(nan[1, 128:256].all()) and bool(nan[2, 256:].all()) and int(nan.sum()) == 128 + 44
    assert bool((got[5] == 0).all()) and bool((got[4].abs() <= 2.0 ** -126).all()) and abs(float(got[3, 0]) / 3e38 - 1) <= 2.0 ** -4


@pytest.mark.parametrize("dim", [1, 4, 31, 100, 128, 130, 301, 512])
def test_store_of_8_bit_rows(ops, dim):
    from aethergraph_b200 import FeatureStore

    x = rand(8, 200, dim)
    codes, scales = ops.encode_f8(x)
    made, viewed = FeatureStore.from_array(x, "f8"), FeatureStore.from_f8(codes, scales)
    want = f.decode(codes.cpu(), scales.cpu()).float()
    ids = torch.tensor([5, 199, 0, 5, 77], device="cuda")
    for store in (made, viewed):
        assert (store.dtype, store.num_nodes, store.feature_dim) == ("f8", 200, dim)
        assert torch.equal(store.gather(ids).cpu(), want[ids.cpu()])
        assert torch.equal(torch.from_numpy(store.features()), want)
        assert torch.equal(torch.from_numpy(store.payload_to_host()).view(200, dim), codes.cpu().contiguous().view(torch.uint8))
        assert torch.equal(torch.from_numpy(store.scales_to_host()), scales.cpu())
    assert torch.equal(ops.decode_f8(codes, scales).cpu(), want)
    with pytest.raises(ValueError):
        FeatureStore.from_array(torch.full((2, dim), float("nan"), device="cuda"), "f8")


# ----------------------------------------------------------------- product --
def product_case(rows, dim, out, seed=1):
    from aethergraph_b200 import ops

    x, w = rand(seed, rows, dim), rand(seed + 1, out, dim)
    x *= 2.0 ** torch.randint(-6, 7, (rows, 1), device="cuda")  # scales far apart
    if rows > 2:
        x[1] = 0
    return (*ops.encode_f8(x), *ops.encode_weight_f8(w))


def check_product(got, a, sa, w, sw, ids=None, bias=None, dtype=torch.bfloat16):
    A, W = f.decode(a.cpu(), sa.cpu()), f.decode_weight(w.cpu(), sw.cpu())
    if ids is not None:
        A = A[ids.cpu().long()]
    want, mags = A @ W.t(), A.abs() @ W.abs().t()
    if bias is not None:
        want, mags = want + wide(bias), mags + wide(bias).abs()
    # the products are exact; at most 128 additions in a block, two products and an addition for each
    # block, the bias: every one within a step (2u) of float32
    blocks = -(-a.shape[1] // 128)
    near(got, want, f.STEP[dtype] * (1 + 2 ** -7) * want.abs() + (128 + 3 * blocks + 2) * 2 * U * mags + LEAST[dtype], "product")


PRODUCTS = [(1, 16, 1), (1, 1024, 1024), (2, 100, 47), (4, 128, 128), (5, 129, 129), (17, 301, 33), (64, 512, 200), (127, 64, 256),
            (128, 1, 8), (129, 256, 130), (300, 602, 172), (1000, 384, 512), (2049, 2000, 96), (700, 1433, 7)]


@pytest.mark.parametrize("rows,dim,out", PRODUCTS)
def test_product(ops, rows, dim, out):
    case = product_case(rows, dim, out)
    for dtype in TYPES:
        bias = rand(5, out) if dtype == torch.bfloat16 else None
        got = ops.product_f8(*case, bias=bias, dtype=dtype)
        assert got.dtype == dtype
        check_product(got, *case, bias=bias, dtype=dtype)


@pytest.mark.parametrize("rows,dim,out", PRODUCTS)
def test_product_by_id(ops, rows, dim, out):
    held = 50
    case = product_case(held, dim, out)
    for kind in (torch.int64, torch.int32):
        ids = torch.randint(0, held, (rows,), generator=torch.Generator().manual_seed(rows), dtype=kind).cuda()
        got = ops.product_f8(*case, ids=ids)
        check_product(got, *case, ids=ids)
        assert torch.equal(got, ops.product_f8(_take(case[0], ids), case[1][ids.long()], *case[2:]))


def _take(codes, ids):
    rows = torch.zeros(len(ids), codes.stride(0), dtype=torch.uint8, device="cuda")
    rows[:, :codes.shape[1]] = codes.view(torch.uint8)[ids.long()]
    return rows.view(torch.float8_e4m3fn)[:, :codes.shape[1]]


@pytest.mark.parametrize("rows", [3, 200])
def test_product_ids_outside(ops, rows):
    case = product_case(20, 256, 64)
    ids = torch.randint(0, 20, (rows,), device="cuda")
    good = ops.product_f8(*case, ids=ids)
    ops.check()
    ids[1] = 20
    ids[rows - 1] = -1
    got = ops.product_f8(*case, ids=ids)
    with pytest.raises(ValueError, match="out of bounds"):
        ops.check()
    ops.check()
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[[1, rows - 1]] = True
    assert not bool(got[bad.cuda()].any()) and torch.equal(got[~bad.cuda()], good[~bad.cuda()])


@pytest.mark.parametrize("dim", [100, 602])
@pytest.mark.parametrize("rows", [3, 150])
def test_product_reads_nothing_beside_its_rows(ops, rows, dim):
    """NaN codes in the pitch's padding, NaN scales of a row that only ids outside would fall back on."""
    a, sa, w, sw = product_case(rows, dim, 70)
    good = ops.product_f8(a, sa, w, sw)
    wide = [torch.full((len(t), t.stride(0) + 16), 0x7F, dtype=torch.uint8, device="cuda") for t in (a, w)]
    for t, v in zip(wide, (a, w)):
        t[:, :dim] = v.view(torch.uint8)
    na, nw = (t.view(torch.float8_e4m3fn)[:, :dim] for t in wide)
    assert torch.equal(ops.product_f8(na, sa, nw, sw), good)
    ids = torch.arange(rows, device="cuda")
    assert torch.equal(ops.product_f8(na, sa, nw, sw, ids=ids), good)
    sa[0] = float("nan")
    ids[:] = rows
    ids[1] = 1
    got = ops.product_f8(na, sa, nw, sw, ids=ids, bias=torch.full((70,), 3.0, device="cuda"))
    assert bool(got[1].isfinite().all()) and not bool(got[0].any()) and not bool(got[2:].any())
    with pytest.raises(ValueError, match="out of bounds"):
        ops.check()


@pytest.mark.parametrize("rows", [2, 300])
def test_product_of_nan_rows_stays_in_them(ops, rows):
    a, sa, w, sw = product_case(rows, 300, 200)
    good = ops.product_f8(a, sa, w, sw)
    sa[0, 1] = float("nan")
    got = ops.product_f8(a, sa, w, sw)
    assert bool(got[0].isnan().all()) and torch.equal(got[1:], good[1:])
    assert ops.product_f8(a[:0], sa[:0], w, sw).shape == (0, 200)


@pytest.mark.parametrize("rows", [3, 500])
def test_product_of_slices(ops, rows):
    """Rows of a larger tensor: pitch wider than the row, rows and weights from the middle."""
    a, sa, w, sw = product_case(rows + 7, 512, 384)
    got = ops.product_f8(a[5:5 + rows, 128:320], sa[5:5 + rows, 1:3].contiguous(), w[128:330, 128:320], sw[1:3, 1:3].contiguous())
    check_product(got, a[5:5 + rows, 128:320].contiguous(), sa[5:5 + rows, 1:3], w[128:330, 128:320].contiguous(), sw[1:3, 1:3])


@pytest.mark.parametrize("out", [96, 128, 200])
def test_product_bias_anywhere(ops, out):
    case = product_case(140, 256, out)
    many = rand(5, out + 1)
    for bias in (many[:out].contiguous(), many[1:]):
        check_product(ops.product_f8(*case, bias=bias, dtype=torch.float32), *case, bias=bias, dtype=torch.float32)


def test_refusals(ops):
    a, sa, w, sw = product_case(8, 64, 16)
    x = rand(1, 8, 64)
    for call in (lambda: ops.dropout(x, 1.5, 1), lambda: ops.dropout(x, 0.5, -1), lambda: ops.dropout(x, 0.5, 1, 1 << 64),
                 lambda: ops.dropout(x.double(), 0.5, 1), lambda: ops.dropout(x[:, :0], 0.5, 1), lambda: ops.dropout(x.sum(), 0.5, 1),
                 lambda: ops.dropout_(x.t(), 0.5, 1), lambda: ops.dropout_(x.clone().requires_grad_(), 0.5, 1),
                 lambda: ops.dropout_(x[:1].expand(8, 64), 0.5, 1),
                 lambda: ops.add_rms_norm(x, torch.ones(63, device="cuda")), lambda: ops.add_rms_norm(x, None, x[:4]),
                 lambda: ops.add_rms_norm(x, None, x.half()), lambda: ops.add_rms_norm(rand(1, 2, 16385)),
                 lambda: ops.add_rms_norm(x.half(), torch.ones(64, device="cuda", dtype=torch.bfloat16)),
                 lambda: ops.add_rms_norm_f8(x.clone().requires_grad_()), lambda: ops.encode_weight_f8(x[0]),
                 lambda: ops.product_f8(a, sa[:4], w, sw), lambda: ops.product_f8(a[:, :63], sa, w, sw),
                 lambda: ops.product_f8(a[:, 8:], sa, w[:, 8:], sw), lambda: ops.product_f8(a, sa, w, sw, ids=torch.zeros(3, device="cuda")),
                 lambda: ops.product_f8(a, sa, w, sw, ids=torch.zeros(3, dtype=torch.int64)),
                 lambda: ops.product_f8(a, sa, w, sw, bias=torch.zeros(15, device="cuda")),
                 lambda: ops.product_f8(a, sa, w, sw, dtype=torch.float64), lambda: ops.product_f8(a, sa, w[:0], sw[:0])):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------- streams and graphs --
def test_other_stream_and_captured_graph(ops):
    """The whole layer on another stream, and captured twice and replayed over new inputs.  The eager calls'
    autograd graphs are gone by then: PyTorch cannot capture a backward pass while one of the same
    leaves, made on another stream, is alive."""
    x, w, res, _ = norm_case(600, 256, torch.bfloat16, 0.2, True, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, res)]
    dy = rand(9, 600, 256, dtype=torch.bfloat16)
    wc, ws = ops.encode_weight_f8(rand(10, 96, 256))

    def layer():
        y, h = ops.add_rms_norm(*leaves, p=0.2, seed=4, offset=1)
        d = ops.dropout(y, 0.1, 4, 2)
        grads = torch.autograd.grad((d, h), leaves, (dy, dy))
        with torch.no_grad():
            out = ops.product_f8(*ops.add_rms_norm_f8(d, w)[:2], wc, ws)
        return (y.detach(), h.detach(), d.detach(), out, *grads)

    eager = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = layer()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = layer()
    with torch.cuda.graph(g2):
        captured2 = layer()
    with torch.no_grad():
        x.copy_(rand(30, 600, 256, dtype=torch.bfloat16))
    want = layer()
    for _ in range(2):
        g.replay()
        g2.replay()
    for a, b, c in zip(want, captured, captured2):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_two_streams_at_once(ops):
    """Calls that overlap share nothing."""
    x, w, res, _ = norm_case(4000, 512, torch.bfloat16, 0.1, True, torch.bfloat16)
    dy = rand(6, 4000, 512, dtype=torch.bfloat16)
    case = product_case(3000, 640, 384)

    def work():
        leaves = [t.detach().requires_grad_() for t in (x, w, res)]
        y, h = ops.add_rms_norm(*leaves, p=0.1, seed=3)
        return [y.detach(), *torch.autograd.grad((y, h), leaves, (dy, dy)), ops.product_f8(*case)]

    want = work()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


# ------------------------------------------------------------ as they are used --
def test_layers_over_a_sampled_batch(ops):
    """Sampled batch -> projection straight from 8-bit rows -> dropout + norm -> 8-bit rows -> next store -> next product."""
    import aethergraph_b200 as ag
    from aethergraph_b200 import synth

    n, dim, hidden = 5000, 100, 72
    g = synth.rmat_graph(n, 60_000, seed=1)
    store = ag.FeatureStore.from_array(rand(1, n, dim), "f8")
    loader = ag.NeighborLoader(g, ag.SamplingConfig(num_neighbors=[10, 5], seed=3), features=store)
    with loader:
        loader.submit(0, synth.seed_batch(n, 64, 3, 0))
        _, sg, x = loader.next_batch()
        n_id = sg.nodes_t.clone()
        decoded = x.clone()
    assert torch.equal(decoded, store.gather(n_id))
    w1, w2 = rand(2, hidden, dim), rand(3, 32, hidden)
    c1, c2 = ops.encode_weight_f8(w1), ops.encode_weight_f8(w2)
    h1 = store.project(n_id, *c1)
    store.check()
    W = f.decode_weight(c1[0].cpu(), c1[1].cpu())
    want = decoded.double().cpu() @ W.t()
    near(h1, want, 2.0 ** -8 * 1.01 * want.abs() + 300 * U * (decoded.double().abs().cpu() @ W.abs().t()), "projection")
    codes, scales, h = ops.add_rms_norm_f8(h1, torch.ones(hidden, device="cuda"), h1)
    nxt = ag.FeatureStore.from_f8(codes, scales)
    ids = torch.arange(0, len(n_id), 2, device="cuda", dtype=torch.int32)
    out = nxt.project(ids, *c2, dtype=torch.float32)
    assert torch.equal(out, ops.product_f8(codes, scales, *c2, ids=ids, dtype=torch.float32))
    check_product(out, codes, scales, *c2, ids=ids, dtype=torch.float32)
    with pytest.raises(ValueError):
        ag.FeatureStore.from_array(rand(1, 4, 8)).project(ids, *c2)


@pytest.mark.parametrize("dim", [21, 64])
def test_typed_batches_over_8_bit_rows(dim):
    """8-bit stores beside others in the loader of a typed graph."""
    import numpy as np

    import aethergraph_b200 as ag

    rng = np.random.default_rng(3)
    e = lambda n, a, b: (rng.integers(0, a, n).astype(np.uint32), rng.integers(0, b, n).astype(np.uint32))  # noqa: E731
    h = ag.HeteroCsrGraph.from_edge_arrays({"a": 300, "b": 200}, [("a", "to", "b", *e(3000, 300, 200)), ("b", "to", "a", *e(3000, 200, 300))])
    stores = {"a": ag.FeatureStore.from_array(rand(1, 300, dim), "f8"), "b": ag.FeatureStore.from_array(rand(2, 200, dim), "bf16")}
    cfg = ag.HeteroSamplingConfig({("a", "to", "b"): [4, 3], ("b", "to", "a"): [4, 3]}, seed=1)
    loader = ag.HeteroNeighborLoader(h, cfg, "b", prefetch_depth=2, features=stores)
    for i in range(3):
        loader.submit(i, np.arange(i * 20, i * 20 + 20))
    for _ in range(3):
        _, sg = loader.next_batch()
        for t in ("a", "b"):
            assert torch.equal(sg.x_t(t), stores[t].gather(sg.nodes_t(t)))
    loader.shutdown()
