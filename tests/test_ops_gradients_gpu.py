"""Gradients of the norm against the definition's, from the h of 32 bits that the forward pass normalised.

The bounds hold no rounding of h to the rows' type: with u = 2^-24, h is off by 2u of the scaled x and u of the sum, its
reciprocal root by 50u and what h's error makes of it, and every product and sum after that by u each.
"""
import pytest
import torch

import ops_formulas as f
from test_ops_gpu import LEAST, U, near, norm_case, ops, rand, wide  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu

# lane groups, several chunks a lane, whole blocks of one, two and four chunks a thread: aligned, even and odd lengths
SHAPES = [(33, 17), (257, 64), (19, 100), (41, 301), (12, 602), (300, 512), (300, 1040), (7, 1031), (170, 2050), (3, 4099), (170, 9000), (5, 9002), (2, 16384)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_norm_gradients_of_the_unrounded_sum(ops, rows, dim, dtype):  # noqa: F811
    eps = float(torch.tensor(1e-5))
    for p, with_res in ((0.25, True), (0.5, False), (0.0, True)):
        x, w, res, m = norm_case(rows, dim, dtype, p, with_res, torch.float32)
        names = ["x", "w"] + ["res"] * with_res
        leaves = [t.requires_grad_() for t in (x, w, res) if t is not None]
        y, h = ops.add_rms_norm(x, w, res, eps=1e-5, p=p, seed=11, offset=5)
        dy, dh = rand(4, rows, dim, dtype=dtype), rand(5, rows, dim, dtype=dtype)
        got = dict(zip(names, torch.autograd.grad((y, h), leaves, (dy, dh))))
        _, h64 = f.norm(wide(x), wide(w), wide(res), eps, m)
        r = 1 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + eps)
        off_h = 2 * U * (wide(x).abs() * (1 if m is None else m)) + U * h64.abs()
        off_r = 50 * U + (off_h * h64.abs()).sum(1, keepdim=True) / (h64 * h64).sum(1, keepdim=True).clamp_min(1e-300)  # relative
        g = wide(dy) * wide(w)
        s, mag = (g * h64).sum(1, keepdim=True), (g.abs() * h64.abs()).sum(1, keepdim=True)
        off_s = (g.abs() * off_h).sum(1, keepdim=True) + 50 * U * mag  # at most 32 additions in a thread and 14 across
        t = wide(dh) + r * g - h64 * r ** 3 / dim * s
        bound = (3 * off_r + 10 * U) * (r * g.abs() + h64.abs() * r ** 3 / dim * mag + wide(dh).abs()) + \
            r ** 3 / dim * (off_h * s.abs() + (h64.abs() + off_h) * off_s)
        step = f.STEP[dtype] * (1 + 2 ** -7)
        if with_res:
            near(got["res"], t, bound + step * (t.abs() + bound) + LEAST[dtype], f"res p {p}")
        mm = 1.0 if m is None else m
        near(got["x"], t * mm, (bound + (step + 3 * U) * (t.abs() + bound)) * mm + LEAST[dtype], f"x p {p}")
        mags = (wide(dy).abs() * h64.abs() * r).sum(0)
        off = (wide(dy).abs() * (off_h + off_r * h64.abs()) * r).sum(0) + (20 + rows / 8) * U * mags
        near(got["w"], (wide(dy) * h64 * r).sum(0), off, f"w p {p}")


@pytest.mark.parametrize("dim", [64, 301])
def test_gradients_of_a_sum_beyond_the_rows_type(ops, dim):  # noqa: F811
    """x + residual passes float16's largest value: h is infinite in float16, y and the gradients of y are not."""
    x, res = (torch.full((4, dim), 4e4, dtype=torch.float16, device="cuda").requires_grad_() for _ in range(2))
    w = torch.ones(dim, device="cuda", requires_grad=True)
    y, h = ops.add_rms_norm(x, w, res)
    assert bool(h.isinf().all())
    dy = rand(4, 4, dim, dtype=torch.float16)
    dx, dw, dres = torch.autograd.grad(y, (x, w, res), dy)
    # y = 1 within 40u, rounded to 1; dw sums dy h r = dy; dx is below float16's steps of dy / 8e4
    near(dw, wide(dy).sum(0), 60 * U * wide(dy).abs().sum(0))
    assert bool(dx.isfinite().all()) and torch.equal(dx, dres) and float(dx.abs().max()) < 2 * float(dy.abs().max()) / 8e4


def test_what_the_gradients_are_made_of_is_watched(ops):  # noqa: F811
    """16-bit rows: x and residual, changed in place before the backward pass, are noticed."""
    x, w, res, _ = norm_case(8, 64, torch.bfloat16, 0.0, True, torch.bfloat16)
    w.requires_grad_()
    for i in range(2):
        y, h = ops.add_rms_norm(x, w, res, p=0.5, seed=1)
        (x, res)[i].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y.sum(), w)
    # made again from rows with a pitch of their own, and from rows laid out otherwise
    wide_x = torch.zeros(8, 96, dtype=torch.bfloat16, device="cuda")
    wide_x[:, 8:72] = x
    want = torch.autograd.grad(ops.add_rms_norm(x, w, res, p=0.5, seed=1)[0].sum(), w)[0]
    for a, b in ((wide_x[:, 8:72], res), (x, res.t().contiguous().t()), (wide_x[:, 8:72].unflatten(0, (2, 4)), res.view(2, 4, 64))):
        assert torch.equal(torch.autograd.grad(ops.add_rms_norm(a, w, b, p=0.5, seed=1)[0].sum(), w)[0], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_inference_mode(ops, dtype):  # noqa: F811
    """Branch or residual from a part of the model that runs in inference mode."""
    x, w, res, _ = norm_case(8, 64, dtype, 0.0, True, dtype)
    w.requires_grad_()
    want = torch.autograd.grad(ops.add_rms_norm(x, w, res, p=0.5, seed=1)[0].sum(), w)[0]
    with torch.inference_mode():
        x2, res2 = x.clone(), res.clone()
    for a, b in ((x2, res), (x, res2), (x2, res2)):
        assert torch.equal(torch.autograd.grad(ops.add_rms_norm(a, w, b, p=0.5, seed=1)[0].sum(), w)[0], want)
