"""Derivatives and transforms that the row operators do not have are refused, not lost."""
import pytest
import torch

from test_ops_cpu import _tangent_calls
from test_ops_gpu import ops, product_case, rand  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_tangents(ops, no_grad):  # noqa: F811
    fwd = torch.autograd.forward_ad
    a, sa, w8, sw = product_case(8, 64, 16)
    with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
        x, w, bias, scales = (fwd.make_dual(t, torch.ones_like(t)) for t in (rand(1, 4, 16), rand(2, 16), rand(3, 16), sa))
        for call in (*_tangent_calls(x, w, rand(4, 4, 16)), lambda: ops.product_f8(a, sa, w8, sw, bias=bias),
                     lambda: ops.product_f8(a, scales, w8, sw), lambda: ops.product_f8(a, sa, w8, fwd.make_dual(sw, sw))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
    torch.testing.assert_close(ops.dropout(rand(1, 4, 16), 0.0, 1), rand(1, 4, 16), rtol=0, atol=0)  # and nothing lingers


def test_functional_transforms(ops):  # noqa: F811
    x = rand(1, 4, 16)
    for call in (lambda: torch.func.grad(lambda v: ops.dropout(v, 0.5, 1).sum())(x), lambda: torch.func.jvp(lambda v: ops.dropout(v, 0.5, 1), (x,), (x,)),
                 lambda: torch.func.vmap(lambda v: ops.add_rms_norm(v)[0])(x), lambda: torch.func.vmap(lambda v: ops.dropout_(v, 0.5, 1))(x)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    assert torch.equal(x, rand(1, 4, 16))


def test_values_kept_with_the_other_sign(ops):  # noqa: F811
    """The imaginary part of a conjugate: memory holds the negative values."""
    z = torch.randn(40, 1, dtype=torch.complex64, device="cuda").conj()
    a, sa, w8, sw = product_case(8, 64, 16)
    other = lambda t: torch._neg_view(-t)  # noqa: E731
    for x in (z.imag, other(rand(1, 40, 24)), other(rand(1, 40, 24).bfloat16())):
        assert x.is_neg()
        same, w, res = x.resolve_neg(), rand(2, x.shape[1]), rand(3, *x.shape, dtype=x.dtype)
        assert torch.equal(ops.dropout(x, 0.5, 1), ops.dropout(same, 0.5, 1))
        for got, want in zip(ops.add_rms_norm(x, other(w), other(res), p=0.5, seed=1), ops.add_rms_norm(same, w, res, p=0.5, seed=1)):
            assert torch.equal(got, want)
        for call in (ops.encode_f8, ops.encode_weight_f8, ops.add_rms_norm_f8):
            for got, want in zip(call(x), call(same)):
                assert torch.equal(got.view(torch.uint8) if got.element_size() == 1 else got, want.view(torch.uint8) if want.element_size() == 1 else want)
        w.requires_grad_()
        grads = [torch.autograd.grad(ops.add_rms_norm(v, w, res, p=0.5, seed=1), w, (g, g))[0] for v, g in ((x, other(res)), (same, res))]
        assert torch.equal(*grads)
        with pytest.raises(ValueError):
            ops.dropout_(x, 0.5, 1)
    bias = rand(5, 16)
    assert torch.equal(ops.product_f8(a, sa, w8, sw, bias=other(bias)), ops.product_f8(a, sa, w8, sw, bias=bias))
    for call in (lambda: ops.product_f8(a, other(sa), w8, sw), lambda: ops.product_f8(a, sa, w8, other(sw)), lambda: ops.decode_f8(a, other(sa))):
        with pytest.raises(ValueError, match="scales"):
            call()
