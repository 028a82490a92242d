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
