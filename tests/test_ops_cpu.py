"""Row operators without a GPU: the random bits' definition, refusals before anything is launched."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import aethergraph_b200 as ag
from aethergraph_b200 import _lib, ops
from oracle import ago

import ops_formulas as f


def test_random_bits_are_the_frameworks_philox():
    seed, offset = 0x1234567890ABCDEF, 0xFEDCBA9800000007
    got = f.lots(5, 21, seed, offset)
    for r, c in ((0, 0), (0, 7), (3, 8), (4, 20), (2, 13)):
        words = ago.philox4x32_10(seed, offset & 0xFFFFFFFF, (r << 32) | (c // 8), offset >> 32)
        word = int(words[(c % 8) // 2])
        assert got[r, c] == (word >> 16 if c % 2 else word & 0xFFFF)


def test_mask_keeps_the_expected_share():
    m = f.mask(2000, 100, 0.25, 7, 0)
    kept = float((m > 0).double().mean())
    # 200 000 independent lots: standard deviation sqrt(.25 * .75 / 2e5) < 0.001; five of them
    assert abs(kept - 0.75) < 0.005
    assert abs(float(m.mean()) - 1.0) < 0.005 / 0.75


def test_ops_is_reached_from_the_package():
    assert ag.ops is ops and "ops" in ag.__all__


@pytest.mark.parametrize("call", [
    lambda x: ops.dropout(x, 0.5, 1), lambda x: ops.dropout_(x, 0.5, 1), lambda x: ops.add_rms_norm(x),
    lambda x: ops.add_rms_norm_f8(x), lambda x: ops.encode_f8(x), lambda x: ops.encode_weight_f8(x),
    lambda x: ops.product_f8(x, x, x, x), lambda x: ag.FeatureStore.from_f8(x, x)])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="CUDA tensor"):
        call(torch.zeros(4, 16))


def _dropout(rows=4, dim=8, dtype=0, p=0.5, ptr=16, y_stride=8):
    return _lib.lib().ag_rows_dropout(ptr, ptr, rows, dim, dim, y_stride, dtype, p, 1, 0, 0, None)


@pytest.mark.parametrize("kw,text", [
    (dict(p=-0.1), "probability"), (dict(p=1.5), "probability"), (dict(p=float("nan")), "probability"),
    (dict(dtype=3), "dtype tag"), (dict(dtype=-1), "dtype tag"), (dict(dim=0), "columns"), (dict(rows=1 << 32), "rows"),
    (dict(ptr=None), "null"), (dict(y_stride=7), "overlap")])
def test_dropout_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        _lib.check(_dropout(**kw))


def _norm(**kw):
    base = dict(x=16, y=16, rows=2, dim=8, x_stride=8, y_stride=8, dtype=0)
    base.update(kw)
    return _lib.lib().ag_rows_norm(C.byref(_lib.Norm(**base)), 0, None)


@pytest.mark.parametrize("kw,text", [
    (dict(dim=16385, y_stride=16385), "16384"), (dict(dim=0), "columns"), (dict(dtype=4), "dtype tag"), (dict(p=2.0), "probability"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(x_stride=1 << 32), "apart"), (dict(x=None), "null"), (dict(y=None), "null"), (dict(codes=16), "null"), (dict(codes=16, scales=16, code_stride=16), "either"),
    (dict(y=None, codes=16, scales=16, code_stride=8), "16 bytes"), (dict(y=None, codes=8, scales=16, code_stride=16), "16 bytes"),
    (dict(weight=16, dtype=1, weight_dtype=2), "weights"), (dict(encode_only=1), "encoding"), (dict(y_stride=4), "overlap"),
    (dict(h=16, h_stride=4), "overlap"), (dict(y=None, codes=16, scales=16, code_stride=16, encode_only=1, residual=16), "encoding")])
def test_norm_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        _lib.check(_norm(**kw))


def _product(**kw):
    base = dict(codes=16, scales=16, weight=16, weight_scales=16, out=16, rows=2, held=2, dim=16, out_dim=4, code_stride=16,
                weight_stride=16, out_stride=4, out_dtype=2)
    base.update(kw)
    return _lib.lib().ag_rows_product(C.byref(_lib.Product(**base)), 0, None)


@pytest.mark.parametrize("kw,text", [
    (dict(codes=None), "null"), (dict(out=None), "null"), (dict(out_dtype=3), "dtype tag"), (dict(dim=0), "range"),
    (dict(out_dim=0), "range"), (dict(rows=3), "held"), (dict(code_stride=24), "16 bytes"), (dict(codes=24), "16 bytes"),
    (dict(weight_stride=8), "16 bytes"), (dict(out_stride=3), "overlap"), (dict(held=1 << 31), "range"), (dict(rows=1 << 31), "range")])
def test_product_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        _lib.check(_product(**kw))


def test_weights_refusals():
    enc = _lib.lib().ag_rows_encode_weight
    for args in ((None, 4, 16, 16, 0, 16, 16, 16), (16, 4, 16, 16, 3, 16, 16, 16), (16, 4, 16, 16, 0, 16, 24, 16), (16, 4, 0, 16, 0, 16, 16, 16)):
        with pytest.raises(ValueError):
            _lib.check(enc(*args, 0, None))


def test_store_refusals():
    out = C.c_void_p()
    make = _lib.lib().ag_features_from_f8
    for args in ((None, 16, 4, 16, 16), (16, 16, 4, 16, 24), (16, 16, 4, 32, 16), (8, 16, 4, 16, 16), (16, 16, 4, 0, 16)):
        with pytest.raises(ValueError):
            _lib.check(make(*args, 0, C.byref(out)))


def test_formulas_agree_with_autograd_and_differences():
    """The gradient that the kernels are held to, against differences of the 64-bit formula."""
    rng = torch.Generator().manual_seed(3)
    x, res, dy, dh = (torch.randn(3, 11, generator=rng, dtype=torch.float64) for _ in range(4))
    w = torch.randn(11, generator=rng, dtype=torch.float64)
    m = f.mask(3, 11, 0.3, 5, 2)
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    y, h = f.norm(leaves[0], leaves[1], leaves[2], 1e-6, m)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))

    def loss(x, w, res):
        y, h = f.norm(x, w, res, 1e-6, m)
        return float((y * dy).sum() + (h * dh).sum())

    for i, g in enumerate(grads):
        d = torch.randn(g.shape, generator=rng, dtype=torch.float64)
        at = [x, w, res]
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - 1e-6 * d, at[i] + 1e-6 * d
        # central difference: 1e-12 of the third derivative, plus rounding 1e-15 / 1e-6
        assert abs((loss(*hi) - loss(*lo)) / 2e-6 - float((g * d).sum())) < 1e-6


def test_mask_of_all_and_nothing():
    assert bool((f.mask(3, 9, 0.0, 1, 0) == 1).all()) and bool((f.mask(3, 9, 1.0, 1, 0) == 0).all())
    assert np.array_equal(f.lots(4, 9, 1, 0)[2:], f.lots(2, 9, 1, 0, first_row=2))


def _norm_back(**kw):
    base = dict(dy=16, h=16, rstd=16, dx=16, rows=2, dim=8, dy_stride=8, h_stride=8, x_stride=8, residual_stride=8, dtype=1)
    base.update(kw)
    return _lib.lib().ag_rows_norm_backward(C.byref(_lib.NormGrad(**base)), 0, None)


@pytest.mark.parametrize("kw,text", [
    (dict(h=None), "null"), (dict(x=16), "either"), (dict(residual=16), "either"), (dict(h=None, x=16, dtype=0), "f32"),
    (dict(weight=16, weight_dtype=2), "weights"),
    (dict(dw=16, scratch=16, scratch_bytes=1 << 40, weight_dtype=3), "weights"), (dict(h=None, x=16, x_stride=1 << 32), "apart"), (dict(h=None, x=16, residual=16, residual_stride=1 << 32), "apart")])
def test_norm_gradient_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        _lib.check(_norm_back(**kw))


def _tangent_calls(x, w, plain):
    """Calls with a tangent in one of their arguments; `plain`: one without."""
    return [lambda: ops.dropout(x, 0.5, 1), lambda: ops.dropout_(x, 0.5, 1), lambda: ops.add_rms_norm(x), lambda: ops.add_rms_norm(plain, w),
            lambda: ops.add_rms_norm(plain, None, x), lambda: ops.add_rms_norm_f8(x), lambda: ops.add_rms_norm_f8(plain, w),
            lambda: ops.add_rms_norm_f8(plain, None, x), lambda: ops.encode_f8(x), lambda: ops.encode_weight_f8(x),
            lambda: ops.product_f8(plain, x, plain, plain)]


@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_tangents_are_refused(no_grad):
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        x, w = (torch.autograd.forward_ad.make_dual(torch.ones(*s), torch.ones(*s)) for s in ((4, 16), (16,)))
        for call in _tangent_calls(x, w, torch.ones(4, 16)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


def test_tracing_is_refused():
    x = torch.ones(4, 16)
    for call in (lambda v: ops.dropout(v, 0.5, 1), lambda v: ops.dropout_(v, 0.5, 1), lambda v: ops.add_rms_norm(v)[0], lambda v: ops.add_rms_norm_f8(v)[0],
                 lambda v: ops.encode_f8(v)[0], lambda v: ops.encode_weight_f8(v)[0], lambda v: ops.product_f8(v, v, v, v)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, x, check_trace=False)


@pytest.mark.parametrize("p", [0.0, 0.5])
def test_dropout_in_place_keeps_its_pitch(p):
    for strides in ((16, 8), (8, 16), (0, 8)):
        with pytest.raises(ValueError, match="in place"):
            _lib.check(_lib.lib().ag_rows_dropout(256, 256, 4, 8, *strides, 0, p, 1, 0, 0, None))


def test_the_package_needs_no_torch_until_it_is_used():
    """A star import, `ops` among its names, without torch and without the extension; the first call asks for both."""
    code = ("import sys; sys.modules['torch'] = None; sys.modules['aethergraph_b200._ops'] = None\n"
            "from aethergraph_b200 import *\n"
            "import aethergraph_b200 as ag\n"
            "assert ops is ag.ops and Graph is ag.Graph\n"
            "try: ops.dropout(None, 0.5, 1)\n"
            "except ImportError: print('asked')\n")
    got = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.strip() == "asked", got.stderr


def test_decode_refusals():
    for args in ((None, 16, 4, 16, 16, 16), (16, None, 4, 16, 16, 16), (16, 16, 4, 16, 16, None), (16, 16, 4, 0, 16, 16), (16, 16, 4, 16, 24, 16), (16, 16, 4, 32, 16, 16),
                 (8, 16, 4, 16, 16, 16), (16, 16, 4, 16, 1 << 32, 16)):
        with pytest.raises(ValueError):
            _lib.check(_lib.lib().ag_rows_decode(*args, 0, None))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.decode_f8(torch.zeros(4, 16), torch.zeros(4, 1))


def test_feature_dropout_of_nothing():
    """A node type without features, without rows in this batch, or with rows of no columns."""
    from aethergraph_b200.pytorch.loader import FeatureDropout

    drop = FeatureDropout(0.5, 1)
    assert drop(None, 0) is None
    for shape in ((0, 8), (5, 0), (0, 0)):
        x = torch.empty(shape)
        assert drop(x, 0) is x
