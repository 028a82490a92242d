"""The forms that many rows take, against 64 bits: norms whose blocks take a second row and several chunks a
thread, products of every tile width whose blocks take several tiles.  Bounds as derived in test_ops_gpu."""
import pytest
import torch

import ops_formulas as f
import test_ops_gpu as base
from test_ops_gpu import LEAST, TYPES, U, near, ops, product_case, rand  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu

# whole blocks of rows beyond the resident ones: aligned and not, two and four chunks a thread
NORMS = [(5000, 1024), (3001, 602), (2501, 1031), (1500, 4096), (700, 9000), (400, 16384)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", NORMS)
def test_norm(ops, rows, dim, dtype):  # noqa: F811
    base.test_norm_forward(ops, rows, dim, dtype)
    base.test_norm_f8(ops, rows, dim, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,dim", NORMS)
def test_norm_gradients(ops, rows, dim, dtype):  # noqa: F811
    base.test_norm_gradients(ops, rows, dim, dtype)


def width_of(rows, out, sms=148):
    """Tile width that the product takes, and tiles a block works on at most."""
    rounds = {w: -(-(-(-rows // 128) * -(-out // w)) // sms) for w in (128, 64, 32)}
    cost = {w: rounds[w] * c for w, c in ((128, 156), (64, 110), (32, 98))}
    width = min((128, 64, 32), key=lambda w: cost[w])
    return width, rounds[width]


# several tiles a block at every width; outputs that leave by TMA and not; columns cut off; 33 scale blocks
PRODUCTS = [(20_011, 256, 250, 128), (38_411, 256, 256, 128), (9_600, 4200, 256, 128), (9_601, 140, 251, 128), (20_011, 129, 60, 64), (19_100, 4200, 130, 64),
            (20_000, 300, 64, 64), (40_001, 130, 30, 32), (40_000, 512, 32, 32)]


@pytest.mark.parametrize("ids", [False, True])
@pytest.mark.parametrize("rows,dim,out,width", PRODUCTS)
def test_product(ops, rows, dim, out, width, ids):  # noqa: F811
    assert width_of(rows, out)[0] == width and width_of(rows, out)[1] > 1
    held = 3000 if ids else rows
    a, sa, w, sw = product_case(held, dim, out)
    A, W = f.decode(a, sa), f.decode_weight(w, sw)
    given, bad = None, None
    if ids:
        given = torch.randint(0, held, (rows,), generator=torch.Generator().manual_seed(rows)).cuda()
        bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
        bad[[5, 19_000 if rows > 19_000 else 9_500, rows - 1]] = True  # in a block's first tile and in a later one
        A = A[given]
        given[bad] = torch.tensor([held, -1, 1 << 40], device="cuda")
    want, mags = A @ W.t(), A.abs() @ W.abs().t()
    for dtype in TYPES:
        bias = rand(5, out) if dtype != torch.float16 else None
        got = ops.product_f8(a, sa, w, sw, ids=given, bias=bias, dtype=dtype)
        full, size = (want, mags) if bias is None else (want + bias.double(), mags + bias.double().abs())
        if ids:
            full, size = full.masked_fill(bad[:, None], 0.0), size.masked_fill(bad[:, None], 0.0)
            with pytest.raises(ValueError, match="out of bounds"):
                ops.check()
        near(got, full, f.STEP[dtype] * (1 + 2 ** -7) * full.abs() + (128 + 3 * sa.shape[1] + 2) * 2 * U * size + LEAST[dtype] * (size > 0), f"{dtype}")
    ops.check()
