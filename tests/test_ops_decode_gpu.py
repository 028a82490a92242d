"""decode_f8 is a call like the others: on the caller's stream, waiting for nothing, in a graph too."""
import pytest
import torch

import ops_formulas as f
from test_ops_gpu import ops, rand  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim", [(0, 8), (1, 1), (3, 16), (200, 100), (2000, 128), (77, 301), (5, 9000)])
def test_values(ops, rows, dim):  # noqa: F811
    codes, scales = ops.encode_f8(rand(1, rows, dim))
    want = f.decode(codes.cpu(), scales.cpu()).float()
    assert torch.equal(ops.decode_f8(codes, scales).cpu(), want)
    wide = torch.full((rows, codes.stride(0) + 32 if rows else 16), 0x7F, dtype=torch.uint8, device="cuda")  # NaN beside the rows
    if rows:
        wide[:, 16:16 + dim] = codes.view(torch.uint8)
        assert torch.equal(ops.decode_f8(wide.view(torch.float8_e4m3fn)[:, 16:16 + dim], scales).cpu(), want)


def test_captured_and_on_another_stream(ops):  # noqa: F811
    x = rand(1, 500, 96)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(100):
            a = a @ a
            a = a / a.abs().max()
        codes, scales = ops.encode_f8(x)
        other = ops.decode_f8(codes, scales)
        waited = side.query()  # the products above take longer than the calls
    assert not waited
    torch.cuda.current_stream().wait_stream(side)
    want = f.decode(codes.cpu(), scales.cpu()).float()
    assert torch.equal(other.cpu(), want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.decode_f8(*ops.encode_f8(x))
    x.neg_()
    g.replay()
    assert torch.equal(out.cpu(), -want)


def test_refusals(ops):  # noqa: F811
    codes, scales = ops.encode_f8(rand(1, 8, 64))
    for call in (lambda: ops.decode_f8(codes, scales[:4]), lambda: ops.decode_f8(codes[:, 8:], scales), lambda: ops.decode_f8(codes.view(torch.uint8), scales),
                 lambda: ops.decode_f8(codes, scales.half())):
        with pytest.raises(ValueError):
            call()
