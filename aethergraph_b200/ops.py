"""Row operators: what a model's layers do to the feature rows of a batch.

    x = ops.dropout(batch.x, 0.5, seed, offset=step)               # mask never stored
    y, h = ops.add_rms_norm(branch, weight, residual, p=0.1, seed=seed, offset=step)
    codes, scales, h = ops.add_rms_norm_f8(branch, weight, residual)  # rows in 8 bits
    out = ops.product_f8(codes, scales, *ops.encode_weight_f8(w))     # and their product

The rows are CUDA tensors of float32, float16 or bfloat16 whose last dimension is the
row; leading dimensions are flattened.  Calls run on the current stream of the rows' device,
wait for nothing and may be captured into a CUDA graph (a backward pass, as with any PyTorch operator,
only while no autograd graph of the same leaves made on another stream is alive).  `dropout`
and `add_rms_norm` have gradients (reverse mode, once: a backward pass with create_graph=True is refused, and so
are inputs with a forward-mode tangent); the 8-bit operators are for inference and have none.
torch.jit.trace is refused: it would keep a call's results as constants.

8-bit rows are a pair (codes, scales): torch.float8_e4m3fn codes [rows, dim], whose row pitch
is a multiple of 16 bytes, and float32 scales [rows, ceil(dim / 128)], value = code * scale.
8-bit weights [out, dim] carry one scale per 128 x 128 block.  `FeatureStore` keeps such
rows under the dtype "f8".

The functions are those of `_ops` (csrc/ops_torch.cpp), which calls the kernels through the C
ABI; like the rest of the package there is no fallback without it.  It is loaded, and torch with it, by the
first call.
"""
from __future__ import annotations

from typing import TYPE_CHECKING

from . import _lib

if TYPE_CHECKING:
    import torch

__all__ = ["add_rms_norm", "add_rms_norm_f8", "check", "decode_f8", "dropout", "dropout_", "encode_f8", "encode_weight_f8",
           "product_f8"]


_loaded = None


def _native():
    global _loaded
    if _loaded is None:
        _lib.lib()  # said in the package's own words if it was never built
        import torch  # noqa: F401  (the extension needs its libraries)

        from . import _ops as _loaded
    return _loaded


def _check_key(seed: int, offset: int) -> None:
    if not 0 <= seed < 1 << 64 or not 0 <= offset < 1 << 64:
        raise ValueError("seed and offset must be in [0, 2**64)")


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """Rows with elements zeroed with probability `p` and the others scaled by 1 / (1 - p).

    `p` is taken to the nearest multiple of 1/65536 and the scale is that of the value taken.
    Which elements fall is a function of (seed, offset, row, column) alone — the same on every
    call, for every type and layout; give every use in a program an `offset` of its own.  The gradient makes the mask again
    instead of storing it.  A dropped element is 0 even where `x` is infinite or NaN."""
    _check_key(seed, offset)
    return _native().dropout(x, p, seed, offset)


def dropout_(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """`dropout` in place, for rows that no gradient is asked of (a batch's own `x`)."""
    _check_key(seed, offset)
    _native().dropout_(x, p, seed, offset)
    return x


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, *, eps: float = 1e-6,
                 p: float = 0.0, seed: int = 0, offset: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = residual + dropout(x), y = h / sqrt(mean(h**2) + eps) * weight, row by row.

    One pass over the rows: sum, statistics and product are held in float32 and rounded once; rows whose squares pass
    float32 (magnitudes beyond about 1e19) come out as zeros.
    Without residual and dropout h is `x` itself.  `weight` is [dim], of x's type or float32; rows have at most 16384 columns.  The
    gradients of x, weight and residual take one pass too; weight's is summed in a fixed order.  They are those of the
    unrounded h: for float16 and bfloat16 rows x and residual are kept for the backward pass (as autograd keeps any operator's
    inputs: changed in place meanwhile, the backward pass is refused), for float32 h.
    `p`, `seed` and `offset` are `dropout`'s."""
    _check_key(seed, offset)
    return _native().add_rms_norm(x, weight, residual, eps, p, seed, offset)


def add_rms_norm_f8(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, *,
                    eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, scales, h): `add_rms_norm` with y as 8-bit rows, encoded where it is computed.  For
    inference: no dropout, no gradient."""
    return _native().add_rms_norm_f8(x, weight, residual, eps)


def encode_f8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales): rows, of at most 16384 columns, in 8 bits.  A block's scale puts its largest magnitude on 448; a block
    that holds an infinity or NaN reads as NaN throughout."""
    return _native().encode_f8(x)


def encode_weight_f8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of weights [out, dim]: one scale per 128 x 128 block, float32
    [ceil(out / 128), ceil(dim / 128)]."""
    return _native().encode_weight_f8(w)


def decode_f8(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """8-bit rows as float32 [rows, dim] (exact: code * scale, one multiplication)."""
    return _native().decode_f8(codes, scales)


def product_f8(codes: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *,
               ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               dtype: torch.dtype | None = None) -> torch.Tensor:
    """rows @ weight.T + bias of 8-bit rows and 8-bit weights, [rows, out] in `dtype` (bfloat16 by default).

    With `ids` (int64, or int32 holding u32 ids) output row i is that of 8-bit row ids[i]; an id outside them
    gives a zero row and an error that `check` raises.  Every block of 128 columns is summed,
    multiplied by its two scales and added up in float32.  `bias` is float32 [out]."""
    return _native().product_f8(codes, scales, weight, weight_scales, ids, bias, dtype)


def check(device: int | None = None) -> None:
    """Raise ValueError if a `product_f8` on the device since the last check saw an id outside its rows (waits for the
    device).  A store's products are checked by the store."""
    import torch

    _lib.check(_lib.lib().ag_rows_check(torch.cuda.current_device() if device is None else int(device)))
