"""Row operators: what a model's layers do to the feature rows of a batch.

    x = ops.dropout(batch.x, 0.5, seed, offset=step)               # mask never stored
    y, h = ops.add_rms_norm(branch, weight, residual, p=0.1, seed=seed, offset=step)
    codes, scales, h = ops.add_rms_norm_f8(branch, weight, residual)  # rows in 8 bits
    out = ops.product_f8(codes, scales, *ops.encode_weight_f8(w))     # and their product

The rows are CUDA tensors of float32, float16 or bfloat16 whose last dimension is the
row; leading dimensions are flattened.  Calls run on the current stream of the rows' device,
wait for nothing and may be captured into a CUDA graph (a backward pass, as with any PyTorch operator,
only while no autograd graph of the same leaves made on another stream is alive).  `dropout` and `add_rms_norm`
have gradients (once differentiable); the 8-bit operators are for inference and have none.

8-bit rows are a pair (codes, scales): torch.float8_e4m3fn codes [rows, dim], whose row pitch
is a multiple of 16 bytes, and float32 scales [rows, ceil(dim / 128)], value = code * scale.
8-bit weights [out, dim] carry one scale per 128 x 128 block.  `FeatureStore` keeps such
rows under the dtype "f8".
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

__all__ = ["add_rms_norm", "add_rms_norm_f8", "check", "decode_f8", "dropout", "dropout_", "encode_f8", "encode_weight_f8",
           "product_f8"]

F8_BLOCK = 128  # columns per scale
_TAG = {torch.float32: _lib.AG_F32, torch.float16: _lib.AG_F16, torch.bfloat16: _lib.AG_BF16}


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    """`t` as [rows, dim] with consecutive columns; copied only where it is laid out otherwise."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.dtype not in _TAG:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    if t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= 0:
        return t
    if t.dim() == 0:
        raise ValueError(f"{what} must have at least one dimension")
    if t.shape[-1] == 0:
        raise ValueError(f"{what} must have at least one column")
    return t.contiguous().view(-1, t.shape[-1])


def _like(t, x: torch.Tensor, what: str) -> torch.Tensor:
    if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{what} must have the shape, type and device of x: got {tuple(t.shape)} {t.dtype} on {t.device}, "
                         f"x is {tuple(x.shape)} {x.dtype} on {x.device}")
    return _rows(t, what)


def _key(seed: int, offset: int) -> tuple[int, int]:
    if not 0 <= seed < 1 << 64 or not 0 <= offset < 1 << 64:
        raise ValueError("seed and offset must be in [0, 2**64)")
    return int(seed), int(offset)


def _differentiable(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ----------------------------------------------------------------- dropout --
def _run_dropout(x: torch.Tensor, y: torch.Tensor, p: float, seed: int, offset: int) -> torch.Tensor:
    rows, out = _rows(x, "x"), y.view(-1, y.shape[-1])
    _lib.check(_lib.lib().ag_rows_dropout(rows.data_ptr(), out.data_ptr(), rows.shape[0], rows.shape[1], rows.stride(0),
                                          out.stride(0), _TAG[x.dtype], p, seed, offset, x.device.index, _stream(x)))
    return y


def _empty_like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset):
        ctx.key = (p, seed, offset)
        return _run_dropout(x, _empty_like(x), p, seed, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return _run_dropout(dy, _empty_like(dy), *ctx.key), None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """Rows with elements zeroed with probability `p` and the others scaled by 1 / (1 - p).

    `p` is taken to the nearest multiple of 1/65536 and the scale is that of the value taken.
    Which elements fall is a function of (seed, offset, row, column) alone — the same on every
    call, for every type and layout; give every use in a program an `offset` of its own.  The gradient makes the mask again
    instead of storing it.  A dropped element is 0 even where `x` is infinite or NaN."""
    seed, offset = _key(seed, offset)
    _rows_only(x)
    if _differentiable(x):
        return _Dropout.apply(x, float(p), seed, offset)
    return _run_dropout(x, _empty_like(x), float(p), seed, offset)


def dropout_(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """`dropout` in place, for rows that no gradient is asked of (a batch's own `x`)."""
    seed, offset = _key(seed, offset)
    _rows_only(x)
    if _differentiable(x):
        raise ValueError("dropout_ is for rows that need no gradient; use dropout")
    if x.dim() != 2 and not x.is_contiguous():
        raise ValueError("dropout_ needs [rows, dim] with consecutive columns, or a contiguous tensor")
    rows = x if x.dim() == 2 else x.view(-1, x.shape[-1])
    if x.shape[-1] > 1 and rows.stride(1) != 1 or rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]:
        raise ValueError("dropout_ needs rows of consecutive columns that do not overlap")
    _lib.check(_lib.lib().ag_rows_dropout(rows.data_ptr(), rows.data_ptr(), rows.shape[0], rows.shape[1],
                                          max(rows.stride(0), rows.shape[1]), max(rows.stride(0), rows.shape[1]), _TAG[x.dtype],
                                          float(p), seed, offset, x.device.index, _stream(x)))
    return x


def _rows_only(x) -> None:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if x.dtype not in _TAG:
        raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must have at least one column, got shape {tuple(x.shape)}")


# -------------------------------------------------------------------- norm --
def _weight(weight, x: torch.Tensor):
    if weight is None:
        return None
    if weight.dim() != 1 or weight.shape[0] != x.shape[-1] or weight.device != x.device or weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"weight must be [{x.shape[-1]}] of {x.dtype} or float32 on {x.device}, got {tuple(weight.shape)} "
                         f"{weight.dtype} on {weight.device}")
    return weight.contiguous()


def _norm_args(rows, res, weight, eps, p=0.0, seed=0, offset=0) -> "_lib.Norm":
    n = _lib.Norm(x=rows.data_ptr(), rows=rows.shape[0], dim=rows.shape[1], x_stride=rows.stride(0), eps=eps, p=p, seed=seed,
                  offset=offset, dtype=_TAG[rows.dtype])
    if res is not None:
        n.residual, n.residual_stride = res.data_ptr(), res.stride(0)
    if weight is not None:
        n.weight, n.weight_dtype = weight.data_ptr(), _TAG[weight.dtype]
    return n


def _run_norm(x, weight, residual, eps, p, seed, offset, want_rstd):
    rows = _rows(x, "x")
    res = None if residual is None else _like(residual, x, "residual")
    w = _weight(weight, x)
    n = _norm_args(rows, res, w, eps, p, seed, offset)
    y = _empty_like(x)
    n.y, n.y_stride = y.data_ptr(), rows.shape[1]
    h = x
    if residual is not None or p > 0:
        h = _empty_like(x)
        n.h, n.h_stride = h.data_ptr(), rows.shape[1]
    rstd = None
    if want_rstd:
        rstd = torch.empty(rows.shape[0], dtype=torch.float32, device=x.device)
        n.rstd = rstd.data_ptr()
    _lib.check(_lib.lib().ag_rows_norm(C.byref(n), x.device.index, _stream(x)))
    return y, h, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, p, seed, offset):
        y, h, rstd = _run_norm(x, weight, residual, eps, p, seed, offset, True)
        ctx.save_for_backward(h, weight, rstd)
        ctx.key = (p, seed, offset)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_res = ctx.needs_input_grad[:3]
        p, seed, offset = ctx.key
        if dy is None and dh is None:
            return (None,) * 7
        rows, w = _rows(h, "h"), None if weight is None else weight.contiguous()
        n = _lib.NormGrad(h=rows.data_ptr(), rstd=rstd.data_ptr(), rows=rows.shape[0], dim=rows.shape[1], h_stride=rows.stride(0),
                          p=p, seed=seed, offset=offset, dtype=_TAG[h.dtype])
        keep = []
        for name, grad in (("dy", dy), ("dh", dh)):
            if grad is not None:
                g = _rows(grad, name)
                keep.append(g)
                setattr(n, name, g.data_ptr())
                setattr(n, name + "_stride", g.stride(0))
        dx = dres = dw = None
        if need_x:
            dx = _empty_like(h)
            n.dx = dx.data_ptr()
        if need_res:
            if p > 0 or not need_x:
                dres = _empty_like(h)
                n.dresidual = dres.data_ptr()
            else:
                dres = dx  # without dropout the two are one
        if w is not None:
            n.weight, n.weight_dtype = w.data_ptr(), _TAG[w.dtype]
        if need_w:
            dw = torch.empty_like(w)
            if dy is None:
                dw.zero_()
            else:
                size = C.c_uint64()
                _lib.check(_lib.lib().ag_rows_norm_backward_scratch(rows.shape[0], rows.shape[1], h.device.index, C.byref(size)))
                scratch = torch.empty(max(size.value, 4), dtype=torch.uint8, device=h.device)
                n.dw, n.scratch, n.scratch_bytes = dw.data_ptr(), scratch.data_ptr(), size.value
        _lib.check(_lib.lib().ag_rows_norm_backward(C.byref(n), h.device.index, _stream(h)))
        return dx, dw, dres, None, None, None, None


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, *, eps: float = 1e-6,
                 p: float = 0.0, seed: int = 0, offset: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = residual + dropout(x), y = h / sqrt(mean(h**2) + eps) * weight, row by row.

    One pass over the rows: sum, statistics and product are held in float32 and rounded once.
    Without residual and dropout h is `x` itself.  `weight` is [dim], of x's type or float32; rows have at most 16384 columns.  The
    gradients of x, weight and residual take one pass too; weight's is summed in a fixed order.
    `p`, `seed` and `offset` are `dropout`'s."""
    seed, offset = _key(seed, offset)
    _rows_only(x)
    if _differentiable(x, weight, residual):
        return _AddRmsNorm.apply(x, weight, residual, float(eps), float(p), seed, offset)
    return _run_norm(x, weight, residual, float(eps), float(p), seed, offset, False)[:2]


# ------------------------------------------------------------- 8-bit rows --
def _empty_f8(rows: int, dim: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    codes = torch.empty((rows, (dim + 15) // 16 * 16), dtype=torch.float8_e4m3fn, device=device)
    return codes[:, :dim], torch.empty((rows, (dim + F8_BLOCK - 1) // F8_BLOCK), dtype=torch.float32, device=device)


def _to_f8(n: "_lib.Norm", x: torch.Tensor, dim: int):
    codes, scales = _empty_f8(n.rows, dim, x.device)
    n.codes, n.scales, n.code_stride = codes.data_ptr(), scales.data_ptr(), codes.stride(0)
    if n.rows:
        _lib.check(_lib.lib().ag_rows_norm(C.byref(n), x.device.index, _stream(x)))
    return codes, scales


def add_rms_norm_f8(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, *,
                    eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, scales, h): `add_rms_norm` with y as 8-bit rows, encoded where it is computed.  For
    inference: no dropout, no gradient."""
    _rows_only(x)
    if _differentiable(x, weight, residual):
        raise ValueError("8-bit rows have no gradient; call add_rms_norm_f8 under torch.no_grad()")
    rows = _rows(x, "x")
    res = None if residual is None else _like(residual, x, "residual")
    w = _weight(weight, x)
    n = _norm_args(rows, res, w, float(eps))
    h = x
    if residual is not None:
        h = _empty_like(x)
        n.h, n.h_stride = h.data_ptr(), rows.shape[1]
    codes, scales = _to_f8(n, x, rows.shape[1])
    return codes, scales, h


def encode_f8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales): rows in 8 bits.  A block's scale puts its largest magnitude on 448; a block
    that holds an infinity or NaN reads as NaN throughout."""
    _rows_only(x)
    if _differentiable(x):
        raise ValueError("8-bit rows have no gradient; call encode_f8 under torch.no_grad()")
    rows = _rows(x, "x")
    n = _norm_args(rows, None, None, 0.0)
    n.encode_only = 1
    return _to_f8(n, x, rows.shape[1])


def encode_weight_f8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of weights [out, dim]: one scale per 128 x 128 block, float32
    [ceil(out / 128), ceil(dim / 128)]."""
    _rows_only(w)
    if w.dim() != 2:
        raise ValueError(f"weights must be [out, dim], got shape {tuple(w.shape)}")
    if _differentiable(w):
        raise ValueError("8-bit weights have no gradient; call encode_weight_f8 under torch.no_grad()")
    rows = _rows(w, "w")
    codes, _ = _empty_f8(rows.shape[0], rows.shape[1], w.device)
    scales = torch.empty(((rows.shape[0] + F8_BLOCK - 1) // F8_BLOCK, (rows.shape[1] + F8_BLOCK - 1) // F8_BLOCK),
                         dtype=torch.float32, device=w.device)
    _lib.check(_lib.lib().ag_rows_encode_weight(rows.data_ptr(), rows.shape[0], rows.shape[1], rows.stride(0), _TAG[w.dtype],
                                                codes.data_ptr(), codes.stride(0), scales.data_ptr(), w.device.index, _stream(w)))
    return codes, scales


def _check_f8(codes, scales, what: str, blocks_of: int) -> None:
    if not isinstance(codes, torch.Tensor) or not codes.is_cuda or codes.dim() != 2 or codes.dtype != torch.float8_e4m3fn:
        raise ValueError(f"{what} must be a CUDA tensor [rows, dim] of torch.float8_e4m3fn")
    rows, dim = codes.shape
    if dim == 0 or dim > 1 and codes.stride(1) != 1 or codes.stride(0) % 16 or codes.stride(0) < dim or codes.data_ptr() % 16:
        raise ValueError(f"{what} must start on 16 bytes, with consecutive columns and a row pitch that is a multiple of 16 bytes")
    want = ((rows + blocks_of - 1) // blocks_of, (dim + F8_BLOCK - 1) // F8_BLOCK)
    if not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or tuple(scales.shape) != want or not scales.is_contiguous() or \
            scales.device != codes.device:
        raise ValueError(f"{what}' scales must be contiguous float32 {list(want)} on {codes.device}")


def decode_f8(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """8-bit rows as float32 [rows, dim] (exact: code * scale, one multiplication)."""
    from .features import FeatureStore

    store = FeatureStore.from_f8(codes, scales)
    return store.gather(torch.arange(codes.shape[0], device=codes.device))


def product_f8(codes: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *,
               ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """rows @ weight.T + bias of 8-bit rows and 8-bit weights, [rows, out] in `dtype`.

    With `ids` (int64, or int32 holding u32 ids) output row i is that of 8-bit row ids[i]; an id outside them
    gives a zero row and an error that `check` raises.  Every block of 128 columns is summed,
    multiplied by its two scales and added up in float32.  `bias` is float32 [out]."""
    _check_f8(codes, scales, "codes", 1)
    held = (codes.data_ptr(), scales.data_ptr(), codes.stride(0), codes.shape[0], codes.shape[1], codes.device.index)
    return _product(held, weight, weight_scales, ids, bias, dtype)


def _product(held, weight, weight_scales, ids, bias, dtype) -> torch.Tensor:
    codes, scales, pitch, rows, dim, index = held
    _check_f8(weight, weight_scales, "weight", F8_BLOCK)
    dev = weight.device
    if dev.index != index or weight.shape[1] != dim:
        raise ValueError(f"weight must be [out, {dim}] on cuda:{index}, got {list(weight.shape)} on {dev}")
    if dtype not in _TAG:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    out_dim = weight.shape[0]
    args = _lib.Product(codes=codes, scales=scales, weight=weight.data_ptr(), weight_scales=weight_scales.data_ptr(), rows=rows,
                        held=rows, dim=dim, out_dim=out_dim, code_stride=pitch, weight_stride=weight.stride(0), out_stride=out_dim,
                        out_dtype=_TAG[dtype])
    if ids is not None:
        if ids.device != dev or ids.dim() != 1 or not ids.is_contiguous() or ids.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"ids must be a contiguous 1-d tensor of dtype int64 or int32 on {dev}")
        rows = ids.shape[0]
        args.ids, args.ids_are_i64, args.rows = ids.data_ptr(), int(ids.dtype == torch.int64), rows
    if bias is not None:
        if bias.device != dev or bias.dtype != torch.float32 or tuple(bias.shape) != (out_dim,) or not bias.is_contiguous():
            raise ValueError(f"bias must be contiguous float32 [{out_dim}] on {dev}")
        args.bias = bias.data_ptr()
    if _differentiable(bias):
        raise ValueError("product_f8 has no gradient; call it under torch.no_grad()")
    if out_dim == 0:
        raise ValueError("weight must have at least one row")
    out = torch.empty((rows, out_dim), dtype=dtype, device=dev)
    args.out = out.data_ptr()
    if rows:
        _lib.check(_lib.lib().ag_rows_product(C.byref(args), index, _stream(weight)))
    return out


def check(device: int | None = None) -> None:
    """Raise ValueError if a product since the last check saw an id outside its rows (waits for the device)."""
    _lib.check(_lib.lib().ag_rows_check(torch.cuda.current_device() if device is None else int(device)))
