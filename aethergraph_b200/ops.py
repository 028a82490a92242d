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
_stream = torch._C._cuda_getCurrentRawStream  # of a device index: a tenth of a microsecond, current_stream() takes two


def _check_rows(x, what: str = "x") -> int:
    """The dtype tag of a CUDA tensor of rows."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    tag = _TAG.get(x.dtype)
    if tag is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what} must have at least one column, got shape {tuple(x.shape)}")
    return tag


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """(tensor, rows, dim, pitch) of `t` as rows of consecutive columns; copied only where it is laid out
    otherwise.  The tensor is to be kept until the call is queued."""
    dim = t.shape[-1]
    if not t.is_contiguous():
        if t.dim() == 2 and (t.stride(1) == 1 or dim == 1) and t.stride(0) >= 0:
            return t, t.shape[0], dim, t.stride(0)
        t = t.contiguous()
    return t, t.numel() // dim, dim, dim


def _empty_like(x: torch.Tensor) -> torch.Tensor:
    """Contiguous, of x's shape."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)


def _check_like(t, x: torch.Tensor, what: str) -> None:
    if not isinstance(t, torch.Tensor) or t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{what} must have the shape, type and device of x: got {_say(t)}, x is {_say(x)}")


def _say(t) -> str:
    return f"{tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__


def _check_key(seed: int, offset: int) -> None:
    if not 0 <= seed < 1 << 64 or not 0 <= offset < 1 << 64:
        raise ValueError("seed and offset must be in [0, 2**64)")


def _once(what: str) -> None:
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} is differentiable once; call the backward pass without create_graph")


# ----------------------------------------------------------------- dropout --
def _run_dropout(x: torch.Tensor, tag: int, p: float, seed: int, offset: int) -> torch.Tensor:
    y = _empty_like(x)
    t, rows, dim, pitch = _rows(x)
    index = x.get_device()
    status = _lib.lib().ag_rows_dropout(t.data_ptr(), y.data_ptr(), rows, dim, pitch, dim, tag, p, seed, offset, index, _stream(index))
    if status:
        _lib.check(status)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tag, p, seed, offset):
        ctx.key = (tag, p, seed, offset)
        return _run_dropout(x, tag, p, seed, offset)

    @staticmethod
    def backward(ctx, dy):
        _once("dropout")
        return _run_dropout(dy, *ctx.key), None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """Rows with elements zeroed with probability `p` and the others scaled by 1 / (1 - p).

    `p` is taken to the nearest multiple of 1/65536 and the scale is that of the value taken.
    Which elements fall is a function of (seed, offset, row, column) alone — the same on every
    call, for every type and layout; give every use in a program an `offset` of its own.  The gradient makes the mask again
    instead of storing it.  A dropped element is 0 even where `x` is infinite or NaN."""
    _check_key(seed, offset)
    tag = _check_rows(x)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dropout.apply(x, tag, p, seed, offset)
    return _run_dropout(x, tag, p, seed, offset)


def dropout_(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """`dropout` in place, for rows that no gradient is asked of (a batch's own `x`)."""
    _check_key(seed, offset)
    tag = _check_rows(x)
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("dropout_ is for rows that need no gradient; use dropout")
    t, rows, dim, pitch = _rows(x)
    if t is not x or rows > 1 and pitch < dim:
        raise ValueError("dropout_ needs rows of consecutive columns that do not overlap")
    index, pitch = x.get_device(), max(pitch, dim)  # the pitch of a single row is free
    _lib.check(_lib.lib().ag_rows_dropout(x.data_ptr(), x.data_ptr(), rows, dim, pitch, pitch, tag, p, seed, offset, index, _stream(index)))
    return x


# -------------------------------------------------------------------- norm --
def _check_weight(weight, x: torch.Tensor) -> None:
    if not isinstance(weight, torch.Tensor) or weight.dim() != 1 or weight.shape[0] != x.shape[-1] or weight.device != x.device or \
            weight.dtype is not x.dtype and weight.dtype is not torch.float32:
        raise ValueError(f"weight must be [{x.shape[-1]}] of {x.dtype} or float32 on {x.device}, got {_say(weight)}")


def _norm_args(x, tag, weight, residual, eps):
    """The call's arguments without its outputs, and the tensors that they name."""
    t, rows, dim, pitch = _rows(x)
    n = _lib.Norm(x=t.data_ptr(), rows=rows, dim=dim, x_stride=pitch, eps=eps, dtype=tag)
    keep = [t]
    if residual is not None:
        r, _, _, n.residual_stride = _rows(residual)
        n.residual = r.data_ptr()
        keep.append(r)
    if weight is not None:
        w = weight.contiguous()
        n.weight, n.weight_dtype = w.data_ptr(), _TAG[w.dtype]
        keep.append(w)
    return n, keep


def _run_norm(x, tag, weight, residual, eps, p, seed, offset, want_rstd):
    n, keep = _norm_args(x, tag, weight, residual, eps)
    n.p, n.seed, n.offset = p, seed, offset
    y = _empty_like(x)
    n.y, n.y_stride = y.data_ptr(), n.dim
    h = x
    if residual is not None or p > 0:
        h = _empty_like(x)
        n.h, n.h_stride = h.data_ptr(), n.dim
    index, rstd = x.get_device(), None
    if want_rstd:
        rstd = x.new_empty(n.rows, dtype=torch.float32)
        n.rstd = rstd.data_ptr()
    status = _lib.lib().ag_rows_norm(C.byref(n), index, _stream(index))
    if status:
        _lib.check(status)
    return y, h, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, tag, eps, p, seed, offset):
        y, h, rstd = _run_norm(x, tag, weight, residual, eps, p, seed, offset, True)
        ctx.save_for_backward(h, weight, rstd)
        ctx.key = (tag, p, seed, offset)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        _once("add_rms_norm")
        if dy is None and dh is None:
            return (None,) * 8
        h, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_res = ctx.needs_input_grad[:3]
        tag, p, seed, offset = ctx.key
        t, rows, dim, pitch = _rows(h)
        n = _lib.NormGrad(h=t.data_ptr(), rstd=rstd.data_ptr(), rows=rows, dim=dim, h_stride=pitch, p=p, seed=seed, offset=offset,
                          dtype=tag)
        keep, index = [t], h.get_device()
        if dy is not None:
            g, _, _, n.dy_stride = _rows(dy)
            n.dy = g.data_ptr()
            keep.append(g)
        if dh is not None:
            g, _, _, n.dh_stride = _rows(dh)
            n.dh = g.data_ptr()
            keep.append(g)
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
        if weight is not None:
            w = weight.contiguous()
            keep.append(w)
            n.weight, n.weight_dtype = w.data_ptr(), _TAG[w.dtype]
            if need_w and dy is not None:
                dw = torch.empty_like(w)
                size = C.c_uint64()
                _lib.check(_lib.lib().ag_rows_norm_backward_scratch(rows, dim, tag, index, C.byref(size)))
                scratch = h.new_empty(size.value, dtype=torch.uint8)
                n.dw, n.scratch, n.scratch_bytes = dw.data_ptr(), scratch.data_ptr(), size.value
        status = _lib.lib().ag_rows_norm_backward(C.byref(n), index, _stream(index))
        if status:
            _lib.check(status)
        return dx, dw, dres, None, None, None, None, None


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, *, eps: float = 1e-6,
                 p: float = 0.0, seed: int = 0, offset: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = residual + dropout(x), y = h / sqrt(mean(h**2) + eps) * weight, row by row.

    One pass over the rows: sum, statistics and product are held in float32 and rounded once.
    Without residual and dropout h is `x` itself.  `weight` is [dim], of x's type or float32; rows have at most 16384 columns.  The
    gradients of x, weight and residual take one pass too; weight's is summed in a fixed order.
    `p`, `seed` and `offset` are `dropout`'s."""
    _check_key(seed, offset)
    tag = _check_rows(x)
    if weight is not None:
        _check_weight(weight, x)
    if residual is not None:
        _check_like(residual, x, "residual")
    if torch.is_grad_enabled() and (x.requires_grad or weight is not None and weight.requires_grad or
                                    residual is not None and residual.requires_grad):
        return _AddRmsNorm.apply(x, weight, residual, tag, eps, p, seed, offset)
    return _run_norm(x, tag, weight, residual, eps, p, seed, offset, False)[:2]


# ------------------------------------------------------------- 8-bit rows --
def _no_gradient(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradient; call it under torch.no_grad()")


def _empty_f8(rows: int, dim: int, like: torch.Tensor) -> torch.Tensor:
    return like.new_empty((rows, (dim + 15) // 16 * 16), dtype=torch.float8_e4m3fn)[:, :dim]


def _to_f8(n: "_lib.Norm", x: torch.Tensor):
    codes = _empty_f8(n.rows, n.dim, x)
    scales = x.new_empty((n.rows, (n.dim + F8_BLOCK - 1) // F8_BLOCK), dtype=torch.float32)
    n.codes, n.scales, n.code_stride = codes.data_ptr(), scales.data_ptr(), (n.dim + 15) // 16 * 16
    index = x.get_device()
    if n.rows:
        _lib.check(_lib.lib().ag_rows_norm(C.byref(n), index, _stream(index)))
    return codes, scales


def add_rms_norm_f8(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, *,
                    eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, scales, h): `add_rms_norm` with y as 8-bit rows, encoded where it is computed.  For
    inference: no dropout, no gradient."""
    tag = _check_rows(x)
    if weight is not None:
        _check_weight(weight, x)
    if residual is not None:
        _check_like(residual, x, "residual")
    _no_gradient("add_rms_norm_f8", x, weight, residual)
    n, keep = _norm_args(x, tag, weight, residual, eps)
    h = x
    if residual is not None:
        h = _empty_like(x)
        n.h, n.h_stride = h.data_ptr(), n.dim
    codes, scales = _to_f8(n, x)
    return codes, scales, h


def encode_f8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales): rows in 8 bits.  A block's scale puts its largest magnitude on 448; a block
    that holds an infinity or NaN reads as NaN throughout."""
    tag = _check_rows(x)
    _no_gradient("encode_f8", x)
    n, keep = _norm_args(x, tag, None, None, 0.0)
    n.encode_only = 1
    return _to_f8(n, x)


def encode_weight_f8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of weights [out, dim]: one scale per 128 x 128 block, float32
    [ceil(out / 128), ceil(dim / 128)]."""
    tag = _check_rows(w, "w")
    if w.dim() != 2:
        raise ValueError(f"weights must be [out, dim], got shape {tuple(w.shape)}")
    _no_gradient("encode_weight_f8", w)
    t, out, dim, pitch = _rows(w)
    codes = _empty_f8(out, dim, w)
    scales = w.new_empty(((out + F8_BLOCK - 1) // F8_BLOCK, (dim + F8_BLOCK - 1) // F8_BLOCK), dtype=torch.float32)
    index = w.get_device()
    _lib.check(_lib.lib().ag_rows_encode_weight(t.data_ptr(), out, dim, pitch, tag, codes.data_ptr(), (dim + 15) // 16 * 16,
                                                scales.data_ptr(), index, _stream(index)))
    return codes, scales


def _check_f8(codes, scales, what: str, blocks_of: int) -> tuple[int, int, int, int]:
    """(rows, dim, pitch, device index) of 8-bit rows."""
    if not isinstance(codes, torch.Tensor) or not codes.is_cuda or codes.dim() != 2 or codes.dtype is not torch.float8_e4m3fn:
        raise ValueError(f"{what} must be a CUDA tensor [rows, dim] of torch.float8_e4m3fn")
    (rows, dim), (pitch, step), index = codes.shape, codes.stride(), codes.get_device()
    if dim == 0 or dim > 1 and step != 1 or pitch % 16 or pitch < dim or codes.data_ptr() % 16:
        raise ValueError(f"{what} must start on 16 bytes, with consecutive columns and a row pitch that is a multiple of 16 bytes")
    want = ((rows + blocks_of - 1) // blocks_of, (dim + F8_BLOCK - 1) // F8_BLOCK)
    if not isinstance(scales, torch.Tensor) or scales.dtype is not torch.float32 or scales.shape != want or not scales.is_contiguous() or \
            not scales.is_cuda or scales.get_device() != index:
        raise ValueError(f"{what}' scales must be contiguous float32 {list(want)} on {codes.device}")
    return rows, dim, pitch, index


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
    rows, dim, pitch, index = _check_f8(codes, scales, "codes", 1)
    return _product((codes.data_ptr(), scales.data_ptr(), pitch, rows, dim, index), weight, weight_scales, ids, bias, dtype)


def _product(held, weight, weight_scales, ids, bias, dtype) -> torch.Tensor:
    codes, scales, pitch, rows, dim, index = held
    out_dim, w_dim, w_pitch, w_index = _check_f8(weight, weight_scales, "weight", F8_BLOCK)
    if w_index != index or w_dim != dim or out_dim == 0:
        raise ValueError(f"weight must be [out, {dim}] on cuda:{index}, got {list(weight.shape)} on {weight.device}")
    tag = _TAG.get(dtype)
    if tag is None:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    args = _lib.Product(codes=codes, scales=scales, weight=weight.data_ptr(), weight_scales=weight_scales.data_ptr(), rows=rows,
                        held=rows, dim=dim, out_dim=out_dim, code_stride=pitch, weight_stride=w_pitch, out_stride=out_dim,
                        out_dtype=tag)
    if ids is not None:
        if not isinstance(ids, torch.Tensor) or not ids.is_cuda or ids.get_device() != index or ids.dim() != 1 or \
                not ids.is_contiguous() or ids.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"ids must be a contiguous 1-d tensor of dtype int64 or int32 on cuda:{index}")
        rows = ids.shape[0]
        args.ids, args.ids_are_i64, args.rows = ids.data_ptr(), ids.dtype is torch.int64, rows
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or not bias.is_cuda or bias.get_device() != index or bias.dtype is not torch.float32 or \
                bias.shape != (out_dim,) or not bias.is_contiguous():
            raise ValueError(f"bias must be contiguous float32 [{out_dim}] on cuda:{index}")
        _no_gradient("a product of 8-bit rows", bias)
        args.bias = bias.data_ptr()
    out = weight_scales.new_empty((rows, out_dim), dtype=dtype)
    if rows:
        args.out = out.data_ptr()
        status = _lib.lib().ag_rows_product(C.byref(args), index, _stream(index))
        if status:
            _lib.check(status)
    return out


def check(device: int | None = None) -> None:
    """Raise ValueError if a product since the last check saw an id outside its rows (waits for the device)."""
    _lib.check(_lib.lib().ag_rows_check(torch.cuda.current_device() if device is None else int(device)))
