"""The row operators' definitions in 64 bits (numpy and torch), for the tests."""
from __future__ import annotations

import numpy as np
import torch

E4M3_MAX = 448.0
TINY = 2.0 ** -126
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of each type


def philox(c0, c1, c2, c3, seed):
    """Philox4x32-10 over uint64 arrays of 32-bit words."""
    c = [np.asarray(v, dtype=np.uint64) for v in (c0, c1, c2, c3)]
    k = [np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32)]
    low, s = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> s) ^ c[1] ^ k[0], b & low, (a >> s) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return c


def lots(rows, dim, seed, offset, first_row=0):
    """The 16 random bits of every element of rows [first_row, first_row + rows)."""
    groups = (dim + 7) // 8
    r, g = np.meshgrid(np.arange(first_row, first_row + rows), np.arange(groups), indexing="ij")
    words = philox(g, r, np.full(g.shape, offset & 0xFFFFFFFF), np.full(g.shape, offset >> 32), seed)
    halves = [h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))]
    return np.stack(halves, 2).reshape(rows, groups * 8)[:, :dim].astype(np.int64)


def mask(rows, dim, p, seed, offset, first_row=0):
    """float64 [rows, dim]: the scale where an element stays, else 0."""
    t = int(np.floor(p * 65536 + 0.5))
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    return torch.from_numpy(np.where(lots(rows, dim, seed, offset, first_row) >= t, scale, 0.0))


def norm(x, w, res, eps, m=None):
    """(y, h) in float64; differentiable."""
    h = x if m is None else x * m
    if res is not None:
        h = h + res
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return (y if w is None else y * w), h


def decode(codes, scales):
    """float64 rows of 8-bit rows."""
    return codes.to(torch.float64) * scales.to(torch.float64).repeat_interleave(128, 1)[:, :codes.shape[1]]


def decode_weight(codes, scales):
    out, dim = codes.shape
    return codes.to(torch.float64) * scales.to(torch.float64).repeat_interleave(128, 0).repeat_interleave(128, 1)[:out, :dim]


def block_peaks(y, rows_of=1):
    """Largest magnitude per `rows_of` x 128 block."""
    rows, dim = y.shape
    y = torch.nn.functional.pad(y.abs(), (0, -dim % 128, 0, -rows % rows_of))
    return y.view(y.shape[0] // rows_of, rows_of, y.shape[1] // 128, 128).amax((1, 3))
