"""Row operators of a layer over a batch's feature rows, sized for timing: dropout whose mask
is a function of (seed, offset, row, column), the root-mean-square norm with the residual's
addition (forward, backward, and with rows of 8-bit floats as output), and the product of
8-bit rows, in order or picked by id, with 8-bit weights.

A case is a dict of plain values.  `prepare` makes the inputs from the seed, `run` makes one
pass, `work` states the bytes and operations that the pass cannot do without, `exact` computes
the same outputs in 64 bits.  With `own` false `run` computes in elementary torch operations.

Random bits: element (r, c) of rows x dim takes 16 bits of Philox4x32-10 with the counter
(c // 8, r, offset's lower and upper word) and the seed as key; of the four words the one
numbered (c % 8) // 2, its lower half for even c.  It is kept if they are at least
T = round(65536 p), and scaled by 65536 / (65536 - T).
8-bit rows: e4m3 codes and one f32 scale per 128 columns of a row (amax / 448); weights
[out, dim] carry one scale per 128 x 128 block.  Row pitches are multiples of 16 bytes.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
BLOCK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -126


def _dropout(name, **kw):
    return dict(dict(name=name, kind="dropout", rows=1 << 10, dim=128, dtype="f32", p=0.5, train=True), **kw)


def _norm(name, **kw):
    return dict(dict(name=name, kind="norm", rows=1 << 10, dim=128, dtype="bf16", p=0.0, residual=True, train=False, f8=False),
                **kw)


def _product(name, **kw):
    return dict(dict(name=name, kind="product", rows=1 << 10, dim=128, out=128, dtype="bf16", ids=False, table=0, bias=False),
                **kw)


def listed():
    return [
        # The seeds' own rows of a small batch: one call, nothing to hide its latency.
        _dropout("dropout_b128", rows=128, dim=128, train=False),
        # Training on batches of 1024 seeds, fanouts 25 and 10 (about 38 000 nodes a batch), rows of 256 bf16.
        _dropout("dropout_b1024_train", rows=38_411, dim=256, dtype="bf16"),
        # Rows whose length is no multiple of a vector load, three hops.
        _dropout("dropout_3hop_odd_train", rows=250_007, dim=301, dtype="f16", p=0.1),
        # One vertex asked for online.
        _norm("norm_one_row", rows=1, dim=1024),
        # A layer of the same training batch: h = residual + dropout(branch), normalised; forward and backward.
        _norm("norm_b1024_train", rows=38_411, dim=256, p=0.1, train=True),
        # The same in full precision, row length odd.
        _norm("norm_odd_train", rows=20_011, dim=602, dtype="f32", p=0.25, train=True),
        # Wide rows, no dropout, no residual.
        _norm("norm_wide_train", rows=16_384, dim=4096, dtype="f16", residual=False, train=True),
        # A layer's output over a whole graph kept as 8-bit rows for the next layer.
        _norm("norm_f8_layer", rows=524_288, dim=512, f8=True),
        # One vertex through a projection: the weights are all there is to read.
        _product("product_one_row", rows=1, dim=1024, out=1024),
        # First layer of the training batch, straight from the stored 8-bit rows.
        _product("product_b1024_by_id", rows=38_411, dim=256, out=256, ids=True, table=2_000_000, bias=True),
        # Odd sizes everywhere, results in full precision.
        _product("product_odd", rows=5_003, dim=602, out=172, dtype="f32"),
        # Layer-wise inference over a graph: large enough that the multiplications bound it.
        _product("product_layer", rows=131_072, dim=2048, out=1024),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["dropout", "norm", "norm", "norm_f8", "product", "product"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "product":
        dim, out = _log(rng, 32, 2048), _log(rng, 16, 1024)
        if rng.random() < 0.5:
            dim, out = -(-dim // 64) * 64, -(-out // 64) * 64
        rows = _log(rng, 1, 131_072)
        ids = rng.random() < 0.5
        c = _product("", rows=rows, dim=dim, out=out, dtype=dtype, ids=ids,
                     table=_log(rng, 1000, max(1000, min(2_000_000, 512_000_000 // dim))) if ids else 0, bias=rng.random() < 0.5)
    else:
        dim = _log(rng, 8, 4096)
        if rng.random() < 0.5:
            dim = -(-dim // 8) * 8
        rows = _log(rng, 1, max(1, min(524_288, 33_000_000 // dim)))
        if kind == "dropout":
            c = _dropout("", rows=rows, dim=dim, dtype=dtype, p=rng.choice([0.1, 0.3, 0.5]), train=rng.random() < 0.7)
        elif kind == "norm":
            c = _norm("", rows=rows, dim=dim, dtype=dtype, p=rng.choice([0.0, 0.1, 0.5]), residual=rng.random() < 0.7,
                      train=rng.random() < 0.6)
        else:
            c = _norm("", rows=rows, dim=dim, dtype=dtype, residual=rng.random() < 0.7, f8=True)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs --
def _rows(gen, rows, dim, dtype):
    """Feature-like rows: columns of unequal size, every 97th row zero (a vertex without features)."""
    x = torch.randn(rows, dim, generator=gen, device="cuda")
    x *= torch.rand(dim, generator=gen, device="cuda") * 2 + 0.1
    if rows > 97:
        x[::97] = 0
    return x.to(dtype)


def _encode_rows(x):
    """e4m3 codes (row pitch a multiple of 16 bytes) and scales of f32 rows."""
    rows, dim = x.shape
    blocks = -(-dim // BLOCK)
    s = torch.nn.functional.pad(x, (0, blocks * BLOCK - dim)).view(rows, blocks, BLOCK).abs().amax(2)
    s = (s / E4M3_MAX).clamp_min(TINY)
    codes = torch.zeros(rows, -(-dim // 16) * 16, dtype=torch.float8_e4m3fn, device=x.device)[:, :dim]
    codes.copy_((x / s.repeat_interleave(BLOCK, 1)[:, :dim]).to(torch.float8_e4m3fn))
    return codes, s


def _encode_weight(w):
    out, dim = w.shape
    ob, kb = -(-out // BLOCK), -(-dim // BLOCK)
    s = torch.nn.functional.pad(w, (0, kb * BLOCK - dim, 0, ob * BLOCK - out)).view(ob, BLOCK, kb, BLOCK).abs().amax((1, 3))
    s = (s / E4M3_MAX).clamp_min(TINY)
    codes = torch.zeros(out, -(-dim // 16) * 16, dtype=torch.float8_e4m3fn, device=w.device)[:, :dim]
    codes.copy_((w / s.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)[:out, :dim]).to(torch.float8_e4m3fn))
    return codes, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, dim, dtype = case["rows"], case["dim"], DTYPES[case["dtype"]]
    s = {"case": case, "seed": seed * 1_000_003 + 17, "offset": seed % 1000}
    if case["kind"] == "product":
        held = case["table"] if case["ids"] else rows
        s["codes"], s["scales"] = _encode_rows(_rows(gen, held, dim, torch.float32))
        s["w"], s["w_scales"] = _encode_weight(torch.randn(case["out"], dim, generator=gen, device="cuda") / math.sqrt(dim))
        if case["ids"]:
            s["ids"] = torch.randint(0, held, (rows,), generator=gen, device="cuda")
        if case["bias"]:
            s["bias"] = torch.randn(case["out"], generator=gen, device="cuda")
        return s
    s["x"] = _rows(gen, rows, dim, dtype).requires_grad_(case["train"])
    if case["kind"] == "norm":
        s["w"] = (1 + 0.2 * torch.randn(dim, generator=gen, device="cuda")).to(dtype).requires_grad_(case["train"])
        if case["residual"]:
            s["res"] = _rows(gen, rows, dim, dtype).requires_grad_(case["train"])
        if case["train"]:
            s["dh"] = torch.randn(rows, dim, generator=gen, device="cuda").to(dtype)
    if case["train"]:
        s["dy"] = torch.randn(rows, dim, generator=gen, device="cuda").to(dtype)
    return s


# -------------------------------------------------------------- plain forms --
def _philox(c0, c1, c2, c3, seed):
    """Philox4x32-10 over int64 tensors that hold 32-bit words."""
    low = 0xFFFFFFFF
    k0, k1 = seed & low, (seed >> 32) & low

    def high(a, m):  # upper word of a 32 x 32 bit product, in 16-bit halves of `a`
        return ((a >> 16) * m + (((a & 0xFFFF) * m) >> 16)) >> 16

    for _ in range(10):
        c0, c1, c2, c3 = (high(c2, 0xCD9E8D57) ^ c1 ^ k0, (c2 * 0xCD9E8D57) & low,
                          high(c0, 0xD2511F53) ^ c3 ^ k1, (c0 * 0xD2511F53) & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _threshold(p):
    return int(math.floor(65536 * p + 0.5))


def _mask(rows, dim, p, seed, offset):
    """f32 [rows, dim]: the scale where an element is kept, else 0."""
    t = _threshold(p)
    groups = -(-dim // 8)
    zero = torch.zeros(rows, groups, dtype=torch.int64, device="cuda")
    words = _philox(zero + torch.arange(groups, device="cuda"), zero + torch.arange(rows, device="cuda")[:, None],
                    zero + (offset & 0xFFFFFFFF), zero + (offset >> 32), seed)
    bits = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 2).view(rows, groups * 8)[:, :dim]
    return (bits >= t).float() * (65536 / max(1, 65536 - t))


def _plain_dropout(s, case):
    dtype = DTYPES[case["dtype"]]
    m = _mask(case["rows"], case["dim"], case["p"], s["seed"], s["offset"])
    y = (s["x"].float() * m).to(dtype)
    return (y, (s["dy"].float() * m).to(dtype)) if case["train"] else y


def _plain_norm(s, case):
    dtype, dim = DTYPES[case["dtype"]], case["dim"]
    x, w = s["x"].float(), s["w"].float()
    m = _mask(case["rows"], dim, case["p"], s["seed"], s["offset"]) if case["p"] else None
    h = x * m if m is not None else x
    if case["residual"]:
        h = h + s["res"].float()
    r = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
    y = h * r * w
    if case["f8"]:
        codes, scales = _encode_rows(y)
        return codes, scales, h.to(dtype)
    got = {"y": y.to(dtype), "h": h.to(dtype)}
    if case["train"]:
        dy = s["dy"].float()
        g = dy * w
        dh = s["dh"].float() + r * g - h * (r ** 3 / dim) * (g * h).sum(1, keepdim=True)
        got["dw"] = (dy * h * r).sum(0).to(dtype)
        got["dx"] = (dh * m if m is not None else dh).to(dtype)
        if case["residual"]:
            got["dres"] = dh.to(dtype)
    return got


def _plain_product(s, case):
    dim, out = case["dim"], case["out"]
    codes, scales = s["codes"], s["scales"]
    if case["ids"]:
        codes, scales = codes.view(torch.uint8)[s["ids"]].view(torch.float8_e4m3fn), scales[s["ids"]]
    a = codes.float() * scales.repeat_interleave(BLOCK, 1)[:, :dim]
    w = s["w"].float() * s["w_scales"].repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)[:out, :dim]
    y = a @ w.t()
    if case["bias"]:
        y = y + s["bias"]
    return y.to(DTYPES[case["dtype"]])


# ----------------------------------------------------------------- one pass --
def _own_dropout(s, case):
    from aethergraph_b200 import ops

    y = ops.dropout(s["x"], case["p"], s["seed"], s["offset"])
    return (y, torch.autograd.grad(y, s["x"], s["dy"])[0]) if case["train"] else y


def _own_norm(s, case):
    from aethergraph_b200 import ops

    x, w, res = s["x"], s["w"], s.get("res")
    if case["f8"]:
        return ops.add_rms_norm_f8(x, w, res, eps=EPS)
    y, h = ops.add_rms_norm(x, w, res, eps=EPS, p=case["p"], seed=s["seed"], offset=s["offset"])
    if not case["train"]:
        return {"y": y, "h": h}
    wrt = (x, w, res) if case["residual"] else (x, w)
    grads = torch.autograd.grad((y, h), wrt, (s["dy"], s["dh"]))
    return dict({"y": y, "h": h}, **dict(zip(("dx", "dw", "dres"), grads)))


def _own_product(s, case):
    from aethergraph_b200 import ops

    return ops.product_f8(s["codes"], s["scales"], s["w"], s["w_scales"], ids=s.get("ids"), bias=s.get("bias"),
                          dtype=DTYPES[case["dtype"]])


def run(state):
    case = state["case"]
    if own:
        return {"dropout": _own_dropout, "norm": _own_norm, "product": _own_product}[case["kind"]](state, case)
    with torch.no_grad():
        return {"dropout": _plain_dropout, "norm": _plain_norm, "product": _plain_product}[case["kind"]](state, case)


def work(case):
    rows, dim = case["rows"], case["dim"]
    n = rows * dim
    if case["kind"] == "product":
        out, blocks = case["out"], -(-dim // BLOCK)
        b = rows * (dim + 4 * blocks + (8 if case["ids"] else 0)) + out * dim + 4 * blocks * -(-out // BLOCK) + \
            (4 * out if case["bias"] else 0) + rows * out * BYTES[case["dtype"]]
        return {"bytes": b, "flops": 2 * rows * dim * out}
    e = BYTES[case["dtype"]]
    if case["kind"] == "dropout":
        return {"bytes": n * e * (4 if case["train"] else 2), "flops": n * (2 if case["train"] else 1)}
    summed = case["residual"] or case["p"] > 0  # otherwise h is x itself and nothing is written for it
    b = n * e * (1 + case["residual"] + summed) + (rows * (dim + 4 * -(-dim // BLOCK)) if case["f8"] else n * e) + dim * e
    f = n * 6
    if case["train"]:  # dy, dh and h read, dx and (where it differs from dx) the residual's gradient written
        b += n * e * (4 + (case["residual"] and case["p"] > 0)) + 2 * dim * e
        f += n * 12
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------ 64 bits --
def _exact_mask(rows, dim, p, seed, offset):
    """The keep mask times its scale, by numpy's 64-bit unsigned products, a slab of rows at a time."""
    t = _threshold(p)
    groups = (dim + 7) // 8
    got = np.empty((rows, dim))
    step = max(1, (1 << 20) // groups)
    for r0 in range(0, rows, step):
        n = min(step, rows - r0)
        ctr = [np.tile(np.arange(groups, dtype=np.uint64), n), np.repeat(np.arange(r0, r0 + n, dtype=np.uint64), groups),
               np.uint64(offset % (1 << 32)), np.uint64(offset // (1 << 32))]
        key = [seed % (1 << 32), (seed // (1 << 32)) % (1 << 32)]
        for _ in range(10):
            a, b = np.uint64(0xD2511F53) * ctr[0], np.uint64(0xCD9E8D57) * ctr[2]
            s32, m32 = np.uint64(32), np.uint64(0xFFFFFFFF)
            ctr = [(b >> s32) ^ ctr[1] ^ np.uint64(key[0]), b & m32, (a >> s32) ^ ctr[3] ^ np.uint64(key[1]), a & m32]
            key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
        u = np.stack(ctr, 1).astype("<u4").view("<u2").reshape(n, groups * 8)[:, :dim]  # little-endian: lower half first
        got[r0:r0 + n] = np.where(u >= t, 65536.0 / max(1, 65536 - t), 0.0)
    return torch.from_numpy(got).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        rows, dim = case["rows"], case["dim"]
        if case["kind"] == "product":
            a, sa = s["codes"].to(torch.float64), s["scales"].to(torch.float64)
            b, sb = s["w"].to(torch.float64), s["w_scales"].to(torch.float64)
            if case["ids"]:
                a, sa = a.index_select(0, s["ids"]), sa.index_select(0, s["ids"])
            y = torch.zeros(rows, case["out"], dtype=torch.float64, device="cuda")
            for k in range(sa.shape[1]):  # block by block, as the definition has it
                cols = slice(k * BLOCK, min(dim, (k + 1) * BLOCK))
                per_out = torch.repeat_interleave(sb[:, k], BLOCK)[:case["out"]]
                y += (a[:, cols] @ b[:, cols].t()) * sa[:, k, None] * per_out
            return y + s["bias"].to(torch.float64) if case["bias"] else y
        m = _exact_mask(rows, dim, case["p"], s["seed"], s["offset"]) if case["kind"] == "dropout" or case["p"] else 1.0
        x = s["x"].to(torch.float64)
        if case["kind"] == "dropout":
            return (x * m, s["dy"].to(torch.float64) * m) if case["train"] else x * m
        h = x * m + (s["res"].to(torch.float64) if case["residual"] else 0.0)
        w = s["w"].to(torch.float64)
        norm = torch.sqrt(torch.sum(h * h, 1, keepdim=True) / dim + EPS)
        u = h / norm
        y = u * w
        if case["f8"]:
            blocks = -(-dim // BLOCK)
            top = torch.stack([y[:, k * BLOCK:(k + 1) * BLOCK].abs().amax(1) for k in range(blocks)], 1)
            scales = torch.clamp(top / E4M3_MAX, min=TINY)
            return y / torch.repeat_interleave(scales, BLOCK, 1)[:, :dim], scales, h
        got = {"y": y, "h": h}
        if case["train"]:
            dy = s["dy"].to(torch.float64)
            du = dy * w
            dh = s["dh"].to(torch.float64) + (du - u * torch.mean(du * u, 1, keepdim=True)) / norm
            got.update(dw=torch.sum(dy * u, 0), dx=dh * m)
            if case["residual"]:
                got["dres"] = dh
        return got
