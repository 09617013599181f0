"""The operators around the search in 64 bits (torch on the CPU), from their
definitions, with bounds on what float32 arithmetic may add to each value."""
from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def d64(t):
    return None if t is None else t.detach().cpu().double()


def assert_close(got, want, bound, name=""):
    """|got - want| <= bound + the rounding of want to got's type, everywhere."""
    unit, tiny = UNIT[got.dtype], TINY[got.dtype]
    got = d64(got)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    room = bound * (1 + unit) + unit * want.abs() + tiny
    bad = ~(same | ((got - want).abs() <= room))
    if bad.any():
        at = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values off; at {at} got {got[at].item()!r}, "
                             f"want {want[at].item()!r}, room {room.expand_as(want)[at].item()!r}")


# ------------------------------------------------------------------ layer norm
def norm(x, w, b, eps):
    """y, its bound, mean, rstd."""
    width = x.shape[1]
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = (c.square().mean(1, keepdim=True) + eps).rsqrt()
    xh = c * rstd
    one = torch.ones(width, dtype=torch.float64)
    w = one if w is None else w
    y = xh * w + (0 if b is None else b)
    # A sum of n terms in any order is off by at most n u sum |terms|; the
    # mean so by width u mean|x|, which moves every deviation.
    off = (width + 8) * U32 * x.abs().mean(1, keepdim=True) * rstd
    xh_off = off * (1 + xh.abs()) + (width + 16) * U32 * xh.abs()
    return y, xh_off * w.abs() + 4 * U32 * y.abs(), mean, rstd, xh, xh_off


def norm_grads(dy, x, w, eps):
    """(dx, dw, db) with a bound each."""
    rows, width = x.shape
    _, _, _, rstd, xh, xh_off = norm(x, w, None, eps)
    w = torch.ones(width, dtype=torch.float64) if w is None else w
    g = dy * w
    mg, mgx = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rstd * (g - mg - xh * mgx)
    n = (width + 16) * U32
    mgx_off = (g.abs() * xh_off).mean(1, keepdim=True) + n * (g * xh).abs().mean(1, keepdim=True)
    dx_off = rstd * (n * g.abs().mean(1, keepdim=True) + xh.abs() * mgx_off + xh_off * mgx.abs()
                     + 4 * U32 * (g.abs() + mg.abs() + (xh * mgx).abs())) + n * dx.abs()
    dw, db = (dy * xh).sum(0), dy.sum(0)
    m = (rows + 8) * U32
    dw_off = (dy.abs() * xh_off).sum(0) + m * (dy * xh).abs().sum(0)
    return (dx, dx_off), (dw, dw_off), (db, m * dy.abs().sum(0))


# ------------------------------------------------------------------ linear
def activate(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * 0.5 * (1 + torch.erf(z / math.sqrt(2)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def linear(x, w, b, name, res):
    """y and its bound, z and its bound.  No activation here is steeper than 1.13."""
    z = x @ w.T
    off = 2 * (x.shape[1] + 8) * U32 * (x.abs() @ w.abs().T)
    if b is not None:
        z = z + b
        off = off + 2 * U32 * (b.abs() + z.abs())
    y = activate(z, name)
    y_off = 1.13 * off + 16 * U32 * z.abs()
    if res is not None:
        y = y + res
        y_off = y_off + 2 * U32 * (y.abs() + res.abs())
    return y, y_off, z, off


def linear_grads(dy, x, w, z, z_off, name, kind):
    """(dx, dw, db) with a bound each, where dz and the kept z are rounded to ``kind``.

    z moves by its rounding and by the product's own bound; no slope here
    changes faster than 0.8."""
    unit = UNIT[kind]
    dz = dy * slope(z, name)
    steep = 0.0 if name in (None, "none", "relu") else 0.8
    dz32_off = dy.abs() * (steep * (unit * z.abs() + z_off * (1 + unit)) + 32 * U32) + 4 * U32 * dz.abs()
    rounded = 0.0 if name in (None, "none") else unit
    dz_off = dz32_off * (1 + unit) + rounded * dz.abs() + TINY[kind]
    m, n = dy.shape
    both = dz.abs() + dz_off
    dx, dw, db = dz @ w, dz.T @ x, dz.sum(0)
    dx_off = dz_off @ w.abs() + 2 * (n + 8) * U32 * (both @ w.abs())
    dw_off = dz_off.T @ x.abs() + 2 * (m + 8) * U32 * (both.T @ x.abs())
    return (dx, dx_off), (dw, dw_off), (db, dz32_off.sum(0) + (m + 8) * U32 * both.sum(0))


# ------------------------------------------------------------------ rows in 8 bits
def quantise(x, group):
    """(codes, scales) of float32 rows, each step rounded to float32 as the definition says."""
    x = x.detach().cpu().float()
    n, width = x.shape
    group = group or width
    codes = torch.zeros((n, width), dtype=torch.int8)
    scales = torch.zeros((n, -(-width // group)))
    for g in range(scales.shape[1]):
        part = x[:, g * group:(g + 1) * group]
        top = part.abs().amax(1)  # NaN where one is
        some = torch.isfinite(top) & (top >= 2.0 ** -100)
        inv = torch.where(some, (1 / top.double()).float() * 127, 0.0)
        code = (part * inv[:, None]).round()
        codes[:, g * group:(g + 1) * group] = torch.where(some[:, None], code, 0.0).to(torch.int8)
        scales[:, g] = torch.where(some, top * torch.tensor(1 / 127), torch.where(torch.isfinite(top), 0.0, top))
    return codes, scales


def quantise_affine(x, lo, step):
    lo, inv = torch.tensor(lo), torch.tensor(1 / step)
    v = (x.detach().cpu().float() - lo) * inv
    return torch.nan_to_num(v, nan=0.0).clamp(0, 255).round().to(torch.uint8)


def stands_for(codes, scales, group, lo, step):
    """The float32 values of rows, as they are read back."""
    c = codes.cpu().float()
    if scales is None:
        return torch.tensor(lo) + torch.tensor(step) * c
    group = group or c.shape[1]
    return c * scales.cpu().repeat_interleave(group, 1)[:, :c.shape[1]]


# ------------------------------------------------------------------ attention over found rows
def attend(q, ids, k, v, scale, cap, bias=None, query_docs=None, row_docs=None, dout=None):
    """From float64 queries [nq][heads][head] and rows [slots][groups][head]:
    a dict of (value, bound) for out, lse and, with dout, dq and dbias."""
    nq, heads, head = q.shape
    slots, groups, _ = k.shape
    found = ids.shape[1]
    hidden = (ids < 0) | (ids >= slots)
    at = torch.where(hidden, 0, ids).long()
    if row_docs is not None:
        hidden = hidden | (row_docs[at] != query_docs[:, None])
    if bias is not None:
        hidden = hidden | (bias == -math.inf)
    kk = torch.where(hidden[:, :, None, None], 0.0, k[at]).repeat_interleave(heads // groups, 2)  # [nq][found][heads][head]
    vv = torch.where(hidden[:, :, None, None], 0.0, v[at]).repeat_interleave(heads // groups, 2)
    s = scale * torch.einsum("qhd,qkhd->qhk", q, kk)
    s_off = (head + 16) * U32 * abs(scale) * torch.einsum("qhd,qkhd->qhk", q.abs(), kk.abs())
    t = torch.zeros_like(s)
    if cap:
        t = torch.tanh(s / cap)
        s = cap * t
        s_off = s_off + 8 * U32 * cap
    if bias is not None:
        s = s + bias[:, None]
        s_off = s_off + 2 * U32 * (s.abs() + bias[:, None].abs())
    s = s.masked_fill(hidden[:, None], -math.inf)
    s_off = torch.where(hidden[:, None], 0.0, s_off)
    if found == 0:
        lse = torch.full((nq, heads), -math.inf, dtype=torch.float64)
    else:
        lse = torch.logsumexp(s, 2)
    p = torch.where(torch.isneginf(s), 0.0, torch.exp(s - lse[..., None].clamp(min=-1e300)))
    worst = s_off.amax(2) if found else torch.zeros((nq, heads), dtype=torch.float64)
    # exp of a difference: its argument's error, itself up to |s| u, and the function's few units.
    size = torch.where(torch.isneginf(s), 0.0, s).abs().amax(2) if found else worst
    rel = 2 * worst + (4 * size + 2 * found + 16) * U32
    out = torch.einsum("qhk,qkhd->qhd", p, vv)
    off = rel[..., None] * torch.einsum("qhk,qkhd->qhd", p, vv.abs())
    r = {"out": (out, off), "lse": (lse, rel + 4 * U32 * torch.where(torch.isinf(lse), 0.0, lse).abs())}
    if dout is not None:
        dp = torch.einsum("qhd,qkhd->qhk", dout, vv)
        dp_off = (head + 16) * U32 * torch.einsum("qhd,qkhd->qhk", dout.abs(), vv.abs())
        big = (p * dp).sum(2, keepdim=True)
        big_off = (p * dp_off).sum(2, keepdim=True) + rel[..., None] * (p * dp.abs()).sum(2, keepdim=True)
        ds = p * (dp - big)
        ds_off = rel[..., None] * p * (dp.abs() + big.abs()) + p * (dp_off + big_off)
        sl = 1 - t * t
        sl_off = 16 * U32 + (2 * s_off / cap if cap else 0.0)
        dq = scale * torch.einsum("qhk,qkhd->qhd", ds * sl, kk)
        # dq as scale (A - D B): each of the two sums carries its own error.
        both = p * (dp.abs() + big.abs())
        dq_off = abs(scale) * torch.einsum("qhk,qkhd->qhd", ds_off + both * (sl_off + (2 * found + 16) * U32), kk.abs())
        r["dq"] = (dq, dq_off)
        r["dbias"] = (ds.sum(1), ds_off.sum(1) + (heads + 4) * U32 * ds.abs().sum(1))
    return r
