"""The operators around the search on the GPU against their 64-bit forms:
layer norm, linear, the 8-bit row cache and attention over found rows, where
sizes, strides and masks can go wrong."""
import math

import pytest
import torch

import memory_plain as plain
from memory_plain import assert_close, d64

pytestmark = pytest.mark.gpu

memory = pytest.importorskip("winnex_madhava.memory")

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
KINDS = [F32, BF16, F16]


def rand(seed, *shape, kind=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(kind).cuda()


# ------------------------------------------------------------------ layer norm
def check_norm(x, w, b, eps, dy):
    y, mean, rstd = memory.layer_norm_forward(x, w, b, eps=eps)
    x64, w64, b64 = d64(x), d64(w), d64(b)
    want, off, m, r, _, _ = plain.norm(x64, w64, b64, eps)
    assert_close(y, want, off, "y")
    n = (x.shape[1] + 8) * plain.U32
    assert_close(mean, m[:, 0], n * x64.abs().mean(1), "mean")
    assert_close(rstd, r[:, 0], r[:, 0] * (n + n * x64.abs().mean(1) * r[:, 0]), "rstd")
    assert torch.equal(memory.layer_norm(x, w, b, eps=eps), y)
    got = memory.layer_norm_backward(dy, x, w, mean, rstd, weight_dtype=None if b is None else b.dtype)
    for name, g, (value, bound) in zip(("dx", "dw", "db"), got, plain.norm_grads(d64(dy), x64, w64, eps)):
        assert_close(g, value, bound, name)
    again = memory.layer_norm_backward(dy, x, w, mean, rstd, weight_dtype=None if b is None else b.dtype)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 768), (3, 7), (9, 256), (5, 264), (17, 301), (4, 520), (33, 1024),
                                        (2, 1032), (5, 1999), (3, 8192), (2, 16384), (700, 48), (2500, 200)])
def test_layer_norm_sizes(kind, rows, width):
    own = rows % 2 == 0  # weights of the rows' type, or float32
    w = rand(1, width, kind=kind if own else F32, scale=0.2, shift=1.0)
    b = rand(2, width, kind=w.dtype, scale=0.2)
    check_norm(rand(3, rows, width, kind=kind, scale=1.5, shift=0.3), w, b, 1e-5, rand(4, rows, width, kind=kind))


@pytest.mark.parametrize("kind", KINDS)
def test_layer_norm_without_weights_and_strided(kind):
    wide = rand(5, 40, 256, kind=kind)
    dy = rand(6, 40, 200, kind=kind)
    check_norm(wide[:, :200], None, None, 1e-6, dy)          # rows with a gap
    check_norm(wide[:, 3:203], None, None, 1e-6, dy)         # that start off a 16-byte boundary
    check_norm(wide[::2, 8:208], rand(7, 200, kind=kind), None, 1e-6, dy[:20])


def test_layer_norm_large_offset_keeps_its_variance():
    x = rand(8, 6, 768, shift=1000.0)
    check_norm(x, rand(9, 768), rand(10, 768), 1e-5, rand(11, 6, 768))


def test_layer_norm_constant_and_non_finite_rows():
    x = torch.ones(4, 300, device="cuda")
    x[1, 5] = math.inf
    x[2, 7] = math.nan
    y, mean, rstd = memory.layer_norm_forward(x, None, None, eps=1e-5)
    assert torch.equal(y[0], torch.zeros_like(y[0])) and torch.equal(y[3], torch.zeros_like(y[3]))
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()


def test_layer_norm_no_rows():
    x = torch.empty(0, 96, device="cuda", dtype=BF16)
    y, mean, rstd = memory.layer_norm_forward(x)
    dx, dw, db = memory.layer_norm_backward(x, x, None, mean, rstd)
    assert y.shape == dx.shape == (0, 96) and not dw.any() and not db.any()


def test_layer_norm_autograd_and_differences():
    x, w, b = rand(12, 5, 50).requires_grad_(), rand(13, 50).requires_grad_(), rand(14, 50).requires_grad_()
    dy = rand(15, 5, 50)
    memory.layer_norm(x, w, b).backward(dy)
    for k, t in enumerate((x, w, b)):
        along = rand(16 + k, *t.shape)
        h = 2.0 ** -6
        args = [v.detach() for v in (x, w, b)]

        def value(sign):
            moved = list(args)
            moved[k] = moved[k] + sign * h * along
            return (d64(memory.layer_norm(*moved)) * d64(dy)).sum()

        slope = (value(1) - value(-1)) / (2 * h)
        # Float32 values of size ~4 in 250 terms over 2h, and the third derivative times h^2.
        room = 250 * 4 * 4 * 2.0 ** -24 / h + 250 * h * h
        assert abs(slope - (d64(t.grad) * d64(along)).sum()) < room


# ------------------------------------------------------------------ linear
def check_linear(x, w, b, name, res, dy):
    y, z = memory.linear_forward(x, w, b, activation=name, residual=res, keep_preactivation=True)
    want, off, z64, z_off = plain.linear(d64(x), d64(w), d64(b), name, d64(res))
    assert_close(y, want, off, "y")
    assert torch.equal(memory.linear(x, w, b, activation=name, residual=res), y)
    assert (z is None) == (name in (None, "none"))
    if z is not None:
        assert_close(z, z64, z_off, "z")
    got = memory.linear_backward(dy, x, w, z, activation=name)
    grads = plain.linear_grads(d64(dy), d64(x), d64(w), z64, z_off, name, x.dtype)
    for label, g, (value, bound) in zip(("dx", "dw", "db"), got, grads):
        assert_close(g, value, bound, label)
    again = memory.linear_backward(dy, x, w, z, activation=name)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


# Integer-valued operands: relu's z is exact and, with a bias off the integers, never 0.
def whole(seed, *shape, kind):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-2, 3, shape, generator=g).to(kind).cuda()


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("name", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [(1, 8, 8), (1, 768, 768), (3, 48, 200), (17, 300, 130), (128, 64, 256),
                                   (129, 72, 264), (200, 1000, 96), (300, 129, 77), (1, 1, 1), (5, 7, 9)])
def test_linear_sizes(kind, name, m, k, n):
    if name == "relu":
        x, w = whole(1, m, k, kind=kind), whole(2, n, k, kind=kind)
        b = torch.full((n,), 0.5, dtype=kind, device="cuda")
    else:
        x, w = rand(1, m, k, kind=kind), rand(2, n, k, kind=kind, scale=k ** -0.5)
        b = rand(3, n, kind=kind, scale=0.1)
    res = rand(4, m, n, kind=kind) if m % 2 else None
    check_linear(x, w, b, name, res, rand(5, m, n, kind=kind))


@pytest.mark.parametrize("m,k,n", [(2000, 256, 128), (1500, 768, 520), (4096, 128, 64), (40, 2048, 640), (64, 4096, 8)])
def test_linear_larger(m, k, n):
    check_linear(rand(1, m, k, kind=BF16), rand(2, n, k, kind=BF16, scale=k ** -0.5), None, "gelu", None,
                 rand(5, m, n, kind=BF16))


@pytest.mark.parametrize("kind", [BF16, F16])
def test_linear_strided_operands(kind):
    m, k, n = 70, 136, 88
    x, w = rand(1, m, 3 * k, kind=kind)[:, k:2 * k], rand(2, n, k + 8, kind=kind, scale=0.1)[:, :k]
    res, dy = rand(3, m, 2 * n, kind=kind)[:, :n], rand(4, m, 2 * n, kind=kind)[:, n:]
    check_linear(x, w, None, "silu", res, dy)
    # Rows that start off a 16-byte boundary, with a stride that is no multiple of it.
    x, w = rand(5, m, k + 5, kind=kind)[:, 3:3 + k], rand(6, n, k + 3, kind=kind, scale=0.1)[:, 1:1 + k]
    res, dy = rand(7, m, n + 5, kind=kind)[:, 5:], rand(8, m, n + 1, kind=kind)[:, :n]
    check_linear(x, w, rand(9, n + 1, kind=kind)[1:], "gelu", res, dy)


def test_linear_no_rows_and_parts():
    x, w = torch.empty(0, 24, device="cuda", dtype=BF16), rand(1, 16, 24, kind=BF16)
    y, z = memory.linear_forward(x, w, activation="gelu", keep_preactivation=True)
    dx, dw, db = memory.linear_backward(y, x, w, z, activation="gelu")
    assert y.shape == (0, 16) and dx.shape == (0, 24) and not dw.any() and not db.any()
    x, dy = rand(2, 30, 24, kind=BF16), rand(3, 30, 16, kind=BF16)
    full = memory.linear_backward(dy, x, w)
    for k in range(3):
        some = memory.linear_backward(dy, x, w, need=tuple(i == k for i in range(3)))
        assert torch.equal(some[k], full[k]) and all(some[i] is None for i in range(3) if i != k)


def test_linear_autograd_leading_dimensions():
    x = rand(1, 2, 9, 40, kind=BF16).requires_grad_()
    w, b = rand(2, 24, 40, kind=BF16, scale=0.2).requires_grad_(), rand(3, 24, kind=BF16).requires_grad_()
    res, dy = rand(4, 2, 9, 24, kind=BF16).requires_grad_(), rand(5, 2, 9, 24, kind=BF16)
    y = memory.linear(x, w, b, activation="gelu", residual=res)
    y.backward(dy)
    _, z = memory.linear_forward(x.detach(), w.detach(), b.detach(), activation="gelu", keep_preactivation=True)
    dx, dw, db = memory.linear_backward(dy, x.detach(), w.detach(), z, activation="gelu")
    assert y.shape == (2, 9, 24)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw) and torch.equal(b.grad, db)
    assert torch.equal(res.grad, dy)


def test_linear_gradients_against_differences():
    """The 64-bit gradients that the kernels are held to are the slopes of the 64-bit forward pass."""
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((6, 10), (7, 10), (7,), (6, 7)))
    for name in ("none", "gelu", "silu", "relu"):
        z = x @ w.T + b
        grads = plain.linear_grads(dy, x, w, z, torch.zeros_like(z), name, F32)
        for k, t in enumerate((x, w, b)):
            along, h = torch.randn(t.shape, generator=g, dtype=torch.float64), 1e-6

            def value(sign):
                a = [x, w, b]
                a[k] = a[k] + sign * h * along
                return (plain.activate(a[0] @ a[1].T + a[2], name) * dy).sum()

            slope = (value(1) - value(-1)) / (2 * h)
            assert abs(slope - (grads[k][0] * along).sum()) < 1e-6 * (1 + abs(slope))


def test_linear_values_out_of_range_stay_visible():
    x = torch.full((4, 64), 300.0, dtype=F16, device="cuda")
    w = torch.full((8, 64), 300.0, dtype=F16, device="cuda")
    assert torch.isinf(memory.linear(x, w)).all()
    x[1, 3] = math.nan
    y = memory.linear(x, w, activation="relu")
    assert torch.isnan(y[1]).all() and torch.isinf(y[0]).all()


# ------------------------------------------------------------------ rows in 8 bits
def new_cache(slots, width, group, code):
    if code == "uint8":
        return memory.RowCache.empty(slots, width, code=code, lo=-3.0, step=6.5 / 255)
    return memory.RowCache.empty(slots, width, group=group)


def check_rows(cache, at, x, kind):
    cache.write(at, x)
    keep = ((at >= 0) & (at < cache.slots)).cpu()
    slots = at.cpu()[keep].long()
    if cache.scales is None:
        codes, scales = plain.quantise_affine(x, cache.lo, cache.step), None
    else:
        codes, scales = plain.quantise(x, cache.group)
        assert torch.equal(torch.nan_to_num(cache.scales.cpu()[slots], nan=-1.0),
                           torch.nan_to_num(scales[keep], nan=-1.0))
    assert torch.equal(cache.codes.cpu()[slots], codes[keep])
    back = cache.read(at, dtype=kind)
    want = plain.stands_for(codes, scales, cache.group, cache.lo, cache.step).to(kind)
    want[~keep] = 0
    assert torch.equal(torch.nan_to_num(back.cpu(), nan=7.0), torch.nan_to_num(want, nan=7.0))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width,group,code", [(1, 0, "int8"), (7, 16, "int8"), (48, 16, "int8"), (64, 64, "int8"),
                                              (300, 32, "int8"), (768, 64, "int8"), (768, 0, "int8"), (200, 48, "int8"),
                                              (1999, 128, "int8"), (1024, 256, "int8"), (520, 512, "int8"),
                                              (2500, 0, "int8"), (136, 112, "int8"),
                                              (128, 0, "uint8"), (7, 0, "uint8"), (301, 0, "uint8"), (768, 0, "uint8")])
def test_rows_written_and_read(kind, width, group, code):
    n, slots = 53, 90
    cache = new_cache(slots, width, group, code)
    at = torch.randperm(slots, generator=torch.Generator().manual_seed(width))[:n].to(torch.int32).cuda()
    at[::7] = -1
    at[3] = slots
    check_rows(cache, at, rand(width, n, width, kind=kind), kind)
    untouched = torch.ones(slots, dtype=torch.bool)
    untouched[at.cpu()[(at >= 0).cpu() & (at < slots).cpu()].long()] = False
    assert not cache.codes.cpu()[untouched].any()
    if cache.scales is not None:
        assert not cache.scales.cpu()[untouched].any()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_strided_unaligned_and_int64(kind):
    slots, width = 40, 96
    base = torch.zeros(slots, 111, dtype=torch.int8, device="cuda")
    scales = torch.zeros(slots, 3, device="cuda")
    at = torch.arange(slots - 1, -1, -1, device="cuda")
    x = rand(1, slots, 2 * width + 1, kind=kind)[:, 3:3 + width]
    check_rows(memory.RowCache(base[:, 5:5 + width], scales, group=32), at, x, kind)
    assert not base[:, :5].any() and not base[:, 5 + width:].any()
    check_rows(memory.RowCache(base[:, :width], scales, group=32), at, x, kind)
    check_rows(memory.RowCache(base[:, 8:8 + width].view(torch.uint8), lo=-2.0, step=0.02), at, x, kind)


def test_rows_extremes():
    x = torch.zeros(12, 64, device="cuda")
    x[0] = 3.4e38
    x[1, 3] = math.inf
    x[2, 40] = math.nan
    x[3, 5] = 2.0 ** -101
    x[4, 5] = 2.0 ** -100
    x[5, 6] = -1e-45
    x[6] = torch.arange(64, device="cuda") + 0.5          # ties to even
    x[6, 63] = 127.0
    x[7, :5] = torch.tensor([-127.0, 0.5, 1.5, 2.5, -0.5])
    check_rows(memory.RowCache.empty(12, 64, group=32), torch.arange(12, device="cuda"), x, F32)
    x[8, :6] = torch.tensor([-math.inf, math.inf, math.nan, -3.0, 3.5, 9.0])
    check_rows(new_cache(12, 64, 0, "uint8"), torch.arange(12, device="cuda"), x, F32)


def test_rows_empty_calls():
    cache = memory.RowCache.empty(5, 32)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    cache.write(none, torch.empty(0, 32, device="cuda"))
    assert cache.read(none).shape == (0, 32)
    nothing = memory.RowCache.empty(0, 32)
    ids = torch.tensor([[0, -1], [3, 7]], device="cuda")
    nothing.write(ids[0].contiguous(), rand(1, 2, 32))
    assert not nothing.read(ids).any() and nothing.read(ids).shape == (2, 2, 32)


# ------------------------------------------------------------------ attention over found rows
def filled(slots, width, group, code, seed):
    cache = memory.RowCache.empty(slots, width, code=code, group=group, lo=-2.0, step=4 / 255)
    cache.write(torch.arange(slots, device="cuda"), rand(seed, slots, width))
    return cache


def held(cache, head):
    """What the codes stand for in 64 bits (the stored scale is a float32 value)."""
    c = cache.codes.cpu().double()
    if cache.scales is None:
        v = float(torch.tensor(cache.lo)) + float(torch.tensor(cache.step)) * c
    else:
        v = c * cache.scales.cpu().double().repeat_interleave(cache.group or cache.width, 1)[:, :cache.width]
    return v.view(cache.slots, -1, head)


def check_attend(q, ids, keys, values, dout, cap=0.0, bias=None, query_docs=None, row_docs=None, scale=None):
    how = dict(cap=cap, bias=bias, query_docs=query_docs, row_docs=row_docs, scale=scale)
    out, lse = memory.attend(q, ids, keys, values, **how)
    head = q.shape[2]
    cpu = [None if t is None else t.cpu() for t in (query_docs, row_docs)]
    want = plain.attend(d64(q), ids.cpu(), held(keys, head), held(values, head), head ** -0.5 if scale is None else scale,
                        cap, d64(bias), *cpu, d64(dout))
    assert_close(out, *want["out"], "out")
    assert_close(lse, *want["lse"], "lse")
    dq, dbias = memory.attend_backward(dout, q, ids, keys, values, lse, **how)
    assert_close(dq, *want["dq"], "dq")
    assert (dbias is None) == (bias is None)
    if bias is not None:
        assert_close(dbias, *want["dbias"], "dbias")
    o2, l2 = memory.attend(q, ids, keys, values, **how)
    g2, b2 = memory.attend_backward(dout, q, ids, keys, values, lse, **how)
    assert torch.equal(out, o2) and torch.equal(lse, l2) and torch.equal(dq, g2)
    assert bias is None or torch.equal(dbias, b2)
    return out, lse, dq


def lists(seed, nq, found, slots):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, slots, (nq, found), generator=g, dtype=torch.int32)
    keep = torch.randint(0, found + 2, (nq, 1), generator=g)
    return torch.where(torch.arange(found) < keep, ids, -1).cuda()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nq,found,groups,shared,head,group,code", [
    (1, 1, 1, 1, 8, 0, "int8"), (1, 32, 4, 3, 64, 64, "int8"), (5, 10, 12, 1, 64, 64, "int8"),
    (3, 7, 2, 4, 40, 16, "int8"), (4, 33, 3, 2, 96, 32, "int8"), (2, 300, 1, 8, 128, 128, "int8"),
    (3, 65, 2, 5, 256, 0, "int8"), (2, 17, 1, 1, 200, 48, "int8"), (4, 20, 2, 2, 32, 0, "uint8"),
    (2, 1500, 2, 2, 64, 64, "int8"), (1, 4096, 1, 3, 24, 16, "int8"), (3, 12, 5, 1, 16, 80, "int8"),
    (2, 40, 3, 7, 72, 0, "uint8"), (300, 3, 2, 1, 64, 32, "int8"), (1, 2000, 8, 16, 128, 64, "int8")])
def test_attend_sizes(kind, nq, found, groups, shared, head, group, code):
    slots = 500
    keys, values = (filled(slots, groups * head, group, code, s) for s in (1, 2))
    q, dout = (rand(s, nq, groups * shared, head, kind=kind) for s in (3, 4))
    ids = lists(nq * found, nq, found, slots)
    check_attend(q, ids, keys, values, dout)
    bias = -3 * torch.rand(nq, found, generator=torch.Generator().manual_seed(5)).cuda()
    docs = torch.randint(0, 2, (slots,), generator=torch.Generator().manual_seed(6), dtype=torch.int32).cuda()
    check_attend(q, ids, keys, values, dout, cap=2.5, bias=bias, query_docs=docs[:nq].contiguous(), row_docs=docs)


@pytest.mark.parametrize("kind", KINDS)
def test_attend_masks(kind):
    slots, found, head = 64, 20, 64
    keys, values = filled(slots, 2 * head, 64, "int8", 1), filled(slots, 2 * head, 64, "int8", 2)
    # Rows that no query may see hold NaN.
    keys.scales[5], values.scales[6] = math.nan, math.inf
    nq = 8
    q, dout = rand(3, nq, 4, head, kind=kind), rand(4, nq, 4, head, kind=kind)
    ids = torch.arange(nq * found, device="cuda", dtype=torch.int32).view(nq, found) % slots
    bias = rand(5, nq, found)
    bias[(ids == 5) | (ids == 6)] = -math.inf
    ids[1] = -1                                  # an empty list
    ids[2] = 2 ** 31 - 1                         # ids past the cache
    bias[3] = -math.inf                          # a mask that leaves nothing
    bias[4][bias[4] != -math.inf] = torch.finfo(F32).min   # the type's lowest value is no mask: all weigh alike
    bias[5, 1:] = -math.inf                      # one entry left
    ids[5, 0] = 9
    out, lse, dq = check_attend(q, ids, keys, values, dout, bias=bias)
    for i in (1, 2, 3):
        assert not out[i].any() and torch.isneginf(lse[i]).all() and not dq[i].any()
    assert torch.isfinite(out).all() and torch.isfinite(dq).all()
    docs = torch.where(torch.arange(slots) % 5 == 0, 1, 0).to(torch.int32).cuda()
    mine = torch.tensor([0, 1, 2, 0, 0, 0, 2, 1], dtype=torch.int32, device="cuda")  # document 2 has no row
    out, lse, _ = check_attend(q, ids, keys, values, dout, bias=bias, query_docs=mine, row_docs=docs)
    assert torch.isneginf(lse[6]).all() and not out[6].any()


@pytest.mark.parametrize("kind", KINDS)
def test_attend_large_scores(kind):
    """Scores of some thousands: the maximum carries the softmax, whatever its place in the list."""
    head, slots, found = 64, 300, 200
    keys, values = filled(slots, head, 0, "int8", 1), filled(slots, head, 0, "int8", 2)
    q, dout = rand(3, 4, 2, head, kind=kind, scale=8), rand(4, 4, 2, head, kind=kind)
    ids = lists(7, 4, found, slots)
    check_attend(q, ids, keys, values, dout, scale=0.5)
    check_attend(q, ids, keys, values, dout, scale=-0.5, cap=50.0)


def test_attend_strided_and_shared_lists():
    head, slots, nq, found = 32, 100, 6, 9
    keys, values = filled(slots, 4 * head, 32, "int8", 1), filled(slots, 4 * head, 32, "uint8", 2)
    q = rand(3, nq, 3, 8, head + 5, kind=BF16)[:, 1, :, 2:2 + head]
    dout = rand(4, nq, 8, head, kind=BF16)
    ids = lists(8, nq, found + 4, slots)[:, 3:3 + found]
    bias = rand(5, nq, found + 1)[:, :found]
    check_attend(q, ids, keys, values, dout, bias=bias)
    check_attend(q, ids[:1].expand(nq, found), keys, values, dout, bias=bias[:1].expand(nq, found))
    # Cache rows of an odd byte stride that start anywhere.
    base = torch.randint(-127, 128, (slots, 4 * head + 9), dtype=torch.int8, device="cuda")
    odd = memory.RowCache(base[:, 3:3 + 4 * head], keys.scales, group=32)
    check_attend(q, ids, odd, values, dout, bias=bias)
    check_attend(q, ids, keys, odd, dout, bias=bias)


def test_attend_nothing():
    keys, values = filled(10, 64, 64, "int8", 1), filled(10, 64, 64, "int8", 2)
    q = rand(1, 3, 2, 64)
    out, lse, dq = check_attend(q, torch.empty(3, 0, dtype=torch.int32, device="cuda"), keys, values, q)
    assert not out.any() and torch.isneginf(lse).all() and not dq.any()
    out, lse = memory.attend(q[:0], torch.empty(0, 4, dtype=torch.int32, device="cuda"), keys, values)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    nothing = memory.RowCache.empty(0, 64)
    out, lse = memory.attend(q, torch.zeros(3, 4, dtype=torch.int32, device="cuda"), nothing, nothing)
    assert not out.any() and torch.isneginf(lse).all()


def test_attend_autograd_and_differences():
    keys, values = filled(50, 64, 16, "int8", 1), filled(50, 64, 16, "int8", 2)
    q, bias = rand(3, 3, 4, 32).requires_grad_(), rand(4, 1, 12).requires_grad_()  # one bias for every query
    ids, dout = lists(9, 3, 12, 50), rand(5, 3, 4, 32)

    def run(q, bias):
        return memory.attend(q, ids, keys, values, cap=3.0, bias=bias.expand(3, 12))[0]

    run(q, bias).backward(dout)
    h = 2.0 ** -6
    for t, other in ((q, bias), (bias, q)):
        along = rand(6, *t.shape)

        def value(sign):
            moved, rest = t.detach() + sign * h * along, other.detach()
            return (d64(run(*((moved, rest) if t is q else (rest, moved)))) * d64(dout)).sum()

        slope = (value(1) - value(-1)) / (2 * h)
        # Float32 outputs of size ~2 in 384 terms over 2h, and the third derivative times h^2.
        assert abs(slope - (d64(t.grad) * d64(along)).sum()) < 384 * 2 * 16 * 2.0 ** -24 / h + 384 * h * h


def test_attend_joins_by_lse():
    """Two halves of a list joined by their lse are the whole list."""
    keys, values = filled(80, 128, 64, "int8", 1), filled(80, 128, 64, "int8", 2)
    q, ids = rand(3, 5, 2, 64), lists(10, 5, 24, 80)
    o, z = memory.attend(q, ids, keys, values)
    parts = [memory.attend(q, ids[:, s], keys, values) for s in (slice(0, 9), slice(9, 24))]
    w = torch.softmax(torch.stack([p[1] for p in parts]).double(), 0)
    joined = torch.nan_to_num(w[0])[..., None] * parts[0][0] + torch.nan_to_num(w[1])[..., None] * parts[1][0]
    assert (joined - o).abs().max() < 64 * 2.0 ** -24 * 4
    total = torch.logaddexp(parts[0][1].double(), parts[1][1].double())
    assert torch.equal(torch.isneginf(total), torch.isneginf(z))
    assert ((total - z)[~torch.isneginf(z)].abs() < 64 * 2.0 ** -24 * 8).all()


# ------------------------------------------------------------------ streams and graphs
def test_other_stream_and_graph():
    """Everything runs on the current stream and can be captured."""
    x, w, b = rand(1, 300, 96, kind=BF16), rand(2, 64, 96, kind=BF16), rand(3, 64, kind=BF16)
    dy = rand(4, 300, 64, kind=BF16)
    cache, cache2 = memory.RowCache.empty(300, 64), memory.RowCache.empty(300, 64)
    at, ids = torch.arange(300, device="cuda"), lists(3, 20, 8, 300)

    def work(cache):
        n, mean, rstd = memory.layer_norm_forward(x)
        y, z = memory.linear_forward(n, w, b, activation="gelu", keep_preactivation=True)
        cache.write(at, y)
        q = y[:20].view(20, 1, 64)
        out, lse = memory.attend(q, ids, cache, cache)
        dq, _ = memory.attend_backward(out, q, ids, cache, cache, lse)
        dn, dw, db = memory.linear_backward(dy, n, w, z, activation="gelu")
        return (out, lse, dq, dw, db, cache.read(at)) + memory.layer_norm_backward(dn, x, None, mean, rstd)

    want = work(cache)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = work(cache2)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = work(cache2)
    cache2.codes.zero_()
    for t in again:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, again))


# ------------------------------------------------------------------ refusals
def refused(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_refusals():
    x, w = rand(1, 4, 32, kind=BF16), rand(2, 8, 32, kind=BF16)
    refused(lambda: memory.layer_norm(x.double()), "float32, bfloat16 or float16")
    refused(lambda: memory.layer_norm(x.t()), "last dimension must be contiguous")
    refused(lambda: memory.layer_norm(x, rand(1, 31)), "vector of 32")
    refused(lambda: memory.layer_norm(x, rand(1, 32, kind=F16)), "float32 or of x's type")
    refused(lambda: memory.layer_norm(x, torch.ones(32)), "is on cpu")
    refused(lambda: memory.layer_norm(x[:, :0]), "at least 1")
    refused(lambda: memory.layer_norm(x.view(2, 2, 32).transpose(0, 1)), "rows of one stride")
    refused(lambda: memory.linear(x.float(), w.float()), "bfloat16 or float16")
    refused(lambda: memory.linear(x, w.half()), "x's type")
    refused(lambda: memory.linear(x, w[:, :31]), "31 columns")
    refused(lambda: memory.linear(x, w, activation="tanh"), "activation")
    refused(lambda: memory.linear(x, w, residual=x), "y's shape")
    refused(lambda: memory.linear(x, w, rand(3, 8)), "bias must have x's type")
    refused(lambda: memory.linear_backward(x[:, :8], x, w, activation="gelu"), "z must be")
    refused(lambda: memory.RowCache.empty(4, 32, group=24), "multiple of 16")
    refused(lambda: memory.RowCache.empty(4, 32, code="int4"), "int8 or uint8")
    refused(lambda: memory.RowCache(torch.zeros(4, 32, dtype=torch.int8, device="cuda")), "scales")
    refused(lambda: memory.RowCache.empty(4, 32, code="uint8", step=0.0), "step")
    cache = memory.RowCache.empty(4, 32)
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    refused(lambda: cache.write(ids, x[:3]), "rows must be 4 x 32")
    refused(lambda: cache.write(ids.float(), x), "int32 or int64")
    refused(lambda: cache.read(ids, dtype=torch.int8), "dtype")
    q = rand(4, 4, 2, 32)
    refused(lambda: memory.attend(q, ids, cache, cache), "ids must be int32")
    refused(lambda: memory.attend(q[..., :20], ids[:, None], cache, cache), "multiple of 8")
    refused(lambda: memory.attend(q[..., :24], ids[:, None], cache, cache), "do not hold heads")
    refused(lambda: memory.attend(q, ids[:, None], cache, memory.RowCache.empty(5, 32)), "one shape")
    refused(lambda: memory.attend(q, ids[:, None], cache, cache, cap=-1.0), "cap")
    refused(lambda: memory.attend(q, ids[:, None], cache, cache, row_docs=ids), "go together")
    refused(lambda: memory.attend(q, ids[:, None], cache, cache, bias=q[:, 0, :1].double()), "bias must be")


def test_attend_lowest_value_everywhere_weighs_alike():
    """A list whose every bias is the type's lowest value is not empty: its entries weigh alike."""
    head, slots, found = 64, 40, 12
    keys, values = filled(slots, head, 0, "int8", 1), filled(slots, head, 0, "int8", 2)
    q, dout = rand(3, 2, 3, head), rand(4, 2, 3, head)
    ids = lists(11, 2, found, slots).clamp(min=0)
    bias = torch.full((2, found), torch.finfo(F32).min, device="cuda")
    out, lse = memory.attend(q, ids, keys, values, bias=bias)
    dq, dbias = memory.attend_backward(dout, q, ids, keys, values, lse, bias=bias)
    k, v = held(keys, head)[:, 0][ids.cpu().long()], held(values, head)[:, 0][ids.cpu().long()]
    mean = v.mean(1)[:, None].expand(2, 3, head)
    assert_close(out, mean, 64 * plain.U32 * v.abs().mean(1)[:, None].expand(2, 3, head), "out")
    dp = torch.einsum("qhd,qkd->qhk", d64(dout), v)
    ds = (dp - dp.mean(2, keepdim=True)) / found
    room = 256 * plain.U32 * torch.einsum("qhd,qkd->qhk", d64(dout).abs(), v.abs()).amax(2, keepdim=True)
    want = head ** -0.5 * torch.einsum("qhk,qkd->qhd", ds, k)
    assert_close(dq, want, room * head ** -0.5 * k.abs().mean(1)[:, None], "dq")
    assert_close(dbias, ds.sum(1), (room / found).sum(1).expand(2, found), "dbias")


def test_example_runs_them_together():
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "memory.py")
    spec = importlib.util.spec_from_file_location("memory_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, hit = example.run(stored=3_000, queries=32, steps=6)
    assert hit == 1.0                     # the asked state is nearest by far (noise 0.1 of its size)
    assert all(math.isfinite(x) for x in losses) and losses[-1] < losses[0]


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("width", [1, 2, 3, 31, 255, 301, 769, 1030, 2047])
def test_layer_norm_rows_that_start_inside_words(kind, width):
    """Contiguous 16-bit rows of odd and even widths, more of them than a launch has warps; the arrays around the
    outputs stay as they are."""
    rows = 5001
    check_norm(rand(1, rows, width, kind=kind), rand(2, width, scale=0.2, shift=1.0), rand(3, width), 1e-5,
               rand(4, rows, width, kind=kind))


@pytest.mark.parametrize("kind", [BF16, F16])
def test_layer_norm_mixed_strides(kind):
    """Rows of odd and even strides together, and bases off a word."""
    x, dy = rand(1, 33, 102, kind=kind)[:, :101], rand(2, 33, 101, kind=kind)
    check_norm(x, None, None, 1e-5, dy)
    check_norm(dy, rand(3, 101, kind=kind), None, 1e-5, x.contiguous())
    check_norm(rand(4, 33, 102, kind=kind)[:, 1:], None, None, 1e-5, rand(5, 33, 104, kind=kind)[:, 2:103])
