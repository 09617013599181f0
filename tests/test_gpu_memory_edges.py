"""Edges of the operators around the search on the GPU: strides that only the C ABI takes, values at the ends of a type's
range, gradients through every output, and what a failed call leaves behind."""
import ctypes
import math

import pytest
import torch

import memory_plain as plain
from helpers import capi
from memory_plain import assert_close, d64

pytestmark = pytest.mark.gpu

memory = pytest.importorskip("winnex_madhava.memory")

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
P, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


def rand(seed, *shape, kind=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(kind).cuda()


def address(t):
    return P(0 if t is None else t.data_ptr())


# ------------------------------------------------------------------ layer norm at strides of the caller's choice
def with_gap(rows, width, gap, kind, seed=None):
    """[rows][width + gap] whose gap, and whole where there is no seed, holds 7."""
    t = torch.full((rows, width + gap), 7.0, dtype=kind, device="cuda")
    if seed is not None:
        t[:, :width] = rand(seed, rows, width, kind=kind, scale=1.5, shift=0.3)
    return t


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("rows,width", [(5, 256), (3001, 256), (5, 512), (700, 768), (9, 1024), (7, 1536), (6, 2048),
                                        (3, 8192), (3, 16384), (5, 767), (5, 2047)])
def test_layer_norm_every_stride_odd(kind, rows, width):
    """16-bit rows, inputs and outputs all an odd number of elements apart: every element is read, summed and written,
    the gaps between rows stay as they are."""
    L = capi()
    L.mdh_layer_norm_forward.argtypes = [P, i64, i32, P, P, i32, i64, i32, ctypes.c_float, P, i64, P, P, P]
    L.mdh_layer_norm_backward_workspace.argtypes, L.mdh_layer_norm_backward_workspace.restype = [i64, i32], i64
    L.mdh_layer_norm_backward.argtypes = [P, i64, P, i64, i32, P, i32, P, P, i64, i32, P, i64, P, P, P, i64, P]
    code, gap, eps = 1 if kind == BF16 else 2, 1 + width % 2, 1e-5
    x, dy = with_gap(rows, width, gap, kind, 1), with_gap(rows, width, gap + 2, kind, 2)
    x[:, width:], dy[:, width:] = math.nan, math.nan          # what lies between rows takes no part
    w, b = rand(3, width, scale=0.2, shift=1.0), rand(4, width)
    y, dx = with_gap(rows, width, gap + 4, kind), with_gap(rows, width, gap, kind)
    mean, rstd = torch.full((rows,), math.nan, device="cuda"), torch.full((rows,), math.nan, device="cuda")
    stream = P(torch.cuda.current_stream().cuda_stream)
    assert L.mdh_layer_norm_forward(address(x), x.stride(0), code, address(w), address(b), 0, rows, width, eps, address(y),
                                    y.stride(0), address(mean), address(rstd), stream) == 0, L.mdh_last_error()
    x64, w64, dy64 = d64(x[:, :width]), d64(w), d64(dy[:, :width])
    want, off, m, r, _, _ = plain.norm(x64, w64, d64(b), eps)
    assert_close(y[:, :width], want, off, "y")
    n = (width + 8) * plain.U32
    assert_close(mean, m[:, 0], n * x64.abs().mean(1), "mean")
    assert_close(rstd, r[:, 0], r[:, 0] * (n + n * x64.abs().mean(1) * r[:, 0]), "rstd")
    assert (y[:, width:] == 7).all()

    size = L.mdh_layer_norm_backward_workspace(rows, width)
    grads = plain.norm_grads(dy64, x64, w64, eps)
    for out in (dx, None):                                    # with the rows' gradient, and the weights' alone
        ws = torch.full((size // 4,), math.nan, device="cuda")
        dw, db = torch.full((width,), math.nan, device="cuda"), torch.full((width,), math.nan, device="cuda")
        assert L.mdh_layer_norm_backward(address(dy), dy.stride(0), address(x), x.stride(0), code, address(w), 0,
                                         address(mean), address(rstd), rows, width, address(out), dx.stride(0),
                                         address(dw), address(db), address(ws), size, stream) == 0, L.mdh_last_error()
        assert_close(dw, *grads[1], "dw")
        assert_close(db, *grads[2], "db")
    assert_close(dx[:, :width], *grads[0], "dx")
    assert (dx[:, width:] == 7).all()


# ------------------------------------------------------------------ linear at the ends of its range
@pytest.mark.parametrize("name", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("rows", [1, 40])
def test_linear_gradients_where_z_leaves_float16(name, rows):
    """z of -90,000 and 90,000 are infinite in float16; the slopes there are 0 and 1."""
    x = torch.full((rows, 1), 300.0, dtype=F16, device="cuda")
    w = torch.tensor([[-300.0], [300.0], [0.25]], dtype=F16, device="cuda")
    y, z = memory.linear_forward(x, w, activation=name, keep_preactivation=True)
    assert torch.isneginf(z[:, 0]).all() and torch.isposinf(z[:, 1]).all()
    assert not y[:, 0].any() and torch.isposinf(y[:, 1]).all()
    dy = torch.tensor([[0.5, 0.25, 1.0]], dtype=F16, device="cuda").expand(rows, 3).contiguous()
    dx, dw, db = memory.linear_backward(dy, x, w, z, activation=name)
    dz = torch.tensor([0.0, 0.25, 1.0], device="cuda")        # 75 is past where either slope differs from 1
    assert torch.equal(dx.float(), torch.full((rows, 1), 0.25 * 300 + 0.25, device="cuda"))
    assert torch.equal(dw.float()[:, 0], 300.0 * rows * dz)
    assert torch.equal(db.float(), rows * dz)


def gelu_tail(kind, n):
    """n values of z in [-12, -1], and there in 64 bits: z, z Phi(z), Phi(z) + z phi(z) and the relative error that
    float32 arithmetic may add to a term.  e^(-z^2 / 2) has that of its argument, a few roundings of z^2 / 2; the rest is
    held to 2^-18."""
    z = torch.linspace(-12, -1, n, dtype=torch.float64).to(kind)
    z64 = z.double()
    cdf = torch.special.erfc(-z64 / math.sqrt(2)) / 2
    density = torch.exp(-z64 * z64 / 2) / math.sqrt(2 * math.pi)
    rel = 2.0 ** -18 + 3 * z64 * z64 * plain.U32
    return z.cuda(), (z64 * cdf, rel * (z64 * cdf).abs()), (cdf + z64 * density, rel * (cdf + (z64 * density).abs()))


@pytest.mark.parametrize("kind", [BF16, F16])
def test_gelu_tail_by_relative_error(kind):
    n = 4096
    z, (want, off), (slope, slope_off) = gelu_tail(kind, n)
    one = torch.ones(1, 1, dtype=kind, device="cuda")
    # The tiles, and the gradient: dx is dz, rounded once to the type (the product's one term is exact).
    y, kept = memory.linear_forward(z[:, None], one, activation="gelu", keep_preactivation=True)
    assert torch.equal(kept[:, 0], z)
    assert_close(y[:, 0], want, off, "y")
    dx, dw, db = memory.linear_backward(torch.ones_like(y), z[:, None], one, kept, activation="gelu")
    assert_close(dx[:, 0], slope, slope_off, "dx")
    # A few rows, and a k that is split over blocks.
    y = memory.linear(one, z[:, None], activation="gelu")
    assert_close(y[0], want, off, "y of one row")
    x, w = (torch.zeros(rows, 4096, dtype=kind, device="cuda") for rows in (16, 256))
    x[:, 70], w[:, 70] = 1, z[::16]
    y = memory.linear(x, w, activation="gelu")
    assert_close(y, want[::16].expand(16, 256), off[::16].expand(16, 256), "y of split k")


def test_linear_expired_wait_is_reported_once():
    """A wait of an earlier product that gave up (its word set from the host) fails the next product, or the call that
    asks, once; forms without waits go on."""
    L = capi()
    x, w = rand(1, 40, 64, kind=BF16), rand(2, 24, 64, kind=BF16)
    want = memory.linear(x, w)
    memory.linear_status()
    for call in (lambda: memory.linear(x, w), lambda: memory.linear_backward(want, x, w), memory.linear_status,
                 lambda: memory.linear_status("cuda:0")):
        assert L.mdh_linear_set_expired() == 0, L.mdh_last_error()
        row = memory.linear(x[:1], w)                          # reads nothing that a wait guards
        with pytest.raises(RuntimeError, match="expired"):
            call()
        memory.linear_status()
        assert torch.equal(memory.linear(x, w), want) and row.shape == (1, 24)
    assert L.mdh_linear_status() == 0


# ------------------------------------------------------------------ attention
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


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("shared,head", [(1, 64), (4, 32), (8, 64), (2, 96), (4, 128)])
def test_attend_query_elements_of_any_size(kind, shared, head):
    """An element of a query counts by its own size, however large another one is: the keys are 0 where the large one is."""
    slots, found, nq = 60, 200, 3
    keys, values = filled(slots, 2 * head, 0, "int8", 1), filled(slots, 2 * head, 0, "int8", 2)
    keys.codes[:, [5, head + 5]] = 0
    q, dout = rand(3, nq, 2 * shared, head, kind=kind), rand(4, nq, 2 * shared, head, kind=kind)
    q[..., 5] = 30000.0 if kind == F16 else 2.0 ** 60
    q[0, ..., 6] = 2.0 ** -20                                  # and small ones stay
    ids = torch.randint(0, slots, (nq, found), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
    out, lse = memory.attend(q, ids, keys, values)
    want = plain.attend(d64(q), ids.cpu(), held(keys, head), held(values, head), head ** -0.5, 0.0)
    assert_close(out, *want["out"], "out")
    assert_close(lse, *want["lse"], "lse")


def slopes64(q, ids, keys, values, bias, cap, dout, dlse):
    """dq and dbias in 64 bits by differentiation of the 64-bit form."""
    head = q.shape[2]
    q64, b64 = d64(q).requires_grad_(), d64(bias).requires_grad_()
    r = plain.attend(q64, ids.cpu(), held(keys, head), held(values, head), head ** -0.5, cap, b64)
    loss = (r["lse"][0] * d64(dlse)).sum()
    if dout is not None:
        loss = loss + (r["out"][0] * d64(dout)).sum()
    return torch.autograd.grad(loss, (q64, b64))


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("nq,found,groups,shared,head", [(3, 20, 2, 3, 64), (2, 1500, 2, 4, 32), (40, 64, 3, 1, 40)])
@pytest.mark.parametrize("through_out", [True, False])
def test_attend_gradient_through_lse(kind, nq, found, groups, shared, head, through_out):
    """A loss of out and lse, and of lse alone."""
    slots, cap = 300, 3.0
    keys, values = (filled(slots, groups * head, 0, "int8", s) for s in (1, 2))
    q, bias = rand(3, nq, groups * shared, head, kind=kind), -torch.rand(nq, found, generator=torch.Generator().manual_seed(4)).cuda()
    ids = torch.randint(-3, slots, (nq, found), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
    dlse = rand(6, nq, groups * shared)
    dout = rand(7, nq, groups * shared, head, kind=kind) if through_out else None
    q.requires_grad_(), bias.requires_grad_()
    out, lse = memory.attend(q, ids, keys, values, cap=cap, bias=bias)
    loss = (lse * dlse).sum() + (0 if dout is None else (out.float() * dout.float()).sum())
    loss.backward()
    dq, dbias = slopes64(q, ids, keys, values, bias, cap, dout, dlse)
    # The bounds for dout alone, and dlse as what it is beside dP: a number of its own size for each entry.
    dp = dlse[..., None].expand(nq, groups * shared, head) / head
    room = plain.attend(d64(q), ids.cpu(), held(keys, head), held(values, head).abs() + 1, head ** -0.5, cap, d64(bias),
                        dout=(0 if dout is None else d64(dout).abs()) + d64(dp).abs())
    assert_close(q.grad, dq, 4 * room["dq"][1], "dq")
    assert_close(bias.grad, dbias, 4 * room["dbias"][1], "dbias")


def test_attend_joined_by_lse_trains_as_one():
    """Two parts of a list joined by their lse inside autograd give the gradients of the whole list, empty parts included."""
    head, slots, nq = 64, 80, 6
    keys, values = filled(slots, 2 * head, 64, "int8", 1), filled(slots, 2 * head, 64, "int8", 2)
    ids = torch.randint(0, slots, (nq, 24), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
    ids[1, :9] = -1
    ids[2, 9:] = -1
    dout = rand(4, nq, 2, head)
    grads = []
    for parts in ([ids], [ids[:, :9], ids[:, 9:]]):
        q = rand(3, nq, 2, head).requires_grad_()
        done = [memory.attend(q, part, keys, values) for part in parts]
        weight = torch.softmax(torch.stack([lse for _, lse in done]), 0)
        sum(w[..., None] * o for w, (o, _) in zip(weight, done)).backward(dout)
        grads.append(d64(q.grad))
    want = plain.attend(d64(rand(3, nq, 2, head)), ids.cpu(), held(keys, head), held(values, head), head ** -0.5, 0.0,
                        dout=d64(dout))["dq"]
    for g in grads:
        assert ((g - want[0]).abs() <= 8 * want[1] + plain.U32 * want[0].abs()).all()


def test_attend_lse_gradient_of_empty_lists():
    """No entry, no gradient, whatever comes back for an lse of -infinity."""
    keys, values = filled(10, 64, 64, "int8", 1), filled(10, 64, 64, "int8", 2)
    q, dout = rand(1, 3, 2, 32), rand(2, 3, 2, 32)
    ids = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    ids[2] = 5
    bias = torch.zeros(3, 4, device="cuda")
    _, lse = memory.attend(q, ids, keys, values, bias=bias)
    dlse = torch.tensor([[math.nan, math.inf], [-math.inf, 3.0], [0.5, 0.5]], device="cuda")
    dq, dbias = memory.attend_backward(dout, q, ids, keys, values, lse, bias=bias, dlse=dlse)
    assert not dq[:2].any() and not dbias[:2].any() and torch.isfinite(dq).all() and dq[2].any()


def test_attend_refuses_another_shape_of_dlse():
    keys = filled(10, 64, 64, "int8", 1)
    q, ids = rand(1, 3, 2, 32), torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    _, lse = memory.attend(q, ids, keys, keys)
    for bad in (lse[:2], lse.double(), lse.t().contiguous().t(), lse.cpu()):
        with pytest.raises(ValueError, match="dlse"):
            memory.attend_backward(q, q, ids, keys, keys, lse, dlse=bad)


# ------------------------------------------------------------------ gradients that nobody asked for
def spied(monkeypatch, name):
    """Records the arguments of a native call."""
    calls, real = [], getattr(memory._native, name)
    monkeypatch.setattr(memory._native, name, lambda *a: (calls.append(a), real(*a))[1])
    return calls


def test_layer_norm_forms_what_is_needed(monkeypatch):
    x, w, b = rand(1, 50, 96, kind=BF16), rand(2, 96), rand(3, 96)
    dy = rand(4, 50, 96, kind=BF16)
    y, mean, rstd = memory.layer_norm_forward(x, w, b)
    full = memory.layer_norm_backward(dy, x, w, mean, rstd)
    calls = spied(monkeypatch, "_layer_norm_backward")
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, True, True)):
        some = memory.layer_norm_backward(dy, x, w, mean, rstd, need=need)
        leaves = [t.clone().requires_grad_(n) for t, n in zip((x, w, b), need)]
        memory.layer_norm(*leaves).backward(dy)
        for n, s, f, leaf in zip(need, some, full, leaves):
            assert torch.equal(s, f) and torch.equal(leaf.grad, f) if n else s is None and leaf.grad is None
        for args in calls:
            assert [args[k] != 0 for k in (11, 13, 14)] == list(need)
            assert (args[15] != 0) == (need[1] or need[2])     # scratch only where sums are formed
        calls.clear()


def test_attend_forms_the_bias_gradient_where_it_is_needed(monkeypatch):
    keys, values = filled(50, 64, 64, "int8", 1), filled(50, 64, 64, "int8", 2)
    q, ids = rand(3, 4, 2, 32), torch.randint(0, 50, (4, 9), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
    bias, dout = rand(4, 4, 9), rand(6, 4, 2, 32)
    out, lse = memory.attend(q, ids, keys, values, bias=bias)
    dq, dbias = memory.attend_backward(dout, q, ids, keys, values, lse, bias=bias)
    calls = spied(monkeypatch, "_attend_backward")
    alone, none = memory.attend_backward(dout, q, ids, keys, values, lse, bias=bias, need=(True, False))
    assert torch.equal(alone, dq) and none is None
    none, alone = memory.attend_backward(dout, q, ids, keys, values, lse, bias=bias, need=(False, True))
    assert none is None and torch.equal(alone, dbias)
    q2 = q.clone().requires_grad_()
    memory.attend(q2, ids, keys, values, bias=bias)[0].backward(dout)
    assert torch.equal(q2.grad, dq)
    assert [[a[k] != 0 for k in (6, 7)] for a in calls] == [[True, False], [True, True], [True, False]]


# ------------------------------------------------------------------ a cache as a corpus
@pytest.mark.parametrize("width", [100, 128])
def test_codes_side_by_side_are_a_corpus(width):
    """The codes of a cache as the corpus of a device index, copied to rows side by side where the cache pads them; the
    ids found are those of the codes."""
    L = capi()
    n, asked, k = 5000, 40, 8
    cache = memory.RowCache.empty(n, width, code="uint8", lo=-3.0, step=6 / 255)
    cache.write(torch.arange(n, device="cuda"), rand(1, n, width))
    assert cache.codes.is_contiguous() == (width % 16 == 0)
    corpus = cache.codes.contiguous()
    queries = corpus[::n // asked][:asked].contiguous()
    torch.cuda.synchronize()
    index = P()
    assert L.mdh_index_create_u8_device(address(corpus), n, width, 1, 0, ctypes.byref(index)) == 0, L.mdh_last_error()
    ids, dist = (torch.full((asked, k), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    assert L.mdh_search_u8_device(index, address(queries), asked, k, address(ids), address(dist), None, None) == 0, L.mdh_last_error()
    assert L.mdh_index_destroy(index) == 0
    far = (queries.double()[:, None] - corpus.double()[None]).square().sum(2)
    want, at = torch.sort(far, dim=1, stable=True)             # ties go to the lowest id
    assert torch.equal(ids.long(), at[:, :k]) and torch.equal(dist.double(), want[:, :k])
    # By distance, the rows found are those that the cache reads back nearest.
    back = cache.read(ids)
    asked_back = cache.read(ids[:, :1].contiguous())
    assert (((back - asked_back).double().square().sum(2) - want[:, :k] * cache.step ** 2).abs() < 1e-3).all()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_codes_are_those_that_torch_makes_on_the_gpu(kind):
    """The definition's products (scale a (1 / 127), inverse 127 (1 / a)) are what torch's quotients compute on a GPU, so
    a program that quantises its rows itself gets the same codes and scales, bit for bit."""
    n, width, group = 20_000, 256, 64
    x = rand(1, n, width, kind=kind, scale=1.7)
    cache = memory.RowCache.empty(n, width, group=group)
    cache.write(torch.arange(n, device="cuda"), x)
    parts = x.float().view(n, -1, group)
    top = parts.abs().amax(2, keepdim=True)
    assert torch.equal(cache.scales, (top / 127)[..., 0])
    assert torch.equal(cache.codes, (parts * (127 / top)).round().to(torch.int8).view(n, width))


