"""Operators around the search, what needs no GPU: the C ABI's refusals, and
the 64-bit forms that the GPU tests compare with (gradients against
differences, codes against their definition)."""
import ctypes
import math

import pytest
import torch

import memory_plain as plain
from helpers import capi
from winnex_madhava import memory

P = ctypes.c_void_p
SOME = P(4096)  # an address that is checked and never read
INVALID, CUDA, UNSUPPORTED = 1, 2, 7


class Rows(ctypes.Structure):
    _fields_ = [("codes", P), ("scales", P), ("slots", ctypes.c_int64), ("stride", ctypes.c_int64),
                ("width", ctypes.c_int32), ("group", ctypes.c_int32), ("code", ctypes.c_int32), ("lo", ctypes.c_double),
                ("step", ctypes.c_double)]


class Attend(ctypes.Structure):
    _fields_ = [("q", P), ("ids", P), ("bias", P), ("query_docs", P), ("row_docs", P), ("q_stride", ctypes.c_int64),
                ("q_head_stride", ctypes.c_int64), ("ids_stride", ctypes.c_int64), ("bias_stride", ctypes.c_int64),
                ("queries", ctypes.c_int64), ("found", ctypes.c_int32), ("heads", ctypes.c_int32),
                ("shared", ctypes.c_int32), ("head", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("scale", ctypes.c_float), ("cap", ctypes.c_float)]


@pytest.fixture(scope="module")
def lib():
    L = capi()
    i32, i64, f = ctypes.c_int32, ctypes.c_int64, ctypes.c_float
    L.mdh_layer_norm_forward.argtypes = [P, i64, i32, P, P, i32, i64, i32, f, P, i64, P, P, P]
    L.mdh_layer_norm_backward.argtypes = [P, i64, P, i64, i32, P, i32, P, P, i64, i32, P, i64, P, P, P, i64, P]
    L.mdh_linear_forward.argtypes = [P, i64, P, i64, P, P, i64, i32, i32, i64, i32, i32, P, i64, P, P, i64, P]
    L.mdh_linear_backward.argtypes = [P, i64, P, i64, P, i64, P, i32, i32, i64, i32, i32, P, P, P, P, i64, P]
    L.mdh_rows_write.argtypes = [P, P, i32, P, i64, i32, i64, P]
    L.mdh_rows_read.argtypes = [P, P, i32, i64, P, i64, i32, P]
    L.mdh_attend.argtypes = [P, P, P, P, P, P, i64, P]
    L.mdh_attend_backward.argtypes = [P, P, P, P, P, P, P, P, i64, P]
    return L


def norm(L, x=SOME, xs=8, dtype=0, w_dtype=0, rows=4, width=8, eps=1e-5):
    return L.mdh_layer_norm_forward(x, xs, dtype, None, None, w_dtype, rows, width, eps, SOME, max(width, 1), None, None,
                                    None)


def test_layer_norm_refusals(lib):
    assert norm(lib, dtype=3) == INVALID and b"dtype" in lib.mdh_last_error()
    assert norm(lib, dtype=1, w_dtype=2) == INVALID and b"weights" in lib.mdh_last_error()
    assert norm(lib, rows=-1) == INVALID
    assert norm(lib, width=0) == INVALID
    assert norm(lib, width=16385, xs=16385) == UNSUPPORTED
    assert norm(lib, x=None) == INVALID
    assert norm(lib, xs=7) == INVALID and b"stride" in lib.mdh_last_error()
    assert norm(lib, eps=-1.0) == INVALID and norm(lib, eps=math.nan) == INVALID
    assert lib.mdh_layer_norm_backward(None, 8, SOME, 8, 0, None, 0, SOME, SOME, 4, 8, SOME, 8, None, None, None, 0,
                                       None) == INVALID


def linear(L, x=SOME, xs=8, w=SOME, ws=8, dtype=1, act=0, rows=4, inner=8, outer=8, ys=8):
    return L.mdh_linear_forward(x, xs, w, ws, None, None, 0, dtype, act, rows, inner, outer, SOME, ys, None, None, 0,
                                None)


def test_linear_refusals(lib):
    assert linear(lib, dtype=0) == INVALID and b"bfloat16" in lib.mdh_last_error()
    assert linear(lib, act=4) == INVALID and linear(lib, act=-1) == INVALID
    assert linear(lib, rows=-1) == INVALID and linear(lib, inner=0) == INVALID and linear(lib, outer=0) == INVALID
    assert linear(lib, rows=2 ** 31) == UNSUPPORTED
    assert linear(lib, x=None) == INVALID and linear(lib, w=None) == INVALID
    assert linear(lib, xs=7) == INVALID and linear(lib, ws=7) == INVALID and linear(lib, ys=7) == INVALID
    # The slope of an activation needs z.
    assert lib.mdh_linear_backward(SOME, 8, SOME, 8, SOME, 8, None, 1, 2, 4, 8, 8, SOME, SOME, SOME, SOME, 1 << 20,
                                   None) == INVALID


def rows(**k):
    return Rows(**{**dict(codes=4096, scales=4096, slots=10, stride=64, width=64, group=32, code=0, lo=0.0, step=1.0), **k})


def test_row_cache_refusals(lib):
    def write(c, bits=32, dtype=0, n=4, stride=64):
        return lib.mdh_rows_write(ctypes.byref(c), SOME, bits, SOME, stride, dtype, n, None)

    for bad in (dict(slots=-1), dict(slots=2 ** 31), dict(width=0), dict(stride=63), dict(code=2), dict(codes=None),
                dict(scales=None), dict(group=8), dict(group=-16), dict(code=1, step=0.0), dict(code=1, step=math.nan),
                dict(code=1, lo=math.inf), dict(code=1, step=1e-45)):
        assert write(rows(**bad)) == INVALID, bad
    assert write(rows(width=65537, stride=70000)) == UNSUPPORTED
    assert write(rows(), bits=16) == INVALID and write(rows(), dtype=5) == INVALID
    assert write(rows(), n=-1) == INVALID and write(rows(), stride=63) == INVALID
    assert lib.mdh_rows_write(None, SOME, 32, SOME, 64, 0, 4, None) == INVALID
    assert lib.mdh_rows_read(ctypes.byref(rows()), SOME, 32, 4, SOME, 63, 0, None) == INVALID


def attend(L, keys=None, values=None, **k):
    a = Attend(**{**dict(q=4096, ids=4096, q_stride=64, q_head_stride=32, ids_stride=5, queries=3, found=5, heads=4,
                         shared=2, head=32, dtype=0, scale=0.1, cap=0.0), **k})
    keys, values = keys or rows(), values or rows()
    return L.mdh_attend(ctypes.byref(a), ctypes.byref(keys), ctypes.byref(values), SOME, SOME, None, 0, None)


def test_attend_refusals(lib):
    for bad in (dict(dtype=3), dict(queries=-1), dict(found=-1), dict(heads=0), dict(shared=0), dict(shared=3),
                dict(ids_stride=4), dict(query_docs=4096), dict(row_docs=4096), dict(scale=math.nan),
                dict(cap=-1.0), dict(cap=math.inf), dict(q=None), dict(ids=None), dict(bias=4096, bias_stride=4),
                dict(heads=2, shared=2)):
        assert attend(lib, **bad) == INVALID, bad
    for head in (12, 264, 0, -8):
        assert attend(lib, head=head) == UNSUPPORTED
    assert attend(lib, values=rows(slots=11)) == INVALID
    assert attend(lib, values=rows(width=32)) == INVALID


def test_workspaces_need_no_gpu_and_take_any_sizes(lib):
    for name, kinds in (("mdh_attend_workspace", [P]), ("mdh_attend_backward_workspace", [P, ctypes.c_int32]),
                        ("mdh_layer_norm_backward_workspace", [ctypes.c_int64, ctypes.c_int32])):
        getattr(lib, name).argtypes, getattr(lib, name).restype = kinds, ctypes.c_int64
    some = dict(queries=3, found=5000, heads=4, shared=2, head=32, dtype=0)
    a = Attend(**some)
    assert lib.mdh_attend_workspace(ctypes.byref(a)) > 0                 # a long list of few queries is cut
    assert lib.mdh_attend_backward_workspace(ctypes.byref(a), 1) >= 3 * 4 * 5000 * 8
    for bad in (dict(heads=0), dict(shared=0), dict(shared=3), dict(head=0), dict(head=2 ** 31 - 1), dict(queries=-1),
                dict(found=-1)):
        a = Attend(**{**some, **bad})
        assert lib.mdh_attend_workspace(ctypes.byref(a)) == 0 and lib.mdh_attend_backward_workspace(ctypes.byref(a), 1) == 0
    assert lib.mdh_attend_workspace(None) == 0
    assert lib.mdh_layer_norm_backward_workspace(0, 768) == 0 and lib.mdh_layer_norm_backward_workspace(10, 0) == 0


def test_no_gpu_no_operator(lib):
    if lib.mdh_device_count() > 0:
        pytest.skip("a GPU is present")
    assert norm(lib) == CUDA and linear(lib) == CUDA and attend(lib) == CUDA
    assert lib.mdh_rows_read(ctypes.byref(rows()), SOME, 32, 4, SOME, 64, 0, None) == CUDA
    assert b"no CUDA device" in lib.mdh_last_error()


def test_python_refuses_cpu_tensors():
    x = torch.zeros(4, 16)
    for call in (lambda: memory.layer_norm(x), lambda: memory.linear(x.bfloat16(), x.bfloat16()),
                 lambda: memory.RowCache(torch.zeros(4, 16, dtype=torch.uint8)),
                 lambda: memory.attend(torch.zeros(1, 1, 16), torch.zeros(1, 1, dtype=torch.int32), None, None)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


# ------------------------------------------------------------------ the 64-bit forms
def rand(g, *shape):
    return torch.randn(shape, generator=g, dtype=torch.float64)


def slope(f, x, along, h=1e-6):
    return (f(x + h * along) - f(x - h * along)) / (2 * h)


def test_layer_norm_gradients_are_the_slopes():
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = rand(g, 4, 9), rand(g, 9), rand(g, 9), rand(g, 4, 9)
    grads = plain.norm_grads(dy, x, w, 1e-5)
    forms = (lambda v: (plain.norm(v, w, b, 1e-5)[0] * dy).sum(), lambda v: (plain.norm(x, v, b, 1e-5)[0] * dy).sum(),
             lambda v: (plain.norm(x, w, v, 1e-5)[0] * dy).sum())
    for f, t, (grad, _) in zip(forms, (x, w, b), grads):
        along = rand(g, *t.shape)
        assert abs(slope(f, t, along) - (grad * along).sum()) < 1e-6


def test_attend_gradients_are_the_slopes():
    g = torch.Generator().manual_seed(1)
    q, k, v, bias, dout = rand(g, 3, 4, 8), rand(g, 20, 2, 8), rand(g, 20, 2, 8), rand(g, 3, 6), rand(g, 3, 4, 8)
    ids = torch.randint(-1, 20, (3, 6), generator=g, dtype=torch.int32)
    ids[1] = -1
    r = plain.attend(q, ids, k, v, 0.3, 2.0, bias, dout=dout)
    for f, t, name in ((lambda x: (plain.attend(x, ids, k, v, 0.3, 2.0, bias)["out"][0] * dout).sum(), q, "dq"),
                       (lambda x: (plain.attend(q, ids, k, v, 0.3, 2.0, x)["out"][0] * dout).sum(), bias, "dbias")):
        along = rand(g, *t.shape)
        assert abs(slope(f, t, along) - (r[name][0] * along).sum()) < 1e-6
    assert not r["out"][0][1].any() and torch.isneginf(r["lse"][0][1]).all() and not r["dq"][0][1].any()


def test_codes_stay_within_half_a_step():
    g = torch.Generator().manual_seed(2)
    x = torch.randn((30, 50), generator=g) * torch.logspace(-20, 20, 30)[:, None]
    codes, scales = plain.quantise(x, 16)
    back = plain.stands_for(codes, scales, 16, 0.0, 1.0)
    step = scales.repeat_interleave(16, 1)[:, :50]
    assert ((back - x).abs() <= step * 0.5001).all() and codes.abs().max() == 127
    u = plain.quantise_affine(x[15:16], -1.0, 0.01)
    inside = (x[15:16] > -1) & (x[15:16] < 1.5)
    assert ((plain.stands_for(u, None, 0, -1.0, 0.01) - x[15:16]).abs()[inside] <= 0.00501).all()
