"""Edges of the operators around the search that need no GPU: sizes at the ends of a call's index arithmetic, and the
definitions of the row cache's codes beside one another."""
import ctypes
import importlib.util
import os

import pytest
import torch

import memory_plain as plain
from helpers import ROOT, capi

P, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
SOME = P(4096)  # an address that is checked and never read
UNSUPPORTED = 7


class Rows(ctypes.Structure):
    _fields_ = [("codes", P), ("scales", P), ("slots", i64), ("stride", i64), ("width", i32), ("group", i32), ("code", i32),
                ("lo", ctypes.c_double), ("step", ctypes.c_double)]


class Attend(ctypes.Structure):
    _fields_ = [("q", P), ("ids", P), ("bias", P), ("query_docs", P), ("row_docs", P), ("q_stride", i64),
                ("q_head_stride", i64), ("ids_stride", i64), ("bias_stride", i64), ("queries", i64), ("found", i32),
                ("heads", i32), ("shared", i32), ("head", i32), ("dtype", i32), ("scale", ctypes.c_float),
                ("cap", ctypes.c_float)]


@pytest.mark.parametrize("rows", [1, 40])
def test_linear_sizes_past_the_index_arithmetic(rows):
    """Column and k indices are 32 bits and run past the size by a tile: sizes near 2^31 are refused before a launch."""
    L = capi()
    L.mdh_linear_forward.argtypes = [P, i64, P, i64, P, P, i64, i32, i32, i64, i32, i32, P, i64, P, P, i64, P]
    L.mdh_linear_backward.argtypes = [P, i64, P, i64, P, i64, P, i32, i32, i64, i32, i32, P, P, P, P, i64, P]
    for inner, outer in ((2 ** 31 - 1, 8), (8, 2 ** 31 - 1), (2 ** 30 + 1, 8), (8, 2 ** 30 + 1)):
        assert L.mdh_linear_forward(SOME, inner, SOME, inner, None, None, 0, 1, 0, rows, inner, outer, SOME, outer, None, SOME,
                                    2 ** 62, None) == UNSUPPORTED, (inner, outer)
        assert L.mdh_linear_backward(SOME, outer, SOME, inner, SOME, inner, None, 1, 0, rows, inner, outer, SOME, SOME, SOME,
                                     SOME, 2 ** 62, None) == UNSUPPORTED, (inner, outer)
    # The slope pass has a block row for each 256 columns.
    outer = 65535 * 256 + 1
    assert L.mdh_linear_backward(SOME, outer, SOME, 8, SOME, 8, SOME, 1, 2, rows, 8, outer, SOME, SOME, SOME, SOME, 2 ** 62,
                                 None) == UNSUPPORTED


def test_attend_lists_past_the_index_arithmetic():
    L = capi()
    L.mdh_attend.argtypes = [P, P, P, P, P, P, i64, P]
    L.mdh_attend_backward.argtypes = [P, P, P, P, P, P, P, P, i64, P]
    cache = Rows(codes=4096, scales=4096, slots=10, stride=64, width=64, group=32, code=0, lo=0.0, step=1.0)
    for found in (2 ** 31 - 1, 2 ** 31 - 1024):
        a = Attend(q=4096, ids=4096, q_stride=64, q_head_stride=32, ids_stride=found, queries=1, found=found, heads=2,
                   shared=1, head=32, dtype=0, scale=0.1, cap=0.0)
        at = ctypes.byref(a), ctypes.byref(cache), ctypes.byref(cache)
        assert L.mdh_attend(*at, SOME, SOME, SOME, 2 ** 62, None) == UNSUPPORTED and b"found" in L.mdh_last_error()
        assert L.mdh_attend_backward(*at, SOME, SOME, SOME, None, SOME, 2 ** 62, None) == UNSUPPORTED


# ------------------------------------------------------------------ one definition of the codes
def test_codes_beside_the_plain_and_exact_forms_of_the_cases():
    """A row's codes and values by the definition (inverse 127 (1 / a) and scale a (1 / 127)) beside the forms that the
    measured cases carry, which divide: the same codes but where a value lies on a step's edge, scales within one unit."""
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    operators = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(operators)
    n, width, group = 400, 96, 32
    x = torch.randn((n, width), generator=torch.Generator().manual_seed(3)) * 1.7
    codes, scales = plain.quantise(x, group)
    want = plain.stands_for(codes, scales, group, 0.0, 1.0).double()
    ids = torch.arange(n, dtype=torch.int32)

    def case():
        return dict(slots=n, width=width, write=n, read=n, group=group, code="int8", type="f32", back="f32", rows=x, slot=ids,
                    ids=ids, codes=torch.zeros((n, width), dtype=torch.int8), scales=torch.zeros((n, 3)), lo=0.0, step=1.0)

    step = scales.double().repeat_interleave(group, 1)
    for form in (operators._rows_plain, operators._exact_rows):
        off = (form(case())["back"].double() - want).abs()
        moved = off > 0.5 * step
        assert moved.sum() <= 2                                 # about one code in a million
        assert (off[~moved] <= 2.0 ** -22 * want[~moved].abs()).all()   # a unit of the scale, a rounding of the value
