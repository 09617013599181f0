"""Operators around the exact search, on CUDA tensors: what makes the rows
that an index holds, and what reads the rows that a search found.

* :func:`layer_norm` and :func:`linear` normalise a model's states and
  project them to rows; both have a backward pass (through autograd, or
  directly with the ``*_forward`` / ``*_backward`` functions).
* :class:`RowCache` stores rows in 8 bits as they are written and reads them
  back by id.  Its ``uint8`` codes are a corpus of the exact u8 search.
* :func:`attend` reads the lists of ids that a search returned: attention of
  each query over its found rows, with a cap on the scores, a bias for each
  entry (a weight on its distance, say) and a document mask.

All run on the tensors' device and on torch's current stream there, do not
wait, and can be captured in a CUDA graph after a first call.  There is no
CPU path.  Wrong shapes, types or devices raise ``ValueError``; a failing
call of the native library raises ``RuntimeError`` with its message.
No counterpart in the reference.
"""
from __future__ import annotations

import torch

from . import _native

__all__ = ["layer_norm", "layer_norm_forward", "layer_norm_backward", "linear", "linear_forward", "linear_backward",
           "RowCache", "attend", "attend_backward"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _require(ok, message):
    if not ok:
        raise ValueError(message)


def _dtype(t, name):
    code = _DTYPES.get(t.dtype)
    _require(code is not None, f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


def _on(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _rows(t, name):
    """``t`` as rows of its last dimension: a 2-D view (rows may be strided)."""
    _require(t.is_cuda, f"{name} must be a CUDA tensor")
    _require(t.dim() >= 1, f"{name} must have at least one dimension")
    if t.dim() != 2:
        try:
            t = t.view(-1, t.shape[-1]) if t.shape[-1] else t.view(0, 0)
        except RuntimeError:
            raise ValueError(f"{name}: its leading dimensions cannot be viewed as rows of one stride") from None
    _require(t.shape[1] <= 1 or t.stride(1) == 1, f"{name}: the last dimension must be contiguous")
    _require(t.shape[0] <= 1 or t.stride(0) >= t.shape[1], f"{name}: rows must not overlap")
    return t


def _vector(t, size, name):
    if t is not None:
        _require(t.dim() == 1 and t.shape[0] == size and t.is_contiguous(),
                 f"{name} must be a contiguous vector of {size}")
    return t


def _ptr(t):
    return 0 if t is None else t.data_ptr()


class _Call:
    """The device of a call, made current, and torch's stream there."""

    def __init__(self, device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)
        self.device = device

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _workspace(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


# ------------------------------------------------------------------ layer norm
def _norm_weights(x2, weight, bias):
    width = x2.shape[1]
    _vector(weight, width, "weight")
    _vector(bias, width, "bias")
    _on(x2.device, weight=weight, bias=bias)
    kinds = {t.dtype for t in (weight, bias) if t is not None}
    _require(len(kinds) <= 1, "weight and bias must have one type")
    kind = kinds.pop() if kinds else x2.dtype
    _require(kind in (torch.float32, x2.dtype), "weight and bias must be float32 or of x's type")
    return kind


def _norm_forward(x, weight, bias, eps, keep):
    x2 = _rows(x, "x")
    code = _dtype(x2, "x")
    rows, width = x2.shape
    _require(width >= 1, "x must have a last dimension of at least 1")
    kind = _norm_weights(x2, weight, bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if keep:
        mean, rstd = torch.empty((2, rows), dtype=torch.float32, device=x.device)
    with _Call(x.device) as stream:
        _native._layer_norm_forward(x2.data_ptr(), x2.stride(0), code, _ptr(weight), _ptr(bias), _DTYPES[kind], rows,
                                    width, eps, y.data_ptr(), width, _ptr(mean), _ptr(rstd), stream)
    return y, mean, rstd


def layer_norm_forward(x, weight=None, bias=None, *, eps=1e-5):
    """``(y, mean, rstd)``: :func:`layer_norm` with the row statistics
    (float32, one for each row) that :func:`layer_norm_backward` takes."""
    return _norm_forward(x, weight, bias, eps, True)


def layer_norm_backward(dy, x, weight, mean, rstd, *, weight_dtype=None):
    """``(dx, dweight, dbias)`` of :func:`layer_norm` from the gradient of y.

    dweight and dbias have the weight's type (``weight_dtype`` where there is
    no weight; default x's type)."""
    x2, dy2 = _rows(x, "x"), _rows(dy, "dy")
    code = _dtype(x2, "x")
    _require(dy.shape == x.shape and dy.dtype == x.dtype, "dy must have x's shape and type")
    rows, width = x2.shape
    _require(width >= 1, "x must have a last dimension of at least 1")
    kind = _norm_weights(x2, weight, None) if weight is not None else weight_dtype or x.dtype
    _require(kind in (torch.float32, x.dtype), "weight_dtype must be float32 or x's type")
    for name, t in (("mean", mean), ("rstd", rstd)):
        _vector(t, rows, name)
        _require(t is not None and t.dtype == torch.float32, f"{name} must be float32")
    _on(x.device, dy=dy, weight=weight, mean=mean, rstd=rstd)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw, db = torch.empty((2, width), dtype=kind, device=x.device)
    size = _native._layer_norm_backward_workspace(rows, width)
    ws = _workspace(size, x.device)
    with _Call(x.device) as stream:
        _native._layer_norm_backward(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), code, _ptr(weight),
                                     _DTYPES[kind], mean.data_ptr(), rstd.data_ptr(), rows, width, dx.data_ptr(),
                                     width, dw.data_ptr(), db.data_ptr(), _ptr(ws), size, stream)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.kind = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(dy.contiguous(), x, weight, mean, rstd, weight_dtype=ctx.kind)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def layer_norm(x, weight=None, bias=None, *, eps=1e-5):
    """Layer norm over the last dimension: ``(x - mean) * rstd * weight + bias``.

    x: float32, bfloat16 or float16, last dimension contiguous (up to 16384);
    weight and bias: float32 or x's type, or None.  Statistics are float32.
    Differentiable in x, weight and bias."""
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


# ------------------------------------------------------------------ linear
def _activation(name):
    code = _ACTIVATIONS.get(name)
    _require(code is not None, f"activation must be one of none, relu, gelu, silu, not {name!r}")
    return code


def _linear_operands(x, weight):
    x2 = _rows(x, "x")
    _require(x2.dtype in (torch.bfloat16, torch.float16), f"x must be bfloat16 or float16, not {x.dtype}")
    _require(weight.dim() == 2 and weight.dtype == x.dtype, "weight must be a matrix of x's type")
    w2 = _rows(weight, "weight")
    _require(w2.shape[1] == x2.shape[1], f"weight has {w2.shape[1]} columns, x rows of {x2.shape[1]}")
    _require(w2.shape[0] >= 1 and w2.shape[1] >= 1, "weight must not be empty")
    _on(x.device, weight=weight)
    return x2, w2


def linear_forward(x, weight, bias=None, *, activation=None, residual=None, keep_preactivation=False):
    """``(y, z)``: :func:`linear`, and with ``keep_preactivation`` the value
    before the activation, in x's type, that :func:`linear_backward` takes
    (None without an activation: its slope is 1)."""
    x2, w2 = _linear_operands(x, weight)
    act = _activation(activation)
    (rows, inner), outer = x2.shape, w2.shape[0]
    shape = x.shape[:-1] + (outer,)
    r2 = None
    if bias is not None:
        _vector(bias, outer, "bias")
        _require(bias.dtype == x.dtype, "bias must have x's type")
    if residual is not None:
        _require(residual.shape == shape and residual.dtype == x.dtype, "residual must have y's shape and x's type")
        r2 = _rows(residual, "residual")
    _on(x.device, bias=bias, residual=residual)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    z = torch.empty(shape, dtype=x.dtype, device=x.device) if keep_preactivation and act else None
    size = _native._linear_forward_workspace(x2.data_ptr(), x2.stride(0), w2.data_ptr(), w2.stride(0), rows, inner,
                                             outer)
    ws = _workspace(size, x.device)
    with _Call(x.device) as stream:
        _native._linear_forward(x2.data_ptr(), x2.stride(0), w2.data_ptr(), w2.stride(0), _ptr(bias), _ptr(r2),
                                0 if r2 is None else r2.stride(0), _DTYPES[x.dtype], act, rows, inner, outer,
                                y.data_ptr(), outer, _ptr(z), _ptr(ws), size, stream)
    return y, z


def linear_backward(dy, x, weight, z=None, *, activation=None, need=(True, True, True)):
    """``(dx, dweight, dbias)`` of :func:`linear` from the gradient of y.

    z: from :func:`linear_forward` (with an activation).  ``need`` says which
    of the three to form; the others are None.  The residual's gradient is dy."""
    x2, w2 = _linear_operands(x, weight)
    act = _activation(activation)
    (rows, inner), outer = x2.shape, w2.shape[0]
    shape = x.shape[:-1] + (outer,)
    _require(dy.shape == shape and dy.dtype == x.dtype, "dy must have y's shape and x's type")
    dy2 = _rows(dy, "dy")
    if act:
        _require(z is not None and z.shape == shape and z.dtype == x.dtype and z.is_contiguous(),
                 "z must be what linear_forward kept: y's shape, x's type, contiguous")
    _on(x.device, dy=dy, z=z)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
    dw = torch.empty((outer, inner), dtype=x.dtype, device=x.device) if need[1] else None
    db = torch.empty(outer, dtype=x.dtype, device=x.device) if need[2] else None
    size = _native._linear_backward_workspace(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0),
                                              w2.data_ptr(), w2.stride(0), act, rows, inner, outer)
    ws = _workspace(size, x.device)
    with _Call(x.device) as stream:
        _native._linear_backward(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), w2.data_ptr(),
                                 w2.stride(0), _ptr(z if act else None), _DTYPES[x.dtype], act, rows, inner, outer,
                                 _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), size, stream)
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, z = linear_forward(x, weight, bias, activation=activation, residual=residual, keep_preactivation=True)
        ctx.save_for_backward(x, weight, z)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        grads = linear_backward(dy.contiguous(), x, weight, z, activation=ctx.activation,
                                need=ctx.needs_input_grad[:3])
        return (*grads, dy if ctx.needs_input_grad[3] else None, None)


def linear(x, weight, bias=None, *, activation=None, residual=None):
    """``activation(x @ weight.T + bias) + residual`` in one kernel.

    x [..., inner] and weight [outer, inner]: bfloat16 or float16, products
    summed in float32; bias [outer], residual [..., outer]; activation None,
    "relu", "gelu" (z Phi(z)) or "silu".  Differentiable in all four."""
    if _wants_grad(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, activation)
    return linear_forward(x, weight, bias, activation=activation, residual=residual)[0]


# ------------------------------------------------------------------ rows in 8 bits
class RowCache:
    """Rows of one width in 8 bits, in the caller's tensors.

    codes [slots, width] int8 with scales [slots, groups] float32: ``group``
    elements (a multiple of 16, or 0 for the whole row) share a scale, a
    element stands for code * scale.  codes uint8: one affine map, an element
    stands for lo + step * code; these codes are a corpus of the exact u8
    search.  :meth:`empty` allocates with the row stride that reads fastest.
    """

    def __init__(self, codes, scales=None, *, group=0, lo=0.0, step=1.0):
        _require(codes.is_cuda and codes.dim() == 2 and codes.dtype in (torch.int8, torch.uint8),
                 "codes must be an int8 or uint8 CUDA matrix")
        slots, width = codes.shape
        _require(width >= 1 and (width == 1 or codes.stride(1) == 1) and (slots <= 1 or codes.stride(0) >= width),
                 "codes must be rows of contiguous elements that do not overlap")
        affine = codes.dtype == torch.uint8
        if affine:
            _require(scales is None, "uint8 codes have no scales")
            _require(step > 0, "step must be positive")
        else:
            _require(group >= 0 and group % 16 == 0, "group must be 0 or a multiple of 16")
            groups = 1 if group == 0 else -(-width // group)
            _require(scales is not None and scales.dtype == torch.float32 and scales.shape == (slots, groups) and
                     scales.is_contiguous(), f"scales must be a contiguous float32 matrix of {slots} x {groups}")
            _on(codes.device, scales=scales)
        self.codes, self.scales, self.group, self.lo, self.step = codes, scales, group, lo, step
        self.slots, self.width, self.device = slots, width, codes.device
        self._native = _native._Rows(codes.data_ptr(), _ptr(scales), slots, max(codes.stride(0), width), width,
                                     0 if affine else group, int(affine), lo, step)

    @classmethod
    def empty(cls, slots, width, *, code="int8", group=64, lo=0.0, step=1.0, device="cuda"):
        """A cache with every row zero codes (int8: zeros; uint8: lo)."""
        _require(code in ("int8", "uint8"), "code must be int8 or uint8")
        _require(slots >= 0 and width >= 1, "slots must be >= 0 and width >= 1")
        _require(group >= 0 and group % 16 == 0, "group must be 0 or a multiple of 16")
        kind = torch.int8 if code == "int8" else torch.uint8
        codes = torch.zeros((slots, -(-width // 16) * 16), dtype=kind, device=device)[:, :width]
        if code == "uint8":
            return cls(codes, lo=lo, step=step)
        groups = 1 if group == 0 else -(-width // group)
        return cls(codes, torch.zeros((slots, groups), device=device), group=group)

    def _ids(self, ids, name, dims=1):
        _require(ids.dtype in (torch.int32, torch.int64) and ids.is_contiguous() and (not dims or ids.dim() == dims),
                 f"{name} must be contiguous int32 or int64" + (" and one-dimensional" if dims else ""))
        _on(self.device, **{name: ids})
        return 32 if ids.dtype == torch.int32 else 64

    def write(self, slots, rows):
        """Quantises rows [n, width] (float32, bfloat16 or float16) into the
        given slots; a slot outside [0, slots) (-1, say) writes nothing.  The
        slots of one call that are inside must differ from one another."""
        bits = self._ids(slots, "slots")
        _require(rows.dim() == 2 and rows.shape == (slots.shape[0], self.width),
                 f"rows must be {slots.shape[0]} x {self.width}")
        r2 = _rows(rows, "rows")
        code = _dtype(r2, "rows")
        _on(self.device, rows=rows)
        with _Call(self.device) as stream:
            _native._rows_write(self._native, slots.data_ptr(), bits, r2.data_ptr(), r2.stride(0), code,
                                slots.shape[0], stream)

    def read(self, ids, dtype=torch.float32):
        """The rows of ids [...] as [..., width] of ``dtype``: what the codes
        stand for, zeros where an id is outside [0, slots)."""
        bits = self._ids(ids, "ids", 0)
        _require(dtype in _DTYPES, f"dtype must be float32, bfloat16 or float16, not {dtype}")
        out = torch.empty(ids.shape + (self.width,), dtype=dtype, device=self.device)
        with _Call(self.device) as stream:
            _native._rows_read(self._native, ids.data_ptr(), bits, ids.numel(), out.data_ptr(), self.width,
                               _DTYPES[dtype], stream)
        return out


# ------------------------------------------------------------------ attention over found rows
def _attend_args(q, ids, keys, values, scale, cap, bias, query_docs, row_docs):
    _require(q.is_cuda and q.dim() == 3, "q must be a CUDA tensor [queries, heads, head]")
    code = _dtype(q, "q")
    queries, heads, head = q.shape
    _require(heads >= 1 and head >= 8 and head % 8 == 0 and head <= 256,
             "q: the head size must be a multiple of 8 up to 256")
    _require(q.stride(2) == 1, "q: the last dimension must be contiguous")
    _require(keys.width == values.width and keys.slots == values.slots, "keys and values must have one shape")
    _require(keys.width % head == 0 and heads % (keys.width // head) == 0,
             f"cache rows of {keys.width} do not hold heads of {head} that {heads} query heads share")
    _require(ids.dim() == 2 and ids.shape[0] == queries and ids.dtype == torch.int32,
             "ids must be int32 [queries, found]")
    found = ids.shape[1]

    def lists(t):  # one list may serve every query (stride 0)
        return (found <= 1 or t.stride(1) == 1) and (queries <= 1 or t.stride(0) >= found or t.stride(0) == 0)

    _require(lists(ids), "ids must be rows of contiguous entries")
    if bias is not None:
        _require(bias.shape == ids.shape and bias.dtype == torch.float32 and lists(bias),
                 "bias must be float32 of ids' shape, its rows contiguous")
    _require((query_docs is None) == (row_docs is None), "query_docs and row_docs go together")
    if query_docs is not None:
        for name, t, n in (("query_docs", query_docs, queries), ("row_docs", row_docs, keys.slots)):
            _vector(t, n, name)
            _require(t.dtype == torch.int32, f"{name} must be int32")
    _on(q.device, ids=ids, bias=bias, query_docs=query_docs, row_docs=row_docs, keys=keys, values=values)
    _require(cap >= 0, "cap must be >= 0")
    return _native._AttendArgs(q.data_ptr(), ids.data_ptr(), _ptr(bias), _ptr(query_docs), _ptr(row_docs),
                               q.stride(0), q.stride(1), ids.stride(0), 0 if bias is None else bias.stride(0),
                               queries, found, heads,
                               heads * head // keys.width, head, code, head ** -0.5 if scale is None else scale, cap)


def _attend(q, ids, keys, values, scale, cap, bias, query_docs, row_docs):
    args = _attend_args(q, ids, keys, values, scale, cap, bias, query_docs, row_docs)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    size = _native._attend_workspace(args)
    ws = _workspace(size, q.device)
    with _Call(q.device) as stream:
        _native._attend(args, keys._native, values._native, out.data_ptr(), lse.data_ptr(), _ptr(ws), size, stream)
    return out, lse


def attend_backward(dout, q, ids, keys, values, lse, *, scale=None, cap=0.0, bias=None, query_docs=None,
                    row_docs=None):
    """``(dq, dbias)`` of :func:`attend` from the gradient of its output and
    its lse; dbias (float32, summed over the heads) is None without a bias.
    The caches are constants."""
    args = _attend_args(q, ids, keys, values, scale, cap, bias, query_docs, row_docs)
    _require(dout.shape == q.shape and dout.dtype == q.dtype and dout.is_contiguous(),
             "dout must be contiguous, of q's shape and type")
    _require(lse.shape == q.shape[:2] and lse.dtype == torch.float32 and lse.is_contiguous(),
             "lse must be what attend returned")
    _on(q.device, dout=dout, lse=lse)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dbias = None if bias is None else torch.empty(ids.shape, dtype=torch.float32, device=q.device)
    size = _native._attend_backward_workspace(args, dbias is not None)
    ws = _workspace(size, q.device)
    with _Call(q.device) as stream:
        _native._attend_backward(args, keys._native, values._native, dout.data_ptr(), lse.data_ptr(), dq.data_ptr(),
                                 _ptr(dbias), _ptr(ws), size, stream)
    return dq, dbias


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, bias, ids, keys, values, scale, cap, query_docs, row_docs):
        out, lse = _attend(q, ids, keys, values, scale, cap, bias, query_docs, row_docs)
        ctx.save_for_backward(q, bias, ids, lse, query_docs, row_docs)
        ctx.rest = (keys, values, scale, cap)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, bias, ids, lse, query_docs, row_docs = ctx.saved_tensors
        keys, values, scale, cap = ctx.rest
        dq, dbias = attend_backward(dout.contiguous(), q, ids, keys, values, lse, scale=scale, cap=cap, bias=bias,
                                    query_docs=query_docs, row_docs=row_docs)
        return (dq, dbias) + (None,) * 7


def attend(q, ids, keys, values, *, scale=None, cap=0.0, bias=None, query_docs=None, row_docs=None):
    """``(out, lse)``: attention of each query over its list of cached rows.

    q [queries, heads, head] (float32, bfloat16 or float16); ids [queries,
    found] int32, as a search returns them; keys and values: :class:`RowCache`
    whose rows hold heads of ``head`` elements that consecutive query heads
    share.  An entry scores ``scale * q . key`` (scale: head^-1/2), capped as
    ``cap * tanh(score / cap)`` where cap > 0, plus bias[query, entry].  It is
    hidden where its id is outside the cache, its bias is -infinity, or
    ``row_docs[id] != query_docs[query]``.  A query whose entries are all
    hidden gives zeros and an lse of -infinity.  lse [queries, heads] joins
    this attention with another over other rows.  ``out`` is differentiable
    in q and bias; lse and the caches are constants, and rows that a query
    read must not be rewritten before its backward pass."""
    if _wants_grad(q, bias):
        return _Attend.apply(q, bias, ids, keys, values, scale, cap, query_docs, row_docs)
    return _attend(q, ids, keys, values, scale, cap, bias, query_docs, row_docs)
