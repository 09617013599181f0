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
           "linear_status", "RowCache", "attend", "attend_backward"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _require(ok, message):
    if not ok:
        raise ValueError(message)


def _dtype(t, name):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


def _device(t, name):
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    return index


def _on(index, t, name):
    if t is not None and t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")


def _rows(t, name):
    """``(rows, width, stride, t)`` of ``t`` as rows of its last dimension
    (2-D rows may be strided); ``t`` is a view of the argument."""
    dims = t.dim()
    if dims == 2:
        rows, width = t.shape
        stride, inner = t.stride()
        if width > 1 and inner != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
        if rows > 1 and stride < width:
            raise ValueError(f"{name}: rows must not overlap")
        return rows, width, stride, t
    if dims == 0:
        raise ValueError(f"{name} must have at least one dimension")
    width = t.shape[-1]
    if t.is_contiguous():
        return t.numel() // width if width else 0, width, width, t
    try:
        return _rows(t.view(-1, width), name)
    except RuntimeError:
        raise ValueError(f"{name}: its leading dimensions cannot be viewed as rows of one stride") from None


def _vector(t, size, name):
    if t.dim() != 1 or t.shape[0] != size or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {size}")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


# The handle of torch's current stream on a device, without building a Stream.
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(index, fn, *args):
    """fn(*args, stream) with device ``index`` current and torch's stream there."""
    if index == torch.cuda.current_device():
        fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            fn(*args, _stream_of(index))


def _like(t):
    """A contiguous tensor of t's shape, type and device, not initialised."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(tuple(t.shape))


def _workspace(size, t):
    return t.new_empty((size,), dtype=torch.uint8) if size else None


# ------------------------------------------------------------------ layer norm
def _norm_weights(index, width, kind, weight, bias):
    """The type of the weights."""
    of = kind
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _vector(t, width, name)
            _on(index, t, name)
            of = t.dtype
            if of != kind and of != torch.float32:
                raise ValueError("weight and bias must be float32 or of x's type")
    if weight is not None and weight.dtype != of:
        raise ValueError("weight and bias must have one type")
    return of


def _norm_forward(x, weight, bias, eps, keep):
    index = _device(x, "x")
    code = _dtype(x, "x")
    rows, width, stride, x2 = _rows(x, "x")
    if width < 1:
        raise ValueError("x must have a last dimension of at least 1")
    kind = _norm_weights(index, width, x.dtype, weight, bias)
    y = _like(x)
    mean = rstd = None
    if keep:
        mean = x.new_empty((rows,), dtype=torch.float32)
        rstd = torch.empty_like(mean)
    _call(index, _native._layer_norm_forward, x2.data_ptr(), stride, code, _ptr(weight), _ptr(bias), _DTYPES[kind],
          rows, width, eps, y.data_ptr(), width, _ptr(mean), _ptr(rstd))
    return y, mean, rstd


def layer_norm_forward(x, weight=None, bias=None, *, eps=1e-5):
    """``(y, mean, rstd)``: :func:`layer_norm` with the row statistics
    (float32, one for each row) that :func:`layer_norm_backward` takes."""
    return _norm_forward(x, weight, bias, eps, True)


def layer_norm_backward(dy, x, weight, mean, rstd, *, weight_dtype=None, need=(True, True, True)):
    """``(dx, dweight, dbias)`` of :func:`layer_norm` from the gradient of y.

    dweight and dbias have the weight's type (``weight_dtype`` where there is
    no weight; default x's type).  ``need`` says which of the three to form;
    the others are None."""
    index = _device(x, "x")
    code = _dtype(x, "x")
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("dy must have x's shape and type")
    rows, width, stride, x2 = _rows(x, "x")
    _, _, dy_stride, dy2 = _rows(dy, "dy")
    if width < 1:
        raise ValueError("x must have a last dimension of at least 1")
    if weight is not None:
        kind = _norm_weights(index, width, x.dtype, weight, None)
    else:
        kind = weight_dtype or x.dtype
        _require(kind in (torch.float32, x.dtype), "weight_dtype must be float32 or x's type")
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        _vector(t, rows, name)
        _require(t.dtype == torch.float32, f"{name} must be float32")
        _on(index, t, name)
    _on(index, dy, "dy")
    dx = _like(x) if need[0] else None
    dw = x.new_empty((width,), dtype=kind) if need[1] else None
    db = x.new_empty((width,), dtype=kind) if need[2] else None
    size = _native._layer_norm_backward_workspace(rows, width) if need[1] or need[2] else 0
    ws = _workspace(size, x)
    _call(index, _native._layer_norm_backward, dy2.data_ptr(), dy_stride, x2.data_ptr(), stride, code, _ptr(weight),
          _DTYPES[kind], mean.data_ptr(), rstd.data_ptr(), rows, width, _ptr(dx), width, _ptr(dw),
          _ptr(db), _ptr(ws), size)
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
        return (*layer_norm_backward(dy.contiguous(), x, weight, mean, rstd, weight_dtype=ctx.kind,
                                     need=ctx.needs_input_grad[:3]), None)


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


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
    """(device, x's rows, weight's rows) as :func:`_rows` gives them."""
    index = _device(x, "x")
    kind = x.dtype
    if kind != torch.bfloat16 and kind != torch.float16:
        raise ValueError(f"x must be bfloat16 or float16, not {kind}")
    if weight.dim() != 2 or weight.dtype != kind:
        raise ValueError("weight must be a matrix of x's type")
    xr, wr = _rows(x, "x"), _rows(weight, "weight")
    if wr[1] != xr[1]:
        raise ValueError(f"weight has {wr[1]} columns, x rows of {xr[1]}")
    if wr[0] < 1 or wr[1] < 1:
        raise ValueError("weight must not be empty")
    _on(index, weight, "weight")
    return index, xr, wr


def linear_forward(x, weight, bias=None, *, activation=None, residual=None, keep_preactivation=False):
    """``(y, z)``: :func:`linear`, and with ``keep_preactivation`` the value
    before the activation, in x's type, that :func:`linear_backward` takes
    (None without an activation: its slope is 1)."""
    index, (rows, inner, xs, x2), (outer, _, ws, w2) = _linear_operands(x, weight)
    act = _activation(activation)
    kind = x.dtype
    shape = x.shape[:-1] + (outer,)
    res = res_stride = 0
    if bias is not None:
        _vector(bias, outer, "bias")
        if bias.dtype != kind:
            raise ValueError("bias must have x's type")
        _on(index, bias, "bias")
    if residual is not None:
        if residual.shape != shape or residual.dtype != kind:
            raise ValueError("residual must have y's shape and x's type")
        _on(index, residual, "residual")
        _, _, res_stride, r2 = _rows(residual, "residual")
        res = r2.data_ptr()
    y = x.new_empty(tuple(shape))
    z = torch.empty_like(y) if keep_preactivation and act else None
    xp, wp = x2.data_ptr(), w2.data_ptr()
    size = _native._linear_forward_workspace(xp, xs, wp, ws, rows, inner, outer)
    space = _workspace(size, x)
    _call(index, _native._linear_forward, xp, xs, wp, ws, _ptr(bias), res, res_stride, _DTYPES[kind], act, rows, inner,
          outer, y.data_ptr(), outer, _ptr(z), _ptr(space), size)
    return y, z


def linear_backward(dy, x, weight, z=None, *, activation=None, need=(True, True, True)):
    """``(dx, dweight, dbias)`` of :func:`linear` from the gradient of y.

    z: from :func:`linear_forward` (with an activation).  ``need`` says which
    of the three to form; the others are None.  The residual's gradient is dy."""
    index, (rows, inner, xs, x2), (outer, _, ws, w2) = _linear_operands(x, weight)
    act = _activation(activation)
    kind = x.dtype
    shape = x.shape[:-1] + (outer,)
    if dy.shape != shape or dy.dtype != kind:
        raise ValueError("dy must have y's shape and x's type")
    _on(index, dy, "dy")
    _, _, dys, dy2 = _rows(dy, "dy")
    if act:
        if z is None or z.shape != shape or z.dtype != kind or not z.is_contiguous():
            raise ValueError("z must be what linear_forward kept: y's shape, x's type, contiguous")
        _on(index, z, "z")
    dx = _like(x) if need[0] else None
    dw = _like(weight) if need[1] else None
    db = x.new_empty((outer,)) if need[2] else None
    xp, wp, dp = x2.data_ptr(), w2.data_ptr(), dy2.data_ptr()
    size = _native._linear_backward_workspace(dp, dys, xp, xs, wp, ws, act, rows, inner, outer)
    space = _workspace(size, x)
    _call(index, _native._linear_backward, dp, dys, xp, xs, wp, ws, _ptr(z if act else None), _DTYPES[kind], act, rows,
          inner, outer, _ptr(dx), _ptr(dw), _ptr(db), _ptr(space), size)
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


def linear_status(device=None):
    """Raises ``RuntimeError``, once, if a device-side wait of an earlier
    :func:`linear` call on the device (default: the current one) expired: what
    was computed since the last report is void.  The next call that runs a
    product says the same; this one covers the last call and the replays of a
    graph.  It does not wait: synchronise first."""
    with torch.cuda.device(device):
        _native._linear_status()


# ------------------------------------------------------------------ rows in 8 bits
class RowCache:
    """Rows of one width in 8 bits, in the caller's tensors.

    codes [slots, width] int8 with scales [slots, groups] float32: ``group``
    elements (a multiple of 16, or 0 for the whole row) share a scale, a
    element stands for code * scale.  codes uint8: one affine map, an element
    stands for lo + step * code; these codes are a corpus of the exact u8
    search.  :meth:`empty` allocates with the row stride that reads fastest, a
    multiple of 16 bytes; what takes a device pointer and no stride (the C ABI's
    index over device memory) wants ``codes.contiguous()``.
    """

    def __init__(self, codes, scales=None, *, group=0, lo=0.0, step=1.0):
        index = _device(codes, "codes")
        affine = codes.dtype == torch.uint8
        if codes.dim() != 2 or not (affine or codes.dtype == torch.int8):
            raise ValueError("codes must be an int8 or uint8 matrix")
        slots, width = codes.shape
        stride, inner = codes.stride()
        if width < 1 or (width > 1 and inner != 1) or (slots > 1 and stride < width):
            raise ValueError("codes must be rows of contiguous elements that do not overlap")
        if affine:
            _require(scales is None, "uint8 codes have no scales")
            _require(step > 0, "step must be positive")
            group = 0
        else:
            _require(group >= 0 and group % 16 == 0, "group must be 0 or a multiple of 16")
            groups = -(-width // group) if group else 1
            if scales is None or scales.dtype != torch.float32 or scales.shape != (slots, groups) or \
                    not scales.is_contiguous():
                raise ValueError(f"scales must be a contiguous float32 matrix of {slots} x {groups}")
            _on(index, scales, "scales")
        self.codes, self.scales, self.group, self.lo, self.step = codes, scales, group, lo, step
        self.slots, self.width, self.index = slots, width, index
        self._native = _native._Rows(codes.data_ptr(), _ptr(scales), slots, stride if stride > width else width, width,
                                     group, affine, lo, step)

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

    def _ids(self, ids, name):
        wide = ids.dtype == torch.int64
        if not (wide or ids.dtype == torch.int32) or not ids.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 or int64")
        _on(self.index, ids, name)
        return 64 if wide else 32

    def write(self, slots, rows):
        """Quantises rows [n, width] (float32, bfloat16 or float16) into the
        given slots; a slot outside [0, slots) (-1, say) writes nothing.  The
        slots of one call that are inside must differ from one another."""
        bits = self._ids(slots, "slots")
        if slots.dim() != 1 or rows.dim() != 2 or rows.shape != (slots.shape[0], self.width):
            raise ValueError(f"slots must be one-dimensional and rows must be {slots.shape[0]} x {self.width}")
        code = _dtype(rows, "rows")
        _on(self.index, rows, "rows")
        n, _, stride, _ = _rows(rows, "rows")
        _call(self.index, _native._rows_write, self._native, slots.data_ptr(), bits, rows.data_ptr(), stride, code, n)

    def read(self, ids, dtype=torch.float32):
        """The rows of ids [...] as [..., width] of ``dtype``: what the codes
        stand for, zeros where an id is outside [0, slots)."""
        bits = self._ids(ids, "ids")
        code = _DTYPES.get(dtype)
        if code is None:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
        out = self.codes.new_empty((*ids.shape, self.width), dtype=dtype)
        _call(self.index, _native._rows_read, self._native, ids.data_ptr(), bits, ids.numel(), out.data_ptr(),
              self.width, code)
        return out


# ------------------------------------------------------------------ attention over found rows
def _list_stride(t, queries, found, name):
    """The row stride of lists [queries, found]; 0 gives every query the same."""
    stride, inner = t.stride()
    if (found > 1 and inner != 1) or (queries > 1 and stride < found and stride != 0):
        raise ValueError(f"{name} must be rows of contiguous entries")
    return stride


def _attend_args(q, ids, keys, values, scale, cap, bias, query_docs, row_docs):
    index = _device(q, "q")
    code = _dtype(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [queries, heads, head]")
    queries, heads, head = q.shape
    q_stride, head_stride, inner = q.stride()
    if heads < 1 or head < 8 or head % 8 or head > 256:
        raise ValueError("q: the head size must be a multiple of 8 up to 256")
    if inner != 1:
        raise ValueError("q: the last dimension must be contiguous")
    width, slots = keys.width, keys.slots
    if values.width != width or values.slots != slots:
        raise ValueError("keys and values must have one shape")
    if width % head or heads % (width // head):
        raise ValueError(f"cache rows of {width} do not hold heads of {head} that {heads} query heads share")
    if keys.index != index or values.index != index:
        raise ValueError(f"keys and values must be on cuda:{index}")
    if ids.dim() != 2 or ids.shape[0] != queries or ids.dtype != torch.int32:
        raise ValueError("ids must be int32 [queries, found]")
    found = ids.shape[1]
    _on(index, ids, "ids")
    ids_stride, bias_stride = _list_stride(ids, queries, found, "ids"), 0
    if bias is not None:
        if bias.shape != ids.shape or bias.dtype != torch.float32:
            raise ValueError("bias must be float32 of ids' shape")
        bias_stride = _list_stride(bias, queries, found, "bias")
        _on(index, bias, "bias")
    if query_docs is not None or row_docs is not None:
        _require(query_docs is not None and row_docs is not None, "query_docs and row_docs go together")
        for t, name, n in ((query_docs, "query_docs", queries), (row_docs, "row_docs", slots)):
            _vector(t, n, name)
            _require(t.dtype == torch.int32, f"{name} must be int32")
            _on(index, t, name)
    if not cap >= 0:
        raise ValueError("cap must be >= 0")
    return index, _native._AttendArgs(q.data_ptr(), ids.data_ptr(), _ptr(bias), _ptr(query_docs), _ptr(row_docs),
                                      q_stride, head_stride, ids_stride, bias_stride, queries, found, heads,
                                      heads * head // width, head, code, head ** -0.5 if scale is None else scale, cap)


def _attend(q, ids, keys, values, scale, cap, bias, query_docs, row_docs):
    index, args = _attend_args(q, ids, keys, values, scale, cap, bias, query_docs, row_docs)
    out = _like(q)
    lse = q.new_empty((q.shape[0], q.shape[1]), dtype=torch.float32)
    size = _native._attend_workspace(args)
    ws = _workspace(size, q)
    _call(index, _native._attend, args, keys._native, values._native, out.data_ptr(), lse.data_ptr(), _ptr(ws), size)
    return out, lse


def attend_backward(dout, q, ids, keys, values, lse, *, scale=None, cap=0.0, bias=None, query_docs=None,
                    row_docs=None, dlse=None, need=(True, True)):
    """``(dq, dbias)`` of :func:`attend` from the gradient of its output and
    its own lse (never one joined with another attention's); dlse is the
    gradient of lse where that took part too.  dbias (float32, summed over the
    heads) is None without a bias.  The caches are constants.  ``need`` says
    which of the two to give; the other is None.  dbias takes 8 bytes of scratch
    for each query, head and entry (4 GB for 8,192 x 16 x 4,096)."""
    index, args = _attend_args(q, ids, keys, values, scale, cap, bias, query_docs, row_docs)
    if dout.shape != q.shape or dout.dtype != q.dtype or not dout.is_contiguous():
        raise ValueError("dout must be contiguous, of q's shape and type")
    if lse.shape != q.shape[:2] or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be what attend returned")
    _on(index, dout, "dout")
    _on(index, lse, "lse")
    if dlse is not None:
        if dlse.shape != lse.shape or dlse.dtype != torch.float32 or not dlse.is_contiguous():
            raise ValueError("dlse must be contiguous float32 of lse's shape")
        _on(index, dlse, "dlse")
    dq = _like(q)
    dbias = q.new_empty(tuple(ids.shape), dtype=torch.float32) if bias is not None and need[1] else None
    size = _native._attend_backward_workspace(args, dbias is not None)
    ws = _workspace(size, q)
    _call(index, _native._attend_backward, args, keys._native, values._native, dout.data_ptr(), lse.data_ptr(),
          _ptr(dlse), dq.data_ptr(), _ptr(dbias), _ptr(ws), size)
    return dq if need[0] else None, dbias


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, bias, ids, keys, values, scale, cap, query_docs, row_docs):
        out, lse = _attend(q, ids, keys, values, scale, cap, bias, query_docs, row_docs)
        ctx.save_for_backward(q, bias, ids, lse, query_docs, row_docs)
        ctx.rest = (keys, values, scale, cap)
        ctx.set_materialize_grads(False)  # a loss mostly leaves lse out
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlse):
        q, bias, ids, lse, query_docs, row_docs = ctx.saved_tensors
        keys, values, scale, cap = ctx.rest
        dout = q.new_zeros(tuple(q.shape)) if dout is None else dout.contiguous()
        dlse = None if dlse is None else dlse.contiguous()
        dq, dbias = attend_backward(dout, q, ids, keys, values, lse, scale=scale, cap=cap, bias=bias,
                                    query_docs=query_docs, row_docs=row_docs, dlse=dlse, need=ctx.needs_input_grad[:2])
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
    this attention with another over other rows.  Both are differentiable in q
    and bias; the caches are constants, and rows that a query read must not be
    rewritten before its backward pass."""
    if _wants_grad(q, bias):
        return _Attend.apply(q, bias, ids, keys, values, scale, cap, query_docs, row_docs)
    return _attend(q, ids, keys, values, scale, cap, bias, query_docs, row_docs)
