"""Cases for the operators around the exact search: layer norm, the projection that makes the rows, the 8-bit row cache
and attention over the rows that a search found.

``listed()`` names the cases, ``draw(rng)`` makes more of the same ranges.  ``run(state)`` is one pass: the framework's
operators where ``own`` is true, else the same operators in elementary torch operations in float32.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-5


def _memory():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "winnex-madhava_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from winnex_madhava import memory

    return memory


# ------------------------------------------------------------------ cases
def listed():
    return [
        # The state of one new token or query, before it is projected: latency.
        {"name": "norm_token", "op": "norm", "rows": 1, "width": 768, "type": "bf16", "weights": "bf16", "train": False},
        # A training step's tokens at the width of the float corpus, with float32 master weights.
        {"name": "norm_train", "op": "norm", "rows": 65_536, "width": 768, "type": "bf16", "weights": "f32", "train": True},
        # Float rows of an odd count at a width that no vector divides.
        {"name": "norm_odd", "op": "norm", "rows": 20_011, "width": 301, "type": "f32", "weights": "f32", "train": True},
        # One query projected to the width of the float corpus: the weights' bytes and latency.
        {"name": "linear_token", "op": "linear", "rows": 1, "inner": 768, "outer": 768, "type": "bf16",
         "activation": "gelu", "residual": False, "train": False},
        # A training step of the widening layer of a projection head.
        {"name": "linear_train", "op": "linear", "rows": 16_384, "inner": 768, "outer": 2_048, "type": "bf16",
         "activation": "gelu", "residual": False, "train": True},
        # A ragged batch on sizes that no tile divides, with a residual.
        {"name": "linear_ragged", "op": "linear", "rows": 5_003, "inner": 300, "outer": 200, "type": "f16",
         "activation": "silu", "residual": True, "train": True},
        # One new row goes into the cache, the rows that a top-10 search found come back with it: latency.
        {"name": "rows_token", "op": "rows", "slots": 100_000, "width": 768, "write": 1, "read": 11, "group": 64,
         "code": "int8", "type": "bf16", "back": "bf16"},
        # A corpus of float rows becomes the u8 codes that the exact search scans, and is read back whole.
        {"name": "rows_corpus", "op": "rows", "slots": 1_000_003, "width": 128, "write": 1_000_003, "read": 1_000_003,
         "group": 0, "code": "uint8", "type": "f32", "back": "f32"},
        # One query with shared heads reads its top-32.
        {"name": "attend_token", "op": "attend", "slots": 100_000, "queries": 1, "found": 32, "heads": 12, "shared": 3,
         "head": 64, "group": 64, "code": "int8", "type": "bf16", "cap": 0.0, "bias": False, "documents": 0,
         "train": False},
        # The batch of the cosine benchmark reads its top-100, each query only rows of its own document set.
        {"name": "attend_batch", "op": "attend", "slots": 1_000_000, "queries": 4_096, "found": 100, "heads": 12,
         "shared": 1, "head": 64, "group": 64, "code": "int8", "type": "bf16", "cap": 0.0, "bias": True,
         "documents": 4, "train": False},
        # A few queries read the longest lists that the clustered search returns.
        {"name": "attend_long", "op": "attend", "slots": 500_000, "queries": 8, "found": 4_096, "heads": 16, "shared": 8,
         "head": 128, "group": 128, "code": "int8", "type": "f16", "cap": 30.0, "bias": True, "documents": 0,
         "train": False},
        # A training step through the memory: gradients of the queries and of the distances' bias.
        {"name": "attend_train", "op": "attend", "slots": 200_000, "queries": 2_048, "found": 64, "heads": 12,
         "shared": 3, "head": 64, "group": 64, "code": "int8", "type": "bf16", "cap": 20.0, "bias": True,
         "documents": 0, "train": True},
    ]


def _between(rng, low, high):
    """A whole number of [low, high], its logarithm spread evenly."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "rows", "attend"])
    if op == "norm":
        width = _between(rng, 7, 8_192)
        kind = rng.choice(["f32", "bf16", "f16"])
        return {"op": op, "rows": _between(rng, 1, min(131_072, 50_000_000 // width)), "width": width, "type": kind,
                "weights": rng.choice(["f32", kind]), "train": rng.random() < 0.6}
    if op == "linear":
        inner, outer = _between(rng, 48, 2_048), _between(rng, 48, 2_048)
        return {"op": op, "rows": _between(rng, 1, min(65_536, 25_000_000_000 // (inner * outer))), "inner": inner,
                "outer": outer, "type": rng.choice(["bf16", "f16"]),
                "activation": rng.choice(["none", "relu", "gelu", "silu"]), "residual": rng.random() < 0.5,
                "train": rng.random() < 0.6}
    if op == "rows":
        width = _between(rng, 7, 2_048)
        slots = _between(rng, 100, min(1_000_000, 120_000_000 // width))
        code = rng.choice(["int8", "uint8"])
        return {"op": op, "slots": slots, "width": width, "write": _between(rng, 1, slots), "read": _between(rng, 1, slots),
                "group": rng.choice([0, 16, 32, 64, 128]) if code == "int8" else 0, "code": code,
                "type": rng.choice(["f32", "bf16", "f16"]), "back": rng.choice(["f32", "bf16", "f16"])}
    head = rng.choice([32, 40, 64, 96, 128])
    groups = rng.choice([1, 2, 4, 8])
    shared = rng.choice([1, 2, 4, 8])
    width = groups * head
    found = _between(rng, 1, 4_096)
    code = rng.choice(["int8", "int8", "uint8"])
    return {"op": op, "slots": _between(rng, 1_000, min(1_000_000, 700_000_000 // width)),
            "queries": _between(rng, 1, max(1, min(8_192, 200_000_000 // (width * found * max(1, shared // 2))))),
            "found": found, "heads": groups * shared, "shared": shared, "head": head,
            "group": rng.choice([16, 32, 64, 0]) if code == "int8" else 0, "code": code,
            "type": rng.choice(["f32", "bf16", "f16"]), "cap": rng.choice([0.0, 0.0, 20.0]),
            "bias": rng.random() < 0.5, "documents": rng.choice([0, 0, 3]), "train": rng.random() < 0.4}


# ------------------------------------------------------------------ inputs
def _normal(gen, shape, kind, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(_TYPES[kind])


def _groups(width, group):
    return 1 if group == 0 else -(-width // group)


def _codes(gen, case, slots, width):
    """A cache that holds rows already: codes with a row stride of 16 bytes, scales as quantised rows have them."""
    held = torch.randint(0, 256, (slots, -(-width // 16) * 16), generator=gen, device="cuda", dtype=torch.uint8)
    if case["code"] == "uint8":
        return held[:, :width], None
    held = held.view(torch.int8)
    held.clamp_(min=-127)
    scales = torch.rand((slots, _groups(width, case["group"])), generator=gen, device="cuda") * 0.02 + 0.01
    return held[:, :width], scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    op, kind = case["op"], case["type"]
    if op == "norm":
        shape = (case["rows"], case["width"])
        s["x"] = _normal(gen, shape, kind) * 1.5 + 0.25
        s["w"] = (1 + _normal(gen, shape[1:], "f32", 0.1)).to(_TYPES[case["weights"]])
        s["b"] = _normal(gen, shape[1:], case["weights"], 0.1)
        s["dy"] = _normal(gen, shape, kind) if case["train"] else None
    elif op == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        s["x"] = _normal(gen, (m, k), kind)
        s["w"] = _normal(gen, (n, k), kind, k ** -0.5)
        s["b"] = _normal(gen, (n,), kind, 0.1)
        s["res"] = _normal(gen, (m, n), kind) if case["residual"] else None
        s["dy"] = _normal(gen, (m, n), kind) if case["train"] else None
    elif op == "rows":
        slots, width, count, reads = case["slots"], case["width"], case["write"], case["read"]
        s["codes"], s["scales"] = _codes(gen, case, slots, width)
        s["rows"] = _normal(gen, (count, width), kind)
        s["slot"] = torch.randperm(slots, generator=gen, device="cuda")[:count].to(torch.int32)
        ids = torch.randperm(slots, generator=gen, device="cuda")[:reads].to(torch.int32)
        ids[: min(reads, count)] = s["slot"][: min(reads, count)]
        if count > 64:
            s["slot"][::61] = -1  # padding rows of a batch
        if reads > 64:
            ids[::53] = -1  # places that the search left empty
        s["ids"], s["lo"], s["step"] = ids, -4.0, 8.0 / 255.0
    else:
        slots, nq, k = case["slots"], case["queries"], case["found"]
        heads, width = case["heads"], case["heads"] // case["shared"] * case["head"]
        s["keys"], s["key_scales"] = _codes(gen, case, slots, width)
        s["values"], s["value_scales"] = _codes(gen, case, slots, width)
        s["lo"], s["step"] = -1.0, 2.0 / 255.0
        s["q"] = _normal(gen, (nq, heads, case["head"]), kind)
        ids = torch.randint(0, slots, (nq, k), generator=gen, device="cuda", dtype=torch.int32)
        kept = torch.randint(-k // 8, 9 * k, (nq, 1), generator=gen, device="cuda")  # some lists end early, few are empty
        s["ids"] = torch.where(torch.arange(k, device="cuda") < kept, ids, -1)
        s["bias"] = None
        if case["bias"]:
            s["bias"] = -4 * torch.rand((nq, k), generator=gen, device="cuda")
            s["bias"].masked_fill_(torch.rand((nq, k), generator=gen, device="cuda") < 0.02, -math.inf)
        s["row_docs"] = s["query_docs"] = None
        if case["documents"]:
            s["row_docs"] = torch.randint(0, case["documents"], (slots,), generator=gen, device="cuda", dtype=torch.int32)
            s["query_docs"] = torch.randint(0, case["documents"], (nq,), generator=gen, device="cuda", dtype=torch.int32)
        s["do"] = _normal(gen, (nq, heads, case["head"]), kind) if case["train"] else None
    return s


# ------------------------------------------------------------------ plain forms
def _norm_plain(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + _EPS).rsqrt()
    xh = (x - mean) * rstd
    out = {"y": (xh * w + b).to(s["x"].dtype)}
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        out |= {"dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0).to(s["w"].dtype), "db": dy.sum(0).to(s["b"].dtype)}
    return out


def _act_plain(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope_plain(z, name):
    if name == "relu":
        return (z > 0).float()
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if name == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    return torch.ones_like(z)


def _linear_plain(s):
    x, w, kind = s["x"].float(), s["w"].float(), s["x"].dtype
    z = x @ w.T + s["b"].float()
    y = _act_plain(z, s["activation"])
    if s["res"] is not None:
        y = y + s["res"].float()
    out = {"y": y.to(kind)}
    if s["train"]:
        dz = s["dy"].float() * _slope_plain(z, s["activation"])
        out |= {"dx": (dz @ w).to(kind), "dw": (dz.T @ x).to(kind), "db": dz.sum(0).to(kind)}
    return out


def _spread(scales, width, group):
    """A scale for each element, from one for each group."""
    return scales.expand(-1, width) if group == 0 else scales.repeat_interleave(group, 1)[:, :width]


def _values(codes, scales, ids, s, width):
    """The rows that cache places stand for, in float32."""
    c = codes[ids].float()
    return s["lo"] + s["step"] * c if scales is None else c * _spread(scales[ids], width, s["group"])


def _rows_plain(s):
    width, group, slots = s["width"], s["group"], s["slots"]
    kept = (s["slot"] >= 0) & (s["slot"] < slots)
    x, at = s["rows"].float()[kept], s["slot"][kept].long()
    if s["code"] == "uint8":
        s["codes"][at] = ((x - s["lo"]) * (1 / s["step"])).clamp(0, 255).round().to(torch.uint8)
    else:
        n = _groups(width, group)
        padded = torch.nn.functional.pad(x, (0, n * group - width if group else 0))
        top = padded.abs().view(x.shape[0], n, -1).amax(2)
        zero = torch.zeros_like(top)
        inv = torch.where(top >= 2.0 ** -100, 127 / top, zero)
        s["scales"][at] = torch.where(top >= 2.0 ** -100, top / 127, zero)
        s["codes"][at] = (x * _spread(inv, width, group)).round().to(torch.int8)
    known = (s["ids"] >= 0) & (s["ids"] < slots)
    back = _values(s["codes"], s["scales"], s["ids"].clamp(0, slots - 1).long(), s, width)
    return {"back": torch.where(known[:, None], back, 0.0).to(_TYPES[s["back"]])}


def _attend_plain(s):
    nq, k, heads, shared, head = s["queries"], s["found"], s["heads"], s["shared"], s["head"]
    groups, slots = heads // shared, s["slots"]
    at = s["ids"].clamp(0, slots - 1).long()
    seen = (s["ids"] >= 0) & (s["ids"] < slots)
    if s["row_docs"] is not None:
        seen = seen & (s["row_docs"][at] == s["query_docs"][:, None])
    if s["bias"] is not None:
        seen = seen & (s["bias"] != -math.inf)
    flat = at.reshape(-1)
    keys = _values(s["keys"], s["key_scales"], flat, s, groups * head).view(nq, k, groups, head).permute(0, 2, 3, 1)
    values = _values(s["values"], s["value_scales"], flat, s, groups * head).view(nq, k, groups, head).permute(0, 2, 1, 3)
    q = s["q"].float().view(nq, groups, shared, head)
    scale, cap = head ** -0.5, s["cap"]
    score, slope = scale * (q @ keys), 1.0
    if cap:
        t = torch.tanh(score / cap)
        score, slope = cap * t, 1 - t * t
    if s["bias"] is not None:
        score = score + s["bias"][:, None, None, :]
    score = torch.where(seen[:, None, None, :], score, -math.inf)
    top = score.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(3, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    o = p @ values
    out = {"o": o.reshape(nq, heads, head).to(s["q"].dtype), "lse": (torch.log(total) + top).view(nq, heads)}
    if s["train"]:
        dp = s["do"].float().view(nq, groups, shared, head) @ values.transpose(2, 3)
        ds = p * (dp - (p * dp).sum(3, keepdim=True))
        out["dq"] = (scale * ((ds * slope) @ keys.transpose(2, 3))).reshape(nq, heads, head).to(s["q"].dtype)
        if s["bias"] is not None:
            out["dbias"] = ds.sum((1, 2))
    return out


# ------------------------------------------------------------------ the framework's operators
def _norm_own(s):
    m = _memory()
    if not s["train"]:
        return {"y": m.layer_norm(s["x"], s["w"], s["b"], eps=_EPS)}
    y, mean, rstd = m.layer_norm_forward(s["x"], s["w"], s["b"], eps=_EPS)
    dx, dw, db = m.layer_norm_backward(s["dy"], s["x"], s["w"], mean, rstd)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _linear_own(s):
    m = _memory()
    if not s["train"]:
        return {"y": m.linear(s["x"], s["w"], s["b"], activation=s["activation"], residual=s["res"])}
    y, z = m.linear_forward(s["x"], s["w"], s["b"], activation=s["activation"], residual=s["res"],
                            keep_preactivation=True)
    dx, dw, db = m.linear_backward(s["dy"], s["x"], s["w"], z, activation=s["activation"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _rows_own(s):
    cache = _memory().RowCache(s["codes"], s["scales"], group=s["group"], lo=s["lo"], step=s["step"])
    cache.write(s["slot"], s["rows"])
    return {"back": cache.read(s["ids"], dtype=_TYPES[s["back"]])}


def _attend_own(s):
    m = _memory()
    keys = m.RowCache(s["keys"], s["key_scales"], group=s["group"], lo=s["lo"], step=s["step"])
    values = m.RowCache(s["values"], s["value_scales"], group=s["group"], lo=s["lo"], step=s["step"])
    how = {"cap": s["cap"], "bias": s["bias"], "query_docs": s["query_docs"], "row_docs": s["row_docs"]}
    o, lse = m.attend(s["q"], s["ids"], keys, values, **how)
    out = {"o": o, "lse": lse}
    if s["train"]:
        out["dq"], dbias = m.attend_backward(s["do"], s["q"], s["ids"], keys, values, lse, **how)
        if dbias is not None:
            out["dbias"] = dbias
    return out


def run(state):
    forms = ({"norm": _norm_own, "linear": _linear_own, "rows": _rows_own, "attend": _attend_own} if own else
             {"norm": _norm_plain, "linear": _linear_plain, "rows": _rows_plain, "attend": _attend_plain})
    return forms[state["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if op == "norm":
        n, e = case["rows"] * case["width"], size[case["type"]]
        passes = 4 if case["train"] else 2
        return {"bytes": n * e * passes + case["width"] * size[case["weights"]] * passes,
                "flops": n * (20 if case["train"] else 8)}
    if op == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        moved = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        if case["train"]:
            moved += m * n + m * k + n * k + n
        return {"bytes": 2 * moved, "flops": (6 if case["train"] else 2) * m * n * k}
    groups = 0 if case["code"] == "uint8" else 4  # bytes of a group's scale
    if op == "rows":
        width = case["width"]
        held = width + groups * _groups(width, case["group"])
        moved = case["write"] * (width * size[case["type"]] + held + 4)
        moved += case["read"] * (held + width * size[case["back"]] + 4)
        return {"bytes": moved, "flops": 4 * width * case["write"] + 2 * width * case["read"]}
    nq, k, heads, head = case["queries"], case["found"], case["heads"], case["head"]
    width = heads // case["shared"] * head
    held = width + groups * _groups(width, case["group"])
    moved = 2 * min(nq * k, case["slots"]) * held + nq * k * (8 if case["bias"] else 4)
    moved += nq * heads * (2 * head * size[case["type"]] + 4)
    if case["train"]:
        moved += nq * heads * 2 * head * size[case["type"]] + (4 * nq * k if case["bias"] else 0)
    return {"bytes": moved, "flops": (12 if case["train"] else 4) * nq * k * heads * head}


# ------------------------------------------------------------------ in 64 bits, from the definitions
def _exact_norm(s):
    x, w, b = (s[n].double() for n in ("x", "w", "b"))
    width = x.shape[1]
    centred = x - x.sum(1, keepdim=True) / width
    spread = torch.sqrt((centred ** 2).sum(1, keepdim=True) / width + _EPS)
    unit = centred / spread
    out = {"y": unit * w + b}
    if s["train"]:
        up = s["dy"].double()
        inner = up * w
        out["db"] = up.sum(0)
        out["dw"] = torch.einsum("rc,rc->c", up, unit)
        along = torch.einsum("rc,rc->r", inner, unit)[:, None] / width
        out["dx"] = (inner - inner.sum(1, keepdim=True) / width - unit * along) / spread
    return out


def _exact_linear(s):
    x, w = s["x"].double(), s["w"].double()
    z = torch.einsum("mk,nk->mn", x, w) + s["b"].double()
    half = torch.special.erf(z / math.sqrt(2)) / 2 + 0.5
    gate = torch.sigmoid(z)
    value, slope = {
        "none": (z, torch.ones_like(z)),
        "relu": (torch.relu(z), torch.heaviside(z, torch.zeros_like(z))),
        "gelu": (z * half, half + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi)),
        "silu": (z * gate, gate + z * gate * (1 - gate)),
    }[s["activation"]]
    out = {"y": value if s["res"] is None else value + s["res"].double()}
    if s["train"]:
        dz = slope * s["dy"].double()
        out |= {"dx": torch.einsum("mn,nk->mk", dz, w), "dw": torch.einsum("mn,mk->nk", dz, x), "db": dz.sum(0)}
    return out


def _exact_held(codes, scales, s):
    """What every place of a cache stands for."""
    c = codes.double()
    if scales is None:
        return s["lo"] + s["step"] * c
    group = s["group"] or c.shape[1]
    of = torch.arange(c.shape[1], device=c.device) // group
    return c * scales.double()[:, of]


def _exact_rows(s):
    # The stored scale, its inverse and the products are 32-bit values by definition: each is rounded to them.
    slots, width = s["slots"], s["width"]
    held = _exact_held(s["codes"], s["scales"], s)
    keep = torch.nonzero(torch.logical_and(s["slot"] >= 0, s["slot"] < slots))[:, 0]
    x, at = s["rows"][keep].double(), s["slot"][keep].long()
    if s["code"] == "uint8":
        off = (x - s["lo"]).float().double()
        inv = torch.tensor(1 / s["step"], dtype=torch.float32).double().item()
        new = torch.round(torch.clip((off * inv).float().double(), 0, 255)) * s["step"] + s["lo"]
    else:
        group = s["group"] or width
        of = torch.arange(width, device=x.device) // group
        n = int(of[-1]) + 1
        top = torch.zeros((x.shape[0], n), dtype=torch.float64, device=x.device)
        top.scatter_reduce_(1, of.expand(x.shape[0], -1), x.abs(), "amax")
        some = top >= 2.0 ** -100
        inv = torch.where(some, 127 / top, 0.0).float().double()
        scale = torch.where(some, top / 127, 0.0).float().double()
        new = torch.round((x * inv[:, of]).float().double()) * scale[:, of]
    held[at] = new
    out = torch.zeros((s["read"], width), dtype=torch.float64, device=x.device)
    found = torch.nonzero(torch.logical_and(s["ids"] >= 0, s["ids"] < slots))[:, 0]
    out[found] = held[s["ids"][found].long()]
    return {"back": out}


def _exact_attend(s):
    nq, heads, shared, head, slots = s["queries"], s["heads"], s["shared"], s["head"], s["slots"]
    outs = []
    step = max(1, 40_000_000 // (s["found"] * heads * head))
    for i in range(0, nq, step):
        ids = s["ids"][i:i + step]
        hidden = torch.logical_or(ids < 0, ids >= slots)
        at = torch.where(hidden, 0, ids).long()
        if s["documents"]:
            hidden = torch.logical_or(hidden, s["row_docs"][at] != s["query_docs"][i:i + step, None])
        extra = torch.zeros(ids.shape, dtype=torch.float64, device=ids.device)
        if s["bias"] is not None:
            extra = s["bias"][i:i + step].double()
            hidden = torch.logical_or(hidden, torch.isneginf(extra))
        rows = []
        for name in ("keys", "values"):
            held = None if s[name[:-1] + "_scales"] is None else s[name[:-1] + "_scales"][at.flatten()]
            rows.append(_exact_held(s[name][at.flatten()], held, s).view(*ids.shape, heads // shared, head)
                        .repeat_interleave(shared, 2))
        k, v = rows
        q = s["q"][i:i + step].double()
        raw = torch.einsum("qhd,qkhd->qhk", q, k) / math.sqrt(head)
        capped = s["cap"] * torch.tanh(raw / s["cap"]) if s["cap"] else raw
        score = (capped + extra[:, None]).masked_fill(hidden[:, None], -math.inf)
        lse = torch.logsumexp(score, 2)
        p = torch.exp(score - torch.where(torch.isneginf(lse), 0.0, lse)[..., None])
        one = {"o": torch.einsum("qhk,qkhd->qhd", p, v), "lse": lse}
        if s["train"]:
            dp = torch.einsum("qhd,qkhd->qhk", s["do"][i:i + step].double(), v)
            ds = p * (dp - torch.einsum("qhk,qhk->qh", p, dp)[..., None])
            if s["bias"] is not None:
                one["dbias"] = ds.sum(1)
            inner = ds * (1 - (capped / s["cap"]) ** 2) if s["cap"] else ds
            one["dq"] = torch.einsum("qhk,qkhd->qhd", inner, k) / math.sqrt(head)
        outs.append(one)
    return {name: torch.cat([o[name] for o in outs]) for name in outs[0]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "rows": _exact_rows, "attend": _exact_attend}[case["op"]](s)
