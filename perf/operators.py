"""A transformer block's operators as cases that can be timed and checked.

A case is a dict of plain values; prepare() builds what a program holds before
the call, run() is one pass, exact() the same outputs in 64 bits. Where `own`
is true run() calls the framework (tensors on the "hip" device); where it is
false it computes the same by elementary torch operations in 32 bits. Kinds:

  rotary     rotation of feature pairs by position: half or interleaved pairs,
             the whole head or its first features, tables scaled for long
             contexts, with or without the gradient
  attention  softmax attention with shared key/value heads whose mask is given
             by rules (causal, prefix, documents, key lengths) and whose scores
             may be capped by a tanh or biased by distance; forward alone (one
             query over a cache among it) or with the three gradients
  adamw      one decoupled-weight-decay Adam step over a list of tensors, with
             the moments in 32 bits or in blocks of 8-bit codes

Tensors are (batch, length, heads, features); "bhld" cases hold them as
(batch, heads, length, features) and pass a transposed view.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256  # elements that share a scale in the 8-bit moments


# ------------------------------------------------------------------ cases --
def _rotary(name, batch, length, heads, dim, **more):
    case = {"kind": "rotary", "batch": batch, "length": length, "heads": heads, "dim": dim, "part": dim, "pairs": "half",
            "scaling": "none", "factor": 1.0, "positions": "offset", "offset": 0, "dtype": "bfloat16", "out": "bfloat16",
            "layout": "blhd", "grad": False, **more}
    return {"name": name, **case} if name else case


def _attention(name, batch, queries, keys, heads, kv_heads, dim, dtype, **more):
    case = {"kind": "attention", "batch": batch, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "causal": True, "cap": 0.0, "bias": False, "documents": 0, "prefix": False,
            "lengths": False, "layout": "blhd", "grad": False, **more}
    return {"name": name, **case} if name else case


def _adamw(name, sizes, bits, **more):
    case = {"kind": "adamw", "sizes": sizes, "bits": bits, "dtype": "float32", "step": 10, **more}
    return {"name": name, **case} if name else case


def listed():
    return [
        # Serving: the queries of one new token of eight requests, far into their texts.
        _rotary("rotary_token", 8, 1, 16, 128, offset=1999),
        # Training: a projection's float32 result turned and rounded for the attention, and its gradient.
        _rotary("rotary_train", 4, 4096, 16, 128, dtype="float32", grad=True),
        # A long text in a scaled context: interleaved pairs of part of an odd-sized head, packed positions.
        _rotary("rotary_long_part", 1, 30011, 8, 80, part=48, pairs="interleaved", scaling="parts", factor=8.0,
                positions="tensor", dtype="float16", out="float16"),
        # The smallest attention call: one token of one request over a short cache.
        _attention("attention_token_short", 1, 1, 477, 16, 2, 64, "float16", lengths=True),
        # Serving: one token of 16 requests over long caches of unequal length, 4 query heads to a cache head.
        _attention("attention_token_long", 16, 1, 8192, 32, 8, 128, "bfloat16", lengths=True, layout="bhld"),
        # Training: a causal layer, forward and backward.
        _attention("attention_train", 2, 4096, 4096, 16, 4, 128, "bfloat16", grad=True),
        # Training on packed documents with capped scores.
        _attention("attention_documents", 1, 8192, 8192, 8, 8, 128, "float16", cap=30.0, documents=24, grad=True),
        # Float32 training with a prefix that sees itself whole, odd sizes.
        _attention("attention_prefix_f32", 2, 1025, 1025, 6, 6, 80, "float32", prefix=True, grad=True),
        # An encoder's forward pass over one long text, scores biased by distance.
        _attention("attention_distance", 1, 8191, 8191, 12, 12, 64, "bfloat16", causal=False, bias=True),
        # A small network's eight weights and biases: launches and host work are all of it.
        _adamw("adamw_small", "1024x72,72,72x72,72,72x40,40,513,1", 32),
        # The benchmark's 1024-4096-4096-1024 network with its biases.
        _adamw("adamw_network", "1024x4096,4096,4096x4096,4096,4096x1024,1024", 32),
        # The same network with its moments in 8 bits, which come back as the values they stand for.
        _adamw("adamw_network_8bit", "1024x4096,4096,4096x4096,4096,4096x1024,1024", 8),
    ]


def _log(rng, lo, hi, step=1):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, step * round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)))


def draw(rng):
    kind = rng.choice(["rotary", "attention", "attention", "token", "adamw"])
    if kind == "rotary":
        dim = 2 * _log(rng, 16, 128, rng.choice([1, 4, 16]))
        part = rng.choice([dim, dim, 2 * _log(rng, 4, dim // 2)])
        heads, batch = _log(rng, 1, 32), _log(rng, 1, 16)
        length = _log(rng, 1, min(32768, max(1, (1 << 25) // (batch * heads * dim))))
        dtype, out = rng.choice([("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float16", "float16")])
        scaling, factor = rng.choice([("none", 1.0), ("linear", 4.0), ("base", 4.0), ("parts", 8.0)])
        return _rotary(None, batch, length, heads, dim, part=part, pairs=rng.choice(["half", "interleaved"]), scaling=scaling,
                       factor=factor, positions=rng.choice(["offset", "tensor"]), offset=_log(rng, 1, 32768), dtype=dtype, out=out,
                       layout=rng.choice(["blhd", "blhd", "bhld"]), grad=rng.random() < 0.5)
    if kind in ("attention", "token"):
        dtype = rng.choice(["bfloat16", "float16", "bfloat16", "float32"])
        dim = _log(rng, 16, 256, rng.choice([1, 8, 16]))
        kv_heads, group, batch = _log(rng, 1, 8), rng.choice([1, 1, 2, 4, 7, 8]), _log(rng, 1, 16)
        more = {"cap": rng.choice([0.0, 0.0, 20.0]), "bias": rng.random() < 0.25, "layout": rng.choice(["blhd", "blhd", "bhld"])}
        if kind == "token":
            keys = _log(rng, 1, min(32768, (1 << 27) // (batch * kv_heads * dim)))
            return _attention(None, batch, min(keys, rng.choice([1, 1, 1, 2, 5])), keys, kv_heads * group, kv_heads, dim, dtype,
                              lengths=rng.random() < 0.7, **more)
        # The scores of the plain form stay under those of the largest listed case, fewer in float32.
        top = (1 << 29 if dtype != "float32" else 1 << 26) / (batch * kv_heads * group) * min(1.0, 128 / dim)
        queries = _log(rng, 1, max(1, min(8192, int(math.sqrt(top)))))
        keys = rng.choice([queries, queries, max(queries, _log(rng, 1, max(1, min(16384, int(top / queries)))))])
        causal = rng.random() < 0.7
        return _attention(None, batch, queries, keys, kv_heads * group, kv_heads, dim, dtype, causal=causal,
                          prefix=causal and rng.random() < 0.3, documents=rng.choice([0, 0, 1, 4, 16]) if keys == queries else 0,
                          lengths=keys != queries and rng.random() < 0.5, grad=rng.random() < 0.6, **more)
    bits = rng.choice([32, 8])
    sizes = ",".join(rng.choice(["%d", "%dx1"]) % _log(rng, 1, 1 << 21) for _ in range(rng.randint(1, 16)))
    return _adamw(None, sizes, bits, dtype=rng.choice(["float32", "float32", "bfloat16"]), step=rng.randint(1, 1000))


# ------------------------------------------------------------------ inputs --
def _type(name):
    return getattr(torch, name)


def _visible_positions(case, rng):
    """The rule's integers, as host arrays: documents of each token, prefixes, key lengths."""
    b, lq, lk = case["batch"], case["queries"], case["keys"]
    docs = prefix = lengths = None
    if case["documents"]:
        docs = np.zeros((b, lk), np.int32)
        for i in range(b):  # documents of unequal length one after the other, then up to 31 tokens of padding
            cuts = np.sort(rng.integers(0, lk, case["documents"] - 1))
            docs[i] = np.searchsorted(cuts, np.arange(lk), side="right")
            docs[i, lk - int(rng.integers(0, min(32, lk))):] = -1
    if case["prefix"]:
        prefix = rng.integers(0, lk // 2 + 1, b).astype(np.int32)
    if case["lengths"]:
        lengths = rng.integers(max(lq, lk // 4), lk + 1, b).astype(np.int32)
    return docs, prefix, lengths


def _slopes(heads):
    """Distance slopes: a geometric series that halves every eighth of the heads."""
    return (2.0 ** (-8.0 * (np.arange(heads) + 1) / heads)).astype(np.float32)


def _sizes(case):
    return [tuple(int(n) for n in s.split("x")) for s in case["sizes"].split(",")]


def _inputs(case, seed):
    """The case's inputs: torch tensors on the GPU of the case's types, and host arrays of its integers."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))

    def normal(shape, dtype, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(_type(dtype))

    def held(b, l, h, d, dtype):
        return normal((b, h, l, d) if case["layout"] == "bhld" else (b, l, h, d), dtype)

    if case["kind"] == "rotary":
        b, l, h, d = case["batch"], case["length"], case["heads"], case["dim"]
        x = {"x": held(b, l, h, d, case["dtype"])}
        if case["grad"]:
            x["dy"] = normal((b, l, h, d), case["out"])
        if case["positions"] == "tensor":  # texts packed one after the other: positions start again
            start = rng.integers(1, l + 1, (b, 1))
            pos = np.arange(l)[None, :]
            x["positions"] = np.where(pos < start, pos, pos - start).astype(np.int32)
        return x
    if case["kind"] == "attention":
        b, h, g, d, t = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["dtype"]
        x = {"q": held(b, case["queries"], h, d, t), "k": held(b, case["keys"], g, d, t), "v": held(b, case["keys"], g, d, t)}
        if case["grad"]:
            x["dy"] = normal((b, case["queries"], h, d), t)
        docs, prefix, lengths = _visible_positions(case, rng)
        slopes = _slopes(h) if case["bias"] else None
        return {**x, **{n: v for n, v in {"docs": docs, "prefix": prefix, "lengths": lengths, "slopes": slopes}.items() if v is not None}}
    x = {"p": [], "g": [], "m": [], "v": []}
    for shape in _sizes(case):
        n = math.prod(shape)
        x["p"].append(normal(shape, case["dtype"], 0.05))
        x["g"].append(normal(shape, case["dtype"], 0.01))
        if case["bits"] == 32:
            x["m"].append(normal(shape, "float32", 0.003))
            x["v"].append(normal(shape, "float32", 0.01).square())
        else:
            blocks = -(-n // BLOCK)
            inside = torch.arange(blocks * BLOCK, device="cuda") < n
            code = lambda lo, hi: torch.randint(lo, hi, (blocks * BLOCK,), generator=gen, device="cuda") * inside  # noqa: E731
            scale = lambda top: torch.rand(blocks, generator=gen, device="cuda") * top + 0.1 * top  # noqa: E731
            x["m"].append((code(-127, 128), scale(0.01)))
            x["v"].append((code(1, 256), scale(3e-4)))
    return x


def _frequencies(case):
    """Radians per position of each pair, in 64 bits."""
    part, factor = case["part"], case["factor"]
    base = 10000.0
    if case["scaling"] == "base":
        base *= factor ** (part / (part - 2)) if part > 2 else 1.0
    f = base ** (-np.arange(0, part, 2, dtype=np.float64) / part)
    if case["scaling"] == "linear":
        f /= factor
    if case["scaling"] == "parts":  # pairs of over 32 turns in 4096 positions stay, those under one turn stretch
        turns = 4096 * f / (2 * math.pi)
        keep = np.clip((turns - 1) / 31, 0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f


def _rows(case):
    """Positions that the rotary table has to hold."""
    return case["length"] + (case["offset"] if case["positions"] == "offset" else 0)


def prepare(case, seed):
    x = _inputs(case, seed)
    if not own:
        for n in ("docs", "prefix", "lengths", "slopes", "positions"):
            if n in x:
                x[n] = torch.from_numpy(x[n]).cuda()
        if case["kind"] == "rotary":
            angle = np.outer(np.arange(_rows(case)), _frequencies(case))
            x["cos"], x["sin"] = (torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))
        return {"case": dict(case), "x": x}
    import ormi_amd

    def leaf(t, grad=False):
        """The same values as a leaf of the framework."""
        if isinstance(t, np.ndarray):
            return ormi_amd.Tensor(t, "hip", dtype=str(t.dtype))
        kept = str(t.dtype).replace("torch.", "")
        return ormi_amd.Tensor(t.float().cpu().numpy(), "hip", requires_grad=grad, dtype=kept)

    out = {}
    if case["kind"] == "adamw":
        out["p"], out["g"] = [leaf(t) for t in x["p"]], [leaf(t) for t in x["g"]]
        if case["bits"] == 32:
            out["s"] = [ormi_amd.AdamState(leaf(m), leaf(v)) for m, v in zip(x["m"], x["v"])]
        else:
            code = lambda c, t: c.cpu().numpy().astype(t)  # noqa: E731
            out["s"] = [ormi_amd.AdamState8.from_codes(tuple(p.shape), code(m[0], np.int8), m[1].cpu().numpy(), code(v[0], np.uint8), v[1].cpu().numpy())
                        for p, m, v in zip(x["p"], x["m"], x["v"])]
    else:
        out = {n: leaf(t, grad=case["grad"] and n in ("x", "q", "k", "v")) for n, t in x.items()}
    if case["kind"] == "rotary":
        out["table"] = ormi_amd.RotaryTable(case["part"], _rows(case), "hip", scaling=case["scaling"], factor=case["factor"], original=4096)
    return {"case": dict(case), "x": out, "event": _event()}


# ------------------------------------------------- the framework's results --
def _library():
    import ctypes
    from pathlib import Path

    import ormi_amd

    lib = ctypes.CDLL(str(Path(ormi_amd.__file__).resolve().parent / "lib" / "libormi_hip.so"))
    lib.ormi_hip_event_record.argtypes = [ctypes.c_void_p]
    lib.ormi_hip_event_create.argtypes = [ctypes.POINTER(ctypes.c_void_p)]
    return lib


def _event():
    """What _hand_over records: an event of the library's stream."""
    import ctypes

    lib, event = _library(), ctypes.c_void_p()
    if lib.ormi_hip_event_create(ctypes.byref(event)) != 0:
        raise RuntimeError("cannot create an event")
    return lib.ormi_hip_event_record, event


class _Shared:
    """A realized tensor's buffer as torch sees it, without a copy; torch keeps
    this object, and so the buffer, as long as it uses the memory."""

    _TYPES = {"float32": "<f4", "bfloat16": "<i2", "float16": "<f2"}

    def __init__(self, tensor):
        self.tensor = tensor
        self.__cuda_array_interface__ = {"shape": tensor.shape, "typestr": self._TYPES[tensor.dtype], "version": 2,
                                         "data": (tensor._node.data.ptr, False)}


def _hand_over(state, **tensors):
    """The realized tensors as torch tensors. Recording the event puts every
    launch that the library still holds back on the stream, where torch's own
    work follows it; it waits for none of them."""
    record, event = state["event"]
    if record(event) != 0:
        raise RuntimeError("cannot record an event")

    def seen(t):
        v = torch.as_tensor(_Shared(t), device="cuda")
        return v.view(torch.bfloat16) if t.dtype == "bfloat16" else v

    return {n: [seen(t) for t in v] if isinstance(v, list) else seen(v) for n, v in tensors.items()}


def _blhd(case, t):
    """A held tensor as (batch, length, heads, features), the framework's or torch's."""
    if case["layout"] == "blhd":
        return t
    return t.transpose(1, 2) if isinstance(t, torch.Tensor) else t.transpose((0, 2, 1, 3))


def run(state):
    return (_RUN_OWN if own else _RUN)[state["case"]["kind"]](state["case"], state, **state["x"])


# ------------------------------------------------------ the framework's calls --
def _rotary_own(case, state, x, table, dy=None, positions=None):
    import ormi_amd

    y = ormi_amd.rotary(_blhd(case, x), table, positions=positions, offset=case["offset"] if positions is None else 0,
                        pairs=case["pairs"], dtype=case["out"])
    if not case["grad"]:
        return _hand_over(state, y=y.realize())
    x.zero_grad()
    total = (y * dy).sum()
    total.backward()
    gx = x.grad
    if case["layout"] == "bhld":
        gx = gx.transpose((0, 2, 1, 3))  # the order the kernel wrote, so that the memory is in the shape's order
    ormi_amd.realize_all(y, gx)
    total.zero_grad_graph()
    return _hand_over(state, y=y, gx=gx)


def _attention_own(case, state, q, k, v, dy=None, docs=None, prefix=None, lengths=None, slopes=None):
    import ormi_amd

    y = ormi_amd.attention(*(_blhd(case, t) for t in (q, k, v)), causal=case["causal"], cap=case["cap"], slopes=slopes,
                           documents=docs, prefix=prefix, lengths=lengths)
    if not case["grad"]:
        return _hand_over(state, y=y.realize())
    for t in (q, k, v):
        t.zero_grad()
    total = (y * dy).sum()
    total.backward()
    grads = [t.grad if case["layout"] == "blhd" else t.grad.transpose((0, 2, 1, 3)) for t in (q, k, v)]
    ormi_amd.realize_all(y, *grads)
    total.zero_grad_graph()
    return _hand_over(state, y=y, gq=grads[0], gk=grads[1], gv=grads[2])


def _adamw_own(case, state, p, g, s):
    import ormi_amd

    p, s = ormi_amd.adamw(p, g, s, step=case["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY)
    m, v = zip(*(t.values() for t in s))
    return _hand_over(state, p=p, m=list(m), v=list(v))


_RUN_OWN = {"rotary": _rotary_own, "attention": _attention_own, "adamw": _adamw_own}


# ------------------------------------------------------------- plain forms --
def _turn(case, x, cos, sin):
    """x's first features turned in pairs; cos and sin are (batch or 1, length, 1, pairs)."""
    part = case["part"]
    turned, rest = x[..., :part], x[..., part:]
    if case["pairs"] == "half":
        a, b = turned[..., : part // 2], turned[..., part // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), rest), -1)


def _rotary_plain(case, state, x, cos, sin, dy=None, positions=None):
    if positions is None:
        at = torch.arange(case["offset"], case["offset"] + case["length"], device="cuda")[None]
    else:
        at = positions.long()
    c, s = cos[at][:, :, None], sin[at][:, :, None]
    out = {"y": _turn(case, _blhd(case, x).float(), c, s).to(_type(case["out"]))}
    if case["grad"]:
        out["gx"] = _turn(case, dy.float(), c, -s).to(_type(case["dtype"]))
    return out


def _seen(case, docs, prefix, lengths):
    """Which keys each query sees, (batch or 1, 1, 1, queries, keys), and the signed distances."""
    lq, lk = case["queries"], case["keys"]
    i, j = torch.arange(lq, device="cuda")[:, None], torch.arange(lk, device="cuda")[None, :]
    end = torch.full((1, 1, 1), lk, device="cuda") if lengths is None else lengths.long()[:, None, None]
    at = i + end - lq  # the queries are the last of the sequence
    seen = j < end
    if case["causal"]:
        near = j <= at
        seen = seen & (near if prefix is None else near | (j < prefix[:, None, None]))
    if docs is not None:
        d = docs[:, lk - lq:, None]
        seen = seen & (d == docs[:, None, :]) & (d >= 0)
    return seen[:, None, None], (at - j)[:, None, None]


def _heads(case, t):
    """(batch, length, heads, features) as (batch, kv heads, group, length, features) in 32 bits."""
    b, l, h, d = t.shape
    return t.float().reshape(b, l, case["kv_heads"], h // case["kv_heads"], d).permute(0, 2, 3, 1, 4)


def _tokens(t):
    """_heads undone."""
    b, g, r, l, d = t.shape
    return t.permute(0, 3, 1, 2, 4).reshape(b, l, g * r, d)


def _attention_plain(case, state, q, k, v, dy=None, docs=None, prefix=None, lengths=None, slopes=None):
    q, k, v = (_heads(case, _blhd(case, t)) for t in (q, k, v))
    seen, away = _seen(case, docs, prefix, lengths)
    scale = 1 / math.sqrt(case["dim"])
    t = (q @ k.transpose(-1, -2)) * scale
    slope = None
    if case["cap"]:
        unit = torch.tanh(t / case["cap"])
        t = unit * case["cap"]
        slope = 1 - unit * unit
    if slopes is not None:
        t = t - slopes.reshape(1, case["kv_heads"], -1, 1, 1) * away.abs()
    t = t.masked_fill(~seen, -math.inf)
    top = t.amax(-1, keepdim=True)
    p = torch.exp(t - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    y = p @ v
    kept = _type(case["dtype"])
    out = {"y": _tokens(y).to(kept)}
    if case["grad"]:
        dy = _heads(case, dy)
        gv = p.transpose(-1, -2) @ dy
        dt = p * (dy @ v.transpose(-1, -2) - (dy * y).sum(-1, keepdim=True))
        if slope is not None:
            dt = dt * slope
        dt = dt * scale
        gq, gk = dt @ k, dt.transpose(-1, -2) @ q
        out["gq"], out["gk"], out["gv"] = _tokens(gq).to(kept), _tokens(gk.sum(2, keepdim=True)).to(kept), _tokens(gv.sum(2, keepdim=True)).to(kept)
    return out


def _codes_plain(x, top, root):
    """x (flat) as whole-number codes of its blocks' scale, and what they stand for:
    sign * (code / top)^root * scale, the scale the block's largest magnitude."""
    n = x.numel()
    blocks = torch.nn.functional.pad(x, (0, -n % BLOCK)).reshape(-1, BLOCK)
    scale = blocks.abs().amax(1, keepdim=True)
    unit = blocks.abs() / torch.where(scale == 0, 1.0, scale)
    unit = torch.sqrt(unit) if root == 2 else torch.sqrt(torch.sqrt(unit))
    code = torch.round(unit * top)
    if root == 4:  # a second moment never becomes zero: the step divides by its root
        code = torch.where(blocks > 0, code.clamp_min(1.0), code)
    return _decode_plain(code * torch.sign(blocks), scale, top, root).reshape(-1)[:n]


def _decode_plain(code, scale, top, root):
    w = code.abs() * (1.0 / top)
    w = w * w
    if root == 4:
        w = w * w
    return torch.sign(code) * (w * scale)


def _moment(case, state, top, root, shape):
    if case["bits"] == 32:
        return state
    code, scale = state
    return _decode_plain(code.float().reshape(-1, BLOCK), scale[:, None], top, root).reshape(-1)[: math.prod(shape)].reshape(shape)


def _adamw_plain(case, state, p, g, m, v):
    c1, c2 = 1 - BETA1 ** case["step"], 1 - BETA2 ** case["step"]
    out = {"p": [], "m": [], "v": []}
    for pi, gi, mi, vi in zip(p, g, m, v):
        pf, gf = pi.float(), gi.float()
        mi = _moment(case, mi, 127, 2, pi.shape) * BETA1 + gf * (1 - BETA1)
        vi = _moment(case, vi, 255, 4, pi.shape) * BETA2 + (gf * gf) * (1 - BETA2)
        step = (mi / c1) / (torch.sqrt(vi / c2) + EPS)
        out["p"].append((pf - LR * (step + DECAY * pf)).to(pi.dtype))
        if case["bits"] == 8:
            mi, vi = (_codes_plain(t.reshape(-1), top, root).reshape(pi.shape) for t, top, root in ((mi, 127, 2), (vi, 255, 4)))
        out["m"].append(mi)
        out["v"].append(vi)
    return out


_RUN = {"rotary": _rotary_plain, "attention": _attention_plain, "adamw": _adamw_plain}


# -------------------------------------------------------------------- work --
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def _pairs_seen(case):
    """Visible (query, key) pairs of one head over the batch, in the mean over the seeds' lengths, prefixes and documents."""
    b, lq, lk = case["batch"], case["queries"], case["keys"]
    end = (max(lq, lk // 4) + lk) / 2 if case["lengths"] else lk
    seen = lq * end
    if case["causal"]:
        seen -= lq * (lq - 1) / 2
    if case["prefix"]:  # a prefix of n adds n (n - 1) / 2 pairs; n is uniform up to half the keys
        top = lk // 2
        seen += top * top / 6 * min(1.0, lq / lk)
    if case["documents"]:  # sum of squares of random cuts
        seen *= 2 / (case["documents"] + 1)
    return b * seen, b * end


def work(case):
    """Bytes: each input read once and each output written once. Flops: the
    products over visible pairs (two forward, five more backward), and a few per element elsewhere."""
    if case["kind"] == "rotary":
        n = case["batch"] * case["length"] * case["heads"] * case["dim"]
        once = n * (_BYTES[case["dtype"]] + _BYTES[case["out"]])
        table = 4 * case["part"] * case["length"]
        return {"bytes": (once + table) * (2 if case["grad"] else 1), "flops": 3 * n * (2 if case["grad"] else 1)}
    if case["kind"] == "attention":
        size = _BYTES[case["dtype"]]
        pairs, keys = _pairs_seen(case)
        q = case["batch"] * case["queries"] * case["heads"] * case["dim"] * size
        kv = keys * case["kv_heads"] * case["dim"] * size
        if case["grad"]:
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * case["heads"] * case["dim"]}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * case["heads"] * case["dim"]}
    n = sum(math.prod(s) for s in _sizes(case))
    size = _BYTES[case["dtype"]]
    if case["bits"] == 32:
        return {"bytes": n * (3 * size + 16), "flops": 16 * n}
    return {"bytes": n * (3 * size + 4 + 8) + 16 * n // BLOCK, "flops": 40 * n}


# ------------------------------------------------------------------- exact --
def _exact_rotary(case, x):
    pos = x["positions"] if "positions" in x else (case["offset"] + np.arange(case["length"]))[None]
    turn = torch.from_numpy(np.exp(1j * (pos[..., None] * _frequencies(case)))).cuda()[:, :, None]

    def turned(t, by):
        t = t.double()
        part = t[..., : case["part"]]
        if case["pairs"] == "half":
            z = torch.complex(*part.chunk(2, -1)) * by
            z = torch.cat((z.real, z.imag), -1)
        else:
            z = torch.view_as_real(torch.complex(part[..., 0::2].contiguous(), part[..., 1::2].contiguous()) * by).flatten(-2)
        return torch.cat((z, t[..., case["part"]:]), -1)

    out = {"y": turned(_blhd(case, x["x"]), turn)}
    if case["grad"]:
        out["gx"] = turned(x["dy"], turn.conj())
    return out


def _exact_attention(case, x):
    """One head of one batch at a time, so that the scores in 64 bits stay small."""
    q, k, v = (_blhd(case, x[n]).double() for n in "qkv")
    lq, lk, group = case["queries"], case["keys"], case["heads"] // case["kv_heads"]
    y = torch.zeros_like(q)
    gq, gk, gv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    j = torch.arange(lk, device="cuda")
    for b in range(case["batch"]):
        end = int(x["lengths"][b]) if "lengths" in x else lk
        at = torch.arange(lq, device="cuda")[:, None] + (end - lq)
        hidden = (j >= end).expand(lq, lk)
        if case["causal"]:
            late = j > at
            hidden = hidden | (late & (j >= int(x["prefix"][b])) if "prefix" in x else late)
        if "docs" in x:
            d = torch.from_numpy(x["docs"][b]).cuda()
            hidden = hidden | (d[lk - lq:, None] != d) | (d < 0)
        blind = hidden.all(1)
        for h in range(case["heads"]):
            kh, vh = k[b, :, h // group], v[b, :, h // group]
            s = q[b, :, h] @ kh.T / math.sqrt(case["dim"])
            bent = torch.tanh(s / case["cap"]) if case["cap"] else None
            if bent is not None:
                s = bent * case["cap"]
            if "slopes" in x:
                s = s - float(x["slopes"][h]) * (at - j).abs()
            p = torch.softmax(s.masked_fill(hidden, -1e300), -1)
            p = p.masked_fill(hidden | blind[:, None], 0.0)
            y[b, :, h] = p @ vh
            if not case["grad"]:
                continue
            dy = x["dy"][b, :, h].double()
            gv[b, :, h // group] += p.T @ dy
            ds = dy @ vh.T
            ds = p * (ds - (p * ds).sum(1, keepdim=True)) / math.sqrt(case["dim"])
            if bent is not None:
                ds *= 1 - bent.square()
            gq[b, :, h] = ds @ kh
            gk[b, :, h // group] += ds.T @ q[b, :, h]
    return {"y": y, "gq": gq, "gk": gk, "gv": gv} if case["grad"] else {"y": y}


def _exact_adamw(case, x):
    """8-bit moments come back as None: a code is defined by the 32-bit value that it rounds."""
    out = {"p": [], "m": [], "v": []}
    t = case["step"]
    for p, g, m, v in zip(x["p"], x["g"], x["m"], x["v"]):
        n = p.numel()
        if case["bits"] == 8:
            m, v = ((c.double().sign() * (c.double().abs() / top) ** power * s.double().repeat_interleave(BLOCK))[:n].reshape(p.shape)
                    for (c, s), top, power in ((m, 127, 2), (v, 255, 4)))
        p, g, m, v = p.double(), g.double(), m.double(), v.double()
        m = m + (1 - BETA1) * (g - m)
        v = v + (1 - BETA2) * (g.square() - v)
        rate = m / (1 - BETA1 ** t) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        out["p"].append(p * (1 - LR * DECAY) - LR * rate)
        out["m"].append(m if case["bits"] == 32 else None)
        out["v"].append(v if case["bits"] == 32 else None)
    return out


_EXACT = {"rotary": _exact_rotary, "attention": _exact_attention, "adamw": _exact_adamw}


def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["kind"]](case, _inputs(case, seed))
