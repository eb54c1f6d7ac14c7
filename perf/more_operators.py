"""A recurrent block's operators as cases that can be timed and checked.

A case is a dict of plain values; prepare() builds what a program holds before
the call, run() is one pass, exact() the same outputs in 64 bits. Where `own`
is true run() calls the framework (tensors on the "hip" device); where it is
false it computes the same by elementary torch operations in 32 bits. Kinds:

  recurrence  h_t = a_t h_{t-1} + b_t per channel, with the gates as values
              (b = x) or as logits (a = sigmoid(g), b = (1 - a) x); the state
              carried in and out, restarts at documents, lengths of a padded
              batch; forward alone (one token among it) or with the gradients
  conv        a short causal convolution per channel, with or without the silu
              after it; the inputs carried in and out, documents, lengths;
              forward alone or with the gradients
  clip        the norm over a list of gradients: alone, with the clipped
              gradients, or with the AdamW step that they go into
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01


# ------------------------------------------------------------------ cases --
def _recurrence(name, batch, length, channels, gate, dtype, **more):
    case = {"kind": "recurrence", "batch": batch, "length": length, "channels": channels, "gate": gate, "dtype": dtype,
            "gate_dtype": dtype, "initial": False, "documents": 0, "lengths": False, "carry": False, "grad": False, **more}
    return {"name": name, **case} if name else case


def _conv(name, batch, length, channels, width, dtype, **more):
    case = {"kind": "conv", "batch": batch, "length": length, "channels": channels, "width": width, "dtype": dtype,
            "activation": "silu", "bias": True, "initial": False, "documents": 0, "lengths": False, "grad": False, **more}
    return {"name": name, **case} if name else case


def _clip(name, sizes, what, **more):
    case = {"kind": "clip", "sizes": sizes, "what": what, "dtype": "float32", "max_norm": 1.0, "step": 10, **more}
    return {"name": name, **case} if name else case


_NETWORK = "1024x4096,4096,4096x4096,4096,4096x1024,1024"


def listed():
    return [
        # Serving: one new token of eight requests, the state carried from token to token.
        _recurrence("recurrence_token", 8, 1, 2048, "logit", "bfloat16", initial=True, carry=True),
        # Serving: the prompts of a padded batch, the states at their ends kept for the tokens that follow.
        _recurrence("recurrence_prompts", 16, 1000, 1024, "logit", "float16", lengths=True, carry=True),
        # Training: a layer, forward and backward.
        _recurrence("recurrence_train", 8, 2048, 4096, "logit", "bfloat16", grad=True),
        # One long text: few channels, many tokens; gates that a float32 map made.
        _recurrence("recurrence_long", 1, 60001, 1024, "value", "bfloat16", gate_dtype="float32", carry=True),
        # Float32 training on packed documents, continued from a state, odd sizes.
        _recurrence("recurrence_documents", 2, 3001, 517, "value", "float32", initial=True, documents=9, carry=True, grad=True),
        # Serving: the convolution's one token, over the inputs carried from the tokens before.
        _conv("conv_token", 8, 1, 2048, 4, "bfloat16", initial=True),
        # Training: a layer, forward and backward.
        _conv("conv_train", 8, 2048, 4096, 4, "bfloat16", grad=True),
        # Packed documents in float32, odd sizes, without the activation.
        _conv("conv_documents", 1, 30011, 1001, 3, "float32", activation="none", documents=24, grad=True),
        # The norm of a small network's gradients, for a log: launches and host work are all of it.
        _clip("norm_small", "1024x72,72,72x72,72,72x40,40,513,1", "norm"),
        # Clipping the benchmark's 1024-4096-4096-1024 network's gradients.
        _clip("clip_network", _NETWORK, "clip"),
        # Seven layers of small 16-bit matrices and vectors: many tensors.
        _clip("clip_many_bf16", ",".join(["512x512,512,512x512,512,512x2048,2048,2048x512,512"] * 7), "clip", dtype="bfloat16"),
        # The network's clipped AdamW step.
        _clip("adamw_clipped", _NETWORK, "adamw"),
    ]


def _log(rng, lo, hi, step=1):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, step * round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)))


def draw(rng):
    kind = rng.choice(["recurrence", "recurrence", "conv", "clip"])
    if kind == "clip":
        dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
        what = rng.choice(["norm", "clip", "clip", "adamw"])
        count = rng.choice([1, 3, 10, {"norm": 300, "clip": 60, "adamw": 20}[what]])
        sizes = ",".join(rng.choice(["%d", "%dx1"]) % _log(rng, 1, 1 << 20) for _ in range(count))
        return _clip(None, sizes, what, dtype=dtype, max_norm=rng.choice([0.1, 1.0, 1e4]), step=rng.randint(1, 1000))
    batch, channels = _log(rng, 1, 16), _log(rng, 8, 4096, rng.choice([1, 8, 64]))
    length = rng.choice([_log(rng, 1, 8), _log(rng, 8, min(65536, max(9, (1 << 25) // (batch * channels))))])
    masks = rng.choice([{}, {}, {"documents": rng.choice([1, 4, 16])}, {"lengths": True}])
    more = {"initial": rng.random() < 0.5, "grad": rng.random() < 0.6, **masks}
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    if kind == "conv":
        return _conv(None, batch, length, channels, rng.randint(1, 8), dtype, activation=rng.choice(["silu", "none"]),
                     bias=rng.random() < 0.7, **more)
    return _recurrence(None, batch, length, channels, rng.choice(["value", "logit"]), dtype,
                       gate_dtype=rng.choice([dtype, "float32"]), carry=rng.random() < 0.5, **more)


# ------------------------------------------------------------------ inputs --
def _type(name):
    return getattr(torch, name)


def _sizes(case):
    return [tuple(int(n) for n in s.split("x")) for s in case["sizes"].split(",")]


def _inputs(case, seed):
    """The case's inputs: torch tensors on the GPU of the case's types, and host arrays of its integers."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))

    def normal(shape, dtype, scale=1.0, mean=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale + mean).to(_type(dtype))

    if case["kind"] == "clip":
        x = {"g": [normal(s, case["dtype"], 0.01) for s in _sizes(case)]}
        if case["what"] == "adamw":
            x["p"] = [normal(s, case["dtype"], 0.05) for s in _sizes(case)]
            x["m"] = [normal(s, "float32", 3e-4) for s in _sizes(case)]
            x["v"] = [normal(s, "float32", 1e-3).square() for s in _sizes(case)]
        return x
    b, l, c = case["batch"], case["length"], case["channels"]
    x = {"x": normal((b, l, c), case["dtype"])}
    if case["documents"]:  # documents of unequal length one after the other, then in every other row up to 31 tokens of padding
        docs = np.zeros((b, l), np.int32)
        for i in range(b):
            cuts = np.sort(rng.integers(0, l, case["documents"] - 1))
            docs[i] = np.searchsorted(cuts, np.arange(l), side="right")
            if i % 2 == 0:
                docs[i, l - int(rng.integers(0, min(32, l))):] = -1
        x["documents"] = docs
    if case["lengths"]:
        x["lengths"] = rng.integers(l // 4, l + 1, b).astype(np.int32)
    if case["kind"] == "conv":
        w = case["width"]
        x["weight"] = normal((c, w), "float32", 1 / math.sqrt(w))
        if case["bias"]:
            x["bias"] = normal((c,), "float32", 0.1)
        if case["initial"]:
            x["initial"] = normal((b, w - 1, c), case["dtype"])
        if case["grad"]:
            x["dy"] = normal((b, l, c), case["dtype"])
        return x
    if case["gate"] == "logit":  # states that remember for some tens of tokens
        x["gates"] = normal((b, l, c), case["gate_dtype"], 1.0, 3.0)
    else:  # for 10 to 1000 tokens, the inputs scaled so that states have the inputs' size
        forget = torch.exp(torch.rand((b, l, c), generator=gen, device="cuda") * math.log(100) + math.log(1e-3))
        x["gates"] = (1 - forget).to(_type(case["gate_dtype"]))
        x["x"] = (x["x"].float() * torch.sqrt(2 * forget)).to(_type(case["dtype"]))
    if case["initial"]:
        x["initial"] = normal((b, c), "float32")
    if case["grad"]:
        x["dy"] = normal((b, l, c), case["dtype"])
        if case["carry"]:
            x["dlast"] = normal((b, c), "float32")
    return x


_LEARNED = ("gates", "x", "initial", "weight", "bias")  # inputs with a gradient, in the order of the outputs


def prepare(case, seed):
    x = _inputs(case, seed)
    if not own:
        for n in ("documents", "lengths"):
            if n in x:
                x[n] = torch.from_numpy(x[n]).cuda()
        return {"case": dict(case), "x": x}
    import ormi_amd

    def leaf(t, grad=False):
        """The same values as a leaf of the framework."""
        if isinstance(t, np.ndarray):
            return ormi_amd.Tensor(t, "hip", dtype=str(t.dtype))
        kept = str(t.dtype).replace("torch.", "")
        return ormi_amd.Tensor(t.float().cpu().numpy(), "hip", requires_grad=grad, dtype=kept)

    if case["kind"] == "clip":
        out = {n: [leaf(t) for t in x[n]] for n in ("g", "p") if n in x}
        if case["what"] == "adamw":
            out["s"] = [ormi_amd.AdamState(leaf(m), leaf(v)) for m, v in zip(x["m"], x["v"])]
    else:
        out = {n: leaf(t, grad=case["grad"] and n in _LEARNED) for n, t in x.items()}
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
        if 0 in t.shape:
            return torch.empty(t.shape, dtype=_type(t.dtype), device="cuda")
        v = torch.as_tensor(_Shared(t), device="cuda")
        return v.view(torch.bfloat16) if t.dtype == "bfloat16" else v

    return {n: [seen(t) for t in v] if isinstance(v, list) else seen(v) for n, v in tensors.items()}


def run(state):
    return (_RUN_OWN if own else _RUN)[state["case"]["kind"]](state["case"], state, **state["x"])


# ------------------------------------------------------ the framework's calls --
def _sequence_own(case, state, y, last, learned, dy, dlast):
    """The results, and with a gradient the learned inputs' gradients."""
    import ormi_amd

    if not case["grad"]:
        ormi_amd.realize_all(y, last)
        return _hand_over(state, y=y, last=last)
    for t in learned.values():
        t.zero_grad()
    total = (y * dy).sum()
    if dlast is not None:
        total = total + (last * dlast).sum()
    total.backward()
    grads = {"g_" + n: t.grad for n, t in learned.items()}
    ormi_amd.realize_all(y, last, *grads.values())
    total.zero_grad_graph()
    return _hand_over(state, y=y, last=last, **grads)


def _recurrence_own(case, state, gates, x, initial=None, documents=None, lengths=None, dy=None, dlast=None):
    import ormi_amd

    y, last = ormi_amd.linear_recurrence(gates, x, initial, gate=case["gate"], documents=documents, lengths=lengths)
    learned = {"gates": gates, "x": x, **({"initial": initial} if initial is not None else {})}
    return _sequence_own(case, state, y, last, learned, dy, dlast)


def _conv_own(case, state, x, weight, bias=None, initial=None, documents=None, lengths=None, dy=None):
    import ormi_amd

    y, last = ormi_amd.causal_conv(x, weight, bias, initial, activation=None if case["activation"] == "none" else case["activation"],
                                   documents=documents, lengths=lengths)
    learned = {"x": x, "weight": weight, **({"bias": bias} if bias is not None else {}), **({"initial": initial} if initial is not None else {})}
    return _sequence_own(case, state, y, last, learned, dy, None)


def _clip_own(case, state, g, p=None, s=None):
    import ormi_amd

    if case["what"] == "norm":
        return _hand_over(state, norm=ormi_amd.grad_norm(g))
    if case["what"] == "clip":
        clipped, norm = ormi_amd.clip_grads(g, case["max_norm"])
        return _hand_over(state, g=clipped, norm=norm)
    p, s = ormi_amd.adamw(p, g, s, step=case["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, max_norm=case["max_norm"])
    m, v = zip(*(t.values() for t in s))
    return _hand_over(state, p=p, m=list(m), v=list(v))


_RUN_OWN = {"recurrence": _recurrence_own, "conv": _conv_own, "clip": _clip_own}


# ------------------------------------------------------------- plain forms --
def _live(case, documents, lengths):
    """Which tokens count, which of them start from nothing, and each one's run of
    one document, (batch or 1, length, 1) each. The first token continues what came before."""
    l = case["length"]
    t = torch.arange(l, device="cuda")
    counts = torch.ones((1, l), dtype=torch.bool, device="cuda")
    runs = torch.zeros((1, l), dtype=torch.long, device="cuda")
    if lengths is not None:
        counts = t < lengths.long()[:, None]
    if documents is not None:
        counts = counts & (documents >= 0)
        runs = torch.cumsum(torch.nn.functional.pad((documents[:, 1:] != documents[:, :-1]).long(), (1, 0)), 1)
    starts = torch.nn.functional.pad(runs[:, 1:] != runs[:, :-1], (1, 0))
    return counts[..., None], starts[..., None], runs[..., None]


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 with h_{-1} = 0, by doubling spans."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat((b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]), 1)
        if 2 * step < a.shape[1]:
            a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return b


def _recurrence_plain(case, state, gates, x, initial=None, documents=None, lengths=None, dy=None, dlast=None):
    counts, starts, _ = _live(case, documents, lengths)
    dead = counts.logical_not() if documents is not None and lengths is None else torch.zeros_like(counts)  # its state is zero
    g, x = gates.float(), x.float()
    keep = torch.sigmoid(g) if case["gate"] == "logit" else g
    take = torch.sigmoid(-g) if case["gate"] == "logit" else None
    b = x * take if take is not None else x
    a = torch.where(counts, torch.where(starts, 0.0, keep), torch.where(dead, 0.0, 1.0))
    b = torch.where(counts, b, 0.0)
    first = torch.zeros_like(b[:, :1]) if initial is None else initial[:, None]
    h = _scan(a, torch.cat((b[:, :1] + a[:, :1] * first, b[:, 1:]), 1))
    out = {"y": torch.where(counts, h, 0.0).to(_type(case["dtype"])), "last": h[:, -1]}
    if not case["grad"]:
        return out
    before = torch.cat((first, h[:, :-1]), 1)
    d = torch.where(counts, dy.float(), 0.0)
    if dlast is not None:
        d = torch.cat((d[:, :-1], d[:, -1:] + dlast[:, None]), 1)
    after = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), 1)  # what a token's state passes on
    l = _scan(after.flip(1), d.flip(1)).flip(1)
    dx = l * take if take is not None else l
    part = torch.where(starts, 0.0, before)
    dg = l * (part - x) * keep * take if take is not None else l * part
    out["g_gates"] = torch.where(counts, dg, 0.0).to(_type(case["gate_dtype"]))
    out["g_x"] = torch.where(counts, dx, 0.0).to(_type(case["dtype"]))
    if initial is not None:
        out["g_initial"] = a[:, 0] * l[:, 0]
    return out


def _conv_plain(case, state, x, weight, bias=None, initial=None, documents=None, lengths=None, dy=None):
    w, l, kept = case["width"], case["length"], _type(case["dtype"])
    counts, _, runs = _live(case, documents, lengths)
    rows = torch.nn.functional.pad(x.float(), (0, 0, w - 1, 0)) if initial is None else torch.cat((initial, x), 1).float()
    runs = torch.cat((runs[:, :1].expand(-1, w - 1, -1), runs), 1)
    taps = [torch.where(counts & (runs[:, j:j + l] == runs[:, w - 1:]), rows[:, j:j + l], 0.0) for j in range(w)]
    z = sum(t * weight[:, j] for j, t in enumerate(taps))
    if bias is not None:
        z = z + bias
    s = torch.sigmoid(z)
    y = z * s if case["activation"] == "silu" else z
    # The inputs that the next token's taps read: the last ones that count, of the last one's document.
    end = torch.full((x.shape[0],), l, device="cuda") if lengths is None else lengths.long()
    at = end[:, None] + torch.arange(w - 1, device="cuda")  # of rows
    of = runs.expand(x.shape[0], -1, -1)[..., 0]
    alive = torch.gather(of, 1, at) == torch.gather(of, 1, (end + w - 2).clamp_min(0)[:, None])
    if documents is not None:
        alive = alive & (documents[torch.arange(x.shape[0], device="cuda"), end - 1] >= 0)[:, None]
    last = torch.where(alive[..., None], torch.gather(rows, 1, at[..., None].expand(-1, -1, x.shape[2])), 0.0)
    out = {"y": torch.where(counts, y, 0.0).to(kept), "last": last.to(kept)}
    if not case["grad"]:
        return out
    dz = dy.float()
    if case["activation"] == "silu":
        dz = dz * (s * (1 + z * (1 - s)))
    dz = torch.where(counts, dz, 0.0)
    drows = torch.zeros_like(rows)
    for j in range(w):
        drows[:, j:j + l] += torch.where(runs[:, j:j + l] == runs[:, w - 1:], dz * weight[:, j], 0.0)
    out["g_x"] = drows[:, w - 1:].to(kept)
    out["g_weight"] = torch.stack([(dz * t).sum((0, 1), dtype=torch.float64) for t in taps], 1).float()
    if bias is not None:
        out["g_bias"] = dz.sum((0, 1), dtype=torch.float64).float()
    if initial is not None:
        out["g_initial"] = drows[:, :w - 1].to(kept)
    return out


def _clip_plain(case, state, g, p=None, m=None, v=None):
    norm = torch.sqrt(sum(t.double().square().sum() for t in g))
    if case["what"] == "norm":
        return {"norm": norm.float()}
    factor = torch.clamp(case["max_norm"] / norm, max=1.0).float()
    if case["what"] == "clip":
        return {"g": [(t.float() * factor).to(t.dtype) for t in g], "norm": norm.float()}
    c1, c2 = 1 - BETA1 ** case["step"], 1 - BETA2 ** case["step"]
    out = {"p": [], "m": [], "v": []}
    for pi, gi, mi, vi in zip(p, g, m, v):
        pf, gf = pi.float(), gi.float() * factor
        mi = mi * BETA1 + gf * (1 - BETA1)
        vi = vi * BETA2 + (gf * gf) * (1 - BETA2)
        step = (mi / c1) / (torch.sqrt(vi / c2) + EPS)
        out["p"].append((pf - LR * (step + DECAY * pf)).to(pi.dtype))
        out["m"].append(mi)
        out["v"].append(vi)
    return out


_RUN = {"recurrence": _recurrence_plain, "conv": _conv_plain, "clip": _clip_plain}


# -------------------------------------------------------------------- work --
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def work(case):
    """Bytes: each input read once and each output written once. Flops: those of
    the formulas per token and channel, or per parameter."""
    if case["kind"] == "clip":
        n, size = sum(math.prod(s) for s in _sizes(case)), _BYTES[case["dtype"]]
        if case["what"] == "adamw":
            return {"bytes": n * (3 * size + 16), "flops": 19 * n}
        return {"bytes": n * size * (2 if case["what"] == "clip" else 1), "flops": (3 if case["what"] == "clip" else 2) * n}
    n, size = case["batch"] * case["length"] * case["channels"], _BYTES[case["dtype"]]
    if case["lengths"]:  # inputs past a length need not be read; outputs are there
        n = n * 0.8125
    if case["kind"] == "conv":
        return {"bytes": n * size * (4 if case["grad"] else 2), "flops": n * case["width"] * (6 if case["grad"] else 2)}
    gate = _BYTES[case["gate_dtype"]]
    flops = 10 if case["gate"] == "logit" else 2
    return {"bytes": n * (2 * gate + 4 * size if case["grad"] else gate + 2 * size), "flops": n * flops * (3 if case["grad"] else 1)}


# ------------------------------------------------------------------- exact --
def _exact_recurrence(case, x):
    """Token after token, then back."""
    b, l, c = x["x"].shape
    docs, ends = x.get("documents"), x.get("lengths")
    h = x["initial"].double() if "initial" in x else torch.zeros((b, c), dtype=torch.float64, device="cuda")
    logit = case["gate"] == "logit"

    def rule(t):
        """Of token t: who counts, who starts from nothing (also: what does not count and forgets), None where all are alike."""
        if docs is not None:
            dead = docs[:, t] < 0
            return [torch.from_numpy(r).cuda()[:, None] for r in (~dead, dead | (docs[:, t] != docs[:, t - 1] if t else False), ~dead)]
        if ends is not None:
            on = torch.from_numpy(t < ends).cuda()[:, None]
            return on, torch.zeros_like(on), on
        return None

    rules = [rule(t) for t in range(l)]
    states = []
    y = torch.empty((b, l, c), dtype=torch.float64, device="cuda")
    for t in range(l):
        if case["grad"]:
            states.append(h)
        g, v = x["gates"][:, t].double(), x["x"][:, t].double()
        a = 1 / (1 + torch.exp(-g)) if logit else g
        v = v / (1 + torch.exp(g)) if logit else v
        if rules[t] is None:
            h = a * h + v
            y[:, t] = h
        else:
            on, cut, _ = rules[t]
            h = torch.where(cut, 0, torch.where(on, a, 1)) * h + torch.where(on, v, 0)
            y[:, t] = torch.where(on, h, 0)
    out = {"y": y, "last": h}
    if not case["grad"]:
        return out
    m = x["dlast"].double() if "dlast" in x else torch.zeros_like(h)  # the gradient of the state that a token leaves, but for its own output
    dg, dx = torch.empty_like(y), torch.empty_like(y)
    for t in range(l - 1, -1, -1):
        g, v = x["gates"][:, t].double(), x["x"][:, t].double()
        d, before = x["dy"][:, t].double(), states.pop()
        on = cut = None
        if rules[t] is not None:
            on, cut, _ = rules[t]
            d, before = torch.where(on, d, 0), torch.where(cut, 0, before)
        s = m + d
        a = 1 / (1 + torch.exp(-g)) if logit else g
        if logit:
            forget = 1 / (1 + torch.exp(g))
            dgt, dxt = s * (before - v) * a * forget, s * forget
        else:
            dgt, dxt = s * before, s
        if on is None:
            m = a * s
        else:
            dgt, dxt = torch.where(on, dgt, 0), torch.where(on, dxt, 0)
            m = torch.where(cut, 0, torch.where(on, a * s, s))
        dg[:, t], dx[:, t] = dgt, dxt
    out["g_gates"], out["g_x"] = dg, dx
    if "initial" in x:
        out["g_initial"] = m
    return out


def _exact_conv(case, x):
    """A batch's document run after the other: each is a convolution of its own, with nothing before it (or the inputs carried in)."""
    w, silu = case["width"], case["activation"] == "silu"
    weight = x["weight"].double()
    bias = x["bias"].double() if "bias" in x else torch.zeros_like(weight[:, 0])
    b, l, c = x["x"].shape
    zeros = lambda *s: torch.zeros(s, dtype=torch.float64, device="cuda")  # noqa: E731
    y, last, dx, di = zeros(b, l, c), zeros(b, w - 1, c), zeros(b, l, c), zeros(b, w - 1, c)
    dw, db = torch.zeros_like(weight), torch.zeros_like(bias)
    for i in range(b):
        end = int(x["lengths"][i]) if "lengths" in x else l
        docs = x["documents"][i] if "documents" in x else np.zeros(l, np.int32)
        edges = [0] + [t for t in range(1, end) if docs[t] != docs[t - 1]] + [end]
        for k, (lo, hi) in enumerate(zip(edges, edges[1:])):
            final = hi == end
            if hi > lo and docs[lo] < 0:
                continue
            head = x["initial"][i].double() if k == 0 and "initial" in x else zeros(w - 1, c)
            rows = torch.cat((head, x["x"][i, lo:hi].double()))
            if final:
                last[i] = rows[rows.shape[0] - (w - 1):] if w > 1 else last[i]
            if hi == lo:
                continue
            views = rows.unfold(0, w, 1)  # (tokens, channels, width)
            z = (views * weight).sum(-1) + bias
            y[i, lo:hi] = z / (1 + torch.exp(-z)) if silu else z
            if not case["grad"]:
                continue
            d = x["dy"][i, lo:hi].double()
            if silu:
                e = torch.exp(-z)
                d = d * (1 + e + z * e) / (1 + e).square()
            dw += (views * d[..., None]).sum(0)
            db += d.sum(0)
            back = torch.cat((zeros(w - 1, c), d, zeros(w - 1, c))).unfold(0, w, 1)  # the outputs that a row reaches
            drows = (back * weight.flip(1)).sum(-1)
            dx[i, lo:hi] = drows[w - 1:]
            if k == 0:
                di[i] = drows[:w - 1]
    out = {"y": y, "last": last}
    if case["grad"]:
        out.update(g_x=dx, g_weight=dw)
        if "bias" in x:
            out["g_bias"] = db
        if "initial" in x:
            out["g_initial"] = di
    return out


def _exact_clip(case, x):
    total = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(t.double()) for t in x["g"]]))
    if case["what"] == "norm":
        return {"norm": total}
    factor = min(1.0, case["max_norm"] / float(total))
    if case["what"] == "clip":
        return {"g": [t.double() * factor for t in x["g"]], "norm": total}
    out = {"p": [], "m": [], "v": []}
    t = case["step"]
    for p, g, m, v in zip(x["p"], x["g"], x["m"], x["v"]):
        p, g, m, v = p.double(), g.double() * factor, m.double(), v.double()
        m = m + (1 - BETA1) * (g - m)
        v = v + (1 - BETA2) * (g.square() - v)
        rate = m / (1 - BETA1 ** t) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        out["p"].append(p * (1 - LR * DECAY) - LR * rate)
        out["m"].append(m)
        out["v"].append(v)
    return out


_EXACT = {"recurrence": _exact_recurrence, "conv": _exact_conv, "clip": _exact_clip}


def exact(case, seed):
    if case["kind"] == "recurrence" and case["length"] * (3 if case["grad"] else 1) > 100000:
        return None  # token by token this takes too long
    with torch.no_grad():
        return _EXACT[case["kind"]](case, _inputs(case, seed))
