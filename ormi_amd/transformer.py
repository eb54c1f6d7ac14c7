"""What a transformer block needs beside products and maps: rotary positions,
masked softmax attention, and the AdamW step over a list of tensors with the
norm over their gradients.

    table = RotaryTable(head_dim, positions)
    q = rotary(x.reshape((batch, length, heads, head_dim)), table, dtype="bfloat16")
    y = attention(q, k, v, causal=True)          # differentiable, lazy like every op
    optimizer = AdamW(parameters, lr=3e-4)       # loss.backward(); optimizer.step(); loss.zero_grad_graph()

Additive to the reference's Python surface (ormi-core/src/ormi_core/tensor.py:10-190),
which has none of them.
"""
from __future__ import annotations

import math

import numpy as np

from ._ext import ormi_backend
from .exceptions import raise_device_mismatch
from .tensor import Tensor, _parse_device

_BLOCK = 256  # elements that share a scale in 8-bit moments


def _node(t, like: Tensor, what: str):
    """The node of an optional operand: a Tensor on the same device, or None."""
    if t is None:
        return None
    if not isinstance(t, Tensor):
        raise TypeError(f"{what} must be a Tensor.")
    if t.device is not like.device and t.device.type != like.device.type:
        raise_device_mismatch(msg=f"{what} is on another device.", got=t.device.type)
    return t._node


# ------------------------------------------------------------------ rotary --
class RotaryTable:
    """Cosines and sines of every position's angles, computed once in 64 bits.

    part: features turned (even); pair p turns by base^(-2 p / part) radians per
    position. For contexts longer than a model was trained on:
      scaling="linear"  every angle is divided by factor
      scaling="base"    the base grows so that the slowest pair is slowed by
                        factor and the fastest is not
      scaling="parts"   pairs that turn over `fast` times within `original`
                        positions stay, those under `slow` times are slowed by
                        factor, those between in proportion
    magnitude multiplies both tables (a temperature of the scores it leads to).
    """

    def __init__(self, part: int, positions: int, device="hip", *, base: float = 10000.0, scaling: str = "none",
                 factor: float = 1.0, original: int | None = None, slow: float = 1.0, fast: float = 32.0,
                 magnitude: float = 1.0):
        if part < 0 or part % 2:
            raise ValueError("part must be even and not negative.")
        if positions < 0:
            raise ValueError("positions must not be negative.")
        if not base > 0 or not factor > 0:
            raise ValueError("base and factor must be positive.")
        if scaling not in ("none", "linear", "base", "parts"):
            raise ValueError("scaling must be none, linear, base or parts.")
        if scaling == "base" and part > 2:
            base = base * factor ** (part / (part - 2))
        turn = base ** (-np.arange(0, part, 2, dtype=np.float64) / max(part, 1))
        if scaling == "linear":
            turn = turn / factor
        elif scaling == "parts":
            if original is None or original < 1 or not fast > slow:
                raise ValueError("scaling by parts needs original >= 1 and fast > slow.")
            keep = np.clip((original * turn / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
            turn = turn * (keep + (1.0 - keep) / factor)
        angle = np.outer(np.arange(positions, dtype=np.float64), turn)
        self.part, self.positions = part, positions
        self.cos = Tensor((np.cos(angle) * magnitude).astype(np.float32), device)
        self.sin = Tensor((np.sin(angle) * magnitude).astype(np.float32), device)


def rotary(x: Tensor, table: RotaryTable, positions: Tensor | None = None, *, offset: int = 0, pairs: str = "half",
           dtype: str | None = None) -> Tensor:
    """x (batch, length, heads, features) with each token's first table.part features turned by its position.

    positions: int32 (length,) or (batch, length); without it token l stands at
    offset + l. A position outside the table makes its token's turned features
    NaN. pairs: "half" turns feature p with p + part / 2, "interleaved" 2 p with
    2 p + 1. dtype: the result's type (x's); one rounding, from float32.
    """
    if pairs not in ("half", "interleaved"):
        raise ValueError("pairs must be half or interleaved.")
    if positions is not None and offset:
        raise ValueError("give positions or an offset, not both.")
    node = ormi_backend.rotary(x._node, _node(table.cos, x, "The table"), _node(table.sin, x, "The table"),
                               _node(positions, x, "positions"), offset, pairs == "interleaved", dtype or x.dtype)
    return Tensor._wrap(node, x.device)


# --------------------------------------------------------------- attention --
def attention(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = False, scale: float | None = None, cap: float = 0.0,
              slopes: Tensor | None = None, documents: Tensor | None = None, prefix: Tensor | None = None,
              lengths: Tensor | None = None) -> Tensor:
    """Softmax attention of q (batch, queries, heads, features) over k and v (batch, keys, kv heads, features).

    Query head h reads key head h // (heads // kv heads). The queries are the
    last of their sequence: query i stands at position length - queries + i.
      scale      of the scores (1 / sqrt(features))
      cap        scores t become cap tanh(t / cap); 0: not capped
      slopes     float32 (heads,): scores lose slope times the distance
      causal     a query sees keys up to its position
      prefix     int32 (batch,): and, causal, every key before the prefix's end
      documents  int32 (batch, keys): tokens see their own document's; a
                 negative one sees nothing and is seen by nothing
      lengths    int32 (batch,): keys that exist (keys); the others do not count, whatever they hold
    A query that sees no key gives zeros. The result and the gradients have q's
    type (float32, bfloat16 or float16); gradients of shared key heads add up.
    Scores and sums are float32. In the 16-bit types the gradient that comes in is
    rounded to the type, and so are weights and score gradients for their products.
    """
    for t, what in ((k, "k"), (v, "v")):
        _node(t, q, what)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.shape and q.shape[-1] else 1.0
    node = ormi_backend.attention(q._node, k._node, v._node, scale, cap, causal, _node(slopes, q, "slopes"),
                                  _node(documents, q, "documents"), _node(prefix, q, "prefix"), _node(lengths, q, "lengths"))
    return Tensor._wrap(node, q.device)


# ------------------------------------------------------------------- AdamW --
class AdamState:
    """A parameter's two moments in float32."""

    bits = 32
    __slots__ = ("m", "v")

    def __init__(self, m: Tensor, v: Tensor):
        self.m, self.v = m, v

    @classmethod
    def zeros(cls, shape, device="hip") -> "AdamState":
        return cls(Tensor(np.zeros(shape, np.float32), device), Tensor(np.zeros(shape, np.float32), device))

    def values(self):
        """The moments as float32 tensors."""
        return self.m, self.v

    def _nodes(self):
        return [self.m._node, self.v._node]

    @classmethod
    def _from(cls, nodes, shape, device):
        return cls(*(Tensor._wrap(n, device) for n in nodes))


class AdamState8:
    """A parameter's two moments in 8 bits: codes in blocks of 256 elements that
    share a scale, the block's largest magnitude. The first moment is
    sign(c) (|c| / 127)^2 scale, the second (c / 255)^4 scale."""

    bits = 8
    __slots__ = ("shape", "parts")

    def __init__(self, shape, parts):
        self.shape, self.parts = tuple(shape), tuple(parts)

    @classmethod
    def zeros(cls, shape, device="hip") -> "AdamState8":
        blocks = -(-math.prod(shape) // _BLOCK)
        return cls.from_codes(shape, np.zeros(blocks * _BLOCK, np.int8), np.zeros(blocks, np.float32),
                              np.zeros(blocks * _BLOCK, np.uint8), np.zeros(blocks, np.float32), device)

    @classmethod
    def from_codes(cls, shape, m_codes, m_scales, v_codes, v_scales, device="hip") -> "AdamState8":
        """From host arrays: int8 and uint8 codes, padded to whole blocks, and float32 scales."""
        blocks = -(-math.prod(shape) // _BLOCK)

        def words(codes, kind):
            codes = np.ascontiguousarray(codes)
            if codes.dtype != kind or codes.size != blocks * _BLOCK:
                raise ValueError(f"codes must be {np.dtype(kind).name}, a whole number of blocks of {_BLOCK}.")
            return Tensor(codes.reshape(-1).view(np.int32), device, dtype="int32")

        def scales(s):
            s = np.ascontiguousarray(s, dtype=np.float32).reshape(-1)
            if s.size != blocks:
                raise ValueError("one scale for each block.")
            return Tensor(s, device)

        return cls(shape, (words(m_codes, np.int8), scales(m_scales), words(v_codes, np.uint8), scales(v_scales)))

    def values(self):
        """The moments that the codes stand for, as float32 tensors."""
        m, v = ormi_backend.adamw_values(self._nodes(), list(self.shape))
        return Tensor._wrap(m, self.parts[0].device), Tensor._wrap(v, self.parts[0].device)

    def _nodes(self):
        return [p._node for p in self.parts]

    @classmethod
    def _from(cls, nodes, shape, device):
        return cls(shape, (Tensor._wrap(n, device) for n in nodes))


def adamw(params, grads, states, *, step: int, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
          weight_decay: float = 0.01, max_norm: float | None = None):
    """One AdamW step over lists of tensors: (new parameters, new states).

    Runs at once (the gradients are realized together), as few launches for
    however many tensors. states: AdamState or AdamState8, one kind per call.
    step counts from 1. What was passed in keeps its values. With max_norm the
    gradients count times min(1, max_norm / grad_norm(grads)), as clip_grads would
    give them but for its rounding of 16-bit ones.
      m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
      p = p - lr ((m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps) + weight_decay p)
    in float32; a 16-bit parameter is rounded to its type once.
    """
    params, grads, states = list(params), list(grads), list(states)
    if any(not isinstance(t, Tensor) for t in params + grads):
        raise TypeError("params and grads must be Tensors.")
    factor = None if max_norm is None else _norm_and_factor(grads, max_norm)[1]
    return _adamw(params, grads, states, step, lr, betas, eps, weight_decay, factor)


def _adamw(params, grads, states, step, lr, betas, eps, weight_decay, factor):
    kinds = {type(s) for s in states}
    if not kinds <= {AdamState, AdamState8} or len(kinds) > 1:
        raise TypeError("states must be all AdamState or all AdamState8.")
    kind = kinds.pop() if kinds else AdamState
    p, s = ormi_backend.adamw([t._node for t in params], [t._node for t in grads], [t._nodes() for t in states], kind.bits, step, lr,
                              betas[0], betas[1], eps, weight_decay, factor)
    return ([Tensor._wrap(n, t.device) for n, t in zip(p, params)],
            [kind._from(n, t.shape, t.device) for n, t in zip(s, params)])


def _check_max_norm(max_norm: float) -> None:
    if not max_norm >= 0:
        raise ValueError("max_norm must not be negative.")


def _norm_and_factor(grads, max_norm: float):
    """The nodes of the norm and of min(1, max_norm / norm)."""
    _check_max_norm(max_norm)
    return ormi_backend.grad_norm([t._node for t in grads], max_norm)


def _grads(grads):
    grads = list(grads)
    if any(not isinstance(t, Tensor) for t in grads):
        raise TypeError("grads must be Tensors.")
    return grads


def grad_norm(grads) -> Tensor:
    """The square root of the sum of all elements' squares, a float32 scalar on the device.

    Runs at once (the gradients are realized together). Squares are added in 64
    bits, in a fixed order. No gradients: 0.
    """
    grads = _grads(grads)
    node = ormi_backend.grad_norm([t._node for t in grads], math.inf)[0]
    return Tensor._wrap(node, grads[0].device if grads else _parse_device("hip"))


def clip_grads(grads, max_norm: float):
    """(the gradients times min(1, max_norm / norm), norm), norm that of grad_norm.

    Nothing waits for the device: the factor stays there. Each product is rounded
    once to its gradient's type. A norm that is NaN makes every element NaN, an
    infinite one makes finite elements 0 and the others NaN (max_norm=inf leaves
    them as they are).
    """
    grads = _grads(grads)
    _check_max_norm(max_norm)
    nodes, norm = ormi_backend.clip_grads([t._node for t in grads], max_norm)
    return [Tensor._wrap(n, t.device) for n, t in zip(nodes, grads)], Tensor._wrap(norm, grads[0].device if grads else _parse_device("hip"))


class AdamW:
    """Keeps the moments of a list of parameters and steps them by their gradients.

        loss.backward()
        optimizer.step()
        loss.zero_grad_graph()

    step() gives each parameter with a gradient a new value: the Tensor object
    stays, its node is a new leaf without a gradient, so a graph that read the
    old one keeps its values. The old leaf's gradient is let go of; those of the
    nodes between point back at what they were computed from, and a loop that
    does not release them with zero_grad_graph keeps every step's graph in
    memory. state_bits: 32, or 8 for moments of a quarter of the size. max_norm:
    the gradients of a step count times min(1, max_norm / norm), norm being theirs
    taken together; self.norm then holds the last step's, on the device.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32, max_norm: float | None = None):
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8.")
        if max_norm is not None:
            _check_max_norm(max_norm)
        self.params = list(params)
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.max_norm, self.norm = max_norm, None
        kind = AdamState if state_bits == 32 else AdamState8
        self.states = [kind.zeros(p.shape, p.device) for p in self.params]
        self.steps = [0] * len(self.params)

    def step(self) -> None:
        by_step: dict = {}
        for i, p in enumerate(self.params):
            if p.grad is not None:
                by_step.setdefault(self.steps[i] + 1, []).append(i)
        factor = None
        if self.max_norm is not None and by_step:
            norm, factor = _norm_and_factor([self.params[i].grad for members in by_step.values() for i in members], self.max_norm)
            self.norm = Tensor._wrap(norm, self.params[0].device)
        for step, members in by_step.items():
            new, states = self._step([self.params[i] for i in members], [self.states[i] for i in members], step, factor)
            for i, p, s in zip(members, new, states):
                self.params[i].zero_grad()  # of the leaf that was: the graph may still hold it
                self.params[i]._node = p._node
                self.states[i] = s
                self.steps[i] = step

    def _step(self, params, states, step: int, factor):
        grads = [p.grad for p in params]
        options = dict(lr=self.lr, betas=self.betas, eps=self.eps, weight_decay=self.weight_decay)
        if factor is None:
            return adamw(params, grads, states, step=step, **options)
        return _adamw(params, grads, states, step, factor=factor, **options)

    def zero_grad(self) -> None:
        for p in self.params:
            p.zero_grad()


__all__ = ["RotaryTable", "rotary", "attention", "AdamState", "AdamState8", "adamw", "AdamW", "grad_norm", "clip_grads"]
