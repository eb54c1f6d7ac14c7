"""What a recurrent block needs beside products and maps: a gated linear
recurrence over the tokens of each channel, and the short causal convolution
that goes before it. Both carry their state from one call to the next.

    x, conv_state = causal_conv(x, weight, bias, conv_state, activation="silu")
    y, state = linear_recurrence(logits, x, state, gate="logit")    # differentiable, lazy like every op

A state without a gradient keeps nothing of its call once it is realized. One with a
gradient (weights that learn are among what it came from) keeps its call, and through
it every call before: pass state.detach() on where gradients are not to go back.

Additive to the reference's Python surface (ormi-core/src/ormi_core/tensor.py:10-190),
which has neither.
"""
from __future__ import annotations

from ._ext import ormi_backend
from .tensor import Tensor
from .transformer import _node


def _wrap(pair, like: Tensor):
    return tuple(Tensor._wrap(n, like.device) for n in pair)


def linear_recurrence(gates: Tensor, x: Tensor, initial: Tensor | None = None, *, gate: str = "value", documents: Tensor | None = None,
                      lengths: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """h_t = a_t h_{t-1} + b_t over the tokens of x (batch, length, channels): (h, the state after the last token).

    gates: a value per token and channel, of x's type or float32
      gate="value"  a = gates, b = x
      gate="logit"  a = sigmoid(gates), b = (1 - a) x
    initial    float32 (batch, channels): the state before the first token (zeros)
    documents  int32 (batch, length): the state starts from zero where the entry
               changes; a token of a negative one gives zeros and leaves zeros
    lengths    int32 (batch,): tokens that exist (all); the others give zeros,
               whatever they hold, and leave the state as it is
    h has x's type, the state is float32 (batch, channels): pass it, or it
    detached, as the next call's initial. Gradients go to gates, x and initial, from h and from the state.
    States are float32, results are rounded once. Gates whose product over some run
    of tokens passes 2^128, which none of magnitude up to 1 do, give results that
    are not finite; a product below 2^-126 is held to 2^-149 of the state before it.
    """
    if gate not in ("value", "logit"):
        raise ValueError("gate must be value or logit.")
    pair = ormi_backend.recurrence(_node(gates, x, "gates"), x._node, _node(initial, x, "initial"), _node(documents, x, "documents"),
                                   _node(lengths, x, "lengths"), gate == "logit")
    return _wrap(pair, x)


def causal_conv(x: Tensor, weight: Tensor, bias: Tensor | None = None, initial: Tensor | None = None, *, activation: str | None = None,
                documents: Tensor | None = None, lengths: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Each channel of x (batch, length, channels) convolved with its own weights over the token and those before it:
    (act(bias + sum_j weight[:, j] x_{t - width + 1 + j}), the inputs that the next token reads).

    weight      float32 (channels, width), width 1 to 8, the token's own last
    bias        float32 (channels,)
    initial     (batch, width - 1, channels) of x's type: the inputs before the first token (zeros)
    activation  None or "silu"
    documents   int32 (batch, length): a token reads inputs from where the entry last
                changed (initial is the first token's); one of a negative document gives zeros
    lengths     int32 (batch,): tokens that exist (all); the others give zeros, whatever they hold
    The result and the inputs kept (batch, width - 1, channels) have x's type: pass the
    latter, or them detached, as the next call's initial. Gradients go to x, weight, bias and initial.
    Sums are float32, results are rounded once.
    """
    if activation not in (None, "silu"):
        raise ValueError('activation must be None or "silu".')
    pair = ormi_backend.conv(x._node, _node(weight, x, "weight"), _node(bias, x, "bias"), _node(initial, x, "initial"),
                             _node(documents, x, "documents"), _node(lengths, x, "lengths"), activation == "silu")
    return _wrap(pair, x)


__all__ = ["linear_recurrence", "causal_conv"]
