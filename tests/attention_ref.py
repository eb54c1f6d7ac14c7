"""Attention in 64 bits by its formula, with bounds on what float32 sums and
16-bit roundings may be off by, for the attention tests.

Per batch and head, with u = 2^-24 and h the half-spacing of the operands' type
against its values (0 for float32): a score t is off by at most e_t = (D + 8) u S + 4 u |t|, S the
sum of |q k| scale, plus the tanh's 5e-7 cap; an exponential by the factor
2 e_t + 4 u against its row's sum, a sum of n of them by n u. Then
  out: sum p |v| (E + h) + h |out|,              E = 2 max e_t + (n + 12) u
  dv:  sum p |dout| (E + h) + h |dv|
  ds:  p ((|dp| + |delta|) (E + h + 1e-6 if capped) + (D + 8) u A + B (h + D u)),
       A = sum |dout v|, B = sum |dout out|; summed into dq and dk, + h of those
where the gradient's delta reads the rounded output. Every term is doubled once
for the second-order ones left out.
"""
import numpy as np

U = 2.0 ** -24
HALF = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # of 8 and 11 significant bits


def visible(lq, lk, causal=False, docs=None, prefix=None, length=None):
    end = lk if length is None else min(max(int(length), 0), lk)
    at = np.arange(lq)[:, None] + end - lq
    j = np.arange(lk)[None, :]
    see = np.broadcast_to(j < end, (lq, lk)).copy()
    if causal:
        near = j <= at
        see &= near if prefix is None else near | (j < prefix)
    if docs is not None:
        own = np.where((at >= 0) & (at < lk), docs[np.clip(at, 0, lk - 1)], -1)
        see &= (own == docs[None, :]) & (own >= 0)
    return see, at - j


def attention(q, k, v, dout=None, *, dtype="float32", causal=False, scale=None, cap=0.0, slopes=None, documents=None,
              prefix=None, lengths=None):
    """{name: (exact, bound)} for out and, with dout, dq, dk, dv."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    b, lq, heads, d = q.shape
    lk, kvh = k.shape[1], k.shape[2]
    scale = 1 / np.sqrt(d) if scale is None else scale
    h = HALF[dtype]
    shapes = {"out": q.shape, "dq": q.shape, "dk": k.shape, "dv": k.shape}
    val = {n: np.zeros(s) for n, s in shapes.items()}
    err = {n: np.zeros(s) for n, s in shapes.items()}
    for bi in range(b):
        see, away = visible(lq, lk, causal, None if documents is None else documents[bi], None if prefix is None else int(prefix[bi]),
                            None if lengths is None else lengths[bi])
        live = see.any(0)
        for hi in range(heads):
            g = hi // (heads // kvh)
            qh = q[bi, :, hi]
            # what no query sees does not matter, whatever stands there
            kh, vh = (np.where(live[:, None], x[bi, :, g], 0.0) for x in (k, v))
            s = qh @ kh.T * scale
            t, bent = s, np.zeros_like(s)
            if cap:
                bent = np.tanh(s / cap)
                t = cap * bent
            if slopes is not None:
                t = t - float(slopes[hi]) * np.abs(away)
            size = np.abs(qh) @ np.abs(kh).T * abs(scale)
            e_t = (d + 8) * U * size + 4 * U * np.abs(t) + 5e-7 * cap
            if slopes is not None:
                e_t = e_t + 4 * U * abs(float(slopes[hi])) * np.abs(away)
            top = np.max(np.where(see, t, -np.inf), 1, keepdims=True, initial=-np.inf)
            p = np.where(see, np.exp(t - np.where(np.isfinite(top), top, 0.0)), 0.0)
            total = p.sum(1, keepdims=True)
            p = p / np.where(total == 0, 1.0, total)
            n = max(lk, lq * (heads // kvh))
            e = 2 * np.max(np.where(see, e_t, 0.0), 1, keepdims=True, initial=0.0) + (n + 12) * U
            out = p @ vh
            val["out"][bi, :, hi] = out
            err["out"][bi, :, hi] = 2 * ((p * (e + h)) @ np.abs(vh)) + h * np.abs(out)
            if dout is None:
                continue
            do = np.asarray(dout, np.float64)[bi, :, hi]
            dp = do @ vh.T
            delta = (do * out).sum(1, keepdims=True)
            slope = 1 - bent * bent
            ds = p * (dp - delta) * slope
            a, bb = np.abs(do) @ np.abs(vh).T, (np.abs(do) * np.abs(out)).sum(1, keepdims=True)
            e_ds = p * ((np.abs(dp) + np.abs(delta)) * (e + h + (1e-6 if cap else 0.0)) + (d + 8) * U * a + bb * (h + d * U)) * slope
            if cap:
                e_ds = e_ds + 1e-6 * p * (np.abs(dp) + np.abs(delta))
            val["dv"][bi, :, g] += p.T @ do
            err["dv"][bi, :, g] += 2 * ((p * (e + h)).T @ np.abs(do))
            val["dq"][bi, :, hi] = ds @ kh * scale
            err["dq"][bi, :, hi] = 2 * (e_ds + (n + 4) * U * np.abs(ds)) @ np.abs(kh) * abs(scale)
            val["dk"][bi, :, g] += ds.T @ qh * scale
            err["dk"][bi, :, g] += 2 * (e_ds + (n + 4) * U * np.abs(ds)).T @ np.abs(qh) * abs(scale)
    for n in ("dq", "dk", "dv"):
        err[n] = err[n] + h * np.abs(val[n])
    tiny = {"float32": 1e-37, "bfloat16": 1e-37, "float16": 2.0 ** -24}[dtype]  # half the least float16 spacing, and more
    return {n: (val[n], err[n] + tiny) for n in (shapes if dout is not None else ["out"])}


def assert_within(got, want, what):
    exact, bound = want
    got = np.asarray(got, np.float64)
    assert got.shape == exact.shape, what
    assert np.isfinite(got).all(), f"{what}: not finite"
    worst = float(np.max(np.abs(got - exact) / bound, initial=0.0))
    assert worst <= 1.0, f"{what}: {worst:.3g} times its bound"
