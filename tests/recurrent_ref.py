"""The recurrence and the convolution token by token in 64 bits, with bounds on what
float32 roundings may put beside them.

u = 2^-24. Every value comes with a majorant: the same sums over absolute values.
"""
import numpy as np

U = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # of 24, 8 and 11 significant bits
TINY = {"float32": 1e-37, "bfloat16": 1e-37, "float16": 2.0 ** -25}


def close(got, want, bound, dtype, what=""):
    """|got - want| <= bound (fp32 roundings) and the last rounding to the type."""
    limit = bound + HALF[dtype] * (np.abs(want) + bound) + TINY[dtype]
    off = np.abs(got.astype(np.float64) - want)
    assert got.shape == want.shape and np.isfinite(got).all(), what
    assert (off <= limit).all(), (what, float((off / limit).max()), np.unravel_index(np.argmax(off / limit), off.shape))


def rules(length, batch, documents, lengths):
    """on, cut (length, batch, 1): tokens that count, and those that forget what was before them."""
    on, cut = np.ones((length, batch, 1), bool), np.zeros((length, batch, 1), bool)
    for b in range(batch):
        end = length if lengths is None else min(max(int(lengths[b]), 0), length)
        for t in range(length):
            if t >= end:
                on[t, b] = False
            elif documents is not None:
                on[t, b] = documents[b, t] >= 0
                cut[t, b] = not on[t, b] or (t > 0 and documents[b, t] != documents[b, t - 1])
    return on, cut


# Roundings per token, in u: the gate (exp2 2, its correction 2, 1 + e 1, the reciprocal 2; 1 - a a product more: at
# most 12 with the input's), the product of gates, the multiply-add: 16. e^-g of a 16-bit logit goes without the
# correction: -g log2 e is off by half a spacing and by the constant's own, together under 2 |g| u of e^-g (logits
# past 88 count as that). A value then passes at most 2 joins of segments, 4 of waves and those of the tiles before
# it (64 for the longest here), whatever its token: 80.
STEP, JOIN = 16, 80


def recurrence(g, x, logit, initial=None, documents=None, lengths=None, dy=None, dlast=None):
    """(values, bounds), dicts of y, last and with dy or dlast dg, dx, dinitial. Masked places may hold anything."""
    batch, length, channels = x.shape
    g, x = (np.moveaxis(t.astype(np.float64), 1, 0) for t in (g, x))
    on, cut = rules(length, batch, documents, lengths)
    g, x = np.where(on, g, 0.0), np.where(on, x, 0.0)
    a, take = (1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))) if logit else (g, np.ones_like(g))
    keep = np.where(cut, 0.0, np.where(on, a, 1.0))
    b = np.where(on, take * x, 0.0)
    h = np.zeros((batch, channels)) if initial is None else initial.astype(np.float64)
    big, err = np.abs(h), np.zeros_like(h)
    hs, bigs, errs = [h], [big], [err]
    step = STEP + (2 * np.minimum(np.abs(g), 88.0) if logit else np.zeros_like(g))
    for t in range(length):
        err = np.abs(keep[t]) * err + step[t] * U * (np.abs(keep[t]) * big + np.abs(b[t]))
        big = np.abs(keep[t]) * big + np.abs(b[t])
        h = keep[t] * h + b[t]
        hs.append(h), bigs.append(big), errs.append(err)
    hs, bigs, errs = (np.stack(s) for s in (hs, bigs, errs))
    errs = errs + JOIN * U * bigs
    values = {"y": np.where(on, hs[1:], 0.0), "last": hs[-1]}
    bounds = {"y": np.where(on, errs[1:], 0.0), "last": errs[-1]}
    if dy is None and dlast is None:
        return _batch_first(values), _batch_first(bounds)
    d = np.zeros_like(x) if dy is None else np.where(on, np.moveaxis(dy.astype(np.float64), 1, 0), 0.0)
    m = np.zeros((batch, channels)) if dlast is None else dlast.astype(np.float64)
    mb, me = np.abs(m), np.zeros_like(m)
    dg, dx, eg, ex = (np.zeros_like(x) for _ in range(4))
    for t in range(length - 1, -1, -1):
        l, lb, le = d[t] + m, np.abs(d[t]) + mb, me + JOIN * U * mb + U * np.abs(d[t])
        prev, pb, pe = (np.where(cut[t], 0.0, s[t]) for s in (hs, bigs, errs))
        if logit:
            dx[t], ex[t] = l * take[t], (le + step[t] * U * lb) * take[t]
            dg[t] = l * (prev - x[t]) * a[t] * take[t]
            eg[t] = ((le + 2 * step[t] * U * lb) * (pb + np.abs(x[t])) + lb * pe) * a[t] * take[t]
        else:
            dx[t], ex[t] = l, le
            dg[t], eg[t] = l * prev, (le + 4 * U * lb) * pb + lb * pe
        me = np.abs(keep[t]) * me + step[t] * U * np.abs(keep[t]) * lb
        mb = np.abs(keep[t]) * lb
        m = keep[t] * l
    values |= {"dg": np.where(on, dg, 0.0), "dx": np.where(on, dx, 0.0), "dinitial": m}
    bounds |= {"dg": np.where(on, eg, 0.0), "dx": np.where(on, ex, 0.0), "dinitial": me + JOIN * U * mb}
    return _batch_first(values), _batch_first(bounds)


def _batch_first(d):
    return {k: np.moveaxis(v, 0, 1) if v.ndim == 3 else v for k, v in d.items()}


def conv(x, weight, bias, silu, initial=None, documents=None, lengths=None, dy=None, dlast=None):
    """(values, bounds), dicts of y, last and with dy or dlast dx, dw, db, dinitial.

    Roundings: width + 1 multiply-adds of z, 6 of the sigmoid and what is made of it
    (and 2 |z| u of e^-z for 16-bit results, as for the recurrence); silu' is at most
    1.1 and its slope at most 1/2, the silu's own at most 1.1. A weight's gradient adds
    32 tokens in a row, 16 runs pairwise, and the rows of the second launch, one for
    each batch and 480 or 512 tokens: at most 40 additions a term and those.
    """
    batch, length, channels = x.shape
    width = weight.shape[1]
    x, weight = x.astype(np.float64), weight.astype(np.float64)
    bias = np.zeros(channels) if bias is None else bias.astype(np.float64)
    on, _ = rules(length, batch, documents, lengths)
    on = np.moveaxis(on, 0, 1)
    rows = np.concatenate([np.zeros((batch, width - 1, channels)) if initial is None else initial.astype(np.float64), x], 1)
    # reads[b, t, j]: token t's tap j exists (row t + j); last_reads[b, j]: that of the token after the last
    reads, last_at, last_reads = np.zeros((batch, length, width), bool), [], np.zeros((batch, max(width - 1, 0)), bool)
    for b in range(batch):
        run = [0] * (width - 1) + [0] * length
        for t in range(1, length):
            run[width - 1 + t] = run[width - 2 + t] + (documents is not None and documents[b, t] != documents[b, t - 1])
        for t in range(length):
            for j in range(width):
                reads[b, t, j] = on[b, t, 0] and run[t + j] == run[t + width - 1]
        end = length if lengths is None else min(max(int(lengths[b]), 0), length)
        last_at.append(end)
        for j in range(width - 1):
            alive = end == 0 or (on[b, end - 1, 0] and run[end + j] == run[end + width - 2])
            last_reads[b, j] = alive
    taps = np.stack([np.where(reads[:, :, j:j + 1], rows[:, j:j + length], 0.0) for j in range(width)], -1)
    z = np.where(on, (taps * weight).sum(-1) + bias, 0.0)
    ez = (width + 1) * U * np.where(on, (np.abs(taps) * np.abs(weight)).sum(-1) + np.abs(bias), 0.0)
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-z))
    values = {"y": z * s if silu else z}
    bounds = {"y": 1.1 * ez + (8 + 2 * np.abs(z)) * U * np.abs(z) * s if silu else ez}
    values["last"] = np.stack([np.where(last_reads[b][:, None], rows[b, last_at[b]:last_at[b] + width - 1], 0.0) for b in range(batch)]) \
        if batch else np.zeros((0, width - 1, channels))
    if dy is None and dlast is None:
        return values, bounds
    d = np.zeros_like(x) if dy is None else np.where(on, dy.astype(np.float64), 0.0)
    slope = s * (1 + z * (1 - s)) if silu else np.ones_like(z)
    dz = d * slope
    edz = np.abs(d) * (0.5 * ez + (12 + 2 * np.abs(z)) * U * (s + np.abs(z) * s)) if silu else np.zeros_like(z)
    drows, erows = np.zeros_like(rows), np.zeros_like(rows)
    for j in range(width):
        r = reads[:, :, j:j + 1]
        drows[:, j:j + length] += np.where(r, dz * weight[:, j], 0.0)
        erows[:, j:j + length] += np.where(r, (edz + (width + 1) * U * np.abs(dz)) * np.abs(weight[:, j]), 0.0)
    if dlast is not None:
        for b in range(batch):
            part = np.where(last_reads[b][:, None], dlast[b].astype(np.float64), 0.0)
            drows[b, last_at[b]:last_at[b] + width - 1] += part
            erows[b, last_at[b]:last_at[b] + width - 1] += U * np.abs(part)
    erows += 2 * U * np.abs(drows)
    adds = (40 + batch * -(-length // 480)) * U
    edz = edz + adds * np.abs(dz)
    values |= {"dx": drows[:, width - 1:], "dinitial": drows[:, :width - 1], "dw": (dz[..., None] * taps).sum((0, 1)), "db": dz.sum((0, 1))}
    bounds |= {"dx": erows[:, width - 1:], "dinitial": erows[:, :width - 1], "dw": (edz[..., None] * np.abs(taps)).sum((0, 1)),
               "db": edz.sum((0, 1))}
    return values, bounds
