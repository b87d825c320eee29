"""Plain 64-bit restatements (numpy) of the operators in embedding, recurrence and microscale, with the error that a
32-bit evaluation in any order may have.  U is half a step of a float: what one rounding to 32 bits may be off."""
import numpy as np
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half the smallest subnormal


def f64(t):
    return None if t is None else t.detach().to("cpu", torch.float64).numpy()


def close(got, want, err, what=""):
    """|got - want| <= err + half a step of got's type, elementwise."""
    g = f64(got)
    assert g.shape == want.shape, (what, g.shape, want.shape)
    lim = err + HALF_STEP[got.dtype] * (np.abs(want) + err) + TINY[got.dtype]
    bad = ~(np.abs(g - want) <= lim)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, np.abs(g - want) - lim, -np.inf)), g.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off, worst at {at}: {g[at]} for {want[at]}, limit {lim[at]}")


# ---- lookup -----------------------------------------------------------------------------------------------------------


def lookup(table, idx, weight, scale):
    idx = idx.reshape(-1)
    out = np.zeros((idx.size, table.shape[1]))
    for i, p in enumerate(idx):
        if 0 <= p < table.shape[0]:
            out[i] = scale * (1.0 if weight is None else weight.reshape(-1)[i]) * table[p]
    return out


def lookup_backward(dout, table, idx, weight, scale):
    """dtable, its error, dweight, its error."""
    idx, d = idx.reshape(-1), dout.reshape(idx.size, -1)
    dt, ab, cnt = np.zeros(table.shape), np.zeros(table.shape), np.zeros(table.shape[0])
    dw, dwa = np.zeros(idx.size), np.zeros(idx.size)
    for i, p in enumerate(idx):
        if 0 <= p < table.shape[0]:
            w = scale * (1.0 if weight is None else weight.reshape(-1)[i])
            dt[p] += w * d[i]
            ab[p] += np.abs(w * d[i])
            cnt[p] += 1
            dw[i] = scale * (d[i] * table[p]).sum()
            dwa[i] = abs(scale) * np.abs(d[i] * table[p]).sum()
    # a term passes the factor's rounding, its own product's and at most cnt additions
    return dt, (cnt[:, None] + 2) * U * ab, dw, (table.shape[1] + 2) * U * dwa


# ---- recurrence -------------------------------------------------------------------------------------------------------


def sequences(x, offsets):
    """[(index of a sequence's steps in x's leading dimensions)]"""
    if offsets is None:
        return [(b, slice(None)) for b in range(x.shape[0])]
    return [(slice(int(offsets[s]), int(offsets[s + 1])),) for s in range(len(offsets) - 1)]


def scan(gate, x, state, offsets, reverse, dh=None, dlast=None):
    """Every output of scan and scan_backward as {name: (value, error)}.  With M the recurrence of magnitudes, each step of
    any split evaluation rounds what it carries at most four times (product of gates, multiply-add, join of stretches)."""
    D, G = x.shape[-1], gate.shape[-1]
    Q, seqs = D // G, sequences(x, offsets)
    S = len(seqs)
    wide = lambda a: np.repeat(a, Q, axis=-1)  # noqa: E731
    z = lambda *s: np.zeros(s)  # noqa: E731
    h, eh, dx, edx = z(*x.shape), z(*x.shape), z(*x.shape), z(*x.shape)
    dg, edg = z(*gate.shape), z(*gate.shape)
    last, elast, ds, eds = z(S, D), z(S, D), z(S, D), z(S, D)
    for s, at in enumerate(seqs):
        xs, a = x[at], wide(gate[at])
        T = xs.shape[0]
        order = range(T - 1, -1, -1) if reverse else range(T)
        c = np.zeros(D) if state is None else state[s].copy()
        m, e = np.abs(c), np.zeros(D)
        prev = {}
        for t in order:
            prev[t] = (c, m, e)
            c = a[t] * c + xs[t]
            m = np.abs(a[t]) * m + np.abs(xs[t])
            e = np.abs(a[t]) * e + 4 * U * m
            h[at][t], eh[at][t] = c, e
        last[s], elast[s] = c, e
        lam = np.zeros(D) if dlast is None else dlast[s].copy()
        ml, el = np.abs(lam), np.zeros(D)
        for t in reversed(order):
            d = 0.0 if dh is None else dh[at][t]
            lam, ml = lam + d, ml + np.abs(d)
            el = el + U * ml
            dx[at][t], edx[at][t] = lam, el
            c, m, e = prev[t]
            fold = lambda v: v.reshape(G, Q).sum(1)  # noqa: E731
            dg[at][t] = fold(lam * c)
            edg[at][t] = fold(el * m + ml * e + el * e) + (Q + 2) * U * fold(ml * m)
            lam, ml = a[t] * lam, np.abs(a[t]) * ml
            el = np.abs(a[t]) * el + 4 * U * ml
        ds[s], eds[s] = lam, el
    return {"h": (h, eh), "last": (last, elast), "dgate": (dg, edg), "dx": (dx, edx), "dstate": (ds, eds)}


# ---- microscaled 4-bit floats -----------------------------------------------------------------------------------------

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """(values, scale bytes) of the 4-bit form of x (rows, width), by distance to the levels; NaN where a block has an
    infinity or NaN."""
    rows, width = x.shape
    nb = -(-width // 32)
    p = np.zeros((rows, nb * 32))
    p[:, :width] = x
    p = p.reshape(rows, nb, 32)
    bad = ~np.isfinite(p).all(2)
    p = np.where(bad[..., None], 0.0, p)
    most = np.abs(p).max(2)
    e = np.where(most > 0, np.clip(np.frexp(np.where(most > 0, most, 1.0))[1] - 1 - 2, -127, 127), -127)
    v = np.abs(p) * 2.0 ** -e.astype(np.float64)[..., None]
    best = np.zeros_like(v)
    for lev in LEVELS[[2, 4, 6, 1, 3, 5, 7]]:  # even codes first, so that an odd one has to be nearer
        best = np.where(np.abs(v - lev) < np.abs(v - best), lev, best)
    val = np.copysign(best, p) * 2.0 ** e.astype(np.float64)[..., None]
    val = np.where(bad[..., None], np.nan, val)
    return val.reshape(rows, -1)[:, :width], np.where(bad, 255, e + 127)


def values(codes, scales, width):
    """What codes and scales stand for."""
    n = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    v = np.where(n > 7, -1.0, 1.0) * LEVELS[n & 7]
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v * np.repeat(s, 32, axis=1)[:, :v.shape[1]])[:, :width]
