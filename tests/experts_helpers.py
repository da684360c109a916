"""Layers of experts in numpy and float64, by their definitions."""
import numpy as np

import oracle


def scores(x, kind, most):
    """Scores of logits [T, E]: those that are not there (-inf, NaN) have none, +inf counts as the
    type's largest finite value."""
    x = np.asarray(x, np.float64)
    there = x > -np.inf
    x = np.where(there, np.minimum(x, most), -np.inf)
    with np.errstate(all="ignore"):
        if kind == "softmax":
            m = x.max(1, keepdims=True)
            e = np.where(there, np.exp(x - m), 0.0)
            p = e / e.sum(1, keepdims=True)
        else:
            p = 1 / (1 + np.exp(-x))
    return x, there, p


def route(logits, top, bias=None, kind="softmax", groups=1, top_groups=None, group_rank=1,
          renormalise=True, scale=1.0, most=float(np.finfo(np.float32).max)):
    """ids [T, top] and weights [T, top] (float64)."""
    x, there, p = scores(logits, kind, most)
    T, E = x.shape
    key = x.copy()
    if bias is not None:
        b = np.asarray(bias, np.float64)
        with np.errstate(invalid="ignore"):
            key = np.where(there & (b > -np.inf), p + b, -np.inf)
    key = np.where(there, key, -np.inf)
    ids = np.full((T, top), -1, np.int64)
    w = np.zeros((T, top))
    size = E // groups
    for t in range(T):
        allowed = key[t] > -np.inf
        if top_groups is not None and top_groups < groups:
            by = p[t] if bias is None and group_rank == 2 else key[t]
            value = np.full(groups, -np.inf)
            for g in range(groups):
                at = np.arange(g * size, (g + 1) * size)
                best = np.sort(by[at][allowed[at]])[::-1][:group_rank]
                if len(best):
                    value[g] = best.sum()
            order = [g for g in np.argsort(-value, kind="stable")[:top_groups] if value[g] > -np.inf]
            allowed &= np.isin(np.arange(E) // size, order)
        k = np.where(allowed, key[t], -np.inf)
        chosen = [e for e in np.argsort(-k, kind="stable")[:top] if allowed[e]]
        ids[t, :len(chosen)] = chosen
        if not chosen:
            continue
        c, z = p[t, chosen], x[t, chosen]
        if renormalise:  # relative to the largest one, where all the chosen scores vanish too
            if kind == "softmax":
                c = np.exp(z - z.max())
            else:
                c = np.exp(np.minimum(z, 0) - min(z.max(), 0)) / (1 + np.exp(-np.abs(z)))
            c = c / c.sum()
        w[t, :len(chosen)] = c * scale
    return ids, w


def arrange(ids, experts, first=0):
    ids = np.asarray(ids, np.int64) - first
    T, top = ids.shape
    flat = ids.ravel()
    mine = (flat >= 0) & (flat < experts)
    order = np.argsort(np.where(mine, flat, experts), kind="stable")
    starts = np.concatenate([[0], np.cumsum(np.bincount(flat[mine], minlength=experts))])
    tokens = np.where(np.arange(T * top) < starts[-1], order // top, -1)
    place = np.full(T * top, -1, np.int64)
    place[order[:starts[-1]]] = np.arange(starts[-1])
    return starts, tokens, place.reshape(T, top)


def ranges(starts, rows):
    """[first, last) of each expert, as the kernels take first rows: the nearest of 0 .. rows, and the
    largest before where they decrease."""
    s = np.maximum.accumulate([min(max(int(x), 0), rows) for x in starts]).tolist()
    return list(zip(s, s[1:]))


def product(a, sfa, b, sfb, starts, rows=None, total=None):
    """(model of the MFMA's sum as bf16 bits, sum |a b|, written) for every row: fp32 sums of the
    oracle's model in one chain along K."""
    total = (a.shape[0] if rows is None else len(rows)) if total is None else total
    n, k = b.shape[1:]
    want = np.zeros((total, n), np.float32)
    mass = np.zeros((total, n))
    written = np.zeros(total, bool)
    for e, (lo, hi) in enumerate(ranges(starts, total)):
        if lo >= hi:
            continue
        m = np.arange(lo, hi) if rows is None else np.asarray(rows[lo:hi])
        ok = (m >= 0) & (m < a.shape[0])
        qa = np.where(ok[:, None], a[np.where(ok, m, 0)], 0).astype(np.uint8)
        sa = np.ascontiguousarray(np.where(ok, sfa[:, np.where(ok, m, 0)], 0).astype(np.float32))
        want[lo:hi] = oracle.gemm_blockscale_mfma(qa, b[e], sa, sfb[e], 128, 0)
        mass[lo:hi] = oracle.blockscale_absdot(qa, b[e], sa, sfb[e], 128)
        written[lo:hi] = True
    return oracle.to_bf16_bits(want), mass, written


def activate(x):
    """The activation in float64 [R, I] of x [R, 2 I], its scales [I / 128, R]."""
    x = np.asarray(x, np.float64)
    g, u = np.split(x, 2, 1)
    with np.errstate(over="ignore"):
        y = u * g / (1 + np.exp(-g))
    amax = np.abs(y).reshape(len(x), -1, 128).max(2)
    return y, np.where(amax > 0, amax / 448, 1.0).T


def combine(y, place, weights):
    """(sums in float64 [T, N], the sum of magnitudes)."""
    y = np.asarray(y, np.float64)
    ok = (place >= 0) & (place < len(y))
    out = np.zeros((len(place), y.shape[1]))
    mass = np.zeros_like(out)
    for j in range(place.shape[1]):
        t = np.flatnonzero(ok[:, j])
        z = np.asarray(weights, np.float64)[t, j, None] * y[place[t, j]]
        out[t] += z
        mass[t] += np.abs(z)
    return out, mass
