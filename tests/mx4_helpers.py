"""A plain MXFP4 key/value cache in numpy and float64: the layout of
include/gcnasm_amd.h byte by byte, attention and eviction by their definitions."""
import numpy as np

VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])


def places(P, D):
    """Byte offsets in a head's page: K codes [P, D/2], V codes [P, D/2], K scales [P, D/32], V
    scales [P, D/32]; the codes' byte x holds elements 2x and 2x + 1."""
    t = np.arange(P)[:, None]
    x = np.arange(D // 2)[None]
    s = np.arange(D // 32)[None]
    piece = D // 32  # bytes of D/16 elements
    kc = t * (D // 2) + x
    vc = P * D // 2 + ((t // 4 * 16 + x // piece) * 4 + t % 4) * piece + x % piece
    ks = P * D + t * (D // 32) + s
    vs = P * D + P * D // 32 + (t // 4 * (D // 32) + s) * 4 + t % 4
    return kc, vc, ks, vs


def values(codes, scales):
    """Packed codes [..., D/2] and scale bytes [..., D/32] as float64 [..., D]."""
    n = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (2 * codes.shape[-1],))
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
        return VALUES[n] * np.repeat(s, 32, -1)


def tokens(cache, table, P, D, n):
    """K, V float64 [n, heads, D] and whether they are there [n] of one sequence's first n tokens."""
    kc, vc, ks, vs = places(P, D)
    t = np.arange(n)
    pages = np.asarray(table)[t // P] if n else np.zeros(0, int)
    there = (pages >= 0) & (pages < cache.shape[0])
    rows = cache[np.where(there, pages, 0)]  # [n, heads, bytes]

    def take(at):
        return np.take_along_axis(rows, at[t % P][:, None, :].repeat(rows.shape[1], 1), 2)

    return values(take(kc), take(ks)), values(take(vc), take(vs)), there


def attention(q, k, v, there, length, n, causal, window, scale, softcap):
    """float64 rows [n, heads, D] of one sequence: out, lse, the weights [kv heads, length], and
    the bounds of what the kernel may be off by: of out and of lse."""
    rows, hq, D = q.shape
    h = k.shape[1]
    out = np.zeros((n, hq, D))
    lse = np.full((n, hq), -np.inf)
    w = np.zeros((h, length))
    out_tol = np.zeros((n, hq, D))
    lse_tol = np.zeros((n, hq))
    t = np.arange(length)
    for i in range(n):
        pos = length - n + i
        seen = there[:length].copy()
        if causal:
            seen &= t <= pos
        if window:
            seen &= t > pos - window
        if not seen.any():
            continue
        for a in range(hq):
            kk, vv = k[:length][seen][:, a * h // hq], v[:length][seen][:, a * h // hq]
            with np.errstate(all="ignore"):
                s = kk @ q[i, a] * scale
                e = (D + 8) * 2.0 ** -23 * abs(scale) * (np.abs(kk) @ np.abs(q[i, a])).max()
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                    e += softcap * 2.0 ** -21
                m = s.max()
                p = np.exp(s - m)
                l = p.sum()
                # scores off by e, the exponent's argument rounded, the logarithm's
                e += 2.0 ** -22 * (np.abs(s).max() + 1)
                lse_tol[i, a] = 2 * e + 2.0 ** -22 * (abs(m + np.log(l)) + 1)
                p = p / l
                out[i, a] = p @ vv
                lse[i, a] = m + np.log(l)
                # probabilities to 8 bits (2^-9 each) and as far off as the scores; the output's
                # own rounding to bf16; sums in fp32
                mass = p @ np.abs(vv)
                out_tol[i, a] = ((2.0 ** -9 + 4 * e + len(s) * 2.0 ** -23) * mass +
                                 2.0 ** -8.9 * np.abs(out[i, a]) + 1e-37)
                w[a * h // hq, np.flatnonzero(seen)] += p
    return out, lse, w, out_tol, lse_tol


def evict(weights, length, keep, recent):
    """Indices kept of one head's weights [>= length]."""
    if length <= keep:
        return np.arange(length)
    old = length - recent
    w = weights[:old].astype(np.float64)
    w = np.where(np.isnan(w), np.inf, w)
    nan = np.isnan(weights[:old])
    order = sorted(range(old), key=lambda j: (-int(nan[j]), -w[j], j))
    return np.concatenate([np.sort(order[:keep - recent]).astype(int), np.arange(old, length)])
