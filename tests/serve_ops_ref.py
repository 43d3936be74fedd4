"""Rotation with head norms, attention behind shared prefixes and sampling from
given numbers in 64 bits, from their definitions (test infrastructure)."""
import math

import numpy as np

import device_ops_ref as ref

EPS = ref.EPS


def rope(x, pos, freq, gain, eps, near):
    """Rows [rows, heads, hd] at positions pos, normed and turned, and what
    rounding allows of it in units of 2^-24 (before the output's own).

    A norm's sum of hd squares in f32 is off by hd 2^-24 of it at most, its
    root by half of that; eps, the division, the root and the two products
    with it and the gain add less than 8. An angle's sine and cosine: f32's
    rounding of a reduced angle of at most pi / 4 and of its product with pi /
    2, then a few operations on numbers up to 1, all in all less than 6; the
    products and their sum 2 more."""
    x = np.asarray(x, dtype=np.float64)
    y = x
    rel = 0.0
    hd = x.shape[-1]
    if gain is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + np.asarray(gain, dtype=np.float64))
        rel = hd / 2 + 8
    half = len(freq)
    # (a position of 31 bits times a float: exact in 64 bits of mantissa)
    t = np.asarray(pos, dtype=np.longdouble)[:, None] * np.asarray(freq, dtype=np.float32).astype(np.longdouble)
    two_pi = 2 * np.longdouble("3.14159265358979323846264338327950288")
    t = (t - np.rint(t / two_pi) * two_pi).astype(np.float64)[:, None, :]
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if near else (slice(0, half), slice(half, 2 * half))
    o, off = y.copy(), np.abs(y) * rel
    o[..., a] = y[..., a] * np.cos(t) - y[..., b] * np.sin(t)
    o[..., b] = y[..., b] * np.cos(t) + y[..., a] * np.sin(t)
    size = np.abs(y[..., a]) + np.abs(y[..., b])
    off[..., a] = off[..., b] = size * (rel + 8)
    return o, off


def rope_tolerance(typ, o, off):
    return off * EPS["f32"] + EPS[typ] * np.abs(o) + (2.0 ** -25 if typ == "f16" else 1e-37)


def attend_shared(q, data, slots, pos, seq, off, pdata, pslots, plen, pseq, poff, sink, scale):
    """As device_ops_ref.attend, every row also seeing its group's prefix."""
    T, hq, hd = q.shape
    hkv = data.shape[1]
    o, pv = np.zeros((T, hq, hd)), np.zeros((T, hq, hd))
    big, cnt = np.zeros((T, hq, 1)), np.zeros((T, hq, 1))
    for h in range(hkv):
        pre = {}
        for g in range(len(plen)):
            r0, r1 = (0, T) if poff is None else (poff[g], poff[g + 1])
            if 0 <= pseq[g] < pdata.shape[0] and 0 < plen[g] < 2 ** 31:
                K, V = ref.get(pdata, pseq[g], h, pslots)
                n = min(plen[g], pslots)
                for r in range(r0, r1):
                    pre[r] = K[:n], V[:n]
        for i in range(len(pos)):
            r0, r1 = (i, i + 1) if off is None else (off[i], off[i + 1])
            if r1 <= r0 or not 0 <= seq[i] < data.shape[0] or pos[i] < 0:
                continue
            last = pos[i] + r1 - r0 - 1
            at = last - (last - np.arange(slots)) % slots
            K, V = ref.get(data, seq[i], h, slots)
            for r in range(r0, r1):
                see = (at >= 0) & (at <= pos[i] + r - r0)
                k, v = K[see], V[see]
                if r in pre:
                    k, v = np.concatenate([pre[r][0], k]), np.concatenate([pre[r][1], v])
                for a in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    with np.errstate(all="ignore"):
                        x = (k @ q[r, a]) * scale
                        m = max([-math.inf if sink is None else sink[a]] + ([x.max()] if len(x) else []))
                        if m == -math.inf:
                            continue
                        e = np.exp(x - m)
                        den = e.sum() + (0.0 if sink is None else math.exp(sink[a] - m))
                        o[r, a] = (e[:, None] * v).sum(0) / den
                        pv[r, a] = (e[:, None] * np.abs(v)).sum(0) / den
                        big[r, a] = (np.abs(k) @ np.abs(q[r, a])).max() * abs(scale) if len(x) else 0.0
                        cnt[r, a] = len(x)
    return o, pv, big, cnt


def sample(x, u, t=1.0, k=0, p=1.0, q=0.0):
    """(token, log probability) of one row."""
    x = np.asarray(x, dtype=np.float64)
    order = [i for i in ref.order(x) if x[i] > -math.inf]   # (no NaN either)
    if not order:
        return -1, math.nan
    if not t > 0:
        return order[0], 0.0
    order = order[:k] if 0 < k < len(x) else order
    m = x[order[0]]
    if m == math.inf:
        w = np.array([float(x[i] == math.inf) for i in order])
    else:
        w = np.exp((x[order] - m) / t)
    c = np.cumsum(w)
    n = len(w)
    if p < 1:
        n = int(np.searchsorted(c, p * c[-1])) + 1   # the fewest that reach p of it
    n = max(1, min(n, int((w >= q).sum())))          # (w goes down)
    c = c[:n]
    u = 0.0 if math.isnan(u) else min(max(u, 0.0), 1.0)
    i = min(int(np.searchsorted(c, u * c[-1], side="right")), int((w[:n] > 0).sum()) - 1)
    return order[i], math.log(w[i]) - math.log(c[-1])
