"""The operators on device memory in 64 bits, from their definitions, and the
4-bit cache's bytes one index at a time (test infrastructure)."""
import math

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # half a step, relative


def quant(x):
    """Blocks of 32 along the last axis: codes, and scale bytes of the blocks.
    x holds numbers of at most 24 bits (any of the tensors' types)."""
    x = np.asarray(x, dtype=np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore"):
        a = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    a = np.where(bad, 1.0, a)
    e = np.full(a.shape, 2, dtype=np.int64)
    for k in range(3, 253):
        e = np.where(a > 7.0 * 2.0 ** (k - 1 - 127), k, e)
    y = np.abs(np.where(bad[..., None], 0.0, b)) / 2.0 ** (e[..., None] - 127)
    # the nearest level, a tie to the even code
    d = np.abs(y[..., None] - LEVELS)
    best = d.min(-1, keepdims=True)
    tied = d == best
    code = np.argmax(tied, -1)
    odd = (code % 2 == 1) & (tied.sum(-1) > 1)
    code = np.where(odd, code + 1, code)
    code = code + 8 * np.signbit(np.where(bad[..., None], 0.0, b))
    return code.reshape(x.shape), np.where(bad, 255, e).astype(np.uint8)


def values(code, scale):
    """Codes [..., hd] and their blocks' scale bytes as numbers."""
    v = np.where(code & 8, -1.0, 1.0) * LEVELS[code & 7]
    s = np.where(scale == 255, math.nan, 2.0 ** (scale.astype(np.float64) - 127))
    return v * np.repeat(s, 32, axis=-1)


def places(hd, s):
    """Byte and shift of slot s's codes in a record (keys, values), and the
    bytes of their scales."""
    d = np.arange(hd)
    m, h = s % 16, s // 16
    jk = d // (hd // 4)
    key = ((jk * 16 + m) * 2 + h) * (hd // 8) + d % (hd // 4) // 2
    jv, ev = m // 4, h * 4 + m % 4
    val = 16 * hd + ((jv * 16 + d // (hd // 16)) * 8 + ev) * (hd // 32) + d % (hd // 16) // 2
    g = np.arange(hd // 32)
    return key, val, d % 2 * 4, 32 * hd + (g * 16 + m) * 2 + h, 33 * hd + (g * 4 + jv) * 8 + ev


def put(data, q, h, slot, kc, ks, vc, vs):
    """One position's codes and scales into a cache's bytes."""
    rec = data[q, h, slot // 32]
    key, val, sh, kb, vb = places(rec.shape[0] // 34, slot % 32)
    for at, c in ((key, kc), (val, vc)):
        for i in range(len(at)):
            rec[at[i]] = (int(rec[at[i]]) & ~(0xF << int(sh[i])) & 0xFF) | (int(c[i]) << int(sh[i]))
    rec[kb], rec[vb] = ks, vs


def get(data, q, h, slots):
    """The keys and values [slots, hd] of a sequence's head."""
    hd = data.shape[-1] // 34
    K, V = np.empty((slots, hd)), np.empty((slots, hd))
    for s in range(32):
        key, val, sh, kb, vb = places(hd, s)
        rec = data[q, h][np.arange(s, slots, 32) // 32]
        K[s::32] = values((rec[:, key] >> sh) & 15, rec[:, kb])
        V[s::32] = values((rec[:, val] >> sh) & 15, rec[:, vb])
    return K, V


def attend(q, data, slots, pos, seq, off, sink, scale):
    """o [rows, hq, hd], and for each output the sum of p |v| and its row's
    largest sum |scale q_d k_d| over the seen positions, with their count."""
    T, hq, hd = q.shape
    hkv = data.shape[1]
    o, pv = np.zeros((T, hq, hd)), np.zeros((T, hq, hd))
    big, cnt = np.zeros((T, hq, 1)), np.zeros((T, hq, 1))
    for i in range(len(pos)):
        r0, r1 = (i, i + 1) if off is None else (off[i], off[i + 1])
        if r1 <= r0 or not 0 <= seq[i] < data.shape[0]:
            continue
        last = pos[i] + r1 - r0 - 1
        idx = np.arange(slots)
        at = last - (last - idx) % slots
        for h in range(hkv):
            K, V = get(data, seq[i], h, slots)
            for r in range(r0, r1):
                see = (at >= 0) & (at <= pos[i] + r - r0)
                for a in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    k, v = K[see], V[see]
                    with np.errstate(all="ignore"):
                        x = (k @ q[r, a]) * scale
                        m = max([-math.inf if sink is None else sink[a]] + ([x.max()] if len(x) else []))
                        if m == -math.inf:
                            continue
                        e = np.exp(x - m)
                        den = e.sum() + (0.0 if sink is None else math.exp(sink[a] - m))
                        o[r, a] = (e[:, None] * v).sum(0) / den
                        pv[r, a] = (e[:, None] * np.abs(v)).sum(0) / den
                        if len(x):
                            big[r, a] = (np.abs(k) @ np.abs(q[r, a])).max() * abs(scale)
                            cnt[r, a] = len(x)
    return o, pv, big, cnt


def attend_tolerance(typ, o, pv, big, cnt, hd, rounded=False):
    """What rounding allows. A score is a sum of at most 3 hd exact products in
    f32, then two multiplications: off by (3 hd + 2) 2^-24 of the sum of its
    terms' sizes. An exponential's relative error is that of its argument
    (in base e) and of exp2 (2 steps) and the subtraction of the maximum
    (2^-24 of a number that the scores' sizes bound). Sums of cnt
    probabilities and of cnt products lose at most cnt 2^-24 each, the pieces'
    joins a few more. A 16-bit output's probabilities are taken to 2^-16 (cut
    to 16 bits), or (rounded: bf16, more than 16 query rows of a key head)
    each rounded once to bf16, by at most half a step, 2^-8. All
    count against sum p |v|, at most twice (in the sum and in the
    denominator); then the output's own rounding."""
    e = EPS["f32"]
    rel = 2 * ((3 * hd + 2) * e * big + 2 * e * big + 4 * e) + (2 * cnt + 32) * e
    if typ != "f32":
        rel = rel + 2 * (2.0 ** -8 if rounded else 2.0 ** -16)
    return rel * pv + EPS[typ] * np.abs(o) + (2.0 ** -25 if typ == "f16" else 1e-37)


def order(x):
    """The indices of a row by value, then lower index; NaN after all."""
    i = np.arange(len(x))
    return np.lexsort((i, -np.where(np.isnan(x), 0.0, x), np.isnan(x)))


def logprobs(x, tok, top):
    """(lp, entropy, rank, top tokens, their lp, E |x - m|) of one row."""
    od = order(x)
    bad = np.isnan(x).any() or (x == math.inf).any()
    if bad:
        lp, ent, ed = np.full(len(x), math.nan), math.nan, 0.0
    elif (x == -math.inf).all():
        lp, ent, ed = np.full(len(x), -math.inf), 0.0, 0.0
    else:
        m = x.max()
        with np.errstate(all="ignore"):
            d = np.where(x == -math.inf, 0.0, x - m)
            e = np.where(x == -math.inf, 0.0, np.exp(d))
            top1 = od[0]
            rest = e.sum() - 1.0 if len(x) < 2 else np.delete(e, top1).sum()
            ls = math.log1p(rest)
            lp = np.where(x == -math.inf, -math.inf, d - ls)
            ed = float((e * -d).sum() / (1.0 + rest))
            ent = ls + ed
    rank = int(np.nonzero(od == tok)[0][0]) if 0 <= tok < len(x) else -1
    return (lp[tok] if rank >= 0 else math.nan), ent, rank, od[:top], lp[od[:top]], ed
