"""The operators on device memory whose speed is measured: their inputs, their
plain form, the calls of ana_amd.ops, and their results in 64 bits.

Three kinds of case, one operator's pass each:

- "store": new keys and values go into a cache held in 4 bits, and the rows
  just stored come back as the values the cache stands for (what a program
  that checks, moves or replays a sequence's state reads). kv4_write, then
  kv4_read.
- "attend": softmax attention of query rows over such a cache. kv4_attend.
- "logprobs": of each row of logits, the log probability and the rank of a
  given token, the distribution's entropy and its likeliest tokens.
  logprobs.

A case is a dict of plain values. For "store" and "attend":

- n sequences in a cache of rings of `slots` positions, hkv heads of hd
  values (hq query heads share them, hq / hkv each);
- past: the tokens the first sequence holds before the call; the others' go
  down evenly to past - past_spread;
- rows: the tokens of the first sequence in the call (0: one token of each
  sequence, the decode form); the others' go down evenly to rows -
  rows_spread;
- sink: whether each query head has a sink logit;
- type: the keys', values', queries' and outputs' ("f32", "bf16", "f16").

For "logprobs": n rows of `vocab` logits, pad more elements between rows, top
alternatives, the logits' type.

The cache's bytes. A cache is uint8 [seqs, hkv, ceil(slots / 32), 34 hd]: a
record holds 32 slots of one head. A value is an E2M1 code (sign, then 0, 0.5,
1, 1.5, 2, 3, 4, 6), 32 values next to each other along a head share an E8M0
scale (a byte b stands for 2^(b - 127), 255 for a block that is not finite;
OCP's microscaling format MXFP4). With D = hd and the even dimension in a
byte's low half, a record is

    keys    [4 j][16 m][2 h][D / 8 bytes]   slot 16 h + m, dims j D / 4 ...
    values  [4 j][16 m][8 e][D / 32 bytes]  slot 16 (e / 4) + 4 j + e % 4, dims m D / 16 ...
    scales of the keys    [D / 32 blocks][16 m][2 h]
    scales of the values  [D / 32 blocks][4 j][8 e]

A block with largest magnitude a takes the least scale with a <= 7 scale, each
value the code nearest to it (ties to the even code; 7 scale is as far from
the largest code as 5 scale is from the two next to it); bytes go from 2 to 252,
where every value is an ordinary number.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------- the cases

def _store(name, type, n, heads, hd, slots, past, past_spread, rows, rows_spread):
    c = {"kind": "store", "type": type, "n": n, "hq": heads, "hkv": heads, "hd": hd, "slots": slots, "past": past,
         "past_spread": past_spread, "rows": rows, "rows_spread": rows_spread, "sink": False}
    return dict(c, name=name) if name else c


def _attend(name, type, n, hq, hkv, hd, slots, past, past_spread, rows, rows_spread, sink):
    c = {"kind": "attend", "type": type, "n": n, "hq": hq, "hkv": hkv, "hd": hd, "slots": slots, "past": past,
         "past_spread": past_spread, "rows": rows, "rows_spread": rows_spread, "sink": sink}
    return dict(c, name=name) if name else c


def _logprobs(name, type, n, vocab, pad, top):
    c = {"kind": "logprobs", "type": type, "n": n, "vocab": vocab, "pad": pad, "top": top}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decode step of a batch of 64 (12 heads of 64, rings of 2048, as
        # the 115M model has them): each sequence's new key and value
        _store("store_64_step", "f32", 64, 12, 64, 2048, 1930, 700, 0, 0),
        # a prefill step of 16 ragged prompts, about 8192 rows
        _store("store_16_prompts", "f32", 16, 12, 64, 2048, 0, 0, 640, 250),
        # the next piece of four long documents, wide heads, 16-bit activations
        _store("store_4_pieces", "bf16", 4, 8, 128, 32768, 20001, 9000, 4096, 0),
        # one user's stream early in its window: a call whose latency counts
        _attend("attend_1_short", "f32", 1, 12, 12, 64, 2048, 300, 0, 0, 0, True),
        # a batch of 64 conversations of all lengths
        _attend("attend_64_ragged", "f32", 64, 12, 12, 64, 2048, 1930, 1700, 0, 0, True),
        # a full batch past the rings' wrap
        _attend("attend_256_full", "f32", 256, 12, 12, 64, 2048, 3000, 900, 0, 0, True),
        # a few very long documents, query heads sharing keys and values
        _attend("attend_4_long", "bf16", 4, 32, 8, 128, 131072, 131071, 30011, 0, 0, False),
        # 16 fresh ragged prompts in one prefill step
        _attend("attend_16_prompts", "f32", 16, 12, 12, 64, 2048, 0, 0, 640, 250, True),
        # the next piece of two long documents
        _attend("attend_2_pieces", "bf16", 2, 16, 4, 128, 32768, 30000, 4001, 1024, 100, False),
        # one user's pick with its alternatives (a streamed answer's log
        # probabilities): vocabulary 32768, as the 115M model's
        _logprobs("logprobs_1", "f32", 1, 32768, 0, 5),
        # the rows of one scoring step
        _logprobs("logprobs_512", "f32", 512, 32768, 0, 20),
        # a training or evaluation batch in 16 bits, an odd vocabulary, padded
        # rows: ties everywhere
        _logprobs("logprobs_3000_odd", "bf16", 3000, 50021, 3, 8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "logprobs", "logprobs"])
    type = rng.choice(["f32", "f32", "bf16", "f16"])
    if kind == "logprobs":
        vocab = _log(rng, 200, 200000)
        return _logprobs("", type, _log(rng, 1, min(4000, 150000000 // vocab)), vocab, rng.choice([0, 0, 1, 5]),
                         rng.choice([0, 1, 5, 20, 40]))
    hd = rng.choice([32, 64, 64, 128])
    hkv = _log(rng, 1, 1536 // hd)
    if rng.random() < 0.5:
        # single tokens over rings of any length
        n, slots = _log(rng, 1, 256), _log(rng, 33, 131072)
        slots = max(33, min(slots, 400000000 // (n * hkv * hd)))
        past = _log(rng, 1, 2 * slots)
        rows = rows_spread = 0
        past_spread = rng.randrange(0, past)
    else:
        # pieces of prompts that end at the rings' end at the latest
        n, rows = _log(rng, 1, 24), _log(rng, 2, 1500)
        rows_spread = rng.randrange(0, rows)
        past = rng.choice([0, _log(rng, 1, max(2, 60000 // n))])
        past_spread = rng.randrange(0, past) if past else 0
        slots = past + rows + rng.randrange(0, 100)
    if kind == "store":
        return _store("", type, n, hkv, hd, slots, past, past_spread, rows, rows_spread)
    hq = hkv * rng.choice([1, 1, 2, 4, 8] if hkv * hd <= 512 else [1, 1, 2])
    return _attend("", type, n, hq, hkv, hd, slots, past, past_spread, rows, rows_spread, rng.random() < 0.5)


# ---------------------------------------------------------------- the inputs

def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _lengths(case):
    """Each sequence's tokens before the call, and in it."""
    n = case["n"]
    past = [case["past"] - case["past_spread"] * i // n for i in range(n)]
    rows = [max(1, case["rows"] - case["rows_spread"] * i // n) for i in range(n)]
    return past, rows


def _generator(seed):
    g = torch.Generator(device=_device())
    g.manual_seed(seed)
    return g


def _normal(g, shape, type):
    return torch.randn(shape, generator=g, device=g.device, dtype=torch.float32).to(TYPES[type])


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "logprobs":
        n, vocab = case["n"], case["vocab"]
        # a head's logits: most tokens far below the few that come into
        # question, more sharply in some rows than in others
        x = torch.randn((n, vocab + case["pad"]), generator=g, device=g.device, dtype=torch.float32)
        sharp = torch.rand((n, 1), generator=g, device=g.device) * 4.0 + 1.0
        logits = x.mul_(sharp).to(TYPES[case["type"]])[:, :vocab]
        # given tokens: likely ones and any others
        likely = (logits.float() + 3.0 * torch.rand((n, vocab), generator=g, device=g.device)).argmax(-1)
        other = torch.randint(0, vocab, (n,), generator=g, device=g.device)
        pick = torch.rand(n, generator=g, device=g.device) < 0.7
        return {"case": case, "logits": logits, "tokens": torch.where(pick, likely, other).to(torch.int32)}
    n, hkv, hd, slots = case["n"], case["hkv"], case["hd"], case["slots"]
    past, rows = _lengths(case)
    total = sum(rows)
    dev = g.device
    # the sequences sit in the cache in any order
    seq = torch.randperm(n, generator=g, device=dev).to(torch.int32)
    s = {"case": case, "seq": seq, "pos": torch.tensor(past, dtype=torch.int32, device=dev), "off": None,
         "total": total, "past": past, "rows": rows}
    if case["rows"]:
        s["off"] = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device=dev)
    data = torch.zeros((n, hkv, -(-slots // 32), 34 * hd), dtype=torch.uint8, device=dev)
    s["data"] = data
    if case["kind"] == "store":
        s["k"] = _normal(g, (total, hkv, hd), case["type"])
        s["v"] = _normal(g, (total, hkv, hd), case["type"])
    else:
        s["q"] = _normal(g, (total, case["hq"], hd), case["type"])
        s["sink"] = torch.randn(case["hq"], generator=g, device=dev) if case["sink"] else None
        s["scale"] = 1.0 / math.sqrt(hd)
        # the live slots hold keys and values as a model makes them, the
        # others what was there before
        live = min(slots, max(p + r for p, r in zip(past, rows)))
        tiles = -(-live // 32)
        for i in range(n):
            k = torch.randn((hkv, tiles * 32, hd), generator=g, device=dev)
            v = torch.randn((hkv, tiles * 32, hd), generator=g, device=dev)
            _put(data[i], k, v)
    if own:
        from ana_amd import ops
        s["cache"] = ops.KV4(data, slots)
    return s


# ---------------------------------------------------------------- the plain form

def _codes(x):
    """Blocks of 32 values [..., 32] as codes 0 .. 15 and a scale byte each."""
    a = x.abs().amax(-1)
    bits = a.view(torch.int32)
    e = ((bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)).clamp(2, 252)
    y = x * ((254 - e) << 23).view(torch.float32).unsqueeze(-1)
    m = y.abs()
    # a tie goes to the even code: the borders 0.25, 1.25, 2.5 and 5 stay below
    c = ((m > 0.25).to(torch.uint8) + (m >= 0.75).to(torch.uint8) + (m > 1.25).to(torch.uint8)
         + (m >= 1.75).to(torch.uint8) + (m > 2.5).to(torch.uint8) + (m >= 3.5).to(torch.uint8)
         + (m > 5.0).to(torch.uint8))
    c += torch.signbit(x).to(torch.uint8) << 3
    bad = ~torch.isfinite(a)
    return torch.where(bad.unsqueeze(-1), 0, c), torch.where(bad, 255, e).to(torch.uint8)


def _pairs(c):
    """Codes packed two a byte, the first in the low half."""
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _parts(data):
    """The four parts of a cache's records as views [..., their extents]."""
    hd = data.shape[-1] // 34
    lead = data.shape[:-1]
    return (data[..., :16 * hd].unflatten(-1, (4, 16, 2, hd // 8)),
            data[..., 16 * hd:32 * hd].unflatten(-1, (4, 16, 2, 4, hd // 32)),
            data[..., 32 * hd:33 * hd].unflatten(-1, (hd // 32, 16, 2)),
            data[..., 33 * hd:].unflatten(-1, (hd // 32, 4, 2, 4))), lead, hd


def _put(data, k, v):
    """k and v [hkv, slots, hd] from slot 0 of one sequence's records (whole
    tiles of 32 slots)."""
    tiles = k.shape[1] // 32
    (ko, vo, ks, vs), _, hd = _parts(data[:, :tiles])
    h = k.shape[0]
    ck, ek = _codes(k.view(h, tiles, 32, hd // 32, 32))
    cv, ev = _codes(v.view(h, tiles, 32, hd // 32, 32))
    # slot 16 h + m, dim j hd / 4 + ...
    ko.copy_(_pairs(ck.reshape(h, tiles, 2, 16, 4, hd // 4)).permute(0, 1, 4, 3, 2, 5))
    # slot 16 x + 4 j + y, dim m hd / 16 + ...
    vo.copy_(_pairs(cv.reshape(h, tiles, 2, 4, 4, 16, hd // 16)).permute(0, 1, 3, 5, 2, 4, 6))
    ks.copy_(ek.view(h, tiles, 2, 16, hd // 32).permute(0, 1, 4, 3, 2))
    vs.copy_(ev.view(h, tiles, 2, 4, 4, hd // 32).permute(0, 1, 5, 3, 2, 4))


_LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _values(codes, scales, table):
    """Bytes [..., 16] of blocks and their scale bytes [...] as values [..., 32]."""
    x = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).flatten(-2)
    s = scales.int()
    f = torch.where(s == 255, math.nan, (s << 23).view(torch.float32))
    return x * f.unsqueeze(-1)


def _table(dev):
    return torch.tensor(_LEVELS + [-x for x in _LEVELS], dtype=torch.float32, device=dev)


def _unpack(data):
    """The keys and values [..., slots, hd] of records [..., tiles, 34 hd]."""
    (ko, vo, ks, vs), lead, hd = _parts(data)
    t, nd = _table(data.device), len(lead)
    a = list(range(nd))
    kc = ko.permute(*a, nd + 2, nd + 1, nd, nd + 3).reshape(*lead, 32, hd // 32, 16)
    vc = vo.permute(*a, nd + 2, nd, nd + 3, nd + 1, nd + 4).reshape(*lead, 32, hd // 32, 16)
    kc = _values(kc, ks.permute(*a, nd + 2, nd + 1, nd).reshape(*lead, 32, hd // 32), t)
    vc = _values(vc, vs.permute(*a, nd + 2, nd + 1, nd + 3, nd).reshape(*lead, 32, hd // 32), t)
    flat = (*lead[:-1], lead[-1] * 32, hd)
    return kc.reshape(flat), vc.reshape(flat)


def _row_places(s):
    """Each row's place in the cache's first axis and its position."""
    case, dev = s["case"], s["data"].device
    if s["off"] is None:
        return s["seq"].long(), s["pos"].long()
    i = torch.repeat_interleave(torch.arange(case["n"], device=dev), s["off"].diff(), output_size=s["total"])
    return s["seq"].long()[i], s["pos"].long()[i] + torch.arange(s["total"], device=dev) - s["off"].long()[i]


def _plain_store(s):
    case = s["case"]
    hd, h, T = case["hd"], case["hkv"], s["total"]
    where, pos = _row_places(s)
    slot = pos % case["slots"]
    tile, m = slot // 32, slot % 32
    (ko, vo, ks, vs), _, _ = _parts(s["data"])
    ck, ek = _codes(s["k"].float().view(T, h, hd // 32, 32))
    cv, ev = _codes(s["v"].float().view(T, h, hd // 32, 32))
    # (the indexed axes come first in an assignment through several of them)
    pk, pv = _pairs(ck.reshape(T, h, 4, hd // 4)), _pairs(cv.reshape(T, h, 16, hd // 16))
    at = (where, slice(None), tile)
    ko[(*at, slice(None), m % 16, m // 16)] = pk
    vo[(*at, m % 16 // 4, slice(None), m // 16, m % 4)] = pv
    ks[(*at, slice(None), m % 16, m // 16)] = ek
    vs[(*at, slice(None), m % 16 // 4, m // 16, m % 4)] = ev
    # the rows back as values
    t = _table(s["data"].device)
    gk = ko[(*at, slice(None), m % 16, m // 16)].reshape(T, h, hd // 32, 16)
    gv = vo[(*at, m % 16 // 4, slice(None), m // 16, m % 4)].reshape(T, h, hd // 32, 16)
    k = _values(gk, ks[(*at, slice(None), m % 16, m // 16)], t)
    v = _values(gv, vs[(*at, slice(None), m % 16 // 4, m // 16, m % 4)], t)
    return k.view(T, h, hd).to(s["k"].dtype), v.view(T, h, hd).to(s["v"].dtype)


def _softmax_sum(sc, seen, v, sink):
    """Rows of scores [..., g, r, slots] (seen where they count) over v
    [..., slots, hd], with the heads' sinks [..., g, 1, 1]."""
    sc = torch.where(seen, sc, -math.inf)
    top = sc.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink)
    e = torch.exp(sc - top)
    den = e.sum(-1, keepdim=True)
    if sink is not None:
        den = den + torch.exp(sink - top)
    shape = e.shape
    o = torch.matmul(e.reshape(*shape[:-3], shape[-3] * shape[-2], shape[-1]), v)
    return o.view(*shape[:-1], v.shape[-1]) / den


def _plain_attend(s):
    case = s["case"]
    n, hq, hkv, hd, slots = case["n"], case["hq"], case["hkv"], case["hd"], case["slots"]
    G = hq // hkv
    q, data = s["q"].float() * s["scale"], s["data"]
    sink = None if s["sink"] is None else s["sink"].view(hkv, G, 1, 1)
    if s["off"] is None:
        # every sequence at once, over as many slots as the longest has live
        live = min(slots, max(s["past"]) + 1)
        k, v = _unpack(data[:, :, :-(-live // 32)][s["seq"].long()])
        sc = torch.matmul(q.view(n, hkv, G, hd), k.transpose(-1, -2)).unsqueeze(-2)
        at = torch.arange(sc.shape[-1], device=q.device)
        seen = at < torch.clamp(s["pos"].long() + 1, max=slots).view(n, 1, 1, 1, 1)
        return _softmax_sum(sc, seen, v, sink).reshape(n, hq, hd).to(s["q"].dtype)
    out, r0 = torch.empty_like(s["q"]), 0
    for i in range(n):
        T, last = s["rows"][i], s["past"][i] + s["rows"][i] - 1
        live = min(slots, last + 1)
        k, v = _unpack(data[:, :, :-(-live // 32)].index_select(0, s["seq"][i:i + 1].long())[0])
        qi = q[r0:r0 + T].view(T, hkv, G, hd).permute(1, 2, 0, 3)
        sc = torch.matmul(qi.reshape(hkv, G * T, hd), k.transpose(-1, -2)).view(hkv, G, T, -1)
        at = torch.arange(sc.shape[-1], device=q.device)
        at = torch.where(at < slots, last - (last - at) % slots, -1)     # the position a slot holds
        p = s["past"][i] + torch.arange(T, device=q.device)
        seen = (at >= 0) & (at <= p[:, None])
        o = _softmax_sum(sc, seen, v, sink)
        out[r0:r0 + T] = o.permute(2, 0, 1, 3).reshape(T, hq, hd).to(out.dtype)
        r0 += T
    return out


def _keys(x):
    """Whole numbers in the order of logits: larger ones first, then the
    lower index."""
    b = x.view(torch.int32).long()
    o = torch.where(b < 0, -(b & 0x7FFFFFFF), b)
    return (o << 32) - torch.arange(x.shape[-1], device=x.device)


def _plain_logprobs(s):
    x, tok, top = s["logits"].float(), s["tokens"].long().unsqueeze(-1), s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = torch.log(z)
    # (sums of p (x - m) are far smaller than those of p x)
    ent = lse - (e * (x - m)).sum(-1, keepdim=True) / z
    own_x = torch.gather(x, 1, tok)
    at = torch.arange(x.shape[-1], device=x.device)
    rank = ((x > own_x) | ((x == own_x) & (at < tok))).sum(-1)
    ids = torch.topk(_keys(x), top, dim=-1).indices
    return {"logprob": (own_x - m - lse).squeeze(-1), "entropy": ent.squeeze(-1), "rank": rank.to(torch.int32),
            "top": ids.to(torch.int32), "top_logprob": torch.gather(x, 1, ids) - m - lse}


def run(s):
    case = s["case"]
    if not own:
        return {"store": _plain_store, "attend": _plain_attend, "logprobs": _plain_logprobs}[case["kind"]](s)
    from ana_amd import ops
    if case["kind"] == "store":
        ops.kv4_write(s["cache"], s["k"], s["v"], s["pos"], seq=s["seq"], off=s["off"])
        return ops.kv4_read(s["cache"], s["pos"], s["total"], seq=s["seq"], off=s["off"], dtype=s["k"].dtype)
    if case["kind"] == "attend":
        return ops.kv4_attend(s["q"], s["cache"], s["pos"], seq=s["seq"], off=s["off"], sink=s["sink"],
                              scale=s["scale"])
    lp, ent, rank, ids, tlp = ops.logprobs(s["logits"], s["tokens"], top=case["top"])
    return {"logprob": lp, "entropy": ent, "rank": rank, "top": ids, "top_logprob": tlp}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    b = BYTES[case["type"]]
    if case["kind"] == "logprobs":
        n, v = case["n"], case["vocab"]
        # an exponential and two sums a logit, and the comparisons
        return {"bytes": n * (v * b + 4.0 * (4 + 2 * case["top"])), "flops": 6.0 * n * v}
    past, rows = _lengths(case)
    total, hd, hkv, hq = sum(rows), case["hd"], case["hkv"], case["hq"]
    code = 34.0 / 32.0 * hd * hkv              # a position's keys and values in the cache
    if case["kind"] == "store":
        one = 2.0 * hkv * hd
        return {"bytes": total * (2.0 * one * b + code), "flops": 4.0 * total * one}
    by, fl = 2.0 * total * hq * hd * b, 0.0
    for p, r in zip(past, rows):
        last = p + r - 1
        by += code * min(case["slots"], last + 1)
        # a row sees the positions up to its own that the ring still holds
        first = max(0, last + 1 - case["slots"])
        fl += 4.0 * hq * hd * sum(range(p + 1 - first, last + 2 - first))
    return {"bytes": by, "flops": fl}


# ---------------------------------------------------------------- in 64 bits

def _nearest(x):
    """Blocks of 32 values in 64 bits, each as the value its code stands for."""
    dev = x.device
    a = x.abs().max(-1, keepdim=True).values
    # the least power of two with a <= 7 of it
    e = torch.ceil(torch.log2(a / 7.0).clamp(min=-125.0))
    e = e + (a > 7.0 * torch.exp2(e)).double() - (a <= 3.5 * torch.exp2(e)).double()
    scale = torch.exp2(e.clamp(min=-125.0))
    levels = torch.tensor(_LEVELS, dtype=torch.float64, device=dev)
    even = torch.tensor([0, 2, 4, 6], device=dev)
    d = ((x / scale).abs().unsqueeze(-1) - levels).abs()
    d[..., even] -= 1e-12
    return torch.copysign(levels[d.argmin(-1)], x) * scale


def _record_bytes(hd):
    """Where in a record each slot's and dimension's key and value codes are
    (the byte, the bits' shift) and their blocks' scales."""
    s, d = np.meshgrid(np.arange(32), np.arange(hd), indexing="ij")
    j, h, m = d // (hd // 4), s // 16, s % 16
    key = ((j * 16 + m) * 2 + h) * (hd // 8) + d % (hd // 4) // 2
    jv, ev, mv = s % 16 // 4, s // 16 * 4 + s % 4, d // (hd // 16)
    val = 16 * hd + ((jv * 16 + mv) * 8 + ev) * (hd // 32) + d % (hd // 16) // 2
    ks = 32 * hd + (d // 32 * 16 + m) * 2 + h
    vs = 33 * hd + (d // 32 * 4 + jv) * 8 + ev
    return [torch.from_numpy(a.reshape(-1)).to(_device()) for a in (key, val, ks, vs, d % 2 * 4)]


def _read64(rec, at):
    """Records [..., 34 hd] as keys and values [..., 32 hd] in 64 bits."""
    key, val, ks, vs, shift = at
    levels = torch.tensor(_LEVELS + [-x for x in _LEVELS], dtype=torch.float64, device=rec.device)
    two = torch.exp2(torch.arange(256, dtype=torch.float64, device=rec.device) - 127.0)
    out = []
    for c, b in ((key, ks), (val, vs)):
        out.append(levels[(rec[..., c].long() >> shift) & 15] * two[rec[..., b].long()])
    return out


def _attend64(case, s):
    hq, hkv, hd, slots = case["hq"], case["hkv"], case["hd"], case["slots"]
    G, at, r0, outs = hq // hkv, _record_bytes(hd), 0, []
    for i in range(case["n"]):
        T, p0 = s["rows"][i], s["past"][i]
        last = p0 + T - 1
        live = min(slots, last + 1)
        o = torch.empty((T, hkv, G, hd), dtype=torch.float64, device=s["q"].device)
        idx = torch.arange(live, device=o.device)
        turn = last // slots * slots
        at_pos = torch.where(idx <= last - turn, turn + idx, turn - slots + idx)
        p = p0 + torch.arange(T, device=o.device)
        hide = at_pos[None, :] > p[:, None]
        for h in range(hkv):
            k, v = (x.view(-1, hd)[:live] for x in _read64(s["data"][int(s["seq"][i]), h, :-(-live // 32)], at))
            kt = k.t().contiguous()
            for g in range(G):
                sc = s["q"][r0:r0 + T, h * G + g].double() @ kt * s["scale"]
                sc = sc.masked_fill(hide, -math.inf)
                if s["sink"] is not None:
                    sc = torch.cat([sc, s["sink"][h * G + g].double().expand(T, 1)], -1)
                o[:, h, g] = torch.softmax(sc, -1)[:, :live] @ v
        outs.append(o.view(T, hq, hd))
        r0 += T
    return torch.cat(outs)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        hd = case["hd"]
        return tuple(_nearest(s[x].double().unflatten(-1, (hd // 32, 32))).flatten(-2) for x in "kv")
    if case["kind"] == "attend":
        return _attend64(case, s)
    n, top = case["n"], case["top"]
    out = {k: [] for k in ("logprob", "entropy", "rank", "top", "top_logprob")}
    for r in range(0, n, 64):
        x = s["logits"][r:r + 64].double()
        tok = s["tokens"][r:r + 64].long()
        lp = torch.log_softmax(x, -1)
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices
        out["logprob"].append(lp[torch.arange(len(tok), device=x.device), tok])
        out["entropy"].append(-(lp.exp() * lp).sum(-1))
        out["rank"].append((order == tok[:, None]).int().argmax(-1).to(torch.int32))
        out["top"].append(order[:, :top].to(torch.int32))
        out["top_logprob"].append(torch.gather(lp, 1, order[:, :top]))
    return {k: torch.cat(v) for k, v in out.items()}
