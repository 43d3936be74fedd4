"""The operators on device memory (ana_amd.ops) on the GPU, against their
definitions in 64 bits (device_ops_ref)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import ana_amd
import device_ops_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from ana_amd import ops as o
    return o


def dev(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device="cuda")


def rand(rs, shape, typ, scale=1.0):
    """Random numbers of a type, on the GPU and in 64 bits."""
    t = torch.tensor(rs.randn(*shape) * scale, dtype=torch.float64).to(TYPES[typ])
    return t.cuda(), t.double().numpy()


def garbage(rs, cache):
    """A cache of whatever bytes."""
    cache.data.copy_(torch.tensor(rs.randint(0, 256, tuple(cache.data.shape)), dtype=torch.uint8))
    return cache.data.cpu().numpy().copy()


def rows_of(pos, off, slots):
    """(row, sequence index, position, kept) of a call's rows."""
    out = []
    for i, p in enumerate(pos):
        r0, r1 = (i, i + 1) if off is None else (off[i], off[i + 1])
        for r in range(r0, r1):
            out.append((r, i, p + r - r0, r1 - 1 - r < slots))
    return out


# (type, key heads, hd, slots, sequences in the cache, pos, seq, off)
STORES = [
    ("f32", 3, 64, 70, 5, [0, 33, 69, 500], [4, 0, 2, 1], None),
    ("bf16", 2, 128, 64, 3, [0, 31, 32], None, None),
    ("f16", 1, 32, 1, 2, [7, 0], [1, 0], None),
    ("f32", 2, 32, 33, 4, [0, 5, 20, 31], [3, 1, 0, 2], [0, 1, 20, 20, 33]),
    ("bf16", 12, 64, 97, 3, [90, 0, 1000], [2, 0, 1], [0, 40, 137, 139]),
    ("f16", 5, 128, 40, 2, [3, 0], [1, 0], [0, 90, 130]),
    ("f32", 1, 64, 2048, 1, [0], None, [0, 1]),
]


def expect_store(before, k, v, pos, seq, off, slots):
    want = before.copy()
    kc, ks = ref.quant(k)
    vc, vs = ref.quant(v)
    seen = set()
    for i in range(len(pos)):
        q = i if seq is None else seq[i]
        n = 1 if off is None else off[i + 1] - off[i]
        if n == 0:
            continue
        fresh = q not in seen and 0 <= q < before.shape[0]
        seen.add(q)
        for r, i2, p, kept in rows_of(pos, off, slots):
            if i2 == i and kept and fresh:
                for h in range(k.shape[1]):
                    ref.put(want, q, h, p % slots, kc[r, h], ks[r, h], vc[r, h], vs[r, h])
    return want


@pytest.mark.parametrize("typ,heads,hd,slots,seqs,pos,seq,off", STORES)
def test_write_and_read(ops, typ, heads, hd, slots, seqs, pos, seq, off):
    rs = np.random.RandomState(1)
    rows = len(pos) if off is None else off[-1]
    k, k64 = rand(rs, (rows, heads, hd), typ)
    v, v64 = rand(rs, (rows, heads, hd), typ, 3.0)
    cache = ops.KV4.empty(seqs, slots, heads, hd)
    before = garbage(rs, cache)
    args = dict(seq=None if seq is None else dev(seq), off=None if off is None else dev(off))
    ops.kv4_write(cache, k, v, dev(pos), **args)
    want = expect_store(before, k64, v64, pos, seq, off, slots)
    got = cache.data.cpu().numpy()
    assert np.array_equal(got, want)
    gk, gv = ops.kv4_read(cache, dev(pos), rows, dtype=TYPES[typ], **args)
    gk, gv = gk.double().cpu().numpy(), gv.double().cpu().numpy()
    for r, i, p, kept in rows_of(pos, off, slots):
        q = i if seq is None else seq[i]
        for h in range(heads):
            K, V = ref.get(want, q, h, slots)
            # (whatever the ring holds there now; every value is one of the type)
            assert np.array_equal(gk[r, h], K[p % slots], equal_nan=True)
            assert np.array_equal(gv[r, h], V[p % slots], equal_nan=True)


def test_write_special_values(ops):
    """Borders between codes, signed zeros, subnormal and huge blocks, blocks
    that are not finite."""
    b = np.zeros((12, 32), dtype=np.float32)
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]
    b[0, :8], b[0, 8:16] = ties, [-t for t in ties]
    b[1, :8] = np.nextafter(np.float32(ties), np.float32(0))
    b[1, 8:16] = np.nextafter(np.float32(ties), np.float32(100))
    b[2] = -0.0
    b[3, :4] = [1e-45, -1e-40, 1e-38, 2.0 ** -126]
    b[4, :4] = [3.4028235e38, -2.9e38, 1e38, 1.0]
    b[5, :3] = [1.0, math.inf, 2.0]
    b[6, 31] = math.nan
    b[7, 0], b[7, 1] = -math.inf, math.nan
    b[8, 0] = 7.0 * 2.0 ** 10
    b[9, 0] = np.nextafter(np.float32(7.0 * 2.0 ** 10), np.float32(np.inf))
    b[10, 0], b[10, 1] = 2.0 ** -125 * 7, 2.0 ** -125 * 0.25
    b[11] = np.linspace(-7, 7, 32)
    k = b.reshape(6, 1, 64)
    v = b[::-1].copy().reshape(6, 1, 64)
    cache = ops.KV4.empty(1, 6, 1, 64)
    off = dev([0, 6])
    ops.kv4_write(cache, torch.tensor(k).cuda(), torch.tensor(v).cuda(), dev([0]), off=off)
    want = expect_store(np.zeros((1, 1, 1, 34 * 64), dtype=np.uint8), k, v, [0], None, [0, 6], 6)
    assert np.array_equal(cache.data.cpu().numpy(), want)
    gk, gv = ops.kv4_read(cache, dev([0]), 6, off=off)
    K, V = ref.get(want, 0, 0, 6)
    assert np.array_equal(gk.double().cpu().numpy()[:, 0], K, equal_nan=True)
    assert np.array_equal(gv.double().cpu().numpy()[:, 0], V, equal_nan=True)
    # float16 outputs round once (and what is too large for them is infinite)
    hk, _ = ops.kv4_read(cache, dev([0]), 6, off=off, dtype=torch.float16)
    assert np.array_equal(hk.cpu().numpy(), torch.tensor(K).half().numpy()[:, None], equal_nan=True)


def test_write_twice_listed_and_placeless(ops):
    rs = np.random.RandomState(2)
    pos, seq, off = [4, 9, 4, 0], [1, 7, 1, 0], [2, 5, 8, 11, 12]
    k, k64 = rand(rs, (15, 2, 32), "f32")
    v, v64 = rand(rs, (15, 2, 32), "f32")
    cache = ops.KV4.empty(3, 50, 2, 32)
    before = garbage(rs, cache)
    ops.kv4_write(cache, k, v, dev(pos), seq=dev(seq), off=dev(off))
    want = expect_store(before, k64, v64, pos, seq, off, 50)
    assert np.array_equal(cache.data.cpu().numpy(), want)
    # rows without a place read as zeros
    gk, gv = ops.kv4_read(cache, dev(pos), 15, seq=dev(seq), off=dev(off))
    assert not gk[5:8].any() and not gv[5:8].any()
    assert torch.equal(gk[2:5], gk[8:11])


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("pos,seq,off,live", [
    ([-1, 5], [0, 0], None, [1]),                                          # a padded entry ahead of the real one
    ([-1, -9, 3, 4, 9], [2, 0, 2, 1, 2], None, [2, 3]),                    # then listed twice
    ([-1, 5], [0, 0], [0, 1, 4], [1]),
    ([-2 ** 31, 7, -40, 60, 0], [1, 1, 2, 2, 1], [1, 41, 44, 44, 50, 55], [1, 3])])
def test_write_after_a_listing_without_a_place(ops, typ, pos, seq, off, live):
    """A listing without a place (its first position below zero) takes
    nothing from a later one of the same sequence: `live` is what is stored."""
    rs = np.random.RandomState(16)
    rows = len(pos) if off is None else off[-1]
    k, k64 = rand(rs, (rows, 2, 64), typ)
    v, v64 = rand(rs, (rows, 2, 64), typ)
    cache = ops.KV4.empty(3, 70, 2, 64)
    want = garbage(rs, cache)
    args = dict(seq=dev(seq), off=None if off is None else dev(off))
    ops.kv4_write(cache, k, v, dev(pos), **args)
    (kc, ks), (vc, vs) = ref.quant(k64), ref.quant(v64)
    for i in live:
        r0, r1 = (i, i + 1) if off is None else (off[i], off[i + 1])
        for r in range(r0, r1):
            for h in range(2):
                ref.put(want, seq[i], h, (pos[i] + r - r0) % 70, kc[r, h], ks[r, h], vc[r, h], vs[r, h])
    assert np.array_equal(cache.data.cpu().numpy(), want)


def test_strided_and_unaligned(ops):
    """q, k and v as views of one tensor, and views off every border."""
    rs = np.random.RandomState(3)
    n, h, hd = 5, 3, 64
    for typ, shift, pad in (("f32", 0, 0), ("f32", 1, 3), ("bf16", 3, 1), ("f16", 8, 8)):
        w = 3 * h * hd + pad
        flat, _ = rand(rs, (n * w + 16,), typ)
        x = flat[shift:shift + n * w].view(n, w)
        q, k, v = (x[:, i * h * hd:(i + 1) * h * hd].view(n, h, hd) for i in range(3))
        a, b = ops.KV4.empty(n, 40, h, hd), ops.KV4.empty(n, 40, h, hd)
        pos = dev([0, 3, 39, 41, 7])
        ops.kv4_write(a, k, v, pos)
        ops.kv4_write(b, k.contiguous(), v.contiguous(), pos)
        assert torch.equal(a.data, b.data)
        out = torch.full((n, 2, h, hd + 2), 9.0, dtype=TYPES[typ], device="cuda")
        ops.kv4_attend(q, a, pos, out=out[:, 1, :, 1:hd + 1])
        assert torch.equal(out[:, 1, :, 1:hd + 1], ops.kv4_attend(q.contiguous(), a, pos))
        assert (out[:, 0] == 9).all() and (out[..., 0] == 9).all() and (out[..., hd + 1] == 9).all()
        # heads before rows
        t = q.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(ops.kv4_attend(t, a, pos), ops.kv4_attend(q.contiguous(), a, pos))


def filled(ops, rs, seqs, slots, heads, hd):
    """A cache whose every slot holds numbers as they come."""
    cache = ops.KV4.empty(seqs, slots, heads, hd)
    for q in range(seqs):
        k, _ = rand(rs, (slots, heads, hd), "f32")
        v, _ = rand(rs, (slots, heads, hd), "f32")
        ops.kv4_write(cache, k, v, dev([0]), seq=dev([q]), off=dev([0, slots]))
    return cache


def check_attend(ops, cache, q, q64, typ, pos, seq, off, sink, scale=None, live=0):
    hd = cache.hd
    sk = None if sink is None else torch.tensor(sink, dtype=torch.float32, device="cuda")
    got = ops.kv4_attend(q, cache, dev(pos), seq=None if seq is None else dev(seq),
                         off=None if off is None else dev(off), sink=sk, scale=scale, live=live)
    sc = hd ** -0.5 if scale is None else scale
    where = list(range(len(pos))) if seq is None else seq
    o, pv, big, cnt = ref.attend(q64, cache.data.cpu().numpy(), cache.slots, pos, where, off,
                                 None if sink is None else np.asarray(sink, dtype=np.float32).astype(np.float64), sc)
    many = np.zeros((len(q64), 1, 1), dtype=bool)
    for i in range(len(pos) if off is not None else 0):
        many[off[i]:off[i + 1]] = (off[i + 1] - off[i]) * (q64.shape[1] // cache.heads) > 16
    tol = np.where(many & (typ == "bf16"), ref.attend_tolerance(typ, o, pv, big, cnt, hd, True),
                   ref.attend_tolerance(typ, o, pv, big, cnt, hd))
    g = got.double().cpu().numpy()
    r0, r1 = (0, len(g)) if off is None else (off[0], off[-1])
    err = np.abs(g - o)[r0:r1]
    assert np.isfinite(g[r0:r1]).all()
    assert (err <= tol[r0:r1]).all(), (err - tol[r0:r1]).max()
    return got


# (type, query heads, key heads, hd, slots, pos, off, sink)
ATTENDS = [
    ("f32", 1, 1, 64, 40, [0], None, False),
    ("f32", 3, 3, 64, 2048, [0, 31, 32, 1000, 2047, 5000], None, True),
    ("bf16", 8, 2, 128, 500, [499, 63, 0, 777], None, False),
    ("f16", 5, 1, 32, 97, [96, 15, 16, 17], None, True),
    ("f32", 34, 2, 32, 70, [69, 3, 70], None, True),          # 17 query heads a key head
    ("bf16", 40, 1, 64, 300, [299, 100], None, True),
    ("f32", 6, 3, 64, 300, [0, 10, 200], [0, 3, 10, 12], True),        # few rows each
    ("f32", 3, 3, 64, 700, [0, 0, 100, 650], [0, 130, 131, 331, 345], True),
    ("f32", 4, 2, 128, 400, [0, 37], [0, 200, 333], False),
    ("bf16", 4, 1, 128, 333, [5, 0], [0, 40, 220], True),
    ("f16", 2, 2, 32, 290, [0, 100, 7], [0, 90, 190, 200], False),
    ("f16", 3, 1, 64, 260, [11], [0, 240], True),
    ("bf16", 2, 2, 64, 129, [0], [0, 129], False),
    ("f32", 2, 1, 64, 64, [50, 200, 3], [0, 40, 100, 103], True),      # past the wrap in the call
    ("bf16", 2, 2, 32, 33, [0, 30], [0, 100, 120], False),             # longer than the ring
]


@pytest.mark.parametrize("typ,hq,hkv,hd,slots,pos,off,sink", ATTENDS)
def test_attend(ops, typ, hq, hkv, hd, slots, pos, off, sink):
    rs = np.random.RandomState(4)
    n = len(pos)
    cache = filled(ops, rs, n + 1, slots, hkv, hd)
    rows = n if off is None else off[-1]
    q, q64 = rand(rs, (rows, hq, hd), typ)
    seq = [(i * 3 + 1) % (n + 1) for i in range(n)] if n % 3 != 2 else None
    check_attend(ops, cache, q, q64, typ, pos, seq, off, rs.randn(hq) if sink else None)


@pytest.mark.parametrize("n,hq,hkv,hd,slots,pos", [
    (1, 2, 2, 64, 20000, 19000), (1, 8, 1, 128, 9000, 30000), (3, 4, 4, 32, 6000, 3100), (40, 12, 12, 64, 300, 290)])
def test_attend_split(ops, n, hq, hkv, hd, slots, pos):
    """Few rows over long rings (pieces that are joined), with and without a
    known length."""
    rs = np.random.RandomState(5)
    cache = filled(ops, rs, n, slots, hkv, hd)
    q, q64 = rand(rs, (n, hq, hd), "f32")
    ps = [max(0, pos - 997 * i) for i in range(n)]
    m = min(n, 3)
    a = check_attend(ops, cache, q[:m], q64[:m], "f32", ps[:m], None, None, rs.randn(hq))
    b = check_attend(ops, cache, q[:m], q64[:m], "f32", ps[:m], None, None, None, live=ps[0] + 1)
    assert a.shape == b.shape
    # a length that is too short only splits badly
    check_attend(ops, cache, q[:m], q64[:m], "f32", ps[:m], None, None, None, live=1)
    # every sequence at once gives what each gives alone, to rounding
    both = ops.kv4_attend(q, cache, dev(ps))
    one = torch.cat([ops.kv4_attend(q[i:i + 1], cache, dev(ps[i:i + 1]), seq=dev([i])) for i in range(m)])
    assert (both[:m] - one).abs().max() <= 1e-5 * one.abs().max()


def pieces_of(ops, cache, n, rows, ragged, hq, live=0):
    """The pieces that a call's slots are cut into at most, by its workspace."""
    r = ops._Rows(n, rows, None, 1, 1 if ragged else None)
    ws = ana_amd.lib().ana_kv4_attend_ws(cache._p, ctypes.byref(r), hq, live)
    return max(1, ws // (4 * rows * hq * (4 + cache.hd)))


# (type, query heads, key heads, hd, slots, pos, off)
LONG = [
    ("f32", 2, 2, 64, 20000, [19001], None), ("bf16", 8, 2, 128, 9000, [8999, 30000], None),
    ("f16", 3, 3, 32, 40000, [33333], None), ("bf16", 20, 1, 64, 6000, [5017], None),
    ("f32", 6, 1, 128, 7000, [6999, 3001, 70], None),
    ("f32", 2, 1, 64, 9001, [9000, 4000], [0, 3, 8]), ("bf16", 4, 2, 64, 9000, [8200], [0, 4]),      # few rows
    ("f16", 4, 1, 128, 5000, [4990, 17], [0, 2, 6]),
    ("f32", 2, 2, 64, 12000, [11000, 3000], [0, 70, 120]), ("bf16", 4, 1, 128, 8000, [7000], [0, 90]),  # many
    ("f16", 2, 1, 32, 20000, [19000], [0, 64])]


@pytest.mark.parametrize("typ,hq,hkv,hd,slots,pos,off", LONG)
def test_long_rings_count_every_slot_once(ops, typ, hq, hkv, hd, slots, pos, off):
    """Keys of zero: every seen slot weighs 1, and an output is the mean of
    the values, whose sums are exact (multiples of 1/2 below 2^22), in
    probabilities, over the pieces and in the join. What is left is a
    reciprocal, a product and the output's rounding. A slot that is lost, or
    counted twice, moves the mean (itself a value over the root of their
    number) by a value over their number."""
    rs = np.random.RandomState(17)
    n, rows = len(pos), len(pos) if off is None else off[-1]
    cache = ops.KV4.empty(n, slots, hkv, hd)
    codes = rs.randint(0, 256, tuple(cache.data.shape)).astype(np.uint8)
    codes[..., :16 * hd] = 0
    codes[..., 32 * hd:] = 127
    cache.data.copy_(torch.tensor(codes))
    assert pieces_of(ops, cache, n, rows, off is not None, hq) > 1
    q, _ = rand(rs, (rows, hq, hd), typ)
    G, e = hq // hkv, 2.0 ** -24
    for sink in (None, 0.0):
        sk = None if sink is None else torch.zeros(hq, device="cuda")
        got = ops.kv4_attend(q, cache, dev(pos), off=None if off is None else dev(off), sink=sk).double().cpu().numpy()
        for i in range(n):
            r0, r1 = (i, i + 1) if off is None else (off[i], off[i + 1])
            last = pos[i] + r1 - r0 - 1
            idx = np.arange(slots)
            at = last - (last - idx) % slots
            for h in range(hkv):
                _, V = ref.get(codes, i, h, slots)
                by_at = np.zeros((r1 - r0, hd))
                for r in range(r0, r1):
                    see = (at >= 0) & (at <= pos[i] + r - r0)
                    by_at[r - r0] = V[see].sum(0) / (see.sum() + (0 if sink is None else 1))
                want = by_at[:, None, :]
                g = got[r0:r1, h * G:(h + 1) * G]
                tol = np.abs(want) * (2 * e + e * e + (0.0 if typ == "f32" else ref.EPS[typ] * (1 + 3 * e))) + \
                    (2.0 ** -25 if typ == "f16" else 0.0)
                assert (np.abs(g - want) <= tol).all(), (i, h, sink)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("slots,pos,seq,off", [
    (5000, [4000, -1, 4990, 10], [1, 0, 9, 2], [5, 8, 11, 14, 17]),            # few rows; two without a place
    (5000, [4000, 70, -3, 4980], [1, 0, 2, 2], [7, 60, 100, 140, 200]),        # many
    (700, [3000, 5, 100], [0, 2, 1], [1, 750, 753, 1500]),                     # longer than the ring: rows that see nothing
    (5000, [3000, -1, 9, 4999], [3, 0, 1, 0], None)])
def test_long_rings_rows_outside(ops, typ, slots, pos, seq, off):
    """Calls in pieces: rows of no sequence stay, rows without a place are
    zeros, rows that see nothing are zeros with a sink and without, and the
    others are what they are whole (the 64-bit test has those)."""
    rs = np.random.RandomState(24)
    n, rows = len(pos), len(pos) if off is None else off[-1] + 9
    cache = filled(ops, rs, 4, slots, 2, 64)
    q, _ = rand(rs, (rows, 4, 64), typ)
    args = dict(seq=dev(seq), off=None if off is None else dev(off))
    assert pieces_of(ops, cache, n, rows, off is not None, 4) > 1
    assert pieces_of(ops, cache, n, rows, off is not None, 4, live=1) == 1
    for sink in (None, torch.tensor(rs.randn(4), dtype=torch.float32, device="cuda")):
        got, whole = (torch.full((rows, 4, 64), 3.0, dtype=TYPES[typ], device="cuda") for _ in range(2))
        ops.kv4_attend(q, cache, dev(pos), sink=sink, out=got, **args)
        ops.kv4_attend(q, cache, dev(pos), sink=sink, out=whole, live=1, **args)
        some = torch.zeros(rows, dtype=torch.bool, device="cuda")     # rows of a sequence
        sees = some.clone()
        for i in range(n):
            r0, r1 = (i, i + 1) if off is None else (off[i], off[i + 1])
            some[r0:r1] = True
            sees[max(r0, r1 - slots):r1] = 0 <= pos[i] and 0 <= seq[i] < 4
        assert (got[~some] == 3).all() and not got[some & ~sees].any()
        assert got[sees].abs().amax((1, 2)).min() > 0
        a, b = got[sees].double(), whole[sees].double()
        # each within attend_tolerance of the formula: scores of sizes up to 10 and
        # sums of up to `slots`, against sum p |v| (below the largest value), twice
        v = ops.kv4_read(cache, dev([0] * 4), 4 * slots, off=dev(np.arange(5) * slots))[1].abs().max()
        tol = 2 * (2 * slots + 4096) * 2.0 ** -24 * v
        if typ == "bf16":
            tol = tol + 2 * (2 * 2.0 ** -8 * v + 2.0 ** -8 * b.abs())
        assert ((a - b).abs() <= tol).all()


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_long_rings_find_every_tile(ops, typ, rows):
    """A query that matches one slot's key takes that slot's value, whichever
    tile it is in, over the pieces' different maxima (the last row of each of
    the call's sequences; the ones before it look elsewhere)."""
    rs = np.random.RandomState(18)
    slots, hd = 6000 + 13, 64
    cache = filled(ops, rs, 1, slots, 1, hd)
    K, V = ref.get(cache.data.cpu().numpy(), 0, 0, slots)
    tiles = -(-slots // 32)
    find = np.minimum(np.arange(tiles) * 32 + rs.randint(0, 32, tiles), slots - 1)
    per = 12
    for at in range(0, tiles, per):
        slot = find[at:at + per]
        n = len(slot)
        q64 = rs.standard_normal((n, rows, 2, hd))
        q64[:, -1] = 4.0 * K[slot][:, None]
        q = torch.tensor(q64.reshape(n * rows, 2, hd)).to(TYPES[typ]).cuda()
        off = None if rows == 1 else dev(np.arange(n + 1) * rows)
        pos = dev([slots - rows] * n)
        seq = dev([0] * n)
        if at == 0:
            assert pieces_of(ops, cache, n, n * rows, rows > 1, 2) > 1
        got = ops.kv4_attend(q, cache, pos, seq=seq, off=off).double().cpu().numpy().reshape(n, rows, 2, hd)[:, -1]
        x = q.double().cpu().numpy().reshape(n, rows, 2, hd)[:, -1] @ K.T * hd ** -0.5
        p = np.exp(x - x.max(-1, keepdims=True))
        want = p @ V / p.sum(-1, keepdims=True)
        # (the slot's weight is all but 1: what a wrong piece gives is off by the values' own size)
        assert (p.max(-1) / p.sum(-1) > 0.99).all()
        assert (np.abs(got - want) <= 0.02 * np.abs(V).max()).all(), at


def test_attend_piece_of_a_long_ring(ops):
    """A prompt's piece over a long past: its slots split, then joined."""
    rs = np.random.RandomState(6)
    cache = filled(ops, rs, 1, 4000, 1, 64)
    q, q64 = rand(rs, (50, 2, 64), "f32")
    check_attend(ops, cache, q, q64, "f32", [3900], None, [0, 50], rs.randn(2))
    q, q64 = rand(rs, (50, 2, 64), "bf16")
    check_attend(ops, cache, q, q64, "bf16", [3900], None, [0, 50], None)


def test_attend_score_sizes(ops):
    """Large scores (one position takes all), a negative and a zero scale."""
    rs = np.random.RandomState(7)
    cache = filled(ops, rs, 2, 200, 2, 64)
    q, q64 = rand(rs, (2, 2, 64), "f32", 30.0)
    for scale in (2.0, -0.3, 0.0):
        check_attend(ops, cache, q, q64, "f32", [199, 77], None, None, [0.0, -math.inf], scale=scale)
    q, q64 = rand(rs, (60, 2, 64), "f32", 30.0)
    for scale in (2.0, -0.3, 0.0):
        check_attend(ops, cache, q, q64, "f32", [10], None, [0, 60], [-50.0, 200.0], scale=scale)
    for typ in ("bf16", "f16"):
        for scale in (2.0, -0.3, 0.0):
            q, q64 = rand(rs, (2, 2, 64), typ, 3.0)
            check_attend(ops, cache, q, q64, typ, [199, 77], None, None, None, scale=scale)
            q, q64 = rand(rs, (60, 2, 64), typ, 3.0)
            check_attend(ops, cache, q, q64, typ, [10], None, [0, 60], [0.5, -2.0], scale=scale)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_attend_ignores_what_it_does_not_see(ops, typ):
    """Slots that hold nothing yet, and later rows' keys and values that are
    not finite, do not change a row; those it sees make it NaN (a value only
    in its own dims)."""
    rs = np.random.RandomState(8)
    cache = ops.KV4.empty(2, 100, 1, 64)
    cache.data.fill_(255)
    k, _ = rand(rs, (40, 1, 64), "f32")
    v, _ = rand(rs, (40, 1, 64), "f32")
    clean = ops.KV4.empty(2, 100, 1, 64)
    off = dev([0, 40])
    ops.kv4_write(clean, k, v, dev([0]), off=off)
    k[30, 0, 5] = math.nan
    v[20, 0, 40] = math.inf
    ops.kv4_write(cache, k, v, dev([0]), off=off)
    q, _ = rand(rs, (40, 2, 64), typ)
    want = ops.kv4_attend(q, clean, dev([0]), off=off)
    got = ops.kv4_attend(q, cache, dev([0]), off=off)
    assert torch.equal(got[:20], want[:20])
    assert torch.equal(got[20:30, :, :32], want[20:30, :, :32]) and got[20:30, :, 32:].isnan().all()
    assert got[30:].isnan().all()
    # row by row, as single tokens and in twos
    for p in (19, 20, 29, 30, 39):
        one = ops.kv4_attend(q[p:p + 1], cache, dev([p]), seq=dev([0]))
        w = ops.kv4_attend(q[p:p + 1], clean, dev([p]), seq=dev([0]))
        if p < 20:
            assert torch.equal(one, w)
        elif p < 30:
            assert torch.equal(one[..., :32], w[..., :32]) and one[..., 32:].isnan().all()
        else:
            assert one.isnan().all()
        two = ops.kv4_attend(q[p - 1:p + 1], cache, dev([p - 1]), seq=dev([0]), off=dev([0, 2]))
        assert torch.equal(two[:1].isnan(), got[p - 1:p].isnan()) and torch.equal(two[1:].isnan(), got[p:p + 1].isnan())
    # the second sequence holds nothing but its first token
    ops.kv4_write(cache, k[:1], v[:1], dev([0]), seq=dev([1]))
    one = ops.kv4_attend(q[:1], cache, dev([0]), seq=dev([1]))
    val, _ = ops.kv4_read(cache, dev([0]), 1, seq=dev([1]), dtype=TYPES[typ])[::-1]
    assert (one - val).abs().max() <= 2.0 ** -7 * val.abs().max()


def test_attend_queries_that_are_not_finite(ops):
    rs = np.random.RandomState(9)
    cache = filled(ops, rs, 1, 64, 1, 64)
    for typ in TYPES:
        q, _ = rand(rs, (40, 1, 64), typ)
        off = dev([0, 40])
        want = ops.kv4_attend(q, cache, dev([0]), off=off)
        q[7, 0, 3], q[9, 0, 0] = math.nan, math.inf
        got = ops.kv4_attend(q, cache, dev([0]), off=off)
        rest = [i for i in range(40) if i not in (7, 9)]
        assert torch.equal(got[rest], want[rest]) and got[[7, 9]].isnan().all()


def test_attend_rows_and_places_outside(ops):
    rs = np.random.RandomState(10)
    cache = filled(ops, rs, 2, 50, 2, 32)
    q, q64 = rand(rs, (60, 2, 32), "f32")
    out = torch.full((60, 2, 32), 3.0, device="cuda")
    # sequences without rows, one with no place in the cache; rows 0 .. 4 and
    # 45 .. 59 are nobody's
    off, pos, seq = [5, 5, 30, 40, 40, 45], [1, 2, 3, 4, 5], [0, 1, 2, 1, -1]
    ops.kv4_attend(q, cache, dev(pos), seq=dev(seq), off=dev(off), out=out)
    assert (out[:5] == 3).all() and (out[45:] == 3).all() and not out[30:45].any()
    want = ops.kv4_attend(q[5:30].contiguous(), cache, dev([2]), seq=dev([1]), off=dev([0, 25]))
    assert torch.equal(out[5:30], want)
    # single rows
    one = ops.kv4_attend(q[:3], cache, dev([3, 4, 5]), seq=dev([5, 1, -1]), sink=torch.zeros(2, device="cuda"))
    assert not one[0].any() and not one[2].any() and one[1].any()
    # no rows, no sequences
    assert ops.kv4_attend(q[:0], cache, dev([]), seq=dev([])).shape == (0, 2, 32)
    ops.kv4_write(cache, q[:0], q[:0], dev([]), seq=dev([]))
    # the same sequence read twice
    twice = ops.kv4_attend(q[:2], cache, dev([9, 9]), seq=dev([1, 1]))
    assert torch.equal(twice[1:], ops.kv4_attend(q[1:2], cache, dev([9]), seq=dev([1])))


def test_positions_below_zero_are_no_place(ops):
    """A padded batch's rows at position -1 (and any other past 2^31 - 1):
    nothing stored, zeros read and attended, also with rows that reach 0."""
    rs = np.random.RandomState(15)
    cache = filled(ops, rs, 3, 100, 1, 64)
    before = cache.data.clone()
    k, _ = rand(rs, (45, 1, 64), "f32")
    off, pos = dev([0, 20, 25, 45]), dev([-5, -1, -2 ** 31])
    ops.kv4_write(cache, k, k, pos, off=off)
    ops.kv4_write(cache, k[:3], k[:3], pos)
    assert torch.equal(cache.data, before)
    a, b = ops.kv4_read(cache, pos, 45, off=off)
    assert not a.any() and not b.any()
    for typ in TYPES.values():
        q = k.expand(45, 2, 64).to(typ).contiguous()
        assert not ops.kv4_attend(q, cache, pos, off=off).any()
        assert not ops.kv4_attend(q[:3], cache, pos).any()
    # the largest position there is
    far = dev([2 ** 31 - 1])
    ops.kv4_write(cache, k[:1], k[:1], far, seq=dev([1]))
    x, _ = ops.kv4_read(cache, far, 1, seq=dev([1]))
    c, s = ref.quant(k[:1].double().cpu().numpy())
    assert np.array_equal(x.double().cpu().numpy(), ref.values(c, s))
    assert ops.kv4_attend(k[:1], cache, far, seq=dev([1])).isfinite().all()


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("slots,hq,off", [
    (300, 2, None), (300, 40, None), (9000, 6, None),              # single rows: few heads, many, in pieces
    (300, 6, [0, 1, 90, 101]), (9000, 6, [0, 3, 40, 200])])        # few and many rows, heads that split a part's rows
def test_attend_in_place(ops, typ, slots, hq, off):
    rs = np.random.RandomState(21)
    cache = filled(ops, rs, 3, slots, 2, 64)
    q, _ = rand(rs, (3 if off is None else off[-1], hq, 64), typ)
    pos, o = dev([slots - 220, 5, slots // 2]), None if off is None else dev(off)
    want = ops.kv4_attend(q, cache, pos, off=o)
    assert ops.kv4_attend(q, cache, pos, off=o, out=q) is q
    assert torch.equal(q, want)


def test_attend_many_sequences(ops):
    """More sequences than a wave has lanes, ragged, some empty."""
    rs = np.random.RandomState(11)
    n = 150
    lens = rs.randint(0, 9, n)
    lens[[3, 70, 149]] = [40, 33, 70]
    lens[[0, 64]] = 0
    off = np.concatenate([[0], np.cumsum(lens)])
    pos = rs.randint(0, 60, n)
    cache = filled(ops, rs, 8, 90, 1, 64)
    seq = rs.randint(0, 8, n)
    q, _ = rand(rs, (int(off[-1]), 3, 64), "f32")
    # (reads only: several sequences may share a place)
    got = ops.kv4_attend(q, cache, dev(pos), seq=dev(seq), off=dev(off))
    for i in (1, 3, 63, 65, 70, 127, 128, 149):
        if lens[i]:
            want = ops.kv4_attend(q[off[i]:off[i + 1]].contiguous(), cache, dev(pos[i:i + 1]), seq=dev(seq[i:i + 1]),
                                  off=dev([0, lens[i]]))
            assert (got[off[i]:off[i + 1]] - want).abs().max() <= 2e-6 * want.abs().max()


def test_far_offsets(ops):
    """A cache past 2^32 bytes: its last sequence, head and slots."""
    seqs, slots, heads, hd = 3, 12000000, 1, 128
    data = torch.empty((seqs, heads, slots // 32, 34 * hd), dtype=torch.uint8, device="cuda")
    cache = ops.KV4(data, slots)
    rs = np.random.RandomState(12)
    k, k64 = rand(rs, (40, 1, hd), "bf16")
    v, v64 = rand(rs, (40, 1, hd), "bf16")
    p = slots - 20
    ops.kv4_write(cache, k, v, dev([p]), seq=dev([2]), off=dev([0, 40]))
    gk, gv = ops.kv4_read(cache, dev([p]), 40, seq=dev([2]), off=dev([0, 40]), dtype=torch.bfloat16)
    c, s = ref.quant(k64)
    assert np.array_equal(gk.double().cpu().numpy(), ref.values(c, s))
    c, s = ref.quant(v64)
    assert np.array_equal(gv.double().cpu().numpy(), ref.values(c, s))


def test_attend_captured(ops):
    """A step (write, then attend) captured once and replayed as positions
    move on, with eager work between the replays, on a stream of its own."""
    rs = np.random.RandomState(13)
    n, h, hd, slots = 6, 2, 64, 5000
    cache, twin = ops.KV4.empty(n, slots, h, hd), ops.KV4.empty(n, slots, h, hd)
    k, _ = rand(rs, (n * 300, h, hd), "f32")
    v, _ = rand(rs, (n * 300, h, hd), "f32")
    off = dev([300 * i for i in range(n + 1)])
    for c in (cache, twin):
        ops.kv4_write(c, k, v, dev([0] * n), off=off)
    pos = dev([300 - 7 * i for i in range(n)])
    qkv, _ = rand(rs, (3, n, h, hd), "f32")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.kv4_attend(qkv[0], twin, pos)       # (loads the kernels)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv4_write(cache, qkv[1], qkv[2], pos)
        out = ops.kv4_attend(qkv[0], cache, pos)
    for step in range(4):
        fresh, _ = rand(rs, (3, n, h, hd), "f32")
        qkv.copy_(fresh)
        g.replay()
        ops.kv4_write(twin, qkv[1], qkv[2], pos)
        want = ops.kv4_attend(qkv[0], twin, pos)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(cache.data, twin.data), step
        pos += 1


def test_deterministic(ops):
    rs = np.random.RandomState(14)
    cache = filled(ops, rs, 3, 3000, 2, 64)
    q, _ = rand(rs, (3, 8, 64), "f32")
    a = [ops.kv4_attend(q, cache, dev([2999, 100, 1500])) for _ in range(5)]
    assert all(torch.equal(a[0], x) for x in a)


def test_two_calls_at_once(ops):
    """Two streams' calls side by side, then two graphs replayed side by
    side: each has its own workspaces, and gives what it gives alone."""
    rs = np.random.RandomState(19)
    work = []
    for i in range(2):
        cache = filled(ops, rs, 2, 9000, 2, 64)
        q, _ = rand(rs, (2, 4, 64), "f32")
        rows, _ = rand(rs, (2, 50021), "f32", 3.0)
        work.append((cache, q, dev([8999 - i, 4000]), rows, dev([7, 40000 + i])))

    def one(w):
        cache, q, pos, rows, tok = w
        return [ops.kv4_attend(q, cache, pos), *ops.logprobs(rows, tok, 20)]

    assert pieces_of(ops, work[0][0], 2, 2, False, 4) > 1
    want = [one(w) for w in work]
    assert not torch.equal(want[0][0], want[1][0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(12):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(one(work[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for g in got[i] for a, b in zip(g, want[i])), i
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], [None] * 2
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            outs[i] = one(work[i])
    for step in range(4):
        for w in work:
            w[1].mul_(1.25)
            w[3].mul_(0.75)
        want = [one(w) for w in work]
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i])), (step, i)


# ---------------------------------------------------------------- log probabilities

def check_logprobs(ops, x, tok, top):
    """x on the GPU; every row against the definition."""
    n, vocab = x.shape
    lp, ent, rank, ids, tlp = ops.logprobs(x, None if tok is None else dev(tok), top)
    x64 = x.double().cpu().numpy()
    e = 2.0 ** -24
    for r in range(n):
        w = ref.logprobs(x64[r], -1 if tok is None else int(tok[r]), top)
        # each exponential: its argument's two roundings and exp2's two steps;
        # a thread's chain of at most 33 sums, then 6 + 16 + 7 more
        ls = e * (2 * w[5] + 4 + 64)
        if math.isnan(w[1]):
            assert math.isnan(float(ent[r]))
        else:
            assert abs(float(ent[r]) - w[1]) <= ls + e * (2 * w[5] * (w[5] + 36) + 64 * w[5] + 2 * abs(w[1])) + 1e-38, r
        assert np.array_equal(ids[r].cpu().numpy(), w[3]), r
        got, want = tlp[r].double().cpu().numpy(), w[4]
        fin = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got == -math.inf, want == -math.inf)
        assert (np.abs(got[fin] - want[fin]) <= ls + 3 * e * np.abs(want[fin])).all(), r
        if tok is not None:
            assert int(rank[r]) == w[2], r
            if not math.isfinite(w[0]):
                assert str(float(lp[r])) == str(float(w[0]))
            else:
                assert abs(float(lp[r]) - w[0]) <= ls + 3 * e * abs(w[0]), r
    return lp, ent, rank, ids, tlp


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("n,vocab,top,pad,shift", [
    (1, 1, 1, 0, 0), (1, 2, 0, 0, 1), (3, 7, 7, 1, 0), (2, 63, 20, 0, 3), (1, 258, 5, 0, 0), (4, 2049, 20, 0, 0),
    (2, 8193, 64, 3, 5), (1, 32768, 5, 0, 0), (3, 50021, 40, 1, 1), (300, 500, 10, 5, 2), (260, 33001, 3, 0, 0),
    (1, 600001, 8, 0, 0)])
def test_logprobs(ops, typ, n, vocab, top, pad, shift):
    rs = np.random.RandomState(20)
    flat = torch.tensor(rs.standard_normal(n * (vocab + pad) + 8) * 3.0).to(TYPES[typ]).cuda()
    x = flat[shift:shift + n * (vocab + pad)].view(n, vocab + pad)[:, :vocab]
    pick = min(n, 6)
    tok = rs.randint(0, vocab, n)
    got = ops.logprobs(x, dev(tok), top)
    sel = np.unique(np.concatenate([[0, n - 1], rs.randint(0, n, pick)]))
    sub = check_logprobs(ops, x[torch.tensor(sel).cuda()], tok[sel], top)
    # the rows of a larger call, to rounding (another split)
    for a, b in zip(got, sub):
        b2 = a[torch.tensor(sel).cuda()]
        if a.dtype == torch.int32:
            assert torch.equal(b2, b)
        else:
            assert torch.allclose(b2, b, rtol=1e-5, atol=1e-5)


def test_logprobs_whole_rows(ops):
    """Whole rows a workgroup (many rows), each against the definition."""
    rs = np.random.RandomState(21)
    x = torch.tensor(rs.standard_normal((300, 3001)) * 4).float().cuda()
    tok = rs.randint(0, 3001, 300)
    lp, ent, rank, ids, tlp = ops.logprobs(x, dev(tok), 20)
    x64 = x.double().cpu().numpy()
    for r in range(0, 300, 7):
        w = ref.logprobs(x64[r], int(tok[r]), 20)
        assert np.array_equal(ids[r].cpu().numpy(), w[3]) and int(rank[r]) == w[2]
        assert abs(float(lp[r]) - w[0]) <= 2e-5 and abs(float(ent[r]) - w[1]) <= 2e-5


@pytest.mark.parametrize("vocab", [5, 1000, 9000])
@pytest.mark.parametrize("n", [9, 300])
def test_logprobs_special_rows(ops, vocab, n):
    """Ties (all of a row, many at the border), masks, NaN and infinities,
    probabilities next to 1."""
    rs = np.random.RandomState(22)
    x = rs.standard_normal((9, vocab)).astype(np.float32)
    x[0] = 1.5                                     # all equal
    x[1] = np.where(rs.rand(vocab) < 0.5, 2.0, -3.0)
    x[2, 1:] = -math.inf                           # one token left
    x[3] = -math.inf                               # none
    x[4, 2] = math.nan
    x[5, 1] = math.inf
    x[6] = np.float32(-3.4028235e38)               # the type's lowest everywhere
    x[6, 3] = 100.0
    x[7, 0], x[7, 1:] = 0.0, -30.0 - rs.rand(vocab - 1)
    x[8, :2] = [0.0, -0.0]
    x[8, 2:] = -1.0
    tok = np.array([vocab - 1, 1, 1, 0, 2, 1, 3, 0, 1])
    reps = -(-n // 9)
    t = torch.tensor(np.tile(x, (reps, 1))[:n]).cuda()
    top = min(40, vocab)
    if n == 9:
        lp, ent, rank, ids, tlp = check_logprobs(ops, t, tok, top)
    else:
        lp, ent, rank, ids, tlp = ops.logprobs(t, dev(np.tile(tok, reps)[:n]), top)
        for r in range(9):
            w = ref.logprobs(x[r].astype(np.float64), int(tok[r]), top)
            assert np.array_equal(ids[r].cpu().numpy(), w[3]) and int(rank[r]) == w[2], r
            assert math.isnan(w[0]) == math.isnan(float(lp[r])), r
        assert torch.equal(ids[:9], ids[9:18]) and torch.equal(rank[:9], rank[9:18])
    # a sure pick keeps its own digits: log p = -sum of the others
    w = ref.logprobs(x[7].astype(np.float64), 0, 1)
    assert abs(float(lp[7]) - w[0]) <= 1e-4 * abs(w[0]) and abs(float(ent[7]) - w[1]) <= 1e-4 * w[1]


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,top", [(40007, 64), (40007, 20), (40007, 1), (70001, 25), (300011, 64), (600001, 64)])
def test_logprobs_pieces_of_ties_and_masks(ops, typ, vocab, top):
    """Rows in pieces whose alternatives no bound separates: ties, masks, NaN,
    sorted rows, all of the largest in one piece."""
    rs = np.random.RandomState(23)
    x = rs.standard_normal((11, vocab)).astype(np.float32)
    x[0] = -0.25                                              # all equal
    x[1] = np.arange(vocab) / 4096.0                          # rising
    x[2] = -np.arange(vocab) / 4096.0                         # falling
    x[3] = -math.inf
    x[3, rs.choice(vocab, 10, replace=False)] = rs.standard_normal(10)
    x[4] = -math.inf
    x[4, rs.choice(vocab, 700, replace=False)] = rs.standard_normal(700)
    x[5] = math.nan
    x[5, rs.choice(vocab, 30, replace=False)] = rs.standard_normal(30)
    x[6] = math.nan
    at = rs.choice(vocab, 23, replace=False)
    x[6, at[:20]], x[6, at[20:]] = -math.inf, [1.0, 2.0, 2.0]
    x[7, 5000:5100] += 10
    x[8] = np.where(rs.rand(vocab) < 0.5, 3.0, 2.0)
    x[9] = math.nan
    x[10] = -math.inf
    t = torch.tensor(x).to(TYPES[typ]).cuda()
    tok = np.concatenate([rs.randint(0, vocab, 7), [5050, vocab - 1, 17, vocab // 2]])
    lp, ent, rank, ids, tlp = ops.logprobs(t, dev(tok), top)
    e = 2.0 ** -24
    x64 = t.double().cpu().numpy()
    for r in range(11):
        w = ref.logprobs(x64[r], int(tok[r]), top)
        assert np.array_equal(ids[r].cpu().numpy(), w[3]) and int(rank[r]) == w[2], r
        # each exponential as in check_logprobs; a thread's chain of at most
        # 66 sums, then 6 + 4 over the workgroup and 6 + 4 in the join
        tol = e * (2 * w[5] + 4 + 86)
        got, want = np.append(tlp[r].double().cpu().numpy(), float(lp[r])), np.append(w[4], w[0])
        fin = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got == -math.inf, want == -math.inf), r
        assert (np.abs(got[fin] - want[fin]) <= tol + 3 * e * np.abs(want[fin])).all(), r


def test_logprobs_token_outside_and_none(ops):
    x = torch.randn(4, 100, device="cuda")
    lp, ent, rank, ids, tlp = ops.logprobs(x, dev([100, -1, 99, 2 ** 31 - 1]), 0)
    assert lp.isnan().tolist() == [True, True, False, True] and rank[[0, 1, 3]].tolist() == [-1, -1, -1]
    assert ids.shape == (4, 0) and tlp.shape == (4, 0)
    lp, ent2, rank, ids, tlp = ops.logprobs(x, None, 3)
    assert lp is None and rank is None and torch.equal(ent, ent2)
    assert ops.logprobs(x[:0], dev([]), 2)[3].shape == (0, 2)


def test_logprobs_captured(ops):
    x = torch.randn(3, 32768, device="cuda")
    tok = dev([5, 6, 7])
    ops.logprobs(x, tok, 5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.logprobs(x, tok, 5)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        tok += 11
        g.replay()
        want = ops.logprobs(x, tok, 5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


# ---------------------------------------------------------------- together

def test_a_served_step(ops):
    """Prompts stored and attended, then single tokens, then the log
    probabilities of what a head makes of the outputs: the two forms agree
    where they see the same, and picks carry rank 0."""
    rs = np.random.RandomState(30)
    n, h, hd, slots = 3, 2, 64, 80
    lens = [50, 7, 20]
    off = np.concatenate([[0], np.cumsum(lens)])
    T = int(off[-1])
    q, _ = rand(rs, (T, 2 * h, hd), "f32")
    k, _ = rand(rs, (T, h, hd), "f32")
    v, _ = rand(rs, (T, h, hd), "f32")
    whole, steps = ops.KV4.empty(n, slots, h, hd), ops.KV4.empty(n, slots, h, hd)
    ops.kv4_write(whole, k, v, dev([0] * n), off=dev(off))
    o = ops.kv4_attend(q, whole, dev([0] * n), off=dev(off))
    last = torch.empty((n, 2 * h, hd), device="cuda")
    for i in range(n):
        for t in range(lens[i]):
            r = int(off[i]) + t
            ops.kv4_write(steps, k[r:r + 1], v[r:r + 1], dev([t]), seq=dev([i]))
            if t == lens[i] - 1:
                last[i] = ops.kv4_attend(q[r:r + 1], steps, dev([t]), seq=dev([i]))[0]
    assert torch.equal(whole.data, steps.data)
    ends = torch.tensor(off[1:] - 1).cuda()
    assert (o[ends] - last).abs().max() <= 2e-6 * last.abs().max()
    w = torch.randn(2 * h * hd, 1000, device="cuda")
    logits = last.view(n, -1) @ w
    picks = logits.argmax(-1).to(torch.int32)
    lp, ent, rank, ids, tlp = ops.logprobs(logits, picks, 4)
    assert rank.tolist() == [0] * n and torch.equal(ids[:, 0], picks) and torch.equal(tlp[:, 0], lp)
    assert (tlp.exp().sum(-1) <= 1.0 + 1e-5).all() and (ent >= 0).all()
