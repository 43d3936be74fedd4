"""Rotation with head norms, attention behind shared prefixes and sampling
(ana_amd.ops) on the GPU, against their definitions in 64 bits
(serve_ops_ref)."""
import math

import numpy as np
import pytest
import torch

import ana_amd
import device_ops_ref as ref
import serve_ops_ref as sref

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


def host(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------------- qk_rope

def freqs(rot, base=10000.0):
    return (base ** (-2.0 * np.arange(rot // 2) / max(rot, 1))).astype(np.float32)


def positions(pos, off, rows):
    """Each row's position; -1 for a row whose sequence has none, -2 of no sequence."""
    out = np.full(rows, -2, dtype=np.int64)
    for i, p in enumerate(pos):
        r0, r1 = (i, i + 1) if off is None else (off[i], off[i + 1])
        out[r0:r1] = p + np.arange(r1 - r0) if p >= 0 else -1
    return out


def check_rope(typ, got, x64, at, freq, gain, eps, near, before=None):
    o, off = sref.rope(x64, np.maximum(at, 0), freq, gain, eps, near)
    o[at == -1], off[at == -1] = 0.0, 0.0
    g = host(got)
    on = at >= -1
    assert (np.abs(g - o)[on] <= sref.rope_tolerance(typ, o, off)[on]).all()
    if before is not None:
        assert np.array_equal(g[~on], before[~on])


# (type, hq, hk, hd, rot, near, norms, pos, off)
ROPES = [
    ("f32", 12, 12, 64, 64, False, True, [300], None),
    ("f32", 1, 1, 16, 16, True, True, [0, 1, 2, 70000], None),
    ("bf16", 32, 8, 128, 128, False, True, [5, 1 << 20, 77], None),
    ("f16", 3, 1, 256, 256, False, True, [9, 0, 123456], None),
    ("f32", 5, 2, 256, 32, True, False, [0, 1000], [0, 33, 90]),
    ("bf16", 7, 7, 80, 80, False, True, [12, 0, 99999], [0, 1, 40, 41]),
    ("f16", 4, 2, 96, 48, False, False, [7, 3], [0, 0, 65]),
    ("f32", 2, 3, 240, 240, False, True, [3, 1, 2, 5], [0, 17, 17, 17, 20]),
    ("bf16", 6, 1, 112, 16, True, True, [0], [0, 100]),
    ("f32", 24, 24, 32, 0, False, True, [4, 5], None),
    ("bf16", 1, 0, 64, 64, True, True, [4, 5, 6], None),
    ("f32", 12, 12, 64, 32, True, True, [0, 40, 7, 900], [0, 700, 1200, 1900, 2500]),
]


@pytest.mark.parametrize("typ,hq,hk,hd,rot,near,norms,pos,off", ROPES)
def test_rope(ops, typ, hq, hk, hd, rot, near, norms, pos, off):
    rs = np.random.RandomState(hd + hq)
    rows = len(pos) if off is None else off[-1]
    q, q64 = rand(rs, (rows, hq, hd), typ)
    k, k64 = rand(rs, (rows, hk, hd), typ, 3.0) if hk else (None, None)
    f = freqs(rot)
    gq, gk = (rs.randn(2, hd) * 0.3).astype(np.float32) if norms else (None, None)
    arr = lambda g: None if g is None else dev(g, torch.float32)  # noqa: E731
    qo, ko = ops.qk_rope(q, k, dev(pos), dev(f, torch.float32), off=None if off is None else dev(off), gq=arr(gq),
                         gk=arr(gk), near=near)
    at = positions(pos, off, rows)
    check_rope(typ, qo, q64, at, f, gq, 1e-5, near)
    assert (ko is None) == (hk == 0)
    if hk:
        check_rope(typ, ko, k64, at, f, gk, 1e-5, near)


@pytest.mark.parametrize("near", [False, True])
def test_rope_far_positions(ops, near):
    """The angles of every position below 2^31, and of the rows after it."""
    rs = np.random.RandomState(3)
    pos = [2 ** 31 - 1, 2 ** 31 - 2 ** 20 - 3, 2 ** 24 + 1, 99999999]
    q, q64 = rand(rs, (8, 2, 64), "f32")
    f = np.concatenate([freqs(32), -freqs(32, 7.0)])
    qo, _ = ops.qk_rope(q, None, dev(pos), dev(f, torch.float32), off=dev([0, 3, 4, 7, 8]), near=near)
    check_rope("f32", qo, q64, positions(pos, [0, 3, 4, 7, 8], 8), f, None, 0.0, near)


@pytest.mark.parametrize("typ", list(TYPES))
def test_rope_strides_and_rows_outside(ops, typ):
    """Views of a projection's output, of any order and alignment, in place
    and elsewhere; sequences without a position, rows of no sequence."""
    rs = np.random.RandomState(4)
    rows, hq, hk, hd = 23, 6, 2, 64
    pos, off = [3, -1, 50, -2 ** 31], [2, 6, 9, 20, 21]
    at = positions(pos, off, rows)
    f = freqs(32)
    g = (rs.randn(hd) * 0.3).astype(np.float32)
    for shift, order in ((0, 0), (1, 0), (0, 1), (3, 1)):
        flat, _ = rand(rs, (rows * (hq + 2 * hk) * hd + shift,), typ)
        x = flat[shift:].view(rows, hq + 2 * hk, hd) if order == 0 else flat[shift:].view(hq + 2 * hk, rows, hd).transpose(0, 1)
        q, k = x[:, :hq], x[:, hq:hq + hk]
        q64, k64, v64 = host(q), host(k), host(x[:, hq + hk:])
        args = dict(off=dev(off), gq=dev(g, torch.float32))
        out = [torch.full((h, rows, hd), 7.5, dtype=TYPES[typ], device="cuda").transpose(0, 1) for h in (hq, hk)]
        ops.qk_rope(q, k, dev(pos), dev(f, torch.float32), out=out, **args)
        check_rope(typ, out[0], q64, at, f, g, 1e-5, False, np.full_like(q64, 7.5))
        check_rope(typ, out[1], k64, at, f, None, 1e-5, False, np.full_like(k64, 7.5))
        ops.qk_rope(q, k, dev(pos), dev(f, torch.float32), out=(q, k), **args)
        check_rope(typ, q, q64, at, f, g, 1e-5, False, q64)
        check_rope(typ, k, k64, at, f, None, 1e-5, False, k64)
        assert np.array_equal(host(x[:, hq + hk:]), v64)


def test_rope_many_short_sequences(ops):
    """Sequences of no, one and a few rows in any order, more than a
    workgroup's rows and lanes."""
    rs = np.random.RandomState(5)
    lens = rs.choice([0, 0, 0, 1, 2, 5, 33], 3000)
    off = np.concatenate([[0], np.cumsum(lens)])
    pos = rs.randint(0, 5000, 3000)
    q, q64 = rand(rs, (int(off[-1]), 2, 32), "bf16")
    f = freqs(32)
    qo, _ = ops.qk_rope(q, None, dev(pos), dev(f, torch.float32), off=dev(off))
    check_rope("bf16", qo, q64, positions(pos, off, int(off[-1])), f, None, 0.0, False)


def test_rope_special_values(ops):
    """A head of zeros stays one, infinities and NaN stay in their own head,
    squares past f32's largest number are not hidden."""
    x = torch.ones((4, 2, 32), device="cuda")
    x[0, 0], x[1, 1, 3], x[2, 0, 5], x[3, 1, 7] = 0.0, math.inf, math.nan, 3e38
    g = torch.zeros(32, device="cuda")
    qo, _ = ops.qk_rope(x, None, dev([1, 2, 3, 4]), dev(freqs(32), torch.float32), gq=g)
    assert (qo[0, 0] == 0).all()
    fin = torch.isfinite(qo).all(-1).cpu().numpy()
    assert fin.tolist() == [[True, True], [True, False], [False, True], [True, True]]
    assert (qo[3, 1] == 0).all()


# ---------------------------------------------------------------- attention behind shared prefixes

def filled(ops, rs, seqs, slots, heads, hd):
    """A cache whose every slot holds numbers as they come."""
    cache = ops.KV4.empty(seqs, slots, heads, hd)
    cache.data.copy_(torch.tensor(rs.randint(0, 256, tuple(cache.data.shape)), dtype=torch.uint8))
    cache.data[..., 32 * hd:] = torch.tensor(rs.randint(124, 128, (*cache.data.shape[:3], 2 * hd)), dtype=torch.uint8)
    return cache


def check_shared(ops, cache, prefix, q, q64, typ, pos, seq, off, plen, pseq, poff, sink, scale=None, **kw):
    d = lambda a: None if a is None else dev(a)  # noqa: E731
    sk = None if sink is None else dev(sink, torch.float32)
    got = ops.kv4_attend_shared(q, cache, dev(pos), prefix, dev(plen), pseq=d(pseq), poff=d(poff), seq=d(seq), off=d(off),
                                sink=sk, scale=scale, **kw)
    sc = cache.hd ** -0.5 if scale is None else scale
    o, pv, big, cnt = sref.attend_shared(q64, cache.data.cpu().numpy(), cache.slots, pos,
                                         list(range(len(pos))) if seq is None else seq, off, prefix.data.cpu().numpy(),
                                         prefix.slots, plen, list(range(len(plen))) if pseq is None else pseq, poff, sink, sc)
    tol = ref.attend_tolerance(typ, o, pv, big, cnt, cache.hd, rounded=typ == "bf16")
    g = host(got)
    first, last = (0, len(pos)) if off is None else (off[0], off[-1])
    assert (np.abs(g - o)[first:last] <= tol[first:last]).all(), np.abs(g - o)[first:last].max()
    return got


# (type, hq, hkv, hd, own slots, pos, off, prefix slots, plen, pseq, poff, sink)
SHARED = [
    ("f32", 2, 2, 64, 40, [0, 5, 39], None, 100, [100], None, None, True),
    ("f32", 4, 1, 32, 33, [70, 3], None, 31, [1], [0], None, False),
    ("bf16", 8, 2, 128, 64, [10, 63, 0, 200, 30], None, 700, [650, 33], [1, 0], [0, 2, 5], False),
    ("f16", 3, 3, 64, 50, [20] * 70, None, 300, [300], None, None, True),
    ("bf16", 16, 1, 64, 50, [20] * 20, None, 1000, [777], None, None, True),
    ("f32", 2, 1, 128, 90, [0, 7, 30], [0, 1, 40, 71], 400, [399, 64], [1, 0], [0, 40, 71], True),
    ("bf16", 4, 4, 64, 200, [0, 50, 3], [0, 70, 100, 180], 513, [513], None, None, False),
    ("f16", 8, 1, 32, 64, [3, 0], [0, 9, 40], 96, [50, 96, 2], [2, 1, 0], [0, 5, 20, 40], False),
    ("f32", 12, 12, 64, 30, [1, 2, 3, 4], None, 40, [39], None, None, False),
]


@pytest.mark.parametrize("typ,hq,hkv,hd,slots,pos,off,pslots,plen,pseq,poff,sink", SHARED)
def test_shared(ops, typ, hq, hkv, hd, slots, pos, off, pslots, plen, pseq, poff, sink):
    rs = np.random.RandomState(6)
    n = len(pos)
    rows = n if off is None else off[-1]
    cache, prefix = filled(ops, rs, n + 1, slots, hkv, hd), filled(ops, rs, len(plen), pslots, hkv, hd)
    q, q64 = rand(rs, (rows, hq, hd), typ)
    seq = rs.permutation(n + 1)[:n].tolist()
    check_shared(ops, cache, prefix, q, q64, typ, pos, seq, off, plen, pseq, poff,
                 rs.randn(hq) if sink else None)


@pytest.mark.parametrize("typ", list(TYPES))
def test_shared_groups_of_all_kinds(ops, typ):
    """Rows before, between and after the groups, groups without rows, without
    a place, of no length and of a length below zero, sequences without a place."""
    rs = np.random.RandomState(7)
    cache, prefix = filled(ops, rs, 12, 40, 2, 64), filled(ops, rs, 3, 500, 2, 64)
    pos, seq = [3, 20, 55, 0, 9, 11, -1, 5, 6, 7, 8], [4, 0, 11, 2, -1, 3, 5, 12, 6, 7, 8]
    q, q64 = rand(rs, (11, 4, 64), typ)
    # rows 1-3, none, 4-5 (no place), 6 (no length), 7 and 8 (below zero, one token), 9-10 of no group
    poff, pseq, plen = [1, 4, 4, 6, 7, 8, 9], [2, 0, 3, 1, 0, 1], [500, 40, 100, 0, -5, 1]
    out = torch.full_like(q, 7.5)
    got = check_shared(ops, cache, prefix, q, q64, typ, pos, seq, None, plen, pseq, poff, None, out=out)
    assert got is out and (out[[4, 6, 7]] == 0).all()
    # ragged sequences, the rows before the first and after the last left as they were
    off = [2, 5, 5, 9]
    out = torch.full_like(q, 7.5)
    check_shared(ops, cache, prefix, q, q64, typ, [30, 4, 0], [1, 0, 5], off, [300, 7], [0, 2], [0, 3, 11], rs.randn(4),
                 out=out)
    assert (out[:2] == 7.5).all() and (out[9:] == 7.5).all()


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 17, 90])
def test_shared_long_prefix(ops, typ, rows):
    """A prefix in many pieces, at lengths around their borders; what its ring
    holds past the length, NaN included, does not matter; hints change nothing
    that is seen."""
    rs = np.random.RandomState(8)
    cache, prefix = filled(ops, rs, rows, 33, 1, 64), filled(ops, rs, 2, 9000, 1, 64)
    prefix.data[0, :, 128:, 32 * 64:] = 255     # from 4096 on
    q, q64 = rand(rs, (rows, 2, 64), typ)
    pos = rs.randint(0, 60, rows).tolist()
    for n, plive in ((4096, 0), (4065, 4096), (33, 0), (32, 32), (1, 0), (2049, 9000)):
        check_shared(ops, cache, prefix, q, q64, typ, pos, None, None, [n], None, None, [0.5, -1.0], plive=plive, live=20)
    # past the ring's end a prefix is what the ring holds
    got = check_shared(ops, cache, prefix, q, q64, typ, pos, None, None, [20000], [1], None, None)
    assert torch.isfinite(got.float()).all()
    # (a NaN that is seen shows)
    got = ops.kv4_attend_shared(q, cache, dev(pos), prefix, dev([4097]))
    assert torch.isnan(got.float()).all()


def own_pieces(ops, cache, rows, hq, pos, off=None):
    """Whether kv4_attend of such a call cuts a sequence's own positions."""
    r = ops._rows(cache, rows, dev(pos), None, None if off is None else dev(off))
    return ops.lib().ana_kv4_attend_ws(cache._p, ops.C.byref(r), hq, 0) > 0


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("typ", list(TYPES))
def test_shared_own_positions_in_pieces(ops, typ, hd):
    """Single rows whose own positions are one piece and many in one call,
    wrapped ones too, behind prefixes of one piece and many, of no length, without
    a place, and of no group; with and without sinks."""
    rs = np.random.RandomState(31)
    pos = [650, 3, 127, 128, 255, 256, 699, 1500, 40, 700, 511, 0]
    cache, prefix = filled(ops, rs, 13, 700, 2, hd), filled(ops, rs, 3, 400, 2, hd)
    q, q64 = rand(rs, (12, 4, hd), typ)
    assert own_pieces(ops, cache, 12, 4, pos)
    seq = rs.permutation(13)[:12].tolist()
    seq[6] = 13                                                        # (no place: zeros)
    poff, pseq, plen = [1, 4, 6, 6, 8, 10], [2, 0, 1, 1, 7], [400, 17, 30, 0, 60]
    for sink in (None, rs.randn(4)):
        got = check_shared(ops, cache, prefix, q, q64, typ, pos, seq, None, plen, pseq, poff, sink)
        assert (got[6] == 0).all()
        check_shared(ops, cache, prefix, q, q64, typ, pos, seq, None, [333], [1], None, sink)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("typ", list(TYPES))
def test_shared_ragged_own_positions_in_pieces(ops, typ, hd):
    """Sequences of few rows and of many (16 pairs of a key head and more) over
    one piece of their own positions and over several, rows before, between and
    after the groups and of no sequence."""
    rs = np.random.RandomState(32)
    off = [2, 42, 45, 45, 65, 66, 68, 100, 109]
    pos = [1500, 3, 9, 700, 1540, 255, 20, 1700]
    cache, prefix = filled(ops, rs, 8, 1600, 1, hd), filled(ops, rs, 2, 400, 1, hd)
    q, q64 = rand(rs, (111, 2, hd), typ)
    assert own_pieces(ops, cache, 111, 2, pos, off)
    seq = rs.permutation(8).tolist()
    poff, pseq, plen = [0, 30, 43, 67, 104], [1, 0, 0, 1], [400, 33, 0, 150]
    for sink in (None, rs.randn(2)):
        out = torch.full_like(q, 7.5)
        check_shared(ops, cache, prefix, q, q64, typ, pos, seq, off, plen, pseq, poff, sink, out=out)
        assert (out[:2] == 7.5).all() and (out[109:] == 7.5).all()
        check_shared(ops, cache, prefix, q, q64, typ, pos, seq, off, [399], [0], None, sink)


def test_shared_without_groups(ops):
    """No prefix for any row: the attention of the rows' own rings."""
    rs = np.random.RandomState(18)
    cache = filled(ops, rs, 3, 70, 2, 64)
    q, _ = rand(rs, (3, 4, 64), "f32")
    pos = dev([5, 69, 200])
    want = ops.kv4_attend(q, cache, pos)
    got = ops.kv4_attend_shared(q, cache, pos, cache, dev([]), poff=dev([0]))
    assert torch.equal(got, want)


def test_shared_is_attention_over_copies(ops):
    """A prefix of 128 tokens and 70 own ones, against rings that hold both."""
    rs = np.random.RandomState(9)
    n, h, hd = 5, 2, 64
    own, whole = filled(ops, rs, n, 96, h, hd), ops.KV4.empty(n, 224, h, hd)
    prefix = filled(ops, rs, 1, 128, h, hd)
    whole.data[:, :, :4], whole.data[:, :, 4:] = prefix.data, own.data
    q, _ = rand(rs, (n, 4, hd), "f32")
    pos = dev([0, 1, 40, 69, 95])
    a = ops.kv4_attend_shared(q, own, pos, prefix, dev([128]))
    b = ops.kv4_attend(q, whole, pos + 128)
    assert (a - b).abs().max() <= 2.0 ** -24 * 1000 * b.abs().max()
    # the prefix in the same cache, and its own place among the sequences'
    both = ops.KV4(torch.cat([own.data, own.data]), 96)
    c = ops.kv4_attend_shared(q, both, pos, both, dev([96]), pseq=dev([7]))
    d = ops.kv4_attend_shared(q, own, pos, own, dev([96]), pseq=dev([2]))
    assert torch.equal(c, d)


def test_shared_in_place_and_strided(ops):
    rs = np.random.RandomState(10)
    for typ in TYPES:
        cache, prefix = filled(ops, rs, 6, 40, 2, 32), filled(ops, rs, 1, 200, 2, 32)
        flat, _ = rand(rs, (6 * 9 * 32 + 1,), typ)
        pos = [5, 6, 7, 39, 80, 0]
        for x in (flat[:-1].view(6, 9, 32)[:, :4], flat[1:].view(9, 6, 32).transpose(0, 1)[:, 2:6]):
            q = x.clone().contiguous()
            want = check_shared(ops, cache, prefix, x, host(x), typ, pos, None, None, [150], None, None, None)
            ops.kv4_attend_shared(x, cache, dev(pos), prefix, dev([150]), out=x)
            assert torch.equal(x, want)
            assert torch.equal(ops.kv4_attend_shared(q, cache, dev(pos), prefix, dev([150])), want)


def check_fine(ops, cache, prefix, q, q64, pos, off, plen, poff, sink, vmax=0.0, **kw):
    """bf16 outputs behind a prefix, with what f16 probabilities allow. Each is
    off by at most half a step: 2^-11 of itself, or, where f16's steps no longer
    shrink with it, 2^-25, the largest being 2^7 at least there, so 2^-32 of the
    largest. That counts in the sum, times a value of the tiles that are in f16
    (vmax at most), and in the denominator."""
    d = lambda a: None if a is None else dev(a)  # noqa: E731
    got = ops.kv4_attend_shared(q, cache, dev(pos), prefix, dev(plen), poff=d(poff), off=d(off),
                                sink=None if sink is None else dev(sink, torch.float32), **kw)
    n = len(pos)
    o, pv, big, cnt = sref.attend_shared(q64, cache.data.cpu().numpy(), cache.slots, pos, list(range(n)), off,
                                         prefix.data.cpu().numpy(), prefix.slots, plen, list(range(len(plen))), poff, sink,
                                         cache.hd ** -0.5)
    tol = ref.attend_tolerance("bf16", o, pv, big, cnt, cache.hd) + 2 * 2.0 ** -11 * pv + 2 * cnt * 2.0 ** -32 * vmax
    far = np.abs(host(got) - o) - tol
    assert (far <= 0).all(), far.max()


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("sink", [False, True])
def test_shared_bf16_probabilities(ops, hd, sink):
    """Few positions of like weight and values that cancel: a probability's
    rounding is what shows in a bf16 output, not the output's own."""
    rs = np.random.RandomState(21)
    cache, prefix = filled(ops, rs, 64, 3, 2, hd), filled(ops, rs, 3, 40, 2, hd)
    q, q64 = rand(rs, (64, 8, hd), "bf16")
    sk = rs.randn(8) if sink else None
    check_fine(ops, cache, prefix, q, q64, [0] * 64, None, [3], None, sk)
    check_fine(ops, cache, prefix, q, q64, [0] * 64, None, [2, 33, 5], [0, 30, 31, 64], sk)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_shared_values_of_any_scale(ops, hd):
    """Blocks of values beyond f16 (and zeros as the cache holds them, and such
    that are not finite) in some tiles, in all, in the last alone."""
    rs = np.random.RandomState(22)
    for at in ([5], [0], [9], [3, 4, 7], list(range(10))):
        cache, prefix = filled(ops, rs, 20, 40, 1, hd), filled(ops, rs, 1, 310, 1, hd)
        for t in at:
            for lo, hi in ((60, 108), (140, 180), (2, 4)):
                n = rs.randint(1, 12)
                prefix.data[0, 0, t, dev(33 * hd + rs.randint(0, hd, n), torch.int64)] = dev(rs.randint(lo, hi, n), torch.uint8)
        q, q64 = rand(rs, (20, 3, hd), "bf16")
        check_fine(ops, cache, prefix, q, q64, rs.randint(0, 40, 20).tolist(), None, [310], None, None)
    q, q64 = rand(rs, (1, 3, hd), "bf16")
    for t, byte in ((2, 255), (9, 255), (2, 250), (2, 0)):
        prefix = filled(ops, rs, 1, 310, 1, hd)
        prefix.data[0, 0, t, 33 * hd] = byte     # (slot 32 t, the first dims)
        got = host(ops.kv4_attend_shared(q, cache, dev([3]), prefix, dev([310])))
        if byte == 255:
            assert np.isnan(got[..., :32]).all() and np.isfinite(got[..., 32:]).all()
        else:
            check_fine(ops, cache, prefix, q, q64, [3], None, [310], None, None)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rows", [3, 50])
def test_shared_values_of_any_scale_in_one_piece(ops, hd, rows):
    """A prefix gone over in one piece, in f16 and from some tile on in bf16, its
    scores rising and falling from tile to tile before that and after."""
    rs = np.random.RandomState(27)
    n = 700
    for first in (0, 1, 9, 20, 21, 22):        # (22: none)
        cache, prefix = filled(ops, rs, rows, 40, 1, hd), filled(ops, rs, 1, n, 1, hd)
        for t in range(22):
            prefix.data[0, 0, t, 32 * hd:33 * hd] = int(rs.randint(120, 130))
        for t in (first, 21 if first < 21 else first):
            if t < 22:
                prefix.data[0, 0, t, dev(33 * hd + rs.randint(0, hd, 5), torch.int64)] = dev(rs.randint(140, 160, 5), torch.uint8)
        q, q64 = rand(rs, (rows, 2, hd), "bf16")
        check_fine(ops, cache, prefix, q, q64, rs.randint(0, 40, rows).tolist(), None, [n], None, rs.randn(2), vmax=6.0, plive=32)


@pytest.mark.parametrize("gap", [5.0, 9.0, 16.0, 20.0, 30.0])
def test_shared_many_light_positions(ops, gap):
    """One position of a prefix far above thousands of others whose weights
    add up, at the start, in the middle and at the end; its value is zero."""
    rs = np.random.RandomState(23)
    hd, n = 64, 8000
    for slot in (0, 4005, 7999):
        cache, prefix = filled(ops, rs, 5, 3, 1, hd), filled(ops, rs, 1, n, 1, hd)
        prefix.data[..., 32 * hd:33 * hd] = 117
        cache.data[..., 32 * hd:33 * hd] = 117
        ref_data = prefix.data.cpu().numpy()
        ref.put(ref_data, 0, 0, slot, [7] * hd, [126] * 2, [0] * hd, [127] * 2)    # keys of 3, values of 0
        prefix.data.copy_(torch.tensor(ref_data))
        q = torch.full((5, 2, hd), gap / 24, device="cuda").bfloat16()            # (a score of gap, the others next to 0)
        check_fine(ops, cache, prefix, q, host(q), [0] * 5, None, [n], None, None, vmax=6.0)


@pytest.mark.parametrize("typ", list(TYPES))
def test_shared_scores_of_any_size(ops, typ):
    """Scores whose own steps are more than a weight's range: the likeliest
    position has all, whether behind the prefix or the row's own."""
    rs = np.random.RandomState(24)
    hd, n, rows = 64, 300, 40
    cache, prefix = filled(ops, rs, rows, 5, 1, hd), filled(ops, rs, 1, n, 1, hd)
    K, V = ref.get(prefix.data.cpu().numpy(), 0, 0, n)
    for big in (1e4,) if typ == "f16" else (1e4, 1e6, 1e7, 3e7, 1e8):
        q, q64 = rand(rs, (rows, 2, hd), typ, big)
        got = host(ops.kv4_attend_shared(q, cache, dev([2] * rows), prefix, dev([n])))
        assert np.isfinite(got).all()
        for r in range(rows):
            own = ref.get(cache.data[r:r + 1].cpu().numpy(), 0, 0, 5)
            k, v = np.concatenate([K, own[0][:3]]), np.concatenate([V, own[1][:3]])
            for h in range(2):
                x = k @ q64[r, h] * hd ** -0.5
                at = np.argsort(x)
                # (a score is off by 3 hd 2^-24 of its terms, in two of them, and 40 is a weight of nothing)
                if x[at[-1]] - x[at[-2]] > 40 + 4 * 3 * hd * 2.0 ** -24 * (np.abs(k) @ np.abs(q64[r, h])).max() * hd ** -0.5:
                    # (e^-40 of the others' values, and a few roundings of the quotient)
                    assert np.abs(got[r, h] - v[at[-1]]).max() <= 6 * 2.0 ** -20, (big, r, h)


# ---------------------------------------------------------------- sampling

def check_sample(ops, x, u, t=1.0, k=0, p=1.0, q=0.0):
    n, vocab = x.shape
    tensors = [torch.is_tensor(a) for a in (t, k, p, q)]
    tok, lp = ops.sample(x, dev(u, torch.float32), t, k, p, q)
    x64, u32 = host(x), np.asarray(u, dtype=np.float32)
    each = [a.cpu().tolist() if on else [float(np.float32(a))] * n for a, on in zip((t, k, p, q), tensors)]
    tok, lp = tok.cpu().tolist(), host(lp)
    for r in range(n):
        want, wlp = sref.sample(x64[r], float(u32[r]), each[0][r], int(each[1][r]), each[2][r], each[3][r])
        assert tok[r] == want, (r, tok[r], want)
        if math.isnan(wlp):
            assert math.isnan(lp[r])
        else:
            # its own rounding; a mass in units of 2^-42 (at most 2^21 half ones)
            assert abs(lp[r] - wlp) <= 2.0 ** -24 * abs(wlp) + 2.0 ** -22 * 2.0 ** -10, r


SETTINGS = [dict(), dict(t=0.0), dict(t=0.7, k=1), dict(t=0.8, k=40, p=0.95), dict(k=64, q=0.05), dict(t=1.3, k=65, p=0.7),
            dict(t=0.5, k=1000), dict(p=0.9), dict(t=1.7, p=0.99, q=0.01), dict(q=0.2), dict(p=0.0), dict(q=1.0),
            dict(t=2.0, k=3000, p=0.9, q=1e-4), dict(k=100), dict(t=1.5, k=256, p=0.8), dict(k=257, q=0.02),
            dict(t=0.9, k=200, p=0.99, q=0.001)]


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("n,vocab,pad,shift", [(7, 1, 0, 0), (5, 2, 1, 0), (6, 17, 0, 1), (9, 258, 3, 0), (4, 4097, 0, 2),
                                               (12, 32768, 0, 0), (3, 32773, 1, 1), (3, 53255, 1, 3), (2, 120001, 5, 1)])
def test_sample(ops, typ, n, vocab, pad, shift):
    rs = np.random.RandomState(vocab)
    flat, _ = rand(rs, (n * (vocab + pad) + shift,), typ, 2.5)
    x = flat[shift:].view(n, vocab + pad)[:, :vocab]
    for s in SETTINGS:
        u = rs.rand(n)
        u[0] = 0.0
        check_sample(ops, x, u, **s)


def test_sample_settings_of_each_row(ops):
    rs = np.random.RandomState(11)
    n = 260
    x, _ = rand(rs, (n, 5003), "f32", 3.0)
    pick = lambda a, d=torch.float32: dev(rs.choice(a, n), d)  # noqa: E731
    check_sample(ops, x, rs.rand(n), t=pick([0.0, -1.0, 0.3, 0.9, 1.0, 2.5, math.nan]),
                 k=pick([0, 1, 2, 5, 64, 65, 300, 5002, 5003, 9999, -1], torch.int32), p=pick([1.0, 0.5, 0.9, 0.999, 2.0, -1.0]),
                 q=pick([0.0, 0.1, 1e-3, 1.0, -1.0]))


@pytest.mark.parametrize("vocab", [700, 9000, 100001])
def test_sample_min_p_outside_0_to_1(ops, vocab):
    """A row's min-p above 1 is 1 (what is as likely as the first stays), one
    that is not above 0, or NaN, is 0."""
    rs = np.random.RandomState(16)
    given, meant = [2.0, 1.0001, math.inf, math.nan, -1.0, -math.inf, 1.0], [1.0, 1.0, 1.0, 0.0, 0.0, 0.0, 1.0]
    x = torch.tensor(np.minimum(np.round(rs.randn(7, vocab)), 1.0), dtype=torch.float32).cuda()   # (many alike, the likeliest too)
    for s in (dict(), dict(top_k=20), dict(top_k=100), dict(top_k=600), dict(top_p=0.9), dict(top_k=50, top_p=0.9)):
        u = rs.rand(7).astype(np.float32)
        u[0] = 0.97
        tok, lp = ops.sample(x, dev(u, torch.float32), min_p=dev(given, torch.float32), **s)
        for r in range(7):
            want, wlp = sref.sample(host(x)[r], float(u[r]), 1.0, s.get("top_k", 0), float(np.float32(s.get("top_p", 1.0))), meant[r])
            assert int(tok[r]) == want, (s, r)
            assert abs(float(lp[r]) - wlp) <= 2.0 ** -24 * abs(wlp) + 2.0 ** -32, (s, r)   # (as in check_sample)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [300, 20000, 70001])
def test_sample_ties(ops, typ, vocab):
    """All logits alike, two values, a mask of -inf and of the type's lowest
    value: more tokens of one weight than any list holds."""
    rs = np.random.RandomState(12)
    low = torch.finfo(TYPES[typ]).min
    rows = [np.zeros(vocab), np.where(rs.rand(vocab) < 0.3, 1.0, 0.5), np.where(rs.rand(vocab) < 0.99, -math.inf, 2.0),
            np.where(rs.rand(vocab) < 0.5, low, -3.0), np.full(vocab, low), np.round(rs.randn(vocab)),
            np.where(np.arange(vocab) == vocab - 1, 0.0, -math.inf), np.where(rs.rand(vocab) < 0.5, -0.0, 0.0)]
    x = torch.tensor(np.stack(rows)).to(TYPES[typ]).cuda()
    for s in (dict(), dict(p=0.5), dict(k=30), dict(k=200, p=0.25), dict(t=0.1, q=0.5), dict(t=100.0, p=0.7), dict(t=0.0)):
        for u in (0.0, 0.31, 0.77, 0.999):
            check_sample(ops, x, [u] * len(rows), **s)


@pytest.mark.parametrize("vocab", [40, 9000, 100001])
def test_sample_not_finite(ops, vocab):
    rs = np.random.RandomState(13)
    x = rs.randn(7, vocab).astype(np.float32)
    x[0, 3], x[0, 17] = math.nan, 40.0
    x[1, [5, 9, 30]] = math.inf
    x[2, 8], x[2, 9], x[2, 10] = math.inf, math.nan, -math.inf
    x[3], x[4] = -math.inf, math.nan
    x[5] = math.nan
    x[5, 20] = -2.0
    x[6, ::2] = math.nan
    for s in (dict(), dict(t=0.0), dict(k=2), dict(k=100, p=0.9), dict(p=0.4, q=0.01), dict(t=1e-30), dict(t=math.inf)):
        for u in (0.0, 0.5, 0.97, math.nan, -1.0):
            check_sample(ops, torch.tensor(x).cuda(), [u] * 7, **s)


def test_sample_temperatures(ops):
    """From one that leaves a token to one that makes them alike, logits next
    to f32's largest."""
    rs = np.random.RandomState(14)
    x = rs.randn(3, 3001).astype(np.float32)
    x[1] *= 1e37
    x[2] *= 1e-30
    for t in (1e-45, 1e-10, 1e-3, 0.05, 30.0, 1e6, 3e38):
        for s in (dict(), dict(p=0.8), dict(k=20), dict(k=90, p=0.5)):
            check_sample(ops, torch.tensor(x).cuda(), rs.rand(3), t=t, **s)


@pytest.mark.parametrize("vocab", [2, 3001, 70001])
def test_sample_temperatures_next_to_zero(ops, vocab):
    """Temperatures down to f32's least number over logits as small as they are:
    next to each other in f32, and far apart for e^x."""
    rs = np.random.RandomState(25)
    x = rs.randn(4, vocab) * np.array([[1e-37], [1e-36], [1e-40], [1e-43]])
    x[0, 0], x[0, 1] = 0.0, -1e-37
    x[1, ::2] -= 1e-35
    x = x.astype(np.float32)
    for t in (1e-45, 1e-43, 1e-40, 1e-38, 2e-37, 2.4e-37, 1e-36):
        for s in (dict(), dict(p=0.8), dict(k=20), dict(k=300, p=0.9), dict(q=0.3, p=0.99)):
            check_sample(ops, torch.tensor(x).cuda(), rs.rand(4), t=t, **s)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [3001, 70001])
def test_sample_temperatures_next_to_none(ops, typ, vocab):
    """At a temperature past every logit tokens at the type's lowest value are
    as likely as the others, whole stretches of them too."""
    rs = np.random.RandomState(26)
    x = torch.tensor(rs.randn(3, vocab)).to(TYPES[typ])
    x[0, 600:] = torch.finfo(TYPES[typ]).min
    x[1, :vocab - 700] = torch.finfo(TYPES[typ]).min
    x[2, 1::2] = -math.inf
    for t in (math.inf, 3e38, 1e38, 1e37):
        for s in (dict(), dict(p=0.8), dict(k=2000), dict(q=0.5)):
            check_sample(ops, x.cuda(), [0.3, 0.9, 0.6], t=t, **s)


def test_sample_numbers_at_the_borders(ops):
    """Masses and numbers that are exact: u at a border takes the next token."""
    x = torch.zeros((9, 8), device="cuda")
    check_sample(ops, x, np.arange(9) / 8.0)
    check_sample(ops, x, np.nextafter(np.float32(np.arange(9) / 8.0), np.float32(0)))
    check_sample(ops, x, np.arange(9) / 8.0, p=0.5)
    tok, lp = ops.sample(x, dev(np.arange(9) / 8.0, torch.float32), top_p=0.5)
    assert tok.tolist() == [0, 0, 1, 1, 2, 2, 3, 3, 3] and (lp + math.log(4.0)).abs().max() < 1e-6


def test_sample_widest_vocabulary(ops):
    rs = np.random.RandomState(15)
    x = torch.zeros((2, 1 << 21), dtype=torch.bfloat16, device="cuda")
    x[1].normal_(generator=torch.Generator("cuda").manual_seed(1))
    for s in (dict(), dict(p=0.3), dict(k=60), dict(k=100000), dict(q=0.5)):
        check_sample(ops, x, rs.rand(2), **s)


@pytest.mark.parametrize("spread", [0.1, 0.17, 0.3, 0.6, 3.0])
def test_sample_long_rows(ops, spread):
    """One bin's tokens from more than a piece's list or all pieces' room takes
    down to a few."""
    rs = np.random.RandomState(17)
    x = torch.tensor(rs.randn(2, 400003) * spread, dtype=torch.float32).cuda()
    x[1, ::2] = x[0, 1::2].mean()
    for s in (dict(), dict(p=0.9), dict(p=0.3, q=0.7), dict(k=400, p=0.9)):
        check_sample(ops, x, rs.rand(2), **s)
    k = dev([0, 400], torch.int32)
    check_sample(ops, x, rs.rand(2), t=dev([0.7, 1.0], torch.float32), k=k, p=0.9)
    check_sample(ops, x, rs.rand(2), t=dev([0.0, 1.3], torch.float32), k=k.flip(0), p=dev([0.5, 0.95], torch.float32))


def test_sample_follows_the_probabilities(ops):
    """Evenly spaced numbers take each token as often as its probability says."""
    n = 4096
    x = torch.tensor([[0.0, 1.0, -1.0, 0.5, 1.0]], device="cuda").expand(n, 5).contiguous()
    tok, _ = ops.sample(x, (torch.arange(n, device="cuda") + 0.5) / n, temperature=0.7)
    p = torch.softmax(x[0].double() / 0.7, -1).cpu().numpy()
    assert (np.abs(np.bincount(tok.cpu().numpy(), minlength=5) / n - p) <= 1.0 / n).all()


def test_sample_rows_do_not_depend_on_each_other(ops):
    rs = np.random.RandomState(16)
    x, _ = rand(rs, (300, 9001), "bf16", 2.0)
    u = dev(rs.rand(300), torch.float32)
    a = ops.sample(x, u, 0.9, 0, 0.95)
    for r in (0, 7, 299):
        b = ops.sample(x[r:r + 1], u[r:r + 1], 0.9, 0, 0.95)
        assert torch.equal(a[0][r:r + 1], b[0]) and torch.equal(a[1][r:r + 1], b[1])
    for _ in range(3):
        b = ops.sample(x, u, 0.9, 0, 0.95)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("typ", list(TYPES))
def test_sample_long_rows_alone_and_in_a_batch(ops, typ):
    """A row in pieces takes the token that it takes whole, to the bit of its
    log probability."""
    rs = np.random.RandomState(33)
    n, vocab = 100, 70001
    x, _ = rand(rs, (n, vocab), typ, 2.0)
    x[3] = 1.0
    x[4, ::3] = -math.inf
    u = dev(rs.rand(n), torch.float32)
    assert ops.lib().ana_row_sample_ws(1, vocab) > 0 and ops.lib().ana_row_sample_ws(n, vocab) == 0
    for s in (dict(), dict(top_p=0.9), dict(temperature=0.0), dict(top_k=40), dict(top_k=500, top_p=0.9), dict(min_p=0.05),
              dict(temperature=2.0, top_p=0.99, min_p=0.001)):
        a = ops.sample(x, u, **s)
        for r0, r1 in ((0, 1), (3, 5), (60, 100)):
            b = ops.sample(x[r0:r1], u[r0:r1], **s)
            assert torch.equal(a[0][r0:r1], b[0]) and torch.equal(a[1][r0:r1], b[1]), (s, r0)


# ---------------------------------------------------------------- a served step of all of them

class Step:
    """Answers to one prompt: a token each through qk_rope, the cache, the
    attention behind the prompt, a head and the sampler."""

    def __init__(self, ops, typ, n=6, hq=4, hkv=2, hd=64, vocab=1000, plen=70, seed=0):
        rs = np.random.RandomState(seed)
        self.ops, self.typ, self.n, self.plen, self.hd = ops, typ, n, plen, hd
        self.x, _ = rand(rs, (n, hq + 2 * hkv, hd), typ)
        self.q, self.k, self.v = self.x[:, :hq], self.x[:, hq:hq + hkv], self.x[:, hq + hkv:]
        self.freq = dev(freqs(hd), torch.float32)
        self.gq, self.gk = (dev(rs.randn(hd) * 0.2, torch.float32) for _ in range(2))
        self.cache, self.prefix = filled(ops, rs, n, 40, hkv, hd), filled(ops, rs, 1, 96, hkv, hd)
        self.pos, self.length = dev(rs.randint(0, 20, n)), dev([plen])
        self.head = rand(rs, (hq * hd, vocab), typ, 0.2)[0]
        self.u = dev(rs.rand(n), torch.float32)

    def run(self):
        o = self.ops
        q, k = o.qk_rope(self.q, self.k, self.pos + self.plen, self.freq, gq=self.gq, gk=self.gk)
        o.kv4_write(self.cache, k, self.v, self.pos)
        att = o.kv4_attend_shared(q, self.cache, self.pos, self.prefix, self.length)
        logits = att.flatten(1).float() @ self.head.float()
        tok, lp = o.sample(logits, self.u, 0.8, 50, 0.95)
        again, *_ = o.logprobs(logits, tok)
        return q, k, att, logits, tok, lp, again


@pytest.mark.parametrize("typ", list(TYPES))
def test_a_served_step_of_answers(ops, typ):
    s = Step(ops, typ)
    q64, k64, at = host(s.q), host(s.k), s.pos.cpu().numpy() + s.plen
    q, k, att, logits, tok, lp, again = s.run()
    check_rope(typ, q, q64, at, s.freq.cpu().numpy(), s.gq.cpu().numpy(), 1e-5, False)
    check_rope(typ, k, k64, at, s.freq.cpu().numpy(), s.gk.cpu().numpy(), 1e-5, False)
    pos = s.pos.cpu().tolist()
    o, pv, big, cnt = sref.attend_shared(host(q), s.cache.data.cpu().numpy(), 40, pos, list(range(s.n)), None,
                                         s.prefix.data.cpu().numpy(), 96, [s.plen], [0], None, None, s.hd ** -0.5)
    assert (np.abs(host(att) - o) <= ref.attend_tolerance(typ, o, pv, big, cnt, s.hd, rounded=typ == "bf16")).all()
    for r in range(s.n):
        want, wlp = sref.sample(host(logits)[r], float(s.u[r]), float(np.float32(0.8)), 50, float(np.float32(0.95)))
        assert int(tok[r]) == want and abs(float(lp[r]) - wlp) <= 2.0 ** -24 * abs(wlp) + 1e-9
    assert (again < 0).all()


def test_served_steps_captured_and_side_by_side(ops):
    """Graphs of whole steps, replayed with the program's own calls between
    them and side by side on two streams, give what eager steps give."""
    steps = [Step(ops, "f32", seed=1), Step(ops, "bf16", n=40, plen=96, seed=2)]
    twins = [Step(ops, "f32", seed=1), Step(ops, "bf16", n=40, plen=96, seed=2)]
    for s in twins:
        s.run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = s.run()
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in steps]
    rs = np.random.RandomState(17)
    for i in range(5):
        want = []
        for s, t in zip(steps, twins):
            fresh, u = rand(rs, tuple(s.x.shape), s.typ)[0], dev(rs.rand(s.n), torch.float32)
            for y in (s, t):
                y.x.copy_(fresh)
                y.u.copy_(u)
                y.pos.add_(1)
            t.cache.data.copy_(s.cache.data)
            want.append(t.run())
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, t, out, w in zip(steps, twins, outs, want):
            assert torch.equal(s.cache.data, t.cache.data), i
            assert all(torch.equal(a, b) for a, b in zip(out, w)), i


class LongStep(Step):
    """A Step whose every launch there is takes part: own positions in pieces with
    the join, rows of logits in pieces with their bins in a workspace."""

    def __init__(self, ops, typ, seed=0, slots=700, **kw):
        super().__init__(ops, typ, seed=seed, vocab=66001, **kw)
        rs = np.random.RandomState(seed)
        self.cache = filled(ops, rs, self.n, slots, self.cache.heads, self.hd)
        self.pos = dev(rs.randint(0, 2 * slots, self.n))
        self.head = self.head * 0.2

    def run(self):
        o = self.ops
        q, k = o.qk_rope(self.q, self.k, self.pos + self.plen, self.freq, gq=self.gq, gk=self.gk)
        o.kv4_write(self.cache, k, self.v, self.pos)
        att = o.kv4_attend_shared(q, self.cache, self.pos, self.prefix, self.length)
        logits = att.flatten(1).float() @ self.head.float()
        tok, lp = o.sample(logits, self.u, 1.3, 0, 0.95, 1e-4)
        return q, k, att, logits, tok, lp


def test_long_steps_captured_and_side_by_side(ops):
    """As test_served_steps_captured_and_side_by_side, of the launches that hand
    counters, bins and pieces on: two graphs of their own workspaces, replayed on
    two streams with other inputs each time."""
    make = lambda: [LongStep(ops, "f32", seed=1), LongStep(ops, "bf16", n=9, plen=96, seed=2)]  # noqa: E731
    steps, twins = make(), make()
    for s in twins:
        assert own_pieces(ops, s.cache, s.n, 4, [0] * s.n) and ops.lib().ana_row_sample_ws(s.n, 66001) > 0
        s.run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in steps]
    rs = np.random.RandomState(34)
    for i in range(5):
        want = []
        for s, t in zip(steps, twins):
            fresh, u = rand(rs, tuple(s.x.shape), s.typ)[0], dev(rs.rand(s.n), torch.float32)
            for y in (s, t):
                y.x.copy_(fresh)
                y.u.copy_(u)
                y.pos.add_(37)
            t.cache.data.copy_(s.cache.data)
            want.append(t.run())
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, t, out, w in zip(steps, twins, outs, want):
            assert torch.equal(s.cache.data, t.cache.data), i
            assert all(torch.equal(a, b) for a, b in zip(out, w)), i
            for r in range(s.n):
                tok, lp = sref.sample(host(out[3])[r], float(s.u[r]), float(np.float32(1.3)), 0, float(np.float32(0.95)),
                                      float(np.float32(1e-4)))
                assert int(out[4][r]) == tok and abs(float(out[5][r]) - lp) <= 2.0 ** -24 * abs(lp) + 1e-9


def test_calls_of_none(ops):
    e = torch.empty
    q, k = ops.qk_rope(e((0, 2, 32), device="cuda"), None, dev([]), dev(freqs(32), torch.float32))
    assert q.shape == (0, 2, 32) and k is None
    cache = ops.KV4.empty(1, 32, 2, 32)
    assert ops.kv4_attend_shared(e((0, 2, 32), device="cuda"), cache, dev([]), cache, dev([5])).shape == (0, 2, 32)
    tok, lp = ops.sample(e((0, 9), device="cuda"), e(0, device="cuda"))
    assert tok.shape == (0,) and lp.shape == (0,)


def test_mirror_checks(ops):
    x, u = torch.zeros((2, 9), device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(ValueError, match="u: a consecutive float32"):
        ops.sample(x, u.double())
    with pytest.raises(ValueError, match="top_k: a consecutive int32"):
        ops.sample(x, u, top_k=u)
    with pytest.raises(ValueError, match="top_k"):
        ops.sample(x, u, top_k=-1)
    with pytest.raises(ana_amd.AnaError, match="temperature"):
        ops.sample(x, u, temperature=-1.0)
    with pytest.raises(ana_amd.AnaError, match="unknown type"):
        ops.sample(x.double(), u)
    q = torch.zeros((2, 2, 32), device="cuda")
    with pytest.raises(ValueError, match="k: "):
        ops.qk_rope(q, q.half(), dev([0, 1]), u)
    with pytest.raises(ana_amd.AnaError, match="turned values"):
        ops.qk_rope(q, q, dev([0, 1]), u)
    cache = ops.KV4.empty(2, 32, 2, 32)
    with pytest.raises(ValueError, match="off: "):
        ops.kv4_attend_shared(q, cache, dev([0, 1]), cache, dev([1]), poff=dev([0]))
    with pytest.raises(ana_amd.AnaError, match="without offsets"):
        ops.kv4_attend_shared(q, cache, dev([0, 1]), cache, dev([1, 1]))
