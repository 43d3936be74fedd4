"""Rotation with head norms, attention behind shared prefixes and sampling
without a GPU: what the C ABI and its mirror refuse before a device is touched,
and the 64-bit forms that the GPU tests compare with."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import ana_amd
import serve_ops_ref as sref
from ana_amd import ops

A = 1 << 20   # an address that is never read: every call here is refused or empty


def cache(**kw):
    d = dict(data=A, device=0, seqs=2, slots=64, heads=2, hd=64)
    d.update(kw)
    return ops._Kv4(*(d[k] for k in ("data", "device", "seqs", "slots", "heads", "hd")))


def rows(**kw):
    d = dict(n=2, rows=2, seq=A, pos=A, off=None)
    d.update(kw)
    return ops._Rows(*(d[k] for k in ("n", "rows", "seq", "pos", "off")))


def mat(p=A, row=256, head=64):
    return ops._Mat(p, row, head)


def by(x):
    return None if x is None else C.byref(x)


def error():
    return ana_amd.lib().ana_error(None).decode()


# ---------------------------------------------------------------- qk_rope

def rope(**kw):
    d = dict(hd=64, r=rows(seq=None), type=0, rot=64, near=0, freq=A, gq=A, gk=A, eps=1e-5, hq=4, q=mat(), qo=mat(), hk=4,
             k=mat(), ko=mat())
    d.update(kw)
    f = None if d["rot"] is None else ops._Rope(d["freq"], d["rot"], d["near"], d["gq"], d["gk"], d["eps"])
    rc = ana_amd.lib().ana_qk_rope(0, d["hd"], by(d["r"]), d["type"], by(f), d["hq"], by(d["q"]), by(d["qo"]), d["hk"],
                                   by(d["k"]), by(d["ko"]), None)
    return rc, error()


@pytest.mark.parametrize("kw,why", [
    (dict(hd=0), "head size"), (dict(hd=8), "head size"), (dict(hd=72), "head size"), (dict(hd=272), "head size"),
    (dict(r=None), "null rows"), (dict(r=rows(pos=None)), "null positions"), (dict(r=rows(rows=3)), "without offsets"),
    (dict(r=rows(rows=1 << 31, off=A)), "2^26"), (dict(r=rows(n=(1 << 26) + 1, rows=0, off=A)), "2^26"),
    (dict(type=3), "unknown type"), (dict(rot=None), "null rotation"), (dict(rot=8), "turned values"),
    (dict(rot=80), "turned values"), (dict(freq=None), "null frequencies"), (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"), (dict(hq=0, hk=0), "heads"), (dict(hq=70000), "heads"), (dict(hk=70000), "heads"),
    (dict(q=None), "null q"), (dict(qo=None), "null q's output"), (dict(k=None), "null k"), (dict(ko=mat(p=None)), "null k's output"),
    (dict(q=mat(p=A + 2)), "border"), (dict(k=mat(row=63)), "overlap"), (dict(qo=mat(row=64, head=64)), "overlap"),
    (dict(ko=mat(row=255)), "overlap")])
def test_refuses_rope(kw, why):
    rc, msg = rope(**kw)
    assert rc == ana_amd.ANA_EINVAL and why in msg


def test_empty_rope():
    assert rope(r=rows(n=0, rows=0))[0] == 0
    assert rope(r=rows(n=2, rows=0, off=A), q=mat(p=None), qo=mat(p=None), k=mat(p=None), ko=mat(p=None))[0] == 0
    # (heads of none are not looked at)
    assert rope(r=rows(n=0, rows=0), hk=0, k=None, ko=None)[0] == 0


# ---------------------------------------------------------------- attention behind prefixes

def shared(**kw):
    d = dict(c=cache(), r=rows(), pc=cache(slots=1024), pre=rows(n=1), type=0, q=mat(), hq=4, o=mat(), ws=A, nws=1 << 40)
    d.update(kw)
    rc = ana_amd.lib().ana_kv4_attend_shared(by(d["c"]), by(d["r"]), by(d["pc"]), by(d["pre"]), d["type"], by(d["q"]),
                                             d["hq"], 0.125, None, by(d["o"]), 0, 0, d["ws"], d["nws"], None)
    return rc, error()


@pytest.mark.parametrize("kw,why", [
    (dict(c=None), "null cache"), (dict(pc=None), "null cache"), (dict(pc=cache(data=None)), "null cache"),
    (dict(pc=cache(heads=1)), "another device"), (dict(pc=cache(hd=32)), "another device"),
    (dict(pc=cache(device=1)), "another device"), (dict(pc=cache(data=A + 4)), "16-byte"), (dict(r=None), "null rows"),
    (dict(pre=None), "null prefixes"), (dict(pre=rows(n=1, pos=None)), "null prefix lengths"),
    (dict(pre=rows(n=1, rows=3)), "not 2"), (dict(pre=rows(n=2)), "without offsets"), (dict(pre=rows(n=0)), "without offsets"),
    (dict(pre=rows(n=3, seq=None, off=A)), "in a cache of 2"), (dict(pre=rows(n=(1 << 26) + 1, off=A)), "2^26"),
    (dict(pre=rows(n=1 << 24, off=A)), "than a launch takes"), (dict(type=7), "unknown type"), (dict(hq=3), "query heads"),
    (dict(q=None), "null q"), (dict(o=mat(row=64)), "overlap"), (dict(ws=None), "workspace"), (dict(ws=A + 8), "16-byte")])
def test_refuses_shared(kw, why):
    rc, msg = shared(**kw)
    assert rc == ana_amd.ANA_EINVAL and why in msg


def test_shared_workspace():
    L = ana_amd.lib()
    args = lambda c=cache(), r=rows(), pc=cache(slots=1 << 16), p=rows(n=1): (by(c), by(r), by(pc), by(p))  # noqa: E731
    need = L.ana_kv4_attend_shared_ws(*args(), 4, 0, 0)
    # a place for each (row, head) of one own piece and one of the prefix at least
    assert need >= 4 * 2 * 4 * 2 * 68 and need % (4 * 68) == 0
    for n in (need - 1, 0):
        rc, msg = shared(pc=cache(slots=1 << 16), nws=n)
        assert rc == ana_amd.ANA_EINVAL and "workspace" in msg
    # a shorter prefix needs no more
    assert L.ana_kv4_attend_shared_ws(*args(), 4, 0, 100) <= need
    for bad in (args(c=cache(hd=48)), args(pc=cache(heads=3)), args(pc=cache(slots=0)), (None,) * 4):
        assert L.ana_kv4_attend_shared_ws(*bad, 4, 0, 0) == 0
    assert L.ana_kv4_attend_shared_ws(*args(), 5, 0, 0) == 0


def test_empty_shared():
    assert shared(r=rows(n=0, rows=0), pre=rows(n=1, rows=0))[0] == 0
    assert shared(r=rows(n=2, rows=0, off=A), pre=rows(n=0, rows=0, off=A), q=mat(p=None), o=mat(p=None))[0] == 0


# ---------------------------------------------------------------- sampling

def sample(**kw):
    d = dict(type=0, logits=A, ld=100, n=2, vocab=100, u=A, tok=A, lp=A, t=1.0, p=1.0, q=0.0, k=0, ts=None, ps=None, qs=None,
             ks=None, s=True, ws=A, nws=1 << 40)
    d.update(kw)
    s = ops._Draw(d["t"], d["p"], d["q"], d["k"], d["ts"], d["ps"], d["qs"], d["ks"]) if d["s"] else None
    rc = ana_amd.lib().ana_row_sample(0, d["type"], d["logits"], d["ld"], d["n"], d["vocab"], d["u"], by(s), d["tok"],
                                      d["lp"], d["ws"], d["nws"], None)
    return rc, error()


@pytest.mark.parametrize("kw,why", [
    (dict(type=-1), "unknown type"), (dict(vocab=0), "vocabulary"), (dict(vocab=(1 << 21) + 1, ld=1 << 22), "vocabulary"),
    (dict(n=1 << 22), "rows"), (dict(ld=99), "overlap"), (dict(s=False), "null settings"), (dict(t=-0.5), "temperature"),
    (dict(t=math.nan), "temperature"), (dict(p=-0.1), "top-p"), (dict(p=1.5), "top-p"), (dict(p=math.nan), "top-p"),
    (dict(q=-0.1), "min-p"), (dict(q=1.1), "min-p"), (dict(q=math.nan), "min-p"), (dict(logits=None), "null"),
    (dict(u=None), "null"), (dict(tok=None), "null"), (dict(lp=None), "null"), (dict(logits=A + 2), "border")])
def test_refuses_sample(kw, why):
    rc, msg = sample(**kw)
    assert rc == ana_amd.ANA_EINVAL and why in msg


def test_sample_workspace():
    """Few long rows take one."""
    L = ana_amd.lib()
    assert L.ana_row_sample_ws(1, 32000) == 0 and L.ana_row_sample_ws(3000, 200000) == 0 and L.ana_row_sample_ws(0, 200000) == 0
    need = L.ana_row_sample_ws(2, 200000)
    assert need > 2 * 8 * 2048
    for kw in (dict(ws=None), dict(nws=need - 1), dict(ws=A + 4)):
        rc, msg = sample(vocab=200000, ld=200000, **kw)
        assert rc == ana_amd.ANA_EINVAL and "workspace" in msg
    assert L.ana_row_sample_ws(1, 0) == 0 and L.ana_row_sample_ws(1, (1 << 21) + 1) == 0


def test_empty_sample():
    assert sample(n=0)[0] == 0


def test_mirror_refuses():
    x = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="not on a GPU"):
        ops.qk_rope(x, None, torch.zeros(2, dtype=torch.int32), torch.zeros(32))
    with pytest.raises(ValueError, match="not on a GPU"):
        ops.sample(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(ValueError, match="consecutive"):
        ops.sample(torch.zeros(5, 4).t(), torch.zeros(4))


# ---------------------------------------------------------------- the 64-bit forms

def test_reference_rope():
    rs = np.random.RandomState(0)
    x, f = rs.randn(3, 2, 32), (10000.0 ** (-np.arange(8) / 8.0)).astype(np.float32)
    for near in (False, True):
        o, off = sref.rope(x, [0, 5, 77], f, None, 1e-5, near)
        assert np.array_equal(o[0], x[0]) and np.array_equal(o[..., 16:], x[..., 16:])
        assert np.allclose((o ** 2).sum(-1), (x ** 2).sum(-1)) and (off >= 0).all()
        a, b = (0, 1) if near else (0, 8)
        z = (x[1, :, a] + 1j * x[1, :, b]) * np.exp(5j * float(f[0]))
        assert np.allclose(o[1, :, a], z.real) and np.allclose(o[1, :, b], z.imag)
    g = rs.randn(32)
    o, _ = sref.rope(x, [0, 0, 0], f, g, 0.0, False)
    assert np.allclose(((o / (1 + g)) ** 2).mean(-1), 1.0)


def test_reference_sample():
    x = np.array([1.0, 3.0, 2.0, 3.0, -math.inf, math.nan])
    p = np.exp(x[:4]) / np.exp(x[:4]).sum()
    got = [sref.sample(x, u)[0] for u in (0.0, p[1] - 1e-9, p[1] + 1e-9, 2 * p[1] + 1e-9, 1 - p[0] + 1e-9, 1.0)]
    assert got == [1, 1, 3, 2, 0, 0]
    assert abs(sref.sample(x, 0.0)[1] - math.log(p[1])) < 1e-12
    assert sref.sample(x, 0.99, k=1) == (1, 0.0) and sref.sample(x, 0.99, t=0.0) == (1, 0.0)
    assert sref.sample(x, 0.99, k=2)[0] == 3 and sref.sample(x, 0.99, p=2 * p[1] - 1e-9)[0] == 3
    assert sref.sample(x, 0.99, p=2 * p[1] + 1e-9)[0] == 2 and sref.sample(x, 0.99, q=0.3)[0] == 2
    assert sref.sample(x, 0.99, q=0.4)[0] == 3 and sref.sample([math.inf, 1, math.inf], 0.6) == (2, -math.log(2.0))
    assert sref.sample([-math.inf, math.nan], 0.5)[0] == -1


def test_reference_shared_is_softmax():
    """A prefix and a sequence's own tokens as one sequence."""
    import device_ops_ref as ref
    rs = np.random.RandomState(2)
    mk = lambda n, t: rs.randint(0, 256, (n, 1, t, 34 * 32)).astype(np.uint8)  # noqa: E731
    data, pdata = mk(2, 1), mk(1, 2)
    for d in (data, pdata):
        d[..., 32 * 32:] = rs.randint(125, 128, (*d.shape[:3], 64))
    q = rs.randn(2, 2, 32)
    o, _, _, cnt = sref.attend_shared(q, data, 32, [3, 7], [1, 0], None, pdata, 64, [40], [0], None, [0.5, -1.0], 0.2)
    for r, (s, n) in enumerate(((1, 4), (0, 8))):
        K, V = ref.get(data, s, 0, 32)
        P, W = ref.get(pdata, 0, 0, 64)
        K, V = np.concatenate([P[:40], K[:n]]), np.concatenate([W[:40], V[:n]])
        w = np.exp(0.2 * K @ q[r, 1])
        assert np.allclose(o[r, 1], w @ V / (w.sum() + math.exp(-1.0))) and cnt[r, 1, 0] == 40 + n
