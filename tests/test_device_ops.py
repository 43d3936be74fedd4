"""The operators on device memory without a GPU: what the C ABI and its
mirror refuse, before a device is touched, and the 64-bit forms that the GPU
tests compare with."""
import ctypes as C
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import ana_amd
import device_ops_ref as ref
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


def mat(p=A, row=128, head=64):
    return ops._Mat(p, row, head)


def write(c, r, k, v, typ=0):
    L = ana_amd.lib()
    ref_ = lambda x: None if x is None else C.byref(x)  # noqa: E731
    out = [L.ana_kv4_write(ref_(c), ref_(r), typ, ref_(k), ref_(v), None),
           L.ana_kv4_read(ref_(c), ref_(r), typ, ref_(k), ref_(v), None)]
    assert out[0] == out[1]
    return out[0], L.ana_error(None).decode()


def attend(c, r, q, o, hq=4, typ=0, ws=A, nws=1 << 40):
    L = ana_amd.lib()
    ref_ = lambda x: None if x is None else C.byref(x)  # noqa: E731
    rc = L.ana_kv4_attend(ref_(c), ref_(r), typ, ref_(q), hq, 0.125, None, ref_(o), 0, ws, nws, None)
    return rc, L.ana_error(None).decode()


BAD_CACHES = [(None, "null cache"), (cache(data=None), "null cache"), (cache(hd=48), "head size"),
              (cache(hd=0), "head size"), (cache(seqs=0), "no sequences"), (cache(slots=0), "no sequences"),
              (cache(heads=0), "no sequences"), (cache(heads=70000), "65535 heads"),
              (cache(slots=0xFFFFFFFF), "slots"), (cache(data=A + 8), "16-byte"),
              (cache(seqs=1 << 31, slots=1 << 30, heads=60000), "beyond any memory")]
BAD_ROWS = [(None, "null rows"), (rows(pos=None), "null positions"), (rows(rows=3), "without offsets"),
            (rows(n=3, rows=3, seq=None), "in a cache of 2"), (rows(rows=1 << 31, off=A), "2^26"),
            (rows(n=(1 << 26) + 1, rows=0, off=A), "2^26")]


@pytest.mark.parametrize("c,why", BAD_CACHES)
def test_refuses_caches(c, why):
    for rc, msg in (write(c, rows(), mat(), mat()), attend(c, rows(), mat(), mat())):
        assert rc == ana_amd.ANA_EINVAL and why in msg


@pytest.mark.parametrize("r,why", BAD_ROWS)
def test_refuses_rows(r, why):
    for rc, msg in (write(cache(), r, mat(), mat()), attend(cache(), r, mat(row=256), mat(row=256))):
        assert rc == ana_amd.ANA_EINVAL and why in msg


@pytest.mark.parametrize("typ", [-1, 3, 77])
def test_refuses_types(typ):
    for rc, msg in (write(cache(), rows(), mat(), mat(), typ), attend(cache(), rows(), mat(), mat(), typ=typ)):
        assert rc == ana_amd.ANA_EINVAL and "unknown type" in msg


@pytest.mark.parametrize("m,why", [(None, "null"), (mat(p=None), "null"), (mat(p=A + 2), "border"),
                                   (mat(row=63), "overlap"), (mat(head=63), "overlap"), (mat(head=0), "overlap")])
def test_refuses_tensors(m, why):
    for rc, msg in (write(cache(), rows(), m, mat()), write(cache(), rows(), mat(), m),
                    attend(cache(), rows(), m, mat(row=256)), attend(cache(), rows(), mat(row=256), m)):
        assert rc == ana_amd.ANA_EINVAL and why in msg


def test_refuses_heads_and_workspaces():
    for hq in (0, 3, 5):
        rc, msg = attend(cache(), rows(), mat(), mat(), hq=hq)
        assert rc == ana_amd.ANA_EINVAL and "query heads" in msg
    # 2^31 pairs; 2^24 workgroups of single rows; of ragged ones
    for c, r, hq in ((cache(), rows(n=1 << 20, rows=1 << 26, off=A), 32), (cache(), rows(n=1 << 23, rows=1 << 23), 2),
                     (cache(), rows(n=1 << 23, rows=9, off=A), 2)):
        rc, msg = attend(c, r, mat(row=64 * hq), mat(row=64 * hq), hq=hq)
        assert rc == ana_amd.ANA_EINVAL and "than a launch takes" in msg
    long = cache(slots=1 << 20)
    need = ana_amd.lib().ana_kv4_attend_ws(C.byref(long), C.byref(rows()), 4, 0)
    assert need > 0 and need % (2 * 4 * 16) == 0
    for ws, n in ((None, need), (A, need - 1), (A + 4, need)):
        rc, msg = attend(long, rows(), mat(row=256), mat(row=256), ws=ws, nws=n)
        assert rc == ana_amd.ANA_EINVAL and "workspace" in msg
    # a known length needs no more of it than the ring
    assert ana_amd.lib().ana_kv4_attend_ws(C.byref(long), C.byref(rows()), 4, 40) == 0


@pytest.mark.parametrize("m", [mat(row=64, head=64), mat(row=127, head=64), mat(row=64, head=127),
                               mat(row=1 << 63, head=1 << 63)])
def test_refuses_outputs_that_overlap(m):
    """Strides that are wide enough one by one, not together."""
    L = ana_amd.lib()
    c, r, ok = cache(), rows(), mat()
    for k, v in ((m, ok), (ok, m)):
        rc = L.ana_kv4_read(C.byref(c), C.byref(r), 0, C.byref(k), C.byref(v), None)
        assert rc == ana_amd.ANA_EINVAL and "overlap" in L.ana_error(None).decode()
    rc, msg = attend(c, r, ok, m, hq=2)
    assert rc == ana_amd.ANA_EINVAL and "overlap" in msg


@pytest.mark.parametrize("heads,hq,hd,slots", [(12, 12, 64, 2048), (24, 24, 64, 60000), (8, 32, 128, 131072), (1, 16, 32, 9000),
                                               (3, 3, 64, 700), (1, 64, 128, 1 << 20)])
@pytest.mark.parametrize("n", [1, 2, 7, 24, 64, 200, 5000])
@pytest.mark.parametrize("each", [0, 1, 2, 4, 16, 100, 1000])
def test_pieces_fill_the_chip_once(heads, hq, hd, slots, n, each):
    """A call is cut into pieces only as far as three workgroups a CU: one for
    each sequence and key head at least (0 rows each: single rows, without
    offsets), and one for every 128 pairs. The workspace tells the pieces."""
    c = cache(seqs=n, slots=slots, heads=heads, hd=hd)
    r = rows(n=n, rows=n * max(each, 1), off=A if each else None)
    ws = ana_amd.lib().ana_kv4_attend_ws(C.byref(c), C.byref(r), hq, 0)
    one = 4 * n * max(each, 1) * hq * (4 + hd)
    assert ws % one == 0
    pieces = max(1, ws // one)
    g = hq // heads
    groups = heads * max(n * (1 if each else -(-g // 16)), n * each * g // 128)
    assert pieces == 1 or pieces * groups <= 3 * 256
    assert pieces <= max(1, -(-slots // 32) // (8 if each else 4))
    # as many as that where the ring is long
    assert pieces == 128 or pieces == max(1, -(-slots // 32) // (8 if each else 4)) or 2 * pieces * groups + 2 * groups > 3 * 256


def test_empty_calls_touch_nothing():
    assert write(cache(), rows(n=0, rows=0), mat(), mat())[0] == 0
    assert attend(cache(), rows(n=0, rows=0), mat(row=256), mat(row=256))[0] == 0
    assert write(cache(), rows(n=2, rows=0, off=A), mat(p=None), mat(p=None))[0] == 0


def test_cache_bytes():
    L = ana_amd.lib()
    assert L.ana_kv4_bytes(3, 65, 2, 64) == 3 * 2 * 3 * 34 * 64
    for bad in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 16), (1, 1, 1, 256), (1, 1, 70000, 64)):
        assert L.ana_kv4_bytes(*bad) == 0


def logprobs(**kw):
    d = dict(device=0, type=0, logits=A, ld=100, n=2, vocab=100, tok=A, top=3, lp=A, ent=A, rank=A, top_tok=A,
             top_lp=A, ws=A, nws=1 << 30)
    d.update(kw)
    L = ana_amd.lib()
    return L.ana_row_logprobs(*d.values(), None), L.ana_error(None).decode()


@pytest.mark.parametrize("kw,why", [
    (dict(type=9), "unknown type"), (dict(vocab=0, top=0), "vocabulary"), (dict(vocab=1 << 22, ld=1 << 22), "vocabulary"),
    (dict(top=65), "alternatives"), (dict(vocab=5, top=6), "alternatives"), (dict(ld=99), "overlap"),
    (dict(logits=None), "null"), (dict(ent=None), "null"), (dict(lp=None), "null"), (dict(rank=None), "null"),
    (dict(top_tok=None), "null"), (dict(top_lp=None), "null"), (dict(logits=A + 2), "border"),
    (dict(n=1 << 24), "at most 16777215"), (dict(vocab=9000, ld=9000, n=1 << 22), "at most 4194303"), (dict(vocab=40000, ld=40000, ws=None), "workspace"),
    (dict(vocab=40000, ld=40000, nws=8), "workspace")])
def test_refuses_logprobs(kw, why):
    rc, msg = logprobs(**kw)
    assert rc == ana_amd.ANA_EINVAL and why in msg


def test_empty_logprobs():
    assert logprobs(n=0)[0] == 0
    assert ana_amd.lib().ana_row_logprobs_ws(1, 0, 0) == 0
    assert ana_amd.lib().ana_row_logprobs_ws(1, 100, 65) == 0


def test_mirror_refuses_host_tensors_and_shapes():
    with pytest.raises(ValueError, match="not on a GPU"):
        ops.KV4(torch.zeros((1, 1, 2, 34 * 64), dtype=torch.uint8), 64)
    with pytest.raises(ValueError, match="not a cache"):
        ops.KV4(torch.zeros((1, 1, 2, 34 * 64), dtype=torch.uint8), 65)
    with pytest.raises(ValueError, match="uint8"):
        ops.KV4(torch.zeros((1, 1, 2, 34 * 64)), 64)
    with pytest.raises(ValueError, match="no cache"):
        ops.KV4.empty(1, 64, 1, 48, device="cpu")
    with pytest.raises(ValueError, match="not on a GPU"):
        ops.logprobs(torch.zeros(2, 5))
    with pytest.raises(ValueError, match="consecutive"):
        ops.logprobs(torch.zeros(5, 4).t())


@pytest.mark.parametrize("first,ok", [("ana_amd.ops, ana_amd; ana_amd.lib()", True), ("torch, ana_amd; ana_amd.lib()", True),
                                      ("ana_amd; ana_amd.lib()", False)])
def test_mirror_refuses_a_second_runtime(first, ok):
    """torch's HIP runtime loaded after libana.so's, where they are not the
    same file, would find no GPU."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = f"import {first}; import torch, glob, os; n = glob.glob(os.path.dirname(torch.__file__) + '/lib/libamdhip64*'); " \
           "print('own' if n else 'shared', flush=True); import ana_amd.ops; print('loaded')"
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=110)
    if ok or r.stdout.startswith("shared"):
        assert r.stdout.endswith("loaded\n"), r.stderr
    else:
        assert r.stdout == "own\n" and "import torch before the first call of ana_amd" in r.stderr


# ---------------------------------------------------------------- the 64-bit forms

def test_reference_layout_is_a_permutation():
    """Every byte half of a record is one value's, every scale byte one block's."""
    for hd in (32, 64, 128):
        half, scale = [], []
        for s in range(32):
            key, val, sh, kb, vb = ref.places(hd, s)
            half += list(key * 2 + sh // 4) + list(val * 2 + sh // 4)
            scale += list(kb) + list(vb)
        assert sorted(half) == list(range(2 * 32 * hd))
        assert sorted(scale) == list(range(32 * hd, 34 * hd))


def test_reference_quantisation():
    x = np.zeros((1, 32))
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]
    c, s = ref.quant(x)
    assert list(c[0, :8]) == [0, 2, 2, 4, 4, 6, 6, 7] and s[0, 0] == 127
    r = np.random.RandomState(0).randn(50, 64).astype(np.float32)
    c, s = ref.quant(r)
    y = ref.values(c, s)
    step = 2.0 ** (s.astype(float) - 127)
    assert (np.abs(r - y) <= np.repeat(step, 32, -1)).all()
    a = np.abs(r).reshape(50, 2, 32).max(-1)
    assert (a <= 7 * step).all() and (a > 3.5 * step).all()


def test_reference_logprobs():
    x = np.random.RandomState(1).randn(40)
    p = np.exp(x) / np.exp(x).sum()
    lp, ent, rank, ids, tlp, _ = ref.logprobs(x, 7, 40)
    assert abs(lp - math.log(p[7])) < 1e-12 and abs(ent + (p * np.log(p)).sum()) < 1e-12
    assert rank == int((x > x[7]).sum()) and np.allclose(np.exp(tlp).sum(), 1.0)


def test_reference_attention_is_softmax():
    rs = np.random.RandomState(2)
    data = rs.randint(0, 256, (1, 1, 2, 34 * 32)).astype(np.uint8)
    data[..., 32 * 32:] = rs.randint(125, 128, (1, 1, 2, 2 * 32))
    q = rs.randn(3, 2, 32)
    o, pv, big, cnt = ref.attend(q, data, 40, [4], [0], [0, 3], None, 0.2)
    K, V = ref.get(data, 0, 0, 40)
    for r in range(3):
        w = np.exp(0.2 * K[:5 + r] @ q[r, 1])
        assert np.allclose(o[r, 1], (w / w.sum()) @ V[:5 + r])
    assert cnt.max() == 7
