"""Contexts whose softmax rings are held in 4 bits (ANA_KV4), against the
model in 64 bits over the rings that the context itself holds, and the log
probabilities of ana_logprobs and ana_score_logprobs_n against the logits."""
import ctypes
import math

import numpy as np
import pytest

import ana_amd
import device_ops_ref as ref
from ana_amd import ckpt
from ana_amd import config as cf
from ana_amd import ops

pytestmark = pytest.mark.gpu

# hd 64 with every arm on, and hd 32 with none; one softmax layer, the last
MID = cf.Config(vocab=258, ctx=64, d=256, f=1024, layers=4, heads=4, rglru=True, qk=True, sinks=True, tied=True)
THIN = cf.Config(vocab=258, ctx=40, d=128, f=256, layers=4, heads=4, rglru=False, qk=False, sinks=False, tied=True)
TOL = {ana_amd.FAST_FP32: 1e-4, ana_amd.BF16: 2e-2}


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4")
    out = {}
    for name, c in (("mid", MID), ("thin", THIN)):
        w = ckpt.init_params(c, "normal", 5, trained=True)
        path = str(d / f"{name}.ftc2")
        ckpt.write(path, c, w)
        out[name] = (c, path, np.asarray(w, dtype=np.float64))
    return out


class Row:
    """One sequence in 64 bits: GLA states of its own, the softmax layer over
    rings that it is given."""

    def __init__(self, c, w):
        self.c = c
        self.blk, fin = cf.layout(c)
        self.w, self.fin = w, w[fin:fin + c.d]
        self.emb = w[:c.vocab * c.d].reshape(c.vocab, c.d)
        self.S = {i: np.zeros((c.heads, c.hd, c.hd)) for i in range(c.layers) if not c.is_softmax(i)}

    def mat(self, at, rows, cols):
        return self.w[at:at + rows * cols].reshape(rows, cols)

    @staticmethod
    def norm(x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * g

    def feed(self, tok, pos, ring):
        """The logits after a token, and the softmax layer's k and v."""
        c, d = self.c, self.c.d
        x = self.emb[tok].copy()
        for i, b in enumerate(self.blk):
            y = self.norm(x, self.w[b.ra:b.ra + d])
            q, k, v = (self.mat(a, d, d) @ y for a in (b.wq, b.wk, b.wv))
            q, k, v = (t.reshape(c.heads, c.hd) for t in (q, k, v))
            if b.gla:
                z = (self.mat(b.wa, d, d) @ y).reshape(c.heads, c.hd)
                q, k = (t / np.sqrt((t * t).sum(-1, keepdims=True) + 1e-6) for t in (q, k))
                sg = 1.0 / (1.0 + np.exp(-z))
                al = sg
                if c.rglru:
                    lam = -np.log1p(np.exp(-self.w[b.lam:b.lam + d])).reshape(c.heads, c.hd)
                    la = np.minimum(8.0 * sg * lam, -float(np.float32(1e-4)))
                    k, al = k * np.sqrt(-np.expm1(2.0 * la)), np.exp(la)
                self.S[i] = self.S[i] * al[:, :, None] + k[:, :, None] * v[:, None, :]
                o = np.einsum("hk,hkv->hv", q, self.S[i])
            else:
                if c.qk:
                    q = self.norm(q, 1.0 + self.w[b.gq:b.gq + c.hd])
                    k = self.norm(k, 1.0 + self.w[b.gk:b.gk + c.hd])
                kv = (k, v)
                live = min(pos, c.ctx - 1) + 1
                K, V = ring
                o = np.zeros((c.heads, c.hd))
                for h in range(c.heads):
                    s = K[:live, h] @ q[h] / math.sqrt(c.hd)
                    snk = self.w[b.sink + h] if c.sinks else -math.inf
                    m = max(s.max(), snk)
                    e = np.exp(s - m)
                    o[h] = e @ V[:live, h] / (e.sum() + math.exp(snk - m))
            x = x + self.mat(b.wo, d, d) @ o.reshape(d)
            y = self.norm(x, self.w[b.rf:b.rf + d])
            g = self.mat(b.wg, c.f, d) @ y
            x = x + self.mat(b.wd, d, c.f) @ (g / (1.0 + np.exp(-g)) * (self.mat(b.wu, c.f, d) @ y))
        return self.emb @ self.norm(x, self.fin), kv


def rings(dec, seq, c):
    a = dec.state(seq, 3).astype(np.float64).reshape(2, c.ctx, c.heads, c.hd)
    return a[0], a[1]


def rel(got, want):
    return float(np.abs(np.asarray(got, np.float64) - want).max() / np.abs(want).max())


def tokens(n, seed, vocab):
    return [int(t) for t in np.random.RandomState(seed).randint(2, vocab, n)]


def held(c, kv, ring, slot, slack):
    """A stored row is its key and value to the codes' rounding: half the
    widest gap, one scale, with `slack` (the mode's own error) of the block's
    largest."""
    for x, r in zip(kv, ring):
        a = np.abs(x.reshape(c.heads, -1, 32)).max(-1, keepdims=True)
        scale = 2.0 ** np.ceil(np.log2(np.maximum(a, 1e-30) * (1 + slack) / 7.0))
        err = np.abs(x - r[slot]).reshape(c.heads, -1, 32)
        assert (err <= scale * (1 + 1e-6) + slack * a).all(), (err / scale).max()


@pytest.mark.parametrize("mode", [ana_amd.FAST_FP32, ana_amd.BF16], ids=["fast_fp32", "bf16"])
@pytest.mark.parametrize("name", ["mid", "thin"])
def test_tokens_one_at_a_time(models, name, mode):
    """Three sequences fed together, token by token, past the ring's wrap."""
    c, path, w = models[name]
    n, T = 3, c.ctx + 9
    toks = [tokens(T, s, c.vocab) for s in range(n)]
    rows = [Row(c, w) for _ in range(n)]
    with ana_amd.Decoder(path, max_seqs=4, numerics=mode | ana_amd.KV4) as dec:
        seqs = [2, 0, 3]
        for t in range(T):
            dec.feed(seqs, [t] * n, [x[t] for x in toks])
            got = dec.logits(seqs) if t % 7 == 0 or t > T - 4 else None
            for i in range(n):
                ring = rings(dec, seqs[i], c)
                want, kv = rows[i].feed(toks[i][t], t, ring)
                held(c, kv, ring, t % c.ctx, 1e-4 if mode == ana_amd.FAST_FP32 else 4e-2)
                if got is not None:
                    assert rel(got[i], want) <= TOL[mode], (t, i)
        # nothing of the sequence left out
        assert not dec.state(1, 3).any()
        dec.reset(0)
        assert not dec.state(0, 3).any() and dec.state(2, 3).any()


@pytest.mark.parametrize("mode", [ana_amd.FAST_FP32, ana_amd.BF16], ids=["fast_fp32", "bf16"])
@pytest.mark.parametrize("name,lens,chunk", [("mid", [50, 7, 64], 64), ("mid", [3, 90, 20], 16), ("thin", [40, 1, 61], 8),
                                             ("mid", [1, 2], 64)])
def test_prompts(models, name, lens, chunk, mode):
    """Prompts in chunks, short of the wrap and past it, then one token each.
    A prompt's rows see the rings as they were at their own position: the
    64-bit rows are given each slot as it was stored."""
    c, path, w = models[name]
    n = len(lens)
    toks = [tokens(k + 1, 10 + i, c.vocab) for i, k in enumerate(lens)]
    with ana_amd.Decoder(path, max_seqs=n, prefill_chunk=chunk, numerics=mode | ana_amd.KV4) as dec:
        # the rings after every piece, so that slots of the last turn are seen before they are overwritten
        rows = [Row(c, w) for _ in range(n)]
        past = [0] * n
        cut = c.ctx if max(lens) <= c.ctx else 8
        while any(past[i] < lens[i] for i in range(n)):
            piece = [toks[i][past[i]:min(lens[i], past[i] + cut)] for i in range(n)]
            before = [rings(dec, i, c) for i in range(n)]
            dec.feeds_n(list(range(n)), past, piece)
            got = dec.logits(list(range(n)))
            for i in range(n):
                K, V = (x.copy() for x in before[i])
                after = rings(dec, i, c)
                for t, tok in enumerate(piece[i]):
                    p = past[i] + t
                    K[p % c.ctx], V[p % c.ctx] = after[0][p % c.ctx], after[1][p % c.ctx]
                    want, kv = rows[i].feed(tok, p, (K, V))
                    held(c, kv, (K, V), p % c.ctx, 1e-4 if mode == ana_amd.FAST_FP32 else 4e-2)
                if piece[i]:
                    assert rel(got[i], want) <= TOL[mode], (i, past[i])
                past[i] += len(piece[i])
        dec.feed(list(range(n)), lens, [toks[i][-1] for i in range(n)])
        got = dec.logits(list(range(n)))
        for i in range(n):
            want, _ = rows[i].feed(toks[i][-1], lens[i], rings(dec, i, c))
            assert rel(got[i], want) <= TOL[mode], i


@pytest.mark.parametrize("n", [1, 6])
def test_loops_are_the_steps(models, n):
    """The token loops (captured steps, and launch by launch) against feeds
    and picks one at a time: the same kernels, so the same picks."""
    c, path, _ = models["mid"]
    prompts = [tokens(5 + 3 * i, 40 + i, c.vocab) for i in range(n)]
    seqs, pos = list(range(n)), [len(p) - 1 for p in prompts]
    mode = ana_amd.FAST_FP32 | ana_amd.KV4
    with ana_amd.Decoder(path, max_seqs=n, numerics=mode) as a, ana_amd.Decoder(path, max_seqs=n, numerics=mode) as b:
        for d in (a, b):
            d.feeds_n(seqs, [0] * n, [p[:-1] for p in prompts])
        last = [p[-1] for p in prompts]
        out = a.generate(seqs, pos, last, 70)
        cur = list(last)
        for k in range(70):
            b.feed(seqs, [p + k for p in pos], cur)
            cur = [int(t) for t in b.top(seqs)]
            assert cur == [int(t) for t in out[:, k]], k
        assert np.array_equal(a.logits(seqs), b.logits(seqs))
        st = ana_amd.Settings(0.8, 40, 0.9)
        rng = np.ascontiguousarray(np.stack([ana_amd.rng_seeded(5 + i) for i in range(n)]))
        x = a.generate(seqs, [p + 70 for p in pos], cur, 9, st, rng)
        assert x.shape == (n, 9) and (x < c.vocab).all()


def test_close_to_fp32_rings(models):
    """Four bits against fp32 rings on the same tokens: the same model, with
    the rings' rounding (a key or value is off by up to a seventh of its
    block's largest) and nothing worse."""
    c, path, _ = models["mid"]
    toks = tokens(60, 3, c.vocab)
    with ana_amd.Decoder(path, numerics=ana_amd.FAST_FP32) as a, \
            ana_amd.Decoder(path, numerics=ana_amd.FAST_FP32 | ana_amd.KV4) as b:
        for d in (a, b):
            d.feeds(0, 0, toks)
        la, lb = a.logits([0])[0], b.logits([0])[0]
        assert 1e-6 < rel(lb, la.astype(np.float64)) < 0.15
        fk, fv = rings(a, 0, c)
        k, v = rings(b, 0, c)
        for x, y in ((fk, k), (fv, v)):
            x, y = x[:60].reshape(-1, 32), y[:60].reshape(-1, 32)
            top = np.abs(x).max(-1, keepdims=True)
            assert (np.abs(x - y) <= top * (2.0 / 7.0) + 1e-6).all()


@pytest.fixture(scope="module")
def long_model(tmp_path_factory):
    """A window of 35 tiles: attention over it is cut into pieces."""
    c = cf.Config(vocab=258, ctx=1100, d=256, f=512, layers=4, heads=4, rglru=True, qk=True, sinks=True, tied=True)
    w = ckpt.init_params(c, "normal", 7, trained=True)
    path = str(tmp_path_factory.mktemp("kv4long") / "long.ftc2")
    ckpt.write(path, c, w)
    for n, rows, off in ((1, 1, False), (3, 3, False), (3, 600, True)):   # single rows; a prefill step's
        k = ops._Kv4(16, 0, 3, c.ctx, c.heads, c.hd)
        r = ops._Rows(n, rows, 1, 1, 1 if off else None)
        assert ana_amd.lib().ana_kv4_attend_ws(ctypes.byref(k), ctypes.byref(r), c.heads, 0) >= 2 * 4 * rows * c.heads * (4 + c.hd)
    return c, path, np.asarray(w, dtype=np.float64)


@pytest.mark.parametrize("mode", [ana_amd.FAST_FP32, ana_amd.BF16], ids=["fast_fp32", "bf16"])
def test_rings_in_pieces(long_model, mode):
    """Prompts over a long past (every row's log probability), then single
    tokens of one and of several sequences, past the wrap too, against the
    64-bit model over the context's own rings."""
    c, path, w = long_model
    lens = [1097, 600, 941]
    toks = [tokens(k + 8, 90 + i, c.vocab) for i, k in enumerate(lens)]
    with ana_amd.Decoder(path, max_seqs=3, numerics=mode | ana_amd.KV4) as dec:
        rows, past, fed = [Row(c, w) for _ in range(3)], [0] * 3, [0] * 3
        for cut in (260, 10 ** 6):
            # (a window scores the token after its last fed one)
            win = [toks[i][past[i]:min(lens[i], past[i] + cut) + 1] for i in range(3)]
            got = dec.score_logprobs_n([0, 1, 2], past, win, top=2)
            for i in range(3):
                ring = rings(dec, i, c)
                for t in range(len(win[i]) - 1):
                    want, kv = rows[i].feed(win[i][t], past[i] + t, ring)
                    if t % 23 == 0 or t + 2 >= len(win[i]):
                        held(c, kv, ring, past[i] + t, 1e-4 if mode == ana_amd.FAST_FP32 else 4e-2)
                    # a logit's error counts twice: in the token's own and in the sum's
                    tol = 2 * TOL[mode] * np.abs(want).max() + 1e-5
                    m = want.max()
                    lp = want[win[i][t + 1]] - m - math.log(np.exp(want - m).sum())
                    assert abs(got[i].logprob[t] - lp) <= tol, (i, past[i] + t)
                past[i] += len(win[i]) - 1
        for t in range(8):
            for seqs in ([1], [2, 0]):
                dec.feed(seqs, [past[i] for i in seqs], [toks[i][past[i]] for i in seqs])
                for i, lg in zip(seqs, dec.logits(seqs)):
                    want, _ = rows[i].feed(toks[i][past[i]], past[i], rings(dec, i, c))
                    assert rel(lg, want) <= TOL[mode], (i, past[i])
                    past[i] += 1


@pytest.mark.parametrize("n", [1, 3])
def test_loops_over_pieces(long_model, n):
    """The token loops (captured steps) over windows in pieces, past the wrap
    too: feeds and picks one at a time give the same."""
    c, path, _ = long_model
    lens = [1080, 350, 800][:n]
    toks = [tokens(k + 1, 70 + i, c.vocab) for i, k in enumerate(lens)]
    seqs = list(range(n))
    mode = ana_amd.FAST_FP32 | ana_amd.KV4
    with ana_amd.Decoder(path, max_seqs=n, numerics=mode) as a, ana_amd.Decoder(path, max_seqs=n, numerics=mode) as b:
        for d in (a, b):
            d.feeds_n(seqs, [0] * n, [t[:-1] for t in toks])
        cur = [t[-1] for t in toks]
        out = [a.generate(seqs, lens, cur, 20), None]
        out[1] = a.generate(seqs, [k + 20 for k in lens], [int(t) for t in out[0][:, -1]], 20)   # the graph again
        for k in range(40):
            b.feed(seqs, [p + k for p in lens], cur)
            cur = [int(t) for t in b.top(seqs)]
            assert cur == [int(t) for t in out[k // 20][:, k % 20]], k
        assert np.array_equal(a.logits(seqs), b.logits(seqs))
        for i in seqs:
            assert np.array_equal(a.state(i, 3), b.state(i, 3))


@pytest.mark.parametrize("n", [1, 3])
def test_loops_that_allocate_nothing(long_model, n):
    """ana_generate_noalloc over 4-bit rings in pieces: the loop's picks."""
    c, path, _ = long_model
    lens = [1085, 350, 800][:n]
    toks = [tokens(k + 1, 70 + i, c.vocab) for i, k in enumerate(lens)]
    seqs = np.arange(n, dtype=np.uint32)
    mode, u32 = ana_amd.FAST_FP32 | ana_amd.KV4, ctypes.POINTER(ctypes.c_uint32)
    with ana_amd.Decoder(path, max_seqs=n, numerics=mode) as a, ana_amd.Decoder(path, max_seqs=n, numerics=mode) as b:
        for d in (a, b):
            d.feeds_n(list(seqs), [0] * n, [t[:-1] for t in toks])
        cur = np.array([t[-1] for t in toks], dtype=np.uint32)
        want = a.generate(list(seqs), lens, [int(t) for t in cur], 25)
        out = np.zeros((n, 25), dtype=np.uint32)
        args = [x.ctypes.data_as(u32) for x in (seqs, np.array(lens, dtype=np.uint32), cur)]
        assert ana_amd.lib().ana_generate_noalloc(b.h, n, *args, 25, None, None, out.ctypes.data_as(u32)) == 0
        assert np.array_equal(out, want)


@pytest.mark.parametrize("mode", [ana_amd.FAST_FP32, ana_amd.BF16], ids=["fast_fp32", "bf16"])
def test_memory(tmp_path, mode):
    """A context with 4-bit rings holds less than one with fp32 rings by the
    rings' difference at least: nothing else of it is larger, and none of the
    fp32 rings' scratch is there."""
    c = cf.Config(vocab=258, ctx=2048, d=256, f=512, layers=4, heads=4, rglru=True, qk=True, sinks=True, tied=True)
    path, n = str(tmp_path / "long.ftc2"), 32
    ckpt.write(path, c, ckpt.init_params(c, "normal", 5))
    def free():
        a, b = ctypes.c_size_t(), ctypes.c_size_t()
        assert ana_amd.lib().hipMemGetInfo(ctypes.byref(a), ctypes.byref(b)) == 0
        return a.value

    held = []
    for m in (mode, mode | ana_amd.KV4):
        with ana_amd.Decoder(path, max_seqs=n, numerics=m):
            pass   # (what the first context of a kind leaves behind)
        before = free()
        with ana_amd.Decoder(path, max_seqs=n, numerics=m):
            held.append(before - free())
    layers = sum(c.is_softmax(i) for i in range(c.layers))
    rings = n * layers * (2 * c.ctx * c.d * 4 - c.heads * (c.ctx // 32) * 34 * c.hd)
    assert held[0] - held[1] >= rings, (held, rings)


def test_refused(models, tmp_path):
    c, path, _ = models["mid"]
    with pytest.raises(ana_amd.AnaError, match="exact mode keeps its rings in fp32"):
        ana_amd.Decoder(path, numerics=ana_amd.EXACT_FP32 | ana_amd.KV4)
    with pytest.raises(ana_amd.AnaError, match="unknown numerics"):
        ana_amd.Decoder(path, numerics=ana_amd.FAST_FP32 | ana_amd.KV4 | 0x200)
    small = str(tmp_path / "s.ftc2")
    ckpt.write(small, cf.SMALL4_V3, ckpt.init_params(cf.SMALL4_V3, "normal", 3))
    with pytest.raises(ana_amd.AnaError, match="head dimensions of 32 and 64"):
        ana_amd.Decoder(small, numerics=ana_amd.FAST_FP32 | ana_amd.KV4)


@pytest.mark.parametrize("mode", [ana_amd.FAST_FP32, ana_amd.BF16], ids=["fast_fp32", "bf16"])
def test_last_positions(models, mode):
    """The largest position of a 4-bit ring is stored and attended; calls that
    reach past it are refused before they change anything."""
    c, path, w = models["mid"]
    far = 2 ** 31 - 1
    with ana_amd.Decoder(path, max_seqs=2, numerics=mode | ana_amd.KV4) as dec:
        rows = [Row(c, w) for _ in range(2)]
        dec.feeds(0, far - 2, [5, 6])
        for t, tok in enumerate((5, 6)):
            rows[0].feed(tok, far - 2 + t, rings(dec, 0, c))
        before = [dec.state(0, i) for i in range(c.layers + 1)]
        for call in (lambda: dec.feed([0], [far + 1], [7]), lambda: dec.feed([1, 0], [0, 2 ** 32 - 1], [7, 7]),
                     lambda: dec.feeds(0, far, [7, 8]), lambda: dec.feeds_n([1, 0], [0, far - 1], [[3], [7, 8, 9]]),
                     lambda: dec.generate([0], [far], [7], 2), lambda: dec.score_n([0], [far], [[7, 8, 9]]),
                     lambda: dec.score_logprobs_n([0], [2 ** 32 - 2], [[7, 8]])):
            with pytest.raises(ana_amd.AnaError, match="below 2\\^31"):
                call()
        assert all(np.array_equal(x, dec.state(0, i)) for i, x in enumerate(before)) and not dec.state(1, 3).any()
        dec.feed([0], [far], [7])
        ring = rings(dec, 0, c)
        want, kv = rows[0].feed(7, far, ring)
        held(c, kv, ring, far % c.ctx, 1e-4 if mode == ana_amd.FAST_FP32 else 4e-2)
        assert rel(dec.logits([0])[0], want) <= TOL[mode]
    with ana_amd.Decoder(path, numerics=mode) as dec:   # (fp32 rings take every position)
        dec.feed([0], [far + 1], [7])


# ---------------------------------------------------------------- log probabilities of a context

MODES = [ana_amd.EXACT_FP32, ana_amd.FAST_FP32, ana_amd.BF16, ana_amd.FAST_FP32 | ana_amd.KV4]


def same(r, logits, tok, top):
    """A row of a Logprobs against the definition on its logits."""
    x = logits.astype(np.float64)
    w = ref.logprobs(x, tok, top)
    e = 2.0 ** -24
    ls = e * (2 * w[5] + 68)
    assert list(r.top) == list(w[3]) and (r.rank is None or int(r.rank) == w[2])
    assert (np.abs(r.top_logprob - w[4]) <= ls + 3 * e * np.abs(w[4])).all()
    assert abs(float(r.entropy) - w[1]) <= ls + e * (2 * w[5] * (w[5] + 36) + 64 * w[5] + 2 * abs(w[1]))
    if r.logprob is not None:
        assert abs(float(r.logprob) - w[0]) <= ls + 3 * e * abs(w[0])


def row(r, i):
    return ana_amd.Logprobs(None if r.logprob is None else r.logprob[i], r.entropy[i],
                            None if r.rank is None else r.rank[i], r.top[i], r.top_logprob[i])


@pytest.mark.parametrize("mode", MODES, ids=["exact", "fast_fp32", "bf16", "fast_kv4"])
def test_logprobs_after_feeds(models, mode):
    c, path, _ = models["mid"]
    n = 6
    with ana_amd.Decoder(path, max_seqs=8, numerics=mode) as dec:
        dec.feeds_n(list(range(n)), [0] * n, [tokens(4 + i, i, c.vocab) for i in range(n)])
        for seqs in ([5, 0, 3], [1], list(range(n))):
            lg = dec.logits(seqs)
            given = [int(t) for t in np.random.RandomState(9).randint(0, c.vocab, len(seqs))]
            r = dec.logprobs(seqs, given, top=7)
            for i in range(len(seqs)):
                same(row(r, i), lg[i], given[i], 7)
            r = dec.logprobs(seqs, top=64)
            assert r.logprob is None and r.rank is None
            for i in range(len(seqs)):
                same(row(r, i), lg[i], -1, 64)
            assert (dec.logprobs(seqs, dec.top(seqs)).rank == 0).all()
        # the probability that ana_stats gives, and its rival
        p, alt, palt = dec.stats([2], [17])
        r = dec.logprobs([2], [17], top=2)
        assert abs(math.exp(r.logprob[0]) - p[0]) <= 1e-5 * p[0]
        assert alt[0] in r.top[0]


@pytest.mark.parametrize("mode", MODES, ids=["exact", "fast_fp32", "bf16", "fast_kv4"])
def test_score_logprobs(models, mode):
    """Windows of all lengths: the summands of score_n, and every row's rank,
    entropy and alternatives as after feeding its tokens."""
    c, path, _ = models["mid"]
    lens = [40, 1, 2, 70, 0]
    toks = [tokens(k, 60 + i, c.vocab) for i, k in enumerate(lens)]
    with ana_amd.Decoder(path, max_seqs=5, prefill_chunk=16, numerics=mode) as dec:
        seqs, zero = list(range(5)), [0] * 5
        got = dec.score_logprobs_n(seqs, zero, toks, top=5)
        assert [g.entropy.size for g in got] == [39, 0, 1, 69, 0]
        for s in seqs:
            dec.reset(s)
        ce = dec.score_n(seqs, zero, toks)
        for g, x in zip(got, ce):
            assert np.allclose(-g.logprob, x, rtol=2e-5, atol=2e-5)
            assert g.top.shape == (x.size, 5)
        assert all(np.array_equal(a.logprob, b.logprob) for a, b in zip(got, got))
        if mode == ana_amd.EXACT_FP32:
            # its logits are those of single feeds, bit for bit
            for s in (0, 3):
                dec.reset(s)
                for t in range(lens[s] - 1):
                    dec.feed([s], [t], [toks[s][t]])
                    same(row(got[s], t), dec.logits([s])[0], toks[s][t + 1], 5)
        # no alternatives
        for s in seqs:
            dec.reset(s)
        none = dec.score_logprobs_n(seqs, zero, toks)
        assert none[0].top.shape == (39, 0) and np.array_equal(none[0].rank, got[0].rank)


@pytest.mark.parametrize("mode", MODES, ids=["exact", "fast_fp32", "bf16", "fast_kv4"])
def test_score_logprobs_repeats(models, mode):
    """The same windows scored twice, and (exact mode) one by one: the same
    numbers, bit for bit."""
    c, path, _ = models["mid"]
    lens = [40, 1, 2, 70, 0]
    toks = [tokens(k, 60 + i, c.vocab) for i, k in enumerate(lens)]
    with ana_amd.Decoder(path, max_seqs=5, prefill_chunk=16, numerics=mode) as dec:
        seqs = list(range(5))
        got = []
        for _ in range(2):
            got.append(dec.score_logprobs_n(seqs, [0] * 5, toks, top=5))
            for s in seqs:
                dec.reset(s)
        for a, b in zip(*got):
            for f in ("logprob", "entropy", "rank", "top", "top_logprob"):
                assert np.array_equal(getattr(a, f), getattr(b, f)), f
        assert got[0][0].logprob.std() > 0.1 and got[0][3].logprob.std() > 0.1
        if mode == ana_amd.EXACT_FP32:
            # (its rows' logits do not depend on what is fed beside them)
            for i in (0, 3):
                one = dec.score_logprobs_n([i], [0], [toks[i]], top=5)[0]
                for f in ("logprob", "entropy", "rank", "top", "top_logprob"):
                    assert np.array_equal(getattr(one, f), getattr(got[0][i], f)), f


def test_logprobs_refused(models):
    c, path, _ = models["mid"]
    with ana_amd.Decoder(path, max_seqs=2) as dec:
        dec.feed([0], [0], [3])
        for kw, why in ((dict(toks=[258]), "outside the vocabulary"), (dict(top=65), "alternatives")):
            with pytest.raises(ana_amd.AnaError, match=why):
                dec.logprobs([0], **kw)
        with pytest.raises(ana_amd.AnaError, match="listed twice"):
            dec.logprobs([0, 0])
        with pytest.raises(ValueError, match="one token per sequence"):
            dec.logprobs([0], [1, 2])
        with pytest.raises(ana_amd.AnaError, match="alternatives"):
            dec.score_logprobs_n([0], [0], [[3, 4]], top=70)
        with pytest.raises(ValueError, match="windows"):
            dec.score_logprobs_n([0], [0], [])
        with pytest.raises(ana_amd.AnaError, match="outside the vocabulary"):
            dec.score_logprobs_n([0], [0], [[3, 999]])
