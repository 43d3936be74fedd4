"""libana's operators on device memory, over torch tensors (include/ana.h,
"operators on device memory"): queries and keys normed and turned by their
positions, keys and values in 4 bits, attention over them, also behind a
prefix that sequences share, and of rows of logits the log probabilities and
tokens from given random numbers.

A ctypes mirror, as ana_amd itself is: every value is computed by libana.so.
torch holds the tensors, allocates outputs and workspaces, and names the
stream: the work is queued on the tensors' device's current stream, can be
captured there, and is not waited for. Tensors of other streams are the
caller's to order, as for any torch operation. The results have no gradient.

torch brings a HIP runtime of its own, which libana.so shares where torch is
loaded first. Loaded after libana.so it starts a second one, which finds no
GPU: import torch, or this module, before the first call of ana_amd.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import ANA_OK, AnaError, lib


def _runtimes() -> set:
    """The HIP runtimes that are loaded, by file."""
    with open("/proc/self/maps") as f:
        return {x.split()[-1] for x in f if "libamdhip64.so" in x}


if len(_runtimes()) > 1:
    raise ImportError("ana_amd.ops: torch was loaded after libana.so and has another HIP runtime than it "
                      f"({', '.join(sorted(_runtimes()))}): import torch before the first call of ana_amd")

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Kv4(C.Structure):
    _fields_ = [("data", C.c_void_p), ("device", C.c_int), ("seqs", C.c_uint32), ("slots", C.c_uint32),
                ("heads", C.c_uint32), ("hd", C.c_uint32)]


class _Rows(C.Structure):
    _fields_ = [("n", C.c_uint32), ("rows", C.c_uint32), ("seq", C.c_void_p), ("pos", C.c_void_p),
                ("off", C.c_void_p)]


class _Mat(C.Structure):
    _fields_ = [("p", C.c_void_p), ("row", C.c_uint64), ("head", C.c_uint64)]


class _Rope(C.Structure):
    _fields_ = [("freq", C.c_void_p), ("rot", C.c_uint32), ("near", C.c_int), ("gq", C.c_void_p), ("gk", C.c_void_p),
                ("eps", C.c_float)]


class _Draw(C.Structure):
    _fields_ = [("temperature", C.c_float), ("top_p", C.c_float), ("min_p", C.c_float), ("top_k", C.c_uint32),
                ("temperatures", C.c_void_p), ("top_ps", C.c_void_p), ("min_ps", C.c_void_p), ("top_ks", C.c_void_p)]


def _check(r: int) -> None:
    if r != ANA_OK:
        raise AnaError(r, lib().ana_error(None).decode())


# the device's current stream as a number (torch.cuda.current_stream makes an
# object of it first: 1.1 us of a call's 12 against 0.1)
_stream = torch._C._cuda_getCurrentRawStream


def _ints(t, n: int, device: torch.device, name: str):
    """A device array of whole numbers: int32, consecutive, n of them."""
    return _array(t, n, torch.int32, device, name)


def _array(t, n: int, dtype, device: torch.device, name: str):
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: a consecutive {str(dtype)[6:]} tensor of {n}, not {tuple(t.shape)} {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    return t.data_ptr()


def _mat(t: torch.Tensor, shape: tuple, dtype, device: torch.device, name: str) -> _Mat:
    if t.shape != shape or t.dtype is not dtype:
        raise ValueError(f"{name}: {shape} {dtype}, not {tuple(t.shape)} {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    a, b, c = t.stride()
    if c != 1:
        raise ValueError(f"{name}: the last axis is not consecutive")
    return _Mat(t.data_ptr(), a, b)


class KV4:
    """A cache of keys and values in 4 bits (MXFP4) for `seqs` sequences:
    rings of `slots` positions, data uint8 [seqs, heads, ceil(slots / 32),
    34 hd] in ana.h's layout. Takes the tensor it is given, as a cache that
    was moved or saved, or (KV4.empty) a new one of zeros."""

    def __init__(self, data: torch.Tensor, slots: int):
        if data.dtype != torch.uint8 or data.dim() != 4 or not data.is_contiguous():
            raise ValueError("KV4: a consecutive uint8 tensor of four axes")
        s, h, t, r = data.shape
        if slots < 1 or t != (slots + 31) // 32 or r % 34 or lib().ana_kv4_bytes(s, slots, h, r // 34) != data.numel():
            raise ValueError(f"KV4: {tuple(data.shape)} is not a cache of {slots} slots")
        self.data, self.slots = data, slots
        self.seqs, self.heads, self.hd = s, h, r // 34
        if not data.is_cuda:
            raise ValueError("KV4 is not on a GPU")
        self.device = data.device
        self._c = _Kv4(data.data_ptr(), self.device.index, s, slots, h, r // 34)
        self._p = C.addressof(self._c)

    @classmethod
    def empty(cls, seqs: int, slots: int, heads: int, hd: int, device="cuda") -> "KV4":
        if lib().ana_kv4_bytes(seqs, slots, heads, hd) == 0:
            raise ValueError(f"KV4: no cache of {seqs} sequences, {slots} slots, {heads} heads of {hd}")
        return cls(torch.zeros((seqs, heads, (slots + 31) // 32, 34 * hd), dtype=torch.uint8, device=device), slots)


def _rows(cache: KV4, rows: int, pos, seq, off) -> _Rows:
    n, dev = pos.numel(), cache.device
    return _Rows(n, rows, _ints(seq, n, dev, "seq"), _ints(pos, n, dev, "pos"), _ints(off, n + 1, dev, "off"))


def kv4_write(cache: KV4, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, seq=None, off=None) -> None:
    """Keys and values [rows, heads, hd] into the cache: sequence i (its
    place seq[i], or i) at positions pos[i] and on, its rows off[i] ..
    off[i + 1] - 1 (or row i alone). ana_kv4_write."""
    rows, dev, dtype = k.shape[0], cache.device, k.dtype
    r = _rows(cache, rows, pos, seq, off)
    shape = (rows, cache.heads, cache.hd)
    km, vm = _mat(k, shape, dtype, dev, "k"), _mat(v, shape, dtype, dev, "v")
    _check(lib().ana_kv4_write(cache._p, C.byref(r), _TYPES.get(dtype, -1), C.byref(km), C.byref(vm),
                               _stream(dev.index)))


def kv4_read(cache: KV4, pos: torch.Tensor, rows: int, seq=None, off=None, dtype=torch.float32):
    """The values that the cache holds at the rows' positions: k and v
    [rows, heads, hd]. Rows that no sequence has are left unset.
    ana_kv4_read."""
    r = _rows(cache, rows, pos, seq, off)
    h, hd, dev = cache.heads, cache.hd, cache.device
    k = torch.empty((rows, h, hd), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    km, vm = _Mat(k.data_ptr(), h * hd, hd), _Mat(v.data_ptr(), h * hd, hd)
    _check(lib().ana_kv4_read(cache._p, C.byref(r), _TYPES.get(dtype, -1), C.byref(km), C.byref(vm),
                              _stream(dev.index)))
    return k, v


def _sink(sink, hq: int, dev: torch.device):
    if sink is not None and (sink.dtype is not torch.float32 or sink.shape != (hq,) or not sink.is_contiguous()
                             or sink.device != dev):
        raise ValueError(f"sink: a consecutive float32 tensor of {hq} on {dev}")


def kv4_attend(q: torch.Tensor, cache: KV4, pos: torch.Tensor, seq=None, off=None, sink=None, scale=None, live: int = 0,
               out=None) -> torch.Tensor:
    """Softmax attention of query rows [rows, hq, hd] over the cache, whose
    own keys and values have been written; each row sees the positions up to
    its own that its ring holds. sink: float32 [hq]; scale: hd ** -0.5 unless
    given; live: the most positions a sequence holds, where the program knows
    it to be fewer than the ring's (only the split of the work depends on
    it); out: where the outputs go, q itself allowed (rows that no sequence has
    stay as they are there). ana_kv4_attend."""
    rows, hq, hd = q.shape
    dev, dtype = cache.device, q.dtype
    r = _rows(cache, rows, pos, seq, off)
    shape = (rows, hq, cache.hd)
    qm = _mat(q, shape, dtype, dev, "q")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
        om = _Mat(out.data_ptr(), hq * hd, hd)
    else:
        om = _mat(out, shape, dtype, dev, "out")
    _sink(sink, hq, dev)
    L, rp = lib(), C.byref(r)
    nb = L.ana_kv4_attend_ws(cache._p, rp, hq, live)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    _check(L.ana_kv4_attend(cache._p, rp, _TYPES.get(dtype, -1), C.byref(qm), hq,
                            cache.hd ** -0.5 if scale is None else scale,
                            None if sink is None else sink.data_ptr(), C.byref(om), live,
                            None if ws is None else ws.data_ptr(), nb, _stream(dev.index)))
    return out


def kv4_attend_shared(q: torch.Tensor, cache: KV4, pos: torch.Tensor, prefix: KV4, plen: torch.Tensor, pseq=None,
                      poff=None, seq=None, off=None, sink=None, scale=None, live: int = 0, plive: int = 0,
                      out=None) -> torch.Tensor:
    """kv4_attend where groups of rows also see a prefix that they share: group
    g has rows poff[g] .. poff[g + 1] - 1 (poff None: one group of all rows) and
    sees the first plen[g] positions of place pseq[g] (or g) of the cache
    `prefix`, besides each row's own sequence in `cache`. plen, pseq: int32
    [groups]; plive: the longest prefix, where the program knows it to be less
    than the ring's. A call of its own takes its workspace anew; captured into
    a graph, it is the graph's. ana_kv4_attend_shared."""
    rows, hq, hd = q.shape
    dev, dtype = cache.device, q.dtype
    r = _rows(cache, rows, pos, seq, off)
    if prefix.device != dev:
        raise ValueError(f"prefix is on {prefix.device}, not on {dev}")
    p = _rows(prefix, rows, plen, pseq, poff)
    shape = (rows, hq, cache.hd)
    qm = _mat(q, shape, dtype, dev, "q")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
        om = _Mat(out.data_ptr(), hq * hd, hd)
    else:
        om = _mat(out, shape, dtype, dev, "out")
    _sink(sink, hq, dev)
    L, rp, pp = lib(), C.byref(r), C.byref(p)
    nb = L.ana_kv4_attend_shared_ws(cache._p, rp, prefix._p, pp, hq, live, plive)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    _check(L.ana_kv4_attend_shared(cache._p, rp, prefix._p, pp, _TYPES.get(dtype, -1), C.byref(qm), hq,
                                   cache.hd ** -0.5 if scale is None else scale,
                                   None if sink is None else sink.data_ptr(), C.byref(om), live, plive, ws.data_ptr(), nb,
                                   _stream(dev.index)))
    return out


def qk_rope(q: torch.Tensor, k, pos: torch.Tensor, freq: torch.Tensor, off=None, gq=None, gk=None, eps: float = 1e-5,
            near: bool = False, out=None):
    """Queries [rows, hq, hd] and keys [rows, hk, hd] (k None: queries alone)
    with each head RMS-normed (gq, gk: float32 [hd], the gain being 1 + g; None:
    not) and its first 2 len(freq) values turned by position times freq, a
    float32 tensor, in pairs of one of each half or, near, of neighbours.
    Sequence i is at positions pos[i] and on, its rows off[i] .. off[i + 1] - 1
    (or row i alone). out: where they go, a pair of tensors, q and k themselves
    allowed; new ones otherwise. (q, k). ana_qk_rope."""
    if not q.is_cuda:
        raise ValueError("q is not on a GPU")
    rows, hq, hd = q.shape
    dev, dtype, n, hk = q.device, q.dtype, pos.numel(), 0 if k is None else k.shape[1]
    if freq.dim() != 1:
        raise ValueError("freq: one axis")
    r = _Rows(n, rows, None, _ints(pos, n, dev, "pos"), _ints(off, n + 1, dev, "off"))
    f = _Rope(_array(freq, freq.numel(), torch.float32, dev, "freq"), 2 * freq.numel(), near,
              _array(gq, hd, torch.float32, dev, "gq"), _array(gk, hd, torch.float32, dev, "gk"), eps)
    qm = _mat(q, (rows, hq, hd), dtype, dev, "q")
    km = None if k is None else _mat(k, (rows, hk, hd), dtype, dev, "k")
    if out is None:
        qo, ko = q.new_empty((rows, hq, hd)), None if k is None else k.new_empty((rows, hk, hd))
        qom, kom = _Mat(qo.data_ptr(), hq * hd, hd), None if k is None else _Mat(ko.data_ptr(), hk * hd, hd)
    else:
        qo, ko = out
        qom = _mat(qo, (rows, hq, hd), dtype, dev, "q's output")
        kom = None if k is None else _mat(ko, (rows, hk, hd), dtype, dev, "k's output")
    _check(lib().ana_qk_rope(dev.index, hd, C.byref(r), _TYPES.get(dtype, -1), C.byref(f), hq, C.byref(qm), C.byref(qom),
                             hk, None if km is None else C.byref(km), None if kom is None else C.byref(kom),
                             _stream(dev.index)))
    return qo, ko


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """A token of each row of logits [n, vocab] from the given random numbers u
    (float32 [n], 0 up to 1), and its log probability among what is kept:
    (tokens int32 [n], logprob float32 [n]). Each setting is a number, or a
    tensor of n for the rows' own (float32; top_k int32): temperature (0 takes
    the likeliest), top_k (0: all), top_p (1: all), min_p (0: all), in that
    order. Tokens follow each other by value, then lower index; the one at
    which the running probability passes u is drawn. ana_row_sample."""
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("sample: rows of logits, each consecutive")
    if not logits.is_cuda:
        raise ValueError("logits is not on a GPU")
    n, vocab = logits.shape
    dev = logits.device
    d = _Draw(1.0, 1.0, 0.0, 0)
    if isinstance(temperature, torch.Tensor):
        d.temperatures = _array(temperature, n, torch.float32, dev, "temperature")
    else:
        d.temperature = temperature
    if isinstance(top_k, torch.Tensor):
        d.top_ks = _array(top_k, n, torch.int32, dev, "top_k")
    elif top_k < 0:
        raise ValueError(f"top_k: {top_k}")
    else:
        d.top_k = min(top_k, vocab)
    if isinstance(top_p, torch.Tensor):
        d.top_ps = _array(top_p, n, torch.float32, dev, "top_p")
    else:
        d.top_p = top_p
    if isinstance(min_p, torch.Tensor):
        d.min_ps = _array(min_p, n, torch.float32, dev, "min_p")
    else:
        d.min_p = min_p
    up = _array(u, n, torch.float32, dev, "u")
    tok = torch.empty(n, dtype=torch.int32, device=dev)
    lp = torch.empty(n, dtype=torch.float32, device=dev)
    L = lib()
    nb = L.ana_row_sample_ws(n, vocab)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    _check(L.ana_row_sample(dev.index, _TYPES.get(logits.dtype, -1), logits.data_ptr(), logits.stride(0), n, vocab, up,
                            C.byref(d), tok.data_ptr(), lp.data_ptr(), None if ws is None else ws.data_ptr(), nb,
                            _stream(dev.index)))
    return tok, lp


def logprobs(logits: torch.Tensor, tokens=None, top: int = 0):
    """Of each row of logits [n, vocab]: the log probability and the rank of
    the given token (tokens int32 [n]; None for neither), the entropy, and
    the `top` likeliest tokens with their log probabilities, ties to the
    lower index: (logprob [n], entropy [n], rank [n], top [n, top],
    top_logprob [n, top]), float32 and int32. Rank counts the tokens before
    it, -1 for a token outside the vocabulary. ana_row_logprobs."""
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logprobs: rows of logits, each consecutive")
    if not logits.is_cuda:
        raise ValueError("logits is not on a GPU")
    n, vocab = logits.shape
    dev = logits.device
    ids = _ints(tokens, n, dev, "tokens")
    L = lib()
    nb = L.ana_row_logprobs_ws(n, vocab, top)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    # the float results and the whole numbers, an allocation each, cut into
    # the tensors that are returned
    g = tokens is not None
    f = torch.empty(n * (1 + g + top), dtype=torch.float32, device=dev)
    i = torch.empty(n * (g + top), dtype=torch.int32, device=dev)
    fp, ip = f.data_ptr(), i.data_ptr()
    _check(L.ana_row_logprobs(dev.index, _TYPES.get(logits.dtype, -1), logits.data_ptr(), logits.stride(0), n, vocab,
                              ids, top, fp + 4 * n if g else None, fp, ip if g else None, ip + 4 * n * g,
                              fp + 4 * n * (1 + g), None if ws is None else ws.data_ptr(), nb, _stream(dev.index)))
    ent, lp, tlp = f.split_with_sizes((n, n * g, n * top))
    rank, ids = i.split_with_sizes((n * g, n * top))
    return lp if g else None, ent, rank if g else None, ids.view(n, top), tlp.view(n, top)
