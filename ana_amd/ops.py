"""libana's operators on device memory, over torch tensors (include/ana.h,
"operators on device memory"): keys and values in 4 bits, attention over
them, and the log probabilities of rows of logits.

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


def _check(r: int) -> None:
    if r != ANA_OK:
        raise AnaError(r, lib().ana_error(None).decode())


# the device's current stream as a number (torch.cuda.current_stream makes an
# object of it first: 1.1 us of a call's 12 against 0.1)
_stream = torch._C._cuda_getCurrentRawStream


def _ints(t, n: int, device: torch.device, name: str):
    """A device array of whole numbers: int32, consecutive, n of them."""
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: a consecutive int32 tensor of {n}, not {tuple(t.shape)} {t.dtype}")
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
    if sink is not None and (sink.dtype is not torch.float32 or sink.shape != (hq,) or not sink.is_contiguous()
                             or sink.device != dev):
        raise ValueError(f"sink: a consecutive float32 tensor of {hq} on {dev}")
    L, rp = lib(), C.byref(r)
    nb = L.ana_kv4_attend_ws(cache._p, rp, hq, live)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    _check(L.ana_kv4_attend(cache._p, rp, _TYPES.get(dtype, -1), C.byref(qm), hq,
                            cache.hd ** -0.5 if scale is None else scale,
                            None if sink is None else sink.data_ptr(), C.byref(om), live,
                            None if ws is None else ws.data_ptr(), nb, _stream(dev.index)))
    return out


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
