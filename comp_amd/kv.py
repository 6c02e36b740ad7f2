"""Quantized key/value cache: writing tokens into it, reading them back, and attention over it.

The part of a decode step beside the GEMVs of comp_amd.host: the projections give new queries, keys and values, `write` puts
the keys and values into the cache as ggml Q4_0 or Q8_0 blocks, and `attend` computes the softmax attention of the queries
over all that the cache holds for their sequences, for one new token a sequence, for several, or for whole prompts.

    cache = KVCache(pages=1024, kv_heads=8, head_dim=128)          # Q4_0, 64 tokens a page
    write(cache, k, v, slots)                                       # k, v [T][8][128]; slots int64 [T]
    out = attend(cache, q, tables, lengths)                         # q [B][heads][128]; one new token a sequence

A page holds `page` consecutive tokens of one sequence; which pages, and in which order, a sequence has stands in its row of
`tables` (int32 page numbers).  Key j of a sequence lies at slot tables[s][j // page] * page + j % page.

As in comp_amd.host, tensors live on a HIP device, calls run on the current torch stream without synchronising, wrong
arguments raise KompArgumentError before anything is launched, and the *_into forms allocate no result.  The values of
`slots`, `tables`, `lengths` and `starts` are on the device, where the kernels check them: a slot outside the cache is left
out (read: zeros), a page outside it hides its keys.  No reference counterpart.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _abi
from .host import _current_device, _need, _raw_stream

_Tensor, _I64, _I32 = torch.Tensor, torch.int64, torch.int32

HEAD_DIMS = (64, 96, 128, 256)
FORMATS = {"q4_0": 0, "q8_0": 2}  # the weight formats' numbers; 16 and 32 code bytes a block of 32
PAIRS = (("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q8_0", "q8_0"))  # (keys, values)
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_CODE_BYTES = {"q4_0": 16, "q8_0": 32}
_BAD = _abi.KompArgumentError


class KVCache:
    """The planes of a quantized cache: `pages` pages of `page` tokens (a power of two, 32 at least) for kv_heads heads of
    head_dim channels (64, 96, 128 or 256).

    k_format and v_format: "q4_0" (18 bytes a block of 32) or "q8_0" (34); values in q8_0 need keys in q8_0.  A new cache
    holds zeros.  The order of the bytes inside a page is the library's own (include/komp_abi.h): write() and read() go
    through it."""

    def __init__(self, pages, kv_heads, head_dim, k_format="q4_0", v_format="q4_0", page=64, device="cuda"):
        if (k_format, v_format) not in PAIRS:
            raise _BAD(f"KVCache: formats {k_format!r}, {v_format!r}; the pairs are {PAIRS}")
        if head_dim not in HEAD_DIMS:
            raise _BAD(f"KVCache: head_dim={head_dim}; one of {HEAD_DIMS}")
        if page < 32 or page > 65536 or page & (page - 1):
            raise _BAD(f"KVCache: page={page} must be a power of two from 32 to 65536")
        if not 1 <= kv_heads <= 65535 or not 0 <= pages < 1 << 31:
            raise _BAD(f"KVCache: kv_heads={kv_heads} (1 to 65535), pages={pages} (0 to 2^31 - 1)")
        if torch.device(device).type != "cuda":
            raise _BAD(f"KVCache: {device}: the cache lives on a HIP device")
        self.pages, self.kv_heads, self.head_dim, self.page = pages, kv_heads, head_dim, page
        self.k_format, self.v_format = k_format, v_format
        blocks = page * (head_dim // 32)
        planes = []
        for fmt in (k_format, v_format):
            planes.append(torch.zeros((pages, kv_heads, blocks * _CODE_BYTES[fmt]), dtype=torch.uint8, device=device))
            planes.append(torch.zeros((pages, kv_heads, blocks), dtype=torch.int16, device=device))
        self.kq, self.ks, self.vq, self.vs = planes
        self._struct = _abi.KvCacheStruct(*(t.data_ptr() for t in planes), pages, kv_heads, head_dim, page,
                                          FORMATS[k_format], FORMATS[v_format])  # fmt: skip
        self._ref = ctypes.addressof(self._struct)
        self._device = self.kq.get_device()
        self._scale = 1.0 / math.sqrt(head_dim)
        self._work = {}  # workspace bytes of attention calls by their sizes

    @property
    def device(self):
        return self.kq.device

    def nbytes(self):
        """Bytes of the four planes."""
        return sum(t.numel() * t.element_size() for t in (self.kq, self.ks, self.vq, self.vs))


def _launch(name, cache, *args):
    """Call a launching ABI entry on the cache's device, with that device's current stream as its last argument."""
    fn = getattr(_abi._lib or _abi.lib(), name)
    dev = cache._device
    if dev == _current_device():
        st = fn(cache._ref, *args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(cache._ref, *args, _raw_stream(dev))
    if st:
        _abi.check(st, name)


def _need_cache(cache):
    if not isinstance(cache, KVCache):
        raise TypeError(f"cache must be a KVCache, got {type(cache).__name__}")


def _need_rows(t, name, cache, heads, what):
    """A [T][heads][head_dim] tensor of a float type whose rows are contiguous, on the cache's device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in TYPES:
        raise _BAD(f"{name} must be f32, f16 or bf16, got {t.dtype}")
    if t.dim() != 3 or (heads is not None and t.shape[1] != heads) or t.shape[2] != cache.head_dim:
        raise _BAD(f"{name} must be [{what}][{'heads' if heads is None else heads}][{cache.head_dim}], got {tuple(t.shape)}")
    if t.get_device() != cache._device:
        raise _BAD(f"{name} is on {t.device}, the cache on {cache.device}")
    if t.numel() and t.stride(2) != 1:
        raise _BAD(f"{name}: the channels of a row must be contiguous (stride(2) == 1)")


def _need_ints(t, name, cache, dtype, shape):
    """A contiguous integer (or f32) tensor of this shape on the cache's device."""
    _need(t, name, dtype, len(shape))
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise _BAD(f"{name} must be a contiguous {list(shape)} tensor, got {tuple(t.shape)}")
    if t.get_device() != cache._device:
        raise _BAD(f"{name} is on {t.device}, the cache on {cache.device}")


# An eager call is mostly host time, so each checks its arguments in one chain of cheap attribute reads first, which implies
# the full checks; those run, and name the fault, when any of it fails.
def _rows_fit(t, cache, heads):
    """True for a tensor that passes _need_rows(t, ..., cache, heads, ...)."""
    if isinstance(t, _Tensor) and t.is_cuda and t.dtype in TYPES and t.dim() == 3:
        shape = t.shape
        return (shape[1] == heads and shape[2] == cache.head_dim and t.stride(2) == 1 and t.get_device() == cache._device)  # fmt: skip
    return False


def _ints_fit(t, cache, dtype, n):
    """True for a contiguous one-dimensional tensor of n elements of this type on the cache's device."""
    return (isinstance(t, _Tensor) and t.is_cuda and t.dtype is dtype and t.dim() == 1 and t.shape[0] == n
            and t.is_contiguous() and t.get_device() == cache._device)  # fmt: skip


def write(cache, k, v, slots):
    """Quantize k, v [T][kv_heads][head_dim] (f32, f16 or bf16; rows contiguous, any strides between them) into the cache's
    slots int64 [T].  A negative slot leaves its token out; slots of one call are to differ.  Returns the cache."""
    if not (type(cache) is KVCache and _rows_fit(k, cache, cache.kv_heads) and _rows_fit(v, cache, cache.kv_heads)
            and v.shape[0] == k.shape[0] and v.dtype is k.dtype and _ints_fit(slots, cache, _I64, k.shape[0])):  # fmt: skip
        _need_cache(cache)
        _need_rows(k, "k", cache, cache.kv_heads, "T")
        _need_rows(v, "v", cache, cache.kv_heads, "T")
        if v.shape[0] != k.shape[0] or v.dtype is not k.dtype:
            raise _BAD(f"k and v must have as many tokens and one type: {tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype}")
        _need_ints(slots, "slots", cache, torch.int64, (k.shape[0],))
    ks, vs = k.stride(), v.stride()
    _launch("komp_kv_write", cache, k.data_ptr(), v.data_ptr(), TYPES[k.dtype], slots.data_ptr(), k.shape[0], ks[0], ks[1],
            vs[0], vs[1])  # fmt: skip
    return cache


def _need_slots(slots, cache):
    n = slots.shape[0] if isinstance(slots, torch.Tensor) and slots.dim() else 0
    if not (type(cache) is KVCache and _ints_fit(slots, cache, _I64, n)):
        _need_cache(cache)
        _need_ints(slots, "slots", cache, torch.int64, (n,))
    return n


def read_into(cache, slots, k, v):
    """read() into preallocated contiguous k, v [T][kv_heads][head_dim] of one type."""
    n = _need_slots(slots, cache)
    for t, name in ((k, "k"), (v, "v")):
        _need_rows(t, name, cache, cache.kv_heads, "T")
        if t.shape[0] != n or not t.is_contiguous() or t.dtype is not k.dtype:
            raise _BAD(f"{name} must be contiguous [{n}][{cache.kv_heads}][{cache.head_dim}], k and v of one type")
    _launch("komp_kv_read", cache, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), TYPES[k.dtype])


def read(cache, slots, dtype=torch.float32):
    """The keys and values that the cache holds at slots int64 [T], as (k, v) [T][kv_heads][head_dim] of dtype: each the
    product of its code and its block's scale, rounded once.  A slot outside the cache gives zeros."""
    n = _need_slots(slots, cache)
    if dtype not in TYPES:
        raise _BAD(f"dtype must be f32, f16 or bf16, got {dtype}")
    shape = (n, cache.kv_heads, cache.head_dim)
    k, v = cache.kq.new_empty(shape, dtype=dtype), cache.kq.new_empty(shape, dtype=dtype)
    _launch("komp_kv_read", cache, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), TYPES[dtype])
    return k, v


def _check_attend(cache, q, out, tables, lengths, starts, max_queries, prefix, slopes, lse):
    """Every check of an attention call's tensors, with its message."""
    _need_cache(cache)
    _need_rows(q, "q", cache, None, "T")
    t, heads = q.shape[0], q.shape[1]
    if heads < 1 or heads % cache.kv_heads:
        raise _BAD(f"q has {heads} heads, which must be a multiple of the cache's {cache.kv_heads}")
    if out is not None:
        _need_rows(out, "out", cache, heads, t)
        if out.shape[0] != t or out.dtype is not q.dtype:
            raise _BAD(f"out must be {list(q.shape)} {q.dtype}, got {list(out.shape)} {out.dtype}")
    _need(tables, "tables", torch.int32, 2)
    batch = tables.shape[0]
    if tables.get_device() != cache._device or (tables.numel() and tables.stride(1) != 1):
        raise _BAD("tables must be [sequences][pages] on the cache's device with contiguous rows")
    _need_ints(lengths, "lengths", cache, torch.int32, (batch,))
    if starts is None:
        if t != batch:
            raise _BAD(f"q has {t} rows for {batch} sequences: give starts, or one row a sequence")
    else:
        _need_ints(starts, "starts", cache, torch.int32, (batch + 1,))
        if max_queries is not None and not 0 <= max_queries <= t:
            raise _BAD(f"max_queries={max_queries} must be from 0 to q's {t} rows")
    if prefix is not None:
        _need_ints(prefix, "prefix", cache, torch.int32, (batch,))
    if slopes is not None:
        _need_ints(slopes, "slopes", cache, torch.float32, (heads,))
    if lse is not None:
        _need_ints(lse, "lse", cache, torch.float32, (t, heads))


def _attend_fits(cache, q, tables, lengths, starts, max_queries, prefix, slopes):
    """True for tensors that pass _check_attend (out and lse aside)."""
    if not (type(cache) is KVCache and isinstance(q, _Tensor) and q.dim() == 3 and isinstance(tables, _Tensor)
            and tables.is_cuda and tables.dtype is _I32 and tables.dim() == 2):  # fmt: skip
        return False
    t, heads = q.shape[0], q.shape[1]
    batch = tables.shape[0]
    return (heads > 0 and heads % cache.kv_heads == 0 and _rows_fit(q, cache, heads) and tables.stride(1) == 1
            and tables.get_device() == cache._device and _ints_fit(lengths, cache, _I32, batch)
            and (t == batch if starts is None else _ints_fit(starts, cache, _I32, batch + 1)
                 and (max_queries is None or 0 <= max_queries <= t))
            and (prefix is None or _ints_fit(prefix, cache, _I32, batch))
            and (slopes is None or _ints_fit(slopes, cache, torch.float32, heads)))  # fmt: skip


def _attend(cache, q, out, tables, lengths, starts, max_queries, max_length, scale, softcap, window, prefix, slopes, lse):
    """Launch an attention call of checked tensors."""
    t, heads = q.shape[0], q.shape[1]
    batch, cols = tables.shape
    if starts is None:
        max_queries = 1 if t else 0
    elif max_queries is None:
        max_queries = t
    if scale is None:
        scale = cache._scale
    elif not abs(scale) <= 2e38:
        raise _BAD(f"scale={scale}: 2e38 at most in magnitude")
    most = cols * cache.page
    max_length = most if max_length is None else max(0, min(int(max_length), most))
    key = (TYPES[q.dtype], t, batch, heads, max_queries, max_length)
    need = cache._work.get(key)
    if need is None:
        v = ctypes.c_int64()
        _abi.call("komp_kv_attend_workspace", cache._ref, *key, ctypes.byref(v))
        if len(cache._work) >= 4096:
            cache._work.clear()
        need = cache._work[key] = v.value
    work = None
    if need:  # kept until the call is on the stream; torch hands the memory to later work of this stream only
        work = cache.kq.new_empty(need)
    qs, os, ts = q.stride(), out.stride(), tables.stride(0)
    _launch("komp_kv_attend", cache, q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), key[0],
            tables.data_ptr(), lengths.data_ptr(), None if starts is None else starts.data_ptr(),
            None if prefix is None else prefix.data_ptr(), None if slopes is None else slopes.data_ptr(), t, batch, heads,
            qs[0], qs[1], os[0], os[1], ts, cols, max_queries, max_length, scale, softcap, window,
            None if work is None else work.data_ptr(), need)  # fmt: skip


def attend_into(cache, q, out, tables, lengths, starts=None, *, max_queries=None, max_length=None, scale=None, softcap=0.0,
                window=0, prefix=None, slopes=None, lse=None):  # fmt: skip
    """attend() into a preallocated out [T][heads][head_dim] of q's type (rows contiguous, any strides between them) and,
    when given, lse f32 [T][heads].  (A call over few rows and many keys still takes a workspace from torch.)"""
    _check_attend(cache, q, out, tables, lengths, starts, max_queries, prefix, slopes, lse)
    _attend(cache, q, out, tables, lengths, starts, max_queries, max_length, scale, softcap, window, prefix, slopes, lse)


def attend(cache, q, tables, lengths, starts=None, *, max_queries=None, max_length=None, scale=None, softcap=0.0, window=0,
           prefix=None, slopes=None, return_lse=False):  # fmt: skip
    """Softmax attention of q [T][heads][head_dim] (f32, f16 or bf16) over the cache: out [T][heads][head_dim] of q's type
    (and with return_lse also the f32 [T][heads] logarithms of the sums of exp(score)).

    Sequence s has lengths[s] keys (int32 [B]; the new tokens' own, already written, among them) in the pages tables[s]
    (int32 [B][pages]); its query rows are starts[s] .. starts[s + 1] - 1 (int32 [B + 1]; None: row s alone), the last ones of
    its positions.  heads is a multiple of the cache's kv_heads, whose head h serves the query heads h * g .. h * g + g - 1.

    A row at position i has score_j = scale * q . k_j (scale: 1 / sqrt(head_dim) by default), capped with softcap > 0 to
    softcap * tanh(score / softcap), less slopes[head] * |i - j| with slopes f32 [heads].  It sees the keys j < length with
    j <= i or j < prefix[s] (int32 [B]), of the past only the nearest `window` ones (itself among them) with window > 0.
    A row that sees nothing gives zeros and an lse of -inf.

    max_queries: the most rows of one sequence (T by default); the results' places of rows past it hold anything (with 0 nothing
    is computed at all).  Give it where starts is given and sequences have a few rows each: one plan serves all sequences, and
    T rows for each of them plan for a prompt.  max_length: an upper bound of the lengths that the launch is planned for (the
    tables' width by default); any value gives the right result.

    Scores, sums and accumulators are f32.  f32 queries keep 22 bits of queries and probabilities; f16 and bf16 queries hold the
    probabilities in f16 (2^-12), bf16 ones of many rows also values times their scales, and keys too where the logarithms are
    not asked for (the results' last bits differ with return_lse)."""
    if not _attend_fits(cache, q, tables, lengths, starts, max_queries, prefix, slopes):
        _check_attend(cache, q, None, tables, lengths, starts, max_queries, prefix, slopes, None)
    out = cache.kq.new_empty(q.shape, dtype=q.dtype)
    lse = cache.kq.new_empty(q.shape[:2], dtype=torch.float32) if return_lse else None
    _attend(cache, q, out, tables, lengths, starts, max_queries, max_length, scale, softcap, window, prefix, slopes, lse)
    return (out, lse) if return_lse else out
