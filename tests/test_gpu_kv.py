"""The quantized key/value cache (comp_amd.kv) on the device, against plain 64-bit forms (tests/kv_ref.py).

Tolerances, from the roundings the kernels make.  With V the largest magnitude among the values:
  f32   queries and probabilities keep 22 bits; a score x (in log2 units, |x| <= 40 in these tests) is held to a few 2^-24 x,
        so a probability is off by at most about 1e-5 of itself: |out - exact| <= 1e-5 V.  A softcap adds cap * log2(e) * a
        few 2^-24 to x (cap 30: 1.5e-5): 3e-5 V.  lse: 1e-5 (4 + |lse|), with a softcap 2e-5 (4 + |lse|).
  f16   P and P' are rounded to f16 (2^-12 each) and so is the output (2^-12): 2^-10 V
  bf16  the output is rounded to bf16 (2^-9): 2^-8 V
Codes and scales are exact."""

import numpy as np
import pytest
import torch

from comp_amd import kv
from tests import kv_ref as R

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOL = {"f32": 1e-5, "f16": 2.0**-10, "bf16": 2.0**-8}
PAIRS = [("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q8_0", "q8_0")]


def normal(shape, seed, dtype="f32"):
    x = np.random.default_rng(seed).normal(size=shape).astype(np.float32)
    return torch.from_numpy(x).to(DTYPES[dtype]).to("cuda")


def poisoned(pages, heads, dim, kf="q4_0", vf="q4_0", page=64):
    """A cache whose unwritten places hold NaN scales: nothing may read them into a result."""
    c = kv.KVCache(pages, heads, dim, kf, vf, page)
    for t in (c.ks, c.vs):
        t.fill_(0x7E00)
    for t in (c.kq, c.vq):
        t.fill_(0xA7)
    return c


class Problem:
    """Sequences in a poisoned cache, their pages in no order; keys and values as the cache keeps them."""

    def __init__(self, lengths, counts, heads, kv_heads, dim, kf, vf, dtype, page=64, seed=0, v_scale=None, k_scale=1.0):
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 2
        order = rng.permutation(pages).astype(np.int32)
        self.tables = np.full((len(lengths), max(need + [1])), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = order[at : at + n]
            at += n
        self.cache = poisoned(pages, kv_heads, dim, kf, vf, page)
        self.lengths, self.counts, self.dtype = lengths, counts, dtype
        self.keys, self.values, self.slots = [], [], []
        for s, n in enumerate(lengths):
            k = normal((n, kv_heads, dim), seed * 1000 + 2 * s, dtype) * k_scale
            v = normal((n, kv_heads, dim), seed * 1000 + 2 * s + 1, dtype)
            if v_scale is not None:
                v = v * torch.from_numpy(v_scale(rng, n)).to(v)[:, None, None]
            j = np.arange(n)
            slots = torch.from_numpy(self.tables[s].astype(np.int64)[j // page] * page + j % page).to("cuda")
            kv.write(self.cache, k, v, slots)
            self.slots.append(slots)
            self.keys.append(R.kept(k.float().cpu().numpy(), kf))
            self.values.append(R.kept(v.float().cpu().numpy(), vf))
        self.q = normal((sum(counts), heads, dim), seed * 1000 + 999, dtype)
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)

    def dev(self, a):
        return torch.from_numpy(np.asarray(a)).to("cuda")

    def args(self, starts=True):
        return (self.cache, self.q, self.dev(self.tables), self.dev(np.asarray(self.lengths, np.int32)),
                self.dev(self.starts) if starts else None)  # fmt: skip

    def check(self, out, lse=None, *, tol=None, q=None, **opts):
        want, want_lse = R.attend((self.q if q is None else q).double().cpu().numpy(), self.keys, self.values, self.counts, **opts)
        big = max([np.abs(v).max() for v in self.values if v.size] + [1e-30])
        tol = TOL[self.dtype] * (3 if opts.get("softcap") and self.dtype == "f32" else 1) if tol is None else tol
        got = out.double().cpu().numpy()
        assert np.isfinite(got).all()
        off = np.abs(got - want).max() / big if got.size else 0.0
        assert off <= tol, f"{off:.3g} of the largest value, {tol:.3g} allowed"
        if lse is not None:
            got = lse.double().cpu().numpy()
            empty = np.isinf(want_lse)
            assert np.array_equal(np.isinf(got), empty)
            bound = (2e-5 if opts.get("softcap") else 1e-5) * (4 + np.abs(want_lse[~empty]))
            assert (np.abs(got - want_lse)[~empty] <= bound).all()


# ---- writing and reading ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", kv.HEAD_DIMS)
@pytest.mark.parametrize("kf,vf", PAIRS)
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 32), (75, 3, 32), (200, 8, 128)])
def test_write_read_exact(kf, vf, dim, dtype, tokens, heads, page):
    """Codes and scales are the oracle quantizers', and a read gives their products; other tokens keep their bytes."""
    cache = poisoned(-(-3 * tokens // page) + 1, heads, dim, kf, vf, page)
    before = [t.clone() for t in (cache.kq, cache.ks, cache.vq, cache.vs)]
    k, v = normal((tokens, heads, dim), 1, dtype), normal((tokens, heads, dim), 2, dtype)
    slots = torch.from_numpy(np.random.default_rng(3).permutation(cache.pages * page)[:tokens]).to("cuda")
    kv.write(cache, k, v, slots)
    for got, x, fmt in zip(kv.read(cache, slots), (k, v), (kf, vf)):
        assert np.array_equal(got.double().cpu().numpy(), R.kept(x.float().cpu().numpy(), fmt))
    for out_type in ("f16", "bf16"):
        for got, x, fmt in zip(kv.read(cache, slots, DTYPES[out_type]), (k, v), (kf, vf)):
            want = torch.from_numpy(R.kept(x.float().cpu().numpy(), fmt)).to(DTYPES[out_type])
            assert torch.equal(got.cpu(), want)
    rest = torch.ones(cache.pages * page, dtype=torch.bool, device="cuda")
    rest[slots] = False
    for got, was in zip(kv.read(cache, rest.nonzero()[:, 0]), "kv"):
        assert torch.isnan(got).all(), was  # the poison of every other token is whole
    # writing the same tokens again into a fresh cache, one at a time, gives the same bytes
    again = poisoned(cache.pages, heads, dim, kf, vf, page)
    for t in range(tokens):
        kv.write(again, k[t : t + 1], v[t : t + 1], slots[t : t + 1])
    for a, b, c in zip((cache.kq, cache.ks, cache.vq, cache.vs), (again.kq, again.ks, again.vq, again.vs), before):
        assert torch.equal(a, b) and not torch.equal(a, c)


@pytest.mark.parametrize("kf,vf", PAIRS)
@pytest.mark.parametrize("first,tokens,dim,page", [(0, 256, 128, 64), (5, 300, 64, 64), (31, 66, 96, 32), (2, 1000, 256, 128),
                                                   (63, 129, 128, 64)])  # fmt: skip
def test_write_runs(kf, vf, first, tokens, dim, page):
    """Consecutive slots from any place in a page on, across pages that are not neighbours, with tokens left out."""
    heads = 2
    cache = poisoned(-(-(first + tokens) // page) + 1, heads, dim, kf, vf, page)
    order = np.random.default_rng(4).permutation(cache.pages)
    j = np.arange(first, first + tokens)
    slots = order[j // page] * page + j % page
    left_out = np.arange(tokens) % 41 == 17
    given = np.where(left_out, np.where(np.arange(tokens) % 2, -1, cache.pages * page + 3), slots)
    k, v = normal((tokens, heads, dim), 5, "bf16"), normal((tokens, heads, dim), 6, "bf16")
    kv.write(cache, k, v, torch.from_numpy(given).to("cuda"))
    for got, x, fmt in zip(kv.read(cache, torch.from_numpy(slots).to("cuda")), (k, v), (kf, vf)):
        got, want = got.double().cpu().numpy(), R.kept(x.float().cpu().numpy(), fmt)
        assert np.array_equal(got[~left_out], want[~left_out]) and np.isnan(got[left_out]).all()
    for got in kv.read(cache, torch.from_numpy(given).to("cuda")):
        assert (got.cpu().numpy()[left_out] == 0).all()


@pytest.mark.parametrize("kf,vf", PAIRS)
def test_write_extreme_blocks(kf, vf):
    """Zeros, ties of both signs, the largest scales, values whose scale is no f16, NaN and infinity."""
    x = np.zeros((12, 1, 64), np.float32)
    x[1, 0, 3], x[1, 0, 7] = 2.5, -2.5
    x[2, 0, 3], x[2, 0, 7] = -2.5, 2.5
    x[3] = 65504.0
    x[4] = -1e-7
    x[5] = 3e-39
    x[6, 0, 40] = 1e4
    x[7, 0, 5] = np.nan
    x[8, 0, 37] = np.inf
    x[9] = 1e30
    x[10, 0, :32] = -np.arange(32)
    x[11] = 1.0
    dev = torch.from_numpy(x).to("cuda")
    cache = poisoned(1, 1, 64, kf, vf)
    slots = torch.arange(12, device="cuda")
    kv.write(cache, dev, dev, slots)
    for got, fmt in zip(kv.read(cache, slots), (kf, vf)):
        got = got.double().cpu().numpy()
        fine = [0, 1, 2, 3, 4, 5, 6, 10, 11]
        assert np.array_equal(got[fine], R.kept(x[fine], fmt))
        assert np.isnan(got[7, 0, :32]).all() and (got[7, 0, 32:] == 0).all()
        assert not np.isfinite(got[8, 0, 32:]).any() and (got[8, 0, :32] == 0).all()
        assert not np.isfinite(got[9]).any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_write_strided(dtype):
    """Keys and values as parts of one projection's output, at odd offsets, and with swapped axes."""
    t, h, d = 37, 3, 64
    base = normal((t, 2 * h * d + 5), 7, dtype)
    k, v = base[:, 1 : 1 + h * d].view(t, h, d), base[:, 2 + h * d : 2 + 2 * h * d].view(t, h, d)
    turned = normal((h, t, d), 8, dtype).transpose(0, 1)
    for a, b in ((k, v), (turned, k)):
        cache = poisoned(2, h, d)
        slots = torch.arange(5, 5 + t, device="cuda")
        kv.write(cache, a, b, slots)
        for got, x in zip(kv.read(cache, slots), (a, b)):
            assert np.array_equal(got.double().cpu().numpy(), R.kept(x.float().cpu().numpy(), "q4_0"))


def test_write_and_read_nothing():
    cache = poisoned(1, 2, 64)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    kv.write(cache, normal((0, 2, 64), 1), normal((0, 2, 64), 1), none)
    k, v = kv.read(cache, none)
    assert k.shape == v.shape == (0, 2, 64)


# ---- attention -------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", kv.HEAD_DIMS)
@pytest.mark.parametrize("kf,vf", PAIRS)
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (5, 1), (40, 2)])
def test_attend_one_token(kf, vf, dim, dtype, heads, kv_heads):
    lengths = [1, 33, 64, 100, 0, 257, 700]
    p = Problem(lengths, [1] * len(lengths), heads, kv_heads, dim, kf, vf, dtype, page=32 if dim == 96 else 64)
    out, lse = kv.attend(*p.args(starts=False), return_lse=True)
    p.check(out, lse)
    assert (out[4] == 0).all() and (lse[4] == -np.inf).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", kv.HEAD_DIMS)
@pytest.mark.parametrize("kf,vf", PAIRS)
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 2)])
def test_attend_several_tokens(kf, vf, dim, dtype, heads, kv_heads):
    """Ragged rows: one, a few, a whole sequence, none."""
    lengths, counts = [70, 5, 300, 33, 9], [5, 5, 40, 0, 1]
    p = Problem(lengths, counts, heads, kv_heads, dim, kf, vf, dtype, seed=1)
    out, lse = kv.attend(*p.args(), max_queries=40, return_lse=True)
    p.check(out, lse)


OPTIONS = [dict(softcap=30.0), dict(window=1), dict(window=45), dict(prefix=[40, 0, 1000, 7]), dict(slopes=True),
           dict(softcap=5.0, window=100, prefix=[90, 3, 0, 1], slopes=True), dict(scale=0.3)]  # fmt: skip


@pytest.mark.parametrize("opts", OPTIONS, ids=lambda o: "-".join(o))
@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f32", 128), ("f16", 96), ("bf16", 128), ("f16", 256)])
def test_attend_options(opts, dtype, dim):
    lengths, counts = [150, 64, 97, 20], [3, 64, 30, 20]
    p = Problem(lengths, counts, 4, 2, dim, "q4_0", "q4_0", dtype, seed=2)
    opts = dict(opts)
    if opts.get("slopes"):
        opts["slopes"] = np.array([0.5, 0.125, 0.01, 0.0], np.float32)
    dev = {k: p.dev(np.asarray(v, np.int32 if k == "prefix" else np.float32)) if k in ("prefix", "slopes") else v
           for k, v in opts.items()}  # fmt: skip
    out, lse = kv.attend(*p.args(), return_lse=True, **dev)
    p.check(out, lse, **opts)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("queries,heads,kv_heads", [(1, 8, 2), (3, 6, 2), (30, 4, 1)])
def test_attend_splits(dtype, queries, heads, kv_heads):
    """Few rows over many keys: the keys are split, whatever the length the launch is planned for."""
    p = Problem([5003, 1200], [queries, queries], heads, kv_heads, 128, "q4_0", "q4_0", dtype, seed=3)
    for bound in (None, 5003, 1, 0, 10**9):
        out, lse = kv.attend(*p.args(), max_queries=queries, max_length=bound, return_lse=True)
        p.check(out, lse)
    window = dict(window=600, softcap=20.0)
    p.check(*kv.attend(*p.args(), max_queries=queries, return_lse=True, **window), **window)


@pytest.mark.parametrize("dtype,queries,dim", [("bf16", 2100, 64), ("f16", 2100, 128), ("f32", 1090, 64), ("f16", 1090, 256)])
def test_attend_prompt(dtype, queries, dim):
    """Enough columns for waves with columns of their own."""
    p = Problem([queries + 77, 40], [queries, 1], 32, 8, dim, "q8_0", "q4_0", dtype, seed=4)
    prefix = np.array([300, 0], np.int32)
    out, lse = kv.attend(*p.args(), max_queries=queries, prefix=p.dev(prefix), return_lse=True)
    p.check(out, lse, prefix=prefix)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("kf,vf", PAIRS)
@pytest.mark.parametrize("kind", ["tiny", "large", "mixed", "rising"])
def test_attend_value_ranges(dtype, kf, vf, kind):
    """Values whose scales are near f16's ends, and scales that differ by far from token to token."""
    scales = {"tiny": lambda r, n: np.full(n, 3e-4), "large": lambda r, n: np.full(n, 3000.0),
              "mixed": lambda r, n: np.exp(r.uniform(-6, 8, n)), "rising": lambda r, n: np.exp(np.linspace(-6, 8, n))}  # fmt: skip
    p = Problem([600, 90], [2, 2], 4, 2, 64, kf, vf, dtype, seed=5, v_scale=lambda r, n: scales[kind](r, n).astype(np.float32))
    p.check(kv.attend(*p.args(), max_queries=2))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("factor", [1e-30, 1e-4, 6.0])
def test_attend_query_ranges(dtype, factor):
    """Queries of any power of two; large ones give one key all the weight."""
    p = Problem([300], [4], 2, 1, 64, "q8_0", "q8_0", dtype, seed=6)
    q = (p.q.float() * factor).to(p.q.dtype)
    scale = 0.125 if factor >= 1e-4 else 1e28
    args = list(p.args())
    args[1] = q
    p.check(kv.attend(*args, scale=scale), q=q, scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("queries", [1, 20])
def test_attend_masked_nonfinite(dtype, queries):
    """NaN and infinite keys and values in places that a row does not see do not reach it; one that it sees does."""
    n = 90
    p = Problem([n], [queries], 4, 2, 64, "q4_0", "q4_0", dtype, seed=7)
    bad = normal((3, 2, 64), 9, dtype)
    bad[0], bad[1, :, 5], bad[2] = float("nan"), float("inf"), -float("inf")
    kv.write(p.cache, bad, bad.flip(0), p.slots[0][10:13])
    want_keys = p.keys[0]
    out = kv.attend(*p.args(), window=n - queries - 13)  # the last row sees from 13 + queries on, the first from 14
    p.check(out, window=n - queries - 13)
    assert want_keys is p.keys[0]
    seen = kv.attend(*p.args())
    assert torch.isnan(seen).all()
    # a later token that is bad is not seen by the rows before it
    p = Problem([n], [20], 4, 2, 64, "q4_0", "q4_0", dtype, seed=7)
    kv.write(p.cache, bad[:1], bad[:1], p.slots[0][n - 5 : n - 4])
    out = kv.attend(*p.args())
    assert torch.isfinite(out[:15]).all() and torch.isnan(out[15:]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_bad_pages_and_lengths(dtype):
    """Pages that the cache does not have hide their keys; lengths end at the tables' end; a length below the rows."""
    p = Problem([200, 100], [1, 1], 4, 2, 64, "q4_0", "q4_0", dtype, seed=8)
    tables = p.tables.copy()
    tables[0, 1], tables[0, 2] = -5, 10**6
    args = list(p.args(starts=False))
    args[2] = p.dev(tables)
    out, lse = kv.attend(*args, return_lse=True)
    hidden = np.r_[0:64, 192:200]
    # (the positions of what is left do not matter without a bias: the row sees all of it)
    want, want_lse = R.attend(p.q.double().cpu().numpy(), [p.keys[0][hidden], p.keys[1]], [p.values[0][hidden], p.values[1]], [1, 1])
    assert np.abs(out.double().cpu().numpy() - want).max() <= TOL[dtype] * np.abs(p.values[0]).max()
    assert np.abs(lse.double().cpu().numpy() - want_lse).max() <= 1e-5 * (4 + np.abs(want_lse).max())
    args = list(p.args(starts=False))
    args[3] = p.dev(np.array([2**31 - 1, -7], np.int32))
    args[2] = p.dev(p.tables[:, :2])  # 128 keys at most
    out = kv.attend(*args)
    keys, values = [p.keys[0][:128], p.keys[1][:0]], [p.values[0][:128], p.values[1][:0]]
    want, _ = R.attend(p.q.double().cpu().numpy(), keys, values, [1, 1])
    assert np.abs(out.double().cpu().numpy() - want).max() <= TOL[dtype] * np.abs(p.values[0]).max()
    # three rows, one key: the first two rows are before the sequence's first key
    p = Problem([1], [3], 4, 2, 64, "q4_0", "q4_0", dtype, seed=8)
    out, lse = kv.attend(*p.args(), return_lse=True)
    assert (out[:2] == 0).all() and (lse[:2] == -np.inf).all()
    assert np.abs(out[2].double().cpu().numpy() - np.repeat(p.values[0][0], 2, axis=0)).max() <= TOL[dtype] * np.abs(p.values[0]).max()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_strided(dtype):
    """Queries as a part of a projection's output at odd offsets; an output with strides; table rows of a wider table."""
    p = Problem([90, 40], [7, 3], 6, 2, 64, "q4_0", "q4_0", dtype, seed=9)
    wide = normal((10, 6 * 64 + 11), 10, dtype)
    wide[:, 3 : 3 + 384] = p.q.reshape(10, -1)
    q = wide[:, 3 : 3 + 384].view(10, 6, 64)
    out = torch.full((6, 11, 65), 7.0, dtype=p.q.dtype, device="cuda")
    view = out[:, 1:, 1:].transpose(0, 1)
    tables = torch.zeros((2, 9), dtype=torch.int32, device="cuda")
    tables[:, : p.tables.shape[1]] = p.dev(p.tables)
    args = list(p.args())
    args[1], args[2] = q, tables[:, : p.tables.shape[1]]
    kv.attend_into(args[0], args[1], view, *args[2:])
    p.check(view)
    assert (out[:, 0] == 7).all() and (out[:, :, 0] == 7).all()


def test_attend_nothing():
    p = Problem([5, 9], [0, 0], 4, 2, 64, "q4_0", "q4_0", "f32")
    assert kv.attend(*p.args()).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_repeats_streams_and_graphs(dtype):
    """The same bits on every call, on another stream, and from a graph replayed between other work."""
    p = Problem([3000, 50, 700], [2, 1, 2], 8, 2, 128, "q4_0", "q4_0", dtype, seed=10)
    args = p.args()
    opts = dict(max_queries=2, return_lse=True)
    want = kv.attend(*args, **opts)
    p.check(*want)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, kv.attend(*args, **opts)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = kv.attend(*args, **opts)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    k, v = normal((5, 2, 128), 11, dtype), normal((5, 2, 128), 12, dtype)
    slots = torch.cat([s[-2:] for s in p.slots])[:5].contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.write(p.cache, k, v, slots)
        got = kv.attend(*args, **opts)
    for seed in range(3):
        k.copy_(normal((5, 2, 128), 20 + seed, dtype))
        graph.replay()
        torch.cuda.synchronize()
        again = kv.attend(*args, **opts)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, again))
        assert not torch.equal(got[0], want[0])


def test_long_cache_offsets():
    """A cache whose planes pass 2^32 bytes: tokens at both ends."""
    pages, heads, dim = 70000, 8, 128  # 64 KiB a page and plane: 4.6 GB each
    cache = kv.KVCache(pages, heads, dim, "q8_0", "q8_0")
    k, v = normal((130, heads, dim), 13, "bf16"), normal((130, heads, dim), 14, "bf16")
    table = np.array([[pages - 1, 0, pages - 2]], np.int32)
    j = np.arange(130)
    slots = torch.from_numpy(table[0].astype(np.int64)[j // 64] * 64 + j % 64).to("cuda")
    kv.write(cache, k, v, slots)
    kept = [R.kept(x.float().cpu().numpy(), "q8_0") for x in (k, v)]
    for got, want in zip(kv.read(cache, slots), kept):
        assert np.array_equal(got.double().cpu().numpy(), want)
    q = normal((1, 16, dim), 15, "f32")
    out = kv.attend(cache, q, torch.from_numpy(table).to("cuda"), torch.tensor([130], dtype=torch.int32, device="cuda"))
    want, _ = R.attend(q.double().cpu().numpy(), [kept[0]], [kept[1]], [1])
    assert np.abs(out.double().cpu().numpy() - want).max() <= TOL["f32"] * np.abs(kept[1]).max()


# ---- refusals --------------------------------------------------------------------------------------------------------


def test_refusals():
    p = Problem([50, 60], [1, 1], 4, 2, 64, "q4_0", "q4_0", "f32")
    cache, q, tables, lengths, starts = p.args()
    k = normal((3, 2, 64), 1)
    slots = torch.arange(3, device="cuda")
    bad = [
        lambda: kv.KVCache(1, 2, 80),
        lambda: kv.KVCache(1, 2, 64, "q4_0", "q8_0"),
        lambda: kv.KVCache(1, 2, 64, page=48),
        lambda: kv.KVCache(1, 2, 64, page=16),
        lambda: kv.KVCache(1, 0, 64),
        lambda: kv.KVCache(1, 2, 64, device="cpu"),
        lambda: kv.write(cache, k, k[:2], slots),
        lambda: kv.write(cache, k, k.half(), slots),
        lambda: kv.write(cache, k, k, slots.int()),
        lambda: kv.write(cache, k, k, slots[:2]),
        lambda: kv.write(cache, k, k, slots.cpu()),
        lambda: kv.write(cache, k.cpu(), k, slots),
        lambda: kv.write(cache, normal((3, 4, 64), 1), k, slots),
        lambda: kv.write(cache, normal((3, 2, 128), 1)[:, :, ::2], k, slots),
        lambda: kv.write(cache, k.double(), k.double(), slots),
        lambda: kv.read(cache, slots, torch.float64),
        lambda: kv.read(cache, slots[::2]),
        lambda: kv.read_into(cache, slots, k, k.half()),
        lambda: kv.attend(cache, q[:, :3], tables, lengths),
        lambda: kv.attend(cache, q[:1], tables, lengths),
        lambda: kv.attend(cache, q[:, :, :32], tables, lengths),
        lambda: kv.attend(cache, q.double(), tables, lengths),
        lambda: kv.attend(cache, q, tables.long(), lengths),
        lambda: kv.attend(cache, q, tables, lengths[:1]),
        lambda: kv.attend(cache, q, tables, lengths, starts[:2]),
        lambda: kv.attend(cache, q, tables, lengths, starts, max_queries=3),
        lambda: kv.attend(cache, q, tables, lengths, softcap=-1.0),
        lambda: kv.attend(cache, q, tables, lengths, softcap=float("nan")),
        lambda: kv.attend(cache, q, tables, lengths, scale=float("inf")),
        lambda: kv.attend(cache, q, tables, lengths, window=-1),
        lambda: kv.attend(cache, q, tables, lengths, prefix=lengths.long()),
        lambda: kv.attend(cache, q, tables, lengths, slopes=torch.zeros(3, device="cuda")),
        lambda: kv.attend_into(cache, q, torch.empty((2, 4, 64), dtype=torch.float16, device="cuda"), tables, lengths),
        lambda: kv.attend_into(cache, q, torch.empty_like(q), tables, lengths, lse=torch.empty((2, 3), device="cuda")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(kv._abi.KompArgumentError):
            call()
            pytest.fail(f"refusal {i} did not come")
    with pytest.raises(TypeError):
        kv.write(None, k, k, slots)
    with pytest.raises(TypeError):
        kv.attend(cache, np.zeros((2, 4, 64)), tables, lengths)


# ---- many columns, and what only their kernel does -------------------------------------------------------------------


@pytest.mark.parametrize("dim", kv.HEAD_DIMS)
@pytest.mark.parametrize("kf,vf", PAIRS)
@pytest.mark.parametrize("opts", [dict(), dict(softcap=20.0, window=130), dict(slopes=True, prefix=[150, 20])], ids=["plain", "cap", "bias"])
def test_attend_many_bf16_without_lse(kf, vf, dim, opts):
    """bf16 without the sums' logarithms scales the keys in the operands too."""
    p = Problem([333, 75], [90, 60], 4, 2, dim, kf, vf, "bf16", seed=12)
    opts = dict(opts)
    if opts.get("slopes"):
        opts["slopes"] = np.array([0.5, 0.125, 0.01, 0.0], np.float32)
    dev = {k: p.dev(np.asarray(v, np.int32 if k == "prefix" else np.float32)) if k in ("prefix", "slopes") else v
           for k, v in opts.items()}  # fmt: skip
    p.check(kv.attend(*p.args(), max_queries=90, **dev), **opts)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kf,vf", PAIRS)
@pytest.mark.parametrize("kind", ["tiny", "large", "mixed", "rising", "keys"])
def test_attend_many_value_ranges(dtype, kf, vf, kind):
    """Scales near f16's ends, far apart from token to token, and large and tiny keys, for many columns."""
    scales = {"tiny": lambda r, n: np.full(n, 3e-4), "large": lambda r, n: np.full(n, 3000.0),
              "mixed": lambda r, n: np.exp(r.uniform(-6, 8, n)), "rising": lambda r, n: np.exp(np.linspace(-6, 8, n)),
              "keys": lambda r, n: np.ones(n)}  # fmt: skip
    p = Problem([300, 90], [70, 70], 4, 2, 64, kf, vf, dtype, seed=13, v_scale=lambda r, n: scales[kind](r, n).astype(np.float32),
                k_scale=2000.0 if kind == "keys" else 1.0)  # fmt: skip
    scale = 0.125 / 2000 if kind == "keys" else 0.125
    p.check(kv.attend(*p.args(), max_queries=70, scale=scale), scale=scale)
    p.check(kv.attend(*p.args(), max_queries=70, scale=-scale), scale=-scale)
    p.check(kv.attend(*p.args(), max_queries=70, scale=0.0), scale=0.0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attend_many_nonfinite(dtype, dim):
    """A token without numbers reaches the rows that see it, in the channels of its block, and no others."""
    n, rows, at = 200, 80, 150  # the rows are positions 120 .. 199
    p = Problem([n], [rows], 4, 2, dim, "q8_0", "q4_0", dtype, seed=14)
    want = kv.attend(*p.args(), max_queries=rows)
    bad_k, bad_v = normal((1, 2, dim), 15, dtype), normal((1, 2, dim), 16, dtype)
    bad_v[0, :, 40] = float("nan")
    kv.write(p.cache, bad_k, bad_v, p.slots[0][at : at + 1])
    out = kv.attend(*p.args(), max_queries=rows)
    sees = at - (n - rows)
    assert torch.equal(out[:sees], want[:sees])
    assert torch.isnan(out[sees:, :, 32:64]).all()
    assert torch.isfinite(out[sees:, :, :32]).all() and torch.isfinite(out[sees:, :, 64:]).all()
    bad_k[0, :, 3] = float("nan")
    kv.write(p.cache, bad_k, bad_v, p.slots[0][at : at + 1])
    out = kv.attend(*p.args(), max_queries=rows)
    assert torch.equal(out[:sees], want[:sees]) and torch.isnan(out[sees:]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [96, 128])
def test_attend_many_splits_and_pages(dtype, dim):
    """Splits of the keys, pages that the cache does not have, rows of no sequence, pages of 32 and 256 tokens."""
    for page in (32, 256):
        p = Problem([3000, 700], [60, 50], 4, 2, dim, "q4_0", "q4_0", dtype, page=page, seed=15)
        for lse in (True, False):
            got = kv.attend(*p.args(), max_queries=60, return_lse=lse)
            p.check(*(got if lse else (got,)))
    tables = p.tables.copy()
    tables[0, 1], tables[0, 3] = -1, 2**31 - 1  # of 256 tokens
    args = list(p.args())
    args[2] = p.dev(tables)
    out = kv.attend(*args, max_queries=60, prefix=p.dev(np.array([3000, 700], np.int32)))
    left = np.r_[0:256, 512:768, 1024:3000]
    prefix = [10**6, 10**6]
    want, _ = R.attend(p.q.double().cpu().numpy(), [p.keys[0][left], p.keys[1]], [p.values[0][left], p.values[1]], p.counts, prefix=prefix)
    assert np.abs(out.double().cpu().numpy() - want).max() <= TOL[dtype] * np.abs(p.values[0]).max()
    # rows before and after those that `starts` gives to the sequences
    more = torch.cat([p.q[:3], p.q, p.q[:5]])
    args = list(p.args())
    args[1], args[4] = more, p.dev(p.starts + 3)
    p.check(kv.attend(*args, max_queries=60)[3:-5])
