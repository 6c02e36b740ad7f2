"""Writing and reading so many tokens that the kernels of 32-token tiles run (tokens * heads past 16384), against the same
tokens a few at a time, whose kernel tests/test_gpu_kv.py holds to the oracle's quantizers, and against those directly.

Every comparison is exact: codes, scales, the bytes of other tokens, and the values read."""

import numpy as np
import pytest
import torch

from comp_amd import kv
from tests import kv_ref as R
from tests.test_gpu_kv import DTYPES, PAIRS, normal, poisoned

pytestmark = pytest.mark.gpu

HEADS = 64
FEW = 200  # tokens of a call of 64 heads that stays with the few-token kernels


def run_slots(first, tokens, pages, page, seed=4):
    """Consecutive tokens from place `first` of their first page on, over pages in no order."""
    order = np.random.default_rng(seed).permutation(pages)
    j = np.arange(first, first + tokens)
    return order[j // page] * page + j % page


def patterns(tokens, pages, page):
    """name -> slots of a call, none twice (the invalid ones aside)."""
    rng, room = np.random.default_rng(6), pages * page
    got = {"from a page's start": run_slots(0, tokens, pages, page)}
    odd = run_slots(13, tokens, pages, page)
    got["from inside a tile"] = odd
    left = odd.copy()
    left[np.arange(tokens) % 41 == 17] = -1
    left[np.arange(tokens) % 53 == 40] = room + 3
    got["tokens left out"] = left
    bad = run_slots(0, tokens, pages, page)
    bad[0], bad[1], bad[5], bad[-1] = -(2**62) - 1, room, -(2**63), 2**62
    got["no slot at the ends"] = bad
    got["first token out"] = np.concatenate([[-7], odd[1:]])
    got["backwards"] = odd[::-1].copy()
    got["no order"] = rng.permutation(room)[:tokens]
    few = [run_slots(5, (tokens + 4 - s) // 5, pages // 5, page, seed=s) + (pages // 5) * page * s for s in range(5)]
    turns = np.empty(tokens, np.int64)  # five sequences in turn: up to five tiles among 32 tokens
    for s in range(5):
        turns[s::5] = few[s]
    got["sequences in turn"] = turns
    got["none"] = np.full(tokens, -1)
    return {k: np.ascontiguousarray(v, np.int64) for k, v in got.items()}


def same(a, b):
    """Equal, a NaN being equal to a NaN."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", kv.HEAD_DIMS)
@pytest.mark.parametrize("kf,vf", PAIRS)
def test_tiles_write(kf, vf, dim, dtype):
    """The planes are those of the tokens written a few at a time, byte for byte; read back they are the oracle's."""
    tokens, pages, page = 517, 45, 32 if dim == 96 else 64
    k, v = normal((tokens, HEADS, dim), 1, dtype), normal((tokens, HEADS, dim), 2, dtype)
    k[7], v[9, :, 5], k[11, :, 3] = 0, float("nan"), 60000.0
    for name, slots in patterns(tokens, pages, page).items():
        print(name, flush=True)
        there = (slots >= 0) & (slots < pages * page)
        on = torch.from_numpy(slots).to("cuda")
        many, few = (poisoned(pages, HEADS, dim, kf, vf, page) for _ in range(2))
        kv.write(many, k, v, on)
        for t in range(0, tokens, FEW):
            kv.write(few, k[t : t + FEW], v[t : t + FEW], on[t : t + FEW])
        for plane in ("kq", "ks", "vq", "vs"):
            assert torch.equal(getattr(many, plane), getattr(few, plane)), (name, plane)
        if there.any():
            heads, some = slice(60, 63), there.nonzero()[0][::7]
            some = some[(some != 7) & (some != 9) & (some != 11)]
            got = kv.read(many, on[torch.from_numpy(some).to("cuda")])
            for g, x, fmt in zip(got, (k, v), (kf, vf)):
                want = R.kept(x[torch.from_numpy(some).to("cuda"), heads].float().cpu().numpy(), fmt)
                assert np.array_equal(g[:, heads].double().cpu().numpy(), want), name


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", kv.HEAD_DIMS)
@pytest.mark.parametrize("kf,vf", PAIRS)
def test_tiles_read(kf, vf, dim, dtype):
    """The same values as read a few at a time; slots outside the cache give zeros, repeated slots what they hold."""
    tokens, pages, page = 517, 45, 32 if dim == 96 else 64
    cache = poisoned(pages, HEADS, dim, kf, vf, page)
    held = torch.from_numpy(np.random.default_rng(8).permutation(pages * page)[:1000]).to("cuda")
    kv.write(cache, normal((1000, HEADS, dim), 3), normal((1000, HEADS, dim), 4), held)
    ways = patterns(tokens, pages, page)
    twice = ways["from inside a tile"].copy()
    twice[40:60] = twice[39]  # within a tile, and across the workgroups' boundary
    twice[300:] = twice[100 : 100 + tokens - 300]
    ways["some again"] = twice
    ways["one slot"] = np.full(tokens, twice[0])
    for name, slots in ways.items():
        print(name, flush=True)
        on = torch.from_numpy(slots).to("cuda")
        got = kv.read(cache, on, DTYPES[dtype])
        parts = [kv.read(cache, on[t : t + FEW], DTYPES[dtype]) for t in range(0, tokens, FEW)]
        for g, p in zip(got, zip(*parts)):
            assert same(g, torch.cat(p)), name
            out = torch.from_numpy(~((slots >= 0) & (slots < pages * page))).to("cuda")
            assert (g[out] == 0).all(), name


@pytest.mark.parametrize("tokens", [255, 256, 257, 287, 288, 320])
@pytest.mark.parametrize("first", [0, 1, 31])
def test_tiles_around_the_threshold(tokens, first):
    """Sizes on both sides of where the tile kernels begin, into preallocated results with strided inputs."""
    cache, dim, page = poisoned(12, HEADS, 64), 64, 64
    base = normal((tokens, 2 * HEADS * dim + 5), 7, "f32")
    k = base[:, 1 : 1 + HEADS * dim].view(tokens, HEADS, dim)
    v = base[:, 2 + HEADS * dim : 2 + 2 * HEADS * dim].view(tokens, HEADS, dim)
    on = torch.from_numpy(run_slots(first, tokens, 12, page)).to("cuda")
    kv.write(cache, k, v, on)
    got = torch.empty((2, tokens, HEADS, dim), device="cuda")
    kv.read_into(cache, on, got[0], got[1])
    for g, x in zip(got, (k, v)):
        assert np.array_equal(g[:, :5].double().cpu().numpy(), R.kept(x[:, :5].cpu().numpy(), "q4_0"))
    rest = torch.ones(12 * page, dtype=torch.bool, device="cuda")
    rest[on] = False
    for g in kv.read(cache, rest.nonzero()[:, 0]):
        assert torch.isnan(g).all()


def test_tiles_graph():
    """A write and a read of many tokens in a graph, replayed between eager work, against the eager calls."""
    tokens, pages, page, dim = 517, 45, 64, 128
    on = torch.from_numpy(patterns(tokens, pages, page)["tokens left out"]).to("cuda")
    k, v = normal((tokens, HEADS, dim), 1, "bf16"), normal((tokens, HEADS, dim), 2, "bf16")
    cache, other = (kv.KVCache(pages, HEADS, dim, "q8_0", "q4_0", page) for _ in range(2))
    kv.write(cache, k, v, on)
    kv.read(cache, on)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.write(cache, k, v, on)
        got = kv.read(cache, on)
    for seed in range(3):
        k.copy_(normal((tokens, HEADS, dim), 20 + seed, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        kv.write(other, k, v, on)
        want = kv.read(other, on)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
