"""Large hidden tokens (tests/test_gpu_kv_hidden.py) where the keys are split over workgroups, beside tokens without numbers,
and in replayed graphs."""

import numpy as np
import pytest
import torch

from comp_amd import kv
from tests import kv_ref as R
from tests.test_gpu_kv import TOL, Problem, normal
from tests.test_gpu_kv_hidden import check

pytestmark = pytest.mark.gpu


def put(p, at, k, v, kf, vf):
    """Token `at` of the only sequence gets the keys k and values v [1][kv heads][channels]."""
    kv.write(p.cache, k, v, p.slots[0][at : at + 1])
    p.keys[0][at : at + 1] = R.kept(k.float().cpu().numpy(), kf)
    p.values[0][at : at + 1] = R.kept(v.float().cpu().numpy(), vf)


def large(shape, seed, dtype):
    return (normal(shape, seed, dtype).float() * (1e4 if dtype == "f16" else 1e5)).to(normal((1,), 0, dtype).dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,n", [(3, 5003), (60, 3001)])
def test_hidden_large_token_in_splits(dtype, dim, rows, n):
    """One split's workgroup meets the token, which only the first rows' window holds, the others do not."""
    p = Problem([n], [rows], 4, 2, dim, "q8_0", "q4_0", dtype, seed=41, v_scale=lambda r, m: np.full(m, 0.01, np.float32))
    window = 700
    put(p, n - rows - window + 2, normal((1, 2, dim), 42, dtype), large((1, 2, dim), 43, dtype), "q8_0", "q4_0")
    check(p, rows, 4, 2, window=window)
    check(p, rows, 4, 2)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sums", [True, False])
def test_hidden_large_token_beside_nan(dtype, sums):
    """A value without a number reaches the rows that see it, in its block's channels, and takes nothing from the exact results
    of those that do not; nor does a large one in the same 32 keys."""
    n, rows, dim = 200, 80, 128
    p = Problem([n], [rows], 4, 2, dim, "q8_0", "q4_0", dtype, seed=44, v_scale=lambda r, m: np.full(m, 0.01, np.float32))
    k, v = normal((1, 2, dim), 45, dtype), normal((1, 2, dim), 46, dtype)
    v[0, :, 40] = float("nan")
    kv.write(p.cache, k, v, p.slots[0][150:151])
    kv.write(p.cache, k, large((1, 2, dim), 47, dtype), p.slots[0][155:156])
    got = kv.attend(*p.args(), max_queries=rows, return_lse=sums)
    out = got[0] if sums else got
    sees, more = 150 - (n - rows), 155 - (n - rows)
    want, _ = R.attend(p.q.double().cpu().numpy(), p.keys, p.values, p.counts)
    big = np.abs(p.values[0]).max()
    assert np.abs(out[:sees].double().cpu().numpy() - want[:sees]).max() <= TOL[dtype] * big
    assert torch.isnan(out[sees:, :, 32:64]).all()
    other = torch.cat([out[sees:, :, :32], out[sees:, :, 64:]], dim=2)
    assert torch.isfinite(other).all()
    assert other[: more - sees].abs().max() <= 2 * float(np.abs(R.kept(v.nan_to_num().float().cpu().numpy(), "q4_0")).max())


@pytest.mark.parametrize("sums", [True, False])
def test_second_pass_in_graphs(sums):
    """bf16 calls whose workgroups begin again, replayed between other work: the eager calls' bits every time."""
    n, rows, dim = 450, 90, 128
    p = Problem([n], [rows], 4, 2, dim, "q4_0", "q4_0", "bf16", seed=48, v_scale=lambda r, m: np.full(m, 0.01, np.float32))
    put(p, n - 20, normal((1, 2, dim), 49, "bf16"), large((1, 2, dim), 50, "bf16"), "q4_0", "q4_0")
    args = p.args()
    kv.attend(*args, max_queries=rows, return_lse=sums)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv.attend(*args, max_queries=rows, return_lse=sums)
    for seed in range(3):
        args[1].copy_(normal(tuple(args[1].shape), 60 + seed, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        want = kv.attend(*args, max_queries=rows, return_lse=sums)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in (zip(got, want) if sums else [(got, want)]))
