"""What a row does not see does not reach its result through other rows either: a token with large, finite keys and values
that only some rows of a call see leaves the others as exact as they are without it.

Each row is held to tests/test_gpu_kv.py's tolerances relative to the largest value that this row itself sees.  A row that
sees a large key has scores of 1e5 beside which those tolerances' |score| <= 40 does not hold: it is held to them where
that key takes all or nothing (its score is 1000 or more away from all others), and its lse is not."""

import numpy as np
import pytest
import torch

from comp_amd import kv
from tests import kv_ref as R
from tests.test_gpu_kv import PAIRS, TOL, Problem, normal

pytestmark = pytest.mark.gpu


def check(p, rows, heads, kv_heads, large_key=None, **opts):
    n, group, dim = p.lengths[0], heads // kv_heads, p.q.shape[2]
    q = p.q.double().cpu().numpy()
    want, want_lse = R.attend(q, p.keys, p.values, p.counts, **opts)
    for sums in (True, False):
        got = kv.attend(*p.args(), max_queries=rows, return_lse=sums, **opts)
        out, lse = got if sums else (got, None)
        out = out.double().cpu().numpy()
        for r in range(rows):
            i = n - rows + r
            lo = max(0, i - opts["window"] + 1) if opts.get("window") else 0
            for h in range(heads):
                if large_key is not None and lo <= large_key <= i:
                    score = p.keys[0][lo : i + 1, h // group] @ q[r, h] * dim**-0.5
                    others = np.delete(score, large_key - lo)
                    if not (score[large_key - lo] > others.max() + 1000 or score[large_key - lo] < others.min() - 1000):
                        continue
                big = np.abs(p.values[0][lo : i + 1, h // group]).max()
                off = np.abs(out[r, h] - want[r, h]).max() / big
                assert off <= TOL[p.dtype], f"row {r}, head {h}, sums {sums}: {off:.3g} of the largest value that it sees"
        if sums:
            sure = np.array([large_key is None or i < large_key for i in range(n - rows, n)])
            lse = lse.double().cpu().numpy()
            assert (np.abs(lse - want_lse) <= 1e-5 * (4 + np.abs(want_lse)))[sure].all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("kf,vf", PAIRS)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("rows,at", [(7, -3), (80, -30)])
@pytest.mark.parametrize("small", [1.0, 0.01])
def test_hidden_large_token(dtype, kf, vf, dim, rows, at, small):
    """The last rows see the token, those before it do not.  Few columns a kv head, and many."""
    large_token(dtype, kf, vf, dim, rows, at, small)


def large_token(dtype, kf, vf, dim, rows, at, small):
    n, heads, kv_heads = 200, 4, 2
    p = Problem([n], [rows], heads, kv_heads, dim, kf, vf, dtype, seed=31, v_scale=lambda r, m: np.full(m, small, np.float32))
    large = 1e4 if dtype == "f16" else 1e5
    k, v = (normal((1, kv_heads, dim), 32 + i, dtype) for i in range(2))
    for what in ("value", "key", "both"):
        print(what, flush=True)
        kk = (k.float() * (large if what != "value" else 1.0)).to(k.dtype)
        vv = (v.float() * (large if what != "key" else small)).to(v.dtype)
        kv.write(p.cache, kk, vv, p.slots[0][n + at : n + at + 1])
        p.keys[0][n + at : n + at + 1] = R.kept(kk.float().cpu().numpy(), kf)
        p.values[0][n + at : n + at + 1] = R.kept(vv.float().cpu().numpy(), vf)
        check(p, rows, heads, kv_heads, large_key=None if what == "value" else n + at)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [7, 80])
def test_hidden_by_a_window(dtype, rows):
    """The first rows' window holds the token, the later rows' does not."""
    n, heads, kv_heads, dim = 300, 4, 2, 128
    p = Problem([n], [rows], heads, kv_heads, dim, "q8_0", "q4_0", dtype, seed=33, v_scale=lambda r, m: np.full(m, 0.01, np.float32))
    window = 100
    at = n - rows - window + 4  # seen by the first rows only
    v = (normal((1, kv_heads, dim), 34, dtype).float() * (1e4 if dtype == "f16" else 1e5)).to(p.q.dtype)
    k = normal((1, kv_heads, dim), 35, dtype)
    kv.write(p.cache, k, v, p.slots[0][at : at + 1])
    p.keys[0][at : at + 1] = R.kept(k.float().cpu().numpy(), "q8_0")
    p.values[0][at : at + 1] = R.kept(v.float().cpu().numpy(), "q4_0")
    check(p, rows, heads, kv_heads, window=window)
