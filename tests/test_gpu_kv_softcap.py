"""Capped scores over the whole range of caps: cap * tanh(score / cap) keeps what an uncapped score keeps.

Tolerances are those of uncapped scores (tests/test_gpu_kv.py): f32 1e-5 of the largest value and lse 1e-5 (4 + |lse|); f16
2^-10, bf16 2^-8.  tanh u has a relative error of a few 2^-24 at any u when it is evaluated without cancellation, so a capped
score is held as an uncapped one is, to a few 2^-24 of itself."""

import numpy as np
import pytest

from comp_amd import kv
from tests import kv_ref as R
from tests.test_gpu_kv import TOL, Problem

pytestmark = pytest.mark.gpu

CAPS = [1e-30, 0.5, 2.0, 5.0, 20.0, 50.0, 300.0, 1e3, 1e5, 1e6, 1e8, 1e20, 1.2e38, 2.0e38, 3.0e38]


def check(p, cap, **opts):
    q = p.q.double().cpu().numpy()
    want, want_lse = R.attend(q, p.keys, p.values, p.counts, softcap=cap, **opts)
    got, lse = kv.attend(*p.args(), max_queries=max(p.counts), softcap=cap, return_lse=True, **opts)
    plain = kv.attend(*p.args(), max_queries=max(p.counts), softcap=cap, **opts)
    big = max(np.abs(v).max() for v in p.values)
    for name, out in (("with lse", got), ("without", plain)):
        off = np.abs(out.double().cpu().numpy() - want).max() / big
        assert off <= TOL[p.dtype], f"cap {cap:g} {name}: {off:.3g} of the largest value"
    off = np.abs(lse.double().cpu().numpy() - want_lse)
    assert (off <= 1e-5 * (4 + np.abs(want_lse))).all(), f"cap {cap:g}: lse off by {off.max():.3g}"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kf,vf", [(64, "q4_0", "q4_0"), (128, "q8_0", "q4_0"), (256, "q8_0", "q8_0")])
@pytest.mark.parametrize("rows", [1, 70])
def test_softcap_range(dtype, dim, kf, vf, rows):
    """A few columns a kv head, and many."""
    p = Problem([300, 90], [rows, rows], 4, 2, dim, kf, vf, dtype, seed=21)
    for cap in CAPS:
        print(cap, flush=True)
        check(p, cap)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 70])
def test_softcap_across_its_bend(dtype, rows):
    """Scores from far below to far above the cap in one call, both signs; a bias and a window after it."""
    p = Problem([400], [rows], 4, 2, 128, "q8_0", "q8_0", dtype, seed=22, k_scale=3.0)
    for scale in (-0.4, 0.02, 0.1):
        for cap in (3.0, 10.0, 25.0):
            check(p, cap, scale=scale)
            check(p, cap, scale=scale, window=77)
