"""Microscaled products at the ends of the scale bytes, of both formats and on every kind of kernel: finite sums within their bound,
sums past f32 infinite, NaN blocks in their own rows and columns alone."""

import numpy as np
import pytest
import torch

from comp_amd import mx
from tests import mx_ref as R

pytestmark = pytest.mark.gpu

LARGEST = float(np.finfo(np.float32).max)
# T, N, K: one column tile with K in registers as one piece a wave and as four, and from memory; batches; tiles through shared memory
SIZES = [(1, 50, 256), (5, 50, 9216), (3, 50, 16416), (20, 50, 256), (100, 50, 256), (1691, 1653, 256)]


def put(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def pack(codes, scales, fmt="e2m1"):
    return mx.pack(put(codes[:, ::2] | codes[:, 1::2] << 4 if fmt == "e2m1" else codes), put(scales), fmt)


def product(xc, xs, fmt, wc, ws):
    """The kernels' product, x's and w's values, and the definition's product with its bound."""
    y = mx.gemm(pack(xc, xs, fmt), pack(wc, ws)).cpu().double().numpy()
    xv, wv = R.values(xc, xs, fmt), R.values(wc, ws, "e2m1")
    with np.errstate(invalid="ignore"):
        return y, xv, wv, *R.product_bound(xv, wv, fmt, "f32")


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_one_row_and_one_column(fmt, size):
    """Every kind of block beside ordinary ones; all values are finite in f32, and so are all sums but those of two rows."""
    t, n, k = size
    g = np.random.default_rng(t)
    xc = g.integers(0, 8 if fmt == "e2m1" else 120, (t, k), dtype=np.uint8)  # positive, up to 240 in e4m3
    wc = g.integers(0, 16, (n, k), dtype=np.uint8)
    xs, ws = np.full((t, k // 32), 127, np.uint8), np.full((n, k // 32), 127, np.uint8)
    top = 246 if fmt == "e4m3" else 251
    xs[:, 1] = top - 10
    ws[:5], ws[5:10] = 0, 1
    ws[10:20, 2] = 20
    ws[20, 3] = 255
    wc[30:40] &= 7
    wc[30:40, 192:224] = 7  # 6, beside the rows' largest values
    if t > 1:
        xs[1, 5] = 255
        xc[2:4, 192:224] = 7 if fmt == "e2m1" else 119
        xs[2:4, 6] = top
    y, xv, wv, want, bound = product(xc, xs, fmt, wc, ws)
    bad = np.zeros((t, n), bool)
    bad[:, 20] = True
    if t > 1:
        bad[1] = True
    assert np.array_equal(np.isnan(xv).any(1)[:, None] | np.isnan(wv).any(1), bad)
    assert np.isnan(y[bad]).all()
    large = np.zeros((t, n), bool)
    large[2:4] = True  # (of ordinary weights: partial sums may pass f32's largest on their way)
    large[:, :10] = False
    inside = ~bad & ~large
    assert (np.abs(xv[inside.any(1)]) @ np.abs(wv[inside.any(0)]).T)[inside[inside.any(1)][:, inside.any(0)]].max() < LARGEST
    assert (np.abs(y - want)[inside] <= bound[inside]).all()  # finite: a NaN or an infinity is not
    if t > 1:
        assert (want[2:4, 30:40] - bound[2:4, 30:40] > LARGEST).all() and (y[2:4, 30:40] == np.inf).all()


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("xs,ws", [(240, 0), (240, 1), (246, 0), (246, 2), (3, 252), (10, 252), (130, 126)])
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_ends(fmt, xs, ws, size):
    """The smallest weights (subnormal in bf16) times large rows, the largest times small rows."""
    t, n, k = size
    g = np.random.default_rng(xs)
    xc = g.integers(0, 16 if fmt == "e2m1" else 256, (t, k), dtype=np.uint8)
    if fmt == "e4m3":
        xc[xc & 127 == 127] = 3
    y, _, _, want, bound = product(xc, np.full((t, k // 32), xs, np.uint8), fmt, g.integers(0, 16, (n, k), dtype=np.uint8),
                                   np.full((n, k // 32), ws, np.uint8))  # fmt: skip
    assert np.abs(want).max() > 2.0**-20 and (np.abs(y - want) <= bound).all()


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("xs,ws", [(0, 252), (1, 250), (2, 246)])
def test_smallest_rows(xs, ws, size):
    """e4m3 rows of the scale bytes 0 to 2 have elements between bf16's multiples of 2^-133: each is off by half of one at most."""
    t, n, k = size
    g = np.random.default_rng(xs)
    xc = g.integers(0, 256, (t, k), dtype=np.uint8)
    xc[xc & 127 == 127] = 3
    y, _, wv, want, bound = product(xc, np.full((t, k // 32), xs, np.uint8), "e4m3", g.integers(0, 16, (n, k), dtype=np.uint8),
                                    np.full((n, k // 32), ws, np.uint8))  # fmt: skip
    assert (np.abs(y - want) <= bound + 2.0**-134 * np.abs(wv).sum(1)).all()


@pytest.mark.parametrize("t", [1, 16, 20])
def test_past_the_largest(t):
    """Scale bytes that only pack() and from_ggml() bring: e2m1 from 253, e4m3 from 247 on.  Values past f32's largest are infinite
    when read; e2m1 rows times e2m1 weights never form them, the products with e4m3 rows do."""
    codes = np.tile(np.array([0, 7, 15, 2], np.uint8), (t, 16))
    values = mx.values(pack(codes, np.full((t, 2), 253, np.uint8))).cpu().numpy()
    assert np.array_equal(values, np.tile(np.array([0, np.inf, -np.inf, 2.0**126], np.float32), (t, 16)))
    e4m3 = np.tile(np.array([0, 0x7E, 0xFE, 0x38], np.uint8), (t, 16))  # 448 and 1
    values = mx.values(pack(e4m3, np.full((t, 2), 247, np.uint8), "e4m3")).cpu().numpy()
    assert np.array_equal(values, np.tile(np.array([0, np.inf, -np.inf, 2.0**120], np.float32), (t, 16)))
    w = np.tile(np.array([1, 7, 2, 2], np.uint8), (50, 16))  # positive weights, 6 * 2^127 among them
    ws = np.full((50, 2), 254, np.uint8)
    x = np.tile(np.array([2, 2, 2, 2], np.uint8), (t, 16))  # ones
    y, _, _, want, bound = product(x, np.full((t, 2), 20, np.uint8), "e2m1", w, ws)
    assert (np.abs(y - want) <= bound).all()
    y, *_ = product(np.full((t, 64), 0x38, np.uint8), np.full((t, 2), 20, np.uint8), "e4m3", w, ws)
    assert (y == np.inf).all()
