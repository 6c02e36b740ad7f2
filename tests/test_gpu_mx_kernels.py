"""Every kernel of the microscaled products on sizes that end inside its tiles, and on K shorter and longer than what it keeps ahead."""

import numpy as np
import pytest
import torch

from comp_amd import _abi, mx
from tests import mx_ref as R

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# (kernel, 16-row tiles of W, of X) -> T, N.  N odd: rows of Y at every alignment.
KERNELS = {("tile", 16, 16): (5737, 5801), ("tile", 8, 8): (1691, 1653), ("stream", 4, 2): (499, 1029), ("stream", 2, 2): (333, 801),
           ("stream", 1, 2): (117, 355)}  # fmt: skip
# one step of 128 and parts of it; a step less, as many as, and more than the tiled kernels keep ahead; parts of a piece of 512
DEPTHS = [32, 96, 160, 256, 416, 512, 672, 1184, 2080]


def random_rows(n, k, fmt, low, high, gen):
    """Rows of random codes and scales -> (Rows, their values in f64), both made on the device."""
    codes = torch.randint(0, 16 if fmt == "e2m1" else 256, (n, k), generator=gen, device="cuda", dtype=torch.uint8)
    if fmt == "e4m3":
        codes[codes & 127 == 127] = 3
    scales = torch.randint(low, high + 1, (n, k // 32), generator=gen, device="cuda", dtype=torch.uint8)
    v = torch.from_numpy(R.table(fmt)).cuda()[codes.int()].view(n, -1, 32) * torch.exp2(scales.double() - 127)[..., None]
    plane = codes[:, ::2] | codes[:, 1::2] << 4 if fmt == "e2m1" else codes
    return mx.pack(plane.contiguous(), scales, fmt), v.view(n, k)


def check(y, x, w, fmt, dtype):
    """mx_ref.product_bound on the device: that many f32 roundings of the magnitudes' sum, and the result's own."""
    want, most = x @ w.T, x.abs() @ w.abs().T
    additions = 4 * (-(-x.shape[1] // (128 if fmt == "e2m1" else 32)) + 8)
    bits, least = {"f32": (24, 2.0**-149), "f16": (11, 2.0**-24), "bf16": (8, 2.0**-133)}[dtype]
    sums = additions * 2.0**-24 * most + 2.0**-149 * additions
    binade = torch.frexp(torch.clamp(want.abs() + sums, min=1e-300)).exponent.double() - 1
    bound = sums + torch.clamp(torch.exp2(binade - bits), min=least / 2)
    off = (y.double() - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max())} of the bound"  # (a NaN is not within it)


@pytest.mark.parametrize("k", DEPTHS)
@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("kernel", KERNELS, ids=lambda k: "%s-%d-%d" % k)
def test_kernel(kernel, fmt, k):
    t, n = KERNELS[kernel]
    assert _abi.mx_gemm_launch(t, n, k) == kernel
    gen = torch.Generator(device="cuda").manual_seed(k)
    x, xv = random_rows(t, k, fmt, 110, 120, gen)
    w, wv = random_rows(n, k, "e2m1", 112, 124, gen)  # (sums that f16 holds)
    for dtype in DTYPES:
        guard = torch.full((t, n + 7), 5.0, dtype=DTYPES[dtype], device="cuda")
        mx.gemm_into(x, w, guard[:, 3 : 3 + n])
        assert bool((guard[:, :3] == 5).all()) and bool((guard[:, 3 + n :] == 5).all())
        check(guard[:, 3 : 3 + n], xv, wv, fmt, dtype)
    assert torch.equal(mx.gemm(x, w, DTYPES[dtype]), guard[:, 3 : 3 + n])


@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("kernel", KERNELS, ids=lambda k: "%s-%d-%d" % k)
def test_places(kernel, fmt):
    """W holds one element a row: each place of K meets its own partner and scale, exactly."""
    t, n = KERNELS[kernel]
    k = 672
    assert _abi.mx_gemm_launch(t, n, k) == kernel
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, xv = random_rows(t, k, fmt, 100, 140, gen)
    codes, scales = np.zeros((n, k), np.uint8), np.zeros((n, k // 32), np.uint8)
    place = np.arange(n) % k
    codes[np.arange(n), place] = 2  # 1.0
    scales[np.arange(n), place // 32] = 127 + np.arange(n) % 7
    w = mx.pack(torch.from_numpy(codes[:, ::2] | codes[:, 1::2] << 4).cuda(), torch.from_numpy(scales).cuda())
    want = xv[:, torch.from_numpy(place).cuda()] * torch.from_numpy(2.0 ** (np.arange(n) % 7)).cuda()
    assert torch.equal(mx.gemm(x, w).double(), want)


@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("kernel", [k for k in KERNELS if k[0] == "tile"], ids=lambda k: "%s-%d-%d" % k)
def test_tiles_replayed(kernel, fmt):
    """In a graph, on other rows each time, with eager products between the replays."""
    t, n = KERNELS[kernel]
    k = 1184
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, w = random_rows(t, k, fmt, 110, 120, gen)[0], random_rows(n, k, "e2m1", 112, 124, gen)[0]
    y = torch.empty((t, n), dtype=torch.bfloat16, device="cuda")
    mx.gemm_into(x, w, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mx.gemm_into(x, w, y)
    for _ in range(3):
        other = torch.randn((t, k), generator=gen, device="cuda")
        mx.quantize_into(other, x)
        y.fill_(7)
        graph.replay()
        assert torch.equal(y, mx.gemm(x, w, torch.bfloat16))
