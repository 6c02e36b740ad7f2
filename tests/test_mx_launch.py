"""Which kernel a microscaled product runs on (the library's plan query; no GPU needed)."""

import pytest

from comp_amd import _abi

STEP, STREAM, TILE = _abi.MX_KERNELS


def test_rows_of_one_tile():
    """Up to 16 rows: kept in registers while K is at most 16384, from memory past that."""
    for n in (1, 17, 4096, 128256, 1 << 26):
        for t in (1, 2, 15, 16):
            for k, kernel in ((32, STEP), (8192, STEP), (8224, STEP), (16384, STEP), (16416, STREAM), (20000, STREAM)):
                assert _abi.mx_gemm_launch(t, n, k) == (kernel, 1, 1)


def test_grids_hold_every_size():
    """Column groups are the grid's second dimension, threads of all row groups fit its first."""
    for t in (17, 100, 8192, 16 * 65535):
        for n in (1, 16, 100, 4096, 1 << 26):
            kernel, rows, cols = _abi.mx_gemm_launch(t, n, 1024)
            assert kernel in (STREAM, TILE) and -(-t // (16 * cols)) <= 65535 and -(-n // (16 * rows)) * 512 < 1 << 32


def test_query_refusals():
    for args in ((0, 5, 64), (5, 0, 64), (-1, 5, 64), (5, 5, 0), (5, 5, 48), (5, 5, 1 << 27), (1 << 20, 5, 64), (5, (1 << 26) + 1, 64),
                 (5, 1 << 26, 1 << 26)):  # fmt: skip
        with pytest.raises(_abi.KompArgumentError):
            _abi.mx_gemm_launch(*args)
    _abi.call("komp_mx_gemm_launch", 5, 5, 64, None, None, None)


def covered(launch, t, n):
    """Rows of X times rows of W that the tiles cover, of a product t x n."""
    _, rows, cols = launch
    return -(-t // (16 * cols)) * 16 * cols * -(-n // (16 * rows)) * 16 * rows


@pytest.mark.parametrize("t", [17, 20, 32])
@pytest.mark.parametrize("n", [28672, 70000, 128256, 131072, 1 << 22])
def test_few_rows_and_many_weights(t, n):
    """One tile of 32 columns holds all of X: no tile whose other columns are thrown away."""
    assert _abi.mx_gemm_launch(t, n, 4096) == (STREAM, 4, 2)


@pytest.mark.parametrize("t", [8192, 32768, 262144, 1 << 19])
@pytest.mark.parametrize("n,rows", [(1, 1), (16, 1), (17, 2), (32, 2), (64, 4)])
def test_many_rows_and_few_weights(t, n, rows):
    launch = _abi.mx_gemm_launch(t, n, 4096)
    assert launch[0] == STREAM and launch[1] <= rows
    assert launch[1] == rows or t == 8192  # (fewer where the larger tiles would not fill the device)


def test_tiles_are_mostly_filled():
    """No tiled kernel where 64 x 32 tiles hold all of X, and 256 x 256 tiles cover at most 5/4 of what 128 x 128 tiles cover."""
    for t in (33, 48, 64, 100, 128, 129, 144, 192, 256, 257, 300, 512, 640, 1041, 4112, 8192, 100000):
        for n in (65, 80, 128, 200, 2048, 6912, 8237, 28672, 33000, 65536, 131072, 131080):
            launch = _abi.mx_gemm_launch(t, n, 4096)
            if launch[0] == TILE:
                assert t > 32
                assert 4 * covered(launch, t, n) <= 5 * covered((TILE, 8, 8), t, n)


# (T, N, K) on both sides of the lines, on 256 CUs: times in the comment at the rule
# fmt: off
MEASURED = [
    (17, 131072, 4096, (STREAM, 4, 2)), (33, 131072, 4096, (TILE, 8, 8)), (128, 131072, 4096, (TILE, 8, 8)),
    (144, 131072, 4096, (TILE, 16, 16)), (300, 131072, 4096, (TILE, 8, 8)), (640, 131072, 4096, (TILE, 16, 16)),
    (32, 28672, 4096, (STREAM, 4, 2)), (48, 28672, 4096, (TILE, 8, 8)), (262144, 64, 1024, (STREAM, 4, 2)),
    (262144, 80, 1024, (TILE, 8, 8)), (262144, 32, 1024, (STREAM, 2, 2)), (8192, 16, 4096, (STREAM, 1, 2)),
    (8192, 14336, 4096, (TILE, 16, 16)), (2048, 4096, 4096, (TILE, 8, 8)), (777, 6912, 2560, (TILE, 8, 8)),
    (256, 14336, 4096, (TILE, 8, 8)), (256, 4096, 14336, (STREAM, 4, 2)), (100, 4096, 4096, (STREAM, 4, 2)),
    (64, 4096, 14336, (STREAM, 2, 2)), (32, 4096, 14336, (STREAM, 1, 2)),
]
# fmt: on


@pytest.mark.parametrize("t,n,k,want", MEASURED)
def test_measured_lines(t, n, k, want):
    assert _abi.mx_gemm_launch(t, n, k) == want
