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
