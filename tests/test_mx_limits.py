"""Products past the sizes that one call takes are refused before anything is launched or allocated."""

import pytest
import torch

from comp_amd import _abi, mx

ROWS, WEIGHTS = (1 << 20) - 16, 1 << 26  # the most rows of X and of W


def held(rows, k, fmt="e2m1"):
    """Rows of any number whose planes are never touched."""
    r = mx.Rows.__new__(mx.Rows)
    r._hold(rows, k, fmt, mx._plane_sizes(rows, k, fmt), torch.zeros(16, dtype=torch.uint8))
    return r


@pytest.fixture
def launches(monkeypatch):
    """The names of what would be launched, and of no tensor but those on a HIP device refused."""
    seen = []
    monkeypatch.setattr(mx, "_launch", lambda name, *args: seen.append(name))
    monkeypatch.setattr(mx, "_need_matrix", lambda *args, **kw: None)
    return seen


@pytest.mark.parametrize("t,n", [(ROWS + 1, 5), (17, WEIGHTS + 1), (3, WEIGHTS + 1), (1 << 30, 5)])
def test_past_the_limits(launches, t, n):
    x, y = torch.zeros(1, 64).expand(t, 64), torch.zeros(1, 1).expand(t, n)
    w = held(n, 64)
    for call in (lambda: mx.linear(x, w), lambda: mx.linear_into(x, w, y), lambda: mx.gemm(held(t, 64), w), lambda: mx.gemm_into(held(t, 64), w, y)):
        with pytest.raises(_abi.KompArgumentError, match="2\\^20 - 16"):
            call()
    assert launches == []


def test_at_the_limits(launches):
    y = torch.zeros(1, 1).expand(ROWS, 5)
    mx.linear_into(torch.zeros(1, 64).expand(ROWS, 64), held(5, 64), y)
    mx.gemm_into(held(ROWS, 64), held(5, 64), y)
    mx.linear_into(torch.zeros(3, 64), held(WEIGHTS, 64), torch.zeros(1, 1).expand(3, WEIGHTS))
    assert launches == ["komp_mx_quantize", "komp_mx_gemm", "komp_mx_gemm", "komp_mx_linear"]
