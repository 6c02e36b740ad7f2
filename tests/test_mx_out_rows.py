"""Results whose rows overlap are refused by the C entries too: two workgroups would write one place."""

import ctypes

import pytest
import torch

from comp_amd import _abi, mx

K, N = 64, 10


def rows(count, fmt=0):
    """A descriptor whose planes are never touched: every call here is refused."""
    return ctypes.byref(_abi.MxRowsStruct(4096, 4096, count, K, fmt))


@pytest.mark.parametrize("less", [1, 5, "all"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("count", [2, 5, 16])
def test_overlapping_rows(count, sign, less):
    stride = lambda width: 0 if less == "all" else sign * (width - less)  # noqa: E731
    for name, args in [("komp_mx_gemm", (rows(count), rows(N), 4096, 0, stride(N))),
                       ("komp_mx_linear", (4096, 0, K, count, 0, rows(N), 4096, 0, stride(N))),
                       ("komp_mx_lookup", (rows(N), 4096, count, 4096, 0, stride(K), 1.0)),
                       ("komp_mx_lookup", (rows(count), None, count, 4096, 0, stride(K), 1.0))]:  # fmt: skip
        with pytest.raises(_abi.KompArgumentError, match="overlap"):
            _abi.call(name, *args, None)


@pytest.mark.gpu
def test_rows_apart():
    """A single row at any stride, and rows one behind the other in either direction."""
    gen = torch.Generator().manual_seed(2)
    w = mx.quantize(torch.randn((N, K), generator=gen).cuda())
    x = torch.randn((5, K), generator=gen).cuda()
    q, ids = mx.quantize(x, "e4m3"), torch.tensor([3, 0, 9, 9, 1], device="cuda")
    want, looked = mx.gemm(q, w), mx.lookup(w, ids)
    stream = torch.cuda.current_stream().cuda_stream
    for sign in (1, -1):
        y, out = torch.zeros(5, N, device="cuda"), torch.zeros(5, K, device="cuda")
        first = 0 if sign > 0 else 4
        _abi.call("komp_mx_gemm", q._ref, w._ref, y[first].data_ptr(), 0, sign * N, stream)
        assert torch.equal(y if sign > 0 else y.flip(0), want)
        y.zero_()
        _abi.call("komp_mx_linear", x.data_ptr(), 0, K, 5, 1, w._ref, y[first].data_ptr(), 0, sign * N, stream)
        assert torch.equal(y if sign > 0 else y.flip(0), want)
        _abi.call("komp_mx_lookup", w._ref, ids.data_ptr(), 5, out[first].data_ptr(), 0, sign * K, 1.0, stream)
        assert torch.equal(out if sign > 0 else out.flip(0), looked)
    y = torch.zeros(N, device="cuda")
    _abi.call("komp_mx_linear", x.data_ptr(), 0, 0, 1, 1, w._ref, y.data_ptr(), 0, 0, stream)
    assert torch.equal(y, want[0])
