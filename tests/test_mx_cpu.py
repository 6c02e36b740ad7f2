"""The microscaled rows' C entries and Python surface without a device: refusals, sizes, names."""

import ctypes

import numpy as np
import pytest
import torch

from comp_amd import _abi, mx
from tests import mx_ref as R


def rows(**over):
    """A descriptor whose planes are never touched: every call here is refused or has nothing to do."""
    f = dict(CODES=4096, SCALES=4096, rows=10, k=64, fmt=0)
    f.update(over)
    return ctypes.byref(_abi.MxRowsStruct(*f.values()))


def refused(name, *args):
    with pytest.raises(_abi.KompArgumentError):
        _abi.call(name, *args)


BAD_ROWS = [dict(k=0), dict(k=48), dict(k=-32), dict(k=1 << 27), dict(rows=-1), dict(rows=1 << 31), dict(rows=1 << 30, k=1 << 20),
            dict(fmt=2), dict(fmt=-1), dict(CODES=None), dict(SCALES=None), dict(CODES=4104), dict(SCALES=4104)]  # fmt: skip


@pytest.mark.parametrize("over", BAD_ROWS, ids=str)
def test_bad_rows(over):
    r = rows(**over)
    refused("komp_mx_quantize", r, 4096, 0, 64, 0, None)
    refused("komp_mx_lookup", r, 4096, 3, 4096, 0, 64, 1.0, None)
    refused("komp_mx_pack", r, 4096, 4096, None)
    refused("komp_mx_unpack", r, 4096, 4096, None)
    refused("komp_mx_gemm", r, rows(), 4096, 0, 10, None)
    refused("komp_mx_gemm", rows(), r, 4096, 0, 10, None)
    refused("komp_mx_linear", 4096, 0, 64, 3, 0, r, 4096, 0, 10, None)


def test_bad_arguments():
    r = rows()
    for args in [(None, 0, 64, 0), (4098, 0, 64, 0), (4097, 1, 64, 0), (4096, 3, 64, 0), (4096, -1, 64, 0), (4096, 0, 1 << 50, 0),
                 (4096, 0, 64, 3), (4096, 0, 64, -1)]:  # fmt: skip
        refused("komp_mx_quantize", r, *args, None)
    for args in [(4096, -1, 4096, 0, 64), (4096, 1 << 31, 4096, 0, 64), (4100, 3, 4096, 0, 64), (4096, 3, None, 0, 64),
                 (4096, 3, 4096, 5, 64), (None, 3, 4096, 0, 64), (4096, 3, 4098, 0, 64)]:  # fmt: skip
        refused("komp_mx_lookup", r, *args, 1.0, None)
    refused("komp_mx_pack", r, None, 4096, None)
    refused("komp_mx_pack", rows(fmt=1), 4096, None, None)  # block_mxfp4 blocks are e2m1
    refused("komp_mx_unpack", r, None, 4096, None)
    refused("komp_mx_unpack", r, 4096, None, None)
    for x, w, args in [(dict(), dict(fmt=1), (4096, 0, 10)), (dict(k=96), dict(), (4096, 0, 10)), (dict(), dict(), (None, 0, 10)),
                       (dict(), dict(), (4096, 3, 10)), (dict(), dict(), (4097, 1, 10)), (dict(rows=1 << 20), dict(), (4096, 0, 10)),
                       (dict(), dict(rows=(1 << 26) + 1), (4096, 0, 10))]:  # fmt: skip
        refused("komp_mx_gemm", rows(**x), rows(**w), *args, None)
    for args in [(None, 0, 64, 3, 0, r, 4096, 0, 10), (4096, 3, 64, 3, 0, r, 4096, 0, 10), (4096, 0, 64, 17, 0, r, 4096, 0, 10),
                 (4096, 0, 64, -1, 0, r, 4096, 0, 10), (4096, 0, 64, 3, 2, r, 4096, 0, 10), (4096, 0, 64, 3, 0, rows(fmt=1), 4096, 0, 10),
                 (4096, 0, 64, 3, 0, r, None, 0, 10), (4096, 0, 64, 3, 0, None, 4096, 0, 10), (4096, 0, 64, 3, 0, r, 4096, 4, 10)]:  # fmt: skip
        refused("komp_mx_linear", *args, None)
    assert "komp_mx_linear" in _abi.last_error()


def test_nothing_to_do():
    none = rows(rows=0, CODES=None, SCALES=None)
    _abi.call("komp_mx_quantize", none, None, 0, 0, 0, None)
    _abi.call("komp_mx_lookup", rows(), 4096, 0, None, 0, 0, 1.0, None)
    _abi.call("komp_mx_lookup", none, None, 0, None, 0, 0, 1.0, None)
    _abi.call("komp_mx_pack", none, None, None, None)
    _abi.call("komp_mx_unpack", none, None, None, None)
    _abi.call("komp_mx_gemm", none, rows(), None, 0, 0, None)
    _abi.call("komp_mx_gemm", rows(), none, None, 0, 0, None)
    _abi.call("komp_mx_linear", None, 0, 0, 0, 1, rows(), None, 0, 0, None)


def test_python_refusals():
    x = torch.zeros(4, 64)
    for call in [lambda: mx.Rows(4, 64, device="cpu"), lambda: mx.Rows(4, 48), lambda: mx.Rows(4, 64, "e5m2"), lambda: mx.Rows(-1, 64),
                 lambda: mx.quantize(x), lambda: mx.gate(x), lambda: mx.gate(x, act="gelu"), lambda: mx.pack(x.byte(), x.byte()),
                 lambda: mx.from_ggml(x.byte(), 4, 64), lambda: mx.pack(x.byte(), x.byte(), "q4_0")]:  # fmt: skip
        with pytest.raises(_abi.KompArgumentError):
            call()
    for call in [lambda: mx.quantize(3), lambda: mx.quantize_into(x, x), lambda: mx.gemm(x, x), lambda: mx.linear(x, x),
                 lambda: mx.lookup(x, x), lambda: mx.values(x), lambda: mx.unpack(None), lambda: mx.gate_into(x, None)]:  # fmt: skip
        with pytest.raises(TypeError):
            call()


def test_komp_name():
    from komp import mx as other

    assert other is mx


def test_reference_of_known_values():
    """The tests' own plain form, on values that are known: the formats' tables, ties, saturation, the smallest scale."""
    x = np.zeros((1, 64))
    x[0, :8] = [7.0, 0.25, 0.75, 1.25, -2.5, -3.5, 5.0, -0.0]
    x[0, 32] = 2.0**-149
    codes, scales = R.quantize(x, "e2m1")
    assert codes[0, :8].tolist() == [7, 0, 2, 2, 8 + 4, 8 + 6, 6, 8] and scales.tolist() == [[127, 0]]
    assert codes[0, 32] == 0  # 2^-149 of 2^-127's steps of half of it
    x[0, :4] = [460.0, 448.0, 2.0**-9, 2.0**-10]
    codes, scales = R.quantize(x, "e4m3")
    assert codes[0, :4].tolist() == [0x7E, 0x7E, 1, 0] and scales[0, 0] == 127
    assert R.quantize(np.full((1, 32), np.inf), "e2m1")[1].tolist() == [[255]]
