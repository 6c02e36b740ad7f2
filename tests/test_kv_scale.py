"""The score's factor: one that is no f32 number, or whose product with log2(e) is none, is refused."""

import ctypes

import pytest

from comp_amd import _abi

BAD = [float("nan"), float("inf"), -float("inf"), 1e39, -1e39, 3e38, -3e38]


@pytest.mark.parametrize("scale", BAD)
def test_scale_refused(scale):
    """By the C entry (the descriptor's planes are never touched; there is no device here to launch on)."""
    c = _abi.KvCacheStruct(4096, 4096, 4096, 4096, 10, 2, 64, 64, 0, 0)
    with pytest.raises(_abi.KompArgumentError, match="scale"):
        _abi.call("komp_kv_attend", ctypes.byref(c), 4096, 4096, None, 0, 4096, 4096, None, None, None, 4, 4, 4, 256, 64, 256, 64, 10,
                  10, 1, 100, scale, 0.0, 0, None, 0, None)  # fmt: skip


@pytest.mark.gpu
@pytest.mark.parametrize("scale", BAD)
def test_kv_attend_scale_refused(scale):
    import torch

    from comp_amd import kv

    cache = kv.KVCache(2, 2, 64)
    tables = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    lengths = torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.ones((1, 4, 64), device="cuda")
    with pytest.raises(_abi.KompArgumentError):
        kv.attend(cache, q, tables, lengths, scale=scale)
    for fine in (2e38, -2e38, 0.0):
        assert torch.equal(kv.attend(cache, q, tables, lengths, scale=fine), torch.zeros_like(q))  # (a new cache's values)
