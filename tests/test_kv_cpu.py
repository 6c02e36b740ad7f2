"""The key/value cache's C entries and Python surface without a device: refusals, plans, names."""

import ctypes

import pytest
import torch

from comp_amd import _abi, kv


def cache(**over):
    """A descriptor whose planes are never touched: every call here is refused, or asks for a plan."""
    f = dict(KQ=4096, KS=4096, VQ=4096, VS=4096, pages=10, heads=2, head_dim=64, page=64, k_fmt=0, v_fmt=0)
    f.update(over)
    return _abi.KvCacheStruct(*f.values())


def refused(name, *args):
    with pytest.raises(_abi.KompArgumentError):
        _abi.call(name, *args)


def workspace(c, type=0, t=4, batch=4, heads=4, max_queries=1, max_length=8192):
    v = ctypes.c_int64(-1)
    _abi.call("komp_kv_attend_workspace", ctypes.byref(c), type, t, batch, heads, max_queries, max_length, ctypes.byref(v))
    return v.value


BAD_CACHES = [dict(head_dim=80), dict(head_dim=0), dict(page=16), dict(page=96), dict(page=1 << 17), dict(heads=0), dict(pages=-1),
              dict(k_fmt=0, v_fmt=2), dict(k_fmt=1), dict(v_fmt=3), dict(KQ=None), dict(VS=None), dict(KS=4098)]  # fmt: skip


@pytest.mark.parametrize("over", BAD_CACHES, ids=str)
def test_bad_caches(over):
    c = ctypes.byref(cache(**over))
    refused("komp_kv_write", c, 4096, 4096, 0, 4096, 3, 128, 64, 128, 64, None)
    refused("komp_kv_read", c, 4096, 3, 4096, 4096, 0, None)
    refused("komp_kv_attend_workspace", c, 0, 4, 4, 4, 1, 100, ctypes.byref(ctypes.c_int64()))


def test_bad_arguments():
    c = ctypes.byref(cache())
    for args in [(4096, 4096, 3, 4096, 3, 128, 64, 128, 64), (4096, 4096, -1, 4096, 3, 128, 64, 128, 64),
                 (None, 4096, 0, 4096, 3, 128, 64, 128, 64), (4096, None, 0, 4096, 3, 128, 64, 128, 64),
                 (4096, 4096, 0, None, 3, 128, 64, 128, 64), (4098, 4096, 0, 4096, 3, 128, 64, 128, 64),
                 (4096, 4096, 0, 4100, 3, 128, 64, 128, 64), (4096, 4096, 0, 4096, -1, 128, 64, 128, 64),
                 (4096, 4096, 0, 4096, 1 << 40, 128, 64, 128, 64)]:  # fmt: skip
        refused("komp_kv_write", c, *args, None)
    for args in [(4096, -3, 4096, 4096, 0), (4096, 3, 4100, 4096, 0), (4096, 3, 4096, None, 0), (None, 3, 4096, 4096, 0),
                 (4096, 3, 4096, 4096, 7)]:  # fmt: skip
        refused("komp_kv_read", c, *args, None)
    refused("komp_kv_write", None, 4096, 4096, 0, 4096, 3, 128, 64, 128, 64, None)
    good = dict(Q=4096, OUT=4096, LSE=None, type=0, TABLES=4096, LENGTHS=4096, STARTS=None, PREFIX=None, SLOPES=None, T=4,
                batch=4, heads=4, qt=256, qh=64, ot=256, oh=64, ts=10, cols=10, max_queries=1, max_length=100, scale=0.1,
                softcap=0.0, window=0, WORK=None, work_bytes=0)  # fmt: skip
    for over in [dict(Q=None), dict(OUT=None), dict(TABLES=None), dict(LENGTHS=None), dict(Q=4098), dict(type=3), dict(T=5),
                 dict(T=-1), dict(heads=3), dict(heads=0), dict(batch=70000, T=70000), dict(max_queries=5), dict(max_queries=-1),
                 dict(T=1 << 24, max_queries=1 << 24, STARTS=4096),
                 dict(max_length=-1), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(window=-1),
                 dict(cols=-1), dict(cols=1 << 40), dict(LSE=4098), dict(SLOPES=4098), dict(max_length=100000)]:  # fmt: skip
        refused("komp_kv_attend", c, *{**good, **over}.values(), None)


def test_nothing_to_do():
    """No tokens and no rows are no error, and launch nothing."""
    c = ctypes.byref(cache())
    _abi.call("komp_kv_write", c, None, None, 0, None, 0, 0, 0, 0, 0, None)
    _abi.call("komp_kv_read", c, None, 0, None, None, 0, None)
    _abi.call("komp_kv_attend", c, *[None] * 3, 0, *[None] * 5, 0, 0, 4, 0, 0, 0, 0, 0, 0, 0, 0, 0.1, 0.0, 0, None, 0, None)


def test_workspace():
    """Splits, and their workspace, where few rows meet many keys; none where the rows fill the device."""
    c = cache(pages=100000)
    assert workspace(c, max_length=100) == 0
    few = workspace(c, max_length=8192)
    assert few > 0 and few % 8 == 0
    assert workspace(c, t=8, batch=8, max_length=8192) > 0
    assert workspace(c, t=0, batch=0, max_queries=0) == 0
    assert workspace(c, t=60000, batch=60000, max_length=8192) == 0
    assert workspace(c, t=4096, batch=1, heads=64, max_queries=4096, max_length=4096) == 0
    for dim in kv.HEAD_DIMS:
        for type in range(3):
            # [split][row][head][dim] f32, then [split][row][head] of two f32
            got = workspace(cache(head_dim=dim), type=type)
            assert any(got == -(-s * 16 * dim * 4 // 256) * 256 + s * 16 * 8 for s in range(2, 65)), (dim, type, got)


def test_python_refusals():
    for args in [dict(head_dim=80), dict(k_format="q4_0", v_format="q8_0"), dict(page=40), dict(k_format="tq2_0"), dict(kv_heads=0),
                 dict(pages=-1), dict(device="cpu")]:  # fmt: skip
        with pytest.raises(_abi.KompArgumentError):
            kv.KVCache(**{**dict(pages=1, kv_heads=1, head_dim=64), **args})
    x = torch.zeros((1, 1, 64))
    for call in (lambda: kv.write(None, x, x, x), lambda: kv.read(None, x), lambda: kv.attend(None, x, x, x)):
        with pytest.raises(TypeError):
            call()


def test_komp_name():
    import komp

    assert komp.kv is kv
