"""Attention calls whose sequences have no query row at most (max_queries = 0) while there are rows: nothing is computed."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch

from comp_amd import _abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES, DIMS = (0, 1, 2), (64, 96, 128, 256)


def descriptor(dim=64):
    """A cache whose planes are never touched."""
    return _abi.KvCacheStruct(4096, 4096, 4096, 4096, 10, 2, dim, 64, 0, 0)


def ask():
    """The workspace of such calls, over the types and head sizes and from one key to many."""
    for dim in DIMS:
        for type in TYPES:
            for length in (0, 1, 640, 1 << 20):
                v = ctypes.c_int64(-1)
                _abi.call("komp_kv_attend_workspace", ctypes.byref(descriptor(dim)), type, 4, 2, 4, 0, length, ctypes.byref(v))
                assert v.value == 0


def test_workspace_without_queries():
    """In a process of its own: a division by zero would end it."""
    r = subprocess.run([sys.executable, "-c", "from tests import test_kv_no_queries as t; t.ask()"], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


def test_attend_without_queries():
    """The call itself launches nothing and needs no workspace (there is no device here to launch on)."""
    c = ctypes.byref(descriptor())
    _abi.call("komp_kv_attend", c, 4096, 4096, None, 0, 4096, 4096, 4096, None, None, 4, 2, 4, 256, 64, 256, 64, 10, 10, 0, 640, 0.1,
              0.0, 0, None, 0, None)  # fmt: skip


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_kv_attend_without_queries(dtype):
    """Through the Python surface: preallocated results keep what they held."""
    from comp_amd import kv

    cache = kv.KVCache(4, 2, 64)
    tables = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    lengths = torch.tensor([70, 3], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda")
    q = torch.ones((4, 4, 64), dtype=dtype, device="cuda")
    out, lse = torch.full_like(q, 5.0), torch.full((4, 4), 6.0, device="cuda")
    kv.attend_into(cache, q, out, tables, lengths, starts, max_queries=0, lse=lse)
    assert (out == 5).all() and (lse == 6).all()
    got, sums = kv.attend(cache, q, tables, lengths, starts, max_queries=0, return_lse=True)
    assert got.shape == q.shape and got.dtype == dtype and sums.shape == (4, 4)
