"""Microscaled rows: 4- and 8-bit floating point elements with a power of two a block of 32, and the products over them.

Beside the integer formats of comp_amd.host: weights in e2m1 (4.25 bits an element, the format MXFP4 of the OCP microscaling
standard and of ggml's block_mxfp4), which the CDNA4 matrix cores multiply as they are, and activations in e2m1 or e4m3.

    w = quantize(weight, "e2m1")                 # weight [N][K] f32, f16 or bf16 -> Rows; or from_ggml(), pack()
    y = linear(x, w)                              # x [T][K] of floats, quantized on the way: decode steps in one launch
    y = gemm(quantize(x, "e4m3"), w)              # the same in two steps, for rows that several products share
    h = gate(y, "e4m3")                           # y [T][2 K] = gate | up -> Rows of silu(gate) * up, for the next product
    e = lookup(table, ids)                        # rows of a quantized table: the embedding

An element is a sign, 2 exponent and 1 mantissa bits (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6) or 4 and 3 (e4m3: up to 448).  A block's
scale is 2^(floor(log2(largest magnitude)) - 2) for e2m1 and - 8 for e4m3 (2^-127 at least); elements are rounded to the nearest,
ties to even, and saturate.  A block that holds an infinity or a NaN is NaN throughout.

As in comp_amd.host, tensors live on a HIP device, calls run on the current torch stream without synchronising, wrong
arguments raise KompArgumentError before anything is launched, and the *_into forms allocate no result.  What is written must not
overlap what the same call reads: no call works in place.  There are no gradients.
No reference counterpart.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _abi
from .host import _current_device, _need, _raw_stream

_Tensor, _I64, _U8 = torch.Tensor, torch.int64, torch.uint8

FORMATS = {"e2m1": 0, "e4m3": 1}
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ACTS = {"silu": 1, "relu2": 2}
LINEAR_ROWS = 16  # rows that linear() quantizes and multiplies in one launch,
LINEAR_VALUES = 98304  # of fewer values than these in all
MAX_ROWS, MAX_WEIGHTS = (1 << 20) - 16, 1 << 26  # of one product
_BAD = _abi.KompArgumentError
_new = object.__new__


class Rows:
    """`rows` rows of k elements (a multiple of 32) in the format "e2m1" or "e4m3", zeros at first.

    codes and scales are the planes; the order of their bytes is the library's own (include/komp_abi.h): quantize(), gate(),
    pack() and from_ggml() write rows, values(), lookup() and unpack() read them."""

    def __init__(self, rows, k, fmt="e2m1", device="cuda"):
        if torch.device(device).type != "cuda":
            raise _BAD(f"Rows: {device}: the rows live on a HIP device")
        sizes = _plane_sizes(rows, k, fmt)
        self._hold(rows, k, fmt, sizes, torch.zeros(sizes[2], dtype=_U8, device=device))

    def _hold(self, rows, k, fmt, sizes, planes):
        # (one allocation for both planes: an eager call is mostly host time)
        self.rows, self.k, self.fmt = rows, k, fmt
        self._planes, self._sizes, self._device = planes, sizes, planes.get_device()
        at = planes.data_ptr()
        self._struct = _abi.MxRowsStruct(at, at + sizes[0], rows, k, FORMATS[fmt])
        self._ref = ctypes.addressof(self._struct)

    @property
    def codes(self):
        return self._planes[: self._sizes[0]].view(-(-self.rows // 16), -1) if self.rows else self._planes.view(0, 0)

    @property
    def scales(self):
        return self._planes[self._sizes[0] :].view(-(-self.rows // 16), -1) if self.rows else self._planes.view(0, 0)

    @property
    def device(self):
        return self._planes.device

    def nbytes(self):
        """Bytes of the two planes."""
        return self._sizes[2]


def _need_format(fmt):
    if fmt not in FORMATS:
        raise _BAD(f"fmt={fmt!r}: one of {tuple(FORMATS)}")


@functools.lru_cache(maxsize=4096)
def _plane_sizes(rows, k, fmt):
    """(bytes of the codes, of the scales, of both)."""
    _need_format(fmt)
    if k < 32 or k % 32 or k > 1 << 26:
        raise _BAD(f"k={k} must be a multiple of 32, from 32 to 2^26")
    tiles, pieces = -(-rows // 16), -(-k // 512)
    if rows < 0 or rows > 0x7FFFFFFF or tiles * pieces > 0x7FFFFFFF:
        raise _BAD(f"{rows} rows of {k} elements")
    codes, scales = tiles * -(-k // 128) * (1024 << FORMATS[fmt]), tiles * pieces * 256
    return codes, scales, codes + scales


def _empty(like, rows, k, fmt):
    """Rows that the next launch writes, places behind the last row and block too."""
    sizes = _plane_sizes(rows, k, fmt)
    r = _new(Rows)
    r._hold(rows, k, fmt, sizes, like.new_empty(sizes[2], dtype=_U8))
    return r


def _launch(name, dev, *args):
    """Call a launching ABI entry on device `dev`, with that device's current stream as its last argument."""
    fn = getattr(_abi._lib or _abi.lib(), name)
    if dev == _current_device():
        st = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, _raw_stream(dev))
    if st:
        _abi.check(st, name)


def _need_rows(r, name):
    if not isinstance(r, Rows):
        raise TypeError(f"{name} must be Rows, got {type(r).__name__}")


def _need_matrix(t, name, cols=None, device=None, rows=None, output=False):
    """A [rows][cols] tensor of a float type whose rows are contiguous (and, to be written, apart)."""
    if (isinstance(t, _Tensor) and t.is_cuda and t.dtype in TYPES and t.dim() == 2 and t.stride(1) == 1
            and (cols is None or t.shape[1] == cols) and (rows is None or t.shape[0] == rows)
            and (device is None or t.get_device() == device)
            and not (output and t.stride(0) < t.shape[1] and t.shape[0] > 1)):  # fmt: skip
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise _BAD(f"{name} is on {t.device}: the operators run on a HIP device only")
    if t.dtype not in TYPES:
        raise _BAD(f"{name} must be f32, f16 or bf16, got {t.dtype}")
    if t.dim() != 2 or (cols is not None and t.shape[1] != cols) or (rows is not None and t.shape[0] != rows):
        raise _BAD(f"{name} must be [{'rows' if rows is None else rows}][{'K' if cols is None else cols}], got {tuple(t.shape)}")
    if device is not None and t.get_device() != device:
        raise _BAD(f"{name} is on {t.device}, the rows on cuda:{device}")
    if t.numel() and t.shape[1] > 1 and t.stride(1) != 1:
        raise _BAD(f"{name}: a row must be contiguous (stride(1) == 1)")
    if output and t.numel() and t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise _BAD(f"{name}: rows overlap (stride(0) = {t.stride(0)})")


def _need_bytes(t, name, shape, device=None):
    """A contiguous uint8 tensor of this shape."""
    _need(t, name, _U8)
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise _BAD(f"{name} must be a contiguous {list(shape)} tensor, got {tuple(t.shape)}")
    if device is not None and t.get_device() != device:
        raise _BAD(f"{name} is on {t.device}, the rows on cuda:{device}")


def _plain(t):
    """The tensor as a plain one: new_empty makes tensors of its argument's type."""
    return t if type(t) is _Tensor else t.as_subclass(_Tensor)


# ---- rows ------------------------------------------------------------------------------------------------------------


def _quantize(x, rows, act):
    _launch("komp_mx_quantize", rows._device, rows._ref, x.data_ptr(), TYPES[x.dtype], x.stride(0), act)
    return rows


def quantize_into(x, rows):
    """quantize() into Rows of x's shape.  Returns them."""
    _need_rows(rows, "rows")
    _need_matrix(x, "x", rows.k, rows._device, rows.rows)
    return _quantize(x, rows, 0)


def quantize(x, fmt="e2m1"):
    """x [R][K] (f32, f16 or bf16; rows contiguous, any stride between them) -> Rows of the format "e2m1" or "e4m3"."""
    _need_matrix(x, "x")
    return _quantize(x, _empty(_plain(x), x.shape[0], x.shape[1], fmt), 0)


def _act(act):
    if act not in ACTS:
        raise _BAD(f"act={act!r}: one of {tuple(ACTS)}")
    return ACTS[act]


def gate_into(x, rows, act="silu"):
    """gate() into Rows of R rows of K elements.  Returns them."""
    number = _act(act)
    _need_rows(rows, "rows")
    _need_matrix(x, "x", 2 * rows.k, rows._device, rows.rows)
    return _quantize(x, rows, number)


def gate(x, fmt="e4m3", act="silu"):
    """x [R][2 K] = [g | u] (f32, f16 or bf16; rows contiguous, any stride between them) -> Rows of silu(g) * u, with act "relu2"
    of max(g, 0)^2 * u: the step between the two products of a gated feed-forward layer.

    The product is that of the exact values, rounded to f32 once (silu(g) = g / (1 + e^-g)); its quantization is quantize()'s."""
    number = _act(act)
    _need_matrix(x, "x")
    if x.shape[1] % 2:
        raise _BAD(f"x must be [R][2 K], got {tuple(x.shape)}")
    return _quantize(x, _empty(_plain(x), x.shape[0], x.shape[1] // 2, fmt), number)


def _need_ids(ids, rows):
    _need(ids, "ids", _I64, 1)
    if not ids.is_contiguous() or ids.get_device() != rows._device:
        raise _BAD(f"ids must be a contiguous tensor on {rows.device}")


def lookup_into(rows, ids, out, scale=1.0):
    """lookup() into out [T][K] (f32, f16 or bf16; rows contiguous, any stride between them that keeps them apart)."""
    _need_rows(rows, "rows")
    _need_ids(ids, rows)
    _need_matrix(out, "out", rows.k, rows._device, ids.shape[0], output=True)
    _launch("komp_mx_lookup", rows._device, rows._ref, ids.data_ptr(), ids.shape[0], out.data_ptr(), TYPES[out.dtype],
            out.stride(0), scale)  # fmt: skip


def _type(dtype):
    if dtype not in TYPES:
        raise _BAD(f"dtype must be f32, f16 or bf16, got {dtype}")
    return TYPES[dtype]


def lookup(rows, ids, dtype=torch.float32, scale=1.0):
    """The rows ids (int64 [T]) as values [T][K] of dtype, each times `scale` in f32 and rounded to dtype: the embedding of a
    quantized table.  The ids are checked on the device: one outside the table gives zeros."""
    _need_rows(rows, "rows")
    _need_ids(ids, rows)
    number = _type(dtype)
    out = rows._planes.new_empty((ids.shape[0], rows.k), dtype=dtype)
    _launch("komp_mx_lookup", rows._device, rows._ref, ids.data_ptr(), ids.shape[0], out.data_ptr(), number, rows.k, scale)
    return out


def values(rows, dtype=torch.float32):
    """All rows as values [rows][K] of dtype.  f32 holds every value below 2^128, bf16 those of magnitude 2^-126 and more exactly;
    past that, which only pack() and from_ggml() bring (scale bytes from 253 on in e2m1, from 247 on in e4m3), they are infinite."""
    _need_rows(rows, "rows")
    number = _type(dtype)
    out = rows._planes.new_empty((rows.rows, rows.k), dtype=dtype)
    _launch("komp_mx_lookup", rows._device, rows._ref, None, rows.rows, out.data_ptr(), number, rows.k, 1.0)
    return out


def pack(codes, scales, fmt="e2m1"):
    """Rows from plain planes on the device: codes uint8 [R][K / 2] (e2m1: element 2 j in the low, 2 j + 1 in the high nibble of
    byte j) or [R][K] (e4m3), scales uint8 [R][K / 32]."""
    _need_format(fmt)
    _need(scales, "scales", _U8, 2)
    n, k = scales.shape[0], scales.shape[1] * 32
    _need_bytes(scales, "scales", scales.shape)
    _need_bytes(codes, "codes", (n, k // 2 if fmt == "e2m1" else k), scales.get_device())
    rows = _empty(_plain(scales), n, k, fmt)
    _launch("komp_mx_pack", rows._device, rows._ref, codes.data_ptr(), scales.data_ptr())
    return rows


def unpack(rows):
    """Rows -> (codes, scales), the plain planes that pack() takes."""
    _need_rows(rows, "rows")
    codes = rows._planes.new_empty((rows.rows, rows.k // 2 if rows.fmt == "e2m1" else rows.k))
    scales = rows._planes.new_empty((rows.rows, rows.k // 32))
    _launch("komp_mx_unpack", rows._device, rows._ref, codes.data_ptr(), scales.data_ptr())
    return codes, scales


def from_ggml(W, n, k):
    """Rows from ggml block_mxfp4 blocks on the device: W uint8, n rows of k / 32 blocks of 17 bytes (for example a GGUF tensor's
    raw bytes), contiguous."""
    _need(W, "W", _U8)
    _plane_sizes(n, k, "e2m1")
    if W.numel() != n * (k // 32) * 17 or not W.is_contiguous():
        raise _BAD(f"W must be {n * (k // 32) * 17} contiguous bytes, got {W.numel()}")
    rows = _empty(_plain(W), n, k, "e2m1")
    _launch("komp_mx_pack", rows._device, rows._ref, W.data_ptr(), None)
    return rows


# ---- products --------------------------------------------------------------------------------------------------------


def _need_weights(w, k, device, t):
    _need_rows(w, "w")
    if w.fmt != "e2m1" or w.k != k or w._device != device:
        raise _BAD(f"w must be e2m1 rows of {k} elements on cuda:{device}, got {w.fmt} rows of {w.k} on {w.device}")
    if t > MAX_ROWS or w.rows > MAX_WEIGHTS:
        raise _BAD(f"{t} x {w.rows} results (2^20 - 16 rows of x and 2^26 of w at most)")


def _gemm(x, w, y, stride):
    _launch("komp_mx_gemm", w._device, x._ref, w._ref, y.data_ptr(), TYPES[y.dtype], stride)


def gemm_into(x, w, y):
    """gemm() into y [T][N] (f32, f16 or bf16; rows contiguous, any stride between them that keeps them apart)."""
    _need_rows(x, "x")
    _need_weights(w, x.k, x._device, x.rows)
    _need_matrix(y, "y", w.rows, x._device, x.rows, output=True)
    _gemm(x, w, y, y.stride(0))


def gemm(x, w, dtype=torch.float32):
    """x Rows [T][K] (e2m1 or e4m3) times w Rows [N][K] (e2m1) -> Y [T][N] of dtype: the sums over K of the products of what the
    elements stand for, in f32, rounded once.  T up to 2^20 - 16, N up to 2^26; the order of the sums depends on the sizes alone.

    In products with e4m3 rows both operands' values are bf16's, which is exact but at the ends: elements of rows with scale bytes 0 to 2
    are rounded to multiples of 2^-133, and weights and rows past f32's largest (see values()) are infinite, so that sums with them
    are infinite or NaN.  Products of e2m1 rows have no such ends."""
    _need_rows(x, "x")
    _need_weights(w, x.k, x._device, x.rows)
    _type(dtype)
    y = w._planes.new_empty((x.rows, w.rows), dtype=dtype)
    _gemm(x, w, y, w.rows)
    return y


def _linear(x, w, y, fmt):
    t = x.shape[0]
    # Each workgroup of the one launch quantizes all rows; two launches cost an eager call 15 us of host time in all.  One launch and two,
    # in a graph, to e4m3 (us): 16 rows through 4096 x 14336 27.5 and 14.7, 8 rows 19.1 and 14.8, 5 rows 16.3 and 14.7, 2 rows 12.7 and
    # 14.7; 16 rows through 4096 x 8192 15.0 and 10.8, through 14336 x 4096 14.3 and 13.3.
    if t > LINEAR_ROWS or t * w.k >= LINEAR_VALUES:
        rows = _empty(w._planes, t, w.k, fmt)  # kept until the calls are on the stream; torch hands it to later work of this stream
        _quantize(x, rows, 0)
        _gemm(rows, w, y, y.stride(0))
    else:
        _launch("komp_mx_linear", w._device, x.data_ptr(), TYPES[x.dtype], x.stride(0), t, FORMATS[fmt], w._ref, y.data_ptr(),
                TYPES[y.dtype], y.stride(0))  # fmt: skip


def linear_into(x, w, y, fmt="e4m3"):
    """linear() into y [T][N] (f32, f16 or bf16; rows contiguous, any stride between them that keeps them apart).  (Rows that
    take two launches still take a workspace for their quantized form from torch.)"""
    _need_format(fmt)
    _need_rows(w, "w")
    _need_matrix(x, "x", w.k, w._device)
    _need_weights(w, w.k, w._device, x.shape[0])
    _need_matrix(y, "y", w.rows, w._device, x.shape[0], output=True)
    _linear(x, w, y, fmt)


def linear(x, w, fmt="e4m3", dtype=None):
    """x [T][K] (f32, f16 or bf16; rows contiguous, any stride between them), quantized to fmt, times w Rows [N][K] (e2m1) -> Y
    [T][N] of dtype (x's by default).  Equal to gemm(quantize(x, fmt), w, dtype) bit for bit; up to LINEAR_ROWS rows of fewer
    than LINEAR_VALUES values in all take one launch.  T and N as gemm()'s."""
    _need_format(fmt)
    _need_rows(w, "w")
    _need_matrix(x, "x", w.k, w._device)
    _need_weights(w, w.k, w._device, x.shape[0])
    dtype = x.dtype if dtype is None else dtype
    _type(dtype)
    y = w._planes.new_empty((x.shape[0], w.rows), dtype=dtype)
    _linear(x, w, y, fmt)
    return y
