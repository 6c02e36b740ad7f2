"""The microscaled rows' operators (comp_amd.mx) against plain 64-bit forms."""

import numpy as np
import pytest
import torch

from comp_amd import _abi, mx
from tests import mx_ref as R

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(1, 32), (2, 96), (15, 128), (16, 160), (17, 512), (33, 544), (5, 2560), (64, 1056), (300, 32), (131, 64), (70, 256), (33, 288)]


def f64(t):
    return t.detach().cpu().double().numpy()


def inputs(n, k, dtype, seed, special=True):
    """Normal values with strong columns, and blocks of every kind: zeros, infinities, NaN, tiny, large, ties, signed zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, k), generator=g) * (1 + 20 * (torch.rand(k, generator=g) < 0.03))
    if special:
        b = x.view(-1, 32)
        tiny, large = (1e-40, 3e38) if dtype != "f16" else (6e-8, 6e4)
        kinds = [lambda r: r.zero_(), lambda r: r.fill_(-0.0), lambda r: r.mul_(tiny), lambda r: r.copy_(large * torch.sign(r)),
                 lambda r: r[7].fill_(float("inf")), lambda r: r[31].fill_(float("nan")),
                 lambda r: r.copy_(torch.arange(32) * 0.25), lambda r: r[1:].zero_(), lambda r: r[0].fill_(float("-inf")),
                 lambda r: r.copy_(torch.tensor([7.9, 6.1, -6.9, 5.0, 0.25, -0.75, 1.25, 2.5] * 4))]  # fmt: skip
        for i in range(1, b.shape[0], 3):
            kinds[(i // 3 + seed) % len(kinds)](b[i])
    return x.to(DTYPES[dtype])


def strided(x, offset=1, extra=3):
    """The same values in rows with a stride of their own, from an odd element on."""
    n, k = x.shape
    buffer = torch.full((n * (k + extra) + offset + 8,), 77.0, dtype=x.dtype, device="cuda")
    view = buffer[offset : offset + n * (k + extra)].view(n, k + extra)[:, :k]
    view.copy_(x)
    return view


def plain_codes(codes, fmt):
    """uint8 plane of unpack() -> one code a byte."""
    c = codes.cpu().numpy()
    return np.stack([c & 15, c >> 4], -1).reshape(c.shape[0], -1) if fmt == "e2m1" else c


def random_rows(n, k, fmt, seed, low=110, high=130):
    """Rows of random codes and scales -> (Rows, their values in f64)."""
    g = np.random.default_rng(seed)
    codes = g.integers(0, 16 if fmt == "e2m1" else 256, (n, k), dtype=np.uint8)
    if fmt == "e4m3":
        codes[codes & 127 == 127] = 3
    scales = g.integers(low, high + 1, (n, k // 32), dtype=np.uint8)
    plane = codes[:, ::2] | codes[:, 1::2] << 4 if fmt == "e2m1" else codes
    r = mx.pack(torch.from_numpy(np.ascontiguousarray(plane)).cuda(), torch.from_numpy(scales).cuda(), fmt)
    return r, R.values(codes, scales, fmt)


def same(a, b):
    assert a.shape == b.shape
    assert np.array_equal(a, b, equal_nan=True) and np.array_equal(np.signbit(a[a == 0]), np.signbit(b[b == 0]))


# ---- rows ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_quantize(fmt, dtype, shape):
    x = inputs(*shape, dtype, shape[1] + shape[0])
    codes, scales = R.quantize(f64(x), fmt)
    for src in (x.cuda(), strided(x)):
        rows = mx.quantize(src, fmt)
        got_codes, got_scales = mx.unpack(rows)
        assert np.array_equal(got_scales.cpu().numpy(), scales)
        assert np.array_equal(plain_codes(got_codes, fmt), codes)
        same(f64(mx.values(rows)), R.values(codes, scales, fmt))


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_quantize_into_used_rows(fmt):
    """The places behind the last row and block are zeros again, whatever the planes held."""
    x = inputs(19, 160, "f32", 5).cuda()
    clean, used = mx.Rows(19, 160, fmt), mx.Rows(19, 160, fmt)
    used.codes.fill_(255)
    used.scales.fill_(255)
    mx.quantize_into(x, clean)
    mx.quantize_into(x, used)
    fresh = mx.quantize(x, fmt)
    for r in (used, fresh):
        assert torch.equal(clean.codes, r.codes) and torch.equal(clean.scales, r.scales)
    codes, scales = mx.unpack(clean)
    again = mx.pack(codes, scales, fmt)
    assert torch.equal(clean.codes, again.codes) and torch.equal(clean.scales, again.scales)


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_all_borders(fmt):
    """Every element's borders and their neighbours, at scales from the smallest to the largest."""
    _, _, high, _ = R.ELEMENTS[fmt]
    half = R.table(fmt)[: 8 if fmt == "e2m1" else 127]
    points = np.concatenate([half, (half[1:] + half[:-1]) / 2]).astype(np.float32)
    points = np.unique(np.concatenate([points, np.nextafter(points, np.float32(1e9)), np.nextafter(points, np.float32(-1))]))
    points = np.concatenate([points, -points])
    top = 2.0**high
    blocks = -(-len(points) // 31)
    x = np.zeros((blocks, 32), np.float32)
    x[:, 0] = top * 1.75
    x[:, 1:].flat[: len(points)] = points
    with np.errstate(over="ignore", under="ignore"):
        all_x = np.concatenate([(x.astype(np.float64) * 2.0**e).astype(np.float32) for e in (-149, -130, -118, -60, 0, 70, 127 - high)])
    rows = mx.quantize(torch.from_numpy(all_x).cuda(), fmt)
    same(f64(mx.values(rows)), R.kept(all_x, fmt))


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_values_of_all_codes(fmt):
    n = 16 if fmt == "e2m1" else 256
    codes = np.tile(np.arange(n, dtype=np.uint8), 256 * 32 // n if n < 32 else 256).reshape(256, -1)
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], codes.shape[1] // 32, 1)
    plane = codes[:, ::2] | codes[:, 1::2] << 4 if fmt == "e2m1" else codes
    rows = mx.pack(torch.from_numpy(np.ascontiguousarray(plane)).cuda(), torch.from_numpy(scales).cuda(), fmt)
    with np.errstate(over="ignore"):
        same(f64(mx.values(rows)), R.values(codes, scales, fmt).astype(np.float32).astype(np.float64))
    back = mx.unpack(rows)
    assert np.array_equal(back[0].cpu().numpy(), plane) and np.array_equal(back[1].cpu().numpy(), scales)


@pytest.mark.parametrize("n,k", [(1, 32), (17, 544), (40, 1024)])
def test_from_ggml(n, k):
    g = np.random.default_rng(n)
    blocks = g.integers(0, 256, (n, k // 32, 17), dtype=np.uint8)
    blocks[..., 0] = g.integers(100, 140, (n, k // 32))
    q = blocks[..., 1:]
    codes = np.concatenate([q & 15, q >> 4], -1).reshape(n, k)
    device = torch.empty(blocks.size + 1, dtype=torch.uint8, device="cuda")[1:]  # bytes at any address
    device.copy_(torch.from_numpy(blocks.reshape(-1)))
    rows = mx.from_ggml(device, n, k)
    same(f64(mx.values(rows)), R.values(codes, blocks[..., 0], "e2m1"))


@pytest.mark.parametrize("act", mx.ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_gate(fmt, dtype, act):
    for n, k in SHAPES:
        x = inputs(n, 2 * k, dtype, n + k)
        want = R.kept(R.gate(f64(x), act), fmt)
        for src in (x.cuda(), strided(x)):
            same(f64(mx.values(mx.gate(src, fmt, act))), want)
    rows = mx.Rows(n, k, fmt)
    assert mx.gate_into(x.cuda(), rows, act) is rows
    same(f64(mx.values(rows)), want)


@pytest.mark.parametrize("act", mx.ACTS)
def test_gate_far_values(act):
    """Gates from the far negative to the far positive, products next to the elements' borders."""
    g = np.concatenate([np.linspace(-120, 120, 4096), np.linspace(-1e-3, 1e-3, 2048), np.geomspace(1e-44, 1e38, 1024),
                        -np.geomspace(1e-44, 1e38, 1024)]).astype(np.float32)  # fmt: skip
    u = np.random.default_rng(1).choice(np.array([1, -1, 0.75, 1.25, 2.5, 1e-30, 1e30, 0], np.float32), g.size)
    x = np.concatenate([g.reshape(64, -1), u.reshape(64, -1)], 1)
    for fmt in mx.FORMATS:
        same(f64(mx.values(mx.gate(torch.from_numpy(x).cuda(), fmt, act))), R.kept(R.gate(x, act), fmt))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_lookup(fmt, dtype):
    for n, k, count in [(1, 32, 1), (9, 32, 700), (20, 64, 129), (37, 96, 50), (50, 256, 77), (30, 288, 33), (100, 544, 17), (16, 2560, 3)]:
        rows, want = random_rows(n, k, fmt, n, 100, 140)
        ids = np.random.default_rng(count).integers(0, n, count)
        if count > 2:
            ids[0], ids[1], ids[2] = -1, n, ids[-1]
        bad = (ids < 0) | (ids >= n)
        for scale in (1.0, 0.3, k**0.5):
            v = (want[np.where(bad, 0, ids)].astype(np.float32) * np.float32(scale)).astype(np.float32)  # rounded to f32 first
            v = f64(torch.from_numpy(np.where(bad[:, None], np.float32(0), v)).to(DTYPES[dtype]))
            got = mx.lookup(rows, torch.from_numpy(ids).cuda(), DTYPES[dtype], scale=scale)
            assert got.dtype is DTYPES[dtype]
            same(f64(got), v)
            guard = torch.full((count, k + 5), 7.0, dtype=DTYPES[dtype], device="cuda")
            mx.lookup_into(rows, torch.from_numpy(ids).cuda(), guard[:, 3 : 3 + k], scale=scale)
            same(f64(guard[:, 3 : 3 + k]), v)
            assert bool((guard[:, :3] == 7).all()) and bool((guard[:, 3 + k :] == 7).all())
    assert mx.lookup(rows, torch.empty(0, dtype=torch.int64, device="cuda")).shape == (0, k)
    assert mx.lookup(rows, torch.tensor([-1], device="cuda"), DTYPES[dtype], scale=float("inf")).abs().max() == 0


@pytest.mark.parametrize("act", mx.ACTS)
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_gate_many(fmt, act):
    """A million products of one block's magnitudes: the blocks whose elements lie next to a border take the 64-bit path."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((512, 2 * 2048), generator=g, device="cuda") * torch.exp2(torch.randint(-8, 9, (512, 1), generator=g, device="cuda"))
    same(f64(mx.values(mx.gate(x, fmt, act))), R.kept(R.gate(f64(x), act), fmt))


# ---- products --------------------------------------------------------------------------------------------------------

PRODUCTS = [(1, 1, 32), (1, 16, 128), (2, 17, 96), (3, 100, 160), (16, 33, 512), (17, 48, 544), (31, 5, 1056), (33, 64, 2560),
            (64, 200, 640), (65, 130, 1024), (100, 257, 96), (130, 300, 1312), (257, 129, 4096), (5, 700, 14336), (3, 40, 20000), (40, 33, 20000), (300, 1100, 1024),
            (1100, 300, 320)]  # fmt: skip


def check_product(y, x, w, fmt, dtype):
    want, bound = R.product_bound(x, w, fmt, dtype)
    off = np.abs(f64(y) - want)
    assert np.isfinite(off).all() and (off <= bound).all(), f"{(off / bound).max()} of the bound"


@pytest.mark.parametrize("shape", PRODUCTS, ids=str)
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_gemm(fmt, shape):
    t, n, k = shape
    x, xv = random_rows(t, k, fmt, 1)
    w, wv = random_rows(n, k, "e2m1", 2)
    for dtype in DTYPES:
        if dtype == "f16":  # what f16 holds
            x, xv = random_rows(t, k, fmt, 3, 110, 120)
        y = mx.gemm(x, w, DTYPES[dtype])
        assert y.dtype is DTYPES[dtype]
        check_product(y, xv, wv, fmt, dtype)
        guard = torch.full((t, n + 7), 5.0, dtype=DTYPES[dtype], device="cuda")
        mx.gemm_into(x, w, guard[:, 2 : 2 + n])
        assert torch.equal(guard[:, 2 : 2 + n], y)
        assert bool((guard[:, :2] == 5).all()) and bool((guard[:, 2 + n :] == 5).all())


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_gemm_places(fmt):
    """One element of a row and one of a column at a time: every place of K meets its own partner."""
    k = 672
    eye = np.zeros((k, k), np.float32)
    np.fill_diagonal(eye, 1.0)
    w = mx.quantize(torch.from_numpy(eye).cuda(), "e2m1")
    x, xv = random_rows(40, k, fmt, 4, 127, 127)
    for t in (3, 20, 40):
        part = mx.quantize(torch.from_numpy(xv[:t].astype(np.float32)).cuda(), fmt)
        same(f64(mx.gemm(part, w)) + 0.0, R.kept(xv[:t], fmt) + 0.0)
    big = mx.quantize(torch.from_numpy(np.tile(xv, (4, 1)).astype(np.float32)).cuda(), fmt)
    same(f64(mx.gemm(big, w)) + 0.0, R.kept(np.tile(xv, (4, 1)), fmt) + 0.0)


@pytest.mark.parametrize("t", [1, 20, 100])
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_gemm_special(fmt, t):
    """Scales from end to end, NaN blocks: each reaches its own row and column alone."""
    k, n = 256, 50
    g = np.random.default_rng(3)
    xc, wc = g.integers(0, 8 if fmt == "e2m1" else 120, (t, k), dtype=np.uint8), g.integers(0, 16, (n, k), dtype=np.uint8)
    xs, ws = np.full((t, k // 32), 127, np.uint8), np.full((n, k // 32), 127, np.uint8)
    ws[:10], xs[:, 1] = 1, 250  # 2^-126 times 2^123
    ws[10:20, 2] = 20
    ws[20, 3] = 255
    if t > 1:
        xs[1, 5] = 255
    low = lambda c: np.ascontiguousarray(c[:, ::2] | c[:, 1::2] << 4)  # noqa: E731
    put = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    x = mx.pack(put(low(xc) if fmt == "e2m1" else xc), put(xs), fmt)
    w = mx.pack(put(low(wc)), put(ws))
    # values and sums are f32's: past its largest they are infinite (values of e4m3; e2m1's are not formed), and where the
    # magnitudes add up to more, a sum may pass it on its way
    xv, wv = R.values(xc, xs, fmt), R.values(wc, ws, "e2m1")
    with np.errstate(all="ignore"):
        if fmt == "e4m3":
            xv = xv.astype(np.float32).astype(np.float64)
        y, largest = f64(mx.gemm(x, w)), float(np.finfo(np.float32).max)
        want, bound = R.product_bound(xv, wv, fmt, "f32")
        most = np.abs(xv) @ np.abs(wv).T
        assert np.array_equal(np.isnan(y)[:, 20], np.full(t, True)) and np.isnan(y)[np.isnan(most)].all()
        inside = most < largest
        assert (inside.any() or fmt == "e4m3") and (np.abs(y - want)[inside] <= bound[inside]).all()
        past = np.isfinite(most) & (np.abs(want) - bound > largest)
        assert (y[past] == np.sign(want[past]) * np.inf).all()
        between = ~np.isnan(most) & ~inside & ~past
        assert (~np.isfinite(y[between]) | (np.abs(y - want)[between] <= bound[between])).all()


@pytest.mark.parametrize("t", [1, 20, 100])
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_gemm_far_scales(fmt, t):
    """Large activations times small weights and the other way round: the powers meet in the product."""
    x, xv = random_rows(t, 256, fmt, 1, 236, 240)
    w, wv = random_rows(50, 256, "e2m1", 2, 6, 14)
    check_product(mx.gemm(x, w), xv, wv, fmt, "f32")
    x, xv = random_rows(t, 256, fmt, 1, 20, 30)
    w, wv = random_rows(50, 256, "e2m1", 2, 230, 236)
    check_product(mx.gemm(x, w), xv, wv, fmt, "f32")


@pytest.mark.parametrize("shape", [(1, 1, 32), (1, 700, 2560), (2, 33, 544), (7, 64, 4096), (16, 50, 96), (5, 17, 14336), (17, 40, 160), (3, 40, 20000), (16, 300, 8192),
                                   (70, 300, 1024)], ids=str)  # fmt: skip
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_linear(fmt, dtype, shape):
    """Equal to quantize and gemm bit for bit, and to the definition within its bound."""
    t, n, k = shape
    x = inputs(t, k, dtype, 11, special=False)
    w, wv = random_rows(n, k, "e2m1", 12, 117, 122)
    for out in DTYPES:
        y = mx.linear(x.cuda(), w, fmt, DTYPES[out])
        assert torch.equal(y, mx.gemm(mx.quantize(x.cuda(), fmt), w, DTYPES[out]))
        assert torch.equal(y, mx.linear(strided(x), w, fmt, DTYPES[out]))
        guard = torch.full((t, n + 3), 5.0, dtype=DTYPES[out], device="cuda")
        mx.linear_into(x.cuda(), w, guard[:, 1 : 1 + n], fmt)
        assert torch.equal(guard[:, 1 : 1 + n], y) and bool((guard[:, 0] == 5).all()) and bool((guard[:, 1 + n :] == 5).all())
        check_product(y, R.kept(f64(x), fmt), wv, fmt, out)
    assert mx.linear(x.cuda(), w, fmt).dtype is DTYPES[dtype]


@pytest.mark.parametrize("t,k", [(5, 9216), (16, 4096), (16, 14336), (16, 20000)])
@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_linear_one_launch(fmt, t, k):
    """The C entry on rows that linear() gives two launches."""
    x = inputs(t, k, "bf16", 2, special=False).cuda()
    w, _ = random_rows(50, k, "e2m1", 3)
    y = torch.zeros(t, 50, device="cuda")
    _abi.call("komp_mx_linear", x.data_ptr(), 2, k, t, mx.FORMATS[fmt], w._ref, y.data_ptr(), 0, 50, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(y, mx.linear(x, w, fmt, torch.float32))


def test_linear_special():
    x = inputs(9, 1056, "f32", 3).cuda()
    w, _ = random_rows(65, 1056, "e2m1", 12)
    for fmt in mx.FORMATS:
        a, b = mx.linear(x, w, fmt), mx.gemm(mx.quantize(x, fmt), w)
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0), b.nan_to_num(0)) and bool(a.isnan().any())


def test_empty():
    w = mx.Rows(0, 64)
    assert mx.linear(torch.zeros(3, 64, device="cuda"), w).shape == (3, 0)
    w, _ = random_rows(5, 64, "e2m1", 1)
    assert mx.linear(torch.zeros(0, 64, device="cuda"), w).shape == (0, 5)
    assert mx.gemm(mx.quantize(torch.zeros(0, 64, device="cuda"), "e4m3"), w).shape == (0, 5)
    assert mx.values(mx.Rows(0, 32)).shape == (0, 32) and mx.unpack(mx.Rows(0, 32))[0].shape == (0, 16)
    assert float(mx.values(mx.Rows(20, 64, "e4m3")).abs().max()) == 0


def test_refusals_on_a_device():
    x, w = torch.zeros(4, 64, device="cuda"), mx.Rows(8, 64)
    y = torch.zeros(4, 8, device="cuda")
    q = mx.quantize(x, "e4m3")
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in [lambda: mx.quantize(x.double()), lambda: mx.quantize(x[:, ::2]), lambda: mx.quantize(x[0]), lambda: mx.quantize(x[:, :40]),
                 lambda: mx.quantize_into(x, mx.Rows(5, 64)), lambda: mx.quantize_into(x, mx.Rows(4, 32)), lambda: mx.gate(x[:, :33]),
                 lambda: mx.gate(x, "fp4"), lambda: mx.gate_into(x, q), lambda: mx.lookup(w, ids.int()), lambda: mx.lookup(w, ids.cpu()),
                 lambda: mx.lookup(w, ids, torch.float64), lambda: mx.lookup_into(w, ids, x[:3]), lambda: mx.values(w, torch.int8),
                 lambda: mx.gemm(q, q), lambda: mx.gemm(q, mx.Rows(8, 96)), lambda: mx.gemm(q, w, torch.float64),
                 lambda: mx.gemm_into(q, w, y[:, :7]), lambda: mx.gemm_into(q, w, y.t()), lambda: mx.gemm_into(q, w, y[:1].expand(4, 8)),
                 lambda: mx.gemm_into(q, w, y.cpu()), lambda: mx.linear(x, w, "fp8"), lambda: mx.linear(x[:, :32], w), lambda: mx.linear(x, q),
                 lambda: mx.linear_into(x, w, y.int()), lambda: mx.linear_into(x, w, y[:3]), lambda: mx.linear(x, w, dtype=torch.int32),
                 lambda: mx.pack(x.byte(), x.byte()[:, :2], "e4m3"), lambda: mx.pack(x.byte(), x[:, :2].byte().contiguous(), "e2m1"),
                 lambda: mx.from_ggml(x.byte(), 4, 64)]:  # fmt: skip
        with pytest.raises(_abi.KompArgumentError):
            call()


# ---- together --------------------------------------------------------------------------------------------------------


class Layer:
    """An embedding, a gated feed-forward layer and the product over the embedding's table again."""

    def __init__(self, vocabulary=300, width=160, inner=224):
        g = torch.Generator().manual_seed(8)
        weight = lambda n, k: torch.randn((n, k), generator=g) * k**-0.5  # noqa: E731
        self.plain = [f64(weight(vocabulary, width) * 8), f64(weight(2 * inner, width)), f64(weight(width, inner))]
        self.table, self.up, self.down = (mx.quantize(torch.from_numpy(p).float().cuda()) for p in self.plain)
        self.plain = [R.kept(p.astype(np.float32), "e2m1") for p in self.plain]

    def run(self, ids, dtype):
        x = mx.lookup(self.table, ids, dtype, scale=0.5)
        h = mx.gate(mx.linear(x, self.up, "e4m3", torch.float32), "e4m3")
        x = mx.gemm(h, self.down, dtype)
        return x, mx.linear(x, self.table, "e2m1", torch.float32)


@pytest.mark.parametrize("t", [1, 5, 40, 90])
def test_layer(t):
    """Each operator's result against the definition over what the one before it gave."""
    layer = Layer()
    ids = torch.from_numpy(np.random.default_rng(t).integers(0, 300, t)).cuda()
    x = mx.lookup(layer.table, ids, torch.float32, scale=0.5)
    same(f64(x), layer.plain[0][ids.cpu().numpy()] * 0.5)
    up = mx.linear(x, layer.up, "e4m3")
    check_product(up, R.kept(f64(x), "e4m3"), layer.plain[1], "e4m3", "f32")
    h = mx.gate(up, "e4m3")
    inner = R.kept(R.gate(f64(up), "silu"), "e4m3")
    same(f64(mx.values(h)), inner)
    y = mx.gemm(h, layer.down)
    check_product(y, inner, layer.plain[2], "e4m3", "f32")
    logits = mx.linear(y, layer.table, "e2m1")
    check_product(logits, R.kept(f64(y), "e2m1"), layer.plain[0], "e2m1", "f32")
    a, b = layer.run(ids, torch.float32)
    assert torch.equal(a, y) and torch.equal(b, logits)


@pytest.mark.parametrize("t", [1, 5, 70])
def test_graph(t):
    """The run captured once and replayed with other ids, eager work between the replays."""
    layer = Layer()
    ids = torch.zeros(t, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.run(ids, torch.bfloat16)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.run(ids, torch.bfloat16)
    for seed in range(4):
        ids.copy_(torch.from_numpy(np.random.default_rng(seed).integers(0, 300, t)))
        graph.replay()
        got = [o.clone() for o in out]
        want = layer.run(ids, torch.bfloat16)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_streams():
    """Calls on two streams at once, each with its own rows."""
    layer = Layer()
    ids = [torch.from_numpy(np.random.default_rng(s).integers(0, 300, 20)).cuda() for s in range(2)]
    want = [layer.run(i, torch.float32) for i in ids]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                got[s] = layer.run(ids[s], torch.float32)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_past_32_bits():
    """Planes of more than 2^32 bytes: the last rows are read, written and multiplied."""
    n, k = 2_200_003, 4096
    scales = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    codes = torch.empty((n, k // 2), dtype=torch.uint8, device="cuda")
    codes.random_(0, 256)
    w = mx.pack(codes, scales)
    assert w.codes.numel() > 1 << 32
    tail = codes[-40:].cpu().numpy()
    tail = np.stack([tail & 15, tail >> 4], -1).reshape(40, k)
    wv = R.values(tail, np.full((40, k // 32), 127, np.uint8), "e2m1")
    ids = torch.arange(n - 40, n, device="cuda")
    same(f64(mx.lookup(w, ids)), wv)
    got = mx.unpack(w)[0]
    assert torch.equal(got[-1000:], codes[-1000:])
    del got
    x = inputs(3, k, "f32", 1, special=False)
    for fmt in mx.FORMATS:
        check_product(mx.linear(x.cuda(), w, fmt)[:, -40:], R.kept(f64(x), fmt), wv, fmt, "f32")
    many = inputs(70, k, "f32", 1, special=False)
    y = mx.linear(many.cuda(), w, "e2m1", torch.bfloat16)
    check_product(y[:, -40:], R.kept(f64(many), "e2m1"), wv, "e2m1", "bf16")
