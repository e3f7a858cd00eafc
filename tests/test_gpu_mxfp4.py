"""MXFP4 on the GPU (ehip_mxfp4_*) against its definition in 64 bits
(mx_util). Quantisation and the panel layout are exact. Products: the codes'
products are exact and the sums fp32, so with k additions of at most one
unit in the last place each (2^-23) an element is within k 2^-23 sum |x||w|,
and independent roundings give sqrt(k) 2^-23 in the 2-norm; sums that fit in
24 bits are exact."""
import numpy as np
import pytest

import mx_util as mx

pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (1, 32), (3, 31), (16, 128), (17, 129), (33, 545), (5, 1000), (40, 2100)]


def _free(*bufs):
    for b in bufs:
        if b is not None:
            b.free()


def _bits(x, dtype):
    """(array for the device, its values) in the type."""
    if dtype == "f32":
        x = np.asarray(x, np.float32)
        return x, x
    if dtype == "f16":
        x = np.asarray(x, np.float16)
        return x.view(np.uint16), x
    b = (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
    return b, (b.astype(np.uint32) << 16).view(np.float32)


def _code(ehip_mod, dtype):
    return {"f32": ehip_mod.WEIGHT_F32, "bf16": ehip_mod.WEIGHT_BF16,
            "f16": ehip_mod.WEIGHT_F16}[dtype]


def _panel_buffers(gctx, ehip_mod, rows, k):
    c, s = ehip_mod.mxfp4_panel_bytes(rows, k)
    bufs = gctx.alloc(c), gctx.alloc(s)
    for b in bufs:
        b.upload(np.full(b.nbytes, 0xAB, np.uint8))
    return bufs


def _quantize(gctx, ehip_mod, x, dtype="f32"):
    raw, _ = _bits(x, dtype)
    rows, k = raw.shape
    dx = gctx.to_device(raw)
    codes, scales = _panel_buffers(gctx, ehip_mod, rows, k)
    assert gctx.mxfp4_quantize(dx, _code(ehip_mod, dtype), rows, k, codes, scales) == 0, \
        gctx.last_error()
    gctx.sync()
    dx.free()
    return codes, scales


def _upload(gctx, codes, scales):
    return tuple(gctx.to_device(a) for a in mx.panels_of(codes, scales))


def _check_panels(codes, scales, want):
    """Bytes equal, but for the sign of zero codes."""
    got = (codes.download(np.uint8, want[0].shape), scales.download(np.uint8, want[1].shape))
    assert np.array_equal(got[1], want[1])

    def halves(a):
        h = np.stack([a & 15, a >> 4])
        return np.where(h == 8, 0, h)

    assert np.array_equal(halves(got[0]), halves(want[0]))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,k", SIZES)
def test_quantize_is_exact(gctx, ehip_mod, rows, k, dtype):
    rng = np.random.default_rng(rows * k)
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-12, 12, (rows, 1)))
    # On the grid's midpoints and beside them, where rounding decides.
    x[rng.random((rows, k)) < 0.5] = rng.choice(np.concatenate([mx.MID, mx.GRID, [7.99, 5.01]]))
    raw, val = _bits(x, dtype)
    codes, scales = _quantize(gctx, ehip_mod, x, dtype)
    _check_panels(codes, scales, mx.panels(*mx.quantize(val.astype(np.float64))))
    y = gctx.alloc(rows * k * 4)
    assert gctx.mxfp4_dequantize(codes, scales, rows, k, y) == 0, gctx.last_error()
    gctx.sync()
    assert np.array_equal(y.download(np.float32, (rows, k)), mx.quantized(val.astype(np.float64)))
    _free(codes, scales, y)


def test_quantize_rounds_every_neighbour(gctx, ehip_mod):
    """Every midpoint and grid value, their fp32 neighbours and both signs, at
    block exponents over fp32's whole range."""
    base = np.concatenate([mx.MID, mx.GRID, [6.5, 7.0]]).astype(np.float32)
    v = np.concatenate([base, np.nextafter(base, np.float32(9)), np.nextafter(base, np.float32(-9))])
    v = np.concatenate([v, -v])
    rows = np.arange(-126, 126)
    x = np.zeros((len(rows), -(-len(v) // 31) * 32), np.float64)
    for i, e in enumerate(rows):
        for j in range(0, len(v), 31):
            part = v[j:j + 31].astype(np.float64) * 2.0**e
            at = j // 31 * 32
            x[i, at] = 6 * 2.0**e  # holds the block's scale
            x[i, at + 1:at + 1 + len(part)] = part
    x = x.astype(np.float32)
    codes, scales = _quantize(gctx, ehip_mod, x)
    _check_panels(codes, scales, mx.panels_of(*mx.quantize(x.astype(np.float64))))
    _free(codes, scales)


def test_quantize_extremes(gctx, ehip_mod):
    x = np.zeros((20, 96), np.float32)
    x[1, 3], x[2, 40], x[3, 95] = np.nan, np.inf, -np.inf
    x[4, 0], x[5, 1], x[6, 2] = 2.0**-149, 2.0**-128, 2.0**-126
    x[7, 0], x[8, 0], x[9, :] = 3.4e38, -2.0**127, np.float32(1.1754942e-38)
    x[10, :32] = np.linspace(0, 1, 32) * 2.0**-127
    codes, scales = _quantize(gctx, ehip_mod, x)
    c, s = mx.quantize(x.astype(np.float64))
    _check_panels(codes, scales, mx.panels(c, s))
    y = gctx.alloc(x.nbytes)
    assert gctx.mxfp4_dequantize(codes, scales, 20, 96, y) == 0
    gctx.sync()
    assert np.array_equal(y.download(np.float32, x.shape), mx.values(c, s, 96), equal_nan=True)
    _free(codes, scales, y)


@pytest.mark.parametrize("rows,k", SIZES)
def test_pack_is_a_permutation(gctx, ehip_mod, rows, k):
    rng = np.random.default_rng(rows + k)
    codes = rng.integers(0, 16, (rows, mx.blocks(k), 32)).astype(np.uint8)
    scales = rng.integers(0, 256, (rows, mx.blocks(k))).astype(np.uint8)
    dc, ds = gctx.to_device(mx.row_bytes(codes)), gctx.to_device(scales)
    pc, ps = _panel_buffers(gctx, ehip_mod, rows, k)
    assert gctx.mxfp4_pack(dc, ds, rows, k, pc, ps) == 0, gctx.last_error()
    gctx.sync()
    codes.reshape(rows, -1)[:, k:] = 0
    want = mx.panels(codes, scales)
    assert np.array_equal(pc.download(np.uint8, want[0].shape), want[0])
    assert np.array_equal(ps.download(np.uint8, want[1].shape), want[1])
    y = gctx.alloc(rows * k * 4)
    assert gctx.mxfp4_dequantize(pc, ps, rows, k, y) == 0
    gctx.sync()
    with np.errstate(over="ignore"):
        ref = mx.values(codes, scales, k).astype(np.float32)
    assert np.array_equal(y.download(np.float32, (rows, k)), ref, equal_nan=True)
    _free(dc, ds, pc, ps, y)


def test_unaligned_rows_quantize_alike(gctx, ehip_mod):
    """x and y four (two) bytes off a 16-byte boundary take the narrow loads."""
    from types import SimpleNamespace
    rows, k = 19, 256
    x = np.random.default_rng(3).standard_normal((rows, k))
    for dtype, size in (("f32", 4), ("bf16", 2), ("f16", 2)):
        raw, val = _bits(x, dtype)
        flat = np.zeros(rows * k + 1, raw.dtype)
        flat[1:] = raw.ravel()
        dx, dy = gctx.to_device(flat), gctx.alloc(4 * (rows * k + 2))
        dy.upload(np.full(rows * k + 2, 7.0, np.float32))
        codes, scales = _panel_buffers(gctx, ehip_mod, rows, k)
        off = SimpleNamespace(ptr=dx.ptr + size)
        assert gctx.mxfp4_quantize(off, _code(ehip_mod, dtype), rows, k, codes, scales) == 0
        assert gctx.mxfp4_dequantize(codes, scales, rows, k, SimpleNamespace(ptr=dy.ptr + 4)) == 0
        gctx.sync()
        out = dy.download(np.float32, (rows * k + 2,))
        assert out[0] == 7.0 and out[-1] == 7.0, "wrote outside y"
        assert np.array_equal(out[1:-1].reshape(rows, k), mx.quantized(val.astype(np.float64)))
        _free(dx, dy, codes, scales)


# ------------------------------------------------------------------- product --

# Rows on both sides of every kernel's limits, widths and k with remainders in
# panels (16), tiles (128) and groups (512).
SHAPES = [(1, 32, 16), (1, 896, 896), (2, 100, 33), (15, 129, 17), (16, 512, 64), (17, 513, 65),
          (32, 640, 48), (33, 2048, 100), (48, 4096, 256), (64, 1000, 129), (65, 700, 300),
          (100, 1536, 1000), (129, 384, 272), (256, 512, 512), (257, 1111, 257), (300, 4096, 520),
          (512, 896, 1300), (513, 160, 1030), (1100, 300, 700), (3, 700, 40), (4, 4200, 33),
          (5, 4200, 33), (600, 1000, 3000)]
# 128 x 128 tiles, and 128 x 256 ones (k from 2048 on) whose k tiles are taken in
# turns of four, two and one.
LARGE = [(1000, 300, 4100), (1030, 2048, 12900), (1025, 2300, 12801), (1030, 2100, 12900)]


def _grid_matrix(rng, rows, k):
    """Codes 0, .5, 1, 1.5, 2 of both signs at scales 2^-1..2^1: products are
    multiples of 2^-4 up to 16, so sums of 2^15 of them are exact in fp32."""
    shape = (rows, mx.blocks(k), 32)
    codes = (rng.integers(0, 5, shape, dtype=np.uint8) |
             (rng.integers(0, 2, shape, dtype=np.uint8) << 3))
    codes.reshape(rows, -1)[:, k:] = 0
    return codes, rng.integers(126, 129, (rows, mx.blocks(k))).astype(np.uint8)


@pytest.mark.parametrize("m,k,n", SHAPES + LARGE)
def test_exact_sums_are_exact(gctx, ehip_mod, m, k, n):
    rng = np.random.default_rng(m * k + n)
    xq, wq = _grid_matrix(rng, m, k), _grid_matrix(rng, n, k)
    bias = rng.integers(-8, 9, n).astype(np.float32)
    bufs = _upload(gctx, *xq) + _upload(gctx, *wq)
    db, dy = gctx.to_device(bias), gctx.alloc(4 * m * n)
    # Exact in fp32 too, whatever the order.
    want = mx.values(*xq, k).astype(np.float32) @ mx.values(*wq, k).T.astype(np.float32)
    for b in (None, db):
        assert gctx.mxfp4_gemm(bufs[0], bufs[1], m, k, bufs[2], bufs[3], n, b, dy) == 0, \
            gctx.last_error()
        gctx.sync()
        assert np.array_equal(dy.download(np.float32, (m, n)), want + (0 if b is None else bias))
    _free(db, dy, *bufs)


def _check(got, x, w, bias, k):
    """got against quantised x, w in 64 bits, within the module's bounds."""
    ref = x @ w.T + (0 if bias is None else bias)
    err = np.abs(got.astype(np.float64) - ref)
    top = np.abs(x) @ np.abs(w).T + (0 if bias is None else np.abs(bias))
    assert (err <= k * 2.0**-23 * top).all(), float((err / top).max())
    assert np.linalg.norm(err) <= np.sqrt(k) * 2.0**-23 * np.linalg.norm(ref)


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_quantises_and_multiplies(gctx, ehip_mod, m, k, n):
    rng = np.random.default_rng(m + k + n)
    x = (rng.standard_normal((m, k)) * np.exp2(rng.integers(-4, 5, (1, k)))).astype(np.float32)
    w = (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
    bias = rng.standard_normal(n).astype(np.float32) if n % 2 else None
    dx, dy = gctx.to_device(x), gctx.alloc(4 * m * n)
    db = gctx.to_device(bias) if bias is not None else None
    wc, ws = _quantize(gctx, ehip_mod, w)
    dy.upload(np.full((m, n), np.nan, np.float32))
    assert gctx.mxfp4_linear(dx, m, k, wc, ws, n, db, dy) == 0, gctx.last_error()
    gctx.sync()
    got = dy.download(np.float32, (m, n))
    _check(got, mx.quantized(x), mx.quantized(w), bias, k)
    # The product over x's panels is the same, bit for bit.
    xc, xs = _quantize(gctx, ehip_mod, x)
    dy.upload(np.full((m, n), np.nan, np.float32))
    assert gctx.mxfp4_gemm(xc, xs, m, k, wc, ws, n, db, dy) == 0, gctx.last_error()
    gctx.sync()
    assert np.array_equal(dy.download(np.float32, (m, n)).view(np.uint32), got.view(np.uint32))
    _free(dx, dy, db, wc, ws, xc, xs)


@pytest.mark.parametrize("m,k,n", [(3, 300, 40), (70, 640, 100), (600, 256, 530)])
def test_nan_blocks_reach_their_rows_only(gctx, ehip_mod, m, k, n):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((m, k)).astype(np.float32)
    w = rng.standard_normal((n, k)).astype(np.float32)
    x[1, k - 1], x[m - 1, 0] = np.nan, np.inf
    w[n // 2, 5] = -np.inf
    dx, dy = gctx.to_device(x), gctx.alloc(4 * m * n)
    wc, ws = _quantize(gctx, ehip_mod, w)
    assert gctx.mxfp4_linear(dx, m, k, wc, ws, n, None, dy) == 0
    gctx.sync()
    got = dy.download(np.float32, (m, n))
    nan = np.zeros((m, n), bool)
    nan[[1, m - 1]], nan[:, n // 2] = True, True
    assert np.array_equal(np.isnan(got), nan)
    _free(dx, dy, wc, ws)


@pytest.mark.parametrize("m", [2, 80, 600])
def test_scales_over_their_whole_range(gctx, ehip_mod, m):
    """Row scales 2^-127..2^103 of x against 1 and 8 in w: results from subnormal
    ones to near fp32's largest."""
    k, n = 256, 260
    rng = np.random.default_rng(m)
    xc, _ = _grid_matrix(rng, m, k)
    wc, _ = _grid_matrix(rng, n, k)
    e = np.linspace(0, 230, m).round().astype(np.uint8)
    xs = np.repeat(e[:, None], k // 32, 1)
    ws = np.full((n, k // 32), 127, np.uint8)
    ws[::2] = 130
    bufs = _upload(gctx, xc, xs) + _upload(gctx, wc, ws)
    dy = gctx.alloc(4 * m * n)
    assert gctx.mxfp4_gemm(bufs[0], bufs[1], m, k, bufs[2], bufs[3], n, None, dy) == 0
    gctx.sync()
    ref = mx.values(xc, xs, k) @ mx.values(wc, ws, k).T
    got = dy.download(np.float32, (m, n))
    normal = np.abs(ref) >= 2.0**-126
    assert np.array_equal(got[normal], ref[normal])
    assert np.abs(got - ref)[~normal].max(initial=0) <= 2.0**-126  # subnormal sums may be flushed
    _free(dy, *bufs)


def test_results_are_deterministic_and_stay_in_y(gctx, ehip_mod):
    from types import SimpleNamespace
    rng = np.random.default_rng(9)
    for m, k, n in ((5, 2048, 100), (90, 2048, 333), (700, 1000, 514)):
        x = rng.standard_normal((m, k)).astype(np.float32)
        wc, ws = _quantize(gctx, ehip_mod, rng.standard_normal((n, k)))
        raw = np.zeros(m * k + 1, np.float32)
        raw[1:] = x.ravel()
        dx, dy = gctx.to_device(raw), gctx.alloc(4 * (m * n + 2))
        outs = []
        for _ in range(2):
            dy.upload(np.full(m * n + 2, 7.0, np.float32))
            assert gctx.mxfp4_linear(SimpleNamespace(ptr=dx.ptr + 4), m, k, wc, ws, n, None,
                                     SimpleNamespace(ptr=dy.ptr + 4)) == 0
            gctx.sync()
            out = dy.download(np.float32, (m * n + 2,))
            assert out[0] == 7.0 and out[-1] == 7.0, "wrote outside y"
            outs.append(out[1:-1])
        assert np.array_equal(outs[0].view(np.uint32), outs[1].view(np.uint32))
        _free(dx, dy, wc, ws)


def test_refusals(gctx, ehip_mod):
    E, L = ehip_mod, ehip_mod.lib()
    b = gctx.alloc(1 << 16)
    p, h, bad = b.ptr, gctx.h, E.INVALID_ARGUMENT
    big = (1 << 21) + 1
    for rows, k in ((0, 4), (4, 0), (-1, 4), (big, 4), (4, big)):
        assert L.ehip_mxfp4_quantize(h, p, 0, rows, k, p, p) == bad
        assert L.ehip_mxfp4_pack(h, p, p, rows, k, p, p) == bad
        assert L.ehip_mxfp4_dequantize(h, p, p, rows, k, p) == bad
        assert L.ehip_mxfp4_gemm(h, p, p, rows, k, p, p, 4, None, p) == bad
        assert L.ehip_mxfp4_linear(h, p, rows, k, p, p, 4, None, p) == bad
        assert L.ehip_mxfp4_gated_linear(h, p, rows, k, p, p, p, p, 4, None, None, 0, p) == bad
    for n in (0, big):
        assert L.ehip_mxfp4_gemm(h, p, p, 4, 4, p, p, n, None, p) == bad
        assert L.ehip_mxfp4_linear(h, p, 4, 4, p, p, n, None, p) == bad
    assert L.ehip_mxfp4_quantize(h, p, 3, 4, 4, p, p) == bad
    for act in (-1, 3):
        assert L.ehip_mxfp4_gated_linear(h, p, 4, 4, p, p, p, p, 4, None, None, act, p) == bad
        assert "activation" in gctx.last_error()
    # null and misaligned operands, one at a time
    quant = [p, 0, 4, 4, p, p]
    for i, v in ((0, None), (4, None), (5, None), (4, p + 8), (5, p + 2)):
        assert L.ehip_mxfp4_quantize(h, *quant[:i], v, *quant[i + 1:]) == bad, (i, v)
    pack = [p, p, 4, 4, p, p]
    for i, v in ((0, None), (1, None), (4, None), (5, None), (4, p + 4)):
        assert L.ehip_mxfp4_pack(h, *pack[:i], v, *pack[i + 1:]) == bad, (i, v)
    deq = [p, p, 4, 4, p]
    for i, v in ((0, None), (1, None), (4, None), (0, p + 4), (1, p + 1)):
        assert L.ehip_mxfp4_dequantize(h, *deq[:i], v, *deq[i + 1:]) == bad, (i, v)
    gemm = [p, p, 4, 4, p, p, 4, None, p]
    for i, v in ((0, None), (1, None), (4, None), (5, None), (8, None), (0, p + 8), (4, p + 8),
                 (5, p + 2)):
        assert L.ehip_mxfp4_gemm(h, *gemm[:i], v, *gemm[i + 1:]) == bad, (i, v)
    lin = [p, 4, 4, p, p, 4, None, p]
    for i, v in ((0, None), (3, None), (4, None), (7, None), (3, p + 8)):
        assert L.ehip_mxfp4_linear(h, *lin[:i], v, *lin[i + 1:]) == bad, (i, v)
    gated = [p, 4, 4, p, p, p, p, 4, None, None, 0, p]
    for i, v in ((0, None), (3, None), (4, None), (5, None), (6, None), (11, None), (5, p + 8)):
        assert L.ehip_mxfp4_gated_linear(h, *gated[:i], v, *gated[i + 1:]) == bad, (i, v)
    b.free()
