"""The gated feed-forward block, act(x Wg^T + bg) * (x Wu^T + bu), over packed
fp32 / bf16 / fp16 weights (ehip_packed_gated_gemm) and MXFP4 ones
(ehip_mxfp4_gated_linear), against 64 bits; both halves of a feed-forward block
in turn, and captured into a graph.

Bounds. A projection's fp32 sum of k products is within e = k 2^-23 (sum |x||w| +
|bias|) of its value (one unit in the last place an addition; the planes of x
and w leave out less than 2^-24 of a term). With |act'| <= 1.13, |act(g)| <= |g|
+ 0.2 and an activation that is off by at most (|g| + 8) 2^-23 of itself (the
hardware's exponential of a rounded product, reciprocal and products):
|y - ref| <= 1.13 eg (|u| + eu) + |act(g)| eu + (|g| + 10) 2^-23 |ref|. In the
2-norm independent roundings give sqrt(k) 2^-23 a projection: bar 4 sqrt(k)
2^-23, and at least 2e-6."""
from types import SimpleNamespace

import numpy as np
import pytest

import mx_util as mx

pytestmark = pytest.mark.gpu

ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _weight(E, rng, n, k, dtype):
    """(bits, values, type) of an [n, k] weight."""
    w = (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
    if dtype == "f32":
        return w, w, E.WEIGHT_F32
    if dtype == "f16":
        h = w.astype(np.float16)
        return h.view(np.uint16), h.astype(np.float32), E.WEIGHT_F16
    b = (w.view(np.uint32) >> 16).astype(np.uint16)
    return b, (b.astype(np.uint32) << 16).view(np.float32), E.WEIGHT_BF16


def _pack(gctx, bits, code):
    n, k = bits.shape
    dw, dwp = gctx.to_device(bits), gctx.alloc(-(-n // 16) * k * 16 * bits.itemsize)
    assert gctx.pack_weight_panels(dw, code, n, k, dwp) == 0, gctx.last_error()
    gctx.sync()
    dw.free()
    return dwp


def _quantize(gctx, E, w):
    n, k = w.shape
    dw = gctx.to_device(np.asarray(w, np.float32))
    bufs = [gctx.alloc(b) for b in E.mxfp4_panel_bytes(n, k)]
    assert gctx.mxfp4_quantize(dw, E.WEIGHT_F32, n, k, *bufs) == 0, gctx.last_error()
    gctx.sync()
    dw.free()
    return bufs


def _check(got, x, wg, wu, bg, bu, act):
    x, wg, wu = (np.asarray(a, np.float64) for a in (x, wg, wu))
    k = x.shape[1]
    zg, zu = (0 if b is None else np.asarray(b, np.float64) for b in (bg, bu))
    g, u = x @ wg.T + zg, x @ wu.T + zu
    eg, eu = (k * 2.0**-23 * (np.abs(x) @ np.abs(w).T + np.abs(z)) for w, z in ((wg, zg), (wu, zu)))
    a = mx.activate(g, act)
    ref = a * u
    err = np.abs(got.astype(np.float64) - ref)
    bar = 1.13 * eg * (np.abs(u) + eu) + np.abs(a) * eu + (np.abs(g) + 10) * 2.0**-23 * np.abs(ref)
    assert (err <= bar).all(), float((err / bar).max())
    assert np.linalg.norm(err) <= max(2e-6, 4 * np.sqrt(k) * 2.0**-23) * np.linalg.norm(ref)


def _bias(rng, n, which):
    return [rng.standard_normal(n).astype(np.float32) if which & b else None for b in (1, 2)]


def _dev(gctx, a):
    return None if a is None else gctx.to_device(a)


# Both sides of the tile rules: rows 1..700, k with and without whole 32s, n
# with remainders in panels and tiles, short and long sums.
SHAPES = [(1, 1, 1), (1, 64, 16), (1, 896, 300), (2, 33, 17), (4, 4096, 96), (7, 100, 129),
          (8, 512, 64), (9, 1000, 111), (16, 96, 250), (17, 64, 256), (31, 130, 257),
          (32, 896, 896), (48, 2048, 200), (64, 160, 130), (65, 999, 129), (130, 300, 70),
          (257, 256, 250), (300, 64, 512), (600, 544, 272),
          # wide enough for each of the larger tiles
          (48, 300, 8200), (600, 97, 4000), (1000, 33, 9002), (520, 70, 12001),
          # and, fp32 weights, for each of theirs
          (130, 1030, 4096), (600, 1030, 1040), (600, 200, 2600), (700, 200, 4096),
          (1000, 96, 8000),
          # bf16 as fp16
          (900, 513, 4100),
          # the steps of tiles of one to four panels split
          (13, 4097, 4100), (20, 3001, 70), (40, 2050, 70), (63, 2050, 70),
          # tiles of 64 x 32 and 48 x 32
          (257, 513, 1030), (70, 700, 70), (2400, 513, 129), (1500, 700, 272)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_packed_gated_against_64_bits(gctx, ehip_mod, m, k, n, dtype):
    E = ehip_mod
    rng = np.random.default_rng(m * k + n)
    x = rng.standard_normal((m, k)).astype(np.float32)
    (gb, gv, code), (ub, uv, _) = (_weight(E, rng, n, k, dtype) for _ in range(2))
    bg, bu = _bias(rng, n, (m + n) % 4)
    act = (m + k + n) % 3
    print(f"[gated] m={m} k={k} n={n} {dtype} act={act} bias={(m + n) % 4}", flush=True)
    raw = np.zeros(m * k + 1, np.float32)
    raw[1:] = x.ravel()
    # x and y four bytes off a 16-byte boundary, and on one
    dx, dy = gctx.to_device(raw), gctx.alloc(4 * (m * n + 2))
    dx2, dy2 = gctx.to_device(x), gctx.alloc(4 * m * n)
    wg, wu, dbg, dbu = _pack(gctx, gb, code), _pack(gctx, ub, code), _dev(gctx, bg), _dev(gctx, bu)
    dy.upload(np.full(m * n + 2, 7.0, np.float32))
    assert gctx.packed_gated_gemm(SimpleNamespace(ptr=dx.ptr + 4), m, k, wg, wu, code, n, dbg, dbu,
                                  act, SimpleNamespace(ptr=dy.ptr + 4)) == 0, gctx.last_error()
    assert gctx.packed_gated_gemm(dx2, m, k, wg, wu, code, n, dbg, dbu, act, dy2) == 0
    gctx.sync()
    out = dy.download(np.float32, (m * n + 2,))
    assert out[0] == 7.0 and out[-1] == 7.0, "wrote outside y"
    got = dy2.download(np.float32, (m, n))
    _check(out[1:-1].reshape(m, n), x, gv, uv, bg, bu, act)
    _check(got, x, gv, uv, bg, bu, act)
    # Again: the same bits.
    assert gctx.packed_gated_gemm(dx2, m, k, wg, wu, code, n, dbg, dbu, act, dy2) == 0
    gctx.sync()
    assert np.array_equal(dy2.download(np.float32, (m, n)).view(np.uint32), got.view(np.uint32))
    for b in (dx, dy, dx2, dy2, wg, wu, dbg, dbu):
        if b is not None:
            b.free()


@pytest.mark.parametrize("m,k,n", [(1, 896, 300), (3, 100, 17), (16, 1030, 64), (33, 512, 100),
                                   (65, 700, 300), (130, 2048, 129), (300, 1111, 520),
                                   (600, 384, 700), (1000, 640, 2050), (1100, 2300, 6605)])
def test_mxfp4_gated_against_64_bits(gctx, ehip_mod, m, k, n):
    E = ehip_mod
    rng = np.random.default_rng(m + k * n)
    x = rng.standard_normal((m, k)).astype(np.float32)
    g, u = ((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32) for _ in range(2))
    bg, bu = _bias(rng, n, (m + n) % 4)
    act = (m + k + n) % 3
    dx, dy, dbg, dbu = gctx.to_device(x), gctx.alloc(4 * (m * n + 2)), _dev(gctx, bg), _dev(gctx, bu)
    wg, wu = _quantize(gctx, E, g), _quantize(gctx, E, u)
    for off in (0, 4):  # y on a 16-byte boundary and off it
        dy.upload(np.full(m * n + 2, 7.0, np.float32))
        assert gctx.mxfp4_gated_linear(dx, m, k, *wg, *wu, n, dbg, dbu, act,
                                       SimpleNamespace(ptr=dy.ptr + off)) == 0, gctx.last_error()
        gctx.sync()
        out = dy.download(np.float32, (m * n + 2,))
        at = off // 4
        assert (out[:at] == 7.0).all() and (out[at + m * n:] == 7.0).all(), "wrote outside y"
        _check(out[at:at + m * n].reshape(m, n), mx.quantized(x), mx.quantized(g), mx.quantized(u),
               bg, bu, act)
    for b in (dx, dy, dbg, dbu, *wg, *wu):
        if b is not None:
            b.free()


@pytest.mark.parametrize("m,k,n", [(1, 128, 64), (8, 896, 100), (40, 64, 256), (300, 512, 256),
                                   (600, 1024, 1040), (900, 514, 4100)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_every_plane_reaches_the_up_projection(gctx, ehip_mod, m, k, n, dtype):
    """With a zero gate weight and bias 64, act(64) = 64 exactly, so y = 64 u. x
    = 1 + 1.5 * 2^-9 + b 2^-18 in three bf16 planes and weights in pairs (w, -w)
    leave u = 2^-18 sum(b w), every partial sum exact in fp32: only the third
    plane is left, to a quarter unit."""
    rng = np.random.default_rng(m + k)
    b = rng.integers(-1, 2, (m, k))
    x = (1 + 1.5 * 2.0**-9 + b * 2.0**-18).astype(np.float32)
    w = np.repeat(rng.choice([-1, 1], (n, k // 2)), 2, axis=1)
    w[:, 1::2] *= -1
    E = ehip_mod
    raw = {"f32": w.astype(np.float32), "f16": w.astype(np.float16).view(np.uint16),
           "bf16": (w.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)}[dtype]
    code = {"f32": E.WEIGHT_F32, "f16": E.WEIGHT_F16, "bf16": E.WEIGHT_BF16}[dtype]
    wu, wg = _pack(gctx, raw, code), _pack(gctx, np.zeros_like(raw), code)
    dx, dy, db = gctx.to_device(x), gctx.alloc(4 * m * n), gctx.to_device(np.full(n, 64, np.float32))
    for act in ACTS.values():
        assert gctx.packed_gated_gemm(dx, m, k, wg, wu, code, n, db, None, act, dy) == 0
        gctx.sync()
        got = dy.download(np.float32, (m, n)).astype(np.float64) * 2.0**12
        assert np.abs(got - b.astype(np.float64) @ w.T.astype(np.float64)).max() <= 0.25
    for buf in (wu, wg, dx, dy, db):
        buf.free()


@pytest.mark.parametrize("act", list(ACTS))
def test_activations_over_their_range(gctx, ehip_mod, act):
    """Weights of zero: y = act(bias_gate) bias_up, both kinds of weights. Far
    into both tails, where results underflow; plus infinity gives infinity, NaN
    and minus infinity NaN (GELU of minus infinity too, 0 times infinity)."""
    E = ehip_mod
    g = np.concatenate([np.linspace(-30, 30, 601), np.geomspace(1e-30, 1e30, 121),
                        -np.geomspace(1e-30, 1e30, 121), [0.0, np.inf, np.nan, -np.inf]])
    g = g.astype(np.float32)
    n = len(g)
    up = np.where(np.arange(n) % 2, 1.0, -2.0).astype(np.float32)
    dbg, dbu = gctx.to_device(g), gctx.to_device(up)
    dx = gctx.to_device(np.ones((2, 32), np.float32))
    outs = []
    for kind in ("packed", "mxfp4"):
        dy = gctx.alloc(8 * n)
        zero = [gctx.alloc(1 << 18) for _ in range(4)]  # zero-filled
        if kind == "packed":
            rc = gctx.packed_gated_gemm(dx, 2, 32, zero[0], zero[1], E.WEIGHT_BF16, n, dbg, dbu,
                                        ACTS[act], dy)
        else:
            rc = gctx.mxfp4_gated_linear(dx, 2, 32, *zero, n, dbg, dbu, ACTS[act], dy)
        assert rc == 0, gctx.last_error()
        gctx.sync()
        outs.append(dy.download(np.float32, (2, n)))
        for b in zero + [dy]:
            b.free()
    fin = np.isfinite(g)
    with np.errstate(over="ignore"):
        ref = mx.activate(g[fin], ACTS[act]) * up[fin]
        big = np.abs(ref) > 3.4e38
    for out in outs:
        assert np.array_equal(out[0], out[1], equal_nan=True)
        got = out[0][fin].astype(np.float64)
        # A quadratic term for GELU's erfc, whose argument is rounded; 2^-126
        # where the exponential or the result is subnormal.
        x = np.abs(g[fin].astype(np.float64))
        bar = (np.minimum(x, 200)**2 * 2 + x.clip(0, 200) + 10) * 2.0**-23 * np.abs(ref) + 2.0**-118
        assert (np.abs(got - ref)[~big] <= bar[~big]).all()
        assert np.isinf(got[big]).all() and (got[big] * ref[big] > 0).all()
        tail = out[0][~fin]
        assert tail[0] == np.inf * up[-3] and np.isnan(tail[1:]).all()
    for b in (dbg, dbu, dx):
        b.free()


@pytest.mark.parametrize("m,k,n", [(2, 160, 100), (20, 160, 100), (600, 1030, 1040)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_non_finite_rows_stay_in_their_rows(gctx, ehip_mod, m, k, n, dtype):
    E = ehip_mod
    rng = np.random.default_rng(m)
    x = rng.standard_normal((m, k)).astype(np.float32)
    (gb, gv, code), (ub, uv, _) = (_weight(E, rng, n, k, dtype) for _ in range(2))
    x[1, 7], x[0, 159] = np.nan, np.inf
    wg, wu = _pack(gctx, gb, code), _pack(gctx, ub, code)
    dx, dy = gctx.to_device(x), gctx.alloc(4 * m * n)
    assert gctx.packed_gated_gemm(dx, m, k, wg, wu, code, n, None, None, 0, dy) == 0
    gctx.sync()
    got = dy.download(np.float32, (m, n))
    assert np.isnan(got[1]).all() and not (np.isfinite(got[0]) & (got[0] != 0)).any()
    if m > 2:
        _check(got[2:], x[2:], gv, uv, None, None, 0)
    for b in (wg, wu, dx, dy):
        b.free()


@pytest.mark.parametrize("m,k,n", [(3, 200, 90), (20, 200, 90), (600, 1030, 1040)])
def test_fp16_subnormal_weights_and_rows_of_any_size(gctx, ehip_mod, m, k, n):
    """Weights among fp16's subnormals (multiples of 2^-24) are exact; rows of x
    from 2^-120 to 2^100, one with a spike 2^20 times the rest, keep their
    precision: beside the module's bound the fp16 planes leave out 2^-39 of a
    row's largest |x| a term. The up bias is zero and the gate's 64 over a zero
    weight, so y = 64 u."""
    E = ehip_mod
    rng = np.random.default_rng(m)
    x = rng.standard_normal((m, k))
    x[0, 5] *= 2.0**20
    x *= np.exp2(np.linspace(-120, 100, m))[:, None]
    x = x.astype(np.float32)
    j = rng.integers(-1023, 1024, (n, k))
    w = (j * 2.0**-24).astype(np.float16)
    assert np.array_equal(w.astype(np.float64), j * 2.0**-24)
    wu = _pack(gctx, w.view(np.uint16), E.WEIGHT_F16)
    wg = _pack(gctx, np.zeros((n, k), np.uint16), E.WEIGHT_F16)
    dx, dy = gctx.to_device(x), gctx.alloc(4 * m * n)
    db = gctx.to_device(np.full(n, 64, np.float32))
    assert gctx.packed_gated_gemm(dx, m, k, wg, wu, E.WEIGHT_F16, n, db, None, 0, dy) == 0
    gctx.sync()
    xd, wd = x.astype(np.float64), w.astype(np.float64)
    err = np.abs(dy.download(np.float32, (m, n)) / 64.0 - xd @ wd.T)
    bar = k * 2.0**-23 * (np.abs(xd) @ np.abs(wd).T)
    bar += 2.0**-39 * np.abs(xd).max(1)[:, None] * np.abs(wd).sum(1)[None]
    assert (err <= bar + 2.0**-126).all(), float((err / (bar + 2.0**-126)).max())
    for b in (wu, wg, dx, dy, db):
        b.free()


@pytest.mark.parametrize("m,k,n", [(3, 200, 90), (20, 200, 90), (70, 999, 129),
                                   (600, 1030, 1040)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_planes_of_rows_of_any_size(gctx, ehip_mod, m, k, n, dtype):
    """Rows of x from 2^-120 to 2^100 keep their precision: beside the module's
    bound, planes below bf16's normal range may be lost, 2^-125 of |w| (of fp32
    weights too: of |x|) a term, and a sum's subnormals, 2^-126 an addition. y =
    64 u, as above."""
    E = ehip_mod
    rng = np.random.default_rng(m)
    x = rng.standard_normal((m, k)) * np.exp2(np.linspace(-120, 100, m))[:, None]
    x = x.astype(np.float32)
    (ub, uv, code), (gb, _, _) = (_weight(E, rng, n, k, dtype) for _ in range(2))
    wu, wg = _pack(gctx, ub, code), _pack(gctx, np.zeros_like(gb), code)
    dx, dy = gctx.to_device(x), gctx.alloc(4 * m * n)
    db = gctx.to_device(np.full(n, 64, np.float32))
    assert gctx.packed_gated_gemm(dx, m, k, wg, wu, code, n, db, None, 0, dy) == 0
    gctx.sync()
    xd, wd = x.astype(np.float64), uv.astype(np.float64)
    err = np.abs(dy.download(np.float32, (m, n)) / 64.0 - xd @ wd.T)
    bar = k * 2.0**-23 * (np.abs(xd) @ np.abs(wd).T) + 2.0**-125 * np.abs(wd).sum(1)[None]
    bar += (2.0**-125 * np.abs(xd).sum(1)[:, None] if dtype == "f32" else 0) + k * 2.0**-126
    assert (err <= bar).all(), float((err / bar).max())
    for b in (wu, wg, dx, dy, db):
        b.free()


@pytest.mark.parametrize("m,k,n", [(1100, 2300, 6605), (1000, 640, 4100), (2500, 2560, 4096)])
def test_mxfp4_passes_on_other_inputs_between(gctx, ehip_mod, m, k, n):
    """Passes that nothing waits between, on two inputs in turn: a tile that is
    read before its loads have landed shows as another pass's values."""
    E = ehip_mod
    rng = np.random.default_rng(m)
    xs = [gctx.to_device(rng.standard_normal((m, k)).astype(np.float32)) for _ in range(2)]
    ys = [gctx.alloc(4 * m * n) for _ in range(2)]
    wg, wu = (_quantize(gctx, E, rng.standard_normal((n, k)).astype(np.float32) / 30)
              for _ in range(2))

    def calls():
        for dx, dy in zip(xs, ys):
            assert gctx.mxfp4_gated_linear(dx, m, k, *wg, *wu, n, None, None, 0, dy) == 0

    calls()
    gctx.sync()
    want = [dy.download(np.uint32, (m, n)) for dy in ys]
    for _ in range(8):
        for _ in range(4):
            calls()
        gctx.sync()
        for dy, w in zip(ys, want):
            assert np.array_equal(dy.download(np.uint32, (m, n)), w)
    for b in (*xs, *ys, *wg, *wu):
        b.free()


@pytest.mark.parametrize("m,k,n,dtype", [(3, 200, 90, "f32"), (20, 200, 90, "f32"),
                                         (600, 1030, 1040, "f32"), (20, 200, 90, "bf16"),
                                         (900, 513, 4100, "bf16")])
def test_weights_of_any_size(gctx, ehip_mod, m, k, n, dtype):
    """Rows of x from 2^-60 to 2^60 and weight rows from 2^-50 to 2^50, a spike
    2^20 times the rest in some of each, keep their precision: beside the module's
    bound 2^-39 of a row's largest |x|, and of a weight row's largest, a term. A
    weight row with an infinity makes its own column non-finite. y = 64 u, as
    above."""
    E = ehip_mod
    rng = np.random.default_rng(m)
    x, w = rng.standard_normal((m, k)), rng.standard_normal((n, k))
    x[0, 5] *= 2.0**20
    w[7::16, 3] *= 2.0**20
    x = (x * np.exp2(np.linspace(-60, 60, m))[:, None]).astype(np.float32)
    w = (w * np.exp2(np.linspace(-50, 50, n))[:, None]).astype(np.float32)
    w[12, 9] = np.inf
    bits, code = w, E.WEIGHT_F32
    if dtype == "bf16":
        bits, code = (w.view(np.uint32) >> 16).astype(np.uint16), E.WEIGHT_BF16
        w = (bits.astype(np.uint32) << 16).view(np.float32)
    wu, wg = _pack(gctx, bits, code), _pack(gctx, np.zeros_like(bits), code)
    dx, dy = gctx.to_device(x), gctx.alloc(4 * m * n)
    db = gctx.to_device(np.full(n, 64, np.float32))
    assert gctx.packed_gated_gemm(dx, m, k, wg, wu, code, n, db, None, 0, dy) == 0
    gctx.sync()
    got = dy.download(np.float32, (m, n)) / 64.0
    assert not np.isfinite(got[:, 12]).any()
    got, w = np.delete(got, 12, 1), np.delete(w, 12, 0)
    xd, wd = np.abs(x.astype(np.float64)), np.abs(w.astype(np.float64))
    ref = x.astype(np.float64) @ w.astype(np.float64).T
    # The last rows' spikes reach 2^60 2^50 2^20, and 64 times that passes fp32's
    # 2^128: such results (a factor of 2 and the bound's share aside) are infinite.
    fits = 64 * np.abs(ref) < 2.0**127
    assert fits.mean() > 0.9 and (64 * xd @ wd.T >= 2.0**127)[~np.isfinite(got)].all()
    err = np.abs(np.where(fits, got - np.where(fits, ref, 0), 0))
    bar = k * 2.0**-23 * (xd @ wd.T)
    bar += 2.0**-39 * (xd.max(1)[:, None] * wd.sum(1)[None] + xd.sum(1)[:, None] * wd.max(1)[None])
    assert (err <= bar + 2.0**-126).all(), float((err / bar).max())
    for b in (wu, wg, dx, dy, db):
        b.free()


def test_two_contexts_at_once(tctx, ehip_mod):
    """Two contexts' calls run side by side on their own streams, each over its own
    workspace: the results of either alone."""
    E, ctxs = ehip_mod, [tctx(), tctx()]
    sizes = [[(300, 512, 520), (20, 4096, 256)], [(257, 640, 400), (70, 4096, 264)]]
    for kind in ("bf16", "mxfp4"):
        rng = np.random.default_rng(7)
        blocks = [[_block(c, E, rng, *s, kind) for s in ss] for c, ss in zip(ctxs, sizes)]
        want = []
        for c, bs in zip(ctxs, blocks):
            want.append([])
            for x, _, (_, _, dy), calls, _ in bs:
                calls()
                c.sync()
                want[-1].append(dy.download(np.float32, x.shape))
                dy.upload(np.full(x.shape, np.nan, np.float32))
        for _ in range(20):
            for bs in zip(*blocks):
                for b in bs:
                    b[3]()
        for c, bs, ws in zip(ctxs, blocks, want):
            c.sync()
            for (x, _, io, _, bufs), w in zip(bs, ws):
                got = io[2].download(np.float32, x.shape)
                assert np.array_equal(got.view(np.uint32), w.view(np.uint32)), kind
                for b in (*io, *bufs):
                    b.free()


# ------------------------------------------------------ the block as one run --

def _block(gctx, E, rng, m, k, n, kind):
    """A feed-forward block's buffers and its calls in order."""
    x = rng.standard_normal((m, k)).astype(np.float32)
    dx, dh, dy = gctx.to_device(x), gctx.alloc(4 * m * n), gctx.alloc(4 * m * k)
    if kind == "mxfp4":
        ws = [(rng.standard_normal(s) / np.sqrt(s[1])).astype(np.float32)
              for s in ((n, k), (n, k), (k, n))]
        g, u, d = (_quantize(gctx, E, w) for w in ws)
        vals = [mx.quantized(w) for w in ws]

        def calls():
            assert gctx.mxfp4_gated_linear(dx, m, k, *g, *u, n, None, None, 0, dh) == 0, \
                gctx.last_error()
            assert gctx.mxfp4_linear(dh, m, n, *d, k, None, dy) == 0, gctx.last_error()
        return x, vals, (dx, dh, dy), calls, [*g, *u, *d]
    ws = [_weight(E, rng, *s, kind) for s in ((n, k), (n, k), (k, n))]
    code = ws[0][2]
    g, u, d = (_pack(gctx, w[0], code) for w in ws)

    def calls():
        assert gctx.packed_gated_gemm(dx, m, k, g, u, code, n, None, None, 0, dh) == 0, \
            gctx.last_error()
        assert gctx.packed_gemm(dh, m, n, d, code, k, None, dy) == 0, gctx.last_error()
    return x, [w[1] for w in ws], (dx, dh, dy), calls, [g, u, d]


@pytest.mark.parametrize("kind", ["mxfp4", "bf16", "f16", "f32"])
@pytest.mark.parametrize("m,k,n", [(1, 896, 1000), (37, 512, 700), (270, 256, 530)])
def test_feed_forward_block(gctx, ehip_mod, kind, m, k, n):
    """Gate and up, then the down projection of their result: each against 64
    bits from its own input, so that no quantisation flips between the two."""
    rng = np.random.default_rng(m)
    x, (g, u, d), (dx, dh, dy), calls, bufs = _block(gctx, ehip_mod, rng, m, k, n, kind)
    calls()
    gctx.sync()
    h, y = dh.download(np.float32, (m, n)), dy.download(np.float32, (m, k))
    q = mx.quantized if kind == "mxfp4" else np.asarray
    _check(h, q(x), g, u, None, None, 0)
    hq = np.asarray(q(h), np.float64)
    ref, top = hq @ np.asarray(d, np.float64).T, np.abs(hq) @ np.abs(d).T
    err = np.abs(y - ref)
    assert (err <= n * 2.0**-23 * top).all()
    assert np.linalg.norm(err) <= np.sqrt(n) * 2.0**-23 * np.linalg.norm(ref)
    for b in (dx, dh, dy, *bufs):
        b.free()


@pytest.mark.parametrize("kind,k", [("mxfp4", 896), ("bf16", 896), ("f32", 896), ("bf16", 4096),
                                    ("f16", 4096)])  # 4096: split tiles
def test_captured_block_replays(tctx, ehip_mod, kind, k):
    """Captured blocks share the context's workspace. Replays after new
    inputs, after eager calls of other sizes, and after the workspace has grown
    past the captured one: each is bit-identical to the eager calls."""
    from ehip import hipgraph
    E, ctx = ehip_mod, tctx()
    rng = np.random.default_rng(1)
    blocks = [_block(ctx, E, rng, m, k, 520, kind) for m in (5, 70, 200, 1)]
    large = _block(ctx, E, rng, 900, k, 2000, kind)
    stream, graphs = hipgraph.Stream(), [hipgraph.Graph() for _ in blocks]
    assert E.lib().ehip_set_stream(ctx.h, stream.h) == 0
    try:
        for b in blocks:
            b[3]()  # the workspace's first growth
        for g, b in zip(graphs, blocks):
            g.capture(stream, b[3])
        for turn in range(4):
            if turn == 2:
                large[3]()
                ctx.sync()
            want = []
            for x, _, (dx, _, dy), calls, _ in blocks:
                dx.upload(rng.standard_normal(x.shape).astype(np.float32))
                calls()
                ctx.sync()
                want.append(dy.download(np.float32, x.shape))
                dy.upload(np.full(x.shape, np.nan, np.float32))
            for g in graphs:
                g.replay(stream)
            ctx.sync()
            for (x, _, (_, _, dy), _, _), w in zip(blocks, want):
                got = dy.download(np.float32, x.shape)
                assert np.array_equal(got.view(np.uint32), w.view(np.uint32)), turn
    finally:
        assert E.lib().ehip_set_stream(ctx.h, None) == 0
        for g in graphs:
            g.close()
        stream.close()
    for x, _, io, _, bufs in [*blocks, large]:
        for b in (*io, *bufs):
            b.free()


def test_capture_without_a_workspace_is_refused(tctx, ehip_mod):
    """A call whose workspace would have to grow inside a capture fails and
    records nothing; the capture itself goes on."""
    from ehip import hipgraph
    E, ctx = ehip_mod, tctx()
    rng = np.random.default_rng(2)
    m, k, n = 40, 300, 64
    dx, dy = ctx.to_device(rng.standard_normal((m, k)).astype(np.float32)), ctx.alloc(4 * m * n)
    w = _quantize(ctx, E, rng.standard_normal((n, k)))
    stream, graph, rcs = hipgraph.Stream(), hipgraph.Graph(), []

    def calls():
        rcs.append(ctx.mxfp4_linear(dx, m, k, *w, n, None, dy))
        rcs.append(ctx.mxfp4_dequantize(*w, n, k, big))

    big = ctx.alloc(4 * n * k)
    assert E.lib().ehip_set_stream(ctx.h, stream.h) == 0
    try:
        graph.capture(stream, calls)
        assert rcs == [E.FAILED_PRECONDITION, 0]
        assert "workspace" in ctx.last_error()
        graph.replay(stream)
        ctx.sync()
    finally:
        assert E.lib().ehip_set_stream(ctx.h, None) == 0
        graph.close()
        stream.close()
    for b in (dx, dy, big, *w):
        b.free()


def test_refusals(gctx, ehip_mod):
    E, L = ehip_mod, ehip_mod.lib()
    b = gctx.alloc(1 << 16)
    p, h, bad = b.ptr, gctx.h, E.INVALID_ARGUMENT
    ok = [p, 4, 4, p, p, E.WEIGHT_BF16, 4, None, None, 0, p]
    for i, v in ((0, None), (1, 0), (1, (1 << 21) + 1), (2, 0), (2, -3), (2, 1 << 22), (3, None),
                 (3, p + 8), (4, None), (4, p + 2), (5, 3), (5, -1), (6, 0), (6, (1 << 21) + 1),
                 (9, 3), (9, -1), (10, None)):
        assert L.ehip_packed_gated_gemm(h, *ok[:i], v, *ok[i + 1:]) == bad, (i, v)
        assert "gated gemm" in gctx.last_error()
    b.free()
