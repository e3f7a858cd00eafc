"""MXFP4 on the host: the panel sizes of the C ABI, and the tests' own 64-bit
definition against cases worked by hand."""
import numpy as np
import pytest

import mx_util as mx


@pytest.mark.parametrize("rows,k,codes,scales", [
    (1, 1, 1024, 256), (16, 128, 1024, 256), (17, 129, 2 * 2 * 1024, 2 * 256),
    (16, 512, 4 * 1024, 256), (33, 513, 3 * 5 * 1024, 3 * 2 * 256),
    (1 << 21, 1 << 21, (1 << 17) * (1 << 14) * 1024, (1 << 17) * (1 << 12) * 256)])
def test_panel_bytes(ehip_mod, rows, k, codes, scales):
    assert ehip_mod.mxfp4_panel_bytes(rows, k) == (codes, scales)
    assert ehip_mod.lib().ehip_mxfp4_panel_bytes(rows, k, None, None) == 0


@pytest.mark.parametrize("rows,k", [(0, 4), (4, 0), (-1, 4), ((1 << 21) + 1, 4), (4, 1 << 22)])
def test_panel_bytes_refuses(ehip_mod, rows, k):
    assert ehip_mod.lib().ehip_mxfp4_panel_bytes(rows, k, None, None) == ehip_mod.INVALID_ARGUMENT


@pytest.mark.parametrize("call,args", [
    ("ehip_mxfp4_quantize", (1, 0, 4, 4, 1, 1)), ("ehip_mxfp4_pack", (1, 1, 4, 4, 1, 1)),
    ("ehip_mxfp4_dequantize", (1, 1, 4, 4, 1)), ("ehip_mxfp4_gemm", (1, 1, 4, 4, 1, 1, 4, 1, 1)),
    ("ehip_mxfp4_linear", (1, 4, 4, 1, 1, 4, 1, 1)),
    ("ehip_mxfp4_gated_linear", (1, 4, 4, 1, 1, 1, 1, 4, 1, 1, 0, 1)),
    ("ehip_packed_gated_gemm", (1, 4, 4, 1, 1, 1, 4, 1, 1, 0, 1))])
def test_calls_without_a_context_are_refused(ehip_mod, call, args):
    assert getattr(ehip_mod.lib(), call)(None, *args) == ehip_mod.INVALID_ARGUMENT


def test_definition_ties_and_scales():
    # Block maximum 4..7.99: scale 1. Ties go to the even code.
    x = np.zeros((1, 64))
    x[0, :14] = [6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, .2501, .7499, -5, -.25, 7.9, 5.001]
    x[0, 32:35] = [2.0**-3, 3 * 2.0**-6, 0]
    codes, scales = mx.quantize(x)
    assert scales.tolist() == [[127, 127 - 5]]
    assert mx.values(codes, scales, 64)[0, :14].tolist() == [
        6, 0, 1, 1, 2, 2, 4, 4, .5, .5, -4, 0, 6, 6]
    assert mx.values(codes, scales, 64)[0, 32:35].tolist() == [2.0**-3, 3 * 2.0**-6, 0]


def test_definition_extremes():
    x = np.zeros((6, 32))
    x[1, 3], x[2, 3], x[3, 5], x[3, 6] = np.nan, -np.inf, 2.0**-149, 2.0**-128
    x[4, 0], x[5, 0] = 3.0e38, 2.0**-126
    codes, scales = mx.quantize(x)
    assert scales[:, 0].tolist() == [0, 255, 255, 0, 127 + 125, 0]
    v = mx.values(codes, scales, 32)
    assert np.isnan(v[1:3]).all() and v[3, 6] == 2.0**-128 and v[3, 5] == 0
    assert v[4, 0] == 6 * 2.0**125 and v[5, 0] == 2.0**-126


def test_panel_helpers_agree():
    rng = np.random.default_rng(0)
    for rows, k in ((1, 1), (17, 130), (40, 1100)):
        codes, scales = mx.quantize(rng.standard_normal((rows, k)))
        for a, b in zip(mx.panels(codes, scales), mx.panels_of(codes, scales)):
            assert np.array_equal(a, b)
