"""MXFP4 by its definition, in NumPy and 64 bits, for the tests: quantisation,
the values of codes and scales, and the panel layout. Also the gated block's
activations."""
from __future__ import annotations

import math

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MID = (GRID[1:] + GRID[:-1]) / 2


def blocks(k: int) -> int:
    return -(-k // 32)


def quantize(x):
    """x [rows, k] -> (codes [rows, blocks, 32] 0..15, scales [rows, blocks]).
    A code is the nearest of the eight magnitudes, the even one of two."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    b = np.zeros((rows, blocks(k) * 32))
    b[:, :k] = x
    b = b.reshape(rows, -1, 32)
    bad = ~np.isfinite(b).all(2)
    b = np.where(bad[:, :, None], 0.0, b)
    top = np.abs(b).max(2)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - 2, -127).clip(-127, 127)
    v = np.abs(b) / np.exp2(e.astype(np.float64))[:, :, None]
    lo, hi = np.searchsorted(MID, v, "left"), np.searchsorted(MID, v, "right")
    code = np.where(lo % 2 == 0, lo, hi) | (np.signbit(b) * 8)
    code[bad] = 0
    return code.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales, k):
    """The values [rows, k] of codes and scales, 64 bits."""
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * s[:, :, None]).reshape(codes.shape[0], -1)[:, :k]


def quantized(x):
    c, s = quantize(x)
    return values(c, s, np.shape(x)[1])


def row_bytes(codes):
    """codes as a checkpoint holds them: two a byte, the even element low."""
    return (codes[:, :, 0::2] | (codes[:, :, 1::2] << 4)).astype(np.uint8)


def panels(codes, scales):
    """(codes, scales) in panels: loops over the layout's own definition."""
    rows, nb = scales.shape
    tiles = -(-nb // 4)
    groups, pn = -(-tiles // 4), -(-rows // 16)
    packed = row_bytes(codes)
    pc = np.zeros((pn, tiles, 64, 16), np.uint8)
    ps = np.zeros((pn, groups, 64, 4), np.uint8)
    for r in range(rows):
        for b in range(nb):
            lane = 16 * (b % 4) + r % 16
            pc[r // 16, b // 4, lane] = packed[r, b]
            ps[r // 16, b // 16, lane, b // 4 % 4] = scales[r, b]
    return pc, ps


def panels_of(codes, scales):
    """panels(), by reshaping (large matrices)."""
    rows, nb = scales.shape
    tiles = -(-nb // 4)
    groups, pn = -(-tiles // 4), -(-rows // 16)
    c = np.zeros((pn * 16, tiles * 4, 16), np.uint8)
    c[:rows, :nb] = row_bytes(codes)
    s = np.zeros((pn * 16, groups * 16), np.uint8)
    s[:rows, :nb] = scales
    pc = c.reshape(pn, 16, tiles, 4, 16).transpose(0, 2, 3, 1, 4).reshape(pn, tiles, 64, 16)
    ps = s.reshape(pn, 16, groups, 4, 4).transpose(0, 2, 4, 1, 3).reshape(pn, groups, 64, 4)
    return np.ascontiguousarray(pc), np.ascontiguousarray(ps)


def activate(x, act):
    """The activations in 64 bits: 0 SiLU, 1 GELU, 2 GELU (tanh)."""
    x = np.asarray(x, np.float64)
    if act == 0:
        u = x
    elif act == 1:
        return 0.5 * x * np.vectorize(math.erfc, otypes=[np.float64])(-x * math.sqrt(0.5))
    else:
        u = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x**3)
    e = np.exp(-np.abs(u))
    return x * np.where(u >= 0, 1 / (1 + e), e / (1 + e))
