"""Plain 64-bit statements of MXFP4: quantisation, products and the MoE layer.

pinned by: brute force over all codes (tests/test_oracle_mxfp4.py).
"""
from __future__ import annotations

import numpy as np

from . import dense

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
TABLE = np.concatenate([VALUES, -VALUES])
BLOCK = 32


def quantize(x):
    """``(packed uint8 [.., K/2], scales uint8 [.., K/32])`` of float x [.., K]."""
    x = np.asarray(x, dtype=np.float64)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    bad = ~np.isfinite(b).all(-1)
    f = np.where(bad[..., None], 0.0, b)
    top = np.abs(f).max(-1)
    _, e = np.frexp(top)                        # top = m 2^e, m in [0.5, 1): floor(log2) = e - 1
    s = np.where(top > 0, np.maximum(e - 1 - 2 + 127, 0), 0)
    v = np.abs(f) / np.exp2(s - 127.0)[..., None]
    code = np.zeros(v.shape, dtype=np.int64)
    for c in range(1, 8):                       # past the middle between c - 1 and c, or at it
        mid = (VALUES[c - 1] + VALUES[c]) / 2   # where c is the even one
        code[(v > mid) | ((v == mid) & (c % 2 == 0))] = c
    code += 8 * np.signbit(f)
    code[bad] = 0
    s = np.where(bad, 255, s)
    code = code.reshape(x.shape).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), s.astype(np.uint8)


def dequantize(packed, scales):
    """float64 values; a scale of 255 is NaN."""
    packed, scales = np.asarray(packed), np.asarray(scales)
    code = np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1],
                                                           2 * packed.shape[-1])
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return TABLE[code] * np.repeat(s, BLOCK, -1)


def tiles(packed, scales, gated=False):
    """One matrix [N, K] in the order of tiles, byte by byte."""
    packed, scales = np.asarray(packed), np.asarray(scales)
    rows, blocks = scales.shape
    halves = [(0, rows // 2), (rows // 2, rows // 2)] if gated else [(0, rows)]
    RT, KB = len(halves) * -(-halves[0][1] // 16), -(-blocks // 4)
    t = np.zeros((RT, KB, 64, 16), dtype=np.uint8)
    ts = np.zeros((RT, -(-KB // 4), 64, 4), dtype=np.uint8)
    for h, (first, n) in enumerate(halves):
        for i in range(n):
            rt, r = (i // 16) * len(halves) + h, i % 16
            for b in range(blocks):
                kb, q = divmod(b, 4)
                t[rt, kb, 16 * q + r] = packed[first + i, 16 * b:16 * b + 16]
                ts[rt, kb // 4, 16 * q + r, kb % 4] = scales[first + i, b]
    return t, ts


def moe_layer(x, w13, w2, ids, weights):
    """float64 layer of x [T, H], w13 [E, 2I, H], w2 [E, H, I] (float64), ids [T, k]."""
    x = np.asarray(x, dtype=np.float64)
    E, I = w13.shape[0], w13.shape[1] // 2
    out = np.zeros((x.shape[0], w2.shape[1]))
    for t in range(x.shape[0]):
        for e, w in zip(ids[t], weights[t]):
            if 0 <= e < E:
                y = w13[e] @ x[t]
                out[t] += float(w) * (w2[e] @ (dense.activation(y[:I], "silu") * y[I:]))
    return out
