"""The MXFP4 oracle against brute force over all codes, and its order of tiles."""
import numpy as np
import pytest

from oracle import mxfp4


def _nearest(v, scale):
    """Codes whose value is nearest to v (v at most 6 scales), the even one of two."""
    off = np.abs(mxfp4.VALUES * scale - abs(v))
    best = np.flatnonzero(off == off.min())
    return int(best[0] if len(best) == 1 else best[best % 2 == 0][0])


@pytest.mark.parametrize("exponent", [-130, -127, -20, 0, 20, 120])
def test_quantize_is_the_nearest_code(exponent):
    rng = np.random.default_rng(exponent + 200)
    x = rng.standard_normal((40, 32)) * 2.0 ** exponent
    x[0, :8] = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0]) * 2.0 ** exponent  # halfway
    packed, s = mxfp4.quantize(x)
    got = np.stack([packed & 15, packed >> 4], -1).reshape(40, 32)
    for row in range(40):
        top = np.abs(x[row]).max()
        scale = 2.0 ** (float(s[row, 0]) - 127)
        assert 4 * scale <= top < 8 * scale or (s[row, 0] == 0 and top < 4 * scale)
        for c in range(32):
            assert got[row, c] & 7 == _nearest(x[row, c], scale)
            assert (got[row, c] >> 3) == np.signbit(x[row, c])


def test_every_code_and_scale_reads_back():
    code = np.tile(np.arange(16, dtype=np.uint8), 2)
    packed = np.tile(code[0::2] | (code[1::2] << 4), (256, 1))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    x = mxfp4.dequantize(packed, scales)
    assert np.isnan(x[255]).all()
    assert np.array_equal(x[127, :8], [0, .5, 1, 1.5, 2, 3, 4, 6])
    assert np.array_equal(x[:255], x[127] * 2.0 ** (np.arange(255) - 127.0)[:, None])
    again, s = mxfp4.quantize(x[:254])          # (a block with a 6 keeps its scale)
    assert np.array_equal(s[:, 0], np.arange(254)) and np.array_equal(again, packed[:254])


def test_special_blocks():
    x = np.zeros((4, 32))
    x[1, 3], x[2, 4], x[3, 5] = np.inf, np.nan, -0.0
    packed, s = mxfp4.quantize(x)
    assert s[:, 0].tolist() == [0, 255, 255, 0]
    assert not packed[:3].any() and packed[3, 2] == 0x80


@pytest.mark.parametrize("rows,blocks,gated", [(1, 1, False), (16, 4, False), (37, 9, False),
                                               (2, 1, True), (40, 17, True)])
def test_tiles_hold_every_block_once(rows, blocks, gated):
    rng = np.random.default_rng(rows)
    packed = rng.integers(0, 256, (rows, blocks * 16), dtype=np.uint8)
    scales = rng.integers(0, 256, (rows, blocks), dtype=np.uint8)
    t, ts = mxfp4.tiles(packed, scales, gated)
    n = rows // 2 if gated else rows
    seen = 0
    for row in range(rows):
        half, i = divmod(row, n)
        rt = (i // 16) * (2 if gated else 1) + (half if gated else 0)
        for b in range(blocks):
            assert np.array_equal(t[rt, b // 4, (b % 4) * 16 + i % 16], packed[row, b * 16:b * 16 + 16])
            assert ts[rt, b // 16, (b % 4) * 16 + i % 16, b // 4 % 4] == scales[row, b]
            seen += 1
    assert seen == rows * blocks and t.astype(int).sum() == packed.astype(int).sum()
    assert ts.astype(int).sum() == scales.astype(int).sum()


def test_moe_layer_against_loops():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, 4))
    w13, w2 = rng.standard_normal((2, 6, 4)), rng.standard_normal((2, 4, 3))
    ids, w = np.array([[0, 1], [1, 1], [-1, 2]]), rng.random((3, 2))
    got = mxfp4.moe_layer(x, w13, w2, ids, w)
    want = np.zeros((3, 4))
    for t in range(3):
        for j in range(2):
            e = ids[t, j]
            if e not in (0, 1):
                continue
            for h in range(4):
                for i in range(3):
                    g, u = (sum(w13[e, r, c] * x[t, c] for c in range(4)) for r in (i, 3 + i))
                    want[t, h] += w[t, j] * w2[e, h, i] * g / (1 + np.exp(-g)) * u
    assert np.allclose(got, want, rtol=1e-12)
