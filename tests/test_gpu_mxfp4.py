"""MXFP4 on the GPU against the 64-bit oracle.

Quantisation, decoding and the order of tiles are exact: compared bit for bit.  Products:
small whole numbers times powers of two make every float32 sum exact, so those are
compared bit for bit too.  Real values are compared within a bound: a float32 sum of K
products in any order, the matrix units truncating (in the 4-bit products each of an
instruction's 128 products and the sum so far), is off by at most (K + K / 128 + 8) *
2^-23 * sum |x w|; the activations' slopes are at most 1.13, the functions are within
2^-20 of their value plus 2^-22 |y|, and the result is rounded once: half a step of its
type.  The layer rounds silu(gate) * up once more, to hidden's type."""
import numpy as np
import pytest
import torch

from oracle import dense, mxfp4
from tests._helpers import banner
from tests._mxfp4_cases import cases

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FLOATS = [torch.bfloat16, torch.float16, torch.float32]


def _np(t):
    return None if t is None else t.double().cpu().numpy()


def _same(a, b):
    """Bit for bit, a NaN being a NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


# ---- quantisation -----------------------------------------------------------------------------

def _hard_rows(rows, K, seed):
    """Values at, next to and between the middles of codes, at many magnitudes."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, K)) * np.exp2(rng.integers(-20, 20, (rows, K // 32)).repeat(32, 1))
    mids = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.9375, -0.0, 0.5, 4])
    pick = rng.random((rows, K)) < 0.4
    hard = rng.choice(mids, (rows, K)) * rng.choice([-1, 1], (rows, K))
    hard = hard * (1 + rng.choice([0, 0, 2.0 ** -8, -2.0 ** -8], (rows, K)))
    hard *= np.exp2(rng.integers(-6, 6, (rows, K // 32)).repeat(32, 1))
    return torch.from_numpy(np.where(pick, hard, x))


@pytest.mark.parametrize("shape", [(1, 32), (1, 2048), (3, 96), (187, 1440), (64, 512), (2, 5, 64),
                                   (7, 14336), (1025, 160), (4096, 32)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_bit_exact(shape, dtype, device):
    from exq_amd.kernels import dequantize_mxfp4, quantize_mxfp4
    banner(f"quantize {shape} {dtype}")
    x = _hard_rows(int(np.prod(shape[:-1])), shape[-1], 5).to(dtype).view(shape)
    packed, scales = quantize_mxfp4(x.cuda())
    want_p, want_s = mxfp4.quantize(_np(x))
    assert packed.shape == (*shape[:-1], shape[-1] // 2) and scales.shape == (*shape[:-1], shape[-1] // 32)
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(packed.cpu().numpy(), want_p)
    for out in FLOATS:
        want = torch.from_numpy(mxfp4.dequantize(want_p, want_s)).to(out)
        assert _same(dequantize_mxfp4(packed, scales, out).cpu(), want)


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_layouts(dtype, device):
    """Column slices, odd strides and starts, expanded and transposed rows, empty ones."""
    from exq_amd.kernels import quantize_mxfp4
    big = torch.randn(40, 331).to(dtype).cuda()
    for x in (big[:, 1:33], big[:, 8:296], big[::3, 32:320], big[:1].expand(9, 331)[:, :320],
              big[:, :40].t()[:, :32], big.view(-1)[3:3 + 64 * 32].view(64, 32), big[:0, :64]):
        packed, scales = quantize_mxfp4(x)
        want = mxfp4.quantize(_np(x))
        assert np.array_equal(packed.cpu().numpy(), want[0])
        assert np.array_equal(scales.cpu().numpy(), want[1])


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_special_values(dtype, device):
    from exq_amd.kernels import dequantize_mxfp4, quantize_mxfp4
    f = torch.finfo(dtype)
    rows = [[0.0], [-0.0], [float("inf")], [-float("inf")], [float("nan")], [f.max], [-f.max, f.tiny],
            [f.tiny], [f.smallest_normal / 4], [2.0 ** -125], [2.0 ** -126, -2.0 ** -127], [1.0, float("nan")]]
    x = torch.zeros(len(rows), 64, dtype=torch.float64)
    for i, r in enumerate(rows):
        x[i, 5:5 + len(r)] = torch.tensor(r, dtype=torch.float64)
        x[i, 32] = 1.0
    x = x.to(dtype)
    packed, scales = quantize_mxfp4(x.cuda())
    want = mxfp4.quantize(_np(x))
    assert np.array_equal(scales.cpu().numpy(), want[1])
    assert np.array_equal(packed.cpu().numpy(), want[0])
    back = dequantize_mxfp4(packed, scales, torch.float32).cpu()
    assert torch.isnan(back[2, :32]).all() and torch.isnan(back[11, :32]).all()
    assert (back[:, 32] == 1).all()


def test_every_code_and_scale_decodes(device):
    from exq_amd.kernels import dequantize_mxfp4
    code = np.tile(np.arange(16, dtype=np.uint8), 2)
    packed = torch.from_numpy(np.tile(code[0::2] | (code[1::2] << 4), (256, 1))).cuda()
    scales = torch.arange(256, dtype=torch.uint8).view(-1, 1).cuda()
    want = torch.from_numpy(mxfp4.dequantize(packed.cpu().numpy(), scales.cpu().numpy()))
    for dtype in FLOATS:
        got, w = dequantize_mxfp4(packed, scales, dtype).cpu(), want.to(torch.float32).to(dtype)
        assert _same(got, w)


@pytest.mark.parametrize("experts,rows,K,gated", [(None, 1, 32, False), (None, 37, 288, False), (3, 16, 512, False),
                                                  (2, 40, 544, True), (None, 2, 64, True), (5, 96, 640, True)])
def test_tiles(experts, rows, K, gated, device):
    from exq_amd.kernels import Mxfp4Weight
    lead = () if experts is None else (experts,)
    g = torch.Generator().manual_seed(rows)
    packed = torch.randint(0, 256, (*lead, rows, K // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(0, 256, (*lead, rows, K // 32), generator=g, dtype=torch.uint8)
    w = Mxfp4Weight.from_packed(packed.cuda(), scales.cuda(), gated)
    for e in range(experts or 1):
        at = (e,) if lead else ()
        t, ts = mxfp4.tiles(packed[at].numpy(), scales[at].numpy(), gated)
        assert np.array_equal(w.tiles[at].cpu().numpy(), t)
        assert np.array_equal(w.tile_scales[at].cpu().numpy(), ts)
    assert (w.rows, w.cols, w.gated) == (rows, K, gated)


# ---- dense products ---------------------------------------------------------------------------

def _codes(rows, K, seed, lo, hi):
    """A stored weight of random codes, its scales 2^lo .. 2^hi."""
    g = torch.Generator().manual_seed(seed)
    packed = torch.randint(0, 256, (rows, K // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(lo + 127, hi + 128, (rows, K // 32), generator=g, dtype=torch.uint8)
    return packed, scales


def _dense(packed, scales):
    return torch.from_numpy(mxfp4.dequantize(packed.numpy(), scales.numpy()))


def _where(a, b):
    bad = (a != b).nonzero()
    return f"{bad.shape[0]} of {a.numel()} differ, first at {bad[0].tolist()}"


# T, K, N: single tokens, tile edges, K below, at and past a tile, odd numbers of blocks
SIZES = [
    (1, 32, 1), (1, 64, 16), (1, 2048, 128), (2, 256, 60), (3, 4096, 48), (5, 160, 33), (8, 96, 37),
    (15, 512, 256), (16, 2816, 512), (17, 128, 100), (31, 1440, 160), (33, 352, 250), (48, 288, 8),
    (63, 2048, 127), (64, 1024, 320), (65, 640, 129), (100, 1280, 384), (127, 32, 257),
    (129, 128, 520), (187, 1440, 203), (256, 256, 256), (257, 192, 264), (300, 2048, 128),
    (384, 448, 640), (513, 1088, 96), (640, 320, 1100), (1025, 96, 255), (1030, 512, 776),
]


@pytest.mark.parametrize("T,K,N", SIZES)
@pytest.mark.parametrize("kind", ["bf16", "f16", "x4"])
@pytest.mark.parametrize("gated", [False, True])
def test_whole_numbers(T, K, N, kind, gated, device):
    """Sums of multiples of 1/16 below 2^20: exact in float32, whatever the order."""
    from exq_amd.kernels import Mxfp4Weight, fused_gated_linear_mxfp4, fused_linear_mxfp4
    banner(f"mxfp4 T={T} K={K} N={N} {kind} gated={gated}")
    rows = 2 * N if gated else N
    if gated:       # the product of two sums has to be exact: a few columns that are not zero
        packed, scales = _codes(rows, K, 1, 0, 0)
        keep = torch.zeros(K // 2, dtype=torch.uint8)
        keep[torch.randperm(K // 2, generator=torch.Generator().manual_seed(9))[:8]] = 255
        packed &= keep
    else:
        packed, scales = _codes(rows, K, 1, -1, 1)
    w = Mxfp4Weight.from_packed(packed.cuda(), scales.cuda(), gated)
    x_scales = None
    if kind == "x4":
        xp, xs = _codes(T, K, 2, -1, 1 if not gated else -1)
        x, x_scales, X = xp.cuda(), xs.cuda(), _dense(xp, xs)
    else:
        dtype = torch.bfloat16 if kind == "bf16" else torch.float16
        X = torch.randint(-3, 4, (T, K), generator=torch.Generator().manual_seed(2)).double()
        x = X.to(dtype).cuda()
    y = X @ _dense(packed, scales).t()
    if gated:
        out = fused_gated_linear_mxfp4(x, w, x_scales=x_scales, activation="relu", out_dtype=torch.float32)
        want = (torch.relu(y[:, :N]) * y[:, N:]).float()
        assert torch.equal(out.cpu(), want), _where(out.cpu(), want)
        return
    out = fused_linear_mxfp4(x, w, x_scales=x_scales, out_dtype=torch.float32)
    assert torch.equal(out.cpu(), y.float()), _where(out.cpu(), y.float())
    g = torch.Generator().manual_seed(3)
    b, r = torch.randint(-40, 41, (N,), generator=g), torch.randint(-90, 91, (T, N), generator=g)
    o = torch.float16 if kind == "f16" else torch.bfloat16
    out = fused_linear_mxfp4(x, w, b.to(o).cuda(), x_scales=x_scales, residual=r.to(o).cuda(), out_dtype=o)
    want = (y + b + r).float().to(o)
    assert torch.equal(out.cpu(), want), _where(out.cpu(), want)


@pytest.mark.parametrize("x4,gated,kernel,T,N", cases())
@pytest.mark.parametrize("K", [96, 672])
def test_every_kernel_at_its_edges(x4, gated, kernel, T, N, K, device):
    """Whole numbers, the sums computed on the GPU in 64 bits from the oracle's values."""
    from exq_amd.kernels import Mxfp4Weight, fused_gated_linear_mxfp4, fused_linear_mxfp4
    banner(f"mxfp4 {kernel} x4={x4} gated={gated} T={T} N={N} K={K}")
    rows = 2 * N if gated else N
    packed, scales = _codes(rows, K, 1, 0, 0)
    if gated:       # (as above: the product of two sums has to be exact)
        keep = torch.zeros(K // 2, dtype=torch.uint8)
        keep[torch.randperm(K // 2, generator=torch.Generator().manual_seed(9))[:8]] = 255
        packed &= keep
    w = Mxfp4Weight.from_packed(packed.cuda(), scales.cuda(), gated)
    if x4:
        xp, xs = _codes(T, K, 2, -1, -1)
        x, x_scales, X = xp.cuda(), xs.cuda(), _dense(xp, xs).cuda()
    else:
        X = torch.randint(-3, 4, (T, K), generator=torch.Generator().manual_seed(2)).double().cuda()
        x, x_scales = X.to(torch.bfloat16), None
    y = torch.mm(X, _dense(packed, scales).cuda().t())
    hold = torch.full((T + 1, -(-N // 4) * 4 + 4), 7.0, device="cuda")
    if gated:
        fused_gated_linear_mxfp4(x, w, x_scales=x_scales, activation="relu", out=hold[:T, :N])
        want = (torch.relu(y[:, :N]) * y[:, N:]).float()
    else:
        fused_linear_mxfp4(x, w, x_scales=x_scales, out=hold[:T, :N])
        want = y.float()
    assert torch.equal(hold[:T, :N], want), _where(hold[:T, :N], want)
    assert (hold[T] == 7.0).all() and (hold[:, N:] == 7.0).all()


def _bounded(X, W, bias, act, residual, out, gated):
    K = X.shape[1]
    B, R = _np(bias), _np(residual)
    dot = np.abs(X) @ np.abs(W).T + (0.0 if B is None else np.abs(B))
    y = X @ W.T + (0.0 if B is None else B)
    ey = (K + K / 128 + 8) * 2.0 ** -23 * dot
    if gated:
        n = W.shape[0] // 2
        g, u = dense.activation(y[:, :n], act), y[:, n:]
        eg = 1.13 * ey[:, :n] + 2.0 ** -20 * np.abs(g) + 2.0 ** -22 * np.abs(y[:, :n])
        ref = g * u
        err = eg * (np.abs(u) + ey[:, n:]) + np.abs(g) * ey[:, n:]
    else:
        ref = dense.activation(y, act)
        err = 1.13 * ey + 2.0 ** -20 * np.abs(ref) + 2.0 ** -22 * np.abs(y)
        if R is not None:
            ref = ref + R
            err = err + 2.0 ** -24 * np.abs(ref)
    tiny = float(torch.finfo(out.dtype).tiny) * float(torch.finfo(out.dtype).eps)
    tol = err + HALF[out.dtype] * (np.abs(ref) + err) + tiny
    off = np.abs(_np(out) - ref)
    assert np.isfinite(_np(out)).all()
    assert (off <= tol).all(), f"worst {float((off / tol).max()):.3f} of the bound"


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh", "sigmoid"])
@pytest.mark.parametrize("T,K,N", [(1, 512, 96), (16, 1024, 80), (50, 352, 65), (130, 768, 144), (520, 256, 512)])
@pytest.mark.parametrize("kind", ["bf16", "f16", "x4"])
def test_real_values(T, K, N, act, kind, device):
    from exq_amd.kernels import Mxfp4Weight, fused_gated_linear_mxfp4, fused_linear_mxfp4, quantize_mxfp4
    banner(f"mxfp4 real T={T} K={K} N={N} {kind} {act}")
    dtype = torch.float16 if kind == "f16" else torch.bfloat16
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, K, generator=g).to(dtype).cuda()
    gated = act is not None
    weight = torch.randn(2 * N, K, generator=g) * 0.05
    x_scales, X = None, _np(x)
    if kind == "x4":
        x, x_scales = quantize_mxfp4(x)
        X = mxfp4.dequantize(x.cpu().numpy(), x_scales.cpu().numpy())
    for out_dtype in (dtype, torch.float32):
        for bias in (None, torch.randn(2 * N, generator=g).to(dtype).cuda()):
            for is_gated in ((False, True) if gated else (False,)):
                rows = 2 * N if is_gated else N
                p, s = quantize_mxfp4(weight[:rows].cuda())
                W = mxfp4.dequantize(p.cpu().numpy(), s.cpu().numpy())
                w = Mxfp4Weight.from_packed(p, s, is_gated)
                b = None if bias is None else bias[:rows]
                if is_gated:
                    out = fused_gated_linear_mxfp4(x, w, b, x_scales=x_scales, activation=act, out_dtype=out_dtype)
                    _bounded(X, W, b, act, None, out, True)
                else:
                    r = torch.randn(T, N, generator=g).to(out_dtype).cuda()
                    out = fused_linear_mxfp4(x, w, b, x_scales=x_scales, activation=act, residual=r, out_dtype=out_dtype)
                    _bounded(X, W, b, act, r, out, False)


@pytest.mark.parametrize("T", [1, 5, 64, 200])
@pytest.mark.parametrize("kind", ["bf16", "f16", "x4"])
def test_strides_and_neighbours(T, kind, device):
    """Column slices and unaligned rows; what lies beside them is neither read nor written."""
    from exq_amd.kernels import Mxfp4Weight, fused_linear_mxfp4
    K, N = 352, 75
    packed, scales = _codes(N, K, 1, -1, 1)
    w = Mxfp4Weight.from_packed(packed.cuda(), scales.cuda())
    for lead, width in ((0, K + 64), (16, K + 48), (3, K + 7), (0, K)):
        if kind == "x4":
            xp, xs = _codes(T, K, 2, -1, 1)
            buf = torch.full((T, lead + width), 0xFF, dtype=torch.uint8).cuda()
            buf[:, lead:lead + K // 2] = xp.cuda()
            x, x_scales, X = buf[:, lead:lead + K // 2], xs.cuda(), _dense(xp, xs)
        else:
            dtype = torch.bfloat16 if kind == "bf16" else torch.float16
            X = torch.randint(-3, 4, (T, K), generator=torch.Generator().manual_seed(2)).double()
            buf = torch.full((T, lead + width), float("nan"), dtype=dtype).cuda()
            buf[:, lead:lead + K] = X.to(dtype).cuda()
            x, x_scales = buf[:, lead:lead + K], None
        y = (X @ _dense(packed, scales).t()).float()
        hold = torch.full((T + 2, N + 9), 7.0).cuda()
        out = fused_linear_mxfp4(x, w, x_scales=x_scales, out=hold[1:-1, 4:4 + N])
        assert torch.equal(out.cpu(), y), _where(out.cpu(), y)
        hold[1:-1, 4:4 + N] = 7.0
        assert (hold == 7.0).all()
        r = torch.randint(-9, 10, (T, N + 5)).float().cuda()
        want = y + r[:, 2:2 + N].cpu()
        fused_linear_mxfp4(x, w, x_scales=x_scales, residual=r[:, 2:2 + N], out=r[:, 2:2 + N])
        assert torch.equal(r[:, 2:2 + N].cpu(), want)
    if kind != "x4":   # one row for all tokens
        out = fused_linear_mxfp4(x[:1].expand(T, K), w, out_dtype=torch.float32)
        assert torch.equal(out.cpu(), y[:1].expand(T, N))
    assert fused_linear_mxfp4(x[:0], w, x_scales=None if x_scales is None else x_scales[:0]).shape == (0, N)


def test_overlaps_are_refused(device):
    """out anywhere in an input but the residual, a workspace in the layer's inputs."""
    from exq_amd.kernels import Mxfp4Weight, fused_experts_mxfp4, fused_linear_mxfp4
    T, K, N = 8, 256, 64
    packed, scales = _codes(N, K, 1, 0, 0)
    w = Mxfp4Weight.from_packed(packed.cuda(), scales.cuda())
    x = torch.ones(T, K, dtype=torch.bfloat16).cuda()
    tail = w.tiles.view(-1)[-2 * T * N:].view(torch.bfloat16).view(T, N)
    wide = Mxfp4Weight(w.tiles, torch.zeros(2 * T * N, dtype=torch.uint8).cuda()[:w.tile_scales.numel()]
                       .view(w.tile_scales.shape), N, K)
    in_scales = wide.tile_scales.view(-1)[:2 * 4 * N].view(torch.bfloat16).view(4, N)
    xp, xs = (t.cuda() for t in _codes(64, K, 2, 0, 0))
    for call in (lambda: fused_linear_mxfp4(x, w, out=tail),
                 lambda: fused_linear_mxfp4(x[:4], wide, out=in_scales),
                 lambda: fused_linear_mxfp4(x, w, out=x[:, :N]),
                 lambda: fused_linear_mxfp4(xp[:1], w, x_scales=xs[:1], out=xp[:1, :N * 2].view(torch.bfloat16)),
                 lambda: fused_linear_mxfp4(x, w, residual=x[:, :N], out=x[:, 1:N + 1])):
        with pytest.raises(ValueError, match="overlap"):
            call()
    h, _, _, w13, w2, ids, wts = _layer(4, 64, 64, 4, 2, torch.bfloat16, 1)
    with pytest.raises(ValueError, match="workspace overlaps"):
        fused_experts_mxfp4(h, w13, w2, wts, ids, workspace=w13.tiles.view(-1))


@pytest.mark.parametrize("T", [3, 70, 300])
@pytest.mark.parametrize("kind", ["bf16", "x4"])
def test_nan_and_infinity_stay_in_their_row_and_column(T, kind, device):
    from exq_amd.kernels import Mxfp4Weight, fused_linear_mxfp4
    K, N = 288, 90
    packed, scales = _codes(N, K, 1, 0, 0)
    scales[7, 3] = 255
    w = Mxfp4Weight.from_packed(packed.cuda(), scales.cuda())
    if kind == "x4":
        xp, xs = _codes(T, K, 2, 0, 0)
        xs[2, 8] = 255
        out = fused_linear_mxfp4(xp.cuda(), w, x_scales=xs.cuda(), out_dtype=torch.float32).cpu()
        X = _dense(xp, xs)
    else:
        X = torch.randint(-3, 4, (T, K), generator=torch.Generator().manual_seed(2)).double()
        X[2, K - 1] = float("nan")
        out = fused_linear_mxfp4(X.to(torch.bfloat16).cuda(), w, out_dtype=torch.float32).cpu()
    want = torch.zeros(T, N)
    fine = torch.ones(T, N, dtype=torch.bool)
    fine[2], fine[:, 7] = False, False
    want = (X.nan_to_num(0.0) @ _dense(packed, scales).nan_to_num(0.0).t()).float()
    assert torch.equal(out[fine], want[fine])
    assert out[~fine].isnan().all()


def test_extreme_scales(device):
    """Weights at both ends of the scales' range, in bfloat16 exactly."""
    from exq_amd.kernels import Mxfp4Weight, fused_linear_mxfp4
    packed, _ = _codes(48, 64, 4, 0, 0)
    packed &= 0x77
    for s in (0, 1, 2, 100, 200, 250):
        scales = torch.full((48, 2), s, dtype=torch.uint8)
        w = Mxfp4Weight.from_packed(packed.cuda(), scales.cuda())
        x = torch.zeros(2, 64, dtype=torch.bfloat16)
        x[0, 5], x[1, 60] = 1.0, 2.0
        out = fused_linear_mxfp4(x.cuda(), w, out_dtype=torch.float32).cpu()
        want = (x.double() @ _dense(packed, scales).t()).float()
        assert torch.equal(out, want)


# ---- MoE layer --------------------------------------------------------------------------------

def _layer(T, H, I, E, k, dtype, seed, ids=None, zipf=0.0):
    from exq_amd.kernels import Mxfp4Weight, quantize_mxfp4
    g = torch.Generator().manual_seed(seed)
    p13, s13 = quantize_mxfp4((torch.randn(E, 2 * I, H, generator=g) * 0.1).cuda())
    p2, s2 = quantize_mxfp4((torch.randn(E, H, I, generator=g) * 0.1).cuda())
    x = torch.randn(T, H, generator=g).to(dtype).cuda()
    if ids is None:
        logits = torch.randn(T, E, generator=g) - zipf * torch.log(torch.arange(E) + 1.0)
        ids = logits.topk(k, -1).indices
    w = torch.rand(T, k, generator=g) + 0.1
    return x, (p13, s13), (p2, s2), Mxfp4Weight.from_packed(p13, s13, True), \
        Mxfp4Weight.from_packed(p2, s2), ids.to(torch.int32).cuda(), w.cuda()


def _layer_bound(x, st13, st2, ids, wts):
    """(reference, bound) [T, H] in float64: the sums' errors, the rounding of silu(gate) * up
    and of the result (added by the caller)."""
    X, T, k = _np(x), x.shape[0], ids.shape[1]
    half = HALF[x.dtype]
    p13, s13, p2, s2 = (t.cpu().numpy() for t in (*st13, *st2))
    E, I, H = p13.shape[0], p13.shape[1] // 2, X.shape[1]
    ref, tol = np.zeros((T, p2.shape[1])), np.zeros((T, p2.shape[1]))
    idn, wn = ids.cpu().numpy(), _np(wts)
    for e in range(E):
        t, j = np.nonzero(idn == e)
        if not t.size:
            continue
        w13, w2 = mxfp4.dequantize(p13[e], s13[e]), mxfp4.dequantize(p2[e], s2[e])
        y = X[t] @ w13.T
        ey = (H + 8) * 2.0 ** -23 * (np.abs(X[t]) @ np.abs(w13).T)
        g, u = dense.activation(y[:, :I], "silu"), y[:, I:]
        eg = 1.13 * ey[:, :I] + 2.0 ** -20 * np.abs(g) + 2.0 ** -22 * np.abs(y[:, :I])
        mid = g * u
        em = eg * (np.abs(u) + ey[:, I:]) + np.abs(g) * ey[:, I:]
        em = em + half * (np.abs(mid) + em) + float(torch.finfo(x.dtype).tiny) * float(torch.finfo(x.dtype).eps)
        out = mid @ w2.T
        eo = em @ np.abs(w2).T + (I + 8) * 2.0 ** -23 * ((np.abs(mid) + em) @ np.abs(w2).T)
        wt = wn[t, j][:, None]
        np.add.at(ref, t, wt * out)
        np.add.at(tol, t, np.abs(wt) * (eo + (k + 2) * 2.0 ** -23 * (np.abs(out) + eo)))
    return ref, tol


def _check_layer(x, st13, st2, w13, w2, ids, wts, **kw):
    from exq_amd.kernels import fused_experts_mxfp4
    out = fused_experts_mxfp4(x, w13, w2, wts, ids, **kw)
    ref, tol = _layer_bound(x, st13, st2, ids, wts)
    tol = tol + HALF[x.dtype] * (np.abs(ref) + tol) + float(torch.finfo(x.dtype).tiny)
    off = np.abs(_np(out) - ref)
    assert np.isfinite(_np(out)).all()
    assert (off <= tol).all(), f"worst {float((off / tol).max()):.3f} of the bound"
    rel = np.linalg.norm(off) / max(np.linalg.norm(ref), 1e-30)
    print(f"[parity] mxfp4 layer T={x.shape[0]} rel_l2={rel:.3e}", flush=True)
    return out


# T, H, I, E, k: one token to prefill, one expert, odd blocks, experts without tokens
LAYERS = [
    (1, 32, 32, 1, 1), (1, 256, 128, 8, 2), (1, 2048, 768, 16, 8), (2, 160, 96, 5, 3), (3, 512, 288, 64, 6),
    (4, 1024, 256, 128, 8), (7, 96, 544, 3, 2), (8, 256, 256, 16, 8), (16, 512, 192, 60, 4), (17, 128, 64, 2, 1),
    (33, 288, 160, 7, 3), (64, 512, 384, 128, 8), (64, 256, 256, 8, 2), (65, 256, 128, 16, 4), (100, 128, 1024, 4, 2),
    (187, 512, 224, 32, 8), (300, 256, 96, 8, 2), (513, 128, 128, 3, 1), (700, 96, 160, 40, 5), (1030, 64, 64, 9, 2),
    # either side of 16, 32, 64, 128 and 512 slots and of 512 and 1,024 experts' routing
    (16, 96, 64, 4, 1), (17, 96, 64, 4, 1), (2, 64, 64, 1024, 16), (3, 64, 64, 1024, 11), (64, 64, 32, 2, 1),
    (65, 64, 32, 1024, 1), (128, 64, 64, 6, 1), (43, 64, 64, 512, 3), (64, 64, 96, 512, 8), (65, 96, 64, 64, 8),
    (40, 64, 64, 600, 4), (129, 64, 32, 1024, 4), (1, 64, 64, 300, 64),
    # 512 and more work-groups of each number of weight tiles a wave, and ragged last ones
    (96, 1056, 160, 64, 4), (40, 2080, 1056, 8, 2), (200, 2048, 1056, 8, 2), (150, 4128, 96, 8, 2),
]


@pytest.mark.parametrize("T,H,I,E,k", LAYERS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer(T, H, I, E, k, dtype, device):
    banner(f"mxfp4 layer T={T} H={H} I={I} E={E} k={k} {dtype}")
    _check_layer(*_layer(T, H, I, E, k, dtype, T + H, zipf=0.8))


@pytest.mark.parametrize("T", [1, 3, 16, 60, 150])
def test_layer_odd_routing(T, device):
    """Ids that repeat within a token, ids of no expert, tokens without any, all on one expert."""
    E, k = 12, 4
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-3, E + 3, (T, k), generator=g)
    ids[::3, 1] = ids[::3, 0]
    ids[T // 2] = -1
    banner(f"mxfp4 odd routing T={T}")
    x, st13, st2, w13, w2, ids, w = _layer(T, 160, 96, E, k, torch.bfloat16, 4, ids)
    w[T // 2] = float("nan")           # (of dropped slots: not read)
    x[T // 2] = float("inf")           # (nor the token's row)
    from exq_amd.kernels import fused_experts_mxfp4
    out = fused_experts_mxfp4(x, w13, w2, w, ids)
    assert (out[T // 2] == 0).all()
    x[T // 2], w[T // 2] = 0.0, 0.0
    assert torch.equal(_check_layer(x, st13, st2, w13, w2, ids, w), out)
    assert torch.equal(fused_experts_mxfp4(x, w13, w2, w, ids.long()), out)
    _check_layer(x, st13, st2, w13, w2, torch.full_like(ids, 5), w)
    none = fused_experts_mxfp4(x, w13, w2, w, torch.full_like(ids, E))
    assert (none == 0).all()


@pytest.mark.parametrize("T", [1, 8, 64, 200])
def test_layer_buffers(T, device):
    """out, workspace of any contents, weights of each type, repeated calls bit for bit."""
    from exq_amd.kernels import fused_experts_mxfp4
    from exq_amd.kernels.mxfp4 import moe_mxfp4_workspace_bytes
    x, st13, st2, w13, w2, ids, w = _layer(T, 256, 128, 16, 4, torch.bfloat16, 7)
    first = _check_layer(x, st13, st2, w13, w2, ids, w)
    need = moe_mxfp4_workspace_bytes(T, 256, 128, 16, 4)
    for fill in (0, 255):
        ws = torch.full((need + 512,), fill, dtype=torch.uint8, device=x.device)
        out = torch.full_like(x, float("nan"))
        got = fused_experts_mxfp4(x, w13, w2, w, ids, out=out, workspace=ws[:need])
        assert got is out and torch.equal(out, first)
        assert (ws[need:] == fill).all()
    for dtype in (torch.float16, torch.bfloat16):
        _check_layer(x, st13, st2, w13, w2, ids, w.to(dtype))
    with pytest.raises(Exception, match="workspace"):
        fused_experts_mxfp4(x, w13, w2, w, ids, workspace=ws[:need - 1])
    with pytest.raises(ValueError, match="overlaps"):
        fused_experts_mxfp4(x, w13, w2, w, ids, out=x)


@pytest.mark.parametrize("T", [2, 40, 130])
def test_layer_row_of_nan(T, device):
    """A token that is not finite spoils no other."""
    from exq_amd.kernels import fused_experts_mxfp4
    x, st13, st2, w13, w2, ids, w = _layer(T, 128, 64, 4, 2, torch.bfloat16, 9)
    first = fused_experts_mxfp4(x, w13, w2, w, ids)
    bad = x.clone()
    bad[1, 3] = float("nan")
    out = fused_experts_mxfp4(bad, w13, w2, w, ids)
    assert out[1].isnan().all()
    out[1] = first[1]
    assert torch.equal(out, first)


# ---- as they are used -------------------------------------------------------------------------

@pytest.mark.parametrize("T", [1, 16, 100])
def test_block(T, device):
    """Router, routed experts and a shared expert onto them, all in MXFP4, in eager mode, on
    another stream and from a replayed graph."""
    from exq_amd.kernels import (Mxfp4Weight, fused_experts_mxfp4, fused_gated_linear_mxfp4, fused_linear,
                                 fused_linear_mxfp4, grouped_topk, quantize_mxfp4)
    H, I, E = 256, 128, 16
    x, st13, st2, w13, w2, _, _ = _layer(T, H, I, E, 4, torch.bfloat16, 11)
    g = torch.Generator().manual_seed(1)
    gate = torch.randn(E, H, generator=g).to(torch.bfloat16).cuda()
    s13 = Mxfp4Weight.quantize((torch.randn(2 * I, H, generator=g) * 0.1).cuda(), gated=True)
    s2 = Mxfp4Weight.quantize((torch.randn(H, I, generator=g) * 0.1).cuda())

    def block(x):
        w, ids = grouped_topk(fused_linear(x, gate, out_dtype=torch.float32), 4, True)
        routed = fused_experts_mxfp4(x, w13, w2, w, ids)
        mid, mid_scales = quantize_mxfp4(fused_gated_linear_mxfp4(x, s13))
        return fused_linear_mxfp4(mid, s2, x_scales=mid_scales, residual=routed, out=routed)

    first = block(x)
    w, ids = grouped_topk(fused_linear(x, gate, out_dtype=torch.float32), 4, True)
    ref, _ = _layer_bound(x, st13, st2, ids, w)
    routed = fused_experts_mxfp4(x, w13, w2, w, ids)
    m, ms = quantize_mxfp4(fused_gated_linear_mxfp4(x, s13))
    shared = fused_linear_mxfp4(m, s2, x_scales=ms, out_dtype=torch.float32)
    assert np.linalg.norm(_np(routed) - ref) <= 5e-3 * np.linalg.norm(ref)
    assert torch.equal(first, (shared + routed.float()).to(torch.bfloat16))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = block(x)
    side.synchronize()
    assert torch.equal(other, first)
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block(xs)
    for seed in range(4):
        new = torch.randn(T, H, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
        want = block(new)
        xs.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want)


@pytest.mark.parametrize("T", [1, 3, 30, 90])
def test_two_streams_at_once(T, device):
    """Calls in flight on two streams: a workspace each."""
    from exq_amd.kernels import fused_experts_mxfp4
    a = _layer(T, 512, 256, 16, 4, torch.bfloat16, 1)
    b = _layer(T, 512, 256, 16, 4, torch.bfloat16, 2)
    want = [fused_experts_mxfp4(x, w13, w2, w, ids) for x, _, _, w13, w2, ids, w in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (x, _, _, w13, w2, ids, w) in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(fused_experts_mxfp4(x, w13, w2, w, ids))
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        assert all(torch.equal(o, ref) for o in got)


def test_two_graphs_at_once(device):
    """Two graphs of the layer, captured one after the other, replayed on two streams."""
    from exq_amd.kernels import fused_experts_mxfp4
    a = _layer(48, 512, 256, 16, 4, torch.bfloat16, 1)
    b = _layer(48, 512, 256, 16, 4, torch.bfloat16, 2)
    want, graphs, outs = [], [], []
    for x, _, _, w13, w2, ids, w in (a, b):
        want.append(fused_experts_mxfp4(x, w13, w2, w, ids))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fused_experts_mxfp4(x, w13, w2, w, ids))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out, ref in zip(outs, want):
        assert torch.equal(out, ref)
