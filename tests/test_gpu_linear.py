"""fused_linear and fused_gated_linear against 64-bit products.

Small whole numbers in the inputs make every float32 sum exact, so those results are
compared bit for bit: a lost, doubled or misplaced k, row or column shows at any size.
Real values are compared within a bound: a float32 sum of K products in any order is
off by at most (K + 8) * 2^-23 * sum |x w| (2^-23, not 2^-24, as the matrix units may
truncate), the activations' slopes are at most 1.13, the functions themselves are within
2^-20 of their value plus 2^-22 |y| (the cancellation of 1 + erf), and the result is
rounded once: half a step of its type."""
import numpy as np
import pytest
import torch

from oracle import dense
from tests._helpers import banner

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _ints(shape, seed, dtype, top=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g).to(dtype)


def _reals(shape, seed, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _np(t):
    return None if t is None else t.double().cpu().numpy()


def _exact(x, w, bias, residual, out, gated):
    """Whole-number inputs: the 64-bit result rounded to the output's type."""
    y = x.double().cpu() @ w.double().cpu().t()
    if bias is not None:
        y = y + bias.double().cpu()
    if gated:
        n = w.shape[0] // 2
        y = torch.relu(y[:, :n]) * y[:, n:]
    if residual is not None:
        y = y + residual.double().cpu()
    want = y.float().to(out.dtype)
    assert torch.equal(out.cpu(), want), _where(out.cpu(), want)


def _where(a, b):
    bad = (a != b).nonzero()
    return f"{bad.shape[0]} of {a.numel()} differ, first at {bad[0].tolist()}"


def _bounded(x, w, bias, act, residual, out, gated):
    K = x.shape[1]
    X, W, B, R = _np(x), _np(w), _np(bias), _np(residual)
    dot = np.abs(X) @ np.abs(W).T + (0.0 if B is None else np.abs(B))
    y = X @ W.T + (0.0 if B is None else B)
    ey = (K + 8) * 2.0 ** -23 * dot
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


# T, K, N: single tokens, every tile's edges, K below, at and past a step, odd layouts
SIZES = [
    (1, 64, 16), (1, 2048, 128), (1, 8, 1), (1, 1000, 2047), (2, 256, 60), (3, 4096, 48), (4, 1, 5),
    (5, 7, 3), (8, 72, 33), (15, 512, 256), (16, 2816, 512), (17, 96, 100), (31, 136, 160),
    (32, 1024, 64), (33, 328, 250), (48, 264, 8), (63, 2048, 127), (64, 2048, 320), (65, 640, 129),
    (100, 1280, 384), (127, 33, 257), (129, 128, 520), (187, 1000, 203), (200, 64, 1032),
    (256, 256, 256), (257, 192, 264), (300, 2048, 128), (384, 448, 640), (513, 1088, 96),
    (640, 320, 1100), (1025, 72, 255), (1030, 512, 776),
]


@pytest.mark.parametrize("T,K,N", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_whole_numbers(T, K, N, dtype, device):
    from exq_amd.kernels import fused_linear
    banner(f"linear T={T} K={K} N={N} {dtype}")
    x, w = _ints((T, K), 1, dtype).cuda(), _ints((N, K), 2, dtype).cuda()
    b, r = _ints((N,), 3, dtype, 40).cuda(), _ints((T, N), 4, dtype, 90).cuda()
    _exact(x, w, None, None, fused_linear(x, w, out_dtype=torch.float32), False)
    _exact(x, w, b, r, fused_linear(x, w, b, residual=r), False)
    _exact(x, w, b.float(), r.float(),
           fused_linear(x, w, b.float(), residual=r.float(), out_dtype=torch.float32), False)


@pytest.mark.parametrize("T,K,N", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gated_whole_numbers(T, K, N, dtype, device):
    from exq_amd.kernels import fused_gated_linear
    banner(f"gated T={T} K={K} I={N} {dtype}")
    # products of two sums below 2^24 / 2: sums of K products of -1, 0, 1
    x, w = _ints((T, K), 5, dtype, 1).cuda(), _ints((2 * N, K), 6, dtype, 1).cuda()
    b = _ints((2 * N,), 7, dtype, 9).cuda()
    out = fused_gated_linear(x, w, activation="relu", out_dtype=torch.float32)
    _exact(x, w, None, None, out, True)
    _exact(x, w, b, None, fused_gated_linear(x, w, b, activation="relu", out_dtype=torch.float32),
           True)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh", "sigmoid"])
@pytest.mark.parametrize("T,K,N", [(1, 512, 96), (16, 1024, 80), (50, 333, 65), (130, 768, 144),
                                   (520, 256, 512)])
def test_activations(act, T, K, N, device):
    from exq_amd.kernels import fused_gated_linear, fused_linear
    banner(f"activation {act} T={T} K={K} N={N}")
    for dtype in (torch.bfloat16, torch.float16):
        x, w = _reals((T, K), 1, dtype).cuda(), _reals((2 * N, K), 2, dtype, 0.1).cuda()
        b, r = _reals((2 * N,), 3, torch.float32).cuda(), _reals((T, 2 * N), 4, dtype).cuda()
        for odt in (None, torch.float32):
            out = fused_linear(x, w, b, activation=act, residual=r, out_dtype=odt)
            _bounded(x, w, b, act, r, out, False)
            if act is not None:
                out = fused_gated_linear(x, w, b, activation=act, out_dtype=odt)
                _bounded(x, w, b, act, None, out, True)


@pytest.mark.parametrize("T,K,N", [(1, 2048, 2048), (16, 8192, 64), (64, 2816, 256),
                                   (187, 1000, 129), (1000, 1024, 512)])
def test_real_values(T, K, N, device):
    from exq_amd.kernels import fused_linear
    banner(f"real values T={T} K={K} N={N}")
    for dtype in (torch.bfloat16, torch.float16):
        x, w = _reals((T, K), 11, dtype).cuda(), _reals((N, K), 12, dtype, 0.02).cuda()
        _bounded(x, w, None, None, None, fused_linear(x, w, out_dtype=torch.float32), False)
        _bounded(x, w, None, None, None, fused_linear(x, w), False)


@pytest.mark.parametrize("T", [1, 7, 40, 200, 700])
def test_strided_rows_and_in_place(T, device):
    """Column slices of wider buffers, misaligned ones among them, an expanded row as x
    and as residual, the result written over the residual; what lies beside is kept."""
    from exq_amd.kernels import fused_gated_linear, fused_linear
    banner(f"strides T={T}")
    K, N = 192, 136
    for dtype in (torch.bfloat16, torch.float16):
        for ox, ow, orr, oo in ((0, 0, 0, 0), (8, 16, 8, 8), (1, 0, 3, 0), (0, 5, 0, 1)):
            xb, wb = _ints((T, K + 40), 1, dtype).cuda(), _ints((N, K + 24), 2, dtype).cuda()
            rb = _ints((T, N + 16), 3, dtype, 50).cuda()
            ob = torch.full((T, N + 32), 7.0, dtype=dtype, device=device)
            x, w, r = xb[:, ox:ox + K], wb[:, ow:ow + K], rb[:, orr:orr + N]
            out = ob[:, oo:oo + N]
            assert fused_linear(x, w, residual=r, out=out) is out
            _exact(x, w, None, r, out, False)
            assert bool((ob[:, :oo] == 7).all()) and bool((ob[:, oo + N:] == 7).all())
            keep = rb.clone()
            fused_linear(x, w, residual=r, out=r)   # in place
            _exact(x, w, None, keep[:, orr:orr + N], r, False)
            assert torch.equal(rb[:, :orr], keep[:, :orr])
            assert torch.equal(rb[:, orr + N:], keep[:, orr + N:])
            g = ob[:, oo:oo + N // 2]
            fused_gated_linear(x, w, activation="relu", out=g)
            _exact(x, w, None, None, g, True)
        x1, r1 = xb[:1, :K].expand(T, K), rb[:1, :N].expand(T, N)
        _exact(x1, w, None, r1, fused_linear(x1, w, residual=r1), False)


def test_refusals_on_the_device(device):
    from exq_amd.kernels import fused_linear
    x = torch.zeros(4, 16, dtype=torch.bfloat16, device=device)
    w = torch.zeros(16, 16, dtype=torch.bfloat16, device=device)
    r = torch.zeros(5, 16, dtype=torch.bfloat16, device=device)
    for kw in (dict(out=x), dict(residual=r[:4], out=r[1:]), dict(out=w[:4]),
               dict(out=r[:4], out_dtype=torch.float32), dict(out=r[:1].expand(4, 16)),
               dict(out=r[:3])):
        with pytest.raises(ValueError):
            fused_linear(x, w, **kw)
    with pytest.raises(RuntimeError, match="different devices"):
        fused_linear(x, w.cpu())
    assert fused_linear(x[:0], w).shape == (0, 16)


def test_special_values(device):
    """Infinities and NaN stay in their rows and columns; fp16 overflows to infinity."""
    from exq_amd.kernels import fused_linear
    banner("linear special values")
    for T in (3, 40, 300):
        x, w = _ints((T, 256), 1, torch.float16).cuda(), _ints((72, 256), 2, torch.float16).cuda()
        want = fused_linear(x, w)
        x2, w2 = x.clone(), w.clone()
        x2[1, 100] = float("nan")
        w2[70, 3] = float("inf")
        x2[:, 3] = 1.0
        w2[:70, 3] = w[:70, 3]
        got = fused_linear(x2, w2)
        ref = x2.float().cpu() @ w2.float().cpu().t()
        assert torch.equal(torch.isnan(got.float().cpu()), torch.isnan(ref))
        assert torch.equal(torch.isinf(got.float().cpu()), torch.isinf(ref))
        rows = [i for i in range(T) if i != 1]
        x3 = x.clone()
        x3[:, 3] = 1.0
        assert torch.equal(got[rows, :70], fused_linear(x3, w)[rows, :70])
        big = fused_linear(torch.full_like(x, 100.0), torch.full_like(w, 100.0))
        assert torch.isinf(big).all() and want.shape == big.shape


def test_large_offsets(device):
    """Rows that start past 2^32 bytes of x, W and out."""
    from exq_amd.kernels import fused_linear
    banner("linear large offsets")
    T, K, N, ld = 300, 128, 160, 8 << 20
    xb = torch.zeros(T * ld, dtype=torch.bfloat16, device=device)
    x = xb.view(T, ld)[:, 64:64 + K]
    x.copy_(_ints((T, K), 1, torch.bfloat16))
    w = _ints((N, K), 2, torch.bfloat16).cuda()
    _exact(x, w, None, None, fused_linear(x, w), False)
    _exact(x[:9], w, None, None, fused_linear(x[:9], w), False)
    wl = xb.view(T, ld)[:N, 4096:4096 + K]
    wl.copy_(w)
    x2 = x.contiguous()
    _exact(x2, w, None, None, fused_linear(x2, wl), False)
    _exact(x2[:5], w, None, None, fused_linear(x2[:5], wl), False)
    out = xb.view(T, ld)[:, 1 << 20:(1 << 20) + N]
    fused_linear(x2, w, out=out)
    _exact(x2, w, None, None, out, False)


def test_two_streams_at_once(device):
    """Calls on two streams, each kernel shape, and calls from tensors made on another
    stream: nothing is shared between them."""
    from exq_amd.kernels import fused_gated_linear, fused_linear
    banner("linear two streams")
    sizes = [(1, 2048, 512), (40, 1024, 256), (100, 777, 300), (300, 512, 640), (1100, 256, 2048),
             (2300, 320, 4100)]
    data = []
    for T, K, N in sizes:
        x, w = _ints((T, K), 1, torch.bfloat16).cuda(), _ints((2 * N, K), 2, torch.bfloat16, 1).cuda()
        data.append((x, w, fused_linear(x, w, out_dtype=torch.float32),
                     fused_gated_linear(x, w, activation="relu")))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for x, w, a, b in (data if i == 0 else data[::-1]):
                    outs.append((fused_linear(x, w, out_dtype=torch.float32), a))
                    outs.append((fused_gated_linear(x, w, activation="relu"), b))
    torch.cuda.synchronize()
    for got, want in outs:
        assert torch.equal(got, want)


def test_every_width_near_the_tiles(device):
    """T and N one below, at and above each tile's edges, K around a step."""
    from exq_amd.kernels import fused_linear
    banner("linear edges")
    for T in (255, 256, 257, 383, 385):
        for N in (255, 256, 257, 513):
            for K in (56, 64, 72, 120, 136):
                x, w = _ints((T, K), T, torch.bfloat16).cuda(), _ints((N, K), N, torch.bfloat16).cuda()
                _exact(x, w, None, None, fused_linear(x, w, out_dtype=torch.float32), False)


@pytest.mark.parametrize("T,K,N", [(2500, 192, 4096), (4100, 136, 4352), (1030, 4096, 520),
                                   (20000, 64, 128), (3, 16384, 72)])
def test_large_shapes_whole_numbers(T, K, N, device):
    """The largest tiles with ragged edges, long contractions, many token blocks."""
    from exq_amd.kernels import fused_gated_linear, fused_linear
    banner(f"large shapes T={T} K={K} N={N}")
    x, w = _ints((T, K), 1, torch.bfloat16, 1).cuda(), _ints((N, K), 2, torch.bfloat16, 1).cuda()
    r = _ints((T, N), 3, torch.bfloat16, 90).cuda()
    out = fused_linear(x, w, residual=r, out_dtype=torch.float32)
    y = x.double() @ w.double().t()
    assert torch.equal(out, (y + r.double()).float())
    half = N // 2 * 2
    g = fused_gated_linear(x, w[:half], activation="relu", out_dtype=torch.float32)
    assert torch.equal(g, (torch.relu(y[:, :half // 2]) * y[:, half // 2:half]).float())


@pytest.mark.parametrize("T,K,N", [(1, 1032, 4096), (5, 264, 8200), (16, 1096, 4104), (13, 135, 4097),
                                   (30, 72, 5000), (32, 2112, 2048), (27, 1025, 8200),
                                   (64, 1160, 1500), (500, 200, 64)])
def test_few_tokens_wide_whole_numbers(T, K, N, device):
    """Streams of 16 and of 32 weight rows on both sides of one round, waves without a
    step of their own, rows of any alignment."""
    from exq_amd.kernels import fused_gated_linear, fused_linear
    banner(f"few tokens, wide T={T} K={K} N={N}")
    for dtype in (torch.bfloat16, torch.float16):
        x, w = _ints((T, K), 1, dtype, 1).cuda(), _ints((N, K), 2, dtype, 1).cuda()
        r = _ints((T, N), 3, dtype, 90).cuda()
        y = x.double() @ w.double().t()
        out = fused_linear(x, w, residual=r, out_dtype=torch.float32)
        assert torch.equal(out, (y + r.double()).float())
        half = N // 2
        g = fused_gated_linear(x, w[:2 * half], activation="relu", out_dtype=torch.float32)
        assert torch.equal(g, (torch.relu(y[:, :half]) * y[:, half:2 * half]).float())


def test_moe_block(device):
    """The operators together, as a block runs them: router projection, grouped routing,
    routed experts, shared expert with its output added onto theirs; eager, and captured
    and replayed with other work between."""
    from exq_amd import synth
    from exq_amd.kernels import (fused_experts, fused_gated_linear, fused_linear, grouped_topk,
                                 pack_experts_int4)
    from oracle import moe
    from tests._helpers import assert_close_rel, oracle_int4_layer
    H, I, S, E, k = 512, 256, 384, 32, 4
    w13, w2 = synth.expert_weights_gpu(E, I, H, 8, device)
    banks = pack_experts_int4(w13) + pack_experts_int4(w2)
    gate = _reals((E, H), 1, torch.bfloat16, 0.05).cuda()
    bias = _reals((E,), 2, torch.float32, 0.05).cuda()
    s13 = _reals((2 * S, H), 3, torch.bfloat16, 0.02).cuda()
    s2 = _reals((H, S), 4, torch.bfloat16, 0.02).cuda()
    for T in (1, 16, 150):
        banner(f"moe block T={T}")
        x = _reals((T, H), 5 + T, torch.bfloat16).cuda()

        def block():
            logits = fused_linear(x, gate, out_dtype=torch.float32)
            w, ids = grouped_topk(logits, k, True, 8, 3, scoring_func="sigmoid",
                                  correction_bias=bias, routed_scaling_factor=2.5)
            routed = fused_experts(x, *banks, w, ids)
            mid = fused_gated_linear(x, s13)
            return logits, w, ids, fused_linear(mid, s2, residual=routed)

        logits, w, ids, out = block()
        _bounded(x, gate, None, None, None, logits, False)
        r_ids, r_w = dense.grouped_topk(_np(logits), k, True, 8, 3, "sigmoid", _np(bias), None, 2.5)
        assert np.array_equal(ids.cpu().numpy(), r_ids)
        np.testing.assert_allclose(_np(w), r_w, rtol=2.0 ** -20)
        ref = oracle_int4_layer(x, *banks, r_ids, r_w)
        ref = ref + dense.linear(dense.gated_linear(_np(x), _np(s13)), _np(s2))
        # three roundings to bf16 (2^-9 rms each at most) beside the layer's own 0.5 %
        assert_close_rel(out, ref.astype(np.float32), 8e-3, f"moe block T={T}")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            block()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            captured = block()
        for _ in range(3):
            for t in captured:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(captured, (logits, w, ids, out)):
                assert torch.equal(a, b)
            block()
            torch.cuda.synchronize()
