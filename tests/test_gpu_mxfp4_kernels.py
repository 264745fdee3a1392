"""Every dense MXFP4 kernel in every type of tokens, over contractions that go round its stages
more than twice, with the whole epilogue and with NaN scales.

Whole numbers: a weight is a multiple of 1/2 up to 6, a token of 1 up to 3 (in MXFP4 of 1/2
up to 6), so sums of 2,080 products are multiples of 1/4 below 2^17, exact in float32 in any
order and in the 4-bit instructions; the product of a gated pair and the result are rounded
once each, as here.  Compared bit for bit with products in 64 bits."""
import pytest
import torch

from exq_amd import _lib
from tests._helpers import banner
from tests._mxfp4_cases import cases

pytestmark = pytest.mark.gpu

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}

# (tokens, gated, kernel, T, N)
KERNELS = [("x4" if x4 else kind, gated, kernel, T, N) for x4, gated, kernel, T, N in cases()
           for kind in (("x4",) if x4 else ("bf16", "f16"))]
FIRST = list({k[:3]: k for k in reversed(KERNELS)}.values())      # one size of each kernel


def _stored(rows, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    packed = torch.randint(0, 256, (rows, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    return packed, torch.full((rows, K // 32), 127, device="cuda", dtype=torch.uint8)


def _values(packed):
    """Values of codes whose scales are 1."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device="cuda")
    return table[torch.stack((packed & 15, packed >> 4), -1).flatten(-2).int()]


def _inputs(kind, gated, T, N, K):
    packed, scales = _stored(2 * N if gated else N, K, 1)
    if kind == "x4":
        x, xs = _stored(T, K, 2)
        return packed, scales, x, xs, _values(x)
    g = torch.Generator(device="cuda").manual_seed(2)
    X = torch.randint(-3, 4, (T, K), generator=g, device="cuda").double()
    return packed, scales, X.to(TYPES[kind]), None, X


def _reaches(kind, gated, kernel, T, N, K):
    got = _lib.lib().exq_linear_mxfp4_kernel(_lib.LinearProblem(
        T, K, N, K // (2 if kind == "x4" else 1), 0, 0, -(-N // 4) * 4 + 4,
        {"x4": _lib.U8, "bf16": _lib.BF16, "f16": _lib.F16}[kind], 0, 0, _lib.F32, 0, gated))
    assert got.decode() == kernel


def _padded(T, N, dtype):
    return torch.full((T + 1, -(-N // 4) * 4 + 4), 7.0, device="cuda", dtype=dtype)


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


@pytest.mark.parametrize("K", [1696, 2080])
@pytest.mark.parametrize("kind,gated,kernel,T,N", KERNELS)
def test_many_stages(kind, gated, kernel, T, N, K, device):
    from exq_amd.kernels import Mxfp4Weight, fused_gated_linear_mxfp4, fused_linear_mxfp4
    banner(f"mxfp4 stages {kernel} {kind} gated={gated} T={T} N={N} K={K}")
    _reaches(kind, gated, kernel, T, N, K)
    packed, scales, x, xs, X = _inputs(kind, gated, T, N, K)
    w = Mxfp4Weight.from_packed(packed, scales, gated)
    y = torch.mm(X, _values(packed).t().contiguous())
    hold = _padded(T, N, torch.float32)
    if gated:
        fused_gated_linear_mxfp4(x, w, x_scales=xs, activation="relu", out=hold[:T, :N])
        y = torch.relu(y[:, :N]) * y[:, N:]
    else:
        fused_linear_mxfp4(x, w, x_scales=xs, out=hold[:T, :N])
    assert torch.equal(hold[:T, :N], y.float())
    assert (hold[T] == 7.0).all() and (hold[:, N:] == 7.0).all()


@pytest.mark.parametrize("kind,gated,kernel,T,N", FIRST)
def test_whole_epilogue(kind, gated, kernel, T, N, device):
    """Bias, activation, residual in place and a result of 16 bits."""
    from exq_amd.kernels import Mxfp4Weight, fused_gated_linear_mxfp4, fused_linear_mxfp4
    K = 224
    banner(f"mxfp4 epilogue {kernel} {kind} gated={gated} T={T} N={N}")
    _reaches(kind, gated, kernel, T, N, K)
    packed, scales, x, xs, X = _inputs(kind, gated, T, N, K)
    w = Mxfp4Weight.from_packed(packed, scales, gated)
    o = torch.float16 if kind == "f16" else torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    b = torch.randint(-40, 41, (packed.shape[0],), generator=g, device="cuda").to(o)
    y = torch.mm(X, _values(packed).t().contiguous()) + b.double()
    hold = _padded(T, N, o)
    if gated:
        fused_gated_linear_mxfp4(x, w, b, x_scales=xs, activation="relu", out=hold[:T, :N])
        want = (torch.relu(y[:, :N]) * y[:, N:]).float().to(o)
    else:
        hold[:T, :N] = torch.randint(-90, 91, (T, N), generator=g, device="cuda").to(o)
        want = (torch.relu(y) + hold[:T, :N].double()).float().to(o)
        fused_linear_mxfp4(x, w, b, x_scales=xs, activation="relu", residual=hold[:T, :N],
                           out=hold[:T, :N])
    assert torch.equal(hold[:T, :N], want)
    assert (hold[T] == 7.0).all() and (hold[:, N:] == 7.0).all()


@pytest.mark.parametrize("kind,gated,kernel,T,N", FIRST)
def test_nan_scales_stay_in_their_row_and_column(kind, gated, kernel, T, N, device):
    from exq_amd.kernels import Mxfp4Weight, fused_gated_linear_mxfp4, fused_linear_mxfp4
    K = 416
    banner(f"mxfp4 nan {kernel} {kind} gated={gated} T={T} N={N}")
    _reaches(kind, gated, kernel, T, N, K)
    packed, scales, x, xs, X = _inputs(kind, gated, T, N, K)
    y = torch.mm(X, _values(packed).t().contiguous())
    column, row = N // 2, T // 2
    scales[column, 12] = 255                      # (the last block, alone in its tile)
    scales[packed.shape[0] - 1, 5] = 255
    bad = torch.zeros(T, N, dtype=torch.bool, device="cuda")
    bad[:, [column, N - 1]] = True
    if T > 1:
        bad[row] = True
        if kind == "x4":
            xs[row, 7] = 255
        else:
            x[row, K - 1] = float("nan")
    w = Mxfp4Weight.from_packed(packed, scales, gated)
    if gated:
        out = fused_gated_linear_mxfp4(x, w, x_scales=xs, activation="relu", out_dtype=torch.float32)
        y = torch.relu(y[:, :N]) * y[:, N:]
    else:
        out = fused_linear_mxfp4(x, w, x_scales=xs, out_dtype=torch.float32)
    y[bad] = float("nan")
    assert _same(out, y.float())
