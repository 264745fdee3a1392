"""Every kernel of fused_linear and fused_gated_linear at its own tile edges, over contractions
that go round its ring of LDS stages more than twice, against 64-bit products.

Whole numbers, so that every float32 sum is exact (plain: at most 7240 products of at most 9;
gated: two sums whose product is below 2^24, which the test asserts) and results are
compared bit for bit: a lost, doubled or misplaced k, row or column shows.  Which kernel a
size reaches is checked without a GPU (tests/test_linear_kernels.py)."""
import pytest
import torch

from tests import _linear_cases as C
from tests._helpers import banner

pytestmark = pytest.mark.gpu

# contraction lengths: at least 2 * stages + 3 steps of the kernel with a part of one at the
# end, even and odd numbers of 64-k blocks for the tiles; then one block and less
STEPS = {"stream 16x16": (7240,), "stream 32x16": (4680,), "stream 16x32": (4680,),
         "stream 32x32": (3656,), "stream 64x32": (2376,), "tile 64x128": (1080, 1096)}


def _lengths(kernel):
    return (*STEPS.get(kernel, (776, 840)), 64, 8)


def _ints(shape, seed, dtype, top):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g, device="cuda", dtype=torch.int16).to(dtype)


def _plain(x, w, T, N, dtype, seed):
    """Three results: float32, the input's type with bias and residual, float32 into a wider
    buffer, whose other columns and rows stay as they are."""
    from exq_amd.kernels import fused_linear
    b, r = _ints((N,), seed + 3, dtype, 40), _ints((T, N), seed + 4, dtype, 90)
    y = x.double() @ w.double().t()
    assert torch.equal(fused_linear(x, w, out_dtype=torch.float32), y.float())
    want = (y + b.double() + r.double()).float()
    assert torch.equal(fused_linear(x, w, b, residual=r), want.to(dtype))
    buf = torch.full((T + 1, N + 12), -7.0, device="cuda")
    fused_linear(x, w, b.float(), residual=r.float(), out=buf[:T, 4:4 + N])
    assert torch.equal(buf[:T, 4:4 + N], want)
    buf[:T, 4:4 + N] = -7.0
    assert bool((buf == -7).all())


def _gated(x, w, T, N, dtype, seed):
    from exq_amd.kernels import fused_gated_linear
    b = _ints((2 * N,), seed + 3, dtype, 9)
    y = x.double() @ w.double().t()
    assert float((y.abs().amax() + 9) ** 2) < 2.0 ** 24
    want = (torch.relu(y[:, :N]) * y[:, N:]).float()
    assert torch.equal(fused_gated_linear(x, w, activation="relu", out_dtype=torch.float32), want)
    y += b.double()
    want = (torch.relu(y[:, :N]) * y[:, N:]).float()
    assert torch.equal(fused_gated_linear(x, w, b, activation="relu"), want.to(dtype))
    buf = torch.full((T + 1, N + 12), -7.0, device="cuda")
    fused_gated_linear(x, w, b.float(), activation="relu", out=buf[:T, 4:4 + N])
    assert torch.equal(buf[:T, 4:4 + N], want)
    buf[:T, 4:4 + N] = -7.0
    assert bool((buf == -7).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kernel,gated,T,N", list(C.aligned()))
def test_aligned_rows(kernel, gated, T, N, dtype, device):
    for K in _lengths(kernel):
        banner(f"{kernel} gated={gated} T={T} K={K} N={N} {dtype}")
        x = _ints((T, K), 1, dtype, 1 if gated else 3)
        w = _ints((N * (2 if gated else 1), K), 2, dtype, 1 if gated else 3)
        (_gated if gated else _plain)(x, w, T, N, dtype, K)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kernel,gated,T,N", list(C.unaligned()))
def test_any_layout(kernel, gated, T, N, dtype, device):
    """Odd rows, rows of four bytes, bases and strides in between."""
    for K, ox, ow, px, pw in ((1001, 0, 0, 0, 0), (1002, 0, 0, 0, 0), (776, 1, 0, 0, 8),
                              (776, 0, 3, 8, 0), (776, 2, 2, 0, 0), (840, 0, 0, 0, 1), (7, 0, 0, 0, 0)):
        banner(f"{kernel} gated={gated} T={T} K={K} N={N} {dtype} {ox} {ow} {px} {pw}")
        rows = N * (2 if gated else 1)
        xb = _ints((T, ox + K + px), 1, dtype, 1 if gated else 3)
        wb = _ints((rows, ow + K + pw), 2, dtype, 1 if gated else 3)
        (_gated if gated else _plain)(xb[:, ox:ox + K], wb[:, ow:ow + K], T, N, dtype, K)


@pytest.mark.parametrize("T,N", [(1537, 7169), (959, 8447), (513, 1100), (300, 4097), (600, 64),
                                 (20, 600), (5, 600)])
def test_rows_far_apart(T, N, device):
    """Rows 8 MiB apart, just inside what one buffer resource covers: the aligned kernels with
    offsets of a lane near 2^31 and rows past 2^32 bytes."""
    from exq_amd.kernels import fused_gated_linear, fused_linear
    K, ld = 136, 4 << 20
    for wide_x in (True, False):
        rows = T if wide_x else N
        if rows < 300:
            continue
        rows = min(rows, 1600)
        t, n = (rows, N) if wide_x else (T, rows)
        banner(f"rows far apart T={t} N={n} {'x' if wide_x else 'W'}")
        buf = torch.empty(rows * ld, dtype=torch.bfloat16, device=device).view(rows, ld)
        x, w = _ints((t, K), 1, torch.bfloat16, 1), _ints((n, K), 2, torch.bfloat16, 1)
        far = buf[:, ld - K:]                    # (the last columns of every row)
        far.copy_(x if wide_x else w)
        y = x.double() @ w.double().t()
        a, b = (far, w) if wide_x else (x, far)
        assert torch.equal(fused_linear(a, b, out_dtype=torch.float32), y.float())
        h = n // 2
        g = fused_gated_linear(a, b[:2 * h], activation="relu", out_dtype=torch.float32)
        assert torch.equal(g, (torch.relu(y[:, :h]) * y[:, h:2 * h]).float())
        del buf, far, a, b


def test_streams_and_replays(device):
    """Every kernel on two streams at once, and captured and replayed with eager calls between."""
    from exq_amd.kernels import fused_gated_linear, fused_linear
    banner("every kernel on two streams, captured and replayed")
    data = []
    for gated, table in ((False, C.PLAIN), (True, C.GATED), (False, C.ANY_PLAIN), (True, C.ANY_GATED)):
        K = 201 if table in (C.ANY_PLAIN, C.ANY_GATED) else 200
        for sizes in table.values():
            T, N = sizes[0]
            x = _ints((T, K), 1, torch.bfloat16, 1)
            w = _ints((N * (2 if gated else 1), K), 2, torch.bfloat16, 1)
            y = x.double() @ w.double().t()
            if gated:
                y = torch.relu(y[:, :N]) * y[:, N:]
            data.append((gated, x, w, y.float()))

    def run(items):
        return [(fused_gated_linear(x, w, activation="relu", out_dtype=torch.float32) if gated
                 else fused_linear(x, w, out_dtype=torch.float32), want) for gated, x, w, want in items]

    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(2):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs += run(data if i == 0 else data[::-1])
    torch.cuda.synchronize()
    assert all(torch.equal(got, want) for got, want in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = run(data)
    for _ in range(3):
        for got, _ in captured:
            got.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(got, want) for got, want in captured)
        assert all(torch.equal(got, want) for got, want in run(data))
