"""grouped_topk where a group's value is small beside what it is the sum of, or past the
largest float32: the order of the groups is that of the 64-bit oracle.

Ids exactly.  The oracle and the kernel both rank in 64 bits, and what their scores may
differ by (2^-52 of a score, rounded at the size of a bias of 1000: 2^-43) is far below the
spacing of the values here (logits some 1e-6 apart)."""
import numpy as np
import pytest
import torch

from oracle import dense
from tests._helpers import banner

pytestmark = pytest.mark.gpu


def _ids_match(logits, bias, k, G, keep, scoring, group_score="top2"):
    from exq_amd.kernels import grouped_topk
    _, ids = grouped_topk(torch.from_numpy(logits).cuda(), k, True, G, keep, scoring_func=scoring,
                          correction_bias=torch.from_numpy(bias).cuda(), group_score=group_score)
    want, _ = dense.grouped_topk(logits, k, True, G, keep, scoring, bias, group_score)
    got = ids.cpu().numpy()
    bad = np.flatnonzero((got != want).any(1))
    assert bad.size == 0, f"{bad.size} of {len(got)} rows, first {got[bad[0]]}, not {want[bad[0]]}"


@pytest.mark.parametrize("E,G,keep", [(8, 4, 2), (32, 2, 1), (64, 16, 5), (256, 8, 4), (512, 16, 7),
                                      (30, 10, 4)])
@pytest.mark.parametrize("size", [24.0, 1000.0])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_opposed_biases_in_a_group(E, G, keep, size, scoring, device):
    """The two best experts of every group have biases of +size and -size, so the roundings of
    their values are far larger than that of the sum of both."""
    banner(f"grouped_topk opposed biases of {size} E={E} G={G} keep={keep} {scoring}")
    rng = np.random.default_rng(E + G)
    T, gs = 400, E // G
    bias = np.full((G, gs), -2.0 * size)
    for g in range(G):
        hi, lo = rng.permutation(gs)[:2]
        bias[g, hi], bias[g, lo] = size, -size
    bias = bias.reshape(E).astype(np.float32)
    for step in (2e-5, 2e-6):
        lg = (rng.standard_normal((T, 1)) + step * rng.standard_normal((T, E))).astype(np.float32)
        for k in (1, min(keep * gs, 2 * keep)):
            _ids_match(lg, bias, k, G, keep, scoring)
        _ids_match(lg, bias, 1, G, keep, scoring, "max")


@pytest.mark.parametrize("E,G,keep", [(16, 8, 5), (32, 16, 7), (16, 4, 2), (48, 2, 1), (24, 6, 4)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_sums_past_the_largest_float(E, G, keep, scoring, device):
    """Sums of two biases beyond the range of float32, below and above, beside groups without
    an expert: 64 bits hold them, and a group with an expert comes before one without."""
    banner(f"grouped_topk sums past the largest float E={E} G={G} keep={keep} {scoring}")
    rng = np.random.default_rng(E)
    gs = E // G
    for sign in (-1.0, 1.0):
        for _ in range(20):
            bias = np.full((G, gs), -np.inf)
            bias[:, :2] = sign * rng.integers(20, 34, (G, 2)) * 1e37
            lg = rng.standard_normal((8, G, gs))
            lg[1:, 0] = -np.inf                         # no expert in the lowest groups
            lg[2:, G // 2] = np.nan
            lg[3:, 0, 0] = 0.0                          # (one)
            _ids_match(lg.reshape(8, E).astype(np.float32), bias.reshape(E).astype(np.float32),
                       2, G, keep, scoring)
    bias = rng.permutation(np.linspace(-1, 1, E) * 3.4e38)
    lg = rng.standard_normal((50, E)).astype(np.float32)
    _ids_match(lg, bias.astype(np.float32), 2, G, keep, scoring)


def test_largest_token_count(device):
    """The largest batch that the call takes, on the kernel with four rows a work-group."""
    banner("grouped_topk 2^26 - 1 tokens")
    from exq_amd.kernels import grouped_topk
    T = (1 << 26) - 1
    g = torch.Generator(device="cuda").manual_seed(3)
    lg = torch.randint(-8, 9, (T, 3), generator=g, device="cuda", dtype=torch.int8).bfloat16()
    w, ids = grouped_topk(lg, 1, True, 3, 2, weights_dtype=torch.bfloat16)
    a, b, c = lg.unbind(1)
    want = torch.where((a >= b) & (a >= c), 0, torch.where(b >= c, 1, 2))
    assert torch.equal(ids[:, 0], want.int())
    assert bool((w == 1).all())
