"""grouped_topk against the 64-bit oracle: ids exactly (the ranking is that of the
scores in 64 bits, ties to the lower id), weights within 2^-20 of the oracle's
relative (an exponential, a division and the final rounding, each a few 2^-24), and
within half a step of a narrower weights type."""
import itertools

import numpy as np
import pytest
import torch

from oracle import dense
from tests._helpers import banner

pytestmark = pytest.mark.gpu


def _check(logits, k, renorm, G=1, keep=1, scoring="softmax", bias=None, group_score=None,
           scale=1.0, n_valid=None, ids_dtype=torch.int32, w_dtype=torch.float32):
    from exq_amd.kernels import grouped_topk
    nv = None if n_valid is None else torch.tensor([n_valid], dtype=torch.int32, device="cuda")
    w, ids = grouped_topk(logits.cuda(), k, renorm, G, keep, scoring_func=scoring,
                          correction_bias=None if bias is None else bias.cuda(),
                          group_score=group_score, routed_scaling_factor=scale,
                          num_token_non_padded=nv, ids_dtype=ids_dtype, weights_dtype=w_dtype)
    torch.cuda.synchronize()
    r_ids, r_w = dense.grouped_topk(logits.double().numpy(), k, renorm, G, keep, scoring,
                                    None if bias is None else bias.double().numpy(), group_score,
                                    scale, n_valid)
    assert ids.dtype == ids_dtype and w.dtype == w_dtype
    got = ids.cpu().numpy().astype(np.int64)
    if group_score == "top2" and bias is None and not np.array_equal(got, r_ids):
        for t in np.flatnonzero((got != r_ids).any(1)):
            assert _tie_of_64_bits(logits[t].double().numpy(), got[t], G, keep, scoring)
            s = dense.grouped_topk(logits[t:t + 1].double().numpy(), logits.shape[1], False,
                                   scoring=scoring, scale=scale)
            assert not renorm
            r_ids[t], r_w[t] = got[t], s[1][0][[list(s[0][0]).index(e) for e in got[t]]]
    assert np.array_equal(got, r_ids)
    # the scale is a float32 in the call: half a step of it; then the type's own rounding
    rtol = 2.0 ** -20 + (0.0 if w_dtype == torch.float32 else torch.finfo(w_dtype).eps / 2)
    np.testing.assert_allclose(w.double().cpu().numpy(), r_w, rtol=rtol,
                               atol=float(torch.finfo(w_dtype).tiny))
    return ids, w


def _tie_of_64_bits(l, ids, G, keep, scoring):
    """Whether `ids` are the best experts of groups that may be the best ones: the sums of
    two scores that 64 bits cannot order are interchangeable.  A score is an exponential
    (off by at most 1 ulp, 2^-52, and so is the 1 + exp of it), a sum and a division
    (2^-53 each), so a sum of two is off by at most 2^-50 of itself on either side, and
    two of them by 2^-49; the logits 6e-8 apart of the test of near ties give sums like
    s(l + 8 d) + s(l + 6 d) and 2 s(l + 7 d), which differ by s''(l) d^2 = 3e-16."""
    x = l.astype(np.longdouble)
    s = 1 / (1 + np.exp(-x)) if scoring == "sigmoid" else np.exp(x - x.max())
    v = np.sort(s.reshape(G, -1), 1)[:, -2:].sum(1)
    edge = np.sort(v)[-keep]
    sure = [g for g in range(G) if v[g] > edge * (1 + 2.0 ** -49)]
    maybe = [g for g in range(G) if abs(v[g] - edge) <= edge * 2.0 ** -49]
    for rest in itertools.combinations(maybe, keep - len(sure)):
        inside = np.isin(np.arange(l.size) // (l.size // G), sure + list(rest))
        best = dense.grouped_topk(np.where(inside, l, -np.inf)[None], ids.size, False,
                                  scoring=scoring)[0][0]
        if np.array_equal(best, ids):
            return True
    return False


def _logits(T, E, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    return torch.from_numpy((rng.standard_normal((T, E)) * scale).astype(np.float32))


SHAPES = [  # T, E, k, groups, kept
    (1, 256, 8, 8, 4), (5, 256, 8, 8, 4), (333, 160, 6, 8, 3), (64, 64, 6, 1, 1), (33, 128, 8, 1, 1),
    (17, 60, 4, 1, 1), (9, 72, 8, 4, 2), (50, 512, 16, 16, 5), (7, 1024, 64, 32, 9),
    (40, 96, 5, 3, 2), (21, 20, 3, 10, 4), (4, 16, 2, 16, 2), (3, 8, 8, 8, 8), (2, 2, 1, 2, 1),
    (6, 1, 1, 1, 1), (130, 288, 16, 8, 3), (66, 352, 12, 16, 11), (12, 640, 10, 64, 7),
    (20, 512, 12, 16, 11), (9, 512, 24, 16, 4), (11, 256, 24, 8, 3), (9, 512, 30, 8, 4), (300, 256, 10, 8, 1),
    (33, 512, 11, 16, 8), (5, 384, 25, 4, 2), (40, 112, 9, 16, 5),
]


@pytest.mark.parametrize("T,E,k,G,keep", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("use_bias", [False, True])
def test_shapes(T, E, k, G, keep, scoring, use_bias, device):
    banner(f"grouped_topk T={T} E={E} k={k} G={G} keep={keep} {scoring} bias={use_bias}")
    rng = np.random.default_rng(E + T)
    scale = 0.2 if scoring == "sigmoid" else 0.3 / E
    bias = torch.from_numpy((scale * rng.standard_normal(E)).astype(np.float32)) if use_bias else None
    lg = _logits(T, E, 100 * E + k)
    for group_score in (("max", "top2") if G > 1 else (None,)):
        for renorm in (True, False):
            _check(lg, k, renorm, G, keep, scoring, bias, group_score, 2.5)


@pytest.mark.parametrize("ldt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bdt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wdt", [torch.float32, torch.bfloat16, torch.float16])
def test_types_and_exact_ties(ldt, bdt, wdt, device):
    """Narrow logits and biases have many equal ranks: the lower id and group win."""
    banner(f"grouped_topk {ldt} bias {bdt} weights {wdt}")
    rng = np.random.default_rng(9)
    lg = torch.from_numpy(rng.standard_normal((70, 256)).astype(np.float32)).to(ldt)
    lg[3] = 0.0
    lg[4, 100:120] = 4.0
    lg[5] = -1.0
    lg[5, 20:30:2] = 0.0
    lg[5, 21:31:2] = -0.0
    bias = torch.from_numpy((rng.integers(-3, 4, 256) / 16).astype(np.float32)).to(bdt)
    for scoring in ("softmax", "sigmoid"):
        for b in (None, bias, torch.zeros(256, dtype=bdt)):
            ids, _ = _check(lg, 8, True, 8, 4, scoring, b, w_dtype=wdt, ids_dtype=torch.int64)
            _check(lg, 8, False, 1, 1, scoring, b, w_dtype=wdt)


def test_near_ties_are_decided_in_64_bits(device):
    """Scores one part in 10^7 or less apart, and group values likewise: float32 sums
    would order them by their roundings."""
    banner("grouped_topk near ties")
    rng = np.random.default_rng(2)
    T, E = 256, 128
    base = rng.standard_normal((T, 1)).astype(np.float32)
    lg = torch.from_numpy(base + (rng.integers(-8, 9, (T, E)) * 6e-8).astype(np.float32))
    # a bias that undoes most of what the logits differ by
    bias = torch.from_numpy((rng.integers(-8, 9, E) * 3e-8 + 0.25).astype(np.float32))
    for scoring in ("softmax", "sigmoid"):
        _check(lg, 8, True, 8, 4, scoring, bias)
        _check(lg, 8, False, 8, 4, scoring, None, "top2")
        _check(lg, 6, False, 1, 1, scoring, bias)


@pytest.mark.parametrize("k", [1, 6, 10, 11, 24])
def test_few_near_ties(k, device):
    """Two scores or two groups of some rows a rounding apart, the others far: among the
    chosen, at the k-th place, below it, and where one is no candidate."""
    banner(f"grouped_topk few near ties k={k}")
    rng = np.random.default_rng(k)
    for E, G, keep in ((256, 1, 1), (256, 8, 4), (96, 4, 2), (512, 16, 12)):
        T = 200
        lg = rng.standard_normal((T, E)).astype(np.float32)
        bias = (0.05 * rng.standard_normal(E)).astype(np.float32)
        r = 1 / (1 + np.exp(-lg.astype(np.float64))) + bias
        order = np.argsort(-r, axis=1)
        for t in range(T):   # expert b's logit set so that its rank value is a's, or next to it
            i = rng.integers(0, min(E - 2, k + 3))
            a, b = order[t, i], order[t, i + 1 + int(rng.integers(0, 2))]
            s = min(max(r[t, a] - bias[b], 1e-3), 1 - 1e-3) + rng.integers(-2, 3) * 2.0 ** -26
            lg[t, b] = np.float32(np.log(s / (1 - s)))
        _check(torch.from_numpy(lg), k, True, G, keep, "sigmoid", torch.from_numpy(bias))
        _check(torch.from_numpy(lg), k, False, G, keep, "sigmoid", torch.from_numpy(bias), "max")
        _check(torch.from_numpy(lg), k, True, G, keep, "softmax", torch.from_numpy(bias / E))


@pytest.mark.parametrize("k", [1, 8, 10, 16, 24])
def test_few_near_ties_of_softmax(k, device):
    """The same for softmax scores with a bias, whose sum over the experts moves with the
    logit that is set: some rows a rounding of 32 bits apart, some of much less."""
    banner(f"grouped_topk few near ties of softmax k={k}")
    rng = np.random.default_rng(50 + k)
    for E, G, keep in ((349, 1, 1), (64, 1, 1), (512, 2, 1), (512, 4, 3), (512, 8, 5), (256, 8, 4),
                       (512, 16, 12)):
        T = 120
        lg = rng.standard_normal((T, E)).astype(np.float32)
        bias = (0.3 / E * rng.standard_normal(E)).astype(np.float32)
        for t in range(T):
            e = np.exp(lg[t].astype(np.float64))
            order = np.argsort(-(e / e.sum() + bias))
            i = rng.integers(0, min(E - 2, k + 3))
            a, b = order[i], order[i + 1 + int(rng.integers(0, 2))]
            d = float(bias[b]) - float(bias[a])
            # e_a / S + bias_a = y / S + bias_b with S = (sum of the others) + y
            y = (e[a] - d * (e.sum() - e[b])) / (1 + d) * (1 + rng.integers(-3, 4) * 2.0 ** -22)
            if y > 1e-3:
                lg[t, b] = np.float32(np.log(y))
        lg[0], lg[1, :] = lg[0, 0], lg[1, :1]           # (all equal: the bias decides)
        lg[2, ::2] = lg[2, 1::2][:lg[2, ::2].size] if E % 2 == 0 else lg[2, ::2]
        for rn in (True, False):
            _check(torch.from_numpy(lg), k, rn, G, keep, "softmax", torch.from_numpy(bias))
        flat = torch.zeros(E)                           # (equal logits tie: the lower id)
        _check(torch.from_numpy(lg), k, True, G, keep, "softmax", flat)
        _check(torch.from_numpy(lg).bfloat16(), k, True, G, keep, "softmax", flat)
        _check(torch.from_numpy(lg * 60).float(), k, False, G, keep, "softmax", flat)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masks(scoring, device):
    """-inf and NaN in logits and bias, rows and groups without an expert left, +inf,
    the type's lowest and largest values, scores that all underflow."""
    banner(f"grouped_topk masks {scoring}")
    inf, nan, big = float("inf"), float("nan"), torch.finfo(torch.float32).max
    lg = _logits(16, 32, 4)
    lg[0] = -inf
    lg[1, 3:] = -inf
    lg[2, ::2] = nan
    lg[3] = nan
    lg[4, 5] = inf
    lg[5, [2, 9]] = inf
    lg[6, 8:] = -big
    lg[7] = -big
    lg[8] = big
    lg[9] = -inf
    lg[9, 31] = 0.0
    lg[10] = torch.linspace(-1000, -900, 32)
    lg[11] = torch.linspace(-1, 1, 32) * big
    lg[12, 8:16] = -inf
    lg[13, :24] = nan
    bias = torch.zeros(32)
    bias[[1, 8]] = -inf
    bias[17] = nan
    bias[20] = 1e30
    bias[21] = inf
    for renorm in (True, False):
        _check(lg, 8, renorm, 4, 2, scoring, None, "max")
        _check(lg, 8, renorm, 1, 1, scoring, None)
        _check(lg, 8, renorm, 4, 2, scoring, bias, "top2")
        _check(lg, 8, renorm, 4, 2, scoring, bias, "max")
        _check(lg, 32, renorm, 1, 1, scoring, bias)
        _check(lg.half(), 8, renorm, 4, 2, scoring, bias, "top2")


def test_no_expert_left_drops_the_token(device):
    """Ids of -1 with weight 0, which the expert layer drops: its output row is zero."""
    from exq_amd import synth
    from exq_amd.kernels import fused_experts, grouped_topk, pack_experts_int4
    banner("grouped_topk into fused_experts")
    w13, w2 = synth.expert_weights_gpu(16, 256, 512, 5, device)
    banks = pack_experts_int4(w13) + pack_experts_int4(w2)
    x = torch.randn(5, 512, device=device).bfloat16()
    lg = _logits(5, 16, 3)
    lg[2] = float("-inf")
    nv = torch.tensor([4], dtype=torch.int32, device=device)
    w, ids = grouped_topk(lg.cuda(), 4, True, 4, 2, num_token_non_padded=nv)
    out = fused_experts(x, *banks, w, ids)
    assert ids[2].tolist() == [-1] * 4 and ids[4].tolist() == [-1] * 4
    assert not out[[2, 4]].any() and bool((out[[0, 1, 3]].abs().amax(1) > 0).all())


def test_padding_and_empty_batches(device):
    banner("grouped_topk padding")
    from exq_amd.kernels import grouped_topk
    lg = _logits(37, 64, 8)
    for n in (0, 1, 36, 37, 50):
        _check(lg, 6, True, 8, 3, "sigmoid", torch.zeros(64), n_valid=n)
    w, ids = grouped_topk(torch.zeros(0, 64, device=device), 6, True)
    assert w.shape == (0, 6) and ids.shape == (0, 6)
    # a strided view of wider logits
    wide = _logits(20, 100, 9).cuda()
    a = grouped_topk(wide[:, 10:74], 6, False, 8, 3)
    b = grouped_topk(wide[:, 10:74].contiguous(), 6, False, 8, 3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_large_batch_and_streams(device):
    """20,001 tokens on a stream of their own; two calls at once give the same."""
    banner("grouped_topk large")
    from exq_amd.kernels import grouped_topk
    rng = np.random.default_rng(1)
    lg = _logits(20001, 256, 12)
    bias = torch.from_numpy((0.1 * rng.standard_normal(256)).astype(np.float32))
    ids, w = _check(lg, 8, True, 8, 4, "sigmoid", bias, scale=2.5)
    g, b = lg.cuda(), bias.cuda()
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            outs.append(grouped_topk(g, 8, True, 8, 4, scoring_func="sigmoid", correction_bias=b,
                                     routed_scaling_factor=2.5))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[1], ids) and torch.equal(o[0], w)
