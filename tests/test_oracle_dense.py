"""The 64-bit statements of grouped routing and of dense products against brute force
over all choices and against torch, and the refusals of the operators (no GPU)."""
import itertools

import numpy as np
import pytest
import torch

from exq_amd import _lib
from exq_amd.kernels import fused_gated_linear, fused_linear, grouped_topk
from oracle import dense


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("use_bias", [False, True])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_grouped_topk_is_the_best_choice(scoring, use_bias, group_score):
    """Among all sets of groups and all k-subsets of their experts."""
    rng = np.random.default_rng(5)
    T, E, G, keep, k = 6, 8, 4, 2, 3
    logits = rng.standard_normal((T, E))
    bias = 0.5 * rng.standard_normal(E) if use_bias else None
    ids, w = dense.grouped_topk(logits, k, True, G, keep, scoring, bias, group_score, 2.0)
    t = torch.from_numpy(logits)
    s = (torch.softmax(t, -1) if scoring == "softmax" else torch.sigmoid(t)).numpy()
    r = s if bias is None else s + bias
    for i in range(T):
        value = [r[i, 2 * g:2 * g + 2].max() if group_score == "max" else r[i, 2 * g:2 * g + 2].sum()
                 for g in range(G)]
        groups = max(itertools.combinations(range(G), keep), key=lambda c: sum(value[g] for g in c))
        room = [e for e in range(E) if e // 2 in groups]
        best = max(itertools.combinations(room, k), key=lambda c: sum(r[i, e] for e in c))
        assert sorted(ids[i]) == sorted(best)
        assert list(ids[i]) == sorted(best, key=lambda e: -r[i, e])
        np.testing.assert_allclose(w[i], 2.0 * s[i, ids[i]] / s[i, ids[i]].sum(), rtol=1e-12)


def test_grouped_topk_masks_and_ties():
    inf, nan = np.inf, np.nan
    ids, w = dense.grouped_topk([[-inf, 1.0, nan, 1.0], [-inf, -inf, nan, -inf],
                                 [0.0, inf, 0.0, inf], [-900.0, -901.0, -inf, -inf]], 3, True,
                                scoring="sigmoid")
    assert ids.tolist() == [[1, 3, -1], [-1, -1, -1], [1, 3, 0], [0, 1, -1]]
    e = np.exp(-1.0)
    np.testing.assert_allclose(w, [[.5, .5, 0], [0, 0, 0], [.4, .4, .2],
                                   [1 / (1 + e), e / (1 + e), 0]], rtol=1e-12)
    ids, _ = dense.grouped_topk([[5.0, 5.0, 5.0, 5.0]], 2, False, 2, 1)
    assert ids.tolist() == [[0, 1]]
    ids, w = dense.grouped_topk([[1.0, 2.0]] * 3, 1, False, n_valid=1)
    assert ids.tolist() == [[1], [-1], [-1]] and w[1, 0] == 0


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh", "sigmoid"])
def test_linear_against_torch(act):
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((5, 7)), rng.standard_normal((6, 7))
    b, r = rng.standard_normal(6), rng.standard_normal((5, 6))
    f = torch.nn.functional
    fn = {None: lambda y: y, "relu": torch.relu, "silu": f.silu, "gelu": f.gelu,
          "gelu_tanh": lambda y: f.gelu(y, approximate="tanh"), "sigmoid": torch.sigmoid}[act]
    tx, tw, tb, tr = map(torch.from_numpy, (x, w, b, r))
    want = fn(f.linear(tx, tw, tb)) + tr
    np.testing.assert_allclose(dense.linear(x, w, b, act, r), want.numpy(), rtol=1e-12, atol=1e-14)
    if act is not None:
        y = f.linear(tx, tw, tb)
        np.testing.assert_allclose(dense.gated_linear(x, w, b, act),
                                   (fn(y[:, :3]) * y[:, 3:]).numpy(), rtol=1e-12, atol=1e-14)


# ---- refusals ---------------------------------------------------------------------------------

def test_grouped_topk_refusals():
    l = torch.zeros(4, 16)
    for args, kw in [((torch.zeros(16), 2, True), {}),
                     ((l.double(), 2, True), {}),
                     ((l, 0, True), {}),
                     ((l, 17, True), {}),
                     ((l, 2, True, 3, 1), {}),
                     ((l, 2, True, 4, 5), {}),
                     ((l, 2, True, 4, 0), {}),
                     ((l, 5, True, 4, 1), {}),
                     ((l, 2, True), dict(scoring_func="tanh")),
                     ((l, 2, True), dict(group_score="mean")),
                     ((l, 2, True), dict(correction_bias=torch.zeros(15))),
                     ((l, 2, True), dict(correction_bias=torch.zeros(16, dtype=torch.float64))),
                     ((l, 2, True), dict(ids_dtype=torch.int16)),
                     ((l, 2, True), dict(num_token_non_padded=torch.zeros(1))),
                     ((l, 2, True), dict(num_token_non_padded=torch.zeros(2, dtype=torch.int32))),
                     ((torch.zeros(2, 1025), 2, True), {}),
                     ((l.clone().requires_grad_(), 2, True), {})]:
        with pytest.raises(ValueError):
            grouped_topk(*args, **kw)
    with pytest.raises(_lib.ExqError, match="HIP device"):
        grouped_topk(l, 2, True)


def test_linear_refusals():
    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    w = torch.zeros(8, 16, dtype=torch.bfloat16)
    for args, kw in [((x[0], w), {}),
                     ((x, w[:, :8]), {}),
                     ((x, w.half()), {}),
                     ((x.float(), w.float()), {}),
                     ((x[:, :0], w[:, :0]), {}),
                     ((x, w[:0]), {}),
                     ((x.t().contiguous().t(), w), {}),
                     ((x, w, torch.zeros(7)), {}),
                     ((x, w, torch.zeros(16)[::2]), {}),
                     ((x, w), dict(activation="tanh")),
                     ((x, w), dict(residual=torch.zeros(4, 7))),
                     ((x, w), dict(residual=torch.zeros(4, 8, dtype=torch.float64))),
                     ((x, w), dict(out=torch.zeros(4, 8, dtype=torch.bfloat16).requires_grad_())),
                     ((x, w.clone().requires_grad_()), {})]:
        with pytest.raises(ValueError):
            fused_linear(*args, **kw)
    for args, kw in [((x, w[:7]), {}), ((x, w[:0]), {}), ((x, w), dict(activation=None)),
                     ((x, w, torch.zeros(4)), {}),
                     ((x.clone().requires_grad_(), w), {})]:
        with pytest.raises(ValueError):
            fused_gated_linear(*args, **kw)
    with pytest.raises(_lib.ExqError, match="HIP device"):
        fused_linear(x, w)
    with torch.no_grad(), pytest.raises(_lib.ExqError, match="HIP device"):
        fused_gated_linear(x, w.clone().requires_grad_())


def test_overlap_rule():
    from exq_amd.kernels.linear import _overlap
    buf = torch.zeros(6, 12)
    a, b = buf[:, :5], buf[:, 5:]
    assert not _overlap(a, 12, b, 12) and not _overlap(b, 12, a, 12)
    assert _overlap(a, 12, buf[:, 4:], 12) and _overlap(buf[:, 4:], 12, a, 12)
    assert not _overlap(buf[:3], 12, buf[3:], 12)
    assert _overlap(buf[:4], 12, buf[3:], 12)
    assert _overlap(b, 12, buf[1:, :5].new_tensor([]).set_(buf.untyped_storage(), 12, (2, 12)), 12)


def test_c_entries_check_arguments():
    L = _lib.lib()

    def route(**kw):
        v = dict(n_tokens=4, n_experts=16, top_k=2, n_groups=4, topk_group=2, logits_dtype=_lib.F32,
                 bias_dtype=_lib.F32, ids_dtype=_lib.I32, weights_dtype=_lib.F32, scoring=0,
                 group_score=0, renormalize=1, scale=1.0)
        v.update(kw)
        st = L.exq_grouped_topk(_lib.RouteProblem(**v), None, None, None, None, None, None)
        return st, L.exq_last_error()

    assert route(n_tokens=0)[0] == 0
    for kw, text in [(dict(logits_dtype=_lib.I32), b"logits dtype"),
                     (dict(ids_dtype=_lib.F32), b"ids dtype"),
                     (dict(weights_dtype=_lib.I8), b"weights dtype"),
                     (dict(scoring=2), b"scoring"), (dict(group_score=-1), b"group_score"),
                     (dict(n_experts=1025), b"n_experts"), (dict(n_groups=3), b"n_groups"),
                     (dict(topk_group=5), b"topk_group"), (dict(top_k=9), b"top_k"),
                     (dict(n_tokens=-1), b"n_tokens"), (dict(n_tokens=1 << 26), b"n_tokens"),
                     ({}, b"null pointer")]:
        st, msg = route(**kw)
        assert st == 1 and text in msg, (kw, msg)

    def lin(residual=None, **kw):
        v = dict(n_tokens=4, in_features=16, out_features=8, x_stride=16, weight_stride=16,
                 residual_stride=8, out_stride=8, act_dtype=_lib.BF16, bias_dtype=_lib.F32,
                 residual_dtype=_lib.F32, out_dtype=_lib.BF16, activation=0, gated=0)
        v.update(kw)
        st = L.exq_linear(_lib.LinearProblem(**v), None, None, None, residual, None, None)
        return st, L.exq_last_error()

    assert lin(n_tokens=0)[0] == 0
    for kw, text in [(dict(act_dtype=_lib.F32), b"x and W"), (dict(out_dtype=_lib.I8), b"out dtype"),
                     (dict(activation=6), b"activation"), (dict(gated=1, residual=1), b"residual"),
                     (dict(in_features=0), b"sizes"), (dict(out_features=0), b"sizes"),
                     (dict(out_features=(1 << 20) + 1), b"sizes"), (dict(n_tokens=-1), b"sizes"),
                     (dict(x_stride=-1), b"strides"), (dict(out_stride=7), b"strides"),
                     ({}, b"null pointer")]:
        st, msg = lin(**kw)
        assert st == 1 and text in msg, (kw, msg)
