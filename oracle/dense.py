"""Plain 64-bit statements of what stands beside the routed experts: routing with
groups of experts, and dense products with an epilogue.

pinned by: brute force over all choices on tiny inputs (tests/test_oracle_dense.py).
"""
from __future__ import annotations

import numpy as np
from scipy.special import erf

_LARGEST = float(np.finfo(np.float32).max)


def grouped_topk(logits, top_k, renormalize, n_groups=1, topk_group=1, scoring="softmax",
                 bias=None, group_score=None, scale=1.0, n_valid=None):
    """``(ids int64 [T, k], weights float64 [T, k])`` of float logits [T, E], row by row."""
    logits = np.asarray(logits, dtype=np.float64)
    T, E = logits.shape
    gs = E // n_groups
    if group_score is None:
        group_score = "max" if bias is None else "top2"
    ids = np.full((T, top_k), -1, dtype=np.int64)
    wts = np.zeros((T, top_k))
    for t in range(T if n_valid is None else min(T, n_valid)):
        l = logits[t]
        there = l > -np.inf                      # (False for NaN)
        if bias is not None:
            there &= np.asarray(bias, dtype=np.float64) > -np.inf
        experts = np.flatnonzero(there)
        if experts.size == 0:
            continue
        l = np.minimum(l, _LARGEST)
        with np.errstate(over="ignore", under="ignore"):
            if scoring == "softmax":
                log_s = l - l[experts].max()
                log_s = log_s - np.log(np.exp(log_s[experts]).sum())
            else:
                log_s = np.minimum(l, 0.0) - np.log1p(np.exp(-np.abs(l)))
            s = np.exp(log_s)
        rank = l if bias is None else s + np.asarray(bias, dtype=np.float64)
        if topk_group < n_groups:
            value = {}
            for e in experts:
                value.setdefault(int(e) // gs, []).append(
                    rank[e] if bias is not None or group_score == "max" else s[e])
            value = {g: (max(v) if group_score == "max" else sum(sorted(v)[-2:]))
                     for g, v in value.items()}
            kept = sorted(value, key=lambda g: (-value[g], g))[:topk_group]
            experts = [e for e in experts if int(e) // gs in kept]
        chosen = sorted(experts, key=lambda e: (-rank[e], e))[:top_k]
        if renormalize:   # (a softmax's ratios are those of the logits, without its sum)
            u = (l if scoring == "softmax" else log_s)[chosen]
            w = np.exp(u - u.max())
            w = w / w.sum()
        else:
            w = s[chosen]
        ids[t, :len(chosen)] = chosen
        wts[t, :len(chosen)] = w * scale
    return ids, wts


def activation(y, name):
    with np.errstate(over="ignore", invalid="ignore"):
        return {None: lambda: y,
                "relu": lambda: np.maximum(y, 0.0),
                "silu": lambda: y / (1.0 + np.exp(-y)),
                "gelu": lambda: 0.5 * y * (1.0 + erf(y * np.sqrt(0.5))),
                "gelu_tanh": lambda: 0.5 * y * (1.0 + np.tanh(np.sqrt(2.0 / np.pi)
                                                              * (y + 0.044715 * y ** 3))),
                "sigmoid": lambda: 1.0 / (1.0 + np.exp(-y))}[name]()


def linear(x, w, bias=None, act=None, residual=None):
    y = np.asarray(x, dtype=np.float64) @ np.asarray(w, dtype=np.float64).T
    if bias is not None:
        y = y + np.asarray(bias, dtype=np.float64)
    y = activation(y, act)
    return y if residual is None else y + np.asarray(residual, dtype=np.float64)


def gated_linear(x, w, bias=None, act="silu"):
    n = np.asarray(w).shape[0] // 2
    bg, bu = (None, None) if bias is None else (bias[:n], bias[n:])
    return linear(x, w[:n], bg, act) * linear(x, w[n:], bu)
