"""The dense half of a MoE block, as measured calls: routing, and products with an epilogue.

``op`` selects the operator:

* ``route``  ``grouped_topk``: softmax or sigmoid scores of the router's logits, an optional
  balancing bias, expert groups, top-k and renormalised, scaled weights;
* ``linear``  ``fused_linear``: ``act(x @ W.T + bias) + residual`` (router projection, the down
  projection of a shared expert added onto the routed experts' output, a dense layer);
* ``gated``  ``fused_gated_linear``: ``act(x @ Wg.T) * (x @ Wu.T)``, the gate / up projection of a
  shared expert or of a dense layer.

Sizes are those of ``exq_amd.synth.CONFIGS`` where a model of theirs has the product, and generic
ones otherwise.  Where ``own`` is false, ``run`` computes the same in elementary torch operations.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_LARGEST = 3.4028234663852886e38   # largest finite float32


def _route(tokens, experts, top_k, groups, top_groups, scoring, bias, renorm, scale, act) -> dict:
    return dict(op="route", tokens=tokens, experts=experts, top_k=top_k, groups=groups,
                top_groups=top_groups, scoring=scoring, bias=bias, renorm=renorm, scale=scale,
                act=act)


def _linear(tokens, k, n, act, out, bias=False, fn="none", residual="none") -> dict:
    return dict(op="linear", tokens=tokens, k=k, n=n, act=act, out=out, bias=bias, fn=fn,
                residual=residual)


def _gated(tokens, k, inter, act, bias=False, fn="silu") -> dict:
    return dict(op="gated", tokens=tokens, k=k, inter=inter, act=act, bias=bias, fn=fn)


def listed() -> list[dict]:
    return [
        # One user generating: the routing of a single token, bound by latency.
        dict(_route(1, 256, 8, 8, 4, "sigmoid", True, True, 2.5, "f32"), name="route_t1"),
        # A ragged prompt through a softmax router whose groups are ranked by their best expert.
        dict(_route(333, 160, 6, 8, 3, "softmax", False, False, 16.0, "bf16"),
             name="route_softmax_t333"),
        # A long prefill batch, router logits in float32.
        dict(_route(16384, 256, 8, 8, 4, "sigmoid", True, True, 2.5, "f32"), name="route_t16384"),
        # The router projection of one decoded token, logits in float32.
        dict(_linear(1, 2048, 128, "bf16", "f32"), name="router_proj_t1"),
        # The router projection of a prefill batch: a tall product with few columns.
        dict(_linear(4096, 2048, 128, "bf16", "f32"), name="router_proj_t4096"),
        # A decode batch: the shared experts' down projection onto the routed experts' output.
        dict(_linear(16, 2816, 2048, "bf16", "bf16", residual="bf16"), name="shared_down_t16"),
        # A short ragged prompt through a dense layer with bias and activation, odd width, fp16.
        dict(_linear(187, 1000, 2047, "f16", "f16", bias=True, fn="gelu", residual="f16"),
             name="dense_odd_t187"),
        # A long prompt through the down projection of a large dense layer.
        dict(_linear(4096, 14336, 4096, "bf16", "bf16", residual="bf16"), name="dense_down_t4096"),
        # The shared experts' gate / up projection of one token: a stream of weights.
        dict(_gated(1, 2048, 2816, "bf16"), name="shared_gate_up_t1"),
        # The same for a full decode batch, in fp16.
        dict(_gated(64, 2048, 2816, "f16"), name="shared_gate_up_t64"),
        # The same for a prefill chunk with a ragged end.
        dict(_gated(2001, 2048, 2816, "bf16"), name="shared_gate_up_t2001"),
        # The largest: a long prompt through the gate / up projection of a large dense layer.
        dict(_gated(4096, 4096, 14336, "bf16"), name="dense_gate_up_t4096"),
    ]


# ---- drawn cases ------------------------------------------------------------------------------

_MAX_FLOPS = 2.0 * 4096 * 4096 * 2 * 14336


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo: int, hi: int) -> int:
    """A width: a multiple of 128 as models have it, of 8, or an odd one."""
    n = _log_int(rng, lo, hi)
    step = rng.choice([128, 128, 128, 64, 8, 1])
    return max(lo, n // step * step)


def draw(rng) -> dict:
    while True:
        case = _draw(rng)
        if work(case)["flops"] <= 0.8 * _MAX_FLOPS:
            return case


def _draw(rng) -> dict:
    op = rng.choice(["route", "route", "linear", "linear", "linear", "gated", "gated"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        experts = groups * rng.randint(max(2, 8 // groups), 512 // groups)
        top_groups = rng.randint(1, groups)
        room = min(16, experts // groups * top_groups)
        scoring = rng.choice(["softmax", "sigmoid"])
        return _route(_log_int(rng, 1, 16384), experts, rng.randint(1, room), groups, top_groups,
                      scoring, rng.random() < (0.7 if scoring == "sigmoid" else 0.3),
                      rng.random() < 0.7, rng.choice([1.0, 2.5, 16.0]),
                      rng.choice(["f32", "f32", "bf16", "f16"]))
    act = rng.choice(["bf16", "bf16", "f16"])
    tokens = _log_int(rng, 1, 4096)
    k = _size(rng, 256, 14336)
    if op == "gated":
        return _gated(tokens, k, _size(rng, 128, 14336), act, rng.random() < 0.25,
                      rng.choice(["silu", "silu", "silu", "gelu", "gelu_tanh"]))
    if rng.random() < 0.3:   # a router's projection
        return _linear(tokens, k, rng.choice([8, 60, 64, 128, 160, 256]), act, "f32",
                       bias=rng.random() < 0.25)
    return _linear(tokens, k, _size(rng, 128, 14336), act, rng.choice([act, act, act, "f32"]),
                   bias=rng.random() < 0.3,
                   fn=rng.choice(["none", "none", "none", "silu", "gelu", "gelu_tanh", "relu"]),
                   residual=rng.choice(["none", act, act, "f32"]))


# ---- inputs -----------------------------------------------------------------------------------

def _generator(seed: int, part: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(1000003 * (seed % (1 << 40)) + part)


def _randn(shape, seed: int, part: int, dtype: torch.dtype, scale: float = 1.0) -> torch.Tensor:
    t = torch.randn(*shape, generator=_generator(seed, part), device="cuda", dtype=torch.float32)
    return t.mul_(scale).to(dtype)


def prepare(case: dict, seed: int) -> dict:
    state = {"case": case}
    act = DTYPES[case["act"]]
    t = case["tokens"]
    if case["op"] == "route":
        n = case["experts"]
        # expert popularity as a trained router's: a Zipf law over a seeded order of the experts
        rank = torch.randperm(n, generator=_generator(seed, 1), device="cuda")
        popular = -0.6 * torch.log(rank.float() + 1.0)
        popular -= popular.mean()
        state["logits"] = (_randn((t, n), seed, 2, torch.float32) + popular).to(act)
        state["bias"] = None
        if case["bias"]:   # the bias that balances them counters the popularity in part
            scale = 0.05 if case["scoring"] == "sigmoid" else 0.1 / n
            state["bias"] = (scale * (torch.randn(n, generator=_generator(seed, 3), device="cuda")
                                      - popular)).contiguous()
        return state
    k = case["k"]
    rows = case["n"] if case["op"] == "linear" else 2 * case["inter"]
    state["x"] = _randn((t, k), seed, 1, act)
    state["w"] = _randn((rows, k), seed, 2, act, 0.02)
    state["bias"] = _randn((rows,), seed, 3, act, 0.1) if case["bias"] else None
    state["residual"] = None
    if case.get("residual", "none") != "none":
        state["residual"] = _randn((t, rows), seed, 4, DTYPES[case["residual"]])
    return state


# ---- one pass ---------------------------------------------------------------------------------

def _own_pass(state: dict):
    from exq_amd.kernels import fused_gated_linear, fused_linear, grouped_topk

    case = state["case"]
    if case["op"] == "route":
        return grouped_topk(state["logits"], case["top_k"], case["renorm"], case["groups"],
                            case["top_groups"], scoring_func=case["scoring"],
                            correction_bias=state["bias"], routed_scaling_factor=case["scale"])
    if case["op"] == "gated":
        return fused_gated_linear(state["x"], state["w"], state["bias"], activation=case["fn"])
    return fused_linear(state["x"], state["w"], state["bias"],
                        activation=None if case["fn"] == "none" else case["fn"],
                        residual=state["residual"], out_dtype=DTYPES[case["out"]])


def _activation(y: torch.Tensor, fn: str) -> torch.Tensor:
    if fn == "silu":
        return y / (1.0 + torch.exp(-y))
    if fn == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if fn == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if fn == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    return y


def _plain_route(state: dict):
    """Ranks in 64 bits: an expert next to the border is decided by its score, not by a rounding."""
    case, bias = state["case"], state["bias"]
    t, n, g = case["tokens"], case["experts"], case["groups"]
    low = float("-inf")
    l = state["logits"].double()
    there = l > low
    if bias is not None:
        there = there & (bias.double() > low)
    l = torch.where(there, l.clamp(max=_LARGEST), low)
    if case["scoring"] == "softmax":
        e = torch.exp(l - l.amax(-1, keepdim=True).clamp(min=-_LARGEST))
        s = e / e.sum(-1, keepdim=True).clamp(min=1.0)
        a = l
    else:
        s = 1.0 / (1.0 + torch.exp(-l))
        a = l.clamp(max=0.0) - torch.log1p(torch.exp(-l.abs()))   # log of the sigmoid
    rank = l if bias is None else torch.where(there, s + bias.double(), low)
    if case["top_groups"] < g:
        inside = rank.view(t, g, n // g)
        if bias is None:
            best = inside.amax(-1)
        else:
            two = torch.sort(inside, dim=-1, descending=True).values[..., :2]
            best = torch.where(two > low, two, torch.zeros_like(two)).sum(-1)
            best = torch.where(two[..., 0] > low, best, low)
        order = torch.sort(best, dim=-1, descending=True, stable=True).indices
        keep = torch.zeros(t, g, dtype=torch.bool, device=l.device)
        keep.scatter_(1, order[:, :case["top_groups"]], True)
        rank = torch.where(keep.unsqueeze(-1), inside, low).view(t, n)
    top = torch.sort(rank, dim=-1, descending=True, stable=True)
    ids = top.indices[:, :case["top_k"]]
    found = top.values[:, :case["top_k"]] > low
    if case["renorm"]:
        a = torch.where(found, torch.gather(a, 1, ids), low)
        w = torch.exp(a - a.amax(-1, keepdim=True).clamp(min=-_LARGEST))
        w = w / w.sum(-1, keepdim=True).clamp(min=1.0)
    else:
        w = torch.where(found, torch.gather(s, 1, ids), torch.zeros((), dtype=s.dtype,
                                                                    device=s.device))
    return ((w * case["scale"]).float(),
            torch.where(found, ids, torch.full_like(ids, -1)).to(torch.int32))


def run(state: dict):
    if own:
        return _own_pass(state)
    case = state["case"]
    if case["op"] == "route":
        return _plain_route(state)
    y = torch.mm(state["x"].float(), state["w"].float().t())
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if case["op"] == "gated":
        i = case["inter"]
        return (_activation(y[:, :i], case["fn"]) * y[:, i:]).to(DTYPES[case["act"]])
    y = _activation(y, case["fn"])
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(DTYPES[case["out"]])


# ---- bounds -----------------------------------------------------------------------------------

def work(case: dict) -> dict:
    """Each input read once, each output written once; 2 flops per multiply-add of a product, and
    one operation per score of a router."""
    t = case["tokens"]
    size = DTYPES[case["act"]].itemsize
    if case["op"] == "route":
        n = case["experts"]
        return {"bytes": float(t * n * size + (4 * n if case["bias"] else 0)
                               + 8 * t * case["top_k"]),
                "flops": float(t * n)}
    rows = case["n"] if case["op"] == "linear" else 2 * case["inter"]
    moved = size * (t + rows) * case["k"] + (size * rows if case["bias"] else 0)
    if case["op"] == "gated":
        moved += size * t * case["inter"]
    else:
        moved += DTYPES[case["out"]].itemsize * t * rows
        if case["residual"] != "none":
            moved += DTYPES[case["residual"]].itemsize * t * rows
    return {"bytes": float(moved), "flops": 2.0 * t * rows * case["k"]}


# ---- 64-bit references ------------------------------------------------------------------------

def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "route":
        # rank by rank: the best group, then the best expert, that is not taken yet
        l = state["logits"].double()
        t, n = l.shape
        g = case["groups"]
        rows = torch.arange(t, device=l.device)
        if case["scoring"] == "softmax":
            score, log_score = torch.softmax(l, -1), torch.log_softmax(l, -1)
        else:
            score, log_score = torch.sigmoid(l), torch.nn.functional.logsigmoid(l)
        rank = l.clone() if state["bias"] is None else score + state["bias"].double()
        per = rank.view(t, g, n // g)
        if state["bias"] is None:
            value = per.max(-1).values
        else:
            value = per.topk(min(2, n // g), -1).values.sum(-1)
        kept = torch.zeros(t, g, dtype=torch.bool, device=l.device)
        for _ in range(case["top_groups"]):
            kept[rows, value.masked_fill(kept, float("-inf")).argmax(-1)] = True
        rank = per.masked_fill(~kept.unsqueeze(-1), float("-inf")).reshape(t, n)
        chosen = []
        for _ in range(case["top_k"]):
            chosen.append(rank.argmax(-1))
            rank[rows, chosen[-1]] = float("-inf")
        ids = torch.stack(chosen, 1)
        if case["renorm"]:
            w = torch.softmax(log_score.gather(1, ids), -1)
        else:
            w = score.gather(1, ids)
        return w * case["scale"], None
    functions = {"none": lambda y: y, "silu": torch.nn.functional.silu,
                 "gelu": torch.nn.functional.gelu, "relu": torch.relu,
                 "gelu_tanh": lambda y: torch.nn.functional.gelu(y, approximate="tanh")}
    fn = functions[case["fn"]]
    x, w = state["x"].double(), state["w"].double()
    b = 0.0 if state["bias"] is None else state["bias"].double()
    y = torch.mm(x, w.t().contiguous()) + b
    if case["op"] == "gated":
        gate, up = y.split(case["inter"], 1)
        return fn(gate) * up
    y = fn(y)
    return y if state["residual"] is None else y + state["residual"].double()
