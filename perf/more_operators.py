"""MXFP4 (microscaled 4-bit floating point) as measured calls.

Blocks of 32 values along a row share a scale ``2**(s - 127)`` (one byte, 255 is NaN); a value is
a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  ``op`` selects the operator:

* ``quant``  ``quantize_mxfp4`` and ``dequantize_mxfp4``: rows to 4 bits and back;
* ``linear``  ``fused_linear_mxfp4``: ``act(x @ W.T + bias) + residual`` with W in MXFP4, x in 16
  bits or (``x4``) quantised to MXFP4 by the caller's own call before the product;
* ``gated``  ``fused_gated_linear_mxfp4``: ``act(x @ Wg.T) * (x @ Wu.T)``, types as for ``linear``;
* ``moe``  ``fused_experts_mxfp4``: a whole MoE layer, ``out[t] = sum_j w[t, j] * down_e(silu(gate_e
  x) * up_e x)``, its experts in MXFP4.

Sizes are those of ``exq_amd.synth.CONFIGS`` where a model of theirs has the layer, and generic
ones otherwise.  Where ``own`` is false, ``run`` computes the same in elementary torch operations.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 32
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quant(rows, k, act) -> dict:
    return dict(op="quant", rows=rows, k=k, act=act)


def _linear(tokens, k, n, act, x4=False, bias=False, fn="none", residual="none", out=None) -> dict:
    return dict(op="linear", tokens=tokens, k=k, n=n, act=act, x4=x4, bias=bias, fn=fn,
                residual=residual, out=out or act)


def _gated(tokens, k, inter, act, x4=False, bias=False, fn="silu") -> dict:
    return dict(op="gated", tokens=tokens, k=k, inter=inter, act=act, x4=x4, bias=bias, fn=fn)


def _moe(tokens, hidden, inter, experts, top_k, act, renorm=True, skew=1.1, padded=0) -> dict:
    return dict(op="moe", tokens=tokens, hidden=hidden, inter=inter, experts=experts, top_k=top_k,
                act=act, renorm=renorm, skew=skew, padded=padded)


def listed() -> list[dict]:
    return [
        # The activations of one decoded token before a product of two MXFP4 operands.
        dict(_quant(1, 2048, "bf16"), name="quant_t1"),
        # Those of a ragged prompt, an odd number of blocks a row, fp16.
        dict(_quant(187, 1440, "f16"), name="quant_odd_t187"),
        # A large weight matrix, quantised once when a model is loaded.
        dict(_quant(28672, 4096, "bf16"), name="quant_weights"),
        # The shared experts' gate / up projection of one token: a stream of weights.
        dict(_gated(1, 2048, 2816, "bf16"), name="shared_gate_up_t1"),
        # A decode batch: their down projection onto the routed experts' output.
        dict(_linear(16, 2816, 2048, "bf16", residual="bf16"), name="shared_down_t16"),
        # A short ragged prompt through a dense layer with bias and activation, odd width, fp16.
        dict(_linear(187, 1440, 2047, "f16", bias=True, fn="gelu", residual="f16"),
             name="dense_odd_t187"),
        # The largest product: a long prompt through the gate / up projection of a dense layer.
        dict(_gated(4096, 4096, 14336, "bf16"), name="dense_gate_up_t4096"),
        # The down projection of that layer with activations in MXFP4 too.
        dict(_linear(4096, 14336, 4096, "bf16", x4=True, residual="bf16"),
             name="dense_down_x4_t4096"),
        # One user generating: a layer of 128 small experts.
        dict(_moe(1, 2048, 768, 128, 8, "bf16"), name="moe_t1"),
        # A decode batch in fp16, router weights not renormalised.
        dict(_moe(16, 2048, 1024, 64, 8, "f16", renorm=False), name="moe_t16"),
        # A full decode batch whose last rows are the padding of a captured size.
        dict(_moe(64, 2048, 768, 128, 8, "bf16", padded=5), name="moe_t64"),
        # A ragged prefill chunk through experts of an odd number of 128-wide tiles.
        dict(_moe(2001, 2048, 1408, 64, 6, "bf16", renorm=False), name="moe_t2001"),
    ]


# ---- drawn cases ------------------------------------------------------------------------------

_MAX_FLOPS = 2.0 * 4096 * 4096 * 2 * 14336


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo: int, hi: int, steps) -> int:
    n, step = _log_int(rng, lo, hi), rng.choice(steps)
    return max(lo, n // step * step)


def draw(rng) -> dict:
    while True:
        case = _draw(rng)
        if work(case)["flops"] <= 0.8 * _MAX_FLOPS:
            return case


def _draw(rng) -> dict:
    op = rng.choice(["quant", "quant", "linear", "linear", "gated", "moe", "moe", "moe"])
    act = rng.choice(["bf16", "bf16", "f16"])
    if op == "quant":
        rows, k = _log_int(rng, 1, 28672), _size(rng, 256, 14336, [512, 128, 32])
        return _quant(max(1, min(rows, (1 << 27) // k)), k, rng.choice(["bf16", "f16", "f32"]))
    if op == "moe":
        experts = rng.choice([8, 16, 60, 64, 128, 160])
        hidden = _size(rng, 512, 4096, [512, 256, 128, 32])
        inter = _size(rng, 256, 4096, [256, 128, 128, 32])
        experts = min(experts, max(8, (1 << 30) // (3 * hidden * inter)))
        tokens = _log_int(rng, 1, 4096)
        top_k = rng.randint(1, min(8, experts))
        return _moe(tokens, hidden, inter, experts, top_k, act, rng.random() < 0.6,
                    rng.choice([0.0, 0.6, 1.1]),
                    rng.randint(1, tokens) // 4 if rng.random() < 0.3 else 0)
    tokens = _log_int(rng, 1, 4096)
    k = _size(rng, 256, 14336, [512, 128, 128, 32])
    width = [128, 128, 128, 64, 8, 1]
    x4 = rng.random() < 0.4
    if op == "gated":
        return _gated(tokens, k, _size(rng, 128, 14336, width), act, x4, rng.random() < 0.25,
                      rng.choice(["silu", "silu", "silu", "gelu", "gelu_tanh"]))
    return _linear(tokens, k, _size(rng, 128, 14336, width), act, x4, rng.random() < 0.3,
                   rng.choice(["none", "none", "none", "silu", "gelu", "gelu_tanh", "relu"]),
                   rng.choice(["none", act, act, "f32"]), rng.choice([act, act, act, "f32"]))


# ---- MXFP4 in elementary operations -----------------------------------------------------------

def _to_mxfp4(x: torch.Tensor):
    """(codes [.., K], scale bytes [.., K / 32]) of finite x [.., K]: the scale is the power of two
    that brings the block's largest magnitude into [4, 8), values go to the nearest code, halfway
    to the even one, and past 6 to 6."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1)
    e = torch.frexp(top).exponent - 1
    s = torch.where(top > 0, (e - 2 + 127).clamp(min=0), torch.zeros_like(e))
    # (2^(127 - s) in two factors, each a normal number)
    half = (127 - s).div(2, rounding_mode="floor")
    v = b.abs() * _power(half).unsqueeze(-1) * _power(127 - s - half).unsqueeze(-1)
    code = ((v > 0.25).to(torch.uint8) + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5)
            + (v >= 3.5) + (v > 5.0))
    code = code + 8 * torch.signbit(b).to(torch.uint8)
    return code.flatten(-2), s.to(torch.uint8)


def _power(e: torch.Tensor) -> torch.Tensor:
    """2^e for whole e in [-126, 127]."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _from_mxfp4(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float32 values of codes [.., K]."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=codes.device)
    s = scales.int()
    half = s >> 1
    v = table[codes.int()].unflatten(-1, (-1, BLOCK))
    v = v * _power(half - 63).unsqueeze(-1) * _power(s - half - 64).unsqueeze(-1)
    return v.flatten(-2)


def _codes(packed: torch.Tensor) -> torch.Tensor:
    """Two codes a byte, the even column in the low four bits."""
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def _packed(codes: torch.Tensor) -> torch.Tensor:
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _tiles(packed: torch.Tensor, scales: torch.Tensor, gated: bool):
    """The order in which the products read a weight [.., N, K]: tiles of 16 rows x 128 columns
    (gate and up tiles in turn), 16 bytes per (block of 32 columns, row); and the scales of four
    tiles along a row together.  Rows are padded to 16, columns to 128 (scales to 512)."""
    pad = torch.nn.functional.pad
    if gated:
        n = packed.shape[-2] // 2
        more = -n % 16
        packed = pad(packed.unflatten(-2, (2, n)), (0, 0, 0, more)).unflatten(-2, (-1, 16))
        scales = pad(scales.unflatten(-2, (2, n)), (0, 0, 0, more)).unflatten(-2, (-1, 16))
        packed = packed.transpose(-4, -3).flatten(-4, -2)
        scales = scales.transpose(-4, -3).flatten(-4, -2)
    more = -packed.shape[-2] % 16
    packed = pad(packed, (0, -packed.shape[-1] % 64, 0, more))
    scales = pad(scales, (0, -scales.shape[-1] % 16, 0, more))
    p = packed.unflatten(-2, (-1, 16)).unflatten(-1, (-1, 4, 16))        # rt, r, kb, q, 16
    s = scales.unflatten(-2, (-1, 16)).unflatten(-1, (-1, 4, 4))         # rt, r, g, i, q
    p = p.movedim(-4, -2).flatten(-3, -2).contiguous()                   # rt, kb, (q, r), 16
    s = s.movedim(-4, -1).movedim(-3, -1).flatten(-3, -2).contiguous()   # rt, g, (q, r), i
    return p, s


# ---- inputs -----------------------------------------------------------------------------------

def _generator(seed: int, part: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(1000003 * (seed % (1 << 40)) + part)


def _randn(shape, seed: int, part: int, dtype: torch.dtype, scale: float = 1.0) -> torch.Tensor:
    t = torch.randn(*shape, generator=_generator(seed, part), device="cuda", dtype=torch.float32)
    return t.mul_(scale).to(dtype)


def _weight(shape, seed: int, part: int, gated: bool) -> dict:
    """A quantised weight [.., N, K] as it is stored (packed, scales) and in the order of tiles."""
    lead = shape[0] if len(shape) == 3 else 1
    some = max(1, (1 << 28) // (shape[-1] * shape[-2]))
    gen, parts = _generator(seed, part), []
    for first in range(0, lead, some):
        w = torch.randn(min(some, lead - first), *shape[-2:], generator=gen, device="cuda")
        codes, s = _to_mxfp4(w.mul_(0.02))
        parts.append((_packed(codes), s))
    packed = torch.cat([p for p, _ in parts]).view(*shape[:-1], shape[-1] // 2)
    scales = torch.cat([s for _, s in parts]).view(*shape[:-1], shape[-1] // BLOCK)
    tiles, tile_scales = _tiles(packed, scales, gated)
    return dict(packed=packed, scales=scales, tiles=tiles, tile_scales=tile_scales,
                rows=shape[-2], cols=shape[-1], gated=gated)


def _logits(case: dict, gen: torch.Generator, device: str) -> torch.Tensor:
    t, n = case["tokens"], case["experts"]
    rank = torch.randperm(n, generator=gen, device=device)
    return (torch.randn(t, n, generator=gen, device=device)
            - case["skew"] * torch.log(rank.float() + 1.0))


def prepare(case: dict, seed: int) -> dict:
    state = {"case": case}
    act = DTYPES[case["act"]]
    if case["op"] == "quant":
        # activations and weights have outliers: a heavy-tailed factor per column
        tail = torch.exp(0.8 * _randn((case["k"],), seed, 2, torch.float32))
        state["x"] = (_randn((case["rows"], case["k"]), seed, 1, torch.float32) * tail).to(act)
        return state
    t = case["tokens"]
    if case["op"] == "moe":
        h, i, n = case["hidden"], case["inter"], case["experts"]
        state["x"] = _randn((t, h), seed, 1, act)
        state["w13"] = _weight((n, 2 * i, h), seed, 2, True)
        state["w2"] = _weight((n, h, i), seed, 3, False)
        p = torch.softmax(_logits(case, _generator(seed, 4), "cuda"), -1)
        w, ids = p.topk(case["top_k"], -1)
        if case["renorm"]:
            w = w / w.sum(-1, keepdim=True)
        ids[t - case["padded"]:] = -1
        state["weights"], state["ids"] = w.contiguous(), ids.to(torch.int32)
        counts = torch.bincount(state["ids"].long().flatten() + 1, minlength=n + 1)[1:]
        state["most"] = int(counts.max())   # rows of the busiest expert
        return state
    k = case["k"]
    gated = case["op"] == "gated"
    rows = 2 * case["inter"] if gated else case["n"]
    state["x"] = _randn((t, k), seed, 1, act)
    state["w"] = _weight((rows, k), seed, 2, gated)
    state["bias"] = _randn((rows,), seed, 3, act, 0.1) if case["bias"] else None
    state["residual"] = None
    if case.get("residual", "none") != "none":
        state["residual"] = _randn((t, rows), seed, 4, DTYPES[case["residual"]])
    return state


# ---- one pass ---------------------------------------------------------------------------------

def _own_pass(state: dict):
    from exq_amd.kernels import (Mxfp4Weight, dequantize_mxfp4, fused_experts_mxfp4,
                                 fused_gated_linear_mxfp4, fused_linear_mxfp4, quantize_mxfp4)

    def handle(w):
        return Mxfp4Weight(w["tiles"], w["tile_scales"], w["rows"], w["cols"], w["gated"])

    case, x = state["case"], state["x"]
    if case["op"] == "quant":
        return dequantize_mxfp4(*quantize_mxfp4(x), dtype=x.dtype)
    if case["op"] == "moe":
        return fused_experts_mxfp4(x, handle(state["w13"]), handle(state["w2"]), state["weights"],
                                   state["ids"])
    x_scales = None
    if case["x4"]:
        x, x_scales = quantize_mxfp4(x)
    if case["op"] == "gated":
        return fused_gated_linear_mxfp4(x, handle(state["w"]), state["bias"], x_scales=x_scales,
                                        activation=case["fn"], out_dtype=DTYPES[case["act"]])
    return fused_linear_mxfp4(x, handle(state["w"]), state["bias"], x_scales=x_scales,
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


def _plain_weight(w: dict) -> torch.Tensor:
    return _from_mxfp4(_codes(w["packed"]), w["scales"])


def _plain_moe(state: dict) -> torch.Tensor:
    case, x, ids, weights = state["case"], state["x"].float(), state["ids"], state["weights"]
    t, k = ids.shape
    i, n, h = case["inter"], case["experts"], case["hidden"]
    flat = ids.flatten().long()
    routed = flat >= 0
    if t * k <= n:   # few slots: the experts of every slot, one by one
        at = flat.clamp(min=0)
        w13 = _from_mxfp4(_codes(state["w13"]["packed"][at]), state["w13"]["scales"][at])
        y = torch.bmm(w13, x.repeat_interleave(k, 0).unsqueeze(-1)).squeeze(-1)
        y = _activation(y[:, :i], "silu") * y[:, i:]
        w2 = _from_mxfp4(_codes(state["w2"]["packed"][at]), state["w2"]["scales"][at])
        y = torch.bmm(w2, y.unsqueeze(-1)).squeeze(-1)
    else:            # rows by expert, as many for each as the busiest has
        most = max(1, state["most"])
        order = torch.argsort(flat, stable=True)
        e = flat[order]
        first = torch.searchsorted(e, torch.arange(n, device=e.device))
        place = e * most + torch.arange(t * k, device=e.device) - first[e.clamp(min=0)]
        place = torch.where(e >= 0, place, n * most)     # (dropped slots: a row of their own)
        rows = torch.zeros(n * most + 1, h, device=x.device).index_copy_(0, place, x[order // k])
        w13 = _plain_weight(state["w13"])
        y = torch.bmm(rows[:-1].view(n, most, h), w13.transpose(1, 2).contiguous())
        y = _activation(y[..., :i], "silu") * y[..., i:]
        del w13
        y = torch.bmm(y, _plain_weight(state["w2"]).transpose(1, 2).contiguous())
        y = torch.cat((y.view(n * most, h), y.new_zeros(1, h)))[place]
        y = torch.empty_like(y).index_copy_(0, order, y)
    y = torch.where(routed.unsqueeze(-1), y * weights.flatten().unsqueeze(-1), torch.zeros_like(y))
    return y.view(t, k, h).sum(1).to(state["x"].dtype)


def run(state: dict):
    if own:
        return _own_pass(state)
    case = state["case"]
    if case["op"] == "quant":
        return _from_mxfp4(*_to_mxfp4(state["x"])).to(state["x"].dtype)
    if case["op"] == "moe":
        return _plain_moe(state)
    x = state["x"].float()
    if case["x4"]:
        x = _from_mxfp4(*_to_mxfp4(x))
    y = torch.mm(x, _plain_weight(state["w"]).t())
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

def _mxfp4_bytes(values: float) -> float:
    return values / 2 + values / BLOCK


def _active_experts(case: dict) -> int:
    """Experts with a token in a batch of this case's routing (one seeded batch)."""
    logits = _logits(case, torch.Generator().manual_seed(1), "cpu")
    ids = logits[: case["tokens"] - case["padded"]].topk(case["top_k"], -1).indices
    return int(ids.unique().numel())


def work(case: dict) -> dict:
    """Each input read once, each output written once (4-bit rows between two calls: written and
    read); 2 flops per multiply-add of a product, and one operation per value quantised."""
    size = DTYPES[case["act"]].itemsize
    if case["op"] == "quant":
        n = case["rows"] * case["k"]
        return {"bytes": float(2 * n * size) + 2 * _mxfp4_bytes(n), "flops": float(2 * n)}
    t = case["tokens"]
    if case["op"] == "moe":
        h, i, k = case["hidden"], case["inter"], case["top_k"]
        moved = (_mxfp4_bytes(_active_experts(case) * 3 * h * i) + 2 * t * h * size + 8 * t * k)
        return {"bytes": float(moved), "flops": 6.0 * (t - case["padded"]) * k * h * i}
    rows = case["n"] if case["op"] == "linear" else 2 * case["inter"]
    n = t * case["k"]
    moved = _mxfp4_bytes(rows * case["k"]) + n * size + (size * rows if case["bias"] else 0)
    if case["x4"]:
        moved += 2 * _mxfp4_bytes(n)
    if case["op"] == "gated":
        moved += size * t * case["inter"]
    else:
        moved += DTYPES[case["out"]].itemsize * t * rows
        if case["residual"] != "none":
            moved += DTYPES[case["residual"]].itemsize * t * rows
    return {"bytes": float(moved), "flops": 2.0 * n * rows}


# ---- 64-bit references ------------------------------------------------------------------------

def _exact_round(x: torch.Tensor) -> torch.Tensor:
    """x [.., K] rounded to MXFP4, by the spacing of the values at each magnitude."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    # (log2 in 64 bits is exact enough to floor: the inputs have 24 bits at most)
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2
    scale = torch.exp2(e.clamp(min=-127))
    v = (b / scale).abs().clamp(max=6.0)
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    v = torch.round(v / step) * step
    return (torch.sign(b) * v.clamp(max=6.0) * scale).flatten(-2)


def _exact_weight(w: dict, e: int | None = None) -> torch.Tensor:
    p, s = (w["packed"], w["scales"]) if e is None else (w["packed"][e], w["scales"][e])
    out = torch.empty(*p.shape[:-1], 2 * p.shape[-1], dtype=torch.float64, device=p.device)
    for col, c in ((0, p % 16), (1, p // 16)):
        m = c % 8
        v = torch.where(m < 2, 0.5 * m, torch.where(m < 4, 0.5 * m, torch.where(
            m < 6, m.double() - 2, 2.0 * m.double() - 8)))
        out[..., col::2] = torch.where(c >= 8, -v.double(), v.double())
    return out * torch.exp2(s.double() - 127).repeat_interleave(BLOCK, -1)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "quant":
        rows = max(1, (1 << 25) // case["k"])
        return torch.cat([_exact_round(x) for x in state["x"].split(rows)])
    x = state["x"].double()
    functions = {"none": lambda y: y, "silu": torch.nn.functional.silu,
                 "gelu": torch.nn.functional.gelu, "relu": torch.relu,
                 "gelu_tanh": lambda y: torch.nn.functional.gelu(y, approximate="tanh")}
    if case["op"] == "moe":
        i = case["inter"]
        out = torch.zeros_like(x)
        for e in range(case["experts"]):
            t, j = torch.nonzero(state["ids"] == e, as_tuple=True)
            if t.numel():
                gate, up = torch.mm(x[t], _exact_weight(state["w13"], e).t()).split(i, 1)
                y = torch.mm(torch.nn.functional.silu(gate) * up,
                             _exact_weight(state["w2"], e).t())
                out.index_add_(0, t, y * state["weights"][t, j].double().unsqueeze(1))
        return out
    fn = functions[case["fn"]]
    if case["x4"]:
        x = _exact_round(x)
    b = 0.0 if state["bias"] is None else state["bias"].double()
    y = torch.mm(x, _exact_weight(state["w"]).t()) + b
    if case["op"] == "gated":
        gate, up = y.split(case["inter"], 1)
        return fn(gate) * up
    y = fn(y)
    return y if state["residual"] is None else y + state["residual"].double()
