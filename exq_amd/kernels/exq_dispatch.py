"""Dispatch primitives on the HIP library.

Mirrors the pybind module ``exq_dispatch_cuda`` of the reference
(exq/kernels/cuda_src/exq_dispatch.cu:312-318: ``dispatch``,
``build_ends_from_slots``, ``gather_hidden``, ``combine``; all write into
caller-allocated outputs and return ``None``) plus the two sgl_kernel entry
points the reference pipeline calls (``moe_align_block_size`` and
``silu_and_mul``, exq/runtime/sglang_backend.py:79, 108-109, 140).
"""
from __future__ import annotations

import functools

import torch

from .. import _lib


def dispatch(router_indices: torch.Tensor, sort_order: torch.Tensor,
             sorted_expert_ids: torch.Tensor, expert_ends: torch.Tensor,
             n_experts: int) -> None:
    """Stable sort of the flat expert ids (exq_dispatch.cu:99-149).

    sort_order/sorted_expert_ids: int64 [n]; expert_ends: int32 [E+1].
    """
    ids = router_indices.reshape(-1)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    dev = _lib.require_gpu(ids, sort_order, sorted_expert_ids, expert_ends)
    n = ids.numel()
    if sort_order.numel() != n or sorted_expert_ids.numel() != n:
        raise ValueError("sort_order / sorted_expert_ids must have n = T*k entries")
    if expert_ends.numel() != n_experts + 1 or expert_ends.dtype != torch.int32:
        raise ValueError("expert_ends must be int32 [n_experts + 1]")
    if sort_order.dtype != torch.int64 or sorted_expert_ids.dtype != torch.int64:
        raise ValueError("sort_order and sorted_expert_ids must be int64")
    L = _lib.lib()
    _lib.check(L.exq_dispatch(ids.data_ptr(), _lib.dtype_code(ids.dtype), n, n_experts,
                              sort_order.data_ptr(), sorted_expert_ids.data_ptr(),
                              expert_ends.data_ptr(), _lib.stream_handle(dev)), "dispatch")


def build_ends_from_slots(sorted_slot_ids: torch.Tensor, flat_router: torch.Tensor,
                          expert_ends: torch.Tensor, sort_order: torch.Tensor,
                          n_active: int, n_experts: int) -> None:
    """Expert boundaries + compacted slot order (exq_dispatch.cu:181-229).

    sorted_slot_ids: int32 [EM] (from moe_align_block_size); flat_router:
    int32 [n_active]; expert_ends: int32 [E+1] (need not be zeroed);
    sort_order: int64 [n_active].
    """
    dev = _lib.require_gpu(sorted_slot_ids, flat_router, expert_ends, sort_order)
    if sorted_slot_ids.dtype != torch.int32 or flat_router.dtype != torch.int32:
        raise ValueError("sorted_slot_ids and flat_router must be int32")
    if expert_ends.dtype != torch.int32 or expert_ends.numel() != n_experts + 1:
        raise ValueError("expert_ends must be int32 [n_experts + 1]")
    if sort_order.dtype != torch.int64 or sort_order.numel() < n_active:
        raise ValueError("sort_order must be int64 with n_active entries")
    L = _lib.lib()
    _lib.check(L.exq_build_ends_from_slots(
        sorted_slot_ids.data_ptr(), sorted_slot_ids.numel(), flat_router.data_ptr(), n_active,
        n_experts, expert_ends.data_ptr(), sort_order.data_ptr(), _lib.stream_handle(dev)),
        "build_ends_from_slots")


def gather_hidden(hidden: torch.Tensor, sort_order: torch.Tensor, out: torch.Tensor,
                  top_k: int) -> None:
    """out[i] = hidden[sort_order[i] // top_k] (exq_dispatch.cu:234-260).

    Unlike the reference (fp16 only, exq_dispatch.cu:256-258) this accepts
    f32, f16 and bf16.
    """
    dev = _lib.require_gpu(hidden, sort_order, out)
    if sort_order.dtype != torch.int64:
        raise ValueError("sort_order must be int64")
    if out.dtype != hidden.dtype or out.shape != (sort_order.numel(), hidden.shape[1]):
        raise ValueError("out must be [n_active, H] with hidden's dtype")
    L = _lib.lib()
    _lib.check(L.exq_gather_hidden(hidden.data_ptr(), _lib.dtype_code(hidden.dtype),
                                   hidden.shape[0], hidden.shape[1], sort_order.data_ptr(),
                                   sort_order.numel(), top_k, out.data_ptr(),
                                   _lib.stream_handle(dev)), "gather_hidden")


def combine(down_out: torch.Tensor, sort_order: torch.Tensor, router_weights: torch.Tensor,
            result: torch.Tensor) -> None:
    """result[t] = sum_j w[t, j] * down_out[pos(t*k+j)] (exq_dispatch.cu:262-310).

    fp32 accumulation in fixed slot order (deterministic); ``result`` has
    ``down_out``'s dtype.
    """
    dev = _lib.require_gpu(down_out, sort_order, router_weights, result)
    T, k = router_weights.shape
    H = down_out.shape[1]
    if result.shape != (T, H) or result.dtype != down_out.dtype:
        raise ValueError("result must be [T, H] with down_out's dtype")
    n_active = sort_order.numel()
    L = _lib.lib()
    ws = _lib.workspace(dev, L.exq_combine_workspace_size(n_active))
    _lib.check(L.exq_combine(down_out.data_ptr(), _lib.dtype_code(down_out.dtype),
                             sort_order.data_ptr(), n_active, router_weights.data_ptr(),
                             _lib.dtype_code(router_weights.dtype), T, k, H, result.data_ptr(),
                             ws.data_ptr(), ws.numel(), _lib.stream_handle(dev)), "combine")


def moe_align_block_size(topk_ids: torch.Tensor, num_experts: int, block_size: int,
                         sorted_token_ids: torch.Tensor, experts_ids: torch.Tensor,
                         num_tokens_post_pad: torch.Tensor, cumsum_buffer: torch.Tensor,
                         pad_sorted_token_ids: bool = True) -> None:
    """Block-padded expert layout, with sgl_kernel's positional signature.

    Called by the reference as ``(topk_ids, E + 1, 16, sorted_ids, expert_blk,
    ntpp, cumsum, True)`` (sglang_backend.py:102-109).
    """
    ids = topk_ids.reshape(-1)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    dev = _lib.require_gpu(ids, sorted_token_ids, experts_ids, num_tokens_post_pad,
                           cumsum_buffer)
    for t in (sorted_token_ids, experts_ids, num_tokens_post_pad, cumsum_buffer):
        if t.dtype != torch.int32:
            raise ValueError("moe_align_block_size outputs must be int32")
    if cumsum_buffer.numel() < num_experts + 1:
        raise ValueError("cumsum_buffer needs num_experts + 1 entries")
    L = _lib.lib()
    _lib.check(L.exq_moe_align_block_size(
        ids.data_ptr(), _lib.dtype_code(ids.dtype), ids.numel(), num_experts, block_size,
        sorted_token_ids.data_ptr(), sorted_token_ids.numel(), experts_ids.data_ptr(),
        experts_ids.numel(), num_tokens_post_pad.data_ptr(), cumsum_buffer.data_ptr(),
        1 if pad_sorted_token_ids else 0, _lib.stream_handle(dev)), "moe_align_block_size")


def silu_and_mul(input: torch.Tensor, out: torch.Tensor) -> None:
    """out = silu(input[:, :I]) * input[:, I:] (gate first), fp32 math."""
    dev = _lib.require_gpu(input, out)
    rows, two_i = input.reshape(-1, input.shape[-1]).shape
    if two_i % 2 or out.numel() != rows * (two_i // 2) or out.dtype != input.dtype:
        raise ValueError("silu_and_mul: out must be [..., I] with input's dtype")
    L = _lib.lib()
    _lib.check(L.exq_silu_and_mul(input.data_ptr(), _lib.dtype_code(input.dtype), rows,
                                  two_i // 2, out.data_ptr(), _lib.stream_handle(dev)),
               "silu_and_mul")


def fused_topk(gating_output: torch.Tensor, topk: int, renormalize: bool,
               ids_dtype: torch.dtype = torch.int32,
               weights_dtype: torch.dtype = torch.float32):
    """Router on the GPU: fp32 softmax over ``gating_output`` [T, E], the top-k
    experts per token (descending, equal logits to the lower id) and their
    softmax weights, divided by their sum when ``renormalize``.

    Returns ``(topk_weights [T, k], topk_ids [T, k])`` like SGLang's
    ``fused_topk``; the reference computes the same routing with
    ``F.softmax`` + ``torch.topk`` + a division by the sum
    (exq/codegen/triton_emitter.py:273-277) and its SGLang hook consumes it as
    ``dispatch_output.topk_output`` (exq/runtime/sglang_backend.py:88-90).
    """
    if gating_output.dim() != 2:
        raise ValueError("gating_output must be [T, E]")
    g = gating_output if gating_output.is_contiguous() else gating_output.contiguous()
    dev = _lib.require_gpu(g)
    T, E = g.shape
    if not 1 <= topk <= min(E, 64):
        raise ValueError(f"topk={topk} must be in [1, min(E, 64)]")
    if E > 1024:
        raise ValueError(f"E={E} > 1024 experts is not supported")
    ids = torch.empty(T, topk, dtype=ids_dtype, device=dev)
    wts = torch.empty(T, topk, dtype=weights_dtype, device=dev)
    L = _lib.lib()
    _lib.check(L.exq_topk_softmax(g.data_ptr(), _lib.dtype_code(g.dtype), T, E, topk,
                                  1 if renormalize else 0, ids.data_ptr(),
                                  _lib.dtype_code(ids.dtype), wts.data_ptr(),
                                  _lib.dtype_code(wts.dtype), _lib.stream_handle(dev)),
               "fused_topk")
    return wts, ids


_SCORING = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}
_FLOAT_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


@functools.lru_cache(maxsize=4096)
def _route_problem(shape, dtype, bias, topk, renormalize, num_expert_group, topk_group,
                   scoring_func, group_score, scale, ids_dtype, weights_dtype):
    """The checked problem of a grouped_topk call, a function of its layouts and options
    alone (so they are checked once; the library only reads the problem)."""
    if len(shape) != 2:
        raise ValueError("gating_output must be [T, E]")
    if dtype not in _FLOAT_DTYPES:
        raise ValueError("gating_output must be float32, float16 or bfloat16")
    T, E = shape
    if not 1 <= E <= 1024:
        raise ValueError(f"E={E} experts is not in [1, 1024]")
    if not 1 <= num_expert_group <= 64 or E % num_expert_group:
        raise ValueError(f"num_expert_group={num_expert_group} must divide E={E} and be at most 64")
    if not 1 <= topk_group <= num_expert_group:
        raise ValueError(f"topk_group={topk_group} must be in [1, num_expert_group]")
    if not 1 <= topk <= min(64, E // num_expert_group * topk_group):
        raise ValueError(f"topk={topk} must be in [1, 64] and fit the experts of topk_group groups")
    if scoring_func not in _SCORING:
        raise ValueError(f"unsupported scoring_func {scoring_func!r}")
    if group_score is None:
        group_score = "max" if bias is None else "top2"
    if group_score not in _GROUP_SCORE:
        raise ValueError(f"unsupported group_score {group_score!r}")
    if ids_dtype not in (torch.int32, torch.int64) or weights_dtype not in _FLOAT_DTYPES:
        raise ValueError("ids must be int32 or int64, weights float32, float16 or bfloat16")
    if bias is not None and (bias[1] not in _FLOAT_DTYPES or tuple(bias[0]) != (E,)):
        raise ValueError(f"correction_bias must be [{E}], float32, float16 or bfloat16")
    code = _lib._TORCH_TO_CODE
    return _lib.RouteProblem(T, E, topk, num_expert_group, topk_group, code[dtype],
                             0 if bias is None else code[bias[1]], code[ids_dtype],
                             code[weights_dtype], _SCORING[scoring_func],
                             _GROUP_SCORE[group_score], 1 if renormalize else 0, scale)


def grouped_topk(gating_output: torch.Tensor, topk: int, renormalize: bool,
                 num_expert_group: int = 1, topk_group: int = 1, *,
                 scoring_func: str = "softmax", correction_bias: torch.Tensor | None = None,
                 group_score: str | None = None, routed_scaling_factor: float = 1.0,
                 num_token_non_padded: torch.Tensor | None = None,
                 ids_dtype: torch.dtype = torch.int32,
                 weights_dtype: torch.dtype = torch.float32):
    """Router with groups of experts, one kernel: softmax or sigmoid scores of
    ``gating_output`` [T, E], ranked by score + ``correction_bias`` [E] (a balancing
    bias; it ranks and never weighs), the ``topk_group`` best of ``num_expert_group``
    groups of consecutive experts, and the ``topk`` best experts in those.

    Returns ``(topk_weights [T, k], topk_ids [T, k])`` like ``fused_topk``: the
    scores of the chosen, divided by their sum when ``renormalize``, times
    ``routed_scaling_factor``; ids in descending order of the ranking, equal values
    to the lower id (equal groups to the lower group).  The ranking is that of the
    scores in 64 bits, whatever the logits' type.  ``group_score``: a group is worth
    its best expert ("max", the default without a bias) or the sum of its two best
    ("top2", the default with one).

    Logits or biases of -inf or NaN mask an expert: it has no part in the softmax,
    the group's value or the choice; a logit of +inf counts as the largest finite
    float32.  Slots that no expert is left for get id -1, which the expert layers
    drop, and weight 0; so do all slots of the rows from ``num_token_non_padded``
    (int32, one element on the device) on, the padding of a captured batch.
    Stream-ordered, graph-capturable, no workspace.  There is no derivative: inputs that
    require a gradient are refused unless gradients are off, and those with a forward-mode
    tangent, which ``torch.no_grad`` leaves on.
    """
    p = _route_problem(
        gating_output.shape, gating_output.dtype,
        None if correction_bias is None else (correction_bias.shape, correction_bias.dtype), topk,
        renormalize, num_expert_group, topk_group, scoring_func, group_score,
        float(routed_scaling_factor), ids_dtype, weights_dtype)
    if num_token_non_padded is not None and (num_token_non_padded.dtype != torch.int32
                                             or num_token_non_padded.numel() != 1):
        raise ValueError("num_token_non_padded must be one int32 element on the device")
    if torch.is_grad_enabled() and (gating_output.requires_grad or (
            correction_bias is not None and correction_bias.requires_grad)):
        raise ValueError("grouped_topk has no backward: call it under torch.no_grad()")
    _lib.refuse_tangents("grouped_topk", gating_output, correction_bias)
    g = gating_output if gating_output.is_contiguous() else gating_output.contiguous()
    dev = _lib.require_gpu(g, correction_bias, num_token_non_padded)
    T = p.n_tokens
    ids = torch.empty(T, topk, dtype=ids_dtype, device=dev)
    wts = torch.empty(T, topk, dtype=weights_dtype, device=dev)
    _lib.launch(_lib.lib().exq_grouped_topk,
                (p, g.data_ptr(), _lib.ptr(correction_bias), _lib.ptr(num_token_non_padded),
                 ids.data_ptr(), wts.data_ptr()), dev.index, "grouped_topk")
    return wts, ids
