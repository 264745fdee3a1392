"""MXFP4 (microscaled 4-bit floating point): quantisation, dense products and the MoE
layer with weights in it, beside the INT4 / INT8 / BF16 ones.

Blocks of 32 values along a row share a scale ``2**(s - 127)``, s one byte (255 is
NaN); a value is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  As stored: ``packed
[.., K/2]`` uint8, the even column in a byte's low half, and ``scales [.., K/32]``
uint8.  The products read a weight in the order of their tiles, which
``Mxfp4Weight.from_packed`` makes once when a model is loaded.  No counterpart in the
reference.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from .. import _lib
from .linear import _ACTIVATIONS, _FLOAT_DTYPES, _GATED, _check_out, _layout, _overlap, _row_stride

_BLOCK = 32


def _refuse_gradients(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no backward: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        _lib.refuse_tangents(what, *tensors)


def _device(first, *others) -> int:
    """The index of the one HIP device that all tensors are on."""
    dev = first.get_device()
    if dev < 0:
        raise _lib.ExqError("exq_amd kernels need tensors on a HIP device (got CPU tensor)")
    for t in others:
        if t is not None and t.get_device() != dev:
            if t.get_device() < 0:
                raise _lib.ExqError("exq_amd kernels need tensors on a HIP device (got CPU tensor)")
            raise _lib.ExqError(f"tensors on different devices: {first.device} and {t.device}")
    return dev


def _aligned(t: torch.Tensor, contiguous: bool = True) -> torch.Tensor:
    """``t``, or a copy that starts at a 16-byte address."""
    if contiguous:
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


# ---- quantisation -----------------------------------------------------------------------------

def quantize_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [.., K]`` (float32 / float16 / bfloat16, K a multiple of 32) to ``(packed
    [.., K/2], scales [.., K/32])``, uint8.

    A block's scale brings its largest magnitude into [4, 8); values go to the nearest
    code, halfway to the even one, and past 6 to 6.  A block with an infinity or a NaN
    reads back as NaN throughout.  Rows must be contiguous, the stride of a matrix's
    rows is free; other layouts are copied first.  Stream-ordered, graph-capturable.
    There is no derivative: an input that requires a gradient is refused unless
    gradients are off, and one with a forward-mode tangent always.
    """
    shape = x.shape
    if not shape or x.dtype not in _FLOAT_DTYPES:
        raise ValueError("x must be [.., K], float32, float16 or bfloat16")
    K = shape[-1]
    if K < _BLOCK or K % _BLOCK:
        raise ValueError(f"the last dimension must be a multiple of 32 (got {K})")
    _refuse_gradients("quantize_mxfp4", x)
    dev = _device(x)
    if len(shape) != 2 or x.stride(1) != 1:
        x = x.reshape(-1, K).contiguous()
    packed = x.new_empty((*shape[:-1], K // 2), dtype=torch.uint8)
    scales = x.new_empty((*shape[:-1], K // _BLOCK), dtype=torch.uint8)
    _lib.launch(_lib.lib().exq_quantize_mxfp4,
                (x.data_ptr(), _lib._TORCH_TO_CODE[x.dtype], x.shape[0], K, x.stride(0),
                 packed.data_ptr(), scales.data_ptr()), dev, "quantize_mxfp4")
    return packed, scales


def _check_stored(packed, scales):
    if packed.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError("packed and scales must be uint8")
    p, s = packed.shape, scales.shape
    if not p or not s or p[-1] < 16 or p[-1] % 16 or p[:-1] != s[:-1] or s[-1] * 16 != p[-1]:
        raise ValueError(f"packed {tuple(p)} and scales {tuple(s)} must be [.., K/2] and "
                         "[.., K/32], K a multiple of 32")


def dequantize_mxfp4(packed: torch.Tensor, scales: torch.Tensor,
                     dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``packed [.., K/2]`` and ``scales [.., K/32]`` back to ``[.., K]`` of ``dtype``
    (float32, bfloat16: every value but the two past their range exactly; float16:
    rounded to nearest)."""
    _check_stored(packed, scales)
    if dtype not in _FLOAT_DTYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    dev = _device(packed, scales)
    packed, scales = _aligned(packed), scales.contiguous()
    shape = packed.shape
    K = shape[-1] * 2
    out = packed.new_empty((*shape[:-1], K), dtype=dtype)
    _lib.launch(_lib.lib().exq_dequantize_mxfp4,
                (packed.data_ptr(), scales.data_ptr(), out.numel() // K, K, out.data_ptr(),
                 _lib._TORCH_TO_CODE[dtype]), dev, "dequantize_mxfp4")
    return out


# ---- weights ----------------------------------------------------------------------------------

class Mxfp4Weight(NamedTuple):
    """A weight ``[N, K]``, or one for each expert ``[E, N, K]``, in the order of tiles.

    ``tiles [.., RT, KB, 64, 16]`` and ``tile_scales [.., RT, ceil(KB / 4), 64, 4]`` uint8
    with KB = ceil(K / 128) and RT = ceil(N / 16): ``tiles[rt, kb, 16 q + r, b]`` is byte b
    of the block 4 kb + q of row 16 rt + r, ``tile_scales[rt, g, 16 q + r, i]`` the scale
    of the block 4 (4 g + i) + q of that row, zeros where there is none.  ``gated``: N
    = 2I, the gate rows first; each half is padded to 16 rows and their tiles alternate.
    """
    tiles: torch.Tensor
    tile_scales: torch.Tensor
    rows: int
    cols: int
    gated: bool = False

    @classmethod
    def from_packed(cls, packed: torch.Tensor, scales: torch.Tensor,
                    gated: bool = False) -> "Mxfp4Weight":
        """From ``packed [.., N, K/2]`` and ``scales [.., N, K/32]``, two or three axes."""
        _check_stored(packed, scales)
        if packed.dim() not in (2, 3) or packed.numel() == 0:
            raise ValueError("packed must be [N, K/2] or [E, N, K/2], not empty")
        lead, (rows, K) = packed.shape[:-2], (packed.shape[-2], packed.shape[-1] * 2)
        if gated and rows % 2:
            raise ValueError("a gated weight is [.., 2I, K]: the gate rows, then the up rows")
        dev = _device(packed, scales)
        packed, scales = _aligned(packed), scales.contiguous()
        RT, KB = _tile_grid(rows, K, gated)
        tiles = torch.empty(*lead, RT, KB, 64, 16, dtype=torch.uint8, device=packed.device)
        tile_scales = torch.empty(*lead, RT, -(-KB // 4), 64, 4, dtype=torch.uint8,
                                  device=packed.device)
        _lib.launch(_lib.lib().exq_tile_mxfp4,
                    (packed.data_ptr(), scales.data_ptr(), lead.numel(), rows, K, int(gated),
                     tiles.data_ptr(), tile_scales.data_ptr()), dev, "Mxfp4Weight.from_packed")
        return cls(tiles, tile_scales, rows, K, bool(gated))

    @classmethod
    def quantize(cls, weight: torch.Tensor, gated: bool = False) -> "Mxfp4Weight":
        """From a float weight ``[N, K]`` or ``[E, N, K]``."""
        return cls.from_packed(*quantize_mxfp4(weight), gated=gated)


def _tile_grid(rows: int, cols: int, gated: bool) -> tuple[int, int]:
    return (2 * -(-(rows // 2) // 16) if gated else -(-rows // 16)), -(-cols // 128)


def _check_weight(w, tiles, tile_scales, experts: bool):
    """Checks of an Mxfp4Weight by its tensors' layouts."""
    (shape, stride, dtype), (s_shape, s_stride, s_dtype) = tiles, tile_scales
    rows, cols, gated = w
    if dtype != torch.uint8 or s_dtype != torch.uint8:
        raise ValueError("tiles and tile_scales must be uint8")
    if rows < 1 or cols < _BLOCK or cols % _BLOCK or (gated and rows % 2):
        raise ValueError(f"a weight of {rows} rows and {cols} columns cannot be in MXFP4 tiles")
    RT, KB = _tile_grid(rows, cols, gated)
    lead = tuple(shape[:1]) if experts else ()
    if tuple(shape) != (*lead, RT, KB, 64, 16) or tuple(s_shape) != (*lead, RT, -(-KB // 4), 64, 4):
        raise ValueError(f"tiles {tuple(shape)} and tile_scales {tuple(s_shape)} do not hold "
                         f"{'weights of each expert' if experts else 'a weight'} of "
                         f"{rows} rows and {cols} columns{' (gated)' if gated else ''}")
    for sh, st in ((shape, stride), (s_shape, s_stride)):
        want = 1
        for n, have in zip(reversed(sh), reversed(st)):
            if n > 1 and have != want:
                raise ValueError("tiles and tile_scales must be contiguous")
            want *= n


def _check_start(address):
    if address & 15:
        raise ValueError("tiles and tile_scales must start at a 16-byte address")


# ---- dense products ---------------------------------------------------------------------------

@functools.lru_cache(maxsize=4096)
def _problem(x, x_scales, w, tiles, tile_scales, bias, residual, out, out_dtype, activation,
             gated) -> _lib.LinearProblem:
    """The checked problem of a call, a function of its tensors' layouts alone."""
    x_shape, x_stride, dtype = x
    rows, K, w_gated = w
    _check_weight(w, tiles, tile_scales, False)
    if bool(w_gated) != bool(gated):
        raise ValueError("a gated product takes a gated weight" if gated
                         else "this weight's gate and up rows are for a gated product")
    if len(x_shape) != 2:
        raise ValueError("x must be [T, K], or [T, K/2] with x_scales")
    n_out, T = rows // 2 if gated else rows, x_shape[0]
    code = _lib._TORCH_TO_CODE
    if x_scales is None:
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("x must be float16 or bfloat16, or packed with x_scales")
        if x_shape[1] != K:
            raise ValueError(f"x {tuple(x_shape)} does not match a weight of {K} columns")
    else:
        if dtype != torch.uint8 or x_scales[2] != torch.uint8:
            raise ValueError("packed x and x_scales must be uint8")
        if x_shape[1] * 2 != K or tuple(x_scales[0]) != (T, K // _BLOCK):
            raise ValueError(f"x {tuple(x_shape)} and x_scales {tuple(x_scales[0])} do not match "
                             f"a weight of {K} columns")
        if (K > _BLOCK and x_scales[1][1] != 1) or (T > 1 and x_scales[1][0] != K // _BLOCK):
            raise ValueError("x_scales must be contiguous")
    ldx, ldr = _row_stride(x_shape, x_stride, "x"), 0
    if bias is not None:
        if bias[2] not in _FLOAT_DTYPES or tuple(bias[0]) != (rows,):
            raise ValueError(f"bias must be [{rows}], float32, float16 or bfloat16")
        if rows > 1 and bias[1][0] != 1:
            raise ValueError("bias must be contiguous")
    if residual is not None:
        if residual[2] not in _FLOAT_DTYPES or tuple(residual[0]) != (T, n_out):
            raise ValueError(f"residual must be [{T}, {n_out}], float32, float16 or bfloat16")
        ldr = _row_stride(residual[0], residual[1], "residual")
    ldo = n_out
    if out is not None:
        if tuple(out[0]) != (T, n_out) or (out_dtype is not None and out[2] != out_dtype):
            raise ValueError(f"out must be [{T}, {n_out}] with dtype {out_dtype or out[2]}")
        out_dtype = out[2]
        ldo = _row_stride(out[0], out[1], "out")
        if T > 1 and ldo < n_out:
            raise ValueError("the rows of out overlap")
    if out_dtype is None:
        out_dtype = dtype if x_scales is None else torch.bfloat16
    if out_dtype not in _FLOAT_DTYPES:
        raise ValueError("out_dtype must be float32, float16 or bfloat16")
    return _lib.LinearProblem(T, K, n_out, ldx, 0, ldr, ldo, code[dtype],
                              0 if bias is None else code[bias[2]],
                              0 if residual is None else code[residual[2]], code[out_dtype],
                              _ACTIVATIONS[activation], gated)


_OUT_DTYPES = (torch.float32, torch.float16, torch.bfloat16)   # by code


def _call(x, weight, bias, x_scales, activation, residual, out_dtype, out, gated, what):
    tiles, tile_scales, rows, cols, w_gated = weight
    w = (rows, cols, w_gated)
    layouts = (_layout(x_scales), w, _layout(tiles), _layout(tile_scales), _layout(bias),
               _layout(residual), _layout(out), out_dtype, activation, gated)
    p = _problem(_layout(x), *layouts)
    _refuse_gradients(what, x, bias, residual, out)
    dev = _device(x, tiles, tile_scales, bias, x_scales, residual, out)
    _check_start(tiles.data_ptr() | tile_scales.data_ptr())
    if x.data_ptr() % 16 or (p.n_tokens > 1 and (p.x_stride * x.element_size() % 16
                                                 or p.x_stride > 1 << 22)):
        x = x.clone(memory_format=torch.contiguous_format)   # (rows at 16-byte addresses)
        p = _problem(_layout(x), *layouts)
    if out is None:
        out = x.new_empty((p.n_tokens, p.out_features), dtype=_OUT_DTYPES[p.out_dtype])
    elif p.n_tokens:
        _check_out(p, out, x, tiles.view(1, -1), bias, residual)
        for t in (tile_scales, x_scales):
            if t is not None and _overlap(out, p.out_stride, t.view(1, -1), t.numel()):
                raise ValueError("out overlaps an input")
    _lib.launch(_lib.lib().exq_linear_mxfp4,
                (p, x.data_ptr(), None if x_scales is None else x_scales.data_ptr(),
                 tiles.data_ptr(), tile_scales.data_ptr(), None if bias is None else bias.data_ptr(),
                 None if residual is None else residual.data_ptr(), out.data_ptr()), dev, what)
    return out


def fused_linear_mxfp4(x: torch.Tensor, weight: Mxfp4Weight, bias: torch.Tensor | None = None, *,
                       x_scales: torch.Tensor | None = None, activation: str | None = None,
                       residual: torch.Tensor | None = None,
                       out_dtype: torch.dtype | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` in one kernel, weight in MXFP4.

    x [T, K] float16 or bfloat16: the weight's values take its type (exactly in
    bfloat16; float16 rounds those below 2^-24 and overflows past 65504).  Or x
    [T, K/2] packed with ``x_scales`` [T, K/32], as ``quantize_mxfp4`` gives them: both
    operands go to the 4-bit matrix instructions.  bias, residual, ``activation`` and
    ``out`` as in ``fused_linear``; returns [T, N] in ``out_dtype`` (default x's,
    bfloat16 for packed x).  Sums in float32, one rounding at the end; the 4-bit
    instructions, which add 128 products and the sum so far at once, drop what lies more
    than 2^23 below the largest of them.  x's row stride is free; rows that do not start
    at 16-byte addresses, or lie more than 2^22 elements apart, are copied first.
    Stream-ordered, graph-capturable, no workspace, no derivative (as ``fused_linear``).
    """
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unsupported activation {activation!r}")
    return _call(x, weight, bias, x_scales, activation, residual, out_dtype, out, 0,
                 "fused_linear_mxfp4")


def fused_gated_linear_mxfp4(x: torch.Tensor, weight: Mxfp4Weight,
                             bias: torch.Tensor | None = None, *,
                             x_scales: torch.Tensor | None = None, activation: str = "silu",
                             out_dtype: torch.dtype | None = None,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """``activation(x @ Wg.T + bg) * (x @ Wu.T + bu)`` in one kernel.

    ``weight``: [2I, K] made with ``gated=True``; bias [2I], the gates' first.  Returns
    [T, I].  Everything else as in ``fused_linear_mxfp4``; ``activation``: "silu",
    "gelu", "gelu_tanh", "relu" or "sigmoid".
    """
    if activation not in _GATED:
        raise ValueError(f"unsupported activation {activation!r}")
    return _call(x, weight, bias, x_scales, activation, None, out_dtype, out, 1,
                 "fused_gated_linear_mxfp4")


# ---- MoE layer --------------------------------------------------------------------------------

@functools.lru_cache(maxsize=4096)
def _moe_problem(shape, dtype, w13, w13_rest, w2, w2_rest, weights, weights_dtype, ids, ids_dtype):
    """(checked problem, workspace bytes) of a layer call, by its tensors' shapes and types."""
    if len(shape) != 2:
        raise ValueError("hidden_states must be [T, H]")
    if len(ids) != 2 or ids != weights or ids[0] != shape[0]:
        raise ValueError("topk_ids / topk_weights must both be [T, k]")
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("hidden_states must be float16 or bfloat16")
    if ids_dtype not in (torch.int32, torch.int64):
        raise ValueError("topk_ids must be int32 or int64")
    if weights_dtype not in _FLOAT_DTYPES:
        raise ValueError("topk_weights must be float32, float16 or bfloat16")
    (tiles13, scales13, rows13, cols13, gated13), (tiles2, scales2, rows2, cols2, gated2) = w13, w2
    if not gated13 or gated2:
        raise ValueError("w13 must be a gated weight and w2 one that is not")
    if len(tiles13) != 5 or len(tiles2) != 5 or tiles2[0] != tiles13[0]:
        raise ValueError("w13 and w2 must hold a weight for each expert, as many the one as the other")
    for w, (tiles_layout, scales_layout) in ((w13, w13_rest), (w2, w2_rest)):
        _check_weight(w[2:], (w[0], *tiles_layout), (w[1], *scales_layout), True)
    T, H, E, I = *shape, tiles13[0], rows13 // 2
    if cols13 != H or (rows2, cols2) != (H, I):
        raise ValueError("the weights' sizes do not match hidden / intermediate sizes")
    code = _lib._TORCH_TO_CODE
    p = _lib.MoeProblem(T, H, I, E, ids[1], 0, _BLOCK, code[dtype], code[ids_dtype],
                        code[weights_dtype])
    need = _lib.lib().exq_moe_mxfp4_workspace_size(p)
    if not need:   # (the library's message: an argument out of its range)
        raise _lib.ExqError(_lib.lib().exq_last_error().decode(errors="replace"))
    return p, need


def _weight_key(w: Mxfp4Weight):
    return ((w.tiles.shape, w.tile_scales.shape, w.rows, w.cols, w.gated),
            ((w.tiles.stride(), w.tiles.dtype), (w.tile_scales.stride(), w.tile_scales.dtype)))


def fused_experts_mxfp4(hidden_states: torch.Tensor, w13: Mxfp4Weight, w2: Mxfp4Weight,
                        topk_weights: torch.Tensor, topk_ids: torch.Tensor, *,
                        activation: str = "silu", out: torch.Tensor | None = None,
                        workspace: torch.Tensor | None = None) -> torch.Tensor:
    """MoE layer with MXFP4 experts: ``out[t] = sum_j w[t, j] * down_e(silu(gate_e x) *
    up_e x)``.

    hidden_states [T, H] float16 / bfloat16; w13 of [E, 2I, H] made with ``gated=True``,
    w2 of [E, H, I]; topk_weights [T, k] float32 / float16 / bfloat16; topk_ids [T, k]
    int32 / int64 (ids outside [0, E) are dropped; a token without experts gets zeros).
    Returns [T, H] in hidden's type.  The weights' values take hidden's type as in
    ``fused_linear_mxfp4``; ``silu(gate) * up`` is rounded to it, as in ``fused_experts``
    (in float16 it becomes infinite past 65504), for the second product's matrix
    instructions, which take two operands of one type.
    Stream-ordered, no synchronisation with the host.  ``workspace``: uint8, at least
    ``moe_mxfp4_workspace_bytes(...)``, not shared by calls that may run at once;
    without one the call uses the calling thread's for the stream, and under graph
    capture one of the graph's.  ``out`` must not overlap an input.  No derivative.
    """
    if activation != "silu":
        raise ValueError(f"unsupported activation {activation!r} (only 'silu')")
    p, need = _moe_problem(hidden_states.shape, hidden_states.dtype, *_weight_key(w13),
                           *_weight_key(w2), topk_weights.shape, topk_weights.dtype,
                           topk_ids.shape, topk_ids.dtype)
    _refuse_gradients("fused_experts_mxfp4", hidden_states, topk_weights, out)
    tiles13, scales13, tiles2, scales2 = w13.tiles, w13.tile_scales, w2.tiles, w2.tile_scales
    dev = _device(hidden_states, topk_weights, topk_ids, tiles13, scales13, tiles2, scales2, out,
                  workspace)
    if dev != torch._C._cuda_getDevice():   # (the stream and its capture are that device's)
        with torch.cuda.device(dev):
            return fused_experts_mxfp4(hidden_states, w13, w2, topk_weights, topk_ids, out=out,
                                       workspace=workspace)
    a13, b13, a2, b2 = (tiles13.data_ptr(), scales13.data_ptr(), tiles2.data_ptr(),
                        scales2.data_ptr())
    _check_start(a13 | b13 | a2 | b2)
    if not (hidden_states.is_contiguous() and topk_ids.is_contiguous()
            and topk_weights.is_contiguous()):
        raise _lib.ExqError("exq_amd kernels need contiguous tensors")
    hidden_states = _aligned(hidden_states)
    if out is None:
        out = torch.empty_like(hidden_states)
    else:
        if out.shape != hidden_states.shape or out.dtype != hidden_states.dtype:
            raise ValueError(f"out must be {tuple(hidden_states.shape)} with dtype "
                             f"{hidden_states.dtype}")
        if not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("out must be contiguous and start at a 16-byte address")
        for t in (hidden_states, topk_weights, topk_ids, tiles13, scales13, tiles2, scales2,
                  workspace):
            if t is not None and t.numel() and out.numel() and _overlap(
                    out.view(1, -1), out.numel(), t.view(1, -1), t.numel()):
                raise ValueError("out overlaps an input")
    if p.n_tokens == 0:
        return out
    if workspace is None:
        workspace = _scratch(out, dev, need)
    else:
        if (workspace.dtype != torch.uint8 or not workspace.is_contiguous()
                or workspace.data_ptr() % 16):
            raise ValueError("workspace must be contiguous uint8 and start at a 16-byte address")
        for t in (hidden_states, topk_weights, topk_ids, tiles13, scales13, tiles2, scales2):
            if _overlap(workspace.view(1, -1), workspace.numel(), t.view(1, -1), t.numel()):
                raise ValueError("workspace overlaps an input")
    _lib.launch(_lib.lib().exq_moe_mxfp4_forward,
                (p, hidden_states.data_ptr(), topk_ids.data_ptr(), topk_weights.data_ptr(),
                 a13, b13, a2, b2, out.data_ptr(), workspace.data_ptr(), workspace.numel()), dev,
                "fused_experts_mxfp4")
    return out


def _scratch(out: torch.Tensor, index: int, need: int) -> torch.Tensor:
    """``_lib.workspace`` of out's device, which is the current one, with less Python where
    the buffer is there (0.5 of a call's 13 us)."""
    if not torch._C._cuda_isCurrentStreamCapturing():
        stream = torch._C._cuda_getCurrentRawStream(index)
        buf = _lib._workspaces.by_key.get((index, stream, "mxfp4"))
        if buf is not None and buf.numel() >= need:
            return buf
    return _lib.workspace(out.device, need, "mxfp4")


def moe_mxfp4_workspace_bytes(n_tokens: int, hidden: int, inter: int, n_experts: int,
                              top_k: int) -> int:
    """Workspace bytes that ``fused_experts_mxfp4`` needs for this problem size."""
    return _lib.lib().exq_moe_mxfp4_workspace_size(
        _lib.MoeProblem(n_tokens, hidden, inter, n_experts, top_k, 0, _BLOCK, _lib.BF16, _lib.I32,
                        _lib.F32))
