"""Dense products with their epilogue, for what stands beside the routed experts of
a MoE block: the router's projection, shared experts and dense layers.

``fused_linear`` adds the bias, applies the activation and adds the residual (the
routed experts' output, for a shared expert's down projection) in the product's
epilogue; ``fused_gated_linear`` is a gate / up projection with the activation and
the product of the halves in it, in place of a product and ``silu_and_mul``.  No
counterpart in the reference, which leaves these layers to SGLang.
"""
from __future__ import annotations

import functools

import torch

from .. import _lib

_ACT_DTYPES = (torch.float16, torch.bfloat16)
_FLOAT_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4,
                "sigmoid": 5}
_GATED = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def _row_stride(shape: tuple, stride: tuple, what: str) -> int:
    """Elements from row to row of a matrix whose rows are contiguous."""
    rows, cols = shape
    if cols > 1 and stride[1] != 1:
        raise ValueError(f"{what} must have contiguous rows (last stride 1)")
    return stride[0] if rows > 1 else cols


def _overlap(a: torch.Tensor, a_stride: int, b: torch.Tensor, b_stride: int) -> bool:
    """Whether two row-strided matrices share bytes (for unequal strides: whether
    their address ranges meet)."""
    def span(t, stride):
        rows, cols = (t.shape[0], t.shape[1]) if t.dim() == 2 else (1, t.shape[0])
        return rows, cols * t.element_size(), stride * t.element_size()
    ra, wa, pa = span(a, a_stride)
    rb, wb, pb = span(b, b_stride)
    a0, b0 = a.data_ptr(), b.data_ptr()
    if a0 + (ra - 1) * pa + wa <= b0 or b0 + (rb - 1) * pb + wb <= a0:
        return False
    if pa == pb and ra > 1 and rb > 1 and wa <= pa and wb <= pb:
        d = (b0 - a0) % pa   # column slices of one buffer lie beside each other
        return d < wa or d + wb > pa
    return True


def _layout(t: torch.Tensor | None):
    return None if t is None else (t.shape, t.stride(), t.dtype)


@functools.lru_cache(maxsize=4096)
def _problem(x, weight, bias, residual, out, out_dtype, activation, gated) -> _lib.LinearProblem:
    """The checked problem of a call, a function of its tensors' layouts alone (so the
    checks are made once for a layout; the library only reads the problem)."""
    (x_shape, x_stride, dtype), (w_shape, w_stride, w_dtype) = x, weight
    if len(x_shape) != 2 or len(w_shape) != 2:
        raise ValueError("x must be [T, K] and weight [N, K]")
    if gated and w_shape[0] % 2:
        raise ValueError("weight must be [2I, K]: the gate rows, then the up rows")
    T, K = x_shape
    n_out = w_shape[0] // 2 if gated else w_shape[0]
    if w_shape[1] != K or K < 1 or n_out < 1:
        raise ValueError(f"weight {tuple(w_shape)} does not match x {tuple(x_shape)}")
    if dtype not in _ACT_DTYPES or w_dtype != dtype:
        raise ValueError("x and weight must both be float16 or both bfloat16")
    ldx, ldw, ldr = _row_stride(x_shape, x_stride, "x"), _row_stride(w_shape, w_stride,
                                                                     "weight"), 0
    if bias is not None:
        if bias[2] not in _FLOAT_DTYPES or tuple(bias[0]) != (w_shape[0],):
            raise ValueError(f"bias must be [{w_shape[0]}], float32, float16 or bfloat16")
        if w_shape[0] > 1 and bias[1][0] != 1:
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
        out_dtype = dtype
    if out_dtype not in _FLOAT_DTYPES:
        raise ValueError("out_dtype must be float32, float16 or bfloat16")
    code = _lib._TORCH_TO_CODE
    return _lib.LinearProblem(T, K, n_out, ldx, ldw, ldr, ldo, code[dtype],
                              0 if bias is None else code[bias[2]],
                              0 if residual is None else code[residual[2]], code[out_dtype],
                              _ACTIVATIONS[activation], gated)


def _check_out(p, out, x, weight, bias, residual):
    """``out`` may be the residual and overlaps nothing else."""
    if p.n_tokens == 0:
        return
    ldo, ldr = p.out_stride, p.residual_stride
    if residual is not None and _overlap(out, ldo, residual, ldr) and not (
            out.data_ptr() == residual.data_ptr() and out.dtype == residual.dtype
            and ldo == ldr):
        raise ValueError("out overlaps the residual without being it")
    if (_overlap(out, ldo, x, p.x_stride) or _overlap(out, ldo, weight, p.weight_stride)
            or (bias is not None and _overlap(out, ldo, bias, bias.numel()))):
        raise ValueError("out overlaps an input")


def _call(x, weight, bias, activation, residual, out_dtype, out, gated, what):
    p = _problem((x.shape, x.stride(), x.dtype), (weight.shape, weight.stride(), weight.dtype),
                 _layout(bias), _layout(residual), _layout(out), out_dtype, activation, gated)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)
                                    or (out is not None and out.requires_grad)):
        raise ValueError(f"{what} has no backward: call it under torch.no_grad()")
    _lib.refuse_tangents(what, x, weight, bias, residual, out)
    dev = x.get_device()
    if dev < 0:
        raise _lib.ExqError("exq_amd kernels need tensors on a HIP device (got CPU tensor)")
    for t in (weight, bias, residual, out):
        if t is not None and t.get_device() != dev:
            raise _lib.ExqError(f"tensors on different devices: {x.device} and {t.device}")
    if out is None:
        out = torch.empty(p.n_tokens, p.out_features, dtype=out_dtype or x.dtype, device=x.device)
    else:
        _check_out(p, out, x, weight, bias, residual)
    _lib.launch(_lib.lib().exq_linear,
                (p, x.data_ptr(), weight.data_ptr(), None if bias is None else bias.data_ptr(),
                 None if residual is None else residual.data_ptr(), out.data_ptr()), dev, what)
    return out


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 activation: str | None = None, residual: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` in one kernel.

    x [T, K] and weight [N, K] float16 or bfloat16; bias [N] and residual [T, N]
    float32 / float16 / bfloat16; returns [T, N] in ``out_dtype`` (default x's;
    float32 for router logits).  ``activation``: None, "relu", "silu", "gelu"
    (erf), "gelu_tanh" or "sigmoid".  Sums in float32, one rounding at the end.
    Rows must be contiguous, row strides are free (column slices, expanded rows).
    ``out`` may be ``residual`` itself, to add in place, and must not overlap any
    other input.  Stream-ordered, graph-capturable, no workspace.  There is no
    derivative: inputs that require a gradient are refused unless gradients are off, and
    those with a forward-mode tangent, which ``torch.no_grad`` leaves on.
    """
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unsupported activation {activation!r}")
    return _call(x, weight, bias, activation, residual, out_dtype, out, 0, "fused_linear")


def fused_gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                       *, activation: str = "silu", out_dtype: torch.dtype | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """``activation(x @ Wg.T + bg) * (x @ Wu.T + bu)`` in one kernel.

    weight [2I, K] holds the I gate rows first, then the I up rows (the layout of
    w13), bias [2I] likewise; returns [T, I].  Types, strides and ``out`` as in
    ``fused_linear``; ``activation``: "silu", "gelu", "gelu_tanh", "relu" or
    "sigmoid".
    """
    if activation not in _GATED:
        raise ValueError(f"unsupported activation {activation!r}")
    return _call(x, weight, bias, activation, None, out_dtype, out, 1, "fused_gated_linear")
