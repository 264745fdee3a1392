"""What the MXFP4 calls refuse, without a GPU: layouts, types, sizes, gradients, tangents."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from exq_amd import _lib
from exq_amd.kernels import (Mxfp4Weight, dequantize_mxfp4, fused_experts_mxfp4,
                             fused_gated_linear_mxfp4, fused_linear_mxfp4, quantize_mxfp4)

u8 = torch.uint8


def _weight(rows, cols, gated=False, experts=None):
    lead = () if experts is None else (experts,)
    RT, KB = (2 * -(-(rows // 2) // 16) if gated else -(-rows // 16)), -(-cols // 128)
    return Mxfp4Weight(torch.zeros(*lead, RT, KB, 64, 16, dtype=u8),
                       torch.zeros(*lead, RT, -(-KB // 4), 64, 4, dtype=u8), rows, cols, gated)


X = torch.zeros(4, 64, dtype=torch.bfloat16)
W = _weight(40, 64)
G = _weight(40, 64, gated=True)


@pytest.mark.parametrize("call,match", [
    (lambda: quantize_mxfp4(torch.zeros(4, 48)), "multiple of 32"),
    (lambda: quantize_mxfp4(torch.zeros(4, 0)), "multiple of 32"),
    (lambda: quantize_mxfp4(torch.zeros(4, 64, dtype=torch.int32)), "float32"),
    (lambda: quantize_mxfp4(torch.zeros(4, 64, requires_grad=True)), "no backward"),
    (lambda: dequantize_mxfp4(torch.zeros(4, 32, dtype=u8), torch.zeros(4, 3, dtype=u8)), "must be"),
    (lambda: dequantize_mxfp4(torch.zeros(4, 24, dtype=u8), torch.zeros(4, 1, dtype=u8)), "must be"),
    (lambda: dequantize_mxfp4(torch.zeros(4, 32), torch.zeros(4, 2, dtype=u8)), "uint8"),
    (lambda: dequantize_mxfp4(torch.zeros(4, 32, dtype=u8), torch.zeros(4, 2, dtype=u8), torch.int8),
     "dtype must be"),
    (lambda: Mxfp4Weight.from_packed(torch.zeros(5, 32, dtype=u8), torch.zeros(5, 2, dtype=u8), True),
     "gated"),
    (lambda: Mxfp4Weight.from_packed(torch.zeros(32, dtype=u8), torch.zeros(2, dtype=u8)), "N, K/2"),
    (lambda: Mxfp4Weight.from_packed(torch.zeros(0, 4, 32, dtype=u8),
                                     torch.zeros(0, 4, 2, dtype=u8)), "not empty"),
    (lambda: fused_linear_mxfp4(X[:, :32], W), "does not match"),
    (lambda: fused_linear_mxfp4(X.float(), W), "float16 or bfloat16"),
    (lambda: fused_linear_mxfp4(X, G), "gated"),
    (lambda: fused_gated_linear_mxfp4(X, W), "gated"),
    (lambda: fused_linear_mxfp4(X.t(), W), "."),
    (lambda: fused_linear_mxfp4(torch.zeros(64, 4, dtype=torch.bfloat16).t(), W), "contiguous rows"),
    (lambda: fused_linear_mxfp4(X, W._replace(rows=57)), "do not hold"),
    (lambda: fused_linear_mxfp4(X, W._replace(cols=48)), "cannot be"),
    (lambda: fused_linear_mxfp4(X, W._replace(tiles=W.tiles.float())), "uint8"),
    (lambda: fused_linear_mxfp4(X, W._replace(tiles=torch.zeros(64, 16, 3, 1, dtype=u8).permute(
        2, 3, 0, 1))), "contiguous"),
    (lambda: fused_linear_mxfp4(X, _weight(40, 64, experts=2)), "do not hold"),
    (lambda: fused_linear_mxfp4(X, W, activation="tanh"), "unsupported activation"),
    (lambda: fused_gated_linear_mxfp4(X, G, activation=None), "unsupported activation"),
    (lambda: fused_linear_mxfp4(X, W, torch.zeros(39)), "bias must be"),
    (lambda: fused_linear_mxfp4(X, W, torch.zeros(80)[::2]), "bias must be contiguous"),
    (lambda: fused_linear_mxfp4(X, W, residual=torch.zeros(4, 39)), "residual must be"),
    (lambda: fused_linear_mxfp4(X, W, out_dtype=torch.int8), "out_dtype"),
    (lambda: fused_linear_mxfp4(X, W, out=torch.zeros(4, 39)), "out must be"),
    (lambda: fused_linear_mxfp4(X, W, out=torch.zeros(1, 40).expand(4, 40)), "overlap"),
    (lambda: fused_linear_mxfp4(X.view(u8)[:, :32], W, x_scales=torch.zeros(4, 3, dtype=u8)), "do not match"),
    (lambda: fused_linear_mxfp4(X[:, :32], W, x_scales=torch.zeros(4, 2, dtype=u8)), "uint8"),
    (lambda: fused_linear_mxfp4(torch.zeros(4, 32, dtype=u8), W, x_scales=torch.zeros(2, 4, dtype=u8).t()),
     "x_scales must be contiguous"),
    (lambda: fused_linear_mxfp4(X.clone().requires_grad_(), W), "no backward"),
    (lambda: fused_linear_mxfp4(X, W, torch.zeros(40, requires_grad=True)), "no backward"),
])
def test_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


IDS = torch.zeros(4, 2, dtype=torch.int32)
WTS = torch.zeros(4, 2)
W13 = _weight(128, 64, True, 3)


@pytest.mark.parametrize("call,match", [
    (lambda: fused_experts_mxfp4(X, W13, _weight(64, 64, experts=2), WTS, IDS), "as many"),
    (lambda: fused_experts_mxfp4(X, W13, _weight(64, 64), WTS, IDS), "each expert"),
    (lambda: fused_experts_mxfp4(X, _weight(128, 64, False, 3), _weight(64, 64, experts=3), WTS, IDS), "gated"),
    (lambda: fused_experts_mxfp4(X, W13, _weight(64, 96, experts=3), WTS, IDS), "sizes"),
    (lambda: fused_experts_mxfp4(X[:, :32], W13, _weight(64, 64, experts=3), WTS, IDS), "sizes"),
    (lambda: fused_experts_mxfp4(X, W13, _weight(64, 64, experts=3), WTS[:3], IDS), "T, k"),
    (lambda: fused_experts_mxfp4(X, W13, _weight(64, 64, experts=3), WTS, IDS.float()), "int32 or int64"),
    (lambda: fused_experts_mxfp4(X, W13, _weight(64, 64, experts=3), WTS, IDS, activation="gelu"), "activation"),
    (lambda: fused_experts_mxfp4(X, W13, _weight(64, 64, experts=3), WTS.requires_grad_(), IDS), "no backward"),
])
def test_layer_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()
    WTS.requires_grad_(False)


@pytest.mark.parametrize("call", [
    lambda: quantize_mxfp4(torch.zeros(4, 64)),
    lambda: dequantize_mxfp4(torch.zeros(4, 32, dtype=u8), torch.zeros(4, 2, dtype=u8)),
    lambda: Mxfp4Weight.quantize(torch.zeros(4, 64)),
    lambda: Mxfp4Weight.from_packed(torch.zeros(4, 32, dtype=u8), torch.zeros(4, 2, dtype=u8)),
    lambda: fused_linear_mxfp4(X, W),
    lambda: fused_gated_linear_mxfp4(X, G),
    lambda: fused_experts_mxfp4(X, W13, _weight(64, 64, experts=3), WTS, IDS),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(_lib.ExqError, match="HIP device"):
        call()


@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_are_refused(no_grad):
    with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        b, r = torch.zeros(40), torch.zeros(4, 40)
        for call in (lambda: quantize_mxfp4(dual(torch.zeros(4, 64))),
                     lambda: fused_linear_mxfp4(dual(X), W),
                     lambda: fused_linear_mxfp4(X, W, dual(b)),
                     lambda: fused_linear_mxfp4(X, W, residual=dual(r)),
                     lambda: fused_gated_linear_mxfp4(dual(X), G),
                     lambda: fused_experts_mxfp4(dual(X), W13, _weight(64, 64, experts=3), WTS, IDS),
                     lambda: fused_experts_mxfp4(X, W13, _weight(64, 64, experts=3), dual(WTS), IDS)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


def test_library_refusals():
    """The C entries check before any launch."""
    L = _lib.lib()
    one = C.c_void_p(1 << 20)

    def linear(**kw):
        a = dict(n_tokens=1, in_features=64, out_features=16, x_stride=64, weight_stride=0,
                 residual_stride=0, out_stride=16, act_dtype=_lib.BF16, bias_dtype=0,
                 residual_dtype=0, out_dtype=_lib.BF16, activation=0, gated=0) | kw
        ptr = a.pop("x", one)
        return L.exq_linear_mxfp4(_lib.LinearProblem(**a), ptr, None, one, one, None,
                                  a.get("res"), one, None)

    assert linear(n_tokens=0) == 0
    for bad in (dict(in_features=48), dict(act_dtype=_lib.F32), dict(act_dtype=_lib.U8),
                dict(out_dtype=_lib.I8), dict(activation=9), dict(n_tokens=-1), dict(x_stride=-8),
                dict(n_tokens=2, out_stride=8), dict(n_tokens=2, x_stride=68), dict(x=None),
                dict(x=C.c_void_p((1 << 20) + 8)), dict(out_features=0)):
        assert linear(**bad) == 1, bad

    def moe(**kw):
        a = dict(n_tokens=4, hidden_size=64, inter_size=64, n_experts=8, top_k=2, n_shared=0,
                 group_size=32, act_dtype=_lib.BF16, ids_dtype=_lib.I32, weights_dtype=_lib.F32) | kw
        p = _lib.MoeProblem(**a)
        need = L.exq_moe_mxfp4_workspace_size(p)
        return need, L.exq_moe_mxfp4_forward(p, one, one, one, one, one, one, one, one, one, 64, None)

    assert moe() [1] == 3 and moe()[0] > 64        # workspace too small
    assert moe(n_tokens=0)[1] == 0
    for bad in (dict(hidden_size=48), dict(inter_size=0), dict(n_experts=1025), dict(top_k=65),
                dict(top_k=0), dict(n_shared=1), dict(group_size=128), dict(act_dtype=_lib.F32),
                dict(ids_dtype=_lib.U8), dict(weights_dtype=_lib.I8), dict(n_tokens=-1)):
        need, status = moe(**bad)
        assert need == 0 and status == 1, bad
    assert moe(n_tokens=1 << 24)[1] == 2           # slots
    assert moe(n_tokens=1 << 22, hidden_size=256, top_k=1)[1] == 2   # hidden past 2 GiB
    assert moe(n_tokens=(1 << 22) - 1, hidden_size=256, top_k=1)[1] == 3
    assert L.exq_quantize_mxfp4(one, _lib.F32, 1, 48, 48, one, one, None) == 1
    assert L.exq_quantize_mxfp4(one, _lib.I32, 1, 64, 64, one, one, None) == 1
    assert L.exq_quantize_mxfp4(one, _lib.F32, 0, 64, 64, None, None, None) == 0
    assert L.exq_dequantize_mxfp4(one, one, 1, 64, C.c_void_p(8), _lib.F32, None) == 1
    assert L.exq_tile_mxfp4(one, one, 1, 5, 64, 1, one, one, None) == 1
