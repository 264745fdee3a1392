"""Inputs with a forward-mode tangent are refused like inputs that require a gradient: the
operators have no derivative, and a result without a tangent would be taken for a constant."""
import pytest
import torch
from torch.autograd import forward_ad

from exq_amd import _lib
from exq_amd.kernels import fused_gated_linear, fused_linear, grouped_topk


def _calls(dual):
    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    w = torch.zeros(8, 16, dtype=torch.bfloat16)
    b, r = torch.zeros(8), torch.zeros(4, 8)
    return [lambda: grouped_topk(dual(r), 2, True),
            lambda: grouped_topk(r, 2, True, correction_bias=dual(b)),
            lambda: grouped_topk(dual(r)[:, ::2], 2, True),
            lambda: fused_linear(dual(x), w), lambda: fused_linear(x, dual(w)),
            lambda: fused_linear(x, w, dual(b)), lambda: fused_linear(x, w, residual=dual(r)),
            lambda: fused_linear(x, w, out=dual(r)),
            lambda: fused_gated_linear(dual(x), w), lambda: fused_gated_linear(x, dual(w)),
            lambda: fused_gated_linear(x, w, dual(b))]


@pytest.mark.parametrize("i", range(11))
@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_are_refused(i, no_grad):
    """Under no_grad too, which does not turn forward mode off."""
    with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        call = _calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))[i]
        with pytest.raises(ValueError, match="forward-mode"):
            call()


@pytest.mark.parametrize("i", range(11))
def test_no_tangent_no_refusal(i):
    """An open level alone changes nothing (here: the refusal of CPU tensors)."""
    with forward_ad.dual_level():
        with pytest.raises(_lib.ExqError, match="HIP device"):
            _calls(lambda t: t)[i]()
