"""A large batch of padding: no slot has an expert."""
import pytest
import torch

from tests._helpers import banner

pytestmark = pytest.mark.gpu


def _us(call):
    times = []
    for _ in range(12):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        call()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    return sorted(times)[6] * 1e3


def test_dropped_batches_are_zeros_and_cost_less_than_routed_ones(device):
    """Every element of out is written once, by all of the chip."""
    from exq_amd.kernels import Mxfp4Weight, fused_experts_mxfp4
    T, H, I, E, k = 4096, 4096, 256, 8, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    w13 = Mxfp4Weight.quantize(torch.randn(E, 2 * I, H, generator=g, device=device) * 0.1, True)
    w2 = Mxfp4Weight.quantize(torch.randn(E, H, I, generator=g, device=device) * 0.1)
    x = torch.randn(T, H, generator=g, device=device).to(torch.bfloat16)
    w = torch.rand(T, k, generator=g, device=device)
    ids = torch.randint(0, E, (T, k), generator=g, device=device)
    none, out = torch.full_like(ids, -1), torch.full_like(x, float("nan"))
    banner("mxfp4 dropped batch")
    dropped = _us(lambda: fused_experts_mxfp4(x, w13, w2, w, none, out=out))
    assert (out == 0).all()
    routed = _us(lambda: fused_experts_mxfp4(x, w13, w2, w, ids, out=out))
    assert out.isfinite().all() and (out != 0).any()
    print(f"dropped {dropped:.0f} us, routed {routed:.0f} us")
    assert dropped < routed
