"""The layer on both sides of the choice between slots and tiles, for small experts and large
ones, against products in 64 bits."""
import pytest
import torch

from tests._helpers import banner

pytestmark = pytest.mark.gpu


def _whole(shape, g, device):
    """An MXFP4 weight of -1, 0 and 1, most of them zero."""
    pick = torch.randint(0, 16, shape, generator=g, device=device)
    return (pick == 1).float() - (pick == 2).float()


# T, H, I, E, k
@pytest.mark.parametrize("T,H,I,E,k", [
    (1, 4096, 4096, 5, 4), (1, 4096, 4096, 6, 5), (4, 4096, 4128, 3, 1), (3, 4096, 4128, 3, 2),
    (1, 4096, 1024, 16, 12), (1, 4096, 1024, 16, 13), (2, 2048, 1408, 9, 8), (16, 1056, 512, 7, 1),
    (17, 1056, 512, 7, 1), (4, 160, 96, 9, 4), (6, 160, 96, 9, 4), (8, 160, 96, 3, 4),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_whole_numbers(T, H, I, E, k, dtype, device):
    """x has one column that is not zero, so gate and up are whole numbers of one product; up
    is 64 where gate is 32 (silu(32) rounds to 32 in 32 bits), and the sums over I and over
    the slots, times router weights of 1/2 and 1, are exact in float32."""
    from exq_amd.kernels import Mxfp4Weight, fused_experts_mxfp4
    banner(f"mxfp4 paths T={T} H={H} I={I} E={E} k={k} {dtype}")
    g = torch.Generator(device=device).manual_seed(T * H + I)
    gate = torch.full((E, I, H), 4.0, device=device)
    up = _whole((E, I, H), g, device)
    down = _whole((E, H, I), g, device)
    w13 = Mxfp4Weight.quantize(torch.cat((gate, up), 1), gated=True)
    w2 = Mxfp4Weight.quantize(down)
    at = torch.randint(0, H, (T,), generator=g, device=device)
    x = torch.zeros(T, H, dtype=dtype, device=device)
    x[torch.arange(T, device=device), at] = 8.0
    ids = torch.randint(-1, E, (T, k), generator=g, device=device)
    w = torch.randint(1, 3, (T, k), generator=g, device=device).float() / 2
    out = fused_experts_mxfp4(x, w13, w2, w, ids)
    want = torch.zeros(T, H, dtype=torch.float64, device=device)
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j])
            if e >= 0:
                mid = 32.0 * 8.0 * up[e, :, at[t]].double()
                want[t] += w[t, j].double() * torch.mv(down[e].double(), mid)
    assert torch.equal(out, want.float().to(dtype))
    assert torch.equal(fused_experts_mxfp4(x, w13, w2, w, ids), out)
