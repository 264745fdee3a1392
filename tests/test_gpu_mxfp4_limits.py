"""Where the MXFP4 operators' arithmetic ends, as their documentation says it."""
import pytest
import torch

from tests._helpers import banner

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 6, 40, 300])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gate_times_up_past_float16(dtype, T, device):
    """silu(256) * 256 is 2^16 in 32 bits: infinite in float16, and 2^16 in bfloat16, where 32
    of them times 2^-4 are 2^17."""
    from exq_amd.kernels import Mxfp4Weight, fused_experts_mxfp4
    banner(f"mxfp4 gate times up {dtype} T={T}")
    H, I = 32, 32
    w13, w2 = torch.zeros(2, 2 * I, H), torch.zeros(2, H, I)
    w13[:, :, 0] = 4.0
    w2[:] = 2.0 ** -4
    w13, w2 = Mxfp4Weight.quantize(w13.to(device), True), Mxfp4Weight.quantize(w2.to(device))
    x = torch.zeros(T, H, dtype=dtype, device=device)
    x[:, 0] = 64.0
    ids = (torch.arange(T, device=device) % 2).view(T, 1)
    out = fused_experts_mxfp4(x, w13, w2, torch.ones(T, 1, device=device), ids)
    assert (out == (float("inf") if dtype == torch.float16 else 2.0 ** 17)).all()


@pytest.mark.parametrize("T", [1, 40, 1500])
@pytest.mark.parametrize("far", [10, 22, 30])
def test_terms_of_far_sizes_in_one_instruction(far, T, device):
    """2^far - 2^far + 36 in one instruction's 128 columns.  The 36, a multiple of 4, is whole
    where 2^far lies at most 2^23 above 4, and may go beyond: the sum is off by at most (128 + 1
    + 8) 2^-23 sum |x w|."""
    from exq_amd.kernels import Mxfp4Weight, fused_linear_mxfp4, quantize_mxfp4
    banner(f"mxfp4 far terms 2^{far} T={T}")
    K, N = 128, 48
    x, w = torch.zeros(T, K), torch.zeros(N, K)
    x[:, 0], x[:, 32], x[:, 64] = 2.0 ** far, 2.0 ** far, 6.0
    w[:, 0], w[:, 32], w[:, 64] = 1.0, -1.0, 6.0
    p, s = quantize_mxfp4(x.to(device))
    out = fused_linear_mxfp4(p, Mxfp4Weight.quantize(w.to(device)), x_scales=s,
                             out_dtype=torch.float32).cpu()
    bound = (128 + 1 + 8) * 2.0 ** -23 * (2.0 * 2.0 ** far + 36.0)
    assert ((out - 36.0).abs() <= (0.0 if far <= 22 else bound)).all()
