"""Two threads that call layers on one stream: each gets what it gets alone, bit for bit (the
layers repeat exactly)."""
import threading

import pytest
import torch

from tests._helpers import banner

pytestmark = pytest.mark.gpu

H, I, E, K = 512, 256, 16, 4


def _inputs(T, seed, device):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(device)
    ids = torch.randn(T, E, generator=g).topk(K, -1).indices.to(torch.int32).to(device)
    return x, ids, (torch.rand(T, K, generator=g) + 0.1).to(device)


def _int4(T, seed, device):
    from exq_amd import synth
    from exq_amd.kernels import fused_experts, pack_experts_int4
    w13, w2 = synth.expert_weights_gpu(E, I, H, seed, device)
    weights = (*pack_experts_int4(w13), *pack_experts_int4(w2))
    x, ids, w = _inputs(T, seed, device)
    return lambda: fused_experts(x, *weights, w, ids)


def _mxfp4(T, seed, device):
    from exq_amd.kernels import Mxfp4Weight, fused_experts_mxfp4
    g = torch.Generator().manual_seed(seed)
    w13 = Mxfp4Weight.quantize((torch.randn(E, 2 * I, H, generator=g) * 0.1).to(device), True)
    w2 = Mxfp4Weight.quantize((torch.randn(E, H, I, generator=g) * 0.1).to(device))
    x, ids, w = _inputs(T, seed, device)
    return lambda: fused_experts_mxfp4(x, w13, w2, w, ids)


def _routed(T, seed, device):
    from exq_amd import synth
    from exq_amd.kernels import moe_int4_forward, pack_experts_int4, unsort_output
    w13, _ = synth.expert_weights_gpu(E, I, H, seed, device)
    packed, scales = pack_experts_int4(w13)
    x, ids, w = _inputs(T, seed, device)
    return lambda: unsort_output(moe_int4_forward(x, packed, scales, ids, E), ids, w, E)


@pytest.mark.parametrize("make", [_int4, _mxfp4, _routed], ids=["int4", "mxfp4", "routed"])
@pytest.mark.parametrize("sizes", [(1, 8), (16, 48), (48, 200), (300, 40)])
def test_threads_on_one_stream(make, sizes, device):
    banner(f"threads {make.__name__} {sizes}")
    calls = [make(T, 3 + i, device) for i, T in enumerate(sizes)]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    start, got, errors = threading.Barrier(2), [[], []], []

    def work(i):
        try:
            start.wait(30)
            for _ in range(40):
                got[i].append(calls[i]())
        except Exception as e:      # (a thread's own is not the test's)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for outs, ref in zip(got, want):
        assert len(outs) == 40 and all(torch.equal(o, ref) for o in outs)
