"""How a layer of few slots runs, told by its workspace: fp32 rows of every slot's result where
it runs on tiles, none where it runs by slots."""
import pytest

from exq_amd.kernels.mxfp4 import moe_mxfp4_workspace_bytes


def _on_tiles(T, H, I, E, k):
    need, n = moe_mxfp4_workspace_bytes(T, H, I, E, k), T * k
    rest = need - 2 * n * I
    assert rest < 16384 or rest >= 4 * n * H
    return rest >= 4 * n * H


@pytest.mark.parametrize("T,H,I,E,k,tiles", [
    (1, 2048, 768, 128, 8, False), (2, 2048, 768, 128, 8, False), (3, 2048, 768, 128, 8, True),
    (1, 8192, 8192, 12, 4, False), (1, 8192, 8192, 12, 5, True), (2, 4096, 14336, 8, 2, False),
    (3, 4096, 14336, 8, 2, True), (1, 6144, 2048, 64, 8, True), (1, 4096, 1024, 64, 8, False),
    (3, 4096, 1024, 64, 4, False), (13, 4096, 1024, 64, 1, True), (16, 2048, 1408, 64, 1, False),
    (17, 2048, 256, 64, 1, True), (64, 2048, 768, 128, 8, True),
])
def test_large_experts_leave_the_slots_early(T, H, I, E, k, tiles):
    """Up to four slots by slots, up to 16 where slots x H x I is at most 3 x 2^24: a slot by
    itself keeps few of its weights on their way."""
    assert _on_tiles(T, H, I, E, k) == tiles
