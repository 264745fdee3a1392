"""Rows whose runs cannot be stored at once: streams for longer than aligned ones, and tiles
again where a product is long enough that its last columns do not count."""
import pytest

from exq_amd import _lib


def _kernel(T, K, N, x4, stride):
    return _lib.lib().exq_linear_mxfp4_kernel(_lib.LinearProblem(
        T, K, N, K, 0, stride, stride, _lib.U8 if x4 else _lib.BF16, 0, 0, _lib.BF16, 0, 0)).decode()


@pytest.mark.parametrize("T,K,N,x4,unaligned,aligned", [
    (100, 1440, 2047, False, "stream", "tile"), (400, 512, 1001, False, "stream", "tile"),
    (400, 512, 2047, False, "tile", "tile"), (187, 4096, 2047, False, "tile", "tile"),
    (187, 4096, 4097, True, "tile", "tile"), (187, 1440, 2047, True, "stream", "tile"),
    (400, 512, 1001, True, "stream", "tile"), (24, 512, 1001, True, "stream", "stream"),
])
def test_unaligned_rows(T, K, N, x4, unaligned, aligned):
    assert _kernel(T, K, N, x4, N).startswith(unaligned)
    assert _kernel(T, K, N, x4, -(-N // 4) * 4).startswith(aligned)
