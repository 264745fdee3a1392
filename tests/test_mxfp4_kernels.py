"""The choice of exq_linear_mxfp4's kernels: each is reached, and by the sizes that the GPU tests
take for it."""
import pytest

from exq_amd import _lib
from tests._mxfp4_cases import CASES, cases


def _kernel(T, N, x4, gated, K=64, stride=None):
    name = _lib.lib().exq_linear_mxfp4_kernel(_lib.LinearProblem(
        T, K, N, K, 0, 0, stride or -(-N // 4) * 4, _lib.U8 if x4 else _lib.BF16, 0, 0, _lib.BF16, 0, gated))
    return name and name.decode()


@pytest.mark.parametrize("x4,gated,kernel,T,N", cases())
def test_sizes_reach_their_kernel(x4, gated, kernel, T, N):
    assert _kernel(T, N, x4, gated) == kernel


def test_every_kernel_has_sizes():
    seen = {(x4, gated): {_kernel(T, N, x4, gated) for T in range(1, 4200, 37)
                          for N in (16, 128, 250, 1000, 2048, 4096, 8192, 16384)}
            for x4 in (False, True) for gated in (False, True)}
    assert {k: set(v) for k, v in CASES.items()} == seen


@pytest.mark.parametrize("x4", [False, True])
def test_unaligned_rows_take_streams_for_longer(x4):
    assert _kernel(187, 2047, x4, False, 1440).startswith("tile")
    assert _kernel(187, 2047, x4, False, 1440, stride=2047) == "stream 32x16"
    assert _kernel(2000, 2047, x4, False, 1440, stride=2047).startswith("tile")


def test_no_kernel_for_no_work_or_a_refused_problem():
    assert _kernel(0, 16, False, False) is None
    assert _kernel(4, 16, False, False, K=48) is None
