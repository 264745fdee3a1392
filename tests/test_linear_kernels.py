"""Which kernel of exq_linear each size of tests/_linear_cases.py reaches, so that a change of
the choice cannot leave a kernel without its tests (no GPU)."""
import pytest
import torch

from exq_amd import _lib
from exq_amd.kernels import linear as L
from tests import _linear_cases as C

KERNELS = {"stream 16x16", "stream 32x16", "stream 16x32", "stream 32x32", "stream 64x32",
           "tile 64x64", "tile 64x128", "tile 128x128", "tile 128x256", "tile 192x256",
           "tile 256x256", "any stream 16x16", "any stream 16x32", "any stream 32x32",
           "any tile 64x64", "any tile 128x128"}


def _kernel(T, K, N, gated=False, x=4096, w=8192, ldx=None, ldw=None):
    code = _lib.BF16
    p = _lib.LinearProblem(T, K, N, K if ldx is None else ldx, K if ldw is None else ldw, N, N, code,
                           code, code, code, 0, int(gated))
    name = _lib.lib().exq_linear_kernel(p, x, w)
    return None if name is None else name.decode()


@pytest.mark.parametrize("kernel,gated,T,N", list(C.aligned()))
def test_aligned_sizes(kernel, gated, T, N):
    for K in (8, 1000, 8192):
        assert _kernel(T, K, N, gated) == kernel


@pytest.mark.parametrize("kernel,gated,T,N", list(C.unaligned()))
def test_sizes_of_any_layout(kernel, gated, T, N):
    assert _kernel(T, 1001, N, gated) == kernel                  # odd rows
    assert _kernel(T, 1002, N, gated) == kernel                  # rows of four bytes
    assert _kernel(T, 1000, N, gated, x=4098) == kernel          # a base in between
    assert _kernel(T, 1000, N, gated, w=8196) == kernel
    assert _kernel(T, 1000, N, gated, ldw=1001) == kernel
    assert _kernel(T, 1000, N, gated, ldx=1 << 23) == kernel     # past one buffer resource
    assert _kernel(T, 1000, N, gated, ldx=4 << 20) != kernel


def test_every_kernel_is_reached():
    both = {(kernel, gated) for kernel, gated, _, _ in [*C.aligned(), *C.unaligned()]}
    narrow = {"stream 16x16", "stream 32x16", "any stream 16x16"}  # not for gated rows
    assert both == {(k, g) for k in KERNELS for g in (False, True) if not (g and k in narrow)}


def test_refused_problems_have_no_kernel():
    assert _kernel(0, 8, 8) is None
    assert _kernel(4, 0, 8) is None
    assert _kernel(4, 8, 8, ldx=-8) is None
    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    p = L._problem(*[(t.shape, t.stride(), t.dtype) for t in (x, x)], None, None, None, None, None, 0)
    assert _lib.lib().exq_linear_kernel(p, x.data_ptr(), x.data_ptr()) is not None
