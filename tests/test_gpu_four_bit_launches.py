"""Launches of the operators that serve from 4 bits: as many as are counted, and none overlaps another where the switch for that is off."""

import pytest
import torch

from test_gpu_kernels import DEV, K

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _kernels(fn) -> int:
    """Kernel nodes of a captured ``fn()`` (nothing is run)."""
    from cuda.bindings import runtime as R

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        keep = fn()
    rc, nodes, n = R.cudaGraphGetNodes(R.cudaGraph_t(graph.raw_cuda_graph()), 1000)
    assert rc == R.cudaError_t.cudaSuccess and 0 < n < 1000, rc
    kinds = [R.cudaGraphNodeGetType(node)[1] for node in nodes[:n]]
    del keep
    return sum(kind == R.cudaGraphNodeType.cudaGraphNodeTypeKernel for kind in kinds)


@pytest.mark.parametrize("m,n,k,dtype", [(1, 6144, 256, BF), (16, 389, 128, BF), (5, 389, 80, F32), (17, 128, 64, BF), (17, 128, 128, BF), (48, 2560, 1280, BF), (64, 148 * 128, 256, BF),
                                         (64, 19456, 256, BF), (200, 256, 64, BF), (256, 148 * 128, 192, BF), (256, 389, 64, BF)])
def test_every_launch_of_a_product_is_counted(m, n, k, dtype):
    """One for few rows, in 32 bits, and where every block has a whole tile; else two."""
    w4, x = K().pack_weight4(torch.randn(n, k, device=DEV), 16), torch.randn(m, k, device=DEV).to(dtype)
    K().linear4(x, w4)                       # (loads the library)
    before = K().launch_count
    made = _kernels(lambda: K().linear4(x, w4))
    assert K().launch_count - before == made
