"""Launches of the operators that serve from 4 bits: as many as are counted, and none overlaps another where the switch for that is off."""

import ctypes

import pytest
import torch

from test_gpu_four_bit import Cache, i32
from test_gpu_kernels import DEV, K

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


class _Edge(ctypes.Structure):
    _fields_ = [("from_port", ctypes.c_ubyte), ("to_port", ctypes.c_ubyte), ("type", ctypes.c_ubyte), ("reserved", ctypes.c_ubyte * 5)]


def _captured(fn):
    """(kernel nodes, edges on which a launch may start before the one in front of it has ended) of a captured ``fn()`` (nothing is run).  The runtime is asked with
    arrays of this function's own; those of the Python binding are given back before they can be read."""
    graph, runtime, room = torch.cuda.CUDAGraph(keep_graph=True), ctypes.CDLL("libcudart.so.12"), 1000
    with torch.cuda.graph(graph):
        keep = fn()
    raw, n, kind = ctypes.c_void_p(int(graph.raw_cuda_graph())), ctypes.c_size_t(room), ctypes.c_int(0)
    nodes, begins, ends, data = (ctypes.c_void_p * room)(), (ctypes.c_void_p * room)(), (ctypes.c_void_p * room)(), (_Edge * room)()
    assert runtime.cudaGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0 and 0 < n.value < room
    kernels = 0
    for node in nodes[:n.value]:
        assert runtime.cudaGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        kernels += kind.value == 0                     # cudaGraphNodeTypeKernel
    n = ctypes.c_size_t(room)
    assert runtime.cudaGraphGetEdges_v2(raw, begins, ends, data, ctypes.byref(n)) == 0 and n.value < room
    del keep
    return kernels, sum(data[i].type == 1 for i in range(n.value))      # cudaGraphDependencyTypeProgrammatic


@pytest.mark.parametrize("m,n,k,dtype", [(1, 6144, 256, BF), (16, 389, 128, BF), (5, 389, 80, F32), (17, 128, 64, BF), (17, 128, 128, BF), (48, 2560, 1280, BF), (64, 148 * 128, 256, BF),
                                         (64, 19456, 256, BF), (200, 256, 64, BF), (256, 148 * 128, 192, BF), (256, 389, 64, BF)])
def test_every_launch_of_a_product_is_counted(m, n, k, dtype):
    """One for few rows, in 32 bits, and where every block has a whole tile; else two."""
    w4, x = K().pack_weight4(torch.randn(n, k, device=DEV), 16), torch.randn(m, k, device=DEV).to(dtype)
    K().linear4(x, w4)                       # (loads the library)
    before = K().launch_count
    made, _ = _captured(lambda: K().linear4(x, w4))
    assert K().launch_count - before == made


@pytest.mark.parametrize("m,n,k,passes", [(48, 2560, 1280, 1), (128, 148 * 128, 256, 1), (129, 389, 64, 2), (200, 2560, 1280, 2), (256, 148 * 128, 256, 2)])
def test_every_launch_of_a_product_with_a_32_bit_result_is_counted(m, n, k, passes):
    """More than 128 rows are two passes; with overlapped launches and without, the same bits."""
    w4, x, y = K().pack_weight4(torch.randn(n, k, device=DEV), 16), torch.randn(m, k, device=DEV).to(BF), {}
    for pdl in (True, None, False):
        y[pdl] = K().linear4(x, w4, out_dtype=F32, pdl=pdl)
        before = K().launch_count
        made, overlapped = _captured(lambda: (x.mul_(1.0), K().linear4(x, w4, out_dtype=F32, pdl=pdl)))
        assert K().launch_count - before == made - 1 and made - 1 in (passes, 2 * passes)
        assert overlapped == {True: made - 1, None: made - 2, False: 0}[pdl]
    assert torch.equal(y[True], y[False]) and torch.equal(y[None], y[False])
    K().check_error_flags()


@pytest.mark.parametrize("m,n,edges", [(4, 389, {True: 1, None: 0, False: 0}), (48, 2560, {True: 2, None: 1, False: 0})])
def test_a_products_launches_follow_the_switch(m, n, edges):
    w4, x, y = K().pack_weight4(torch.randn(n, 1280, device=DEV)), torch.randn(m, 1280, device=DEV).to(BF), {}
    for pdl, want in edges.items():
        y[pdl] = torch.empty(m, n, dtype=BF, device=DEV)
        K().linear4(x, w4, y[pdl], pdl=pdl)
        assert _captured(lambda: (x.mul_(1.0), K().linear4(x, w4, y[pdl], pdl=pdl)))[1] == want, pdl
    assert torch.equal(y[True], y[False]) and torch.equal(y[None], y[False])


@pytest.mark.parametrize("dtype,rows,lens,edges", [(BF, 2, 200, {True: 1, None: 0, False: 0}), (BF, 160, 2100, {True: 2, None: 1, False: 0}), (F32, 1, 700, {True: 1, None: 1, False: 0})])
def test_attentions_launches_follow_the_switch(dtype, rows, lens, edges):
    c, out = Cache([lens], 1, 64, 64, 64, dtype), {}
    c.fill()
    q, slot, pos = torch.randn(rows, 2, 64, device=DEV).to(dtype), i32([0] * rows), i32([lens - 1 - i for i in range(rows)])
    for pdl, want in edges.items():
        out[pdl] = torch.empty(rows, 128, dtype=dtype, device=DEV)
        call = lambda: K().attn4_rows(q, c.k, c.v, c.pt, slot, pos, out[pdl], 0.125, None, 64, lens, pdl=pdl)
        call()
        assert _captured(lambda: (q.mul_(1.0), call()))[1] == want, pdl
    assert torch.equal(out[True], out[False]) and torch.equal(out[None], out[False])
