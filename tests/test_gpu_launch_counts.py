"""kernel_launches counts what a call enqueues: the kernel nodes of a graph that captures it."""
import ctypes as C

import pytest
import torch

import mgg_osdi23_b200 as mgg
from mgg_osdi23_b200 import api

pytestmark = pytest.mark.gpu


def kernels_of(call):
    """(kernel nodes of the captured call, what kernel_launches went up by)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        before = api.kernel_launches[0]
        call()
        counted = api.kernel_launches[0] - before
    cuda, raw, n = C.CDLL("libcuda.so.1"), C.c_void_p(graph.raw_cuda_graph()), C.c_size_t()
    assert cuda.cuGraphGetNodes(raw, None, C.byref(n)) == 0
    if n.value == 0:
        return 0, counted
    nodes = (C.c_void_p * n.value)()
    assert cuda.cuGraphGetNodes(raw, nodes, C.byref(n)) == 0
    found = 0
    for i in range(n.value):
        kind = C.c_int()
        assert cuda.cuGraphNodeGetType(C.c_void_p(nodes[i]), C.byref(kind)) == 0
        found += kind.value == 0                                    # CU_GRAPH_NODE_TYPE_KERNEL
    return found, counted


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(0, 8), (70, 100), (9, 8192), (9, 8200), (9, 8201), (9, 10_240), (9, 10_241), (9, 10_248), (3, 16_384)])
def test_layer_norm(n, d, t):
    x, dy = torch.randn(n, d, device="cuda").to(t), torch.randn(n, d, device="cuda").to(t)
    mean, rstd, dx, out = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda"), torch.empty_like(x), torch.empty_like(x)
    dw, db = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    found, counted = kernels_of(lambda: mgg.layer_norm_forward(out, x))
    assert found == counted
    for args, kw in (((dx,), {}), ((dx,), dict(dweight=dw, dbias=db)), ((None,), dict(dbias=db))):
        found, counted = kernels_of(lambda: mgg.layer_norm_backward(args[0], dy, x, mean, rstd, **kw))
        assert found == counted, (bool(kw), args[0] is None)
    # rows that start off a 16-byte boundary
    if n:
        odd = torch.empty(n * d + 1, device="cuda", dtype=t)[1:].view(n, d).copy_(x)
        for args, kw in (((dx,), dict(dweight=dw)), ((None,), dict(dweight=dw))):
            found, counted = kernels_of(lambda: mgg.layer_norm_backward(args[0], dy, odd, mean, rstd, **kw))
            assert found == counted


@pytest.mark.parametrize("n,c", [(0, 5), (100, 47), (20, 300), (9, 5000)])
def test_class_log_probabilities(n, c):
    z, labels = torch.randn(n, c, device="cuda"), torch.zeros(n, device="cuda", dtype=torch.int32)
    lp, stats, dz = torch.empty(n, device="cuda"), torch.zeros(n, 2, device="cuda"), torch.empty(n, c, device="cuda")
    for call in (lambda: mgg.class_logprob_forward(lp, z, labels, stats=stats), lambda: mgg.class_logprob_backward(dz, z, labels, stats, lp)):
        found, counted = kernels_of(call)
        assert found == counted


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k,m", [(0, 16, 24), (50, 16, 24), (100_000, 8, 8), (3000, 64, 4), (200, 256, 128), (100_000, 128, 128)])
def test_grouped_products(n, k, m, t):
    x, w, dy = torch.randn(n, k, device="cuda").to(t), torch.randn(2, k, m, device="cuda").to(t), torch.randn(n, m, device="cuda").to(t)
    ptr = torch.tensor([0, n // 3, n], device="cuda", dtype=torch.int32)
    out, dx, dw = torch.empty(n, m, device="cuda", dtype=t), torch.empty(n, k, device="cuda", dtype=t), torch.empty(2, k, m, device="cuda")
    for call in (lambda: mgg.grouped_dense_forward(out, x, w, ptr), lambda: mgg.grouped_dense_backward(dx, None, dy, x, w, ptr),
                 lambda: mgg.grouped_dense_backward(None, dw, dy, x, w, ptr), lambda: mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)):
        found, counted = kernels_of(call)
        assert found == counted


def test_a_refused_call_counts_nothing():
    x = torch.randn(4, 8, device="cuda")
    before = api.kernel_launches[0]
    with pytest.raises(mgg.MggbError):
        mgg.layer_norm_forward(torch.empty_like(x), x, eps=-1.0)
    with pytest.raises(mgg.MggbError):
        mgg.class_logprob_backward(torch.empty_like(x), x, None, torch.zeros(4, 2, device="cuda"), None)
    with pytest.raises(mgg.MggbError):
        mgg.grouped_dense_forward(x, x, torch.zeros(1, 8, 8, device="cuda"), torch.tensor([0, 4], device="cuda", dtype=torch.int32))
    assert api.kernel_launches[0] == before
