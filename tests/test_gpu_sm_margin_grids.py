"""The number of SMs that persistent kernels leave free (tn_set_sm_margin), as the loss and its gradient keep it."""
import ctypes as C

import pytest
import torch

from tannic_b200 import ops as tb
from test_gpu_sm_margin import data

pytestmark = pytest.mark.gpu


class KernelNode(C.Structure):  # CUDA_KERNEL_NODE_PARAMS
    _fields_ = [("func", C.c_void_p), ("grid", C.c_uint * 3), ("block", C.c_uint * 3), ("shared", C.c_uint), ("params", C.c_void_p),
                ("extra", C.c_void_p), ("kern", C.c_void_p), ("ctx", C.c_void_p)]


def captured_launches(call):
    """(kernel name, blocks, threads of a block) of every launch that `call` makes."""
    cuda = C.CDLL("libcuda.so.1")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        keep = call()
    raw = C.c_void_p(graph.raw_cuda_graph())
    count = C.c_size_t(0)
    assert cuda.cuGraphGetNodes(raw, None, C.byref(count)) == 0
    nodes = (C.c_void_p * count.value)()
    assert cuda.cuGraphGetNodes(raw, nodes, C.byref(count)) == 0
    found = []
    for node in nodes:
        kind = C.c_int(-1)
        assert cuda.cuGraphNodeGetType(C.c_void_p(node), C.byref(kind)) == 0
        if kind.value != 0:
            continue
        p = KernelNode()
        assert cuda.cuGraphKernelNodeGetParams_v2(C.c_void_p(node), C.byref(p)) == 0
        name = C.c_char_p()
        if p.func:
            assert cuda.cuFuncGetName(C.byref(name), C.c_void_p(p.func)) == 0
        else:
            assert cuda.cuKernelGetName(C.byref(name), C.c_void_p(p.kern)) == 0
        found.append((name.value.decode(), p.grid[0] * p.grid[1] * p.grid[2], p.block[0] * p.block[1] * p.block[2]))
    del keep
    return found


# (tokens, hidden, type), the persistent kernel of the loss and that of its gradient, None where theirs are not persistent
CASES = {
    "one token of 16 bits": (1, 4096, torch.bfloat16, "few_loss_kernel", "half_grad_kernel"),
    "eight tokens of 16 bits": (8, 2048, torch.float16, "loss_gemm", "half_grad_kernel"),
    "sixteen tokens of 16 bits": (16, 2048, torch.bfloat16, "loss_gemm", "half_grad_kernel"),
    "many tokens of 16 bits": (300, 256, torch.bfloat16, "loss_gemm", "loss_gemm"),
    "four tokens of float32": (4, 4096, torch.float32, "few_loss_kernel", "few_grad_kernel"),
    "twenty tokens of float32": (20, 256, torch.float32, None, None),
    "many tokens of float32": (100, 256, torch.float32, "loss_gemm", "loss_gemm"),
}


@pytest.mark.parametrize("name", CASES)
def test_persistent_kernels_leave_the_margin(name):
    tokens, hidden, dtype, forward, backward = CASES[name]
    h, w, t, g = data(tokens, hidden, 40000, dtype)
    lse = tb.linear_cross_entropy(h, w, t)[1]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    calls = {forward: lambda: tb.linear_cross_entropy(h, w, t), backward: lambda: tb.linear_cross_entropy_grad(g, h, w, t, lse)}
    for kernel, call in calls.items():
        if kernel is None:
            continue
        call()
        full = [(b, n) for k, b, n in captured_launches(call) if kernel in k]
        tb.sm_margin(40)
        try:
            less = [(b, n) for k, b, n in captured_launches(call) if kernel in k]
        finally:
            tb.sm_margin(0)
        assert full and len(full) == len(less)
        # none of these has more than 512 threads on an SM, in one block or two
        assert max(b * n for b, n in full) > (sms - 40) * 256
        assert all(b * n <= (sms - 40) * 512 for b, n in less), less


@pytest.mark.parametrize("name", CASES)
def test_results_under_a_margin(name):
    tokens, hidden, dtype, _, _ = CASES[name]
    h, w, t, g = data(tokens, hidden, 3001, dtype, 1)
    loss, lse = tb.linear_cross_entropy(h, w, t)
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    for margin in (1, 40, 64):
        tb.sm_margin(margin)
        try:
            again = tb.linear_cross_entropy(h, w, t)
            grads = tb.linear_cross_entropy_grad(g, h, w, t, lse)
        finally:
            tb.sm_margin(0)
        # sums over the vocabulary are cut elsewhere: a few units of 2^-24 of the largest term, and the result's own rounding
        step = torch.finfo(dtype).eps
        assert bool(((again[0] - loss).abs() <= 2.0 ** -20 * lse.abs()).all()) and bool(((again[1] - lse).abs() <= 2.0 ** -20 * lse.abs()).all())
        assert torch.equal(grads[1], dw)
        scale = (g.abs()[:, None] * w.float().abs().amax()).expand(dh.shape)
        assert bool(((grads[0].float() - dh.float()).abs() <= step * dh.float().abs() + 2.0 ** -18 * scale).all())
    assert tb.device_errors() == 0
