"""Normalisation into its own operand where rows share 16-byte chunks: the chunks that cover a row hold bytes of its neighbours, which
other threads are writing just then."""
import ctypes as C

import pytest
import torch

from tannic_b200 import _abi as A
from tannic_b200 import ops as tb
from test_gpu_layer_norm import check_backward, check_forward, data

pytestmark = pytest.mark.gpu

# a row per warp (every step of it), a row per block, the looping kernels; rows that start at every offset from a boundary
COLS = [1, 3, 33, 71, 100, 271, 301, 511, 601, 767, 1001, 1023, 1025, 2049, 4099, 8191, 8193, 16383, 16401]


def offset(t):
    """The same elements, starting one element behind a 16-byte boundary."""
    return torch.nn.functional.pad(t.reshape(-1), (1, 0))[1:].reshape(t.shape)


def gradient_into(dy, x, mean, rstd, w, dx):
    dw, db = torch.empty_like(w), torch.empty_like(w)
    rec = [tb.desc(t) for t in (dy, x, mean, rstd, w, dx, dw, db)]
    A.check(A.lib().tn_layer_norm_grad(*[C.byref(r) for r in rec], tb.current_stream(x)))
    return dx, dw, db


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("shift", [False, True])
def test_unaligned_rows_in_place(shift, cols, dtype):
    rows = min(20000, 2_000_000 // cols + 5)
    x, dy, w, b = data((rows, cols), dtype, cols)
    if shift:
        x, dy = offset(x), offset(dy)
    y, mean, rstd = tb.layer_norm(x, w, b, stats=True)
    check_forward(x, w, b, 1e-5, (y, mean, rstd))
    want = tb.layer_norm_grad(dy, x, mean, rstd, w)
    check_backward(dy, x, mean, rstd, w, want)
    into = offset(x) if shift else x.clone()
    assert tb.layer_norm(into, w, b, out=into) is into and torch.equal(into, y)
    for name in ("dy", "x"):
        args = {"dy": offset(dy) if shift else dy.clone(), "x": offset(x) if shift else x.clone()}
        dx, dw, db = gradient_into(args["dy"], args["x"], mean, rstd, w, args[name])
        assert torch.equal(dx, want[0]) and torch.equal(dw, want[1]) and torch.equal(db, want[2]), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [71, 271, 1001, 4099, 8193])
def test_what_lies_around_unaligned_rows_is_left_alone(cols, dtype):
    rows = 37
    x, dy, w, b = data((rows, cols), dtype, cols)
    y, mean, rstd = tb.layer_norm(x, w, b, stats=True)
    want = tb.layer_norm_grad(dy, x, mean, rstd, w)
    n = rows * cols
    for before in (1, 3, 5):
        out, grad = (torch.full((n + before + 9,), 7.0, device="cuda", dtype=dtype) for _ in range(2))
        tb.layer_norm(x, w, b, out=out[before:before + n].view(rows, cols))
        gradient_into(dy, x, mean, rstd, w, grad[before:before + n].view(rows, cols))
        assert torch.equal(out[before:before + n].view(rows, cols), y) and torch.equal(grad[before:before + n].view(rows, cols), want[0])
        for buf in (out, grad):
            assert bool((buf[:before] == 7.0).all()) and bool((buf[before + n:] == 7.0).all())
