"""What tn_layer_norm and tn_layer_norm_grad refuse, and with which status. Every check runs before a device is touched, so
records that name device 0 and an address that nothing reads are enough (no GPU needed)."""
import ctypes as C

import pytest
import torch

from tannic_b200 import _abi as A
from tannic_b200 import ops as tb

FAKE = 1 << 20


def rec(shape, dtype=A.BFLOAT16, device=0, strides=None):
    if strides is None:
        strides, run = [], 1
        for n in reversed(shape):
            strides.insert(0, run)
            run *= n
    return A.make_tensor(FAKE, tuple(shape), tuple(strides), dtype, device)


def ref(t):
    return None if t is None else C.byref(t)


def forward(x, w=None, b=None, y="like", mean=None, rstd=None, eps=1e-5):
    y = rec([x.shape.sizes[i] for i in range(x.rank)], x.dtype) if y == "like" else y
    return A.lib().tn_layer_norm(ref(x), ref(w), ref(b), ref(y), ref(mean), ref(rstd), A.StreamT(0), eps)


def backward(x, dy="like", mean="stat", rstd="stat", w=None, dx="like", dw=None, db=None):
    shape = [x.shape.sizes[i] for i in range(x.rank)]
    like = rec(shape, x.dtype)
    stat = rec(shape[:-1], A.FLOAT32)
    pick = lambda t: like if t == "like" else stat if t == "stat" else t  # noqa: E731
    return A.lib().tn_layer_norm_grad(ref(pick(dy)), ref(x), ref(pick(mean)), ref(pick(rstd)), ref(w), ref(pick(dx)), ref(dw), ref(db), A.StreamT(0))


X = lambda: rec((4, 64))  # noqa: E731

FORWARD = {
    "integer input": (lambda: forward(rec((4, 64), A.INT32)), A.UNSUPPORTED_DTYPE),
    "complex input": (lambda: forward(rec((4, 64), A.COMPLEX64)), A.UNSUPPORTED_DTYPE),
    "rank 0": (lambda: forward(rec(())), A.ERROR),
    "empty last axis": (lambda: forward(rec((4, 0))), A.ERROR),
    "host input": (lambda: forward(rec((4, 64), device=None)), A.INCOMPATIBLE_DEVICES),
    "host result": (lambda: forward(X(), y=rec((4, 64), device=None)), A.INCOMPATIBLE_DEVICES),
    "result elsewhere": (lambda: forward(X(), y=rec((4, 64), device=1)), A.INCOMPATIBLE_DEVICES),
    "no result": (lambda: forward(X(), y=None), A.ERROR),
    "result dtype": (lambda: forward(X(), y=rec((4, 64), A.FLOAT16)), A.UNSUPPORTED_DTYPE),
    "result shape": (lambda: forward(X(), y=rec((64, 4))), A.ERROR),
    "result rank": (lambda: forward(X(), y=rec((256,))), A.ERROR),
    "strided result": (lambda: forward(X(), y=rec((4, 64), strides=(128, 1))), A.ERROR),
    "weight length": (lambda: forward(X(), rec((63,))), A.ERROR),
    "weight rank": (lambda: forward(X(), rec((1, 64))), A.ERROR),
    "weight dtype": (lambda: forward(X(), rec((64,), A.FLOAT16)), A.UNSUPPORTED_DTYPE),
    "float32 rows with 16-bit weight": (lambda: forward(rec((4, 64), A.FLOAT32), rec((64,))), A.UNSUPPORTED_DTYPE),
    "strided weight": (lambda: forward(X(), rec((64,), strides=(2,))), A.ERROR),
    "broadcast weight": (lambda: forward(X(), rec((64,), strides=(0,))), A.ERROR),
    "host weight": (lambda: forward(X(), rec((64,), device=None)), A.INCOMPATIBLE_DEVICES),
    "weight and bias dtypes": (lambda: forward(X(), rec((64,)), rec((64,), A.FLOAT32)), A.UNSUPPORTED_DTYPE),
    "bias length": (lambda: forward(X(), None, rec((65,))), A.ERROR),
    "mean dtype": (lambda: forward(X(), mean=rec((4,))), A.UNSUPPORTED_DTYPE),
    "float64 mean dtype": (lambda: forward(rec((4, 64), A.FLOAT64), mean=rec((4,), A.FLOAT32)), A.UNSUPPORTED_DTYPE),
    "mean length": (lambda: forward(X(), mean=rec((5,), A.FLOAT32)), A.ERROR),
    "strided rstd": (lambda: forward(X(), rstd=rec((4,), A.FLOAT32, strides=(2,))), A.ERROR),
    "negative eps": (lambda: forward(X(), eps=-1e-6), A.ERROR),
    "eps not a number": (lambda: forward(X(), eps=float("nan")), A.ERROR),
}
BACKWARD = {
    "integer input": (lambda: backward(rec((4, 64), A.INT64)), A.UNSUPPORTED_DTYPE),
    "empty last axis": (lambda: backward(rec((4, 0)), mean=rec((4,), A.FLOAT32), rstd=rec((4,), A.FLOAT32)), A.ERROR),
    "no dy": (lambda: backward(X(), dy=None), A.ERROR),
    "dy dtype": (lambda: backward(X(), dy=rec((4, 64), A.FLOAT32)), A.UNSUPPORTED_DTYPE),
    "dy shape": (lambda: backward(X(), dy=rec((4, 65))), A.ERROR),
    "dy elsewhere": (lambda: backward(X(), dy=rec((4, 64), device=1)), A.INCOMPATIBLE_DEVICES),
    "no dx": (lambda: backward(X(), dx=None), A.ERROR),
    "strided dx": (lambda: backward(X(), dx=rec((4, 64), strides=(65, 1))), A.ERROR),
    "no mean": (lambda: backward(X(), mean=None), A.ERROR),
    "no rstd": (lambda: backward(X(), rstd=None), A.ERROR),
    "rstd length": (lambda: backward(X(), rstd=rec((3,), A.FLOAT32)), A.ERROR),
    "weight length": (lambda: backward(X(), w=rec((3,))), A.ERROR),
    "dweight dtype": (lambda: backward(X(), w=rec((64,)), dw=rec((64,), A.FLOAT32)), A.UNSUPPORTED_DTYPE),
    "dbias dtype": (lambda: backward(X(), w=rec((64,), A.FLOAT32), db=rec((64,))), A.UNSUPPORTED_DTYPE),
    "dweight length": (lambda: backward(X(), w=rec((64,)), dw=rec((32,))), A.ERROR),
    "strided dbias": (lambda: backward(X(), w=rec((64,)), db=rec((64,), strides=(4,))), A.ERROR),
    "host dx": (lambda: backward(X(), dx=rec((4, 64), device=None)), A.INCOMPATIBLE_DEVICES),
}


@pytest.mark.parametrize("name", FORWARD)
def test_forward_refuses(name):
    call, status = FORWARD[name]
    assert call() == status
    assert b"layer_norm" in A.lib().tn_last_error()


@pytest.mark.parametrize("name", BACKWARD)
def test_backward_refuses(name):
    call, status = BACKWARD[name]
    assert call() == status
    assert b"layer_norm_grad" in A.lib().tn_last_error()


def test_null_input():
    assert A.lib().tn_layer_norm(None, None, None, None, None, None, A.StreamT(0), 1e-5) == A.ERROR
    assert A.lib().tn_layer_norm_grad(None, None, None, None, None, None, None, None, A.StreamT(0)) == A.ERROR


def test_python_rank_0():
    with pytest.raises(ValueError):
        tb.layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError):
        tb.layer_norm_grad(torch.tensor(1.0), torch.tensor(1.0), torch.tensor(1.0), torch.tensor(1.0))
