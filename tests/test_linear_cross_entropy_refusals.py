"""What tn_linear_cross_entropy and its gradient refuse, and with which status. Every check runs before a device is touched, so
records that name device 0 and an address that nothing reads are enough (no GPU needed)."""
import ctypes as C

import pytest

from tannic_b200 import _abi as A

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


DEFAULT = object()


def forward(h=DEFAULT, w=DEFAULT, t=DEFAULT, loss=DEFAULT, lse=DEFAULT):
    h = rec((4, 6, 64)) if h is DEFAULT else h
    w = rec((100, 64)) if w is DEFAULT else w
    t = rec((4, 6), A.INT64) if t is DEFAULT else t
    loss, lse = (rec((4, 6), A.FLOAT32) if x is DEFAULT else x for x in (loss, lse))
    return A.lib().tn_linear_cross_entropy(ref(h), ref(w), ref(t), ref(loss), ref(lse), A.StreamT(0), -100)


def backward(g=DEFAULT, h=DEFAULT, w=DEFAULT, t=DEFAULT, lse=DEFAULT, dh=DEFAULT, dw=DEFAULT):
    h = rec((4, 6, 64)) if h is DEFAULT else h
    w = rec((100, 64)) if w is DEFAULT else w
    t = rec((4, 6), A.INT64) if t is DEFAULT else t
    g, lse = (rec((4, 6), A.FLOAT32) if x is DEFAULT else x for x in (g, lse))
    dh = rec((4, 6, 64)) if dh is DEFAULT else dh
    dw = rec((100, 64)) if dw is DEFAULT else dw
    return A.lib().tn_linear_cross_entropy_grad(ref(g), ref(h), ref(w), ref(t), ref(lse), ref(dh), ref(dw), A.StreamT(0), -100)


COMMON = {
    "no hidden states": (dict(h=None), A.ERROR),
    "no weights": (dict(w=None), A.ERROR),
    "no targets": (dict(t=None), A.ERROR),
    "integer operands": (dict(h=rec((4, 6, 64), A.INT32), w=rec((100, 64), A.INT32)), A.UNSUPPORTED_DTYPE),
    "float64 operands": (dict(h=rec((4, 6, 64), A.FLOAT64), w=rec((100, 64), A.FLOAT64)), A.UNSUPPORTED_DTYPE),
    "two types": (dict(w=rec((100, 64), A.FLOAT16)), A.UNSUPPORTED_DTYPE),
    "float targets": (dict(t=rec((4, 6), A.FLOAT32)), A.UNSUPPORTED_DTYPE),
    "int16 targets": (dict(t=rec((4, 6), A.INT16)), A.UNSUPPORTED_DTYPE),
    "rank 0": (dict(h=rec(())), A.ERROR),
    "weights of rank 1": (dict(w=rec((64,))), A.ERROR),
    "weights of rank 3": (dict(w=rec((1, 100, 64))), A.ERROR),
    "hidden sizes": (dict(w=rec((100, 65))), A.ERROR),
    "empty hidden axis": (dict(h=rec((4, 6, 0)), w=rec((100, 0))), A.ERROR),
    "empty vocabulary": (dict(w=rec((0, 64))), A.ERROR),
    "targets' shape": (dict(t=rec((6, 4), A.INT64)), A.ERROR),
    "targets' rank": (dict(t=rec((24,), A.INT64)), A.ERROR),
    "host hidden states": (dict(h=rec((4, 6, 64), device=None)), A.INCOMPATIBLE_DEVICES),
    "host targets": (dict(t=rec((4, 6), A.INT64, device=None)), A.INCOMPATIBLE_DEVICES),
    "weights elsewhere": (dict(w=rec((100, 64), device=1)), A.INCOMPATIBLE_DEVICES),
    "vocabulary of 2^31": (dict(w=rec((1 << 31, 64))), A.ERROR),
    "lse's type": (dict(lse=rec((4, 6))), A.UNSUPPORTED_DTYPE),
    "lse's shape": (dict(lse=rec((24,), A.FLOAT32)), A.ERROR),
    "lse elsewhere": (dict(lse=rec((4, 6), A.FLOAT32, device=1)), A.INCOMPATIBLE_DEVICES),
}
FORWARD = {
    "no output": (dict(loss=None, lse=None), A.ERROR),
    "loss type": (dict(loss=rec((4, 6))), A.UNSUPPORTED_DTYPE),
    "loss shape": (dict(loss=rec((4,), A.FLOAT32)), A.ERROR),
    "strided loss": (dict(loss=rec((4, 6), A.FLOAT32, strides=(12, 2))), A.ERROR),
    "host loss": (dict(loss=rec((4, 6), A.FLOAT32, device=None)), A.INCOMPATIBLE_DEVICES),
}
BACKWARD = {
    "no grad": (dict(g=None), A.ERROR),
    "no lse": (dict(lse=None), A.ERROR),
    "no output": (dict(dh=None, dw=None), A.ERROR),
    "grad type": (dict(g=rec((4, 6))), A.UNSUPPORTED_DTYPE),
    "grad shape": (dict(g=rec((), A.FLOAT32)), A.ERROR),
    "dhidden type": (dict(dh=rec((4, 6, 64), A.FLOAT32)), A.UNSUPPORTED_DTYPE),
    "dhidden shape": (dict(dh=rec((24, 64))), A.ERROR),
    "strided dhidden": (dict(dh=rec((4, 6, 64), strides=(768, 128, 1))), A.ERROR),
    "dweight type": (dict(dw=rec((100, 64), A.FLOAT32)), A.UNSUPPORTED_DTYPE),
    "dweight shape": (dict(dw=rec((64, 100))), A.ERROR),
    "strided dweight": (dict(dw=rec((100, 64), strides=(1, 100))), A.ERROR),
    "dweight elsewhere": (dict(dw=rec((100, 64), device=1)), A.INCOMPATIBLE_DEVICES),
}


@pytest.mark.parametrize("name", [*COMMON, *FORWARD])
def test_forward_refuses(name):
    if name in COMMON:
        call, status = COMMON[name]
    else:
        call, status = FORWARD[name]
    assert forward(**call) == status
    assert b"linear_cross_entropy" in A.lib().tn_last_error()


@pytest.mark.parametrize("name", [*COMMON, *BACKWARD])
def test_backward_refuses(name):
    call, status = BACKWARD[name] if name in BACKWARD else COMMON[name]
    assert backward(**call) == status
    assert b"linear_cross_entropy_grad" in A.lib().tn_last_error()
