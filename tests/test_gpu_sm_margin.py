"""The loss and its gradient while another thread changes the number of SMs that persistent kernels leave free (tn_set_sm_margin)."""
import threading

import pytest
import torch

from tannic_b200 import _abi as A
from tannic_b200 import ops as tb

pytestmark = pytest.mark.gpu


def data(tokens, hidden, vocab, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(vocab, hidden, generator=gen, device="cuda") / hidden ** 0.5).to(dtype)
    t = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    return h, w, t, torch.rand(tokens, generator=gen, device="cuda")


@pytest.mark.parametrize("tokens,hidden,dtype", [(300, 128, torch.bfloat16), (4, 2048, torch.float16), (1, 4096, torch.bfloat16), (3, 1024, torch.float32)])
def test_margin_changed_by_another_thread(tokens, hidden, dtype):
    """A call keeps to the margin that it found: its result is one of the two that the two margins give."""
    h, w, t, g = data(tokens, hidden, 30000, dtype, 2)
    margins = (0, 60)
    want = []
    try:
        for m in margins:
            tb.sm_margin(m)
            loss, lse = tb.linear_cross_entropy(h, w, t)
            want.append((loss, lse, lse))
        lse = want[0][1]
        for i, m in enumerate(margins):
            tb.sm_margin(m)
            want[i] = want[i][:2] + (tb.linear_cross_entropy_grad(g, h, w, t, lse),)
        stop = threading.Event()

        def toggle():
            lib = A.lib()
            while not stop.is_set():
                for m in margins:
                    lib.tn_set_sm_margin(m)

        thread = threading.Thread(target=toggle)
        thread.start()
        try:
            for _ in range(100):
                got = [(tb.linear_cross_entropy(h, w, t), tb.linear_cross_entropy_grad(g, h, w, t, lse)) for _ in range(10)]
                for (loss, z), (dh, dw) in got:
                    assert any(torch.equal(loss, o[0]) and torch.equal(z, o[1]) for o in want)
                    assert any(torch.equal(dh, o[2][0]) for o in want), float((dh.float() - want[0][2][0].float()).abs().max())
                    assert torch.equal(dw, want[0][2][1])
        finally:
            stop.set()
            thread.join()
    finally:
        tb.sm_margin(0)
