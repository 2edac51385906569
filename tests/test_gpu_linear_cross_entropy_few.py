"""The cross entropy of a linear layer for a few tokens, where other kernels run: one pass over the weights (one token, float32 up to
four; the gradient of 16 bits up to sixteen), tiles of mma.sync (float32, up to 64 tokens). Same checks and tolerances as for many."""
import pytest
import torch

from tannic_b200 import ops as tb
from test_gpu_linear_cross_entropy import DTYPES, IGNORE, both, check_grad, check_loss, data

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 7, 8, 9])
@pytest.mark.parametrize("hidden,vocab", [(64, 1000), (1000, 33), (71, 5003), (4096, 777), (4100, 300), (3, 1), (8, 4), (513, 9)])
def test_sizes(tokens, hidden, vocab, dtype):
    both(*data(tokens, hidden, vocab, dtype, tokens + hidden))


@pytest.mark.parametrize("tokens", [15, 16, 17, 31, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("hidden,vocab", [(64, 1000), (72, 129), (71, 128), (33, 127), (1024, 5003), (4, 1), (500, 3)])
def test_float32_tiles(tokens, hidden, vocab):
    both(*data(tokens, hidden, vocab, torch.float32, tokens + hidden, ignored=0.2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 4, 8])
def test_wide_rows_and_large_vocabulary(tokens, dtype):
    both(*data(tokens, 6000, 500, dtype, 1))   # beyond the gradient's registers
    if dtype == torch.float32:
        both(*data(tokens, 14000, 200, dtype, 1))  # and, for four tokens, the loss's shared memory
    both(*data(tokens, 128, 50257, dtype, 2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pattern", [[True, False, False, False], [False, True, True], [True, True, True, True], [True], [False, True] * 9, [True] * 40])
def test_ignored_and_undefined_tokens(pattern, dtype):
    n = len(pattern)
    h, w, t, g = data(n, 200, 600, dtype, 3)
    out = torch.tensor(pattern, device="cuda")
    t[out] = IGNORE
    _, lse, want = both(h, w, t, g)
    h2, g2, lse2 = h.clone(), g.clone(), lse.clone()
    h2[out], g2[out], lse2[out] = float("nan"), float("inf"), float("nan")
    got = tb.linear_cross_entropy_grad(g2, h2, w, t, lse2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_target_outside_the_vocabulary(dtype):
    h, w, t, g = data(3, 200, 600, dtype, 4)
    clean, lse = tb.linear_cross_entropy(h, w, t)
    t[1] = 600
    loss, lse2 = tb.linear_cross_entropy(h, w, t)
    assert torch.equal(lse, lse2) and bool(torch.isnan(loss[1])) and torch.equal(loss[[0, 2]], clean[[0, 2]])
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    assert bool(torch.isnan(dh[1]).all()) and bool(torch.isfinite(dh[[0, 2]]).all()) and bool(torch.isnan(dw).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("view", ["pitch", "odd pitch", "offset", "transposed", "expanded rows"])
def test_views(view, dtype):
    make = {
        "pitch": lambda m: torch.nn.functional.pad(m, (0, 8))[..., : m.shape[-1]],
        "odd pitch": lambda m: torch.nn.functional.pad(m, (0, 3))[..., : m.shape[-1]],
        "offset": lambda m: torch.nn.functional.pad(m.reshape(-1), (1, 0))[1:].reshape(m.shape),
        "transposed": lambda m: m.transpose(-1, -2).contiguous().transpose(-1, -2),
        "expanded rows": lambda m: m[:1].expand(m.shape),
    }[view]
    for tokens in (3, 20):
        h, w, t, g = data(tokens, 264, 301, dtype, 5)
        both(make(h), w, t, g)
        both(h, make(w), t, g)
        both(h, w, t.int(), g[:1].expand(tokens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [4, 40])
def test_one_of_the_gradients_and_same_bits(tokens, dtype):
    h, w, t, g = data(tokens, 768, 3000, dtype, 6)
    loss, lse = tb.linear_cross_entropy(h, w, t)
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    assert torch.equal(tb.linear_cross_entropy_grad(g, h, w, t, lse, dweight=False)[0], dh)
    assert torch.equal(tb.linear_cross_entropy_grad(g, h, w, t, lse, dhidden=False)[1], dw)
    for _ in range(3):
        again = tb.linear_cross_entropy(h, w, t)
        assert torch.equal(again[0], loss) and torch.equal(again[1], lse)
        assert all(torch.equal(p, q) for p, q in zip(tb.linear_cross_entropy_grad(g, h, w, t, lse), (dh, dw)))


def test_logits_far_apart():
    h, w, t, g = data(4, 64, 600, torch.bfloat16, 7, scale=40.0)
    both(h, w, t, g)
    best = (h.float() @ w.float().T).argmax(-1)
    both(h, w, best, g)


@pytest.mark.parametrize("tokens,dtype", [(2, torch.bfloat16), (2, torch.float32), (30, torch.float32)])
def test_captured_and_replayed(tokens, dtype):
    h, w, t, g = data(tokens, 512, 2000, dtype, 8)
    loss, lse = tb.linear_cross_entropy(h, w, t)
    want = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = tb.linear_cross_entropy(h, w, t)
        grads = tb.linear_cross_entropy_grad(g, h, w, t, out[1])
    torch.cuda.synchronize()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], loss) and all(torch.equal(p, q) for p, q in zip(grads, want))
    check_loss(h, w, t, out)
    check_grad(g, h, w, t, out[1], grads)


@pytest.mark.parametrize("tokens,dtype", [(3, torch.bfloat16), (3, torch.float32), (20, torch.float32), (200, torch.float16)])
def test_rows_behind_the_results_are_left_alone(tokens, dtype):
    import ctypes as C
    from tannic_b200 import _abi as A
    h, w, t, g = data(tokens, 264, 301, dtype, 9)
    lse = tb.linear_cross_entropy(h, w, t)[1]
    big_h, big_w = (torch.full((m.shape[0] + 4, m.shape[1]), 7.0, dtype=m.dtype, device="cuda") for m in (h, w))
    rec = [tb.desc(x) for x in (g, h, w, t, lse, big_h[:tokens], big_w[:301])]
    A.check(A.lib().tn_linear_cross_entropy_grad(*[C.byref(r) for r in rec], tb.current_stream(h), IGNORE))
    check_grad(g, h, w, t, lse, (big_h[:tokens], big_w[:301]))
    assert bool((big_h[tokens:] == 7.0).all()) and bool((big_w[301:] == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hidden,vocab", [(8, 1), (40, 7), (264, 10007), (768, 9), (1696, 4801), (2048, 2000), (2056, 3001), (3456, 2500), (4096, 5003)])
@pytest.mark.parametrize("tokens", [1, 5, 8, 9])
def test_one_pass_of_sixteen_bits(tokens, hidden, vocab, dtype):
    both(*data(tokens, hidden, vocab, dtype, 10))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hidden,vocab", [(8, 3), (512, 10007), (520, 41), (1024, 7001), (1032, 999), (2048, 5003), (2056, 300)])
@pytest.mark.parametrize("tokens", [9, 12, 16, 17])
def test_one_pass_of_two_tiles(tokens, hidden, vocab, dtype):
    h, w, t, g = data(tokens, hidden, vocab, dtype, 12, ignored=0.2)
    both(h, w, t, g)
    lse = tb.linear_cross_entropy(h, w, t)[1]
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    assert torch.equal(tb.linear_cross_entropy_grad(g, h, w, t, lse, dweight=False)[0], dh)
    assert torch.equal(tb.linear_cross_entropy_grad(g, h, w, t, lse, dhidden=False)[1], dw)


def test_small_and_infinite_gradients():
    """float16's d would be lost unscaled; one infinite gradient leaves the other tokens' rows as they are."""
    h, w, t, g = data(6, 264, 3000, torch.float16, 11)
    both(h, w, t, g * 2.0**-20)
    lse = tb.linear_cross_entropy(h, w, t)[1]
    want = tb.linear_cross_entropy_grad(g, h, w, t, lse)[0]
    keep = [0, 1, 2, 4, 5]
    rest = g.clone()
    rest[3] = 0.0
    same = tb.linear_cross_entropy_grad(rest, h, w, t, lse)[0]
    g[3] = float("inf")
    got, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    assert torch.equal(got[keep], same[keep]) and not bool(torch.isfinite(got[3]).any()) and not bool(torch.isfinite(dw).any())
    assert bool(torch.isfinite(want).all())
