"""The cross entropy of a linear layer and its gradient (tn_linear_cross_entropy, tn_linear_cross_entropy_grad) against the
formulas in 64 bits.

Where the tolerances come from. A tensor-core step adds 16 exact products to a float32 accumulator; whatever its order, that is at most
17 roundings (or truncations) of 2^-23 relative to the sum of the magnitudes, so a product over K is off by at most
1.1 K 2^-23 sum |a b| (float32 operands take six passes: 6.6 K; their split leaves 3 2^-24 more per factor pair). The log-sum-exp moves by no
more than the largest error of a logit; its exponentials, sums and logarithm add a few dozen roundings. d is rounded to the
operands' type (torch.finfo(t).eps / 2 relative; float32: 24 bits in three parts), the results once more.
"""
import pytest
import torch

from tannic_b200 import _abi as A
from tannic_b200 import ops as tb

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
DTYPES = HALVES + [torch.float32]
IGNORE = -100
U = 2.0 ** -24


def steps(k, dtype):
    return (6.6 if dtype == torch.float32 else 1.1) * (k + 16) * 2 * U + (6 * U if dtype == torch.float32 else 0.0)


def data(tokens, hidden, vocab, dtype, seed, ignored=0.0, scale=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lead = (tokens,) if isinstance(tokens, int) else tuple(tokens)
    h = torch.randn(*lead, hidden, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(vocab, hidden, generator=gen, device="cuda") * (scale if scale is not None else 1.5 / hidden ** 0.5)).to(dtype)
    t = torch.randint(0, vocab, lead, generator=gen, device="cuda")
    t = torch.where(torch.rand(lead, generator=gen, device="cuda") < ignored, torch.full_like(t, IGNORE), t)
    g = torch.rand(lead, generator=gen, device="cuda") * 2 - 0.5
    return h, w, t, g


def check_loss(h, w, t, got, ignore=IGNORE):
    loss, lse = got
    H, W = h.double().reshape(-1, h.shape[-1]), w.double()
    T = t.reshape(-1).long()
    logits = H @ W.T
    el = steps(h.shape[-1], h.dtype) * (H.abs() @ W.abs().T)
    want = torch.logsumexp(logits, -1)
    tol_lse = el.amax(-1) + 100 * U + 2 * U * want.abs()
    assert loss.shape == t.shape and lse.shape == t.shape and loss.dtype == lse.dtype == torch.float32
    err = (lse.double().reshape(-1) - want).abs()
    assert bool((err <= tol_lse).all()), float((err / tol_lse).max())
    keep = T != ignore
    at = torch.where(keep, T, torch.zeros_like(T))
    lt, elt = logits.gather(1, at[:, None])[:, 0], el.gather(1, at[:, None])[:, 0]
    want = torch.where(keep, want - lt, torch.zeros_like(want))
    tol = torch.where(keep, tol_lse + elt + 2 * U * (want.abs() + lt.abs()), torch.zeros_like(want))
    err = (loss.double().reshape(-1) - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def check_grad(g, h, w, t, lse, got, ignore=IGNORE):
    dh, dw = got
    k = h.shape[-1]
    H, W, T = h.double().reshape(-1, k), w.double(), t.reshape(-1).long()
    n, v = H.shape[0], W.shape[0]
    keep = T != ignore
    G = torch.where(keep, g.reshape(-1).double(), torch.zeros(n, dtype=torch.float64, device=H.device))
    Hk = torch.where(keep[:, None], H, torch.zeros_like(H))
    x = Hk @ W.T - torch.where(keep, lse.reshape(-1).double(), torch.zeros_like(G))[:, None]
    p = torch.where(keep[:, None], x.exp(), torch.zeros_like(x))
    el = steps(k, h.dtype) * (Hk.abs() @ W.abs().T)
    # p from its logit: the logit's error, the subtraction, the exponential and the product with grad
    ed = p * (el + 2 * U * x.abs() + 12 * U) * 1.01 * G.abs()[:, None]
    # The power of two is taken with subnormal results flushed: a probability below 2^-126, the smallest normal number, may be zero. That
    # is at most 2^-126 |grad| for an entry of d, and 2^-126 sum |grad| |h| for one of dweight, of which the tolerance knew nothing.
    ed += 2.0 ** -126 * G.abs()[:, None]
    at = torch.where(keep, T, torch.zeros_like(T))
    d = p.clone()
    d.scatter_add_(1, at[:, None], -keep.double()[:, None])
    d *= G[:, None]
    half = 2 * U if h.dtype == torch.float32 else torch.finfo(h.dtype).eps / 2
    ed += half * d.abs() * 1.01 + 4 * U * d.abs()
    if h.dtype == torch.float16:  # below float16's normal numbers, at a scale that brings the largest grad to 2^13 or more
        ed += 2.0 ** -25 * 2.0 ** -13 * G.abs().max()
    if dh is not None:
        want = d @ W
        tol = ed @ W.abs() + steps(v, h.dtype) * (d.abs() @ W.abs()) + (torch.finfo(h.dtype).eps / 2 + 2 * U) * want.abs() * 1.01
        tol += 2.0 ** -25 if h.dtype == torch.float16 else 1e-40
        err = (dh.double().reshape(-1, k) - want).abs()
        assert bool((err <= tol).all()), ("dhidden", float((err / tol).max()))
        assert dh.shape == h.shape and dh.dtype == h.dtype
        assert not bool(dh.reshape(-1, k)[~keep].any())
    if dw is not None:
        want = d.T @ Hk
        tol = ed.T @ Hk.abs() + steps(n, h.dtype) * (d.abs().T @ Hk.abs()) + (torch.finfo(h.dtype).eps / 2 + 2 * U) * want.abs() * 1.01
        tol += 2.0 ** -25 if h.dtype == torch.float16 else 1e-40
        err = (dw.double() - want).abs()
        assert bool((err <= tol).all()), ("dweight", float((err / tol).max()))
        assert dw.shape == w.shape and dw.dtype == w.dtype


def both(h, w, t, g, **kw):
    loss, lse = tb.linear_cross_entropy(h, w, t, **kw)
    check_loss(h, w, t, (loss, lse), kw.get("ignore_index", IGNORE))
    got = tb.linear_cross_entropy_grad(g, h, w, t, lse, **kw)
    check_grad(g, h, w, t, lse, got, kw.get("ignore_index", IGNORE))
    assert tb.device_errors() == 0
    return loss, lse, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 2, 31, 127, 128, 129, 300])
def test_token_counts(tokens, dtype):
    both(*data(tokens, 64, 700, dtype, tokens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 63, 64, 65, 255, 256, 257, 288, 511, 513, 5001])
def test_vocabulary_sizes(vocab, dtype):
    both(*data(70, 72, vocab, dtype, vocab))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hidden", [1, 3, 7, 8, 9, 31, 63, 64, 65, 127, 128, 197, 256, 264, 513, 768])
def test_hidden_sizes(hidden, dtype):
    both(*data(70, hidden, 300, dtype, hidden))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(4, 1024, 8000), (1, 2000, 4099), (1000, 16, 33), (513, 520, 1025), (2500, 128, 2500)])
def test_larger(shape, dtype):
    both(*data(*shape, dtype, 5, ignored=0.2))


@pytest.mark.parametrize("dtype", DTYPES)
def test_several_pieces_of_the_vocabulary(dtype):
    # a piece of d is at most half a GiB, but at least 4096 entries: these take two
    both(*data(65536 if dtype != torch.float32 else 20000, 40, 5003, dtype, 6, ignored=0.1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ignored", [0.0, 0.3, 0.99, 1.0])
def test_ignored_tokens(ignored, dtype):
    h, w, t, g = data(200, 64, 500, dtype, 7, ignored=ignored)
    loss, lse, (dh, dw) = both(h, w, t, g)
    assert not bool(loss[t == IGNORE].any())
    if ignored == 1.0:
        assert not bool(dh.any()) and not bool(dw.any())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("hidden", [64, 61])
def test_no_target_at_all_writes_zeros_everywhere(hidden, dtype):
    h, w, t, g = data(200, hidden, 500, dtype, 7, ignored=1.0)
    _, lse = tb.linear_cross_entropy(h, w, t)
    poison = torch.full((500 * hidden + 64,), 3.0, dtype=dtype, device="cuda")  # the pool hands this memory out again
    del poison
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    assert not bool(dh.any()) and not bool(dw.any())


def test_ignored_index_inside_the_vocabulary():
    h, w, t, g = data(100, 64, 50, torch.bfloat16, 8)
    t[::3] = 7
    both(h, w, t, g, ignore_index=7)


@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_may_hold_anything(dtype):
    h, w, t, g = data(150, 64, 500, dtype, 9, ignored=0.4)
    _, lse, want = both(h, w, t, g)
    out = t == IGNORE
    h2, g2, lse2 = h.clone(), g.clone(), lse.clone()
    h2[out], g2[out], lse2[out] = float("nan"), float("inf"), float("nan")
    loss2, _ = tb.linear_cross_entropy(h2, w, t)
    assert not bool(loss2[out].any()) and bool(torch.isfinite(loss2).all())
    got = tb.linear_cross_entropy_grad(g2, h2, w, t, lse2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [-1, 500, 2 ** 31 - 1, 2 ** 40, -(2 ** 40)])
def test_target_outside_the_vocabulary(bad, dtype):
    h, w, t, g = data(150, 64, 500, dtype, 10)
    clean, lse = tb.linear_cross_entropy(h, w, t)
    t[77] = bad
    loss, lse2 = tb.linear_cross_entropy(h, w, t)
    assert torch.equal(lse, lse2) and bool(torch.isnan(loss[77]))
    others = torch.arange(150, device="cuda") != 77
    assert torch.equal(loss[others], clean[others])
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    assert bool(torch.isnan(dh[77]).all()) and bool(torch.isfinite(dh[others]).all()) and bool(torch.isnan(dw).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_and_undefined_rows(dtype):
    h, w, t, g = data(150, 64, 500, dtype, 11)
    clean, lse = tb.linear_cross_entropy(h, w, t)
    h[3], h[140, 5] = float("nan"), float("inf")
    loss, lse2 = tb.linear_cross_entropy(h, w, t)
    bad = torch.zeros(150, dtype=torch.bool, device="cuda")
    bad[3] = bad[140] = True
    assert bool(torch.isnan(loss[bad]).all()) and torch.equal(loss[~bad], clean[~bad]) and torch.equal(lse2[~bad], lse[~bad])


def test_logits_far_apart():
    # logits of several thousand: nothing overflows, a certain token has loss 0 and a vanishing gradient
    h, w, t, g = data(140, 64, 600, torch.bfloat16, 12, scale=40.0)
    loss, lse, _ = both(h, w, t, g)
    best = (h.float() @ w.float().T).argmax(-1)
    loss, lse, (dh, dw) = both(h, w, best, g)
    assert float(loss.median()) < 1e-2


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 1e4])
def test_upstream_gradients_of_any_size(size, dtype):
    h, w, t, g = data(130, 64, 700, dtype, 13)
    both(h, w, t, g * size) if size <= 1.0 or dtype == torch.bfloat16 else both(h, w, t, g * 100.0)


def test_upstream_gradient_zero_and_expanded():
    h, w, t, g = data(130, 64, 700, torch.float16, 14, ignored=0.2)
    _, lse = tb.linear_cross_entropy(h, w, t)
    dh, dw = tb.linear_cross_entropy_grad(torch.zeros_like(g), h, w, t, lse)
    assert not bool(dh.any()) and not bool(dw.any())
    one = torch.tensor(0.125, device="cuda")
    got = tb.linear_cross_entropy_grad(one.expand(130), h, w, t, lse)
    want = tb.linear_cross_entropy_grad(torch.full((130,), 0.125, device="cuda"), h, w, t, lse)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("view", ["pitch", "odd pitch", "offset", "transposed", "step", "expanded rows"])
def test_views(view, dtype):
    make = {
        "pitch": lambda m: torch.nn.functional.pad(m, (0, 8))[..., : m.shape[-1]],
        "odd pitch": lambda m: torch.nn.functional.pad(m, (0, 3))[..., : m.shape[-1]],
        "offset": lambda m: torch.nn.functional.pad(m.reshape(-1), (1, 0))[1:].reshape(m.shape),
        "transposed": lambda m: m.transpose(-1, -2).contiguous().transpose(-1, -2),
        "step": lambda m: m.repeat_interleave(2, -1)[..., ::2],
        "expanded rows": lambda m: m[:1].expand(m.shape),
    }[view]
    h, w, t, g = data(133, 72, 301, dtype, 15, ignored=0.1)
    both(make(h), w, t, g)
    both(h, make(w), t, g)
    both(make(h), make(w), t.int(), g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shifted_sequences(dtype):
    # the usual call: position i predicts token i + 1, everything a slice of [batch, length]
    h, w, t, g = data((3, 50), 64, 300, dtype, 16, ignored=0.1)
    both(h[:, :-1], w, t[:, 1:], g[:, 1:])
    both(h.permute(1, 0, 2), w, t.T, g.T)


def test_rank_one_hidden():
    h, w, t, g = data((), 64, 300, torch.bfloat16, 17)
    loss, lse, (dh, dw) = both(h, w, t, g)
    assert loss.shape == () and dh.shape == (64,)


def test_no_tokens():
    h, w, t, g = data(0, 64, 300, torch.bfloat16, 18)
    loss, lse = tb.linear_cross_entropy(h, w, t)
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    assert loss.numel() == 0 and dh.shape == (0, 64) and not bool(dw.any())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_one_of_the_gradients(dtype):
    h, w, t, g = data(200, 64, 500, dtype, 19, ignored=0.2)
    _, lse = tb.linear_cross_entropy(h, w, t)
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    only_h = tb.linear_cross_entropy_grad(g, h, w, t, lse, dweight=False)
    only_w = tb.linear_cross_entropy_grad(g, h, w, t, lse, dhidden=False)
    assert only_h[1] is None and only_w[0] is None
    assert torch.equal(only_h[0], dh) and torch.equal(only_w[1], dw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_on_every_run(dtype):
    h, w, t, g = data(700, 256, 3000, dtype, 20, ignored=0.2)
    first = tb.linear_cross_entropy(h, w, t)
    grads = tb.linear_cross_entropy_grad(g, h, w, t, first[1])
    for _ in range(4):
        again = tb.linear_cross_entropy(h, w, t)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        assert all(torch.equal(p, q) for p, q in zip(grads, tb.linear_cross_entropy_grad(g, h, w, t, again[1])))


def test_gradient_against_differences():
    # float32, with steps of a power of two so that the moved operands are exact
    h, w, t, g = data(6, 16, 40, torch.float32, 21)
    h, w = (torch.round(x * 64) / 64 for x in (h, w))
    _, lse = tb.linear_cross_entropy(h, w, t)
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    value = lambda h, w: float((tb.linear_cross_entropy(h, w, t)[0].double() * g.double()).sum())  # noqa: E731
    step = 2.0 ** -6
    for index, grad in ((0, dh), (1, dw)):
        for at in range(0, grad.numel(), 11):
            up, down = [h.clone(), w.clone()], [h.clone(), w.clone()]
            up[index].view(-1)[at] += step
            down[index].view(-1)[at] -= step
            slope = (value(*up) - value(*down)) / (2 * step)
            # third derivative of a token's loss along one operand: at most 2 |other operand|^3 summed over the six tokens,
            # times step^2 / 6; rounding of the six losses (1e-6 each) over the step
            reach = float((w if index == 0 else h).abs().max())
            tol = 6 * 1.5 * 2 * reach ** 3 * step ** 2 / 6 + 6 * 1.5 * 1e-6 / step
            assert abs(slope - float(grad.reshape(-1)[at])) < tol, (index, at, slope, float(grad.reshape(-1)[at]), tol)


def test_captured_twice_and_replayed():
    h, w, t, g = data(300, 128, 1000, torch.bfloat16, 22, ignored=0.2)
    loss, lse = tb.linear_cross_entropy(h, w, t)
    want = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = tb.linear_cross_entropy(h, w, t)
                grads = tb.linear_cross_entropy_grad(g, h, w, t, out[1])
            graphs.append((graph, out, grads))
    torch.cuda.synchronize()
    for graph, _, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, out, grads in graphs:
        assert torch.equal(out[0], loss) and all(torch.equal(p, q) for p, q in zip(grads, want))
    # other data and other ignored tokens in the same memory
    h2, _, t2, g2 = data(300, 128, 1000, torch.bfloat16, 23, ignored=0.6)
    for to, new in ((h, h2), (t, t2), (g, g2)):
        to.copy_(new)
    loss, lse = tb.linear_cross_entropy(h, w, t)
    want = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    torch.cuda.synchronize()
    graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[1][1][0], loss) and all(torch.equal(p, q) for p, q in zip(graphs[1][2], want))


def test_two_calls_at_once_on_two_streams():
    sets = [data(400, 128, 3000, torch.bfloat16, s, ignored=0.3) for s in (24, 25)]
    want = []
    for h, w, t, g in sets:
        lse = tb.linear_cross_entropy(h, w, t)[1]
        want.append(tb.linear_cross_entropy_grad(g, h, w, t, lse) + (lse,))
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, (h, w, t, g) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                lse = tb.linear_cross_entropy(h, w, t)[1]
                got[i] = tb.linear_cross_entropy_grad(g, h, w, t, lse) + (lse,)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_fewer_sms():
    h, w, t, g = data(300, 128, 3000, torch.bfloat16, 26, ignored=0.1)
    loss, lse = tb.linear_cross_entropy(h, w, t)
    tb.sm_margin(40)
    try:
        again = tb.linear_cross_entropy(h, w, t)
        both(h, w, t, g)
    finally:
        tb.sm_margin(0)
    assert torch.equal(loss, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_then_loss_and_back(dtype):
    """The end of a network as it is trained: norm, linear layer, mean loss over the tokens that count, and the gradients of
    everything, against the same chain in 64 bits."""
    x, w, t, _ = data((4, 60), 128, 1000, dtype, 27, ignored=0.25)
    gen = torch.Generator(device="cuda").manual_seed(28)
    gamma = (1 + 0.1 * torch.randn(128, generator=gen, device="cuda")).to(dtype)
    beta = (0.1 * torch.randn(128, generator=gen, device="cuda")).to(dtype)
    y, mean, rstd = tb.layer_norm(x, gamma, beta, stats=True)
    loss, lse = tb.linear_cross_entropy(y, w, t)
    up = (1.0 / (t != IGNORE).sum()).float().expand(t.shape)
    dy, dw = tb.linear_cross_entropy_grad(up, y, w, t, lse)
    dx, dgamma, dbeta = tb.layer_norm_grad(dy, x, mean, rstd, gamma)

    leaves = [v.double().requires_grad_() for v in (x, gamma, beta, w)]
    X, Ga, Be, W = leaves
    c = X - X.mean(-1, keepdim=True)
    Y = c * (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * Ga + Be
    lp = torch.log_softmax(Y @ W.T, -1)
    keep = t != IGNORE
    total = -(lp.gather(-1, t.clamp(min=0)[..., None])[..., 0] * keep).sum() / keep.sum()
    total.backward()
    # every tensor between two kernels is rounded once, every result once: a handful of half steps of the
    # largest entry of each gradient (errors of an element follow the row's scale, not its own)
    half = 2.0 ** -18 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    assert abs(float((loss.double() * keep).sum() / keep.sum()) - float(total)) < 4 * half * float(Y.abs().max())
    for name, got, want in zip(("x", "gamma", "beta", "weight"), (dx, dgamma, dbeta, dw), (v.grad for v in leaves)):
        err = float((got.double() - want).abs().max() / want.abs().max())
        assert err < 8 * half, (name, err)
