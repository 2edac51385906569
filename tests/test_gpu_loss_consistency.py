"""What the gradient of a linear layer's cross entropy makes of the forward pass's log-sum-exp, where small differences count: nearly
certain tokens, small probabilities, and sums over very many tokens."""
import pytest
import torch

from tannic_b200 import ops as tb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 2, 4, 8, 9, 16, 17, 40, 64, 100, 128, 129, 300])
@pytest.mark.parametrize("hidden", [1024, 2048, 4096])
def test_nearly_certain_tokens(hidden, tokens, dtype):
    """Logits of 20 made of products of one sign, where a sum that is cut off drifts most, and about 1e-3 left for the other entries:
    d = p - 1 of the target is the difference of two numbers near 20. The forward pass's lse has to belong to the logits that the
    gradient forms."""
    vocab = 512
    gen = torch.Generator(device="cuda").manual_seed(tokens + hidden)
    u = torch.randn(hidden, generator=gen, device="cuda").abs()
    u /= u.sum() * (2 / torch.pi) ** 0.5
    h = torch.randn(tokens, hidden, generator=gen, device="cuda").abs().to(dtype)
    size = torch.rand(vocab, 1, generator=gen, device="cuda") + 6.2
    size[0] = 20.0
    w = (size * u).to(dtype)
    t = torch.zeros(tokens, dtype=torch.int64, device="cuda")
    g = torch.ones(tokens, device="cuda")
    _, lse = tb.linear_cross_entropy(h, w, t)
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse)
    H, W = h.double(), w.double()
    logits = H @ W.T
    exact = torch.logsumexp(logits, -1)
    others = (logits[:, 1:] - exact[:, None]).exp()
    d = torch.cat([-others.sum(-1, keepdim=True), others], 1)
    # Along u, dh is d . (W u); the target's part is 20 d_0, the others' about -7 d_0 in all, so a relative error of d_0 becomes 20 / 13 of it.
    # lse is rounded to float32, at most half a unit of numbers from 16 to 32, which is 2^-19, and so are its logarithm and the
    # difference: three units. Where one kernel forms the logits of both passes they are the same, whatever their error. Where two do,
    # each adds up at most K / 32 partial sums in float32: a running sum that grows evenly to 20 rounds to units of 2^-19 for
    # a fifth of the additions, half of that for two fifths, a quarter for one fifth, and so on: a variance of 0.3125 / 12 units^2 each. Six standard
    # deviations of the two together. d and dh are rounded to the type.
    same = 5 <= tokens <= 32 or tokens > 64 if dtype == torch.float32 else tokens > 16
    units = 3 if same else 3 + 6 * (2 * (hidden / 32) * 0.3125 / 12) ** 0.5
    along = dh.double() @ u.double()
    want = (d @ W) @ u.double()
    slack = units * 2.0 ** -19 * 20 / 13 / d[:, 0].abs()
    step = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 8 * U
    tol = (slack + 3 * step) * want.abs() * (1 + 1e-3)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * u.double().sum()
    err = (along - want).abs()
    assert bool((err <= tol).all()), (float((err / want.abs()).max()), float((tol / want.abs()).min()))
    # the same for the target's row of dweight: the sum of d_0 h over the tokens
    v = H.mean(0)
    want = (d[:, 0] @ H) @ v
    slack = units * 2.0 ** -19 / float(d[:, 0].abs().min())
    err = (dw[0].double() @ v - want).abs()
    tol = (slack + 3 * step) * want.abs() * (1 + 1e-3)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * v.abs().sum()
    assert bool(err <= tol), (float(err / want.abs()), float(tol / want.abs()))


@pytest.mark.parametrize("tokens", [1, 3, 5, 16, 17, 32, 33, 64, 65, 200])
def test_small_probabilities_of_float32(tokens):
    """One token counts, its hidden state is 1 and the weights are the logits themselves: a row of dweight is exp(logit - lse) grad and
    nothing else. lse = 0 and grad = 1 make it the exponential of a float32 that is known exactly."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    w = (-60 * torch.rand(20000, 1, generator=gen, device="cuda")).contiguous()
    h = torch.ones(tokens, 1, device="cuda")
    t = torch.full((tokens,), -100, device="cuda", dtype=torch.int64)
    t[tokens // 2] = 0
    zero, one = torch.zeros(tokens, device="cuda"), torch.ones(tokens, device="cuda")
    _, dw = tb.linear_cross_entropy_grad(one, h, w, t, zero)
    want = w.double().exp()
    want[0] -= 1
    # exp of float32 within two units of 2^-23; d scaled and back, its three parts (or two tf32) and the result's rounding: three more of 2^-24,
    # and the two tf32 leave 2^-22
    tol = torch.full_like(want, 11 * U)
    if 5 <= tokens <= 32:
        # The logit is a product of two tf32 parts: a part is rounded to eleven bits, 2^-11 relative at most, so what the second one leaves
        # of w is 2^-22 |w|, which exp passes on.
        tol += 2.0 ** -22 * w.double().abs()
    err = ((dw.double() - want) / want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("tokens", [1, 3, 5, 16, 17, 32, 33, 64, 65, 200])
def test_small_probabilities_of_short_weights(tokens):
    """The same over weights of ten bits, which every split of float32 leaves as they are."""
    w = (-torch.arange(960, device="cuda").float() / 16)[:, None].contiguous()
    h = torch.ones(tokens, 1, device="cuda")
    t = torch.full((tokens,), -100, device="cuda", dtype=torch.int64)
    t[tokens // 2] = 0
    zero, one = torch.zeros(tokens, device="cuda"), torch.ones(tokens, device="cuda")
    _, dw = tb.linear_cross_entropy_grad(one, h, w, t, zero)
    want = w.double().exp()
    want[0] -= 1
    assert float(dw[0]) == 0.0
    err = ((dw.double() - want) / want)[1:].abs()
    assert float(err.max()) <= 11 * U, float(err.max() / U)  # as above


@pytest.mark.parametrize("tokens", [3, 16, 40, 200])
def test_logits_at_the_ends_of_float32(tokens):
    """Entries that lie as far below the log-sum-exp as float32 goes have no probability, and an undefined logit stays undefined."""
    w = torch.tensor([0.0, -1.0, -80.0, -150.0, -1e4, -1e30, -3.0e38], device="cuda")[:, None].contiguous()
    h = torch.ones(tokens, 1, device="cuda")
    t = torch.zeros(tokens, device="cuda", dtype=torch.int64)
    g = torch.ones(tokens, device="cuda")
    loss, lse = tb.linear_cross_entropy(h, w, t)
    want = torch.logsumexp(w.double()[:, 0], 0)
    assert bool(((lse.double() - want).abs() <= 8 * U).all()) and torch.equal(loss, lse)
    dh, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse, dhidden=False)
    assert bool(torch.isfinite(dw).all()) and bool((dw[3:].abs() <= 1e-40 * tokens).all())
    assert abs(float(dw[2]) / (tokens * float((w.double()[2, 0] - want).exp())) - 1) <= 64 * U
    w[1] = float("nan")
    assert bool(torch.isnan(tb.linear_cross_entropy_grad(g, h, w, t, lse)[1][1]).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sums_over_very_many_tokens(dtype):
    """A million positive terms to an element of dweight: an accumulator that cuts off what falls below its last place would lose
    about a thousandth, more than the result's rounding."""
    tokens, hidden, vocab = 1 << 20, 16, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    h = (torch.rand(tokens, hidden, generator=gen, device="cuda") + 0.5).to(dtype)
    w = (torch.randn(vocab, hidden, generator=gen, device="cuda") * 0.1).to(dtype)
    t = torch.full((tokens,), vocab - 1, device="cuda")
    g = torch.full((tokens,), 0.01, device="cuda")
    _, lse = tb.linear_cross_entropy(h, w, t)
    _, dw = tb.linear_cross_entropy_grad(g, h, w, t, lse, dhidden=False)
    want = torch.zeros(vocab, hidden, dtype=torch.float64, device="cuda")
    for i in range(0, tokens, 1 << 17):
        H = h[i:i + (1 << 17)].double()
        p = (H @ w.double().T).softmax(-1)
        p[:, -1] -= 1.0
        want += (p * 0.01).T @ H
    rel = (dw.double() - want) / want
    # every result is rounded by at most half a step, d's roundings are evened out over the tokens; the logits are right to a few 2^-24
    assert float(rel.abs().max()) <= torch.finfo(dtype).eps / 2 * (1 + 1e-2) + 40 * U, float(rel.abs().max())
    # and on the whole nothing is lost: the roundings of 1024 results, uniform within half a step, have a mean of a thirtieth of its third
    # root; five times that
    spread = torch.finfo(dtype).eps / 2 / 3 ** 0.5 / (vocab * hidden) ** 0.5
    assert abs(float(rel.mean())) <= 5 * spread + 40 * U, float(rel.mean())
