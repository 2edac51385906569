"""Errors of a linear layer's logits and gradients on the whole, and what they may be. Used by tests on the GPU, and by one on the CPU that
shows that the limits tell the kernels' arithmetic from arithmetic in fewer bits."""
import torch

U = 2.0 ** -24

# In units of 2^-24 of the logits' root mean square. The tensor cores cut an accumulator off after every step; the kernels let one take
# 4 (16 bits, up to 128 tokens) to 12 (float32 in two tf32 parts) steps from zero, each good for about a unit at most, and add up in
# float32 from there: sqrt(4096 / 32) / 2 roundings of half a unit more at the most, 3.
LOGIT_LIMIT = 12 + 3


def logit_errors(logits, tokens, hidden, dtype, one_sign, device):
    """(rms, mean signed) error of `logits(h, w)`, for a single row w, relative to the logits' root mean square, in units of 2^-24."""
    errors, exact = [], []
    for seed in range(-(-512 // tokens)):
        gen = torch.Generator(device=device).manual_seed(1000 * hidden + seed)
        h = torch.randn(tokens, hidden, generator=gen, device=device)
        w = torch.randn(1, hidden, generator=gen, device=device) * 1.5 / hidden ** 0.5
        if one_sign:
            h, w = h.abs(), w.abs()
        h, w = h.to(dtype), w.to(dtype)
        want = (h.double() * w.double()).sum(-1)
        errors.append(logits(h, w).double().reshape(-1) - want)
        exact.append(want)
    e, x = torch.cat(errors), torch.cat(exact)
    scale = x.square().mean().sqrt() * U
    return float(e.square().mean().sqrt() / scale), float((e * x.sign()).mean() / scale)


# Gradients in float32, root mean square relative to the result's own: a probability passes on its logit's error (logits of about 1.5, off by a
# third of the limit for random operands), the rounding of l - lse (up to 16, so half a unit of 2^-20, a third root of that in the mean: 5),
# the sums add a third of the limit once more. Added up plainly.
GRADIENT_LIMIT = (1.5 + 1.0) * LOGIT_LIMIT / 3 + 5 + 2.5


def gradient_data(tokens, hidden, vocab, dtype, device, seed=0):
    gen = torch.Generator(device=device).manual_seed(tokens + hidden + seed)
    h = torch.randn(tokens, hidden, generator=gen, device=device).to(dtype)
    w = (torch.randn(vocab, hidden, generator=gen, device=device) * 1.5 / hidden ** 0.5).to(dtype)
    t = torch.randint(0, vocab, (tokens,), generator=gen, device=device)
    return h, w, t, torch.rand(tokens, generator=gen, device=device) + 0.5


def exact_d(g, h, w, t, lse):
    p = (h.double() @ w.double().T - lse.double()[:, None]).exp()
    p.scatter_add_(1, t[:, None], torch.full_like(p[:, :1], -1.0))
    return p * g.double()[:, None]


def gradient_errors(gradient, tokens, hidden, vocab, device):
    """Root mean square errors of (dhidden, dweight) of `gradient(g, h, w, t, lse)` in float32, in units of 2^-24."""
    h, w, t, g = gradient_data(tokens, hidden, vocab, torch.float32, device)
    lse = torch.logsumexp(h.double() @ w.double().T, -1).float()
    d = exact_d(g, h, w, t, lse)
    out = []
    for got, want in zip(gradient(g, h, w, t, lse), (d @ w.double(), d.T @ h.double())):
        out.append(float(((got.double() - want).square().mean() / want.square().mean()).sqrt() / U))
    return out


def few_d_limit(dtype, hidden):
    """What d may be off by, relative, when it is read off a row of `hidden` results, each rounded by half a step at most: rms, four times what
    the roundings leave in the mean."""
    return 4 * torch.finfo(dtype).eps / 2 / 3 ** 0.5 / hidden ** 0.5


def d_from_dweight(gradient, tokens, hidden, vocab, dtype, device):
    """Root mean square relative error of d of the one token that counts, from the rows d h of dweight."""
    h, w, t, g = gradient_data(tokens, hidden, vocab, dtype, device)
    lse = torch.logsumexp(h.double() @ w.double().T, -1).float()
    n = tokens // 2
    d = exact_d(g, h, w, t, lse)[n]
    t = torch.where(torch.arange(tokens, device=device) == n, t, torch.full_like(t, -100))
    dw = gradient(g, h, w, t, lse)[1].double()
    x = h[n].double()
    return float((((dw @ x) / (x @ x)) / d - 1).square().mean().sqrt())


def d_from_dhidden(gradient, tokens, hidden, dtype, device):
    """The same of every token over a vocabulary of two entries, from the rows d_0 w_0 + d_1 w_1 of dhidden."""
    errors = []
    for seed in range(-(-64 // tokens)):
        h, w, t, g = gradient_data(tokens, hidden, 2, dtype, device, seed)
        lse = torch.logsumexp(h.double() @ w.double().T, -1).float()
        W = w.double()
        want = exact_d(g, h, w, t, lse) @ W
        got = gradient(g, h, w, t, lse)[0].double()
        along = W[0] - W[1]
        errors.append((got @ along) / (want @ along) - 1)
    return float(torch.cat(errors).square().mean().sqrt())
