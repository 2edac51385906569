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
