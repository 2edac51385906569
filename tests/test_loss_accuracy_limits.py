"""The limits of loss_accuracy.py tell the kernels' arithmetic from arithmetic in fewer bits: both are written out here, on the CPU."""
import pytest
import torch

from loss_accuracy import GRADIENT_LIMIT, LOGIT_LIMIT, d_from_dhidden, d_from_dweight, exact_d, few_d_limit, gradient_errors, logit_errors

HIDDEN = [64, 512, 4096]


def rounded(x, bits):
    """x with `bits` significant bits."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 2.0 ** bits) / 2.0 ** bits, e)


def cut_off(x):
    m, e = torch.frexp(x)
    return torch.ldexp(torch.trunc(m * 2.0 ** 24) / 2.0 ** 24, e)


def parts(x, bits, n):
    out, rest = [], x.double()
    for _ in range(n):
        out.append(rounded(rest, bits))
        rest = rest - out[-1]
    return out


def on_tensor_cores(passes, steps):
    """Sums of products of rows, `steps` steps of 16 columns to an accumulator that is cut off after each; `passes`: pairs of parts that
    go through the columns of one accumulator one after the other."""
    rows, hidden = passes[0][0].shape
    total = torch.zeros(rows, dtype=torch.float64)
    for k in range(0, hidden, 16 * steps):
        acc = torch.zeros_like(total)
        for a, b in passes:
            for s in range(k, min(hidden, k + 16 * steps), 16):
                acc = cut_off(acc + (a[:, s:s + 16] * b[:, s:s + 16]).sum(1))
        total = (total + acc).float().double()
    return total.float()


def split(h, w, bits, n, which, steps):
    a, b = parts(h, bits, n), parts(w.expand_as(h), bits, n)
    return on_tensor_cores([(a[i], b[j]) for i, j in which], steps)


SIX = [(2, 0), (1, 1), (0, 2), (1, 0), (0, 1), (0, 0)]
RIGHT = {
    "float32": lambda h, w: h @ w[0],
    "three parts of 8 bits": lambda h, w: split(h, w, 8, 3, SIX, 8),
    "two parts of 11 bits": lambda h, w: split(h, w, 11, 2, [(1, 0), (0, 1), (0, 0)], 2),
}
WRONG = {
    "two parts of 8 bits": lambda h, w: split(h, w, 8, 2, [(1, 1), (1, 0), (0, 1), (0, 0)], 8),
    "one part of 8 bits": lambda h, w: split(h, w, 8, 1, [(0, 0)], 8),
    "one part of 11 bits": lambda h, w: split(h, w, 11, 1, [(0, 0)], 2),
    "weights of 11 bits": lambda h, w: (h.double() * rounded(w.double(), 11)).sum(-1).float(),
    "largest products first, one accumulator": lambda h, w: split(h, w, 8, 3, SIX[::-1], 256),
}


@pytest.mark.parametrize("hidden", HIDDEN)
@pytest.mark.parametrize("name", RIGHT)
def test_logits_in_float32_pass(name, hidden):
    for one_sign in (False, True):
        rms, signed = logit_errors(RIGHT[name], 128, hidden, torch.float32, one_sign, "cpu")
        assert rms <= LOGIT_LIMIT / 2 and abs(signed) <= LOGIT_LIMIT / 2, (rms, signed)


@pytest.mark.parametrize("hidden", HIDDEN)
@pytest.mark.parametrize("name", WRONG)
def test_logits_in_fewer_bits_do_not(name, hidden):
    errors = [e for one_sign in (False, True) for e in logit_errors(WRONG[name], 128, hidden, torch.float32, one_sign, "cpu")]
    assert max(abs(e) for e in errors) > LOGIT_LIMIT, errors


@pytest.mark.parametrize("hidden", [1024, 4096])
def test_an_accumulator_for_all_of_k_grows_with_it(hidden):
    """bfloat16: sixteen blocks to an accumulator keep the error of 1024 columns, one for all columns does not."""
    at = lambda hidden, steps: logit_errors(lambda h, w: on_tensor_cores([(h.double(), w.expand_as(h).double())], steps), 128, hidden,  # noqa: E731
                                            torch.bfloat16, True, "cpu")[0]
    assert at(hidden, 64) <= 1.5 * at(1024, 64)
    if hidden == 4096:
        assert at(hidden, 256) > 2.5 * at(1024, 64)


def gradient(h_of, d_of):
    def run(g, h, w, t, lse):
        H, W = h_of(h), h_of(w)
        keep = t >= 0
        at = torch.where(keep, t, torch.zeros_like(t))
        d = torch.where(keep[:, None], d_of(exact_d(g, H, W, at, lse)), torch.zeros(1, dtype=torch.float64))
        return (d @ W.double()).to(h.dtype), (d.T @ H.double()).to(w.dtype)
    return run


def of_parts(bits, n):
    return lambda x: sum(parts(x, bits, n))


def in_float32(g, h, w, t, lse):
    d = (h @ w.T - lse[:, None]).exp()
    d.scatter_add_(1, t[:, None], torch.full_like(d[:, :1], -1.0))
    d = d * g[:, None]
    return d @ w, d.T @ h


@pytest.mark.parametrize("tokens", [3, 16, 200])
@pytest.mark.parametrize("hidden", HIDDEN)
def test_gradients(hidden, tokens):
    errors = lambda f: gradient_errors(f, tokens, hidden, 512, "cpu")  # noqa: E731
    assert max(errors(in_float32)) <= GRADIENT_LIMIT / 2
    assert max(errors(gradient(of_parts(8, 3), of_parts(8, 3)))) <= GRADIENT_LIMIT / 2
    assert max(errors(gradient(of_parts(11, 2), of_parts(11, 2)))) <= GRADIENT_LIMIT / 2
    for h_of, d_of in ((of_parts(8, 2), of_parts(8, 3)), (of_parts(8, 3), of_parts(8, 2)), (of_parts(11, 1), of_parts(11, 2)), (of_parts(11, 2), of_parts(11, 1))):
        assert max(errors(gradient(h_of, d_of))) > GRADIENT_LIMIT, errors(gradient(h_of, d_of))


@pytest.mark.parametrize("dtype,bits", [(torch.float16, 11), (torch.bfloat16, 8)])
@pytest.mark.parametrize("tokens", [1, 8])
def test_d_of_two_parts(tokens, dtype, bits):
    same = lambda x: x  # noqa: E731
    limit = few_d_limit(dtype, 2048)
    for n, passes in ((2, True), (1, False)):
        f = gradient(same, of_parts(bits, n))
        assert (d_from_dweight(f, tokens, 2048, 300, dtype, "cpu") <= limit) is passes
        assert (d_from_dhidden(f, tokens, 2048, dtype, "cpu") <= limit) is passes
