"""How far the results of the cross entropy of a linear layer and of its gradient are off on the whole: root mean square and mean signed error
against 64 bits. The bounds of single elements in the other files hold for every order of every sum; these here are what the arithmetic
does to random operands, and would not hold for a kernel that dropped a part of its operands."""
import pytest
import torch

from loss_accuracy import GRADIENT_LIMIT, LOGIT_LIMIT, d_from_dhidden, d_from_dweight, few_d_limit, gradient_errors, logit_errors
from tannic_b200 import ops as tb
from test_gpu_linear_cross_entropy import both, data

pytestmark = pytest.mark.gpu

# types and numbers of tokens of which one kernel each forms the logits
FORWARD = [(1, torch.float32), (4, torch.float32), (5, torch.float32), (16, torch.float32), (17, torch.float32), (64, torch.float32),
           (65, torch.float32), (300, torch.float32), *((n, t) for n in (1, 2, 16, 17, 128) for t in (torch.float16, torch.bfloat16))]


def forward(h, w):
    """Over a vocabulary of one entry the log-sum-exp is the logit itself."""
    return tb.linear_cross_entropy(h, w, torch.zeros(h.shape[0], dtype=torch.int64, device="cuda"))[1]


@pytest.mark.parametrize("one_sign", [False, True])
@pytest.mark.parametrize("tokens,dtype", FORWARD)
@pytest.mark.parametrize("hidden", [64, 72, 512, 1032, 4096])
def test_logits(hidden, tokens, dtype, one_sign):
    rms, signed = logit_errors(forward, tokens, hidden, dtype, one_sign, "cuda")
    assert rms <= LOGIT_LIMIT and abs(signed) <= LOGIT_LIMIT, (rms, signed)
    assert tb.device_errors() == 0


@pytest.mark.parametrize("one_sign", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hidden", [1032, 2048, 4096])
def test_logits_of_many_tokens_do_not_drift_with_the_columns(hidden, dtype, one_sign):
    """More than 128 tokens of 16 bits: an accumulator takes 1024 columns, 64 steps, which are good for two units each at most and some
    roundings beside; what it leaves out does not grow beyond that."""
    at = lambda hidden: logit_errors(forward, 300, hidden, dtype, one_sign, "cuda")  # noqa: E731
    base, rms = at(1024)[0], at(hidden)[0]
    assert rms <= 1.5 * base and base <= 2 * 64 + 3, (rms, base)


@pytest.mark.parametrize("tokens", [3, 4, 5, 16, 17, 32, 33, 64, 65, 200, 300])
@pytest.mark.parametrize("hidden", [64, 72, 512, 1000, 4096])
def test_float32_gradients(hidden, tokens):
    errors = gradient_errors(tb.linear_cross_entropy_grad, tokens, hidden, 512, "cuda")
    assert max(errors) <= GRADIENT_LIMIT, errors


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 2, 5, 8, 9, 16])
def test_d_of_a_few_tokens_of_16_bits(tokens, dtype):
    """Two parts of the operands' type: far better than the results show one by one."""
    limit = few_d_limit(dtype, 2048)
    for error in (d_from_dweight(tb.linear_cross_entropy_grad, tokens, 2048, 300, dtype, "cuda"),
                  d_from_dhidden(tb.linear_cross_entropy_grad, tokens, 2048, dtype, "cuda")):
        assert error <= limit, (error, limit)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [100, 129, 300])
@pytest.mark.parametrize("hidden", [1032, 2048, 4096])
def test_wide_rows_of_many_tokens(hidden, tokens, dtype):
    both(*data(tokens, hidden, 700, dtype, hidden + tokens, ignored=0.1))
