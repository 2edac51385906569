"""How far the results of the cross entropy of a linear layer and of its gradient are off on the whole: root mean square and mean signed error
against 64 bits. The bounds of single elements in the other files hold for every order of every sum; these here are what the arithmetic
does to random operands, and would not hold for a kernel that dropped a part of its operands."""
import pytest
import torch

from loss_accuracy import LOGIT_LIMIT, logit_errors
from tannic_b200 import ops as tb

pytestmark = pytest.mark.gpu

# types and numbers of tokens of which one kernel each forms the logits
FORWARD = [(1, torch.float32), (4, torch.float32), (5, torch.float32), (16, torch.float32), (17, torch.float32), (64, torch.float32),
           (65, torch.float32), (300, torch.float32)]


@pytest.mark.parametrize("one_sign", [False, True])
@pytest.mark.parametrize("tokens,dtype", FORWARD)
@pytest.mark.parametrize("hidden", [64, 72, 512, 1032, 4096])
def test_logits(hidden, tokens, dtype, one_sign):
    """Over a vocabulary of one entry the log-sum-exp is the logit itself."""
    rms, signed = logit_errors(lambda h, w: tb.linear_cross_entropy(h, w, torch.zeros(h.shape[0], dtype=torch.int64, device="cuda"))[1],
                               tokens, hidden, dtype, one_sign, "cuda")
    assert rms <= LOGIT_LIMIT and abs(signed) <= LOGIT_LIMIT, (rms, signed)
    assert tb.device_errors() == 0
