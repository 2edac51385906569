"""What a synchronising call costs beside the wait: the error counters it reads back."""
import pytest
import torch
from torch.profiler import ProfilerActivity, profile

from tannic_b200 import _abi as A
from tannic_b200 import ops as tb

pytestmark = pytest.mark.gpu


def test_one_copy_for_each_counter():
    """One for the tensor-core kernels (products, convolutions, losses), one for the reductions."""
    a = torch.randn(256, 256, device="cuda", dtype=torch.bfloat16)
    tb.matmul(a, a)
    stream = tb.current_stream(a)
    A.check(A.lib().tn_stream_synchronize(stream))
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as p:
        for _ in range(10):
            A.check(A.lib().tn_stream_synchronize(stream))
        torch.cuda.synchronize()
    copies = sum(e.count for e in p.key_averages() if "Memcpy DtoH" in e.key)
    assert copies == 20, [(e.key, e.count) for e in p.key_averages()]
