"""What a synchronising call costs beside the wait: the error counters it reads back."""
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def test_one_copy_for_each_counter():
    """One for the tensor-core kernels (products, convolutions, losses), one for the reductions. In a process of its own, since the
    profiler that counts the copies stays with the process it was used in."""
    script = f"import sys\nsys.path.insert(0, {str(ROOT)!r})\n" + textwrap.dedent("""
        import torch
        from torch.profiler import ProfilerActivity, profile
        from tannic_b200 import _abi as A, ops as tb
        a = torch.randn(256, 256, device="cuda", dtype=torch.bfloat16)
        tb.matmul(a, a)
        stream = tb.current_stream(a)
        A.check(A.lib().tn_stream_synchronize(stream))
        with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as p:
            for _ in range(10):
                A.check(A.lib().tn_stream_synchronize(stream))
            torch.cuda.synchronize()
        print("COPIES", sum(e.count for e in p.key_averages() if "Memcpy DtoH" in e.key))
    """)
    done = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
    copies = int(done.stdout.split("COPIES")[1])
    if copies == 0:
        pytest.skip("the profiler records nothing on this machine")
    assert copies == 20, done.stdout
