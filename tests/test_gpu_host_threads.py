"""Normalisation and loss called from two host threads: what one thread asks for takes nothing from the other."""
import concurrent.futures

import pytest
import torch

from tannic_b200 import ops as tb

pytestmark = pytest.mark.gpu

IGNORE = -100


def norm(cols, dtype):
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x, dy = (torch.randn(5, cols, generator=gen, device="cuda").to(dtype) for _ in range(2))
    w = torch.randn(cols, generator=gen, device="cuda").to(dtype)
    _, mean, rstd = (t.clone() for t in tb.layer_norm(x, w, stats=True))
    return lambda: tb.layer_norm(x, w, stats=True), lambda: tb.layer_norm_grad(dy, x, mean, rstd, w)


def loss(tokens, hidden, dtype):
    gen = torch.Generator(device="cuda").manual_seed(hidden)
    h, w = (torch.randn(n, hidden, generator=gen, device="cuda").to(dtype) for n in (tokens, 64))
    t = torch.arange(tokens, device="cuda")
    g = torch.ones(tokens, device="cuda")
    lse = tb.linear_cross_entropy(h, w, t)[1].clone()
    return lambda: tb.linear_cross_entropy(h, w, t), lambda: tb.linear_cross_entropy_grad(g, h, w, t, lse)


# two sizes of one kernel, the first with more shared memory than the second
SIZES = {
    "norm, aligned": lambda: [norm(c, torch.float32)[0] for c in (8192, 4096)],
    "norm, unaligned": lambda: [norm(c, torch.float32)[0] for c in (8191, 4099)],
    "norm gradient, aligned": lambda: [norm(c, torch.bfloat16)[1] for c in (8192, 4096)],
    "norm gradient, unaligned": lambda: [norm(c, torch.float32)[1] for c in (8191, 4099)],
    "norm gradient, long rows": lambda: [norm(c, torch.float32)[1] for c in (16384, 12288)],
    "loss, one token of 16 bits": lambda: [loss(1, c, torch.bfloat16)[0] for c in (40000, 12000)],
    "loss, four tokens of float32": lambda: [loss(4, c, torch.float32)[0] for c in (12000, 4000)],
    "loss gradient, four tokens of float32": lambda: [loss(4, c, torch.float32)[1] for c in (4096, 2048)],
    "loss gradient, four tokens of 16 bits": lambda: [loss(4, c, torch.float16)[1] for c in (4096, 2048)],
}


@pytest.mark.parametrize("name", SIZES)
def test_one_kernel_at_two_sizes_in_two_threads(name):
    large, small = SIZES[name]()
    with concurrent.futures.ThreadPoolExecutor(1) as one, concurrent.futures.ThreadPoolExecutor(1) as two:
        def on(pool, call):
            def run():
                with torch.cuda.stream(torch.cuda.default_stream()):
                    return [t for t in call() if t is not None]
            return pool.submit(run).result()

        want = on(one, large), on(two, small)
        for _ in range(3):  # each thread has made its call before, and has it again after the other's
            got = on(one, large), on(two, small)
            torch.cuda.synchronize()
            for a, b in zip(want, got):
                assert all(torch.equal(p, q) for p, q in zip(a, b))
        # and both at once
        both = [pool.submit(lambda call=call: [call() for _ in range(200)][-1]) for pool, call in ((one, large), (two, small))]
        for a, b in zip(want, both):
            assert all(torch.equal(p, q) for p, q in zip(a, [t for t in b.result() if t is not None]))
