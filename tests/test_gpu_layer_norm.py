"""Layer normalisation and its gradient (tn_layer_norm, tn_layer_norm_grad) against the formula in 64 bits.

The tolerance of every element is the rounding that the arithmetic can cause, with u = 2^-24 (2^-53 for float64): one half step of
the result's type (torch.finfo(t).eps / 2 relative), and for a sum of n terms added in a tree of depth d at most d u times the
sum of the magnitudes. A thread adds at most 32 elements of a row (a thousandth of it where the row is longer than 16384), then
come five shuffles and at most 32 warps.
"""
import pytest
import torch

from tannic_b200 import _abi as A
from tannic_b200 import ops as tb

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32, torch.float64]


def unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def depth(cols):
    return max(32, cols // 1024 + 1) + 5 + 32


def reference(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    z = c * rstd
    y = z
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean.squeeze(-1), rstd.squeeze(-1)


def check_forward(x, w, b, eps, got):
    """`got` = (y, mean, rstd) of x; x may be any view."""
    y, mean, rstd = got
    want, m, r = reference(x, w, b, eps)
    u, d, cols = unit(x.dtype), depth(x.shape[-1]), x.shape[-1]
    wide = x.double()
    em = (d + 2) * u * wide.abs().mean(-1)                                   # of the mean
    var = (wide - m.unsqueeze(-1)).square().mean(-1)
    # of the variance: the tree, the subtraction (relative 2 u twice in the square), and the mean's error squared and
    # times the sum of the rounded differences
    ev = (d + 6) * u * var + em.square() + 2 * em * 2 * u * (wide - m.unsqueeze(-1)).abs().mean(-1)
    er = r * (0.5 * ev / (var + eps) + 6 * u) * (1 + 1e-3)                       # square root, quotient, conversion of eps
    assert bool(((mean.double() - m).abs() <= em).all()), float((mean.double() - m).abs().max())
    assert bool(((rstd.double() - r).abs() <= er + (r == float("inf")).double()).all()), float((rstd.double() - r).abs().max())
    wabs = w.double().abs() if w is not None else 1.0
    c = (wide - m.unsqueeze(-1)).abs()
    tol = wabs * ((em.unsqueeze(-1) + u * c) * r.unsqueeze(-1) + c * er.unsqueeze(-1) + 3 * u * c * r.unsqueeze(-1))
    tol = tol * (1 + 1e-3) + 2 * u * want.abs() + torch.finfo(x.dtype).eps / 2 * want.abs() * (1 + 1e-3)
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step below the smallest normal number
    bad = ((y.double() - want).abs() > tol) | ~torch.isfinite(y.double())
    assert not bool(bad.any()), (int(bad.sum()), float((y.double() - want).abs().max()))
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()


def check_backward(dy, x, mean, rstd, w, got):
    dx, dw, db = got
    cols = x.shape[-1]
    u, d = unit(x.dtype), depth(cols)
    X, D = x.double().reshape(-1, cols), dy.double().reshape(-1, cols)
    m, r = mean.double().reshape(-1, 1), rstd.double().reshape(-1, 1)
    z = (X - m) * r
    ez = 3 * u * z.abs()
    g = D * w.double() if w is not None else D
    mg, mgz = g.mean(-1, keepdim=True), (g * z).mean(-1, keepdim=True)
    want = r * (g - mg - z * mgz)
    e = u * g.abs() + (d + 3) * u * g.abs().mean(-1, keepdim=True) + z.abs() * (d + 8) * u * (g * z).abs().mean(-1, keepdim=True) \
        + ez * mgz.abs() + 4 * u * (g.abs() + mg.abs() + (z * mgz).abs())
    tol = r * e * (1 + 1e-3) + (u + torch.finfo(x.dtype).eps / 2) * want.abs() * (1 + 1e-3)
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    err = (dx.double().reshape(-1, cols) - want).abs()
    assert bool((err <= tol).all()), (int((err > tol).sum()), float((err / tol).max()))
    if w is None:
        assert dw is None and db is None
        return
    rows = X.shape[0]
    for name, got_p, terms in (("dweight", dw, D * z), ("dbias", db, D)):
        want_p = terms.sum(0)
        tol = (rows + 80) * u * terms.abs().sum(0) + torch.finfo(w.dtype).eps / 2 * want_p.abs() * (1 + 1e-3)
        if w.dtype == torch.float16:
            tol = tol + 2.0 ** -25
        err = (got_p.double() - want_p).abs()
        assert bool((err <= tol).all()), (name, float((err / tol).max()))
        assert got_p.dtype == w.dtype


def data(shape, dtype, seed, params="same"):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64) * 1.7 + 0.4).to(dtype)
    dy = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64).to(dtype)
    if params is None:
        return x, dy, None, None
    pt = dtype if params == "same" else params
    w = (1 + 0.3 * torch.randn(shape[-1], generator=gen, device="cuda", dtype=torch.float64)).to(pt)
    b = (0.3 * torch.randn(shape[-1], generator=gen, device="cuda", dtype=torch.float64)).to(pt)
    return x, dy, w, b


def both(x, dy, w, b, eps=1e-5):
    got = tb.layer_norm(x, w, b, eps=eps, stats=True)
    check_forward(x, w, b, eps, got)
    check_backward(dy, x, got[1], got[2], w, tb.layer_norm_grad(dy, x, got[1], got[2], w))


# one column; around every change of variant; odd lengths; one vector more and less
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 31, 197, 255, 256, 264, 511, 768, 1001, 1024, 1032, 2047, 2056, 4096, 4097, 8192, 8200, 16383, 16384, 16400, 40001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_row_lengths(cols, dtype):
    both(*data((5, cols), dtype, cols))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 1000, 3001])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [96, 768, 2304])
def test_row_counts(rows, dtype, cols):
    both(*data((rows, cols), dtype, rows))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cols", [1, 200, 333, 1024, 3000, 16384, 20000])
def test_float32_parameters(dtype, cols):
    both(*data((9, cols), dtype, 3, torch.float32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_no_parameters_and_one_of_them(dtype):
    x, dy, w, b = data((6, 264), dtype, 4)
    both(x, dy, None, None)
    for pair in ((w, None), (None, b)):
        check_forward(x, *pair, 1e-5, tb.layer_norm(x, *pair, stats=True))
    _, mean, rstd = tb.layer_norm(x, stats=True)
    dx, dw, db = tb.layer_norm_grad(dy, x, mean, rstd, w, bias=False)
    assert db is None
    full = tb.layer_norm_grad(dy, x, mean, rstd, w)
    assert torch.equal(full[0], dx) and torch.equal(full[1], dw)


@pytest.mark.parametrize("view", ["pitch", "odd pitch", "transposed", "expanded", "sliced columns", "permuted", "offset", "step"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views(view, dtype):
    make = {
        "pitch": lambda t: torch.cat([t, t], -1)[..., : t.shape[-1]],
        "odd pitch": lambda t: torch.nn.functional.pad(t, (0, 3))[..., : t.shape[-1]],
        "transposed": lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2),
        "expanded": lambda t: t[:1].expand(t.shape),
        "sliced columns": lambda t: torch.nn.functional.pad(t, (8, 8))[..., 8:-8],
        "permuted": lambda t: t.permute(1, 0, 2).contiguous().permute(1, 0, 2),
        "offset": lambda t: torch.nn.functional.pad(t.reshape(-1), (1, 0))[1:].reshape(t.shape),
        "step": lambda t: t.repeat_interleave(2, -1)[..., ::2],
    }[view]
    x, dy, w, b = data((4, 6, 264), dtype, 9)
    both(make(x), make(dy), w, b)
    # parameters that start off a 16-byte boundary
    w1, b1 = (torch.nn.functional.pad(t, (1, 0))[1:] for t in (w, b))
    both(x, dy, w1, b1)


def test_large_offset_keeps_its_digits():
    # a mean a thousand times the deviation: the squares' difference would leave nothing
    x, dy, w, b = data((8, 1024), torch.float32, 5)
    both(x + 2000.0, dy, w, b)


def test_constant_rows_infinities_and_nan():
    x = torch.full((3, 512), 2.5, device="cuda", dtype=torch.float32)
    w, b = torch.full((512,), 3.0, device="cuda"), torch.arange(512, device="cuda", dtype=torch.float32)
    y, mean, rstd = tb.layer_norm(x, w, b, stats=True)
    assert torch.equal(y, b.expand(3, 512)) and bool((mean == 2.5).all())
    assert bool(((rstd - 1e-5 ** -0.5).abs() <= 8 * 2.0 ** -24 * 1e-5 ** -0.5).all())
    # a row with an infinity or a NaN is NaN; its neighbours are untouched
    x = data((4, 512), torch.float32, 6)[0]
    clean = tb.layer_norm(x)
    x2 = x.clone()
    x2[1, 7], x2[2, 500] = float("inf"), float("nan")
    got = tb.layer_norm(x2)
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[2]).all())
    assert torch.equal(got[0], clean[0]) and torch.equal(got[3], clean[3])


@pytest.mark.parametrize("cols", [264, 20000])
def test_result_in_place(cols):
    x, dy, w, b = data((7, cols), torch.bfloat16, 8)
    y, mean, rstd = tb.layer_norm(x, w, b, stats=True)
    want = tb.layer_norm_grad(dy, x, mean, rstd, w)
    x2 = x.clone()
    assert torch.equal(tb.layer_norm(x2, w, b, out=x2), y) and torch.equal(x2, y)
    import ctypes as C
    for name in ("dy", "x"):
        args = {"dy": dy.clone(), "x": x.clone()}
        dw, db = torch.empty_like(w), torch.empty_like(b)
        ref = {k: C.byref(tb.desc(t)) for k, t in args.items()}
        A.check(A.lib().tn_layer_norm_grad(ref["dy"], ref["x"], C.byref(tb.desc(mean)), C.byref(tb.desc(rstd)), C.byref(tb.desc(w)), ref[name],
                                           C.byref(tb.desc(dw)), C.byref(tb.desc(db)), tb.current_stream(x)))
        assert torch.equal(args[name], want[0]) and torch.equal(dw, want[1]) and torch.equal(db, want[2])


def test_no_rows():
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    y, mean, rstd = tb.layer_norm(x, w, w, stats=True)
    assert y.shape == x.shape and mean.numel() == 0
    dx, dw, db = tb.layer_norm_grad(x, x, mean, rstd, w)
    assert dx.shape == x.shape and not bool(dw.any()) and not bool(db.any())


def test_rank_one_and_many_axes():
    x, dy, w, b = data((300,), torch.float32, 10)
    both(x, dy, w, b)
    x, dy, w, b = data((2, 1, 3, 1, 2, 40), torch.float16, 11)
    both(x, dy, w, b)


def test_same_bits_on_every_run():
    x, dy, w, b = data((5000, 768), torch.bfloat16, 12)
    y, mean, rstd = tb.layer_norm(x, w, b, stats=True)
    first = tb.layer_norm_grad(dy, x, mean, rstd, w)
    for _ in range(5):
        again = tb.layer_norm_grad(dy, x, mean, rstd, w)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_gradient_against_differences():
    x, dy, w, b = data((3, 40), torch.float64, 13)
    _, mean, rstd = tb.layer_norm(x, w, b, stats=True)
    dx, dw, db = tb.layer_norm_grad(dy, x, mean, rstd, w)
    value = lambda x, w, b: float((tb.layer_norm(x, w, b) * dy).sum())  # noqa: E731
    h = 1e-5
    for tensors, index, grad in (((x, w, b), 0, dx), ((x, w, b), 1, dw), ((x, w, b), 2, db)):
        flat = grad.reshape(-1)
        for at in range(0, flat.numel(), 7):
            up, down = ([t.clone() for t in tensors] for _ in range(2))
            up[index].view(-1)[at] += h
            down[index].view(-1)[at] -= h
            slope = (value(*up) - value(*down)) / (2 * h)
            # third derivatives of a row of order one: h^2 times a few; the values' rounding over h
            assert abs(slope - float(flat[at])) < 1e-7 * (1 + abs(slope)), (index, at)


def test_captured_and_replayed_on_another_stream():
    x, dy, w, b = data((500, 768), torch.bfloat16, 14)
    y, mean, rstd = tb.layer_norm(x, w, b, stats=True)
    want = tb.layer_norm_grad(dy, x, mean, rstd, w)
    other = [data((500, 768), torch.bfloat16, 15)[i] for i in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):  # two graphs, each with its own scratch memory inside
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = tb.layer_norm(x, w, b, stats=True)
                grads = tb.layer_norm_grad(dy, x, out[1], out[2], w)
            graphs.append((g, out, grads))
    torch.cuda.synchronize()
    for g, out, grads in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, out, grads in graphs:
        assert torch.equal(out[0], y) and all(torch.equal(p, q) for p, q in zip(grads, want))
    keep_x, keep_dy = x.clone(), dy.clone()
    x.copy_(other[0])
    dy.copy_(other[1])
    y2, mean2, rstd2 = tb.layer_norm(x, w, b, stats=True)
    want2 = tb.layer_norm_grad(dy, x, mean2, rstd2, w)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], y2) and all(torch.equal(p, q) for p, q in zip(graphs[0][2], want2))
    x.copy_(keep_x)
    dy.copy_(keep_dy)


def test_rows_behind_the_tensor_are_left_alone():
    buf = torch.full((10, 200), 7.0, device="cuda", dtype=torch.float16)
    x, dy, w, b = data((6, 200), torch.float16, 16)
    tb.layer_norm(x, w, b, out=buf[:6])
    assert bool((buf[6:] == 7.0).all())
