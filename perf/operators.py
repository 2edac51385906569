"""Timing cases of the operators at the two ends of a network's last layer: layer normalisation and
the softmax cross entropy of a linear layer over a large vocabulary, each with its gradient.

`run` evaluates one case: in its plain form (elementary torch operations in float32, rounded once at
the end) or, where `own` is set, through `tannic_b200.ops`.
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
EPS = 1e-5
IGNORE = -100


def listed():
    return [
        # the norm in front of every layer while one token at a time is generated: latency
        {"name": "norm: one token", "op": "norm", "dtype": "bf16", "params": "bf16", "rows": 1, "cols": 4096},
        # a batch of 256 images of 197 patches, 12 heads of 64
        {"name": "norm: image patches", "op": "norm", "dtype": "bf16", "params": "bf16", "rows": 256 * 197, "cols": 768},
        # odd row length: no row but the first starts on a 16-byte boundary
        {"name": "norm: odd rows", "op": "norm", "dtype": "f32", "params": "f32", "rows": 4099, "cols": 1001},
        # the backward pass over a batch of eight sequences of 2048 tokens
        {"name": "norm gradient: long rows", "op": "norm_grad", "dtype": "bf16", "params": "bf16", "rows": 8 * 2048, "cols": 4096},
        # the patches again, float16 activations and float32 parameters (mixed-precision training)
        {"name": "norm gradient: image patches", "op": "norm_grad", "dtype": "fp16", "params": "f32", "rows": 256 * 197, "cols": 768},
        # one image: a small batch, where the reduction over rows is the latency
        {"name": "norm gradient: one image", "op": "norm_grad", "dtype": "f32", "params": "f32", "rows": 197, "cols": 768},
        # scoring one token against the whole vocabulary: reading the weights is the work
        {"name": "loss: one token", "op": "loss", "dtype": "bf16", "tokens": 1, "hidden": 4096, "vocab": 131072, "ignored": 0.0},
        # an evaluation batch, no extent a multiple of a tile
        {"name": "loss: ragged", "op": "loss", "dtype": "fp16", "tokens": 4095, "hidden": 768, "vocab": 50257, "ignored": 0.1},
        # full precision, a small model
        {"name": "loss: float32", "op": "loss", "dtype": "f32", "tokens": 512, "hidden": 1024, "vocab": 14336, "ignored": 0.0},
        # a training step's largest product
        {"name": "loss gradient: large", "op": "loss_grad", "dtype": "bf16", "tokens": 8192, "hidden": 4096, "vocab": 131072, "ignored": 0.02},
        # a padded batch: a third of the tokens carry no target
        {"name": "loss gradient: ragged", "op": "loss_grad", "dtype": "fp16", "tokens": 1021, "hidden": 768, "vocab": 50257, "ignored": 0.33},
        # adapting to a handful of tokens: the weights' gradient is the traffic
        {"name": "loss gradient: few tokens", "op": "loss_grad", "dtype": "bf16", "tokens": 4, "hidden": 4096, "vocab": 32000, "ignored": 0.0},
    ]


def _spread(rng, low, high):
    """A size between low and high, even over its logarithm; every second one is made odd."""
    n = int(round(low * (high / low) ** rng.random()))
    if rng.random() < 0.5:
        n |= 1
    else:
        n -= n % 8
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "loss", "loss_grad"])
    dtype = rng.choice(["bf16", "fp16", "f32"] if op.startswith("norm") else ["bf16", "fp16", "bf16", "f32"])
    if op.startswith("norm"):
        cols = _spread(rng, 64, 16384)
        rows = _spread(rng, 1, min(65536, 16384 * 4096 // cols))
        return {"op": op, "dtype": dtype, "params": rng.choice([dtype, "f32"]), "rows": rows, "cols": cols}
    vocab = _spread(rng, 1000, 131072)
    hidden = _spread(rng, 64, 4096)
    # float32 products cost several times those of 16-bit operands
    most = 8192 * 4096 * 131072 // (16 if dtype == "f32" else 1)
    tokens = _spread(rng, 1, min(8192, most // (vocab * hidden)))
    return {"op": op, "dtype": dtype, "tokens": tokens, "hidden": hidden, "vocab": vocab, "ignored": rng.choice([0.0, 0.1, 0.5])}


def _normal(gen, shape, dtype, mean=0.0, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).add_(mean).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"op": case["op"]}
    if case["op"].startswith("norm"):
        rows, cols, params = case["rows"], case["cols"], DTYPES[case["params"]]
        # a residual stream: channels of different offset and width
        offset = torch.randn(cols, generator=gen, device="cuda") * 0.5
        width = torch.rand(cols, generator=gen, device="cuda") * 2.0 + 0.25
        s["x"] = torch.randn(rows, cols, generator=gen, device="cuda").mul_(width).add_(offset).to(dtype)
        s["weight"] = _normal(gen, (cols,), params, 1.0, 0.2)
        s["bias"] = _normal(gen, (cols,), params, 0.0, 0.2)
        if case["op"] == "norm_grad":
            s["dy"] = _normal(gen, (rows, cols), dtype, 0.0, 1.0)
            wide = s["x"].double()
            mean = wide.mean(-1)
            rstd = ((wide - mean[:, None]).square().mean(-1) + EPS).rsqrt()
            s["mean"], s["rstd"] = mean.float(), rstd.float()
        return s
    tokens, hidden, vocab = case["tokens"], case["hidden"], case["vocab"]
    # logits with a standard deviation of about 1.3, as an initialised head gives; every second token
    # points towards its target, as after training
    s["weight"] = _normal(gen, (vocab, hidden), dtype, 0.0, 1.28 / hidden ** 0.5)
    targets = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    pull = torch.rand(tokens, 1, generator=gen, device="cuda") * 4.0 * (torch.arange(tokens, device="cuda")[:, None] % 2)
    s["hidden"] = (torch.randn(tokens, hidden, generator=gen, device="cuda") + pull * s["weight"][targets].float()).to(dtype)
    left_out = torch.rand(tokens, generator=gen, device="cuda") < case["ignored"]
    s["targets"] = torch.where(left_out, torch.full_like(targets, IGNORE), targets)
    if case["op"] == "loss_grad":
        s["lse"] = _plain_loss(s["hidden"], s["weight"], s["targets"])[1]
        # the gradient of the mean over the tokens that count; float16 training scales its loss, or
        # most of the weights' gradient would round to zero
        count = (~left_out).sum().clamp(min=1)
        s["grad"] = ((4096.0 if case["dtype"] == "fp16" else 1.0) / count).float().expand(tokens).contiguous()
    return s


def _plain_norm(x, weight, bias):
    wide = x.float()
    mean = wide.mean(-1)
    centred = wide - mean[:, None]
    rstd = 1.0 / (centred.square().mean(-1) + EPS).sqrt()
    y = centred * rstd[:, None] * weight.float() + bias.float()
    return y.to(x.dtype), mean, rstd


def _plain_norm_grad(dy, x, mean, rstd, weight):
    normal = (x.float() - mean[:, None]) * rstd[:, None]
    out = dy.float()
    g = out * weight.float()
    dx = (g - g.mean(-1)[:, None] - normal * (g * normal).mean(-1)[:, None]) * rstd[:, None]
    return dx.to(x.dtype), (out * normal).sum(0).to(weight.dtype), out.sum(0).to(weight.dtype)


def _plain_loss(hidden, weight, targets):
    logits = hidden.float() @ weight.float().T
    top = logits.amax(-1)
    lse = (logits - top[:, None]).exp().sum(-1).log() + top
    counts = targets != IGNORE
    at = torch.where(counts, targets, torch.zeros_like(targets))
    loss = torch.where(counts, lse - logits.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    return loss, lse


def _plain_loss_grad(grad, hidden, weight, targets, lse):
    wide_h, wide_w = hidden.float(), weight.float()
    d = (wide_h @ wide_w.T - lse[:, None]).exp()
    counts = targets != IGNORE
    at = torch.where(counts, targets, torch.zeros_like(targets))
    rows = torch.arange(d.shape[0], device=d.device)
    d[rows, at] -= 1.0
    d *= torch.where(counts, grad, torch.zeros_like(grad))[:, None]
    return (d @ wide_w).to(hidden.dtype), (d.T @ wide_h).to(weight.dtype)


def run(s):
    if own:
        from tannic_b200 import ops
        if s["op"] == "norm":
            return ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, stats=True)
        if s["op"] == "norm_grad":
            return ops.layer_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
        if s["op"] == "loss":
            return ops.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], ignore_index=IGNORE)
        return ops.linear_cross_entropy_grad(s["grad"], s["hidden"], s["weight"], s["targets"], s["lse"], ignore_index=IGNORE)
    if s["op"] == "norm":
        return _plain_norm(s["x"], s["weight"], s["bias"])
    if s["op"] == "norm_grad":
        return _plain_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
    if s["op"] == "loss":
        return _plain_loss(s["hidden"], s["weight"], s["targets"])
    return _plain_loss_grad(s["grad"], s["hidden"], s["weight"], s["targets"], s["lse"])


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"].startswith("norm"):
        psize = 4 if case["params"] == "f32" else 2
        rows, cols = case["rows"], case["cols"]
        if case["op"] == "norm":  # x in, y out, two parameter rows in, two statistics a row out
            return {"bytes": 2 * rows * cols * size + 2 * cols * psize + 8 * rows, "flops": 7 * rows * cols}
        # x and dy in, dx out, the statistics and the weight in, two parameter gradients out
        return {"bytes": 3 * rows * cols * size + 3 * cols * psize + 8 * rows, "flops": 13 * rows * cols}
    n, h, v = case["tokens"], case["hidden"], case["vocab"]
    if case["op"] == "loss":  # operands and targets in, loss and log-sum-exp out
        return {"bytes": (n + v) * h * size + 16 * n, "flops": 2 * n * h * v}
    # operands, targets, log-sum-exp and upstream gradient in, two gradients out; three products
    return {"bytes": 2 * (n + v) * h * size + 16 * n, "flops": 6 * n * h * v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("norm"):
        x, weight = s["x"].double(), s["weight"].double()
        if case["op"] == "norm":
            var, mean = torch.var_mean(x, dim=-1, correction=0)
            rstd = (var + EPS).pow(-0.5)
            y = torch.addcmul(s["bias"].double(), (x - mean.unsqueeze(1)).mul_(rstd.unsqueeze(1)), weight)
            return y, mean, rstd
        cols, dy = case["cols"], s["dy"].double()
        r, m = s["rstd"].double().unsqueeze(1), s["mean"].double().unsqueeze(1)
        z = (x - m) * r
        # the Jacobian of the row, applied from its two rank-one terms
        t = dy * weight
        row_sum, row_dot = t.sum(1, keepdim=True), (t * z).sum(1, keepdim=True)
        return r / cols * (cols * t - row_sum - z * row_dot), torch.einsum("rc,rc->c", dy, z), dy.sum(0)
    w, targets = s["weight"].double(), s["targets"]
    n, step = case["tokens"], max(1, (1 << 28) // case["vocab"])
    if case["op"] == "loss":
        loss, lse = [], []
        for a in range(0, n, step):
            logits, t = s["hidden"][a:a + step].double() @ w.T, targets[a:a + step]
            z = torch.logsumexp(logits, dim=1)
            keep = (t != IGNORE).nonzero()[:, 0]
            one = torch.zeros_like(z)
            one[keep] = z[keep] - logits[keep, t[keep]]
            loss.append(one)
            lse.append(z)
        return torch.cat(loss), torch.cat(lse)
    d_hidden, d_weight = [], torch.zeros_like(w)
    for a in range(0, n, step):
        h, t = s["hidden"][a:a + step].double(), targets[a:a + step]
        p = torch.mm(h, w.T).sub_(s["lse"][a:a + step].double().unsqueeze(1)).exp_()
        keep = (t != IGNORE).nonzero()[:, 0]
        up = torch.zeros_like(s["lse"][a:a + step], dtype=torch.float64)
        up[keep] = s["grad"][a:a + step][keep].double()
        p[keep, t[keep]] -= 1.0
        p.mul_(up.unsqueeze(1))
        d_hidden.append(p @ w)
        d_weight.addmm_(p.T, h)
    return torch.cat(d_hidden), d_weight
