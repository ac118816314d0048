"""The work of the cleartext operators, as measured cases.

The model whose table, Linears and activations the backend evaluates under
encryption is trained in the clear on the same card.  A training step takes
each operator forward and backward; scoring in the clear takes single rows
forward.

Kinds:
  norm   layer norm of `rows` vectors of `width`
  mlp    the gated feed-forward block, width -> hidden -> width
  loss   softmax cross entropy of `rows` vectors against a table of `vocab`
         rows; `ignored` of them carry no target
`train`: forward and backward, gradients returned; else forward alone.
`dtype` is the type of the inputs and weights; `params` that of a norm's
weight and bias.
"""
import math

import torch

own = False

IGNORE = -100
EPS = 1e-5
# degree-3 activation of the encrypted model, lowest degree first
CUBIC = (-0.0320, 0.2195, 0.5706, 0.2048)


def norm(rows, width, dtype, params, train):
    return dict(kind="norm", rows=rows, width=width, dtype=dtype, params=params, train=train)


def mlp(rows, width, hidden, dtype, act, train):
    return dict(kind="mlp", rows=rows, width=width, hidden=hidden, dtype=dtype, act=act, train=train)


def loss(rows, width, vocab, ignored, dtype, train):
    return dict(kind="loss", rows=rows, width=width, vocab=vocab, ignored=ignored, dtype=dtype, train=train)


def listed():
    return [
        # one vector normalised while a model is scored: the smallest call, its launch counts
        dict(name="norm_one", **norm(1, 512, "bfloat16", "bfloat16", False)),
        # an ordinary training step's norm
        dict(name="norm_train", **norm(8192, 1024, "bfloat16", "bfloat16", True)),
        # a ragged batch of a width that no vector load divides, in the precision that the encrypted tables keep
        dict(name="norm_ragged", **norm(4097, 1001, "float32", "float32", True)),
        # the largest: long rows, many of them, weights kept in 32 bits
        dict(name="norm_large", **norm(32768, 4096, "bfloat16", "float32", True)),
        # one vector through the block: weights are read once, nothing else counts
        dict(name="mlp_one", **mlp(1, 1024, 4096, "bfloat16", "silu", False)),
        # a ragged batch, a hidden width that no tile or vector load divides
        dict(name="mlp_ragged", **mlp(1537, 1000, 2731, "float16", "gelu", True)),
        # the lookup's 416 outputs through a block with the encrypted model's activation, in 32 bits
        dict(name="mlp_cubic", **mlp(2048, 416, 512, "float32", "cubic", True)),
        # the largest block: matrix products
        dict(name="mlp_train", **mlp(8192, 2048, 8192, "bfloat16", "silu", True)),
        # the score of one candidate among 65536: the table is read once
        dict(name="loss_one", **loss(1, 1024, 65536, 0, "bfloat16", False)),
        # the 416 outputs against a table of an odd number of rows, in 32 bits
        dict(name="loss_ragged", **loss(1999, 416, 50021, 0, "float32", True)),
        # an ordinary training step, a seventh of its positions without a target
        dict(name="loss_train", **loss(4096, 1024, 65536, 585, "bfloat16", True)),
        # the largest: a step whose logits would take 2 GiB in 16 bits
        dict(name="loss_large", **loss(8192, 2048, 131072, 0, "bfloat16", True)),
    ]


def _spread(rng, low, high, step):
    """A size in [low, high], even on the logarithm; every second one a multiple of `step`."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5:
        n = -(-n // step) * step
    return max(low, min(high, n))


def draw(rng):
    kind = rng.choice(["norm", "mlp", "loss"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    train = rng.random() < 0.67
    if kind == "norm":
        return norm(_spread(rng, 1, 32768, 64), _spread(rng, 16, 4096, 16), dtype, rng.choice([dtype, "float32"]), train)
    if kind == "mlp":
        return mlp(_spread(rng, 1, 8192, 64), _spread(rng, 64, 2048, 16), _spread(rng, 64, 8192, 16), dtype,
                   rng.choice(["silu", "gelu", "cubic"]), train)
    rows = _spread(rng, 1, 8192, 64)
    return loss(rows, _spread(rng, 16, 2048, 16), _spread(rng, 256, 131072, 64), rng.randrange(0, rows // 2 + 1), dtype, train)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    rows, width = case["rows"], case["width"]

    def normal(*shape, std=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(to)

    s = dict(case=dict(case))
    if case["kind"] == "norm":
        par = getattr(torch, case["params"])
        # activations of a residual stream: a mean and a spread of their own in every row
        spread = torch.rand(rows, 1, generator=gen, device=dev) * 3 + 0.5
        mean = torch.randn(rows, 1, generator=gen, device=dev) * 0.5
        s["x"] = (torch.randn(rows, width, generator=gen, device=dev) * spread + mean).to(dtype)
        s["weight"] = (1 + 0.1 * torch.randn(width, generator=gen, device=dev)).to(par)
        s["bias"] = normal(width, std=0.1, to=par)
        if case["train"]:
            s["grad"] = normal(rows, width)
    elif case["kind"] == "mlp":
        hidden = case["hidden"]
        s["x"] = normal(rows, width)
        s["gate"] = normal(hidden, width, std=width ** -0.5)
        s["up"] = normal(hidden, width, std=width ** -0.5)
        s["down"] = normal(width, hidden, std=hidden ** -0.5)
        if case["train"]:
            s["grad"] = normal(rows, width)
    else:
        vocab = case["vocab"]
        s["table"] = normal(vocab, width, std=1.5 * width ** -0.5)
        # ids of a heavy-tailed frequency, and vectors that already lean towards them
        u = torch.rand(rows, generator=gen, device=dev, dtype=torch.float64)
        target = (torch.exp(u * math.log(vocab)) - 1).long().clamp_(0, vocab - 1)
        lean = torch.rand(rows, 1, generator=gen, device=dev) * 3
        s["x"] = (torch.randn(rows, width, generator=gen, device=dev) + lean * s["table"][target].float()).to(dtype)
        target[torch.randperm(rows, generator=gen, device=dev)[:case["ignored"]]] = IGNORE
        s["target"] = target
        if case["train"]:
            # the mean over the rows that have a target, each of a weight of its own; 16-bit floats are
            # trained with a scaled loss
            scale = 4096.0 if case["dtype"] == "float16" else 1.0
            kept = max(1, rows - case["ignored"])
            s["grad"] = (torch.rand(rows, generator=gen, device=dev) + 0.5) * (scale / kept)
    return s


def run(state):
    return _own(state) if own else _plain(state)


# ---- the framework's operators -------------------------------------------------


def _own(s):
    from helrm_amd import cleartext as ct
    case = s["case"]
    if case["kind"] == "norm":
        if not case["train"]:
            return ct.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        y, mean, rstd = ct.layer_norm_forward(s["x"], s["weight"], s["bias"], EPS)
        return (y,) + ct.layer_norm_backward(s["grad"], s["x"], s["weight"], mean, rstd)
    if case["kind"] == "mlp":
        act = CUBIC if case["act"] == "cubic" else case["act"]
        weights = (s["gate"], s["up"], s["down"])
        if not case["train"]:
            return ct.gated_mlp(s["x"], *weights, act)
        y, saved = ct.gated_mlp_forward(s["x"], *weights, act)
        return (y,) + ct.gated_mlp_backward(s["grad"], s["x"], *weights, saved, act)
    losses, lse = ct.cross_entropy_forward(s["x"], s["table"], s["target"], IGNORE)
    if not case["train"]:
        return losses, lse
    return (losses, lse) + ct.cross_entropy_backward(s["grad"], s["x"], s["table"], s["target"], lse, IGNORE)


# ---- the plain forms: elementary operations in 32 bits, rounded once ----------------


def _activation(name, g):
    """act(g) and its derivative."""
    if name == "silu":
        sig = 1 / (1 + torch.exp(-g))
        return g * sig, sig * (1 + g * (1 - sig))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    c0, c1, c2, c3 = CUBIC
    return ((c3 * g + c2) * g + c1) * g + c0, (3 * c3 * g + 2 * c2) * g + c1


def _plain(s):
    case = s["case"]
    x = s["x"].float()
    if case["kind"] == "norm":
        w = s["weight"].float()
        centred = x - x.mean(dim=1, keepdim=True)
        rstd = 1 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
        hat = centred * rstd
        y = (hat * w + s["bias"].float()).to(s["x"].dtype)
        if not case["train"]:
            return y
        dy = s["grad"].float()
        dhat = dy * w
        dx = rstd * (dhat - dhat.mean(dim=1, keepdim=True) - hat * (dhat * hat).mean(dim=1, keepdim=True))
        par = s["weight"].dtype
        return y, dx.to(s["x"].dtype), (dy * hat).sum(dim=0).to(par), dy.sum(dim=0).to(par)
    if case["kind"] == "mlp":
        dtype = s["x"].dtype
        gate, up, down = s["gate"].float(), s["up"].float(), s["down"].float()
        g, u = x @ gate.t(), x @ up.t()
        a, da = _activation(case["act"], g)
        h = a * u
        y = (h @ down.t()).to(dtype)
        if not case["train"]:
            return y
        dy = s["grad"].float()
        dh = dy @ down
        dg, du = dh * u * da, dh * a
        return (y, (dg @ gate + du @ up).to(dtype), (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype), (dy.t() @ h).to(dtype))
    table, target = s["table"].float(), s["target"]
    kept = target != IGNORE
    at = torch.where(kept, target, 0)
    logits = x @ table.t()
    top = logits.amax(dim=1)
    lse = top + torch.log(torch.exp(logits - top[:, None]).sum(dim=1))
    losses = torch.where(kept, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    lse = torch.where(kept, lse, 0.0)
    if not case["train"]:
        return losses, lse
    dlogits = torch.exp(logits - lse[:, None])
    del logits
    dlogits.scatter_add_(1, at[:, None], torch.full_like(dlogits[:, :1], -1.0))
    dlogits = torch.where(kept[:, None], dlogits, 0.0) * s["grad"][:, None]
    dtype = s["x"].dtype
    return losses, lse, (dlogits @ table).to(dtype), (dlogits.t() @ x).to(dtype)


# ---- the definitions in 64 bits ---------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "norm":
        var, mu = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        inv = torch.rsqrt(var + EPS)
        w = s["weight"].double()
        y = torch.addcmul(s["bias"].double(), (x - mu) * inv, w)
        if not case["train"]:
            return y
        dy = s["grad"].double()
        t = dy * w
        # through the mean and through the variance, one at a time
        dvar = -0.5 * inv ** 3 * torch.sum(t * (x - mu), dim=1, keepdim=True)
        dmu = -inv * torch.sum(t, dim=1, keepdim=True)
        dx = t * inv + dvar * 2 * (x - mu) / case["width"] + dmu / case["width"]
        dw = torch.einsum("tn,tn->n", dy, (x - mu) * inv)
        return y, dx, dw, torch.ones(case["rows"], dtype=torch.float64, device=dy.device) @ dy
    if case["kind"] == "mlp":
        wg, wu, wd = (s[k].double() for k in ("gate", "up", "down"))
        g = torch.mm(x, wg.T).requires_grad_()
        if case["act"] == "silu":
            act = g * torch.sigmoid(g)
        elif case["act"] == "gelu":
            act = g * torch.special.ndtr(g)
        else:
            act = sum(c * g ** k for k, c in enumerate(CUBIC))
        u = torch.mm(x, wu.T)
        h = act.detach() * u
        y = torch.mm(h, wd.T)
        if not case["train"]:
            return y
        dy = s["grad"].double()
        dh = torch.mm(dy, wd)
        (dg,) = torch.autograd.grad(act, g, dh * u)
        du = dh * act.detach()
        return y, torch.mm(dg, wg) + torch.mm(du, wu), torch.mm(dg.T, x), torch.mm(du.T, x), torch.mm(dy.T, h)
    # one block of rows after another, so that the logits fit
    rows, vocab, width = case["rows"], case["vocab"], case["width"]
    table = s["table"].double()
    losses = torch.zeros(rows, dtype=torch.float64, device=x.device)
    norms = torch.zeros_like(losses)
    dx, dtable = torch.zeros_like(x), torch.zeros_like(table)
    for row in range(0, rows, 1024):
        part = slice(row, min(rows, row + 1024))
        idx = torch.nonzero(s["target"][part] != IGNORE)[:, 0] + row
        if not len(idx):
            continue
        tgt = s["target"][idx]
        logp = torch.log_softmax(torch.mm(x[idx], table.T), dim=1)
        pick = logp[torch.arange(len(idx), device=x.device), tgt]
        losses[idx] = -pick
        norms[idx] = torch.sum(x[idx] * table[tgt], dim=1) - pick
        if case["train"]:
            prob = logp.exp_()
            prob[torch.arange(len(idx), device=x.device), tgt] -= 1
            prob *= s["grad"][idx].double()[:, None]
            dx[idx] = torch.mm(prob, table)
            dtable += torch.mm(prob.T, x[idx])
        del logp
    return (losses, norms, dx, dtable) if case["train"] else (losses, norms)


def work(case):
    rows, width, size = case["rows"], case["width"], {"float32": 4}.get(case["dtype"], 2)
    if case["kind"] == "norm":
        par = {"float32": 4}.get(case["params"], 2)
        if not case["train"]:
            return {"bytes": 2 * rows * width * size + 2 * width * par, "flops": 8 * rows * width}
        return {"bytes": 4 * rows * width * size + 4 * width * par, "flops": 20 * rows * width}
    if case["kind"] == "mlp":
        weights, data = 3 * width * case["hidden"] * size, rows * width * size
        if not case["train"]:
            return {"bytes": weights + 2 * data, "flops": 6 * rows * width * case["hidden"]}
        return {"bytes": 2 * weights + 4 * data, "flops": 18 * rows * width * case["hidden"]}
    kept, vocab = rows - case["ignored"], case["vocab"]
    if not case["train"]:
        return {"bytes": (vocab + kept) * width * size + 16 * rows, "flops": 2 * kept * vocab * width}
    return {"bytes": 2 * (vocab + rows) * width * size + 20 * rows, "flops": 6 * kept * vocab * width}
