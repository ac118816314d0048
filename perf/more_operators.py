"""The work of the cleartext operators that feed and judge a model, as measured cases.

A model whose table is looked up under encryption is trained in the clear:
its ids become rows of the table, and besides the targets of a cross entropy it
learns from a larger model's answers and from pairs of answers of which one is
preferred.

Kinds:
  embed   rows of a table for `tokens` ids, `ignored` of them without one,
          times `scale`; the table's gradient from the rows'
  teach   distillation: `rows` vectors against a table of `vocab` rows, a
          teacher's `top` logits and their ids for each; a row has from 1 to
          `top` of them where `ragged`, and `ignored` rows have none
  prefer  pairs of sequences of token losses, up to `length` tokens each, with
          those of a reference model; in padded rows, or one behind the other
          with `packed`
`train`: forward and backward, gradients returned; else forward alone.
`dtype` is the type of the vectors and the table, `teacher` that of a teacher's
logits; token losses are float32.
"""
import math

import torch

own = False

IGNORE = -100


def embed(tokens, width, vocab, ignored, scale, dtype, train):
    return dict(kind="embed", tokens=tokens, width=width, vocab=vocab, ignored=ignored, scale=scale, dtype=dtype, train=train)


def teach(rows, width, vocab, top, ragged, ignored, temperature, dtype, teacher, train):
    return dict(kind="teach", rows=rows, width=width, vocab=vocab, top=top, ragged=ragged, ignored=ignored, temperature=temperature,
                dtype=dtype, teacher=teacher, train=train)


def prefer(pairs, length, packed, reference, loss, smoothing, average, train):
    return dict(kind="prefer", pairs=pairs, length=length, packed=packed, reference=reference, loss=loss, smoothing=smoothing,
                average=average, train=train)


def listed():
    return [
        # one id while a model is scored: the smallest call, its launch counts
        dict(name="embed_one", **embed(1, 512, 65536, 0, 1.0, "bfloat16", False)),
        # the 26 categorical ids of 2048 samples, tables of 16 columns one behind the other, in 32 bits
        dict(name="embed_narrow", **embed(26 * 2048, 16, 26 * 2000, 0, 1.0, "float32", True)),
        # a ragged batch of a width that no vector load divides, a tenth of it padding
        dict(name="embed_ragged", **embed(4099, 1001, 50021, 410, 31.64, "float16", True)),
        # an ordinary training step: far more rows in the table than ids
        dict(name="embed_train", **embed(16384, 1024, 65536, 0, 32.0, "bfloat16", True)),
        # the largest: long rows, as many ids as rows, the commonest id several thousand times
        dict(name="embed_large", **embed(131072, 2048, 131072, 0, 1.0, "bfloat16", True)),
        # how far one vector's scores are from a teacher's: the table is read once
        dict(name="teach_one", **teach(1, 1024, 65536, 32, False, 0, 1.0, "bfloat16", "float32", False)),
        # the lookup's 416 outputs in 32 bits, a teacher cut at a probability: 1 to 17 logits a row
        dict(name="teach_ragged", **teach(1999, 416, 50021, 17, True, 100, 2.0, "float32", "float32", True)),
        # an ordinary training step, a seventh of its positions without a teacher's answer
        dict(name="teach_train", **teach(4096, 1024, 65536, 64, False, 585, 1.5, "bfloat16", "bfloat16", True)),
        # the largest: a step whose logits would take 2 GiB in 16 bits
        dict(name="teach_large", **teach(8192, 2048, 131072, 64, False, 0, 2.0, "bfloat16", "float32", True)),
        # one pair scored
        dict(name="prefer_one", **prefer(1, 200, False, True, "logistic", 0.0, False, False)),
        # an ordinary training step of packed answers
        dict(name="prefer_packed", **prefer(128, 1500, True, True, "logistic", 0.1, False, True)),
        # the largest: long answers in padded rows
        dict(name="prefer_large", **prefer(512, 8192, False, True, "logistic", 0.0, False, True)),
    ]


def _spread(rng, low, high, step):
    """A size in [low, high], even on the logarithm; every second one a multiple of `step`."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5:
        n = -(-n // step) * step
    return max(low, min(high, n))


def draw(rng):
    kind = rng.choice(["embed", "teach", "prefer"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    train = rng.random() < 0.67
    if kind == "embed":
        tokens = _spread(rng, 1, 131072, 64)
        width = _spread(rng, 16, 1024 if dtype == "float32" else 2048, 16)
        return embed(tokens, width, _spread(rng, 256, 131072, 64), rng.randrange(0, tokens // 2 + 1),
                     rng.choice([1.0, width ** 0.5]), dtype, train)
    if kind == "teach":
        rows = _spread(rng, 1, 8192, 64)
        # (a float32 product is several of 16 bits)
        width = _spread(rng, 16, 512 if dtype == "float32" else 2048, 16)
        vocab = _spread(rng, 256, 65536 if dtype == "float32" else 131072, 64)
        return teach(rows, width, vocab, _spread(rng, 1, 128, 8), rng.random() < 0.5, rng.randrange(0, rows // 2 + 1),
                     rng.choice([1.0, 2.0, rng.uniform(0.5, 4.0)]), dtype, rng.choice([dtype, "float32"]), train)
    loss = rng.choice(["logistic", "logistic", "hinge"])
    return prefer(_spread(rng, 1, 512, 8), _spread(rng, 1, 8192, 64), rng.random() < 0.5, rng.random() < 0.75, loss,
                  rng.choice([0.0, 0.1]) if loss == "logistic" else 0.0, rng.random() < 0.3, train)


def _margin(case):
    """beta and the margin of a pair's loss: without a reference the ratios are whole log probabilities."""
    return (2.0 if case["average"] else 0.1), (0.0 if case["reference"] else 0.5)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))

    def normal(*shape, std=1.0, to=torch.float32):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(to)

    def common(*shape, n):
        """Ids below n of a heavy-tailed frequency."""
        u = torch.rand(*shape, generator=gen, device=dev, dtype=torch.float64)
        return (torch.exp(u * math.log(n)) - 1).long().clamp_(0, n - 1)

    def some(n, k):
        return torch.randperm(n, generator=gen, device=dev)[:k]

    s = dict(case=dict(case))
    if case["kind"] == "embed":
        dtype = getattr(torch, case["dtype"])
        tokens, width, vocab = case["tokens"], case["width"], case["vocab"]
        s["table"] = normal(vocab, width, std=width ** -0.5, to=dtype)
        s["ids"] = common(tokens, n=vocab)
        s["ids"][some(tokens, case["ignored"])] = IGNORE
        if case["train"]:
            s["grad"] = normal(tokens, width, to=dtype)
    elif case["kind"] == "teach":
        dtype = getattr(torch, case["dtype"])
        rows, width, vocab, top = (case[k] for k in ("rows", "width", "vocab", "top"))
        s["table"] = normal(vocab, width, std=1.5 * width ** -0.5, to=dtype)
        # different ids in a row, the common ones oftener, in the order of falling logits
        ids = common(rows, top, n=vocab - top + 1).sort(dim=1).values + torch.arange(top, device=dev)
        ids = ids.gather(1, torch.rand(rows, top, generator=gen, device=dev).argsort(dim=1))
        step = -torch.log(torch.rand(rows, top, generator=gen, device=dev) + 1e-6)
        s["logits"] = (12 - step.cumsum(dim=1) * (8 / top)).to(getattr(torch, case["teacher"]))
        # vectors that already lean towards the teacher's answer
        lean = torch.rand(rows, 1, generator=gen, device=dev) * 3
        s["x"] = (normal(rows, width) + lean * s["table"][ids[:, 0]].float()).to(dtype)
        if case["ragged"]:
            there = torch.randint(1, top + 1, (rows, 1), generator=gen, device=dev)
            ids = torch.where(torch.arange(top, device=dev) < there, ids, IGNORE)
        ids[some(rows, case["ignored"])] = IGNORE
        s["ids"] = ids
        if case["train"]:
            # the mean over the rows that have a teacher, each of a weight of its own; 16-bit floats are
            # trained with a scaled loss
            scale = 4096.0 if case["dtype"] == "float16" else 1.0
            kept = max(1, rows - case["ignored"])
            s["grad"] = (torch.rand(rows, generator=gen, device=dev) + 0.5) * (scale / kept)
    else:
        pairs, length = case["pairs"], case["length"]
        # answers from an eighth of the longest on, evenly (so that a batch's size is the case's), behind a question that
        # is the same for both and counts in neither
        low = (length + 7) // 8
        lengths = low + torch.arange(2 * pairs, device=dev) * (length - low) // max(1, 2 * pairs - 1)
        lengths = lengths[some(2 * pairs, 2 * pairs)].view(pairs, 2)
        asked = torch.randint(0, (length + 7) // 8, (pairs, 1), generator=gen, device=dev).expand(pairs, 2)
        at = torch.arange(length, device=dev)
        counts = (at >= asked[..., None]) & (at < lengths[..., None])
        target = torch.where(counts, torch.randint(0, 65536, (pairs, 2, length), generator=gen, device=dev), IGNORE)
        token = -torch.log(torch.rand(pairs, 2, length, generator=gen, device=dev) + 1e-6)
        losses = torch.where(counts, 1.8 * token, 0.0)
        reference = torch.where(counts, (losses + normal(pairs, 2, length, std=0.3)).clamp_(min=0), 0.0)
        s["target"], s["losses"], s["reference"] = target, losses, reference
        if case["packed"]:
            inside = (at < lengths[..., None])
            for k in ("target", "losses", "reference"):
                s[k] = s[k][inside]
            s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), lengths.reshape(-1).cumsum(0)])
        else:
            s["offsets"] = None
        if not case["reference"]:
            s["reference"] = None
        if case["train"]:
            s["grad"] = (torch.rand(pairs, generator=gen, device=dev) + 0.5) / pairs
    return s


def run(state):
    return _own(state) if own else _plain(state)


# ---- the framework's operators -------------------------------------------------


def _own(s):
    from helrm_amd import cleartext as ct
    case = s["case"]
    if case["kind"] == "embed":
        y = ct.embedding_forward(s["ids"], s["table"], case["scale"], IGNORE)
        if not case["train"]:
            return y
        return y, ct.embedding_backward(s["grad"], s["ids"], case["vocab"], case["scale"], IGNORE)
    if case["kind"] == "teach":
        t = case["temperature"]
        losses, lse, saved = ct.distillation_forward(s["x"], s["table"], s["ids"], s["logits"], t, IGNORE)
        if not case["train"]:
            return losses, lse
        return (losses, lse) + ct.distillation_backward(s["grad"], s["x"], s["table"], s["ids"], lse, saved, t, IGNORE)
    beta, margin = _margin(case)
    values, ratios, slopes = ct.preference_forward(s["losses"], s["reference"], s["target"], s["offsets"], beta, margin, case["loss"],
                                                   case["smoothing"], case["average"], IGNORE)
    if not case["train"]:
        return values, ratios
    return values, ratios, ct.preference_backward(s["grad"], s["losses"], slopes, s["target"], s["offsets"], IGNORE)


# ---- the plain forms: elementary operations in 32 bits (the sums over tokens in 64), rounded once ----


def _plain(s):
    case = s["case"]
    if case["kind"] == "embed":
        table, ids, scale = s["table"], s["ids"], case["scale"]
        kept = ids != IGNORE
        at = torch.where(kept, ids, 0)
        y = torch.where(kept[:, None], table[at].float() * scale, 0.0).to(table.dtype)
        if not case["train"]:
            return y
        dy = torch.where(kept[:, None], s["grad"].float(), 0.0)
        dtable = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
        dtable.index_add_(0, at, dy)
        return y, (dtable * scale).to(table.dtype)
    if case["kind"] == "teach":
        t = case["temperature"]
        x, table, ids = s["x"].float(), s["table"].float(), s["ids"]
        there = ids != IGNORE
        kept = there.any(dim=1)
        at = torch.where(there, ids, 0)
        teacher = torch.where(there, s["logits"].float() / t, -math.inf)
        teacher = torch.where(kept[:, None], teacher, 0.0)
        teacher = teacher - teacher.amax(dim=1, keepdim=True)
        logp = teacher - torch.log(torch.exp(teacher).sum(dim=1, keepdim=True))
        p = torch.where(there, torch.exp(logp), 0.0)
        logits = x @ table.t()
        logits /= t
        best = logits.amax(dim=1)
        lse = best + torch.log(torch.exp(logits - best[:, None]).sum(dim=1))
        logq = logits.gather(1, at) - lse[:, None]
        losses = torch.where(there, p * (logp - logq), 0.0).sum(dim=1) * (t * t)
        out = losses, torch.where(kept, lse, 0.0)
        if not case["train"]:
            return out
        dlogits = torch.exp(logits - lse[:, None])
        del logits
        dlogits.scatter_add_(1, at, -p)
        dlogits = torch.where(kept[:, None], dlogits, 0.0) * (s["grad"] * t)[:, None]
        dtype = s["x"].dtype
        return out + ((dlogits @ table).to(dtype), (dlogits.t() @ x).to(dtype))
    counts = s["target"] != IGNORE
    token = -s["losses"].double() if s["reference"] is None else s["reference"].double() - s["losses"].double()
    token = torch.where(counts, token, 0.0)
    if s["offsets"] is None:
        ratios, number = token.sum(dim=2), counts.sum(dim=2)
    else:
        lengths = s["offsets"][1:] - s["offsets"][:-1]
        sequence = torch.repeat_interleave(torch.arange(2 * case["pairs"], device=lengths.device), lengths, output_size=token.numel())
        ratios = torch.zeros(2 * case["pairs"], dtype=torch.float64, device=lengths.device).index_add_(0, sequence, token).view(-1, 2)
        number = torch.zeros(2 * case["pairs"], dtype=torch.int64, device=lengths.device).index_add_(0, sequence, counts.long()).view(-1, 2)
    each = 1.0 / number.clamp(min=1) if case["average"] else torch.ones_like(ratios)
    ratios = ratios * each
    beta, margin = _margin(case)
    m = beta * (ratios[:, 0] - ratios[:, 1]) - margin
    if case["loss"] == "logistic":
        e = case["smoothing"]
        tail = torch.log(1 + torch.exp(-m.abs()))
        values = (1 - e) * (tail + (-m).clamp(min=0)) + e * (tail + m.clamp(min=0))
        slope = -(1 - e) / (1 + torch.exp(m)) + e / (1 + torch.exp(-m))
    else:
        values = (1 - m).clamp(min=0)
        slope = torch.where(m < 1, -1.0, 0.0).double()
    any_token = number.sum(dim=1) > 0
    values = torch.where(any_token, values, 0.0)
    if not case["train"]:
        return values.float(), ratios.float()
    # of each token's loss: the preferred sequence's ratio falls with it
    d = (s["grad"].double() * slope * beta)[:, None] * each * torch.tensor([-1.0, 1.0], dtype=torch.float64, device=m.device)
    d = d[..., None] if s["offsets"] is None else d.reshape(-1)[sequence]
    return values.float(), ratios.float(), torch.where(counts, d, 0.0).float()


# ---- the definitions in 64 bits ---------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embed":
        idx = torch.nonzero(s["ids"] != IGNORE)[:, 0]
        rows = s["ids"][idx]
        y = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device=rows.device)
        y[idx] = s["table"][rows].double() * case["scale"]
        if not case["train"]:
            return y
        order = rows.argsort(stable=True)
        dtable = torch.zeros(s["table"].shape, dtype=torch.float64, device=rows.device)
        # the products of a few columns at a time with the ids' incidence, as running sums over sorted ids
        ends = torch.searchsorted(rows[order], torch.arange(case["vocab"] + 1, device=rows.device))
        for c in range(0, case["width"], 256):
            run_ = torch.zeros(len(idx) + 1, min(256, case["width"] - c), dtype=torch.float64, device=rows.device)
            torch.cumsum(s["grad"][idx[order], c:c + 256].double(), dim=0, out=run_[1:])
            dtable[:, c:c + 256] = (run_[ends[1:]] - run_[ends[:-1]]) * case["scale"]
        return y, dtable
    if case["kind"] == "teach":
        rows, vocab, width, t = case["rows"], case["vocab"], case["width"], case["temperature"]
        x, table = s["x"].double(), s["table"].double()
        losses = torch.zeros(rows, dtype=torch.float64, device=x.device)
        norms = torch.zeros_like(losses)
        dx, dtable = torch.zeros_like(x), torch.zeros_like(table)
        have = (s["ids"] != IGNORE)
        for row in range(0, rows, 1024):
            idx = torch.nonzero(have[row:row + 1024].any(dim=1))[:, 0] + row
            if not len(idx):
                continue
            z = torch.mm(x[idx], table.T) / t
            norms[idx] = torch.logsumexp(z, dim=1)
            logq = z.sub_(norms[idx][:, None])
            # the teacher's distribution over the whole table
            low = torch.full_like(s["logits"][idx].double(), -math.inf)
            logp = torch.log_softmax(torch.where(have[idx], s["logits"][idx].double() / t, low), dim=1)
            dense = torch.zeros_like(logq)
            for j in range(case["top"]):
                at = torch.nonzero(have[idx, j])[:, 0]
                v = s["ids"][idx[at], j]
                losses[idx[at]] += t * t * torch.exp(logp[at, j]) * (logp[at, j] - logq[at, v])
                dense[at, v] += torch.exp(logp[at, j])
            if case["train"]:
                d = (logq.exp_() - dense) * (t * s["grad"][idx].double())[:, None]
                dx[idx] = torch.mm(d, table)
                dtable += torch.mm(d.T, x[idx])
            del z, logq, dense
        return (losses, norms, dx, dtable) if case["train"] else (losses, norms)
    beta, margin = _margin(case)
    counts = s["target"] != IGNORE
    rho = -s["losses"].double()
    if s["reference"] is not None:
        rho = rho + s["reference"].double()
    rho = (rho * counts).requires_grad_()
    if s["offsets"] is None:
        sums, number = rho.sum(-1), counts.sum(-1)
    else:
        zero = torch.zeros(1, dtype=torch.float64, device=rho.device)
        run_ = torch.cat([zero, rho.cumsum(0)])
        sums = (run_[s["offsets"][1:]] - run_[s["offsets"][:-1]]).view(-1, 2)
        number = torch.cat([zero, counts.double().cumsum(0)])
        number = (number[s["offsets"][1:]] - number[s["offsets"][:-1]]).view(-1, 2)
    if case["average"]:
        sums = sums / number.clamp(min=1)
    m = beta * (sums[:, 0] - sums[:, 1]) - margin
    if case["loss"] == "logistic":
        values = -(1 - case["smoothing"]) * torch.nn.functional.logsigmoid(m) - case["smoothing"] * torch.nn.functional.logsigmoid(-m)
    else:
        values = torch.relu(1 - m)
    values = values * (number.sum(1) > 0)
    if not case["train"]:
        return values.detach(), sums.detach()
    (d,) = torch.autograd.grad(values, rho, s["grad"].double())
    return values.detach(), sums.detach(), -d * counts


def work(case):
    if case["kind"] == "embed":
        size = {"float32": 4}.get(case["dtype"], 2)
        tokens, kept, width, vocab = case["tokens"], case["tokens"] - case["ignored"], case["width"], case["vocab"]
        # a row that several ids name is read once: no more rows than the table has
        once = {"bytes": (min(kept, vocab) + tokens) * width * size + 8 * tokens, "flops": kept * width}
        if not case["train"]:
            return once
        return {"bytes": once["bytes"] + (kept + vocab) * width * size + 8 * tokens, "flops": 3 * kept * width}
    if case["kind"] == "teach":
        size, held = {"float32": 4}.get(case["dtype"], 2), {"float32": 4}.get(case["teacher"], 2)
        rows, kept, width, vocab, top = case["rows"], case["rows"] - case["ignored"], case["width"], case["vocab"], case["top"]
        teacher = rows * top * (8 + held)
        if not case["train"]:
            return {"bytes": (vocab + kept) * width * size + teacher + 8 * rows, "flops": 2 * kept * vocab * width}
        return {"bytes": 2 * (vocab + rows) * width * size + teacher + 12 * rows, "flops": 6 * kept * vocab * width}
    # sequences are from an eighth of the longest to all of it, nine sixteenths at the mean; padded rows are read whole
    tokens = 2 * case["pairs"] * case["length"]
    if case["packed"]:
        tokens = tokens * 9 // 16
    each = 4 + 8 + (4 if case["reference"] else 0)
    return {"bytes": tokens * (each + (4 if case["train"] else 0)) + 20 * case["pairs"], "flops": tokens * (4 if case["train"] else 3)}
