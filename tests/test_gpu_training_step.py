"""The cleartext operators together, as a training step takes them: ids into rows
of a table, norm, block, and three losses against the same table: targets, a
teacher's top logits, and pairs of sequences of which one is preferred.  Against
the same step in 64 bits by torch's autograd on the CPU, and captured in a graph.

Bounds: every operator's own are tested by themselves; a whole step is held to
the size of its gradients, 2^-12 of the largest of each parameter's in float32
(a chain of some ten operators, each within 2^-16 of its result's size: sums of up
to 2^7 terms), 2^-4 in bfloat16 (2^-8 a rounding, some ten of them in a row)."""
import pytest
import torch

import cleartext_ref as ref
from test_gpu_cleartext import DEV, ct, seeded  # noqa: F401

pytestmark = pytest.mark.gpu

PAIRS, LENGTH, ITEMS, WIDTH, HIDDEN, TOP = 6, 21, 150, 24, 40, 9
SCALE, BETA, WARMTH = 4.0, 0.5, 2.0


def batch(seed):
    gen = seeded(seed)
    ids = torch.randint(ITEMS, (PAIRS, 2, LENGTH), generator=gen)
    target = torch.randint(ITEMS, (PAIRS, 2, LENGTH), generator=gen)
    off = torch.arange(LENGTH) >= torch.randint(LENGTH // 2, LENGTH + 1, (PAIRS, 2, 1), generator=gen)
    ids[off], target[off] = -100, -100                      # padding
    taught = torch.rand(PAIRS, 2, LENGTH, ITEMS, generator=gen).argsort(-1)[..., :TOP]
    taught[off | (torch.rand(PAIRS, 2, LENGTH, generator=gen) < 0.2)] = -100
    logits = torch.randn(PAIRS, 2, LENGTH, TOP, generator=gen) * 2
    reference = torch.rand(PAIRS, 2, LENGTH, generator=gen) * 8
    return [t.to(DEV) for t in (ids, target, taught, logits, reference)]


def parameters(dtype):
    gen = seeded(0)
    made = [torch.randn(ITEMS, WIDTH, generator=gen) * 0.4, 1 + 0.1 * torch.randn(WIDTH, generator=gen), 0.1 * torch.randn(WIDTH, generator=gen),
            *(torch.randn(*s, generator=gen) * s[1] ** -0.5 for s in ((HIDDEN, WIDTH), (HIDDEN, WIDTH), (WIDTH, HIDDEN)))]
    return [p.to(dtype).to(DEV).requires_grad_() for p in made]


def step(ct, params, ids, target, taught, logits, reference):  # noqa: F811
    table, weight, bias, gate, up, down = params
    x = ct.embedding(ids, table, SCALE)
    x = ct.gated_mlp(ct.layer_norm(x, weight, bias), gate, up, down, ref.CUBIC)
    tokens = ct.cross_entropy(x, table, target, reduction="none")
    kept = (target != -100).sum()
    taken = tokens.sum() / kept
    return taken + ct.distillation(x, table, taught, logits, WARMTH) + ct.preference(tokens, reference, target, beta=BETA)


def plain(params, ids, target, taught, logits, reference):
    table, weight, bias, gate, up, down = params
    gone = ids == -100
    x = torch.where(gone[..., None], 0.0, table[ids.clamp(min=0)] * SCALE)
    x = torch.nn.functional.layer_norm(x, (WIDTH,), weight, bias)
    x = (ref.act(ref.CUBIC, x @ gate.T)[0] * (x @ up.T)) @ down.T
    z = x @ table.T
    tokens = torch.where(gone, 0.0, -torch.log_softmax(z, -1).gather(-1, target.clamp(min=0)[..., None])[..., 0])
    loss = tokens.sum() / (~gone).sum()
    there = taught != -100
    p = torch.softmax(torch.where(there, logits / WARMTH, -1e30), -1) * there
    q = torch.log_softmax(z / WARMTH, -1).gather(-1, taught.clamp(min=0))
    each = WARMTH ** 2 * torch.where(there, p * (p.clamp(min=1e-300).log() - q), 0.0).sum(-1)
    loss = loss + each.sum() / there.any(-1).sum()
    ratios = torch.where(gone, 0.0, reference - tokens).sum(-1)
    return loss - torch.nn.functional.logsigmoid(BETA * (ratios[:, 0] - ratios[:, 1])).mean()


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2.0 ** -12), (torch.bfloat16, 2.0 ** -4)])
def test_a_training_step(ct, dtype, tol):  # noqa: F811
    params, data = parameters(dtype), batch(1)
    loss = step(ct, params, *data)
    loss.backward()
    exact = [ref.d(p).requires_grad_() for p in params]
    want = plain(exact, *(t.cpu() if t.dtype == torch.int64 else ref.d(t) for t in data))
    want.backward()
    assert abs(loss.item() - want.item()) <= tol * (1 + abs(want.item()))
    for name, p, e in zip(("table", "weight", "bias", "gate", "up", "down"), params, exact, strict=True):
        assert p.grad.dtype == dtype
        worst = ((ref.d(p.grad) - e.grad).abs().max() / e.grad.abs().max()).item()
        assert worst <= tol, f"{name}: {worst}"


def test_a_captured_step_is_the_eager_one(ct):  # noqa: F811
    params, data = parameters(torch.bfloat16), batch(2)

    def run():
        for p in params:
            p.grad = None
        loss = step(ct, params, *data)
        return loss.detach(), torch.autograd.grad(loss, params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = run()
    for seed in (3, 4, 5):
        for old, new in zip(data, batch(seed), strict=True):
            old.copy_(new)
        with torch.no_grad():
            params[3].mul_(0.9)
        loss.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        eager = run()
        assert torch.equal(loss, eager[0])
        for a, b in zip(grads, eager[1], strict=True):
            assert torch.equal(a, b)
        del eager
