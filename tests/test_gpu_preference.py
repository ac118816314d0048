"""The loss of pairs of sequences against a plain 64-bit implementation: padded
rows and sequences in a line, lengths from none to several shares, tokens that
do not count, infinities and NaN, strides, streams and graphs.

Bounds: sums are of 64 bits, so a result is within its own rounding of the
formula's, and what cancels in it of the sums' size times 2^-48 (2^5 terms'
roundings at the most in 2^-53); a gradient has three roundings."""
import pytest
import torch

import cleartext_ref as ref
from test_gpu_cleartext import DEV, F32, ct, seeded  # noqa: F401

pytestmark = pytest.mark.gpu

IGNORE = -100
F64 = 2.0 ** -48


def f32(v):
    return float(torch.tensor(v))     # as the entry point takes it


def sequences(losses, reference, target, offsets, ignore):
    """(token differences, whether they count) of each sequence."""
    losses = ref.d(losses)
    d = (0.0 if reference is None else ref.d(reference)) - losses
    counts = torch.ones_like(losses, dtype=torch.bool) if target is None else target.cpu() != ignore
    if offsets is None:
        return list(zip(d.flatten(0, -2), counts.flatten(0, -2)))
    o = offsets.cpu().tolist()
    return [(d[a:b], counts[a:b]) for a, b in zip(o, o[1:])]


def plain(losses, reference, target, offsets, beta, margin, kind, smoothing, average, ignore):
    """values, ratios, slopes, and the sums' sizes."""
    s = sequences(losses, reference, target, offsets, ignore)
    r = torch.tensor([d[c].sum().item() for d, c in s], dtype=torch.float64).view(-1, 2)
    size = torch.tensor([d[c].abs().sum().item() for d, c in s], dtype=torch.float64).view(-1, 2)
    n = torch.tensor([int(c.sum()) for _, c in s], dtype=torch.float64).view(-1, 2)
    each = 1 / n.clamp(min=1) if average else torch.ones_like(n)
    r, size = r * each, size * each
    m = beta * (r[:, 0] - r[:, 1]) - margin
    if kind == "hinge":
        v, g = (1 - m).clamp(min=0), torch.where(m.isnan(), m, -(m < 1).double())
    else:
        v, g = torch.nn.functional.softplus(-m) * (1 - smoothing), -torch.sigmoid(-m) * (1 - smoothing)
        if smoothing:
            v, g = v + smoothing * torch.nn.functional.softplus(m), g + smoothing * torch.sigmoid(m)
    v = torch.where(n.sum(1) > 0, v, 0.0)
    return v, r, torch.stack([-g * beta * each[:, 0], g * beta * each[:, 1]], 1), size


def pref_check(ct, losses, reference=None, target=None, offsets=None, beta=0.1, margin=0.0, kind="logistic", smoothing=0.0, average=False,  # noqa: F811
               ignore=IGNORE):
    beta, margin, smoothing = f32(beta), f32(margin), f32(smoothing)
    values, ratios, slopes = ct.preference_forward(losses, reference, target, offsets, beta, margin, kind, smoothing, average, ignore)
    v, r, g, size = plain(losses, reference, target, offsets, beta, margin, kind, smoothing, average, ignore)
    lead = losses.shape[:-2] if offsets is None else (offsets.shape[0] // 2,)
    assert values.shape == lead and ratios.shape == slopes.shape == (*lead, 2)
    cut = (size.sum(1) * abs(beta) + abs(margin) + 1) * F64
    ref.check(ratios.view(-1, 2), r, r.abs() * F32 + size * F64 + 1e-45, 1.0, "ratios")
    ref.check(values.view(-1), v, v.abs() * (F32 + F64) + cut + 1e-45, 1.0, "values")
    ref.check(slopes.view(-1, 2), g, g.abs() * (F32 + F64) + abs(beta) * cut[:, None] + 1e-45, 1.0, "slopes")
    grad = (torch.rand(lead, generator=seeded(3)) + 0.5).to(DEV)
    d = ct.preference_backward(grad, losses, slopes, target, offsets, ignore)
    assert d.shape == losses.shape
    want = torch.zeros(losses.shape, dtype=torch.float64)
    g = g * ref.d(grad).view(-1, 1)
    if offsets is None:
        want += g.view(*lead, 2, 1)
    else:
        o = offsets.cpu().tolist()
        for k, (a, b) in enumerate(zip(o, o[1:])):
            want[a:b] = g.view(-1)[k]
    if target is not None:
        want[target.cpu() == ignore] = 0
    scale = abs(beta) * ref.d(grad).max().item() * cut.max().item() if len(cut) else 0
    ref.check(d, want, want.abs() * 3 * F32 + scale + 1e-44, 1.0, "dlosses")
    assert torch.equal(ct.preference_backward(grad, losses, slopes, target, offsets, ignore), d)
    return values, ratios, slopes, d


def batch(gen, pairs, length, counted=0.8):
    losses = -torch.log(torch.rand(pairs, 2, length, generator=gen) + 1e-6) * 1.8
    reference = losses + 0.3 * torch.randn(pairs, 2, length, generator=gen)
    target = torch.where(torch.rand(pairs, 2, length, generator=gen) < counted, torch.randint(0, 1000, (pairs, 2, length), generator=gen), IGNORE)
    return losses.to(DEV), reference.to(DEV), target.to(DEV)


FORMS = [dict(), dict(kind="hinge"), dict(smoothing=0.1, margin=0.5), dict(average=True, beta=2.0), dict(kind="hinge", margin=-1.0, average=True, beta=5.0),
         dict(smoothing=1.0), dict(beta=0.0), dict(beta=-0.3)]


@pytest.mark.parametrize("pairs,length", [(0, 5), (1, 0), (3, 1), (1, 200), (7, 65), (5, 1025), (300, 3), (257, 16), (257, 17), (257, 64), (300, 65), (256, 256), (256, 257), (2, 4097), (1, 40001),
                                          (3, 16385), (40, 9000)])
def test_preference(ct, pairs, length):  # noqa: F811
    gen = seeded(pairs + length)
    losses, reference, target = batch(gen, pairs, length)
    for k, form in enumerate(FORMS):
        pref_check(ct, losses, reference if k % 3 else None, target if k % 2 else None, **form)


@pytest.mark.parametrize("pairs,mean", [(0, 4), (1, 300), (5, 1), (7, 90), (300, 5), (300, 40), (300, 200), (100, 1200), (2, 30000), (33, 3000)])
def test_sequences_in_a_line(ct, pairs, mean):  # noqa: F811
    gen = seeded(pairs + mean)
    lengths = (torch.rand(2 * pairs, generator=gen) ** 3 * 4 * mean).long()       # many short, a few long; some without tokens
    lead, tail = (3, 5) if mean != 90 else (0, 0)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]) + lead
    n = int(offsets[-1]) + tail
    losses, reference, target = (t.reshape(-1)[:n].contiguous() for t in batch(gen, 1, n))
    for k, form in enumerate(FORMS):
        *_, d = pref_check(ct, losses, reference if k % 3 else None, target if k % 2 else None, offsets.to(DEV), **form)
        assert not d[:lead].any() and not d[n - tail:].any()


def test_rows_and_a_line_agree(ct):  # noqa: F811
    losses, reference, target = batch(seeded(1), 20, 300)
    rows = ct.preference_forward(losses, reference, target, beta=0.2)
    line = ct.preference_forward(losses.view(-1), reference.view(-1), target.view(-1), torch.arange(0, 41 * 300, 300, device=DEV), beta=0.2)
    for a, b in zip(rows, line, strict=True):
        ref.check(a, ref.d(b), ref.d(b).abs(), 2 * F32, "rows and a line")


@pytest.mark.parametrize("pairs,length", [(4, 30), (300, 30), (3, 20000)])
def test_what_does_not_count_reaches_nothing(ct, pairs, length):  # noqa: F811
    losses, reference, target = batch(seeded(pairs), pairs, length, 0.5)
    target[0], target[1, 0], target[2, 1] = IGNORE, IGNORE, IGNORE
    first = pref_check(ct, losses, reference, target)
    gone = target == IGNORE
    losses[gone], reference[gone] = float("nan"), float("-inf")
    values, ratios, slopes = ct.preference_forward(losses, reference, target)
    d = ct.preference_backward((torch.rand(pairs, generator=seeded(3)) + 0.5).to(DEV), losses, slopes, target)
    for a, b in zip(first, (values, ratios, slopes, d), strict=True):
        assert torch.equal(a, b)
    assert values[0] == 0 and not d[gone].any()
    # a pair without tokens is left out of the mean, one with a single sequence is not
    total = ct.preference(losses, reference, target)
    ref.check(total, ref.d(values).sum() / (pairs - 1), ref.d(values).sum() / (pairs - 1), 2 * F32, "mean")
    assert ct.preference(losses, reference, torch.full_like(target, IGNORE)).item() == 0


def test_infinities_and_nan(ct):  # noqa: F811
    losses, reference, _ = batch(seeded(2), 6, 50)
    inf = float("inf")
    losses[0, 0, 3] = inf          # the preferred one is impossible
    losses[1, 1, 7] = inf          # the other one is
    losses[2, 0, 1], losses[2, 1, 1] = inf, inf
    losses[3, 0, 5] = float("nan")
    reference[4, 1, 2] = -inf
    for kind in ("logistic", "hinge"):
        values, ratios, slopes = ct.preference_forward(losses, reference, beta=0.1, kind=kind)
        assert values[0] == inf and values[1] == 0 and torch.isnan(values[2:4]).all() and values[4] == 0 and torch.isfinite(values[5])
        assert ratios[0, 0] == -inf and ratios[1, 1] == -inf and torch.isnan(ratios[3, 0]) and torch.isfinite(ratios[5]).all()
        assert slopes[0].tolist() == [f32(0.1), -f32(0.1)] and not slopes[1].any() and torch.isnan(slopes[2:4]).all()
    # margins at which exp overflows, and where its inverse is all that is left
    for m in (-1e6, -800.0, -100.0, -30.0, 30.0, 100.0, 800.0, 1e6):
        one = torch.zeros(1, 2, 1, device=DEV)
        one[0, 1, 0] = m
        pref_check(ct, one, beta=1.0)
        pref_check(ct, one, beta=1.0, smoothing=0.25)


def test_offsets_that_are_none(ct):  # noqa: F811
    # they read and write within the line, and say so with a NaN
    losses = torch.rand(50, generator=seeded(1)).to(DEV)
    for bad in ([0, 10, 5, 20, 50], [-3, 10, 20, 30, 50], [0, 10, 20, 30, 51], [0, 1 << 62, 5, -(1 << 62), 7], [50, 40, 30, 20, 10]):
        offsets = torch.tensor(bad, device=DEV)
        guard = torch.full((150,), 7.0, device=DEV)
        values, ratios, slopes = ct.preference_forward(losses, offsets=offsets)
        assert torch.isnan(values).any()
        from helrm_amd.backend import PreferenceArgs
        d = guard[50:100]
        ct._call("PreferenceGrad", PreferenceArgs(offsets=offsets.data_ptr(), slope=slopes.data_ptr(), dvalue=torch.ones(2, device=DEV).data_ptr(),
                                                  dloss=d.data_ptr(), pairs=2, length=50, ignore=IGNORE), losses.device)
        assert (guard[:50] == 7).all() and (guard[100:] == 7).all() and not (d == 7).any()


def test_long_sums_that_cancel(ct):  # noqa: F811
    # 2^17 tokens of which each differs by 2^-12 of itself: in 32 bits the sums would lose the difference
    losses, _, _ = batch(seeded(4), 2, 1 << 17)
    reference = losses * (1 + 2.0 ** -12)
    reference[:, 1] = losses[:, 1] * (1 - 2.0 ** -12)
    pref_check(ct, losses, reference, beta=0.01)


def test_layouts(ct):  # noqa: F811
    losses, reference, target = batch(seeded(5), 12, 40)
    first = pref_check(ct, losses, reference, target)
    wide = torch.full((12, 2, 90), 7.0, device=DEV)
    wide[..., 3:43] = losses
    held = torch.full((12, 2, 50), 7, device=DEV)
    held[..., 9:49] = target
    turned = [t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in (losses, reference, target)]
    spread = torch.zeros(12, 2, 80, device=DEV)
    spread[..., ::2] = reference
    for other in ((wide[..., 3:43], reference, held[..., 9:49]), turned, (losses, spread[..., ::2], target)):
        for a, b in zip(first, pref_check(ct, *other), strict=True):
            assert torch.equal(a, b)
    three = pref_check(ct, losses.view(3, 4, 2, 40), reference.view(3, 4, 2, 40), target.view(3, 4, 2, 40))
    assert torch.equal(three[0].view(12), first[0])
    single = pref_check(ct, losses[0], reference[0], target[0])
    assert single[0].shape == () and torch.equal(single[0], first[0][0])
    pref_check(ct, losses[:1].expand(12, 2, 40), reference[:, :1].expand(12, 2, 40), target)
    pref_check(ct, losses.view(-1)[::2], reference.view(-1)[1::2], None, torch.tensor([0, 100, 300, 310, 480], device=DEV))


def test_autograd_and_reductions(ct):  # noqa: F811
    losses, reference, target = batch(seeded(6), 9, 70)
    leaf = losses.clone().requires_grad_()
    values, _, slopes = ct.preference_forward(losses, reference, target, smoothing=0.1)
    out = ct.preference(leaf, reference, target, smoothing=0.1, reduction="none")
    grad = torch.rand(9, generator=seeded(1)).to(DEV)
    out.backward(grad)
    assert torch.equal(out, values) and torch.equal(leaf.grad, ct.preference_backward(grad, losses, slopes, target))
    for reduction, each in (("mean", 1.0 / 9), ("sum", 1.0)):
        leaf.grad = None
        total = ct.preference(leaf, reference, target, smoothing=0.1, reduction=reduction)
        total.backward()
        ref.check(total, ref.d(values).sum() * each, ref.d(values).sum() * each, 2 * F32, reduction)
        assert torch.equal(leaf.grad, ct.preference_backward(torch.full((9,), each, device=DEV), losses, slopes, target))
    line, offsets = losses.view(-1).clone().requires_grad_(), torch.arange(0, 19 * 70, 70, device=DEV)
    ct.preference(line, reference.view(-1), target.view(-1), offsets, smoothing=0.1, reduction="sum").backward()
    assert torch.equal(line.grad.view(9, 2, 70), leaf.grad)
    (g,) = torch.autograd.grad(ct.preference(leaf, reference, target).square(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    with torch.no_grad():
        assert not ct.preference(leaf, reference, target).requires_grad
    assert ct.preference(losses[:0], reference[:0]).item() == 0


@pytest.mark.parametrize("form", FORMS[:5])
def test_against_differences(ct, form):  # noqa: F811
    losses, reference, target = batch(seeded(7), 30, 20)
    step = torch.randn(30, 2, 20, generator=seeded(8)).to(DEV)
    leaf = losses.clone().requires_grad_()
    ct.preference(leaf, reference, target, reduction="sum", **form).backward()
    h = 2.0 ** -6
    s = [ct.preference(losses + k * h * step, reference, target, reduction="none", **form).double() for k in (1, -1)]
    got, want = (s[0] - s[1]) / (2 * h), (leaf.grad.double() * step).sum((1, 2))
    move = abs(form.get("beta", 0.1)) * step.double().abs().sum((1, 2))      # of m, a step of 1
    if form.get("average"):
        move = abs(form["beta"]) * step.double().abs().amax((1, 2)) * 2
    # third derivatives of softplus are under 0.1; a hinge may be crossed by pairs within h * move of it
    values, ratios, _ = ct.preference_forward(losses, reference, target, **form)
    if form.get("kind") == "hinge":
        m = form.get("beta", 0.1) * (ratios[:, 0] - ratios[:, 1]).double() - form.get("margin", 0.0)
        fine = (m - 1).abs() > h * move + 1e-4
        assert fine.sum() > 5
        got, want, move, values = got[fine], want[fine], move[fine], values[fine]
    off = h * h * 0.1 / 6 * move ** 3 + (values.double().abs() + 1) * 64 * F32 / h
    assert ((got - want).abs() <= off).all(), ((got - want).abs() / off).max()


def test_streams_and_graphs(ct):  # noqa: F811
    side = torch.cuda.Stream()
    cases = [batch(seeded(k), pairs, length) for k, (pairs, length) in enumerate(((1, 30), (300, 20), (9, 700), (2, 30000)))]
    offsets = torch.tensor([0, 10, 11, 30000, 59000, 60000, 120000], device=DEV)
    torch.cuda.synchronize()

    def all_of():
        out = []
        for losses, reference, target in cases:
            values, ratios, slopes = ct.preference_forward(losses, reference, target)
            out += [values, ratios, ct.preference_backward(values, losses, slopes, target), ct.preference(losses, reference, target)]
        line = cases[3][0].view(-1)
        values, ratios, slopes = ct.preference_forward(line, offsets=offsets)
        return out + [values, ratios, ct.preference_backward(values, line, slopes, offsets=offsets)]

    first = all_of()
    with torch.cuda.stream(side):
        second = all_of()
    side.synchronize()
    for a, b in zip(first, second, strict=True):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_of()
    for turn in range(3):
        for losses, reference, target in cases:
            losses.mul_(1.01)
            target.copy_(target.roll(1, -1))
        offsets[1:-1].add_(7)
        for t in held:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, all_of(), strict=True):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits(ct):  # noqa: F811
    n = (1 << 32) + 1000
    line = torch.zeros(n, device=DEV)
    line[-900:] = torch.rand(900, generator=seeded(1)).to(DEV)
    offsets = torch.tensor([0, n - 900, n - 500, n - 400, n - 100], device=DEV)
    values, ratios, slopes = ct.preference_forward(line, offsets=offsets)
    end = ref.d(line[-900:])
    want = torch.tensor([[0.0, -end[:400].sum()], [-end[400:500].sum(), -end[500:800].sum()]], dtype=torch.float64)
    ref.check(ratios, want, want.abs(), 2 * F32, "ratios")
    d = ct.preference_backward(torch.ones(2, device=DEV), line, slopes, offsets=offsets)
    assert (d[:n - 900] == slopes[0, 0]).all() and (d[n - 500:n - 400] == slopes[1, 0]).all() and (d[n - 400:n - 100] == slopes[1, 1]).all()
    assert not d[n - 100:].any()


def test_refusals(ct):  # noqa: F811
    losses, reference, target = batch(seeded(0), 4, 6)
    values, ratios, slopes = ct.preference_forward(losses, reference, target)
    line, offsets = losses.view(-1), torch.tensor([0, 10, 20], device=DEV)
    for call, message in ((lambda: ct.preference(losses, reference[:3], target), "reference"),
                          (lambda: ct.preference(losses, reference.double(), target), "reference"),
                          (lambda: ct.preference(losses, reference, target.int()), "target"),
                          (lambda: ct.preference(losses, reference, target.cpu()), "target"),
                          (lambda: ct.preference(losses, reference, target.view(4, 6, 2)), "target"),
                          (lambda: ct.preference(line, offsets=offsets.cpu()), "offsets"),
                          (lambda: ct.preference(line, offsets=offsets.int()), "offsets"),
                          (lambda: ct.preference_backward(values[:3], losses, slopes, target), "grad"),
                          (lambda: ct.preference_backward(values.double(), losses, slopes, target), "grad"),
                          (lambda: ct.preference_backward(values, losses, slopes[:, :1], target), "slopes"),
                          (lambda: ct.preference_backward(values, losses, slopes.double(), target), "slopes")):
        with pytest.raises(ValueError, match=message):
            call()


def test_offsets_that_descend_write_each_token_once(ct):  # noqa: F811
    # [0, 10, 20, 5, 8, 9, 12]: the first and the third pair are ascending by themselves and share tokens
    gen = seeded(11)
    cases = [([0, 10, 20, 5, 8, 9, 12], 24), ([0, -(1 << 63), (1 << 63) - 1, 9, 3, 1 << 32, 40], 33)]
    for pairs, length in ((3, 40), (200, 3000), (3000, 50000)):
        o = torch.randint(0, length + 1, (2 * pairs + 1,), generator=gen)
        cases += [(o.tolist(), length), (o.sort().values.roll(pairs).tolist(), length)]
    for o, length in cases:
        losses, offsets = torch.rand(length, generator=gen).to(DEV), torch.tensor(o, device=DEV)
        values, ratios, slopes = ct.preference_forward(losses, offsets=offsets)
        o = torch.tensor(o)
        descends = o[1:] < o[:-1]
        assert torch.equal(values.isnan().cpu(), descends.view(-1, 2).any(1)) and values.isnan().any()
        grad = torch.ones_like(values)
        slopes = torch.arange(1.0, 2 * len(values) + 1, device=DEV).view(-1, 2)   # finite ones: which sequence's it is can be read off
        d = ct.preference_backward(grad, losses, slopes, offsets=offsets)
        for _ in range(20):
            assert torch.equal(ct.preference_backward(grad, losses, slopes, offsets=offsets).nan_to_num(-1.0), d.nan_to_num(-1.0))
        d, t = d.cpu(), torch.arange(length)
        s = (d.nan_to_num(1.0).long() - 1).clamp(min=0)
        holds = (d > 0) & (o[s] <= t) & (t < o[s + 1])
        assert (holds | d.isnan() | ((d == 0) & ((t < o[0]) | (t >= o[-1])))).all()


@pytest.mark.parametrize("pairs,long", [(1, 30000), (40, 70000), (300, 10000), (70000, 4001)])
def test_a_long_sequence_among_short_ones(ct, pairs, long):  # noqa: F811
    gen = seeded(pairs)
    lengths = torch.randint(0, 9, (2 * pairs,), generator=gen)
    lengths[torch.randint(2 * pairs, (pairs // 3,), generator=gen)] = 0
    lengths[pairs] = long                                       # many sequences without tokens stand beside one another too
    lengths[pairs + 1:pairs + 1 + pairs // 2] = 0
    lead, tail = 2500, 1031
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]) + lead
    n = int(offsets[-1]) + tail
    losses, reference, target = (t.reshape(-1)[:n].contiguous() for t in batch(gen, 1, n))
    for form in (dict(), dict(average=True, beta=2.0)):
        *_, d = pref_check(ct, losses, reference, target, offsets.to(DEV), **form)
        assert not d[:lead].any() and not d[n - tail:].any()
    pref_check(ct, losses[:n - 3], None, None, offsets.to(DEV))


def test_infinities_where_one_side_counts_nothing(ct):  # noqa: F811
    # a smoothing of 1 leaves log(1 + exp m) alone, of 0 log(1 + exp -m): the other one's infinity is no 0 * inf
    losses = torch.ones(2, 2, 3, device=DEV)
    losses[0, 0, 1] = losses[1, 1, 1] = float("inf")           # m is -inf, inf
    for smoothing, values, slopes in ((0.0, [float("inf"), 0.0], [[0.5, -0.5], [0.0, 0.0]]), (1.0, [0.0, float("inf")], [[0.0, 0.0], [-0.5, 0.5]]),
                                      (0.5, [float("inf")] * 2, [[0.25, -0.25], [-0.25, 0.25]])):
        v, _, s = ct.preference_forward(losses, beta=0.5, smoothing=smoothing)
        assert v.tolist() == values and s.tolist() == slopes


@pytest.mark.parametrize("tail", [0, 1, 7, 2048])
@pytest.mark.parametrize("pairs", [3, 600, 40000, 600000])
def test_gradients_of_a_long_line(ct, pairs, tail):  # noqa: F811
    # eight tokens a thread; a token's gradient is one product of the pair's and its sequence's, or 0
    gen = seeded(pairs + tail)
    lengths = torch.randint((1 << 19) // pairs, (1 << 21) // pairs + 2, (2 * pairs,), generator=gen)
    lengths[torch.randint(2 * pairs, (pairs // 2,), generator=gen)] = 0
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]) + 11
    n = int(offsets[-1]) + tail
    assert n >= 1 << 20
    line, target = torch.zeros(n, device=DEV), torch.where(torch.rand(n, generator=gen) < 0.8, 5, IGNORE).to(DEV)
    grad, slopes = torch.randn(pairs, generator=gen).to(DEV), torch.randn(pairs, 2, generator=gen).to(DEV)
    d = ct.preference_backward(grad, line, slopes, target, offsets.to(DEV))
    want = torch.zeros(n, device=DEV)
    want[11:n - tail] = (grad[:, None] * slopes).view(-1).repeat_interleave(lengths.to(DEV))
    assert torch.equal(d, torch.where(target != IGNORE, want, 0.0))
    assert torch.equal(ct.preference_backward(grad, line, slopes, offsets=offsets.to(DEV)), want)
