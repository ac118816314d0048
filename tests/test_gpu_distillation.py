"""Distillation from a teacher's top logits against a plain 64-bit
implementation: types, one row to several tiles, odd widths, tables in several
pieces, rows whose entries are few, none, named twice or outside the table,
infinities, strides, graphs.

Bounds.  A logit is a sum of `width` terms and scaled: L = (width + 14) 2^-24 of
its size.  A teacher's probability comes from an exponential of an argument of
up to A and a sum of `top`: e = (2 A + top + 10) 2^-24 relative.  The rest is as
for the cross entropy (test_gpu_cleartext)."""
import pytest
import torch

import cleartext_ref as ref
from test_gpu_cleartext import DEV, F32, TYPES, ct, normal, seeded  # noqa: F401

pytestmark = pytest.mark.gpu

IGNORE = -100


def tensors(gen, rows, width, vocab, top, dtype, teacher=None, none=0.0, ragged=False, lean=2.0):
    table = normal(gen, vocab, width, std=1.5 * width ** -0.5, dtype=dtype)
    ids = torch.rand(rows, vocab, generator=gen).topk(top, dim=1).indices if vocab * rows < 1 << 24 else \
        (torch.randint(vocab - top + 1, (rows, top), generator=gen).sort(1).values + torch.arange(top))
    logits = (normal(gen, rows, top, std=2.0) + 5).to(teacher or dtype)
    x = (normal(gen, rows, width) + lean * table[ids[:, 0].to(DEV)].float()).to(dtype)
    if ragged:
        ids = torch.where(torch.arange(top) < torch.randint(1, top + 1, (rows, 1), generator=gen), ids, IGNORE)
    ids[torch.rand(rows, generator=gen) < none] = IGNORE
    grad = ((torch.rand(rows, generator=gen) + 0.5) * (64.0 if dtype == torch.float16 else 1.0 / max(1, rows))).to(DEV)
    return x, table, ids.to(DEV), logits, grad


def plain(x, table, ids, logits, grad, t, ignore=IGNORE):
    """Losses, lse, dx, dtable in 64 bits and, for each, the sizes that its bound is made of."""
    x, table, ids, logits, grad = ref.d(x), ref.d(table), ids.cpu(), ref.d(logits), ref.d(grad)
    rows, (vocab, width) = len(x), table.shape
    size = table.abs()
    out = dict(losses=torch.zeros(rows), lse=torch.zeros(rows), spread=torch.zeros(rows), size=torch.zeros(rows), reach=0.0, scale=0.0)
    out = {k: v.double() if torch.is_tensor(v) else v for k, v in out.items()}
    d, q_, p_ = (torch.zeros(rows, vocab, dtype=torch.float64) for _ in range(3))
    for i in range(rows):
        there = (ids[i] != ignore) & (logits[i] != -float("inf"))
        if not there.any():
            continue
        k, l = ids[i][there], logits[i][there]
        z = table @ x[i] / t
        out["scale"] = max(out["scale"], (size @ x[i].abs() / t).nan_to_num(posinf=0.0).max().item())
        lse = torch.logsumexp(z, 0)
        out["lse"][i] = lse
        if ((k < 0) | (k >= vocab)).any():
            out["losses"][i] = float("nan")
            d[i] = float("nan")
            continue
        w = torch.softmax((l - l.max()) / t, 0)
        p = torch.zeros(vocab, dtype=torch.float64).index_add_(0, k, w)
        at = torch.nonzero(p > 0)[:, 0]
        term = p[at].log() - (z[at] - lse)
        out["losses"][i] = t * t * (p[at] * term).sum()
        out["spread"][i] = (p[at] * term.abs()).sum()
        out["size"][i] = (p[at] * (p[at].log().abs() + z[at].abs() + lse.abs())).sum()
        out["reach"] = max(out["reach"], ((l.max() - l[w > 1e-30]) / t).max().item())
        q_[i] = torch.exp(z - lse) * (t * grad[i]).abs()
        p_[i] = p * (t * grad[i]).abs()
        d[i] = (torch.exp(z - lse) - p) * t * grad[i]
    keep = ((ids != ignore) & (logits != -float("inf"))).any(1)
    out["kept"] = keep
    out["dx"], out["sx"], out["qx"], out["px"] = (m @ n for m, n in ((d, table), (d.abs(), table.abs()), (q_, table.abs()), (p_, table.abs())))
    x = torch.where(keep[:, None], x, 0.0)
    out["dtable"], out["st"], out["qt"], out["pt"] = (m.T @ n for m, n in ((d, x), (d.abs(), x.abs()), (q_, x.abs()), (p_, x.abs())))
    return out


def teach_check(ct, x, table, ids, logits, grad, t=1.0, ignore=IGNORE, once=False):  # noqa: F811
    t = float(torch.tensor(t))                     # as the entry point takes it
    rows, (vocab, width), top = x.shape[0], table.shape, ids.shape[1]
    u = ref.U[x.dtype]
    want = plain(x, table, ids, logits, grad, t, ignore)
    losses, lse, saved = ct.distillation_forward(x, table, ids, logits, t, ignore)
    logit = (width + 14) * F32 * want["scale"]
    e = (2 * want["reach"] + top + 10) * F32
    off = logit * 2 + (14 + vocab / 64) * F32 * (1 + want["lse"].abs())
    ref.check(lse, want["lse"], off, 1.0, "lse")
    ref.check(losses, want["losses"], t * t * (logit + off + e * (1 + want["spread"]) + (top + 12) * F32 * want["size"]) + 1e-30, 1.0, "losses")
    none = ~want["kept"]
    assert (losses.cpu()[none] == 0).all() and (lse.cpu()[none] == 0).all()
    dx, dtable = ct.distillation_backward(grad, x, table, ids, lse, saved, t, ignore)
    assert dx.dtype == x.dtype and dtable.dtype == x.dtype
    tol, soft = (vocab + rows + 60) * F32 + (0 if once else 2.1 * u), 4 * logit + 10 * F32
    least = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126      # subnormal results
    for name, got, s, q, p in (("dx", dx, "sx", "qx", "px"), ("dtable", dtable, "st", "qt", "pt")):
        size = want[s] * tol + want[q] * soft + want[p] * e + least
        if once:
            size = u * want[name].abs() + 1.01 * (size + want[s] * 2 * u * u)
        ref.check(got, want[name], size.nan_to_num(0.0), 1.0, name)
    assert (dx.cpu()[none] == 0).all()
    again = ct.distillation_backward(grad, x, table, ids, lse, saved, t, ignore)
    for a, b in zip((dx, dtable), again, strict=True):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    return losses, lse, dx, dtable


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab,top", [(1, 1, 1, 1), (1, 16, 4096, 5), (1, 416, 999, 64), (2, 8, 2, 2), (7, 33, 65, 3), (16, 64, 256, 17),
                                                  (17, 513, 300, 1), (50, 100, 257, 4), (64, 40, 500, 130), (65, 416, 1300, 33), (130, 24, 2500, 100),
                                                  (257, 136, 512, 12), (600, 16, 100, 7), (40, 100, 1500, 1024), (3, 300, 2000, 700)])
def test_distillation(ct, dtype, rows, width, vocab, top):  # noqa: F811
    gen = seeded(rows + vocab + top)
    for k, t in enumerate((1.0, 2.5)):
        teach_check(ct, *tensors(gen, rows, width, vocab, top, dtype, torch.float32 if k else dtype, none=0.2 * k, ragged=bool(k)), t)


# each product in large tiles, whole and split; the last ones: a table in several pieces
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab,top", [(33, 261, 24001, 9), (515, 4099, 515, 40), (1027, 131, 8197, 20), (2100, 24, 32050, 64)])
def test_large_tiles(ct, dtype, rows, width, vocab, top):  # noqa: F811
    teach_check(ct, *tensors(seeded(rows), rows, width, vocab, top, dtype, none=0.1, ragged=True), 0.75)


# so many entries of such width that their scores are picked out of the product's tiles, small and large ones
PICKED = [(520, 2000, 700, 200), (1040, 1040, 3000, 64), (300, 2000, 2000, 400), (300, 8000, 2000, 512), (2040, 520, 8100, 40), (1000, 2000, 129, 129), (1000, 2000, 300, 66)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab,top", PICKED)
def test_scores_out_of_the_tiles(ct, dtype, rows, width, vocab, top):  # noqa: F811
    gen = seeded(rows + top)
    x, table, ids, logits, grad = tensors(gen, rows, width, vocab, top, dtype, none=0.1, ragged=True)
    ids[1, :3] = torch.tensor([0, vocab - 1, vocab // 2])
    teach_check(ct, x, table, ids, logits, grad, 1.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab,top", PICKED[:3])
def test_scores_out_of_the_tiles_of_odd_entries(ct, dtype, rows, width, vocab, top):  # noqa: F811
    gen = seeded(rows)
    x, table, ids, logits, grad = tensors(gen, rows, width, vocab, top, dtype, none=0.1, ragged=True)
    full = torch.randint(vocab, (top,), generator=gen).to(DEV)
    ids[3], ids[4], ids[5], ids[6] = full, full[0], full.sort().values, full.sort(descending=True).values     # ids again and again
    ids[7, ::2] = IGNORE
    logits[8] = torch.finfo(dtype).min
    logits[9, 1:] = -float("inf")
    logits[10] = -float("inf")
    teach_check(ct, x, table, ids, logits, grad, 0.7)
    ids[20, 3], ids[21, 0], ids[22], logits[23, 1] = vocab, -1, 1 << 40, float("nan")
    ids[23, 1] = 5
    losses, lse, saved = ct.distillation_forward(x, table, ids, logits, 1.0)
    dx, dtable = ct.distillation_backward(grad, x, table, ids, lse, saved, 1.0)
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[20:24] = True
    assert torch.equal(torch.isnan(losses).cpu(), bad) and torch.equal(torch.isnan(dx).any(1).cpu(), bad) and torch.isfinite(lse).all()
    assert torch.isnan(dtable).all()


def test_scores_out_of_the_tiles_of_several_launches(ct):  # noqa: F811
    # 4,096 x 1,025 tiles go in two launches, cut at column 131,328; all vectors but a few are 0
    rows, vocab, width, top = 1 << 20, (1 << 18) + 200, 1024, 64
    gen = torch.Generator(DEV).manual_seed(3)
    table = (torch.randn(vocab, width, generator=gen, device=DEV) * 0.03).bfloat16()
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEV)
    some = torch.cat([torch.arange(40), torch.arange(rows // 2 - 20, rows // 2 + 20), torch.arange(rows - 40, rows)]).to(DEV)
    x[some] = torch.randn(len(some), width, generator=gen, device=DEV).bfloat16()
    ids = torch.randint(vocab // top, (rows, top), generator=gen, device=DEV) * top + torch.arange(top, device=DEV)     # different in a row
    ids[some, :4] = torch.tensor([131327, 131328, vocab - 1, 131584], device=DEV)
    logits = torch.randn(rows, top, generator=gen, device=DEV)
    losses, lse, _ = ct.distillation_forward(x, table, ids, logits)
    p = torch.softmax(logits.double(), 1)
    ref.check(lse[40:1000], torch.full((960,), float(vocab), dtype=torch.float64).log(), torch.ones(960), 1e-5, "lse")
    want = (p * (p.log() + torch.tensor(float(vocab), dtype=torch.float64).log().item())).sum(1)
    z = x[some].double() @ table.double().T
    norm = torch.logsumexp(z, 1)
    want[some] = (p[some] * (p[some].log() - z.gather(1, ids[some]) + norm[:, None])).sum(1)
    ref.check(lse[some], norm.cpu(), torch.ones(len(some)), 1e-4, "lse")
    ref.check(losses, want.cpu(), torch.ones(rows), 2e-4, "losses")


def test_two_pieces_of_16_bits(ct):  # noqa: F811
    x, table, ids, logits, grad = tensors(seeded(8), 2100, 24, 64100, 4, torch.bfloat16)
    ids[:4, 0] = torch.tensor([63487, 63488, 64099, 0])     # beside the cut, and at the ends
    teach_check(ct, x, table, ids, logits, grad, 2.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width,vocab", [(1, 72, 264), (3, 264, 1000), (17, 64, 4096), (40, 100, 301), (64, 520, 1300), (94, 172, 3000),
                                              (130, 64, 4100), (256, 264, 700)])
def test_few_rows_round_once(ct, dtype, rows, width, vocab):  # noqa: F811
    teach_check(ct, *tensors(seeded(rows + vocab), rows, width, vocab, 16, dtype), 1.0, once=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,none", [(1, 1.0), (40, 0.5), (300, 0.1), (300, 0.97), (300, 1.0)])
def test_rows_without_a_teacher(ct, dtype, rows, none):  # noqa: F811
    x, table, ids, logits, grad = tensors(seeded(rows), rows, 40, 333, 6, dtype, none=none)
    gone = (ids == IGNORE).all(1)
    logits[5::7] = -float("inf")             # no entry either
    ids[3::7, 2] = IGNORE
    logits[:, 3][ids[:, 3] == IGNORE] = float("nan")
    gone |= (logits == -float("inf")).all(1)
    def both():
        losses, lse, saved = ct.distillation_forward(x, table, ids, logits, 1.5)
        return (losses, lse) + ct.distillation_backward(grad, x, table, ids, lse, saved, 1.5)
    clean = both()
    x[gone] = float("nan")                   # what such a row holds reaches nothing
    grad[gone] = float("inf")
    dirty = both()
    for a, b in zip(clean, dirty, strict=True):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    if gone.all():
        assert not any(t.any() for t in dirty)
    x[gone] = 0
    grad[gone] = 0
    teach_check(ct, x, table, ids, logits, grad, 1.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 40, 300])
def test_an_id_named_twice_and_ids_outside(ct, dtype, rows):  # noqa: F811
    x, table, ids, logits, grad = tensors(seeded(rows), rows, 24, 50, 9, dtype)
    ids[:, 5] = ids[:, 1]
    ids[::2, 8] = ids[::2, 1]
    ids[1::3] = ids[1::3, :1]                # one row of the table alone
    losses, *_ = teach_check(ct, x, table, ids, logits, grad, 1.3)
    assert torch.isfinite(losses).all()
    ids[1, 4], ids[2, 0] = 50, -1
    losses, lse, dx, dtable = teach_check(ct, x, table, ids, logits, grad, 1.3)
    assert torch.isnan(losses).cpu().tolist() == [i in (1, 2) for i in range(rows)] == torch.isnan(dx).any(1).cpu().tolist()
    assert torch.isnan(dtable).all() and torch.isfinite(lse).all()
    # an ignore_index inside the table
    ids[1, 4], ids[2, 0] = 7, 7
    teach_check(ct, x, table, ids, logits, grad, 1.3, ignore=7)


def test_a_models_own_answer_has_no_loss(ct):  # noqa: F811
    # a teacher that knows all of the table and says what the model says
    gen = seeded(2)
    x, table = normal(gen, 90, 32), normal(gen, 60, 32, std=0.2)
    ids = torch.rand(90, 60, generator=gen).argsort(1).to(DEV)
    logits = (x.double() @ table.double().T).gather(1, ids).float()
    grad = torch.ones(90, device=DEV)
    losses, lse, saved = ct.distillation_forward(x, table, ids, logits, 2.0)
    dx, dtable = ct.distillation_backward(grad, x, table, ids, lse, saved, 2.0)
    size = (x.abs() @ table.abs().T).max().item() * 60 * F32
    assert losses.abs().max().item() <= 4 * 4 * size and dx.abs().max().item() <= 4 * 60 * size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 70])
def test_infinities_and_lowest_values(ct, dtype, rows):  # noqa: F811
    low = torch.finfo(dtype).min
    x, table, ids, logits, grad = tensors(seeded(rows), rows, 33, 200, 8, dtype)
    # teachers' logits: the lowest value beside others has no weight, alone it has all of it, whatever the temperature
    logits[0, 1:] = low
    logits[1] = low
    logits[2, :4] = -float("inf")
    for t in (0.5, 1.0, 4.0):
        teach_check(ct, x, table, ids, logits, grad, t)
    logits[0, 2], logits[1, 3] = float("inf"), float("nan")
    losses, lse, saved = ct.distillation_forward(x, table, ids, logits, 2.0)
    assert torch.isnan(losses).cpu().tolist() == [i < 2 for i in range(rows)] and torch.isfinite(lse).all()
    dx, _ = ct.distillation_backward(grad, x, table, ids, lse, saved, 2.0)
    assert torch.isnan(dx).any(1).cpu().tolist() == [i < 2 for i in range(rows)]
    # table rows masked through a constant coordinate: without probability; with a teacher on one of them the loss is infinite
    x, table, ids, logits, grad = tensors(seeded(rows), rows, 33, 200, 8, dtype)
    ids[ids == 11] = 12
    x[:, 7] = 1.0
    table[:, 7] = 0.0
    table[11, 7] = low
    losses, lse, saved = ct.distillation_forward(x, table, ids, logits, 1.0)
    want = plain(x, torch.cat([table[:11], table[12:]]), torch.where(ids > 11, ids - 1, ids), logits, grad, 1.0)
    assert (losses.cpu() - want["losses"]).abs().max() < 1e-4 and (lse.cpu() - want["lse"]).abs().max() < 1e-4
    dx, dtable = ct.distillation_backward(grad, x, table, ids, lse, saved, 1.0)
    assert torch.isfinite(dx).all() and not dtable[11].any()
    table[11, 7] = -float("inf")
    ids[0, 0] = 11
    losses, lse, _ = ct.distillation_forward(x, table, ids, logits, 1.0)
    assert losses[0] == float("inf") and torch.isfinite(losses[1:]).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(ct, dtype):  # noqa: F811
    x, table, ids, logits, grad = tensors(seeded(5), 24, 40, 90, 5, dtype)
    def both(x, table, ids, logits, grad):
        losses, lse, saved = ct.distillation_forward(x, table, ids, logits, 1.5)
        return (losses, lse) + ct.distillation_backward(grad, x, table, ids, lse, saved, 1.5)
    first = both(x, table, ids, logits, grad)
    wide, tall = torch.full((24, 131), 7.0, dtype=dtype, device=DEV), torch.full((180, 77), 7.0, dtype=dtype, device=DEV)
    wide[:, 3:43], tall[::2, 1:41] = x, table
    for other in (both(wide[:, 3:43], tall[::2, 1:41], ids, logits, grad),
                  both(x.t().contiguous().t(), table.t().contiguous().t(), ids.t().contiguous().t(), logits.t().contiguous().t(), grad),
                  both(x.view(4, 6, 40), table, ids.view(4, 6, 5), logits.view(4, 6, 5), grad.view(4, 6)),
                  both(x.view(4, 6, 40), table, ids, logits.view(24, 5), grad)):
        for a, b in zip(first, other, strict=True):
            assert torch.equal(a.reshape(-1), b.reshape(-1))
    # one gradient for all rows
    same = both(x, table, ids, logits, grad[:1].expand(24))
    for a, b in zip(same, both(x, table, ids, logits, grad[:1].repeat(24)), strict=True):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [5, 100])
def test_autograd_and_reductions(ct, rows):  # noqa: F811
    x, table, ids, logits, grad = tensors(seeded(4), rows, 24, 70, 6, torch.float32)
    ids[3] = IGNORE
    losses, lse, saved = ct.distillation_forward(x, table, ids, logits, 2.0)
    a, b = x.clone().requires_grad_(), table.clone().requires_grad_()
    out = ct.distillation(a, b, ids, logits, 2.0, reduction="none")
    out.backward(grad)
    dx, dtable = ct.distillation_backward(grad, x, table, ids, lse, saved, 2.0)
    assert torch.equal(out, losses) and torch.equal(a.grad, dx) and torch.equal(b.grad, dtable)
    for reduction, each in (("mean", 1.0 / (rows - 1)), ("sum", 1.0)):
        a.grad = b.grad = None
        total = ct.distillation(a, b, ids, logits, 2.0, reduction=reduction)
        total.backward()
        assert abs(total.item() - losses.double().sum().item() * each) <= 4 * F32 * losses.abs().double().sum().item() * each
        want = ct.distillation_backward(torch.full((rows,), each, device=DEV), x, table, ids, lse, saved, 2.0)
        assert torch.equal(a.grad, want[0]) and torch.equal(b.grad, want[1])
        with torch.no_grad():
            assert torch.equal(ct.distillation(a, b, ids, logits, 2.0, reduction=reduction), total.detach())
    assert ct.distillation(x[:0], table, ids[:0], logits[:0]).item() == 0
    b.grad = None
    ct.distillation(x[:0], b, ids[:0], logits[:0], reduction="sum").backward()
    assert b.grad.shape == table.shape and not b.grad.any()
    nothing = ct.distillation(a, b, torch.full_like(ids, IGNORE), logits)
    a.grad = None
    nothing.backward()
    assert nothing.item() == 0 and not a.grad.any()
    (g,) = torch.autograd.grad(ct.distillation(a, b, ids, logits).square(), a, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    # one of the two without a gradient
    a.grad = None
    ct.distillation(a, table, ids, logits, 2.0, reduction="sum").backward()
    assert torch.equal(a.grad, want[0])


def test_against_differences(ct):  # noqa: F811
    x, table, ids, logits, _ = tensors(seeded(9), 20, 12, 40, 5, torch.float32)
    gen = seeded(10)
    sx, st = normal(gen, 20, 12), normal(gen, 40, 12)
    a, b = x.clone().requires_grad_(), table.clone().requires_grad_()
    ct.distillation(a, b, ids, logits, 1.5, reduction="sum").backward()
    slope = (a.grad.double() * sx).sum() + (b.grad.double() * st).sum()
    h = 2.0 ** -6
    up, down = (ct.distillation(x + k * h * sx, table + k * h * st, ids, logits, 1.5, reduction="none").double().sum() for k in (1, -1))
    # the same difference in 64 bits says what the step itself costs
    exact = [plain(x.double() + k * h * sx.double(), table.double() + k * h * st.double(), ids, logits, torch.ones(20), 1.5)["losses"].sum() for k in (1, -1)]
    step = abs((exact[0] - exact[1]).item() / (2 * h) - slope.item())
    assert abs(((up - down) / (2 * h) - slope).item()) <= step + 20 * 2.25 * 200 * F32 / h
    assert step <= 0.05 * abs(slope.item()) + 1


def test_streams_and_graphs(ct):  # noqa: F811
    side = torch.cuda.Stream()
    cases = [tensors(seeded(k), rows, 40, vocab, 7, dtype, none=0.1, ragged=True)
             for k, (rows, vocab, dtype) in enumerate(((3, 300, torch.float32), (50, 700, torch.bfloat16), (300, 900, torch.float16)))]
    cases.append(tensors(seeded(9), 520, 2000, 700, 200, torch.bfloat16, none=0.1))
    torch.cuda.synchronize()

    def all_of():
        out = []
        for x, table, ids, logits, grad in cases:
            losses, lse, saved = ct.distillation_forward(x, table, ids, logits, 2.0)
            out += [losses, lse, *ct.distillation_backward(grad, x, table, ids, lse, saved, 2.0), ct.distillation(x, table, ids, logits, 2.0)]
        return out

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
        for x, table, ids, logits, grad in cases:
            x.mul_(-0.9)
            ids.copy_(ids.roll(1, 0))
            logits.copy_(logits.roll(1, 1))
        for t in held:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, all_of(), strict=True):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits(ct):  # noqa: F811
    # a table of more than 2^32 bytes, whose last rows alone are not 0
    vocab, width = (1 << 31) // 512 + 300, 512
    gen = seeded(1)
    table = torch.zeros(vocab, width, dtype=torch.bfloat16, device=DEV)
    table[-40:] = normal(gen, 40, width, std=0.2, dtype=torch.bfloat16)
    ids = (vocab - 1 - torch.rand(20, 40, generator=gen).argsort(1)[:, :6]).to(DEV)
    x, logits, grad = normal(gen, 20, width, dtype=torch.bfloat16), normal(gen, 20, 6), torch.full((20,), 0.1, device=DEV)
    losses, lse, saved = ct.distillation_forward(x, table, ids, logits, 1.0)
    z = ref.d(x) @ ref.d(table[-40:]).T
    want = torch.logsumexp(torch.cat([z, torch.full((20, 1), float(vocab - 40), dtype=torch.float64).log()], 1), 1)
    logp = torch.log_softmax(ref.d(logits), 1)
    logq = z.gather(1, ids.cpu() - (vocab - 40)) - want[:, None]
    ref.check(lse, want, torch.ones(20), 2e-4, "lse")
    ref.check(losses, (logp.exp() * (logp - logq)).sum(1), torch.ones(20), 4e-4, "losses")
    dx, dtable = ct.distillation_backward(grad, x, table, ids, lse, saved, 1.0)
    d = (z - want[:, None]).exp().scatter_add(1, ids.cpu() - (vocab - 40), -logp.exp()) * 0.1
    ref.check(dtable[-40:], d.T @ ref.d(x), d.abs().T @ ref.d(x).abs() + 1e-3, 2.0 ** -7, "dtable")
    ref.check(dx, d @ ref.d(table[-40:]), d.abs() @ ref.d(table[-40:]).abs() + 1e-3, 2.0 ** -7, "dx")


def test_refusals(ct):  # noqa: F811
    x, table, ids, logits, grad = tensors(seeded(0), 6, 8, 20, 3, torch.bfloat16)
    losses, lse, saved = ct.distillation_forward(x, table, ids, logits)
    for call, message in ((lambda: ct.distillation(x, table, ids.int(), logits), "ids: torch.int32"),
                          (lambda: ct.distillation(x, table, ids.cpu(), logits), "ids: torch.int64 on cpu"),
                          (lambda: ct.distillation(x, table, ids[:4], logits[:4]), "ids: 4 rows, not 6"),
                          (lambda: ct.distillation(x, table, ids, logits[:, :2]), "logits"),
                          (lambda: ct.distillation(x, table, ids, logits.half()), "logits: torch.float16"),
                          (lambda: ct.distillation(x, table.float(), ids, logits), "table"),
                          (lambda: ct.distillation_backward(grad[:5], x, table, ids, lse, saved), "grad"),
                          (lambda: ct.distillation_backward(grad.bfloat16(), x, table, ids, lse, saved), "grad"),
                          (lambda: ct.distillation_backward(grad, x, table, ids, lse[:5], saved), "lse"),
                          (lambda: ct.distillation_backward(grad, x, table, ids[:, :2], lse, saved), "saved"),
                          (lambda: ct.distillation_backward(grad, x, table, ids, lse, (saved[0][:5], saved[1])), "saved")):
        with pytest.raises(ValueError, match=message):
            call()
