"""The cleartext operators against plain 64-bit implementations: types,
lengths from none to long ones, odd sizes, strides, masks that leave nothing,
NaN in masked rows, other streams, graphs, and what they refuse.  Bounds are
derived in cleartext_ref."""
import pytest
import torch

import cleartext_ref as ref
from helrm_amd.backend import HipError

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
F32 = 2.0 ** -24
DEV = "cuda"


@pytest.fixture(scope="module")
def ct():
    from helrm_amd import cleartext
    return cleartext


def normal(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen) * std).to(dtype).to(DEV)


def seeded(n):
    return torch.Generator().manual_seed(n)


# ---- layer norm ------------------------------------------------------------------


def norm_check(ct, x, w, b, dy, eps=1e-5):
    u, up = ref.U[x.dtype], ref.U[w.dtype]
    rows, width = x.shape[0], x.shape[1]
    # (x - mu) r is a difference of float32 values of the row's largest size
    x64 = ref.d(x)
    y64, mu64, r64, h64 = ref.layer_norm(x, w, b, eps)
    big = (x64.abs().amax(1, keepdim=True) + 1e-30) * r64[:, None] if rows else x64
    slop = (width + 30) * F32
    y, mean, rstd = ct.layer_norm_forward(x, w, b, eps)
    size = big * ref.d(w).abs() + (0 if b is None else ref.d(b).abs()) + 1e-30
    ref.check(y, y64, size * slop + u * y64.abs(), 1.0, "y")
    ref.check(mean, mu64, x64.abs().amax(1) + 1e-30 if rows else mu64, slop, "mean")
    assert torch.equal(ct.layer_norm(x, w, b, eps), y)
    dx64, dw64, db64 = ref.layer_norm_grad(dy, x, w, eps)
    dx, dw, db = ct.layer_norm_backward(dy, x, w, mean, rstd, has_bias=b is not None)
    t = ref.d(dy).abs() * ref.d(w).abs()
    hs = h64.abs() + big * slop
    sx = r64[:, None] * (t + t.mean(1, keepdim=True) + hs * (t * (hs + big)).mean(1, keepdim=True)) if rows else t
    ref.check(dx, dx64, sx * slop * (1 + big) + u * dx64.abs(), 1.0, "dx")
    row_slop = (rows + 30) * F32
    dy64 = ref.d(dy).abs()
    ref.check(dw, dw64, row_slop * (dy64 * hs).sum(0) + slop * (dy64 * (big + hs * big * big)).sum(0) + up * dw64.abs() + 1e-30, 1.0, "dw")
    if b is None:
        assert db is None
    else:
        ref.check(db, db64, row_slop * dy64.sum(0) + up * db64.abs() + 1e-30, 1.0, "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(0, 8), (1, 1), (1, 512), (3, 7), (5, 1001), (33, 64), (257, 416), (70, 2048), (9, 4097),
                                        (4, 9000), (2, 40000)])
def test_layer_norm(ct, dtype, rows, width):
    gen = seeded(rows * 31 + width)
    x = normal(gen, rows, width, std=2.0, dtype=dtype) + 0.5
    for params in {dtype, torch.float32}:
        w = normal(gen, width, std=0.2, dtype=params) + 1
        norm_check(ct, x, w, normal(gen, width, dtype=params), normal(gen, rows, width, dtype=dtype), eps=1e-3)


def test_layer_norm_without_bias_far_from_zero_and_constant_rows(ct):
    gen = seeded(5)
    x = normal(gen, 6, 96) + 1000.0          # the spread is 1/1000 of the mean
    x[4] = 3.0                               # no spread at all
    norm_check(ct, x, normal(gen, 96), None, normal(gen, 6, 96), eps=1e-2)
    y = ct.layer_norm(x, torch.ones(96, device=DEV), torch.full((96,), 0.25, device=DEV))
    assert torch.equal(y[4], torch.full((96,), 0.25, device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_layouts(ct, dtype):
    gen = seeded(8)
    w, b = normal(gen, 40, dtype=dtype), normal(gen, 40, dtype=dtype)
    wide = normal(gen, 12, 131, dtype=dtype)
    dy = normal(gen, 12, 40, dtype=dtype)
    for x in (wide[:, :40], wide[:, 3:43], wide[::2, 1:41], wide[:, 2:82:2], normal(gen, 40, 12, dtype=dtype).t()):
        norm_check(ct, x, w, b, dy[: x.shape[0]], eps=1e-3)
    flat = wide[:12, :40].contiguous()
    three = ct.layer_norm(flat.view(3, 4, 40), w, b)
    assert torch.equal(three.view(12, 40), ct.layer_norm(flat, w, b))
    one = normal(gen, 1, 40, dtype=dtype)
    norm_check(ct, one.expand(12, 40), w, b, dy, eps=1e-3)
    norm_check(ct, flat, w, b, one.expand(12, 40), eps=1e-3)


def test_layer_norm_of_a_nan_row_stays_in_its_row(ct):
    gen = seeded(2)
    x = normal(gen, 5, 64)
    x[2, 3] = float("nan")
    x[3, 5] = float("inf")
    y = ct.layer_norm(x, torch.ones(64, device=DEV))
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).any()
    assert torch.isfinite(y[[0, 1, 4]]).all()


@pytest.mark.parametrize("width", [7, 520, 1032])
def test_layer_norm_of_equal_values_whose_mean_overflows_times_rstd(ct, width):
    # 2^114 and its sum are exact, h is 0: dx = r (w dy - mean(w dy)), r = 10^6
    x = torch.full((3, width), 2.0 ** 114, device=DEV)
    w, dy = torch.ones(width, device=DEV), normal(seeded(7), 3, width)
    y, mean, rstd = ct.layer_norm_forward(x, w, None, 1e-12)
    assert (y == 0).all() and (mean == 2.0 ** 114).all()
    dx, dw, _ = ct.layer_norm_backward(dy, x, w, mean, rstd, has_bias=False)
    assert (dw == 0).all()
    t = ref.d(dy)
    ref.check(dx, 1e6 * (t - t.mean(1, keepdim=True)), 1e6 * (t.abs() + t.abs().mean(1, keepdim=True)), (width + 30) * F32, "dx")


def test_layer_norm_offsets_beyond_32_bits(ct):
    rows, width = (1 << 31) // 4096 + 5, 4096
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEV)
    gen = seeded(1)
    tail = normal(gen, 7, width, dtype=torch.bfloat16)
    x[-7:] = tail
    w, b = normal(gen, width, dtype=torch.bfloat16), normal(gen, width, dtype=torch.bfloat16)
    y, mean, rstd = ct.layer_norm_forward(x, w, b)
    assert torch.equal(y[-7:], ct.layer_norm(tail, w, b))
    dx, dw, db = ct.layer_norm_backward(x, x, w, mean, rstd)
    small = ct.layer_norm_backward(tail, tail, w, mean[-7:].contiguous(), rstd[-7:].contiguous())
    assert torch.equal(dx[-7:], small[0])
    ref.check(dw, ref.d(small[1]), ref.d(small[1]).abs() + 1e-3, 2.0 ** -7, "dw")


# ---- gated feed-forward block -----------------------------------------------------


def mlp_check(ct, x, gate, up, down, dy, act):
    u = ref.U[x.dtype]
    rows, (hidden, width) = x.shape[0], gate.shape
    sizes = ref.mlp_sizes(dy, x, gate, up, down, act)
    y, saved = ct.gated_mlp_forward(x, gate, up, down, act)
    # one rounding of the hidden values, one of the result; three sums of K terms behind one another, and the
    # activation's slope of what the first is off
    sums = 2 * (2 * width + hidden + rows + 40) * F32
    ref.check(y, ref.mlp(x, gate, up, down, act), sizes[0], sums + 2.1 * u, "y")
    assert torch.equal(ct.gated_mlp(x, gate, up, down, act), y)
    got = ct.gated_mlp_backward(dy, x, gate, up, down, saved, act)
    want = ref.mlp_grad(dy, x, gate, up, down, act)
    # float16 values below 2^-14 are rounded to a multiple of 2^-24
    least = 2.0 ** -24 * (1 + hidden + rows) if x.dtype == torch.float16 else 0.0
    for name, g, r, s in zip(("dx", "dgate", "dup", "ddown"), got, want, sizes[1:]):
        ref.check(g, r, s + (least * 4) / (2.1 * u), sums + 2.1 * u, name)


def mlp_tensors(gen, rows, width, hidden, dtype):
    return (normal(gen, rows, width, dtype=dtype), normal(gen, hidden, width, std=width ** -0.5, dtype=dtype),
            normal(gen, hidden, width, std=width ** -0.5, dtype=dtype), normal(gen, width, hidden, std=hidden ** -0.5, dtype=dtype),
            normal(gen, rows, width, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,hidden", [(1, 1, 1), (1, 64, 256), (2, 416, 512), (5, 30, 17), (16, 128, 264), (33, 72, 136),
                                               (65, 129, 300), (128, 256, 128), (200, 96, 1000), (300, 520, 40), (1000, 16, 24)])
def test_gated_mlp(ct, dtype, rows, width, hidden):
    gen = seeded(rows + width + hidden)
    x, gate, up, down, dy = mlp_tensors(gen, rows, width, hidden, dtype)
    acts = ["silu", "gelu", ref.CUBIC]
    mlp_check(ct, x, gate, up, down, dy, acts[(rows + hidden) % 3])


# each product of the block in large tiles, whole and in sums split along k, none of the sizes a multiple of a tile
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,hidden", [(2051, 4099, 33), (1541, 33, 2565), (2051, 33, 4099), (33, 1027, 2565), (131, 4099, 2565),
                                               (131, 2565, 4099), (131, 4099, 1285), (2565, 131, 1541)])
def test_gated_mlp_large_tiles(ct, dtype, rows, width, hidden):
    x, gate, up, down, dy = mlp_tensors(seeded(rows + width), rows, width, hidden, dtype)
    mlp_check(ct, x, gate, up, down, dy, "gelu")


# up to 64 rows the intermediates are held in two parts, off by u^2: only the result is rounded to its type
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width,hidden", [(1, 72, 64), (3, 264, 1000), (17, 64, 72), (40, 100, 301), (64, 520, 128)])
def test_gated_mlp_of_few_rows_rounds_once(ct, dtype, rows, width, hidden):
    x, gate, up, down, dy = mlp_tensors(seeded(rows + hidden), rows, width, hidden, dtype)
    u, least = ref.U[dtype], 2.0 ** -24 * (1 + hidden + rows) * 4 if dtype == torch.float16 else 0.0
    tol = 2 * (2 * width + hidden + rows + 40) * F32 + 2 * u * u
    y, saved = ct.gated_mlp_forward(x, gate, up, down, "silu")
    got = (y, *ct.gated_mlp_backward(dy, x, gate, up, down, saved, "silu"))
    want = (ref.mlp(x, gate, up, down, "silu"), *ref.mlp_grad(dy, x, gate, up, down, "silu"))
    for name, g, r, size in zip(("y", "dx", "dgate", "dup", "ddown"), got, want, ref.mlp_sizes(dy, x, gate, up, down, "silu")):
        ref.check(g, r, u * r.abs() + 1.01 * (size * tol + least), 1.0, name)


@pytest.mark.parametrize("act", ["silu", "gelu", ref.CUBIC])
@pytest.mark.parametrize("rows", [1, 40])
def test_gated_mlp_activations(ct, act, rows):
    gen = seeded(3)
    x, gate, up, down, dy = mlp_tensors(gen, rows, 48, 80, torch.float32)
    mlp_check(ct, x * (4 if isinstance(act, str) else 1), gate, up, down, dy, act)


def test_gated_mlp_saturated_activations_are_finite(ct):
    x = torch.tensor([[100.0], [-100.0], [1e4], [-1e4]], device=DEV)
    one = torch.ones(1, 1, device=DEV)
    for act in ("silu", "gelu"):
        y, saved = ct.gated_mlp_forward(x, one, one, one, act)
        assert torch.equal(y, torch.tensor([[1e4], [0.0], [1e8], [0.0]], device=DEV)) or act == "silu"
        assert torch.isfinite(y).all() and y[1].abs() < 1e-30 and y[3] == 0
        for g in ct.gated_mlp_backward(torch.ones_like(x), x, one, one, one, saved, act):
            assert torch.isfinite(g).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_mlp_layouts(ct, dtype):
    gen = seeded(12)
    rows, width, hidden = 37, 48, 56
    x, gate, up, down, dy = mlp_tensors(gen, rows, width, hidden, dtype)

    def inside(t, at):  # the same values, one row after `at + a few` elements of another
        wide = torch.full((t.shape[0], t.shape[1] + 11), float("nan"), dtype=dtype, device=DEV)
        wide[:, at:at + t.shape[1]] = t
        return wide[:, at:at + t.shape[1]]

    want = ct.gated_mlp_forward(x, gate, up, down)
    grads = ct.gated_mlp_backward(dy, x, gate, up, down, want[1])
    for at in (0, 1, 8):
        tensors = [inside(t, at) for t in (x, gate, up, down, dy)]
        y, saved = ct.gated_mlp_forward(*tensors[:4])
        assert torch.equal(y, want[0]) and torch.equal(saved, want[1])
        for g, w in zip(ct.gated_mlp_backward(tensors[4], *tensors[:4], saved), grads):
            assert torch.equal(g, w)
    turned = [t.t().contiguous().t() for t in (x, gate, up, down)]
    assert torch.equal(ct.gated_mlp(*turned), want[0])
    assert torch.equal(ct.gated_mlp(x.view(1, rows, width), gate, up, down)[0], want[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_mlp_no_rows(ct, dtype):
    gen = seeded(1)
    x, gate, up, down, dy = mlp_tensors(gen, 0, 13, 9, dtype)
    y, saved = ct.gated_mlp_forward(x, gate, up, down)
    assert y.shape == (0, 13)
    dx, dgate, dup, ddown = ct.gated_mlp_backward(dy, x, gate, up, down, saved)
    assert dx.shape == (0, 13)
    for g in (dgate, dup, ddown):
        assert torch.equal(g, torch.zeros_like(g))


# ---- cross entropy -----------------------------------------------------------------


def ce_check(ct, x, table, target, grad, ignore=-100):
    u = ref.U[x.dtype]
    rows, (vocab, width) = x.shape[0], table.shape
    kept = target.cpu() != ignore
    losses, lse = ct.cross_entropy_forward(x, table, target, ignore)
    l64, s64 = ref.cross_entropy(x, table, target, ignore)
    # a logit is a sum of `width` terms; exponentials and their sum
    scale = (ref.d(x).nan_to_num().abs()[kept] @ ref.d(table).abs().T).amax().item() if kept.any() else 0.0
    logit = (width + 12) * F32 * scale
    off = logit * 2 + (12 + vocab / 64) * F32 * (1 + s64.abs().nan_to_num())
    ref.check(losses, l64, off, 1.0, "losses")
    ref.check(lse, s64, off, 1.0, "lse")
    assert (losses.cpu()[~kept] == 0).all() and (lse.cpu()[~kept] == 0).all()
    dx, dtable = ct.cross_entropy_backward(grad, x, table, target, lse, ignore)
    dx64, dt64, sx, st, px, pt = ref.cross_entropy_grad(grad, x, table, target, ignore)
    tol, soft = (vocab + rows + 60) * F32 + 2.1 * u, 4 * logit + 8 * F32
    least = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126      # subnormal results
    ref.check(dx, dx64, sx * tol + px * soft + least, 1.0, "dx")
    ref.check(dtable, dt64, st * tol + pt * soft + least, 1.0, "dtable")
    assert (dx.cpu()[~kept] == 0).all()


def ce_tensors(gen, rows, width, vocab, dtype, ignored=0.0, lean=2.0):
    table = normal(gen, vocab, width, std=1.5 * width ** -0.5, dtype=dtype)
    target = torch.randint(vocab, (rows,), generator=gen).to(DEV)
    x = (normal(gen, rows, width) + lean * table[target].float()).to(dtype)
    if ignored:
        target[torch.rand(rows, generator=gen).to(DEV) < ignored] = -100
    grad = ((torch.rand(rows, generator=gen) + 0.5) * (64.0 if dtype == torch.float16 else 1.0 / max(1, rows))).to(DEV)
    return x, table, target, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab", [(1, 1, 1), (1, 16, 4096), (1, 416, 999), (2, 8, 2), (7, 33, 65), (16, 64, 256),
                                              (50, 100, 257), (65, 416, 1300), (130, 24, 2500), (257, 136, 512), (600, 16, 100)])
def test_cross_entropy(ct, dtype, rows, width, vocab):
    x, table, target, grad = ce_tensors(seeded(rows + vocab), rows, width, vocab, dtype)
    ce_check(ct, x, table, target, grad)


# each product of the loss in large tiles, whole and split; the last: a table in two pieces in float32
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab", [(261, 33, 24001), (33, 261, 24001), (2051, 4099, 515), (131, 4099, 4099), (1027, 131, 8197),
                                              (4099, 33, 12001)])
def test_cross_entropy_large_tiles(ct, dtype, rows, width, vocab):
    x, table, target, grad = ce_tensors(seeded(rows + vocab), rows, width, vocab, dtype, ignored=0.2)
    ce_check(ct, x, table, target, grad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width,vocab", [(1, 72, 264), (3, 264, 1000), (17, 64, 4096), (40, 100, 301), (64, 520, 1300)])
def test_cross_entropy_of_few_rows_rounds_once(ct, dtype, rows, width, vocab):
    x, table, target, grad = ce_tensors(seeded(rows + vocab), rows, width, vocab, dtype)
    _, lse = ct.cross_entropy_forward(x, table, target)
    u, least = ref.U[dtype], 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126
    logit = (width + 12) * F32 * (ref.d(x).abs() @ ref.d(table).abs().T).amax().item()
    tol, soft = (vocab + rows + 60) * F32 + 2 * u * u, 4 * logit + 8 * F32
    dx64, dt64, sx, st, px, pt = ref.cross_entropy_grad(grad, x, table, target)
    for name, g, r, size, p in zip(("dx", "dtable"), ct.cross_entropy_backward(grad, x, table, target, lse), (dx64, dt64), (sx, st), (px, pt)):
        ref.check(g, r, u * r.abs() + 1.01 * (size * tol + p * soft + least), 1.0, name)


def test_cross_entropy_of_two_pieces_of_16_bits(ct):
    x, table, target, grad = ce_tensors(seeded(8), 2100, 24, 64100, torch.bfloat16)
    target[:3] = torch.tensor([63487, 63488, 64099])     # beside the cut, and the last row
    ce_check(ct, x, table, target, grad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,ignored", [(1, 1.0), (40, 0.5), (300, 0.1), (300, 0.97), (300, 1.0)])
def test_cross_entropy_ignored_rows(ct, dtype, rows, ignored):
    x, table, target, grad = ce_tensors(seeded(rows), rows, 40, 333, dtype, ignored)
    gone = target == -100
    clean = ct.cross_entropy_backward(grad, x, table, target, ct.cross_entropy_forward(x, table, target)[1])
    x[gone] = float("nan")                   # what a masked row holds reaches nothing
    grad[gone] = float("inf")
    if gone.all():
        losses, lse = ct.cross_entropy_forward(x, table, target)
        dx, dtable = ct.cross_entropy_backward(grad, x, table, target, lse)
        for t in (losses, lse, dx, dtable):
            assert torch.equal(t, torch.zeros_like(t))
        return
    ce_check(ct, x, table, target, grad)
    again = ct.cross_entropy_backward(grad, x, table, target, ct.cross_entropy_forward(x, table, target)[1])
    assert torch.equal(again[0], clean[0]) and torch.equal(again[1], clean[1])


def test_cross_entropy_ignore_index_inside_the_table_and_targets_outside(ct):
    x, table, target, grad = ce_tensors(seeded(4), 9, 24, 50, torch.float32)
    target[3] = 7
    ce_check(ct, x, table, target, grad, ignore=7)
    target[1], target[5] = 50, -1
    losses, lse = ct.cross_entropy_forward(x, table, target)
    want, lse64 = ref.cross_entropy(x, table, target)
    assert torch.isnan(losses).cpu().tolist() == torch.isnan(want).tolist() == [i in (1, 5) for i in range(9)]
    assert torch.isfinite(lse).all()
    dx, dtable = ct.cross_entropy_backward(grad, x, table, target, lse)
    assert torch.isnan(dx).any(1).cpu().tolist() == [i in (1, 5) for i in range(9)]


@pytest.mark.parametrize("dtype", TYPES)
def test_cross_entropy_large_and_equal_logits(ct, dtype):
    width, vocab = 16, 700
    x = torch.zeros(4, width, device=DEV, dtype=dtype)
    table = torch.zeros(vocab, width, device=DEV, dtype=dtype)
    table[:, 0] = 100
    table[5, 0], table[600, 0] = 120, -120
    x[0, 0], x[1, 0], x[2, 0] = 100, -100, 1          # logits of 1e4, both signs; row 3: all equal
    target = torch.tensor([5, 600, 0, 3], device=DEV)
    ce_check(ct, x, table, target, torch.ones(4, device=DEV))
    losses, lse = ct.cross_entropy_forward(x, table, target)
    assert losses[0] == 0 and losses[1] == 0
    assert abs(lse[3].item() - torch.log(torch.tensor(float(vocab))).item()) < 1e-5


def test_cross_entropy_infinite_and_nan_inputs_stay_in_their_rows(ct):
    x, table, target, grad = ce_tensors(seeded(6), 5, 20, 300, torch.float32)
    x[1, 2], x[3, 0] = float("nan"), float("inf")
    losses, lse = ct.cross_entropy_forward(x, table, target)
    assert not torch.isfinite(losses[1]) and not torch.isfinite(losses[3])
    assert torch.isfinite(losses[[0, 2, 4]]).all() and torch.isfinite(lse[[0, 2, 4]]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_cross_entropy_layouts(ct, dtype):
    x, table, target, grad = ce_tensors(seeded(9), 45, 56, 310, dtype, 0.2)
    want = ct.cross_entropy_forward(x, table, target)
    grads = ct.cross_entropy_backward(grad, x, table, target, want[1])
    for at in (0, 1, 8):
        def inside(t):
            wide = torch.full((t.shape[0], t.shape[1] + 11), float("nan"), dtype=dtype, device=DEV)
            wide[:, at:at + t.shape[1]] = t
            return wide[:, at:at + t.shape[1]]
        got = ct.cross_entropy_forward(inside(x), inside(table), target)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for g, w in zip(ct.cross_entropy_backward(grad, inside(x), inside(table), target, got[1]), grads):
            assert torch.equal(g, w)
    got = ct.cross_entropy_forward(x.view(9, 5, 56), table.t().contiguous().t(), target.view(9, 5))
    assert torch.equal(got[0].view(-1), want[0])
    assert torch.equal(ct.cross_entropy_backward(grad[:1].expand(45), x, table, target, want[1])[0],
                       ct.cross_entropy_backward(grad[:1].repeat(45), x, table, target, want[1])[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_cross_entropy_no_rows(ct, dtype):
    x, table, target, grad = ce_tensors(seeded(1), 0, 12, 31, dtype)
    losses, lse = ct.cross_entropy_forward(x, table, target)
    dx, dtable = ct.cross_entropy_backward(grad, x, table, target, lse)
    assert losses.shape == (0,) and dx.shape == (0, 12)
    assert torch.equal(dtable, torch.zeros_like(table))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-6, 1.0, 3e4])
def test_cross_entropy_gradient_scales(ct, dtype, size):
    """Gradients of the logits far below and above a 16-bit float's normal range keep their precision."""
    x, table, target, _ = ce_tensors(seeded(2), 20, 32, 3000, dtype)
    grad = torch.full((20,), size, device=DEV)
    lse = ct.cross_entropy_forward(x, table, target)[1]
    dx, dtable = ct.cross_entropy_backward(grad, x, table, target, lse)
    dx64, dt64, sx, st, _, _ = ref.cross_entropy_grad(grad, x, table, target)
    tol = 2.1 * ref.U[dtype] + 1e-3
    least = 2.0 ** -24 if dtype == torch.float16 else 0.0
    top = 65504.0 if dtype == torch.float16 else float("inf")
    for name, g, w, s in (("dx", dx, dx64, sx), ("dtable", dtable, dt64, st)):
        fits = w.abs() < top * 0.99
        ref.check(torch.where(fits.to(DEV), g, 0), torch.where(fits, w, 0), s * tol + least, 1.0, name)


def test_cross_entropy_table_offsets_beyond_32_bits(ct):
    vocab, width = (1 << 31) // 512 + 300, 512
    table = torch.zeros(vocab, width, dtype=torch.bfloat16, device=DEV)
    gen = seeded(1)
    table[-200:] = normal(gen, 200, width, std=0.1, dtype=torch.bfloat16)
    x = normal(gen, 3, width, dtype=torch.bfloat16)
    target = torch.tensor([vocab - 1, 5, vocab - 150], device=DEV)
    losses, lse = ct.cross_entropy_forward(x, table, target)
    z = ref.d(x) @ ref.d(table[-200:]).T
    s = torch.log(torch.exp(z).sum(1) + (vocab - 200))
    picked = torch.stack([z[0, 199], torch.zeros((), dtype=torch.float64), z[2, 50]])
    ref.check(lse, s, torch.ones(3), 1e-4, "lse")
    ref.check(losses, s - picked, torch.ones(3), 1e-4, "losses")
    dx, dtable = ct.cross_entropy_backward(torch.ones(3, device=DEV), x, table, target, lse)
    p = torch.exp(z - s[:, None])
    p[0, 199] -= 1
    p[2, 50] -= 1
    ref.check(dtable[-200:], p.T @ ref.d(x), p.abs().T @ ref.d(x).abs(), 2.0 ** -6, "dtable")
    ref.check(dx, p @ ref.d(table[-200:]), p.abs() @ ref.d(table[-200:]).abs(), 2.0 ** -6, "dx")


def test_cross_entropy_of_more_rows_than_one_launch_has_workgroups(ct):
    # a table of more than 2^24 rows that has to be laid out (bfloat16 of an odd width); equal logits but for a few rows
    vocab, width, rows = (1 << 24) + 77, 3, 20
    gen = seeded(2)
    table = torch.zeros(vocab, width, dtype=torch.bfloat16, device=DEV)
    table[-50:] = normal(gen, 50, width, dtype=torch.bfloat16)
    x = normal(gen, rows, width, std=3.0, dtype=torch.bfloat16)
    target = torch.arange(vocab - rows, vocab, device=DEV)
    losses, lse = ct.cross_entropy_forward(x, table, target)
    z = ref.d(x) @ ref.d(table[-50:]).T
    s = torch.log(torch.exp(z).sum(1) + (vocab - 50))
    at = torch.arange(rows)
    ref.check(lse, s, torch.ones(rows), 1e-4, "lse")
    ref.check(losses, s - z[at, 50 - rows + at], torch.ones(rows), 1e-4, "losses")
    dx, dtable = ct.cross_entropy_backward(torch.ones(rows, device=DEV), x, table, target, lse)
    p = torch.exp(z - s[:, None])
    p[at, 50 - rows + at] -= 1
    ref.check(dx, p @ ref.d(table[-50:]), p.abs() @ ref.d(table[-50:]).abs(), 2.0 ** -6, "dx")
    ref.check(dtable[-50:], p.T @ ref.d(x), p.abs().T @ ref.d(x).abs(), 2.0 ** -6, "dtable")


def test_cross_entropy_of_more_vectors_than_one_launch_has_workgroups(ct):
    rows = (1 << 24) + 99
    gen = seeded(3)
    x = torch.zeros(rows, 1, dtype=torch.bfloat16, device=DEV)
    x[-40:] = normal(gen, 40, 1, dtype=torch.bfloat16)
    table = normal(gen, 2, 1, dtype=torch.bfloat16)
    target = torch.zeros(rows, dtype=torch.int64, device=DEV)
    losses, lse = ct.cross_entropy_forward(x, table, target)
    z = ref.d(x[-40:]) @ ref.d(table).T
    s = torch.logsumexp(z, 1)
    ref.check(lse[-40:], s, torch.ones(40), 1e-5, "lse")
    ref.check(losses[-40:], s - z[:, 0], torch.ones(40), 1e-5, "losses")
    grad = torch.zeros(rows, device=DEV)
    grad[-40:] = 1.0
    dx, dtable = ct.cross_entropy_backward(grad, x, table, target, lse)
    p = torch.exp(z - s[:, None])
    p[:, 0] -= 1
    ref.check(dx[-40:], p @ ref.d(table), p.abs() @ ref.d(table).abs(), 2.0 ** -6, "dx")
    ref.check(dtable, p.T @ ref.d(x[-40:]), p.abs().T @ ref.d(x[-40:]).abs(), 2.0 ** -6, "dtable")
    assert not dx[:-40].any()


def test_cross_entropy_of_more_tiles_than_one_launch_has(ct):
    # 64 x 65538 tiles of 256 x 256: two launches
    rows, vocab, width = 16384, (1 << 24) + 300, 8
    gen = seeded(4)
    table = torch.zeros(vocab, width, dtype=torch.bfloat16, device=DEV)
    some = torch.cat([torch.arange(100, 120), torch.arange((1 << 23) - 300, (1 << 23) + 600, 15), torch.arange(vocab - 40, vocab)])
    table[some.to(DEV)] = normal(gen, len(some), width, dtype=torch.bfloat16)
    x = normal(gen, rows, width, std=2.0, dtype=torch.bfloat16)
    at = torch.randint(len(some), (rows,), generator=gen)
    losses, lse = ct.cross_entropy_forward(x, table, some[at].to(DEV))
    z = ref.d(x) @ ref.d(table[some.to(DEV)]).T
    top = z.amax(1).clamp(min=0)
    s = top + torch.log(torch.exp(z - top[:, None]).sum(1) + (vocab - len(some)) * torch.exp(-top))
    ref.check(lse, s, torch.ones(rows), 1e-4, "lse")
    ref.check(losses, s - z[torch.arange(rows), at], torch.ones(rows), 1e-4, "losses")


# ---- gradients against differences, autograd -------------------------------------------


def along(f, at, direction, step):
    return (f(at + step * direction) - f(at - step * direction)) / (2 * step)


def test_gradients_against_differences(ct):
    """float32 gradients along random directions against central differences of the 64-bit definition, whose own error
    is of the order of step^2 = 1e-8."""
    gen = seeded(21)
    x, gate, up, down, dy = mlp_tensors(gen, 6, 20, 28, torch.float32)
    w, b = normal(gen, 20), normal(gen, 20)
    y, mean, rstd = ct.layer_norm_forward(x, w, b)
    dx, dw, db = ct.layer_norm_backward(dy, x, w, mean, rstd)
    r = ref.d(dy)
    for got, at, f in ((dx, x, lambda t: (ref.layer_norm(t, w, b, 1e-5)[0] * r).sum()),
                       (dw, w, lambda t: (ref.layer_norm(x, t, b, 1e-5)[0] * r).sum()),
                       (db, b, lambda t: (ref.layer_norm(x, w, t, 1e-5)[0] * r).sum())):
        v = torch.randn(at.shape, generator=gen, dtype=torch.float64)
        want = along(f, ref.d(at), v, 1e-4)
        assert abs((ref.d(got) * v).sum() - want) <= 1e-4 * (1 + abs(want))
    for act in ("silu", "gelu", ref.CUBIC):
        y, saved = ct.gated_mlp_forward(x, gate, up, down, act)
        grads = ct.gated_mlp_backward(dy, x, gate, up, down, saved, act)
        args = [x, gate, up, down]
        for k, got in enumerate(grads):
            v = torch.randn(args[k].shape, generator=gen, dtype=torch.float64)
            want = along(lambda t: (ref.mlp(*[ref.d(a) if i != k else t for i, a in enumerate(args)], act) * r).sum(), ref.d(args[k]), v, 1e-4)
            assert abs((ref.d(got) * v).sum() - want) <= 1e-4 * (1 + abs(want))
    x, table, target, grad = ce_tensors(gen, 11, 20, 90, torch.float32, 0.2)
    lse = ct.cross_entropy_forward(x, table, target)[1]
    dx, dtable = ct.cross_entropy_backward(grad, x, table, target, lse)
    for got, at, f in ((dx, x, lambda t: (ref.cross_entropy(t, table, target)[0] * ref.d(grad)).sum()),
                       (dtable, table, lambda t: (ref.cross_entropy(x, t, target)[0] * ref.d(grad)).sum())):
        v = torch.randn(at.shape, generator=gen, dtype=torch.float64)
        want = along(f, ref.d(at), v, 1e-4)
        assert abs((ref.d(got) * v).sum() - want) <= 1e-4 * (1 + abs(want))


def test_autograd(ct):
    gen = seeded(30)
    x, gate, up, down, dy = (t.requires_grad_() for t in mlp_tensors(gen, 10, 24, 32, torch.float32))
    w, b = normal(gen, 24).requires_grad_(), normal(gen, 24).requires_grad_()
    table, target = normal(gen, 70, 24).requires_grad_(), torch.randint(70, (2, 5), generator=gen).to(DEV)
    target[1, 3] = -100
    n = ct.layer_norm(x, w, b)
    out = x + ct.gated_mlp(n, gate, up, down, ref.CUBIC)
    loss = ct.cross_entropy(out.view(2, 5, 24), table, target)
    loss.backward()
    n1, mean, rstd = ct.layer_norm_forward(x.detach(), w.detach(), b.detach())
    y1, saved = ct.gated_mlp_forward(n1, gate.detach(), up.detach(), down.detach(), ref.CUBIC)
    o1 = x.detach() + y1
    losses, lse = ct.cross_entropy_forward(o1, table.detach(), target.view(-1))
    assert torch.allclose(loss, losses.sum() / 9, rtol=1e-6)
    do, dt = ct.cross_entropy_backward(torch.full((10,), 1.0, device=DEV) / 9, o1, table.detach(), target.view(-1), lse)
    dn, dg, du, dd = ct.gated_mlp_backward(do, n1, gate.detach(), up.detach(), down.detach(), saved, ref.CUBIC)
    dx, dw, db = ct.layer_norm_backward(dn, x.detach(), w.detach(), mean, rstd)
    for got, want in ((table.grad, dt), (gate.grad, dg), (up.grad, du), (down.grad, dd), (w.grad, dw), (b.grad, db), (x.grad, do + dx)):
        assert torch.allclose(got, want, rtol=1e-5, atol=1e-8)
    with torch.no_grad():
        assert torch.equal(ct.cross_entropy(out, table, target.view(-1), reduction="none"), losses)
        assert ct.cross_entropy(out, table, torch.full((10,), -100, device=DEV)).item() == 0.0


# ---- streams, graphs, repetition ---------------------------------------------------------


def steps(ct, gen_seed=40, dtype=torch.bfloat16):
    gen = seeded(gen_seed)
    x, gate, up, down, dy = mlp_tensors(gen, 150, 72, 200, dtype)
    w, b = normal(gen, 72, dtype=dtype), normal(gen, 72, dtype=dtype)
    _, table, target, grad = ce_tensors(gen, 150, 72, 900, dtype, 0.2)

    def step():
        n, mean, rstd = ct.layer_norm_forward(x, w, b)
        y, saved = ct.gated_mlp_forward(n, gate, up, down)
        losses, lse = ct.cross_entropy_forward(y, table, target)
        dy, dt = ct.cross_entropy_backward(grad, y, table, target, lse)
        grads = ct.gated_mlp_backward(dy, n, gate, up, down, saved)
        return [n, y, losses, lse, dt, *grads, *ct.layer_norm_backward(grads[0], x, w, mean, rstd)]
    return step, (x, table)


@pytest.mark.parametrize("dtype", TYPES)
def test_same_result_every_time_and_on_another_stream(ct, dtype):
    step, _ = steps(ct, dtype=dtype)
    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    for a, b, c in zip(first, second, step()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_graph_replays(ct):
    step, (x, table) = steps(ct)
    for _ in range(2):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        x.mul_(0.9)
        table.add_(0.01)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b), k


# ---- refusals ---------------------------------------------------------------------------


def test_refusals(ct):
    gen = seeded(1)
    x, gate, up, down, dy = mlp_tensors(gen, 4, 8, 12, torch.float32)
    w = normal(gen, 8)
    with pytest.raises(ValueError, match="not on the GPU"):
        ct.layer_norm(x.cpu(), w)
    with pytest.raises(ValueError, match="float64"):
        ct.layer_norm(x.double(), w.double())
    with pytest.raises(ValueError, match="weight"):
        ct.layer_norm(x, w[:7])
    with pytest.raises(ValueError, match="weight"):
        ct.layer_norm(x, w.half())
    with pytest.raises(ValueError, match="bias"):
        ct.layer_norm(x.half(), w.half(), w)
    y, mean, rstd = ct.layer_norm_forward(x, w)
    with pytest.raises(ValueError, match="grad"):
        ct.layer_norm_backward(dy[:3], x, w, mean, rstd)
    with pytest.raises(ValueError, match="mean"):
        ct.layer_norm_backward(dy, x, w, mean[:3], rstd)
    with pytest.raises(ValueError, match="up: 11 rows"):
        ct.gated_mlp(x, gate, up[:11], down)
    with pytest.raises(ValueError, match="down"):
        ct.gated_mlp(x, gate, up, down[:, :11])
    with pytest.raises(ValueError, match="gate"):
        ct.gated_mlp(x, gate.half(), up, down)
    with pytest.raises(ValueError, match="tanh"):
        ct.gated_mlp(x, gate, up, down, "tanh")
    with pytest.raises(ValueError, match="four coefficients"):
        ct.gated_mlp(x, gate, up, down, (1.0, 2.0))
    _, saved = ct.gated_mlp_forward(x, gate, up, down)
    with pytest.raises(ValueError, match="saved"):
        ct.gated_mlp_backward(dy, x, gate, up, down, saved[:, :3])
    target = torch.zeros(4, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="target"):
        ct.cross_entropy(x, gate, target.int())
    with pytest.raises(ValueError, match="target"):
        ct.cross_entropy(x, gate, target[:3])
    with pytest.raises(ValueError, match="table"):
        ct.cross_entropy(x, gate[:0], target)
    with pytest.raises(ValueError, match="last dimension"):
        ct.cross_entropy(x[:, :7], gate, target)
    with pytest.raises(ValueError, match="reduction"):
        ct.cross_entropy(x, gate, target, reduction="median")
    assert torch.isfinite(ct.cross_entropy(x, gate, target))


def test_workspace_refusals(ct):
    from helrm_amd.backend import LayerNormArgs
    gen = seeded(1)
    x, w = normal(gen, 4, 8), normal(gen, 8)
    mean, rstd = torch.zeros(2, 4, device=DEV)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    a = LayerNormArgs(x=x.data_ptr(), ldx=8, weight=w.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(), dy=x.data_ptr(), lddy=8,
                      dx=dx.data_ptr(), lddx=8, dweight=dw.data_ptr(), rows=4, width=8)
    space = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    a.workspace, a.workspaceBytes = space.data_ptr(), 16
    with pytest.raises(HipError, match="workspace too small"):
        ct._call("LayerNormGrad", a, x.device)
    a.workspace, a.workspaceBytes = space.data_ptr() + 8, space.numel() - 8
    with pytest.raises(HipError, match="aligned"):
        ct._call("LayerNormGrad", a, x.device)
