"""The cleartext operators at the limits of a launch and of a type, against
plain 64-bit implementations.  Bounds as in cleartext_ref."""
import ctypes

import pytest
import torch

import cleartext_ref as ref
from test_gpu_cleartext import DEV, F32, ce_tensors, ct, mlp_tensors, normal, seeded  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2])
def test_layer_norm_of_more_columns_than_one_launch_sums(ct, rows):  # noqa: F811
    # the sums of the weights' gradients, 1,024 threads for 16 columns, would be 2^32 threads and some
    width = (1 << 26) + 9
    gen = torch.Generator(DEV).manual_seed(rows)
    x, dy = (torch.randn(rows, width, generator=gen, device=DEV).bfloat16() for _ in range(2))
    w = (1 + 0.1 * torch.randn(width, generator=gen, device=DEV)).bfloat16()
    y, mean, rstd = ct.layer_norm_forward(x, w, w)
    dx, dw, db = ct.layer_norm_backward(dy, x, w, mean, rstd)
    x, w, dy = x.double(), w.double(), dy.double()
    var, mu = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    r = (var + 1e-5).rsqrt()
    h, t = (x - mu) * r, dy * w
    slop, u = (width / 256 + 30) * F32, ref.U[torch.bfloat16]      # 256 threads' sums
    want = r * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
    for name, got, value, size in (("y", y, h * w + w, (1 + h.abs()) * w.abs()), ("dx", dx, want, t.abs() + 1 + h.abs()),
                                   ("dw", dw, (dy * h).sum(0), (dy.abs() * (1 + h.abs())).sum(0)), ("db", db, dy.sum(0), dy.abs().sum(0) * F32)):
        assert ((got.double() - value).abs() <= size * slop + u * value.abs()).all(), name


def test_cross_entropy_of_small_tiles_in_several_launches(ct):  # noqa: F811
    # 17 rows take tiles of 128 x 128, 2^23 and 3 of them, in three launches; equal logits but for a few rows
    rows, vocab, width = 17, (1 << 30) + 300, 8
    gen = seeded(5)
    table = torch.zeros(vocab, width, dtype=torch.bfloat16, device=DEV)
    some = torch.cat([torch.arange(100, 120), torch.arange((1 << 28) - 300, (1 << 28) + 600, 15), torch.arange((1 << 29) - 200, (1 << 29) + 200, 9),
                      torch.arange(3 << 28, (3 << 28) + 40), torch.arange(vocab - 40, vocab)])
    table[some.to(DEV)] = normal(gen, len(some), width, std=3.0, dtype=torch.bfloat16)
    x = normal(gen, rows, width, std=2.0, dtype=torch.bfloat16)
    at = torch.randint(len(some), (rows,), generator=gen)
    losses, lse = ct.cross_entropy_forward(x, table, some[at].to(DEV))
    z = ref.d(x) @ ref.d(table[some.to(DEV)]).T
    s = torch.logsumexp(torch.cat([z, torch.full((rows, 1), float(vocab - len(some)), dtype=torch.float64).log()], 1), 1)
    ref.check(lse, s, torch.ones(rows), 1e-4, "lse")
    ref.check(losses, s - z[torch.arange(rows), at], torch.ones(rows), 1e-4, "losses")


def test_cross_entropy_of_more_vectors_than_one_launch_has_waves(ct):  # noqa: F811
    # a wave a row would be 2^32 threads and some
    rows = (1 << 26) + 37
    gen = seeded(6)
    x = torch.zeros(rows, 1, dtype=torch.bfloat16, device=DEV)
    table = normal(gen, 2, 1, dtype=torch.bfloat16)
    some = torch.cat([torch.arange(70), torch.arange((1 << 25) - 10, (1 << 25) + 10), torch.arange(rows - 70, rows)])
    x[some.to(DEV)] = normal(gen, len(some), 1, dtype=torch.bfloat16)
    target = torch.ones(rows, dtype=torch.int64, device=DEV)
    losses, lse = ct.cross_entropy_forward(x, table, target)
    z = ref.d(x[some.to(DEV)]) @ ref.d(table).T
    s = torch.logsumexp(z, 1)
    ref.check(lse[some.to(DEV)], s, torch.ones(len(some)), 1e-5, "lse")
    ref.check(losses[some.to(DEV)], s - z[:, 1], torch.ones(len(some)), 1e-5, "losses")
    empty = torch.ones(rows, dtype=torch.bool, device=DEV)
    empty[some.to(DEV)] = False
    assert ((losses[empty] - 0.6931472).abs() < 1e-6).all() and ((lse[empty] - 0.6931472).abs() < 1e-6).all()


# ---- infinities, the types' lowest values, overflow ------------------------------------


def special_check(got, want, size, tol, what):
    """The infinities and NaN of `want`; what is finite there within tol * size."""
    got, want = ref.d(got), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in the wrong places"
    assert torch.equal(torch.where(torch.isinf(got), got, 0), torch.where(torch.isinf(want), want, 0)), f"{what}: infinities"
    fine = torch.isfinite(want)
    ref.check(torch.where(fine, got, 0), torch.where(fine, want, 0), torch.where(fine, size, 0), tol, what)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [3, 40, 70, 300])
@pytest.mark.parametrize("mask", ["-inf", "lowest", "near"])
def test_cross_entropy_of_table_rows_masked_through_a_constant_coordinate(ct, dtype, rows, mask):  # noqa: F811
    width, vocab, column = 33, 700, 7
    x, table, target, grad = ce_tensors(seeded(rows), rows, width, vocab, dtype)
    low = torch.finfo(dtype).min
    value = {"-inf": float("-inf"), "lowest": low, "near": low * (1 - 2.0 ** -12) if dtype == torch.float32 else low / 2}[mask]
    gone = torch.arange(vocab) % 3 == 1
    x[:, column] = 1.0
    table[:, column] = 0
    table[gone.to(DEV), column] = value
    target = target // 3 * 3
    losses, lse = ct.cross_entropy_forward(x, table, target)
    dx, dtable = ct.cross_entropy_backward(grad, x, table, target, lse)
    # the same without the masked rows
    left = table.cpu()[~gone]
    at = (torch.cumsum(~gone, 0) - 1)[target.cpu()]
    l64, s64 = ref.cross_entropy(x, left, at)
    logit = (width + 12) * F32 * (ref.d(x).abs() @ ref.d(left).abs().T).amax().item()
    off = logit * 2 + (12 + vocab / 64) * F32 * (1 + s64.abs())
    ref.check(losses, l64, off, 1.0, "losses")
    ref.check(lse, s64, off, 1.0, "lse")
    dx64, dt64, sx, st, px, pt = ref.cross_entropy_grad(grad, x, left, at)
    tol, soft = (vocab + rows + 60) * F32 + 2.1 * ref.U[dtype], 4 * logit + 8 * F32
    least = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126
    assert not dtable.cpu()[gone].any()
    ref.check(dtable.cpu()[~gone], dt64, st * tol + pt * soft + least, 1.0, "dtable")
    if mask == "-inf":      # 0 times an infinity
        assert torch.isnan(dx[:, column]).all()
        dx[:, column] = 0
        dx64[:, column] = 0
    ref.check(dx, dx64, sx * tol + px * soft + least, 1.0, "dx")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 17, 40, 70, 300])
@pytest.mark.parametrize("where", ["gate", "up", "down", "x", "grad"])
def test_gated_mlp_with_one_infinite_factor(ct, dtype, rows, where):  # noqa: F811
    x, gate, up, down, dy = mlp_tensors(seeded(rows), rows, 24, 40, dtype)
    x[:, 5] = x[:, 5].abs() + 0.5
    {"gate": gate, "up": up, "down": down, "x": x, "grad": dy}[where][min(rows - 1, 2) if where in ("x", "grad") else 2, 5] = float("inf")
    y, saved = ct.gated_mlp_forward(x, gate, up, down, "silu")
    got = (y, *ct.gated_mlp_backward(dy, x, gate, up, down, saved, "silu"))
    want = (ref.mlp(x, gate, up, down, "silu"), *ref.mlp_grad(dy, x, gate, up, down, "silu"))
    u = ref.U[dtype]
    tol = 2 * (2 * 24 + 40 + rows + 40) * F32 + 2.1 * u
    least = 2.0 ** -24 * (1 + 40 + rows) * 4 / (2.1 * u) if dtype == torch.float16 else 0.0
    for name, g, w, size in zip(("y", "dx", "dgate", "dup", "ddown"), got, want, ref.mlp_sizes(dy, x, gate, up, down, "silu")):
        special_check(g, w, size + least, tol, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 17, 40, 70, 300])
def test_gated_mlp_with_a_weight_of_the_types_largest_value(ct, dtype, rows):  # noqa: F811
    x, gate, up, down, dy = mlp_tensors(seeded(rows), rows, 24, 40, dtype)
    x *= 0.25
    down[2, 5] = torch.finfo(dtype).max
    y = ct.gated_mlp(x, gate, up, down, "silu")
    assert torch.isfinite(y).all()
    ref.check(y, ref.mlp(x, gate, up, down, "silu"), ref.mlp_sizes(dy, x, gate, up, down, "silu")[0], 2 * (2 * 24 + 40 + 40) * F32 + 2.1 * ref.U[dtype], "y")


@pytest.mark.parametrize("rows", [3, 40, 70, 300])
def test_products_beyond_float32_are_infinite(ct, rows):  # noqa: F811
    # 10^30 times weights of 10^15 and less: the corrections overflow too, with either sign
    x, gate, up, down, _ = mlp_tensors(seeded(rows), rows, 24, 40, torch.float32)
    x[:, 4] *= 1e30
    gate[::2, 4] *= 1e15
    gate[1::4, 4] *= 1e8
    _, saved = ct.gated_mlp_forward(x, gate, up, down, "silu")
    want = ref.d(x) @ ref.d(gate).T
    want[want.abs() > torch.finfo(torch.float32).max] *= float("inf")
    assert torch.isinf(want).any() and torch.isfinite(want).any()
    special_check(saved[0], want, ref.d(x).abs() @ ref.d(gate).abs().T, 2.0 ** -20, "g")


@pytest.mark.parametrize("rows", [3, 40, 70, 136, 300])
def test_float32_products_are_as_exact_as_float32s(ct, rows):  # noqa: F811
    """One term in every sum but dx's: each of the products' six parts counts.  A product is off by what the three left
    out come to, 1.5 2^-23 at most, and two roundings; y and the weights' gradients are three products behind one another."""
    n = 136
    gen = seeded(rows)
    x, dy, down = torch.zeros(rows, n), torch.zeros(rows, n), torch.zeros(n, n)
    x[torch.arange(rows), torch.randint(n, (rows,), generator=gen)] = torch.randn(rows, generator=gen)
    dy[rows // 2] = torch.randn(n, generator=gen)
    down[torch.arange(n), torch.randperm(n, generator=gen)] = torch.randn(n, generator=gen)
    gate, up = normal(gen, n, n), normal(gen, n, n)
    x, dy, down, act = x.to(DEV), dy.to(DEV), down.to(DEV), (8.0, 0.25, 0.0, 0.0)
    y, saved = ct.gated_mlp_forward(x, gate, up, down, act)
    for got, w in zip(saved, (gate, up)):
        want = ref.d(x) @ ref.d(w).T
        ref.check(got, want, want.abs(), 1.25 * 2.0 ** -22, "a projection")
    _, *got = ct.gated_mlp_backward(dy, x, gate, up, down, saved, act)
    _, *want = ref.mlp_grad(dy, x, gate, up, down, act)
    for name, g, w in zip(("y", "dgate", "dup", "ddown"), (y, *got), (ref.mlp(x, gate, up, down, act), *want)):
        ref.check(g, w, w.abs(), 2.0 ** -19, name)


# ---- forward mode -----------------------------------------------------------------------


@pytest.mark.parametrize("which", range(12))
def test_no_tensor_with_a_tangent_is_taken(ct, which):  # noqa: F811
    from torch.autograd import forward_ad
    x, gate, up, down, dy = mlp_tensors(seeded(1), 4, 8, 12, torch.float32)
    w, b = normal(seeded(2), 8), normal(seeded(3), 8)
    target = torch.zeros(4, dtype=torch.int64, device=DEV)
    _, mean, rstd = ct.layer_norm_forward(x, w, b)
    _, saved = ct.gated_mlp_forward(x, gate, up, down)
    losses, lse = ct.cross_entropy_forward(x, gate, target)
    calls = [(ct.layer_norm, [x, w, b]), (ct.gated_mlp, [x, gate, up, down]), (ct.cross_entropy, [x, gate, target]),
             (lambda g: ct.layer_norm_backward(g, x, w, mean, rstd), [dy]), (lambda g: ct.gated_mlp_backward(g, x, gate, up, down, saved), [dy]),
             (lambda g: ct.cross_entropy_backward(g, x, gate, target, lse), [losses])]
    call, args, k = [(f, a, k) for f, a in calls for k in range(len(a)) if a[k] is not target][which % 12]
    with forward_ad.dual_level():
        args[k] = forward_ad.make_dual(args[k], torch.ones_like(args[k]))
        with pytest.raises(NotImplementedError, match="tangent"):
            call(*args)


# ---- leading dimensions -----------------------------------------------------------------


def test_gradients_of_other_leading_dimensions(ct):  # noqa: F811
    x, gate, up, down, dy = mlp_tensors(seeded(1), 45, 8, 12, torch.float32)
    w, target = normal(seeded(2), 8), torch.arange(45, device=DEV) % 12
    _, mean, rstd = ct.layer_norm_forward(x, w)
    _, saved = ct.gated_mlp_forward(x, gate, up, down)
    losses, lse = ct.cross_entropy_forward(x, gate, target)

    def calls(x, dy, losses, lse):
        return [lambda: ct.layer_norm_backward(dy, x, w, mean, rstd), lambda: ct.gated_mlp_backward(dy, x, gate, up, down, saved),
                lambda: ct.cross_entropy_backward(losses, x, gate, target, lse)]

    want = [call() for call in calls(x, dy, losses, lse)]
    for lead in ((9, 5), (45,), (1, 45), (9, 1, 5)):
        for other in (lead, (45,)):
            for got, w_ in zip(calls(x.view(*other, 8), dy.view(*lead, 8), losses.view(lead), lse.view(lead)), want):
                got = got()
                assert got[0].shape == (*other, 8) and all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, w_))
    x = x.view(9, 5, 8)
    for call in calls(x, dy.view(5, 9, 8), losses.view(5, 9), lse) + [lambda: ct.cross_entropy_backward(losses, x, gate, target, lse.view(5, 9))]:
        with pytest.raises(ValueError, match="leading dimensions"):
            call()


# ---- errors of others -------------------------------------------------------------------


def test_an_error_of_an_earlier_call_is_not_the_operators(ct):  # noqa: F811
    # an allocation that fails leaves its error behind until somebody asks for the last one
    # (torch's own kernels, copies among them, ask for it, and so there are none in these calls)
    x, w, down = normal(seeded(1), 4, 8), normal(seeded(2), 8), normal(seeded(3), 8, 4)
    want = ct.layer_norm(x, w)
    with open("/proc/self/maps") as f:
        hip = ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64.so" in line))
    hip.hipMalloc.argtypes = [ctypes.c_void_p, ctypes.c_size_t]
    for call in (lambda: ct.layer_norm(x, w), lambda: ct.gated_mlp(x, x, x, down)):
        pointer = ctypes.c_void_p()
        assert hip.hipMalloc(ctypes.byref(pointer), 1 << 60) != 0
        call()
    assert torch.equal(ct.layer_norm(x, w), want)


# ---- the mean and the sum of the losses -----------------------------------------------------


@pytest.mark.parametrize("rows", [0, 1, 5, 4095, 8191, 8192, 300001, (1 << 21) + 3])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_cross_entropy_totals(ct, rows, reduction):  # noqa: F811
    # 64-bit sums, one rounding (the losses as the operator leaves them)
    x, table, target, _ = ce_tensors(seeded(rows), rows, 8, 16, torch.float32, 0.3)
    losses = ct.cross_entropy(x, table, target, reduction="none")
    got = ct.cross_entropy(x.view(rows, 1, 8), table, target.view(rows, 1), reduction=reduction)
    n = max(1, int((target != -100).sum())) if reduction == "mean" else 1
    want = ref.d(losses).sum() / n
    ref.check(got, want, want.abs(), 2.0 ** -24 + 2.0 ** -40, reduction)
    x, table = x.requires_grad_(), table.requires_grad_()
    total = ct.cross_entropy(x, table, target, reduction=reduction)
    assert torch.equal(total, got)
    (2.0 * total).backward()
    lse = ct.cross_entropy_forward(x.detach(), table.detach(), target)[1]
    grad = torch.full((rows,), 2.0 / n, dtype=torch.float64, device=DEV).float()
    for a, b in zip((x.grad, table.grad), ct.cross_entropy_backward(grad, x.detach(), table.detach(), target, lse)):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-9)


def test_cross_entropy_totals_of_nothing_and_of_nan(ct):  # noqa: F811
    x, table, target, _ = ce_tensors(seeded(1), 20000, 8, 16, torch.float32)
    gone = torch.full_like(target, -100)
    for reduction in ("mean", "sum"):
        assert ct.cross_entropy(x, table, gone, reduction=reduction).item() == 0.0
        target[777] = 16                       # outside the table
        assert torch.isnan(ct.cross_entropy(x, table, target, reduction=reduction))
        assert ct.cross_entropy(x, table, gone, ignore_index=-100, reduction=reduction).item() == 0.0


@pytest.mark.parametrize("rows", [1000, 70000, 300000, 3000000])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_cross_entropy_totals_in_a_graph(ct, rows, reduction):  # noqa: F811
    # (with torch's sum every replay after the first had the first one's value, from some 100,000 rows on)
    x, table, target, _ = ce_tensors(seeded(rows), rows, 8, 16, torch.float32, 0.2)
    x, table = x.requires_grad_(), table.requires_grad_()

    def step():
        total = ct.cross_entropy(x, table, target, reduction=reduction)
        return (total, *torch.autograd.grad(total, (x, table)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.mul_(0.9)
            target[k::5] = -100
        want = step()
        torch.randn(1 << 22, device=DEV).sum()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k
