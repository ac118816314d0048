"""The cleartext operators at the limits of a launch and of a type, against
plain 64-bit implementations.  Bounds as in cleartext_ref."""
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
