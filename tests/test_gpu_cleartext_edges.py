"""The cleartext operators at the limits of a launch and of a type, against
plain 64-bit implementations.  Bounds as in cleartext_ref."""
import pytest
import torch

import cleartext_ref as ref
from test_gpu_cleartext import DEV, F32, ce_tensors, ct, mlp_tensors, normal, seeded  # noqa: F401

pytestmark = pytest.mark.gpu


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
