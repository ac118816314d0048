"""The embedding and its gradient against a plain 64-bit implementation: types,
lengths from none to several tiles of the sort, runs of equal ids that end
anywhere, odd widths, strides, ids without a row, other streams and graphs.

Bounds: a row is one product and one rounding of it; a gradient is a sum of n
float32 terms, within (n + 1) 2^-24 of the sum of their absolute values, times
a scale (one rounding more), rounded once."""
import pytest
import torch

import cleartext_ref as ref
from helrm_amd.backend import HipError
from test_gpu_cleartext import DEV, F32, TYPES, ct, normal, seeded  # noqa: F401

pytestmark = pytest.mark.gpu

LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # half of it is a subnormal's rounding
IGNORE = -100


def heavy(gen, n, vocab):
    """Ids of which the first ones are common."""
    return (torch.exp(torch.rand(n, generator=gen, dtype=torch.float64) * torch.log(torch.tensor(float(vocab)))) - 1).long().clamp_(0, vocab - 1)


def want(ids, table, grad, scale, ignore=IGNORE):
    """(rows, gradient, sum of absolute values, terms of each row of the table)."""
    ids, table, grad = ids.cpu().reshape(-1), ref.d(table), ref.d(grad)
    rows = torch.zeros(len(ids), table.shape[1], dtype=torch.float64)
    inside = (ids >= 0) & (ids < len(table)) & (ids != ignore)
    rows[inside] = table[ids[inside]] * scale
    rows[~inside & (ids != ignore)] = float("nan")
    d, s, n = torch.zeros_like(table), torch.zeros_like(table), torch.zeros(len(table))
    d.index_add_(0, ids[inside], grad.reshape(-1, table.shape[1])[inside])
    s.index_add_(0, ids[inside], grad.reshape(-1, table.shape[1])[inside].abs())
    n.index_add_(0, ids[inside], torch.ones(int(inside.sum())))
    return rows, d * scale, s * abs(scale), n


def embed_check(ct, ids, table, grad, scale, ignore=IGNORE):  # noqa: F811
    scale = float(torch.tensor(scale))            # as the entry point takes it
    rows, d, s, n = want(ids, table, grad, scale, ignore)
    u, least = ref.U[table.dtype], LEAST[table.dtype]
    y = ct.embedding_forward(ids, table, scale, ignore)
    assert y.shape == (*ids.shape, table.shape[1]) and y.dtype == table.dtype
    ref.check(y.reshape(rows.shape), rows, rows.abs().nan_to_num(0) * (u + F32) + least, 1.0, "y")
    dtable = ct.embedding_backward(grad, ids, table.shape[0], scale, ignore)
    assert dtable.dtype == table.dtype and dtable.is_contiguous()
    ref.check(dtable, d, s * (n[:, None] + 2) * F32 + d.abs() * u + least, 1.0, "dtable")
    assert not dtable.cpu()[n == 0].any()
    assert torch.equal(ct.embedding_backward(grad, ids, table.shape[0], scale, ignore), dtable)
    return y, dtable


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,width,vocab", [(0, 8, 5), (1, 1, 1), (1, 512, 300), (3, 7, 2), (15, 8, 40), (16, 9, 3), (17, 16, 100), (65, 33, 64), (255, 2056, 30),
                                                (256, 12, 5000), (257, 12, 5000), (256, 20000, 3),
                                                (200, 416, 1000), (1000, 1001, 50), (1024, 3, 511), (1025, 64, 512), (700, 2048, 9000), (37, 4097, 20),
                                                (5000, 24, 4000), (5120, 24, 400), (5121, 24, 400), (8191, 5, 3), (8192, 16, 70000), (8193, 16, 300), (12289, 40, 260000), (16384, 24, 9000), (16385, 24, 9000),
                                                (20000, 4, 1), (30011, 130, 5000), (32768, 12, 70000), (32769, 12, 70000),
                                                (70001, 8, 600), (33000, 8, 65534),
                                                (33000, 8, 65535), (65536, 5, 300), (65535, 8, 65534), (65537, 5, 300)])
def test_embedding(ct, dtype, tokens, width, vocab):  # noqa: F811
    gen = seeded(tokens + 7 * width + vocab)
    table, grad = normal(gen, vocab, width, dtype=dtype), normal(gen, tokens, width, dtype=dtype)
    for k, ids in enumerate((torch.randint(vocab, (tokens,), generator=gen), heavy(gen, tokens, vocab))):
        if k:
            ids[torch.rand(tokens, generator=gen) < 0.2] = IGNORE
        embed_check(ct, ids.to(DEV), table, grad, (1.0, 5.6568542)[k])


@pytest.mark.parametrize("width", [4, 72, 1536])
def test_runs_that_end_anywhere(ct, width):  # noqa: F811
    # pieces are 16 to 64 ids: runs of every length about them, in an order of ids that is not theirs
    gen = seeded(width)
    lengths = [1, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 127, 128, 129, 1, 1, 200, 1000, 3, 2500, 5]
    ids = torch.cat([torch.full((n,), 3 * k) for k, n in enumerate(lengths)])
    for ids in (ids, ids[torch.randperm(len(ids), generator=gen)], torch.cat([ids, ids, ids]), ids[torch.randperm(len(ids), generator=gen)][:250]):
        embed_check(ct, ids.to(DEV), normal(gen, 70, width), normal(gen, len(ids), width), 1.0)


@pytest.mark.parametrize("width", [3, 24, 600])
def test_runs_over_groups_of_pieces(ct, width):  # noqa: F811
    # so many ids that pieces' sums are added in groups of 32 before: runs of about one, two and many groups, that begin and end anywhere
    gen = seeded(width)
    lengths = [1, 15, 500, 511, 512, 513, 1023, 1024, 1025, 3, 2000, 16, 16, 4096, 40, 9000, 30000, 1, 700, 700, 700, 20]
    ids = torch.cat([torch.full((n,), 2 * k) for k, n in enumerate(lengths)])
    ids = torch.cat([ids, 2 * len(lengths) + torch.arange(max(0, 66000 - len(ids))) // 3])
    for ids in (ids, ids[torch.randperm(len(ids), generator=gen)]):
        embed_check(ct, ids.to(DEV), normal(gen, int(ids.max()) + 2, width), normal(gen, len(ids), width), 1.0)


def test_a_run_over_groups_of_rows_wider_than_a_workgroup(ct):  # noqa: F811
    # the last pack of a row overlaps one of another turn's
    width = 1024 * 8 + 3
    n = 4200 * 64 + 5
    ids = torch.full((n,), 1)
    ids[::1000] = 0
    grad = torch.randn(n, width, generator=torch.Generator(DEV).manual_seed(1), device=DEV).bfloat16()
    d = ct.embedding_backward(grad, ids.to(DEV), 3)
    for v in (0, 1):
        rows = grad[(ids == v).to(DEV)]
        want, size = (sum(part.double().sum(0) for part in t.split(4096)) for t in (rows, rows.abs()))
        # a term is in at most 64 additions of its piece, 32 of its group and 132 of the groups
        assert ((d[v].double() - want).abs() <= size * 230 * F32 + want.abs() * ref.U[torch.bfloat16]).all()
    assert not d[2].any()


@pytest.mark.parametrize("more", [0, 500])
def test_equal_ids_are_added_in_their_order(ct, more):  # noqa: F811
    # 2^24 + 1 + 1 + ... in float32 stays 2^24, 1 + 1 + ... + 2^24 does not: each id's rows are in order within a piece
    ids = torch.tensor([4, 2] * 8 + [5] * more, device=DEV)
    grad = torch.ones(16 + more, 8, device=DEV)
    grad[0], grad[15] = 2.0 ** 24, 2.0 ** 24
    d = ct.embedding_backward(grad, ids, 6)
    assert (d[4] == 2.0 ** 24).all() and (d[2] == 2.0 ** 24 + 8).all()      # (7 + 2^24, to the even neighbour)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [50, 700, 9000])
def test_ids_without_a_row(ct, dtype, tokens):  # noqa: F811
    gen = seeded(tokens)
    table = normal(gen, 33, 40, dtype=dtype)
    ids = torch.randint(33, (tokens,), generator=gen)
    grad = normal(gen, tokens, 40, dtype=dtype)
    for k, bad in enumerate((IGNORE, 33, -1, 1 << 31, 1 << 32, (1 << 32) + 3, -(1 << 63), (1 << 63) - 1)):
        ids[k::11] = bad
        grad[k::11] = float("nan")                     # reaches nothing
    y, d = embed_check(ct, ids.to(DEV), table, grad, 2.0)
    assert torch.isfinite(d).all()
    # an ignore_index that is a row of the table: that row is zeros, and takes nothing back
    y, d = embed_check(ct, ids.clamp(0, 32).to(DEV), table, torch.nan_to_num(grad), 1.0, ignore=5)
    assert not y.cpu()[ids.clamp(0, 32) == 5].any() and not d[5].any()
    nothing = torch.full((tokens,), IGNORE, device=DEV)
    assert not ct.embedding(nothing, table).any() and not ct.embedding_backward(grad, nothing, 33).any()


def test_infinities_and_nan_stay_in_their_rows(ct):  # noqa: F811
    gen = seeded(3)
    table, grad = normal(gen, 10, 20), normal(gen, 300, 20)
    ids = torch.randint(9, (300,), generator=gen).to(DEV)
    ids[5], ids[6], ids[7] = 9, 9, 1
    table[2, 3], table[3, 0] = float("inf"), float("nan")
    grad[5, 1], grad[6, 1], grad[7, 2] = float("inf"), float("-inf"), float("nan")
    y, d = ct.embedding_forward(ids, table), ct.embedding_backward(grad, ids, 10)
    assert torch.equal(y.nan_to_num(7.0), table[ids].nan_to_num(7.0))
    where = torch.zeros(10, 20, dtype=torch.bool, device=DEV)
    where[9, 1] = where[1, 2] = True
    assert torch.equal(torch.isnan(d), where)


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(ct, dtype):  # noqa: F811
    gen = seeded(8)
    ids = torch.randint(30, (4, 6), generator=gen).to(DEV)
    wide, tall = normal(gen, 30, 131, dtype=dtype), normal(gen, 24, 131, dtype=dtype)
    for cut in ((slice(None), slice(0, 40)), (slice(None), slice(3, 43)), (slice(None), slice(1, 81, 2)), (slice(None), slice(1, 4))):
        table, grad = wide[cut], tall[cut]
        embed_check(ct, ids, table, grad.reshape(4, 6, -1), 1.5)
        embed_check(ct, ids.view(24), table, grad, 1.5)
    embed_check(ct, ids.t(), wide.t().contiguous().t()[:, :40], tall[:, :40].reshape(6, 4, 40), 1.0)
    embed_check(ct, ids[:1, :1].expand(4, 6), wide, tall[:1].expand(24, 131).view(4, 6, 131), 1.0)
    embed_check(ct, ids[::2, 1::2], wide[::2][:15].repeat(2, 1), tall[:6].view(2, 3, 131), 1.0)
    y = ct.embedding(ids[0, 0], wide)
    assert y.shape == (131,) and torch.equal(y, wide[ids[0, 0]])


def test_autograd(ct):  # noqa: F811
    gen = seeded(4)
    ids = torch.randint(50, (7, 9), generator=gen).to(DEV)
    ids[2, 3] = IGNORE
    table, grad = normal(gen, 50, 12), normal(gen, 7, 9, 12)
    leaf = table.clone().requires_grad_()
    y = ct.embedding(ids, leaf, 3.0)
    y.backward(grad)
    assert torch.equal(y, ct.embedding_forward(ids, table, 3.0))
    assert torch.equal(leaf.grad, ct.embedding_backward(grad, ids, 50, 3.0))
    # a gradient that one value stands for
    leaf.grad = None
    ct.embedding(ids, leaf).sum().backward()
    assert torch.equal(leaf.grad, ct.embedding_backward(torch.ones(7, 9, 12, device=DEV), ids, 50))
    assert not ct.embedding(ids, table).requires_grad
    with torch.no_grad():
        assert not ct.embedding(ids, leaf).requires_grad
    (g,) = torch.autograd.grad(ct.embedding(ids, leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


def test_against_differences(ct):  # noqa: F811
    gen = seeded(9)
    ids = torch.randint(6, (40,), generator=gen).to(DEV)
    table, weight, step = normal(gen, 6, 5), normal(gen, 40, 5), normal(gen, 6, 5)
    leaf = table.clone().requires_grad_()
    (ct.embedding(ids, leaf, 0.7).tanh() * weight).sum().backward()
    h = 2.0 ** -7
    up, down = ((ct.embedding(ids, table + k * h * step, 0.7).double().tanh() * weight).sum() for k in (1, -1))
    # third derivatives of tanh are at most 2: h^2 / 6 * 2 * sum |0.7 step|^3; three roundings of a row in each of the two sums; the gradient's own
    off = h * h / 3 * (0.343 * step.double().abs().pow(3)[ids] * weight.abs()).sum()
    off += ((0.7 * (table.abs() + step.abs()))[ids] * weight.abs()).double().sum() * 3 * F32 / h + (step[ids] * weight).abs().double().sum() * 64 * F32
    assert abs(((up - down) / (2 * h) - (leaf.grad.double() * step).sum()).item()) <= off.item()


def test_offsets_beyond_32_bits(ct):  # noqa: F811
    vocab, width = (1 << 31) // 1024 + 9, 1024
    gen = seeded(1)
    table = torch.zeros(vocab, width, dtype=torch.bfloat16, device=DEV)
    table[-5:] = normal(gen, 5, width, dtype=torch.bfloat16)
    ids = torch.randint(vocab - 5, vocab, (100,), generator=gen).to(DEV)
    assert torch.equal(ct.embedding(ids, table), table[ids])
    del table
    tokens = vocab
    grad = torch.zeros(tokens, width, dtype=torch.bfloat16, device=DEV)
    grad[-5:] = normal(gen, 5, width, dtype=torch.bfloat16)
    ids = torch.arange(tokens, device=DEV).flip(0)
    assert torch.equal(ct.embedding_backward(grad, ids, vocab), grad.flip(0))
    one = ct.embedding_backward(grad, torch.full_like(ids, 3), 5)         # one run over all pieces
    ref.check(one[3], ref.d(grad[-5:]).sum(0), ref.d(grad[-5:]).abs().sum(0), 6 * F32 + ref.U[torch.bfloat16], "dtable")
    assert not one[[0, 1, 2, 4]].any()


def test_more_tiles_than_a_workgroup_adds_up(ct):  # noqa: F811
    # 2^20 ids are 256 tiles of the sort
    tokens, width, vocab = (1 << 20) + 77, 4, 1 << 19
    gen = seeded(11)
    ids = heavy(gen, tokens, vocab)
    ids[::97] = IGNORE
    embed_check(ct, ids.to(DEV), normal(gen, vocab, width), normal(gen, tokens, width), 1.0)


def test_the_largest_ids(ct):  # noqa: F811
    # a table of 2^31 - 1 rows: keys of 31 bits, and one more for ids without a row
    vocab = (1 << 31) - 1
    ids = torch.tensor([vocab - 1, 0, vocab, vocab - 2, IGNORE, vocab - 1], device=DEV)
    grad = torch.arange(1.0, 7.0, device=DEV).bfloat16().view(6, 1)
    d = ct.embedding_backward(grad, ids, vocab)
    assert d[torch.tensor([0, vocab - 2, vocab - 1], device=DEV), 0].tolist() == [2.0, 4.0, 7.0]
    assert sum(int(d[k:k + (1 << 28)].count_nonzero()) for k in range(0, vocab, 1 << 28)) == 3
    assert ct.embedding(ids, d)[:, 0].nan_to_num(-1.0).tolist() == [7.0, 2.0, -1.0, 4.0, 0.0, 7.0]


def test_streams_and_graphs(ct):  # noqa: F811
    gen = seeded(6)
    side = torch.cuda.Stream()
    cases = []
    for tokens, width, vocab in ((100, 24, 40), (500, 24, 40), (10000, 24, 300), (3000, 520, 9000)):
        ids = heavy(gen, tokens, vocab).to(DEV)
        cases.append((ids, normal(gen, vocab, width), normal(gen, tokens, width)))
    torch.cuda.synchronize()

    def all_of():
        return [t for ids, table, grad in cases for t in (ct.embedding_forward(ids, table, 2.0), ct.embedding_backward(grad, ids, len(table), 2.0))]

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
        for ids, table, grad in cases:
            ids.copy_(heavy(gen, len(ids), len(table)))
            grad.mul_(-1.5)
        for t in held:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, all_of(), strict=True):
            assert torch.equal(a, b)


def test_refusals(ct):  # noqa: F811
    table, ids, grad = torch.zeros(5, 8, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(3, 8, device=DEV)
    for call, message in ((lambda: ct.embedding(ids.int(), table), "ids: torch.int32"),
                          (lambda: ct.embedding(ids.cpu(), table), "ids: torch.int64 on cpu"),
                          (lambda: ct.embedding(ids, table[:0]), "no rows"),
                          (lambda: ct.embedding(ids, table.double()), "table"),
                          (lambda: ct.embedding(ids, table, ignore_index=1 << 63), "ignore_index"),
                          (lambda: ct.embedding_backward(grad, ids, 0), "no rows"),
                          (lambda: ct.embedding_backward(grad, ids, 1 << 31), "most is"),
                          (lambda: ct.embedding_backward(grad, ids[:2], 5), "grad: 3 rows, not 2")):
        with pytest.raises(ValueError, match=message):
            call()
    from helrm_amd.backend import EmbeddingArgs
    ct.embedding(ids, table)
    many, rows = ids.repeat(100), grad.repeat(100, 1)
    with pytest.raises(HipError, match="workspace too small"):
        ct._call("EmbeddingGrad", EmbeddingArgs(ids=many.data_ptr(), dy=rows.data_ptr(), lddy=8, dtable=table.data_ptr(), workspace=256, workspaceBytes=8,
                                                tokens=300, width=8, vocab=5, ignore=IGNORE, scale=1.0), table.device)


@pytest.mark.parametrize("vocab", [(1 << 18) + 1, (1 << 27) + 1, (1 << 31) - 1])
@pytest.mark.parametrize("tokens", [257, 1025, 5120, 5121, 20000, 40000, 600001])
def test_keys_of_many_digits(ct, tokens, vocab):  # noqa: F811
    # two to four passes of digits (and one more key for ids without a row), in one workgroup, of tiles that are merged, and by digits' counts
    gen = seeded(tokens)
    ids = torch.randint(vocab, (tokens,), generator=gen)
    ids[::5] = ids[1::5][:1] ^ (1 << torch.arange(len(ids[::5])) % 31)        # that differ by a single bit
    ids[::7] = ids[:len(ids[::7])]                                             # some twice, some oftener
    ids[3::11], ids[4::11] = vocab - 1 - torch.arange(len(ids[3::11])) % 3, torch.arange(len(ids[4::11])) % 3
    ids[5::11] = vocab                                                         # outside, and ignored below
    ids[6::11] = IGNORE
    ids = torch.where(ids > vocab, ids - vocab, ids)
    inside = (ids >= 0) & (ids < vocab)
    grad = (torch.arange(tokens) % 3 - 1.0).to(torch.bfloat16).view(tokens, 1)  # sums of whole numbers are exact in float32, and rounded once
    d = ct.embedding_backward(grad.to(DEV), ids.to(DEV), vocab)
    rows, of = ids[inside].unique(return_inverse=True)
    sums = torch.zeros(len(rows), dtype=torch.float64).index_add_(0, of, grad[inside, 0].double())
    assert torch.equal(d[rows.to(DEV), 0].cpu(), sums.to(torch.bfloat16))
    assert sum(int(d[k:k + (1 << 28)].count_nonzero()) for k in range(0, vocab, 1 << 28)) == int(sums.count_nonzero())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [40000, 530000])
def test_ids_without_a_row_among_many(ct, dtype, tokens):  # noqa: F811
    # sorted by digits' counts, which every workgroup adds up, or a launch before
    test_ids_without_a_row(ct, dtype, tokens)


def test_streams_and_graphs_of_many_ids(ct):  # noqa: F811
    gen = seeded(7)
    side = torch.cuda.Stream()
    cases = []
    # digits' counts; groups of pieces; a launch that adds up counts; tiles that are merged
    for tokens, width, vocab in ((40000, 24, 300), (70000, 8, 300000), (530001, 4, 9000), (32768, 40, 700)):
        cases.append((heavy(gen, tokens, vocab).to(DEV), normal(gen, vocab, width), normal(gen, tokens, width)))
    torch.cuda.synchronize()

    def all_of():
        return [t for ids, table, grad in cases for t in (ct.embedding_forward(ids, table, 2.0), ct.embedding_backward(grad, ids, len(table), 2.0))]

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
        for ids, table, grad in cases:
            ids.copy_(heavy(gen, len(ids), len(table)))
            ids[turn::13] = (IGNORE, len(table), -1)[turn]
            grad.mul_(-1.5)
        for t in held:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, all_of(), strict=True):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
