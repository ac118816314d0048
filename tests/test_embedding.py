"""What the embedding refuses without a GPU: every check is made on the host
before anything is launched."""
import ctypes

import pytest

from helrm_amd.backend import EmbeddingArgs, load_library

SOME = 1 << 20      # a pointer that is not followed


@pytest.fixture(scope="module")
def lib():
    lib = load_library()
    for name in ("Embedding", "EmbeddingGrad"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    lib.EmbeddingGradWorkspace.argtypes, lib.EmbeddingGradWorkspace.restype = [ctypes.c_void_p], ctypes.c_long
    return lib


def args(**kw):
    a = EmbeddingArgs(ids=SOME, table=SOME, ldtable=8, y=SOME, ldy=8, dy=SOME, lddy=8, dtable=SOME, tokens=4, width=8, vocab=16, ignore=-100,
                      scale=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(lib, call, a, message):
    assert getattr(lib, call)(ctypes.byref(a) if a is not None else None, None) == -1
    assert message in lib.GetLastError().decode(), lib.GetLastError()


def test_refusals_of_the_entry_points(lib):
    for call in ("Embedding", "EmbeddingGrad"):
        refused(lib, call, None, "no arguments")
        refused(lib, call, args(type=3), "unknown element type")
        for tokens in (-1, 1 << 30, 1 << 40):
            refused(lib, call, args(tokens=tokens), "number of tokens")
        for width in (0, -1, (1 << 31) - 1023):
            refused(lib, call, args(width=width), "width")
        refused(lib, call, args(vocab=0), "table rows")
        refused(lib, call, args(ids=None), "ids")
    refused(lib, "Embedding", args(table=None), "table")
    refused(lib, "Embedding", args(ldtable=7), "table")
    refused(lib, "Embedding", args(y=None), ": y")
    refused(lib, "Embedding", args(ldy=7), ": y")
    refused(lib, "EmbeddingGrad", args(dy=None), "dy")
    refused(lib, "EmbeddingGrad", args(lddy=7), "dy")
    refused(lib, "EmbeddingGrad", args(dtable=None), "dtable")
    assert lib.EmbeddingGradWorkspace(ctypes.byref(args())) == 0           # (few ids take none)
    need = lib.EmbeddingGradWorkspace(ctypes.byref(args(tokens=1000)))
    assert need > 0 and lib.EmbeddingGradWorkspace(ctypes.byref(args(type=3))) == -1
    assert lib.EmbeddingGradWorkspace(ctypes.byref(args(tokens=1000, ids=None, dy=None, dtable=None))) == need
    assert lib.EmbeddingGradWorkspace(ctypes.byref(args(tokens=100000))) > need
    assert lib.EmbeddingGradWorkspace(ctypes.byref(args(tokens=100000, width=800))) > lib.EmbeddingGradWorkspace(ctypes.byref(args(tokens=100000)))
    refused(lib, "EmbeddingGrad", args(tokens=1000, workspace=SOME, workspaceBytes=need - 1), "workspace too small")
    refused(lib, "EmbeddingGrad", args(tokens=1000, workspace=SOME + 8, workspaceBytes=need), "aligned")


def test_refusals_of_the_tensors():
    torch = pytest.importorskip("torch")
    from torch.autograd import forward_ad

    from helrm_amd import cleartext as ct
    ids, table, grad = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(5, 4), torch.zeros(2, 3, 4)
    one = torch.zeros(1, 1)
    for call, message in ((lambda: ct.embedding(ids, table), "not on the GPU"),
                          (lambda: ct.embedding(ids, table[0]), "table: not a matrix"),
                          (lambda: ct.embedding(ids, table[:, :0]), "table: not a matrix"),
                          (lambda: ct.embedding(ids, table.double()), "table: torch.float64"),
                          (lambda: ct.embedding(ids, one.expand(1 << 31, 1)), "most is"),
                          (lambda: ct.embedding(ids, one.expand(1, 1 << 31)), "most is"),
                          (lambda: ct.embedding_backward(grad, ids, 5), "not on the GPU"),
                          (lambda: ct.embedding_backward(grad, ids.view(3, 2), 5), "grad: leading dimensions"),
                          (lambda: ct.embedding_backward(torch.zeros(()), ids, 5), "grad: no last dimension"),
                          (lambda: ct.embedding_backward(one.expand(1, 1 << 31), ids, 5), "most is")):
        with pytest.raises(ValueError, match=message):
            call()
    with forward_ad.dual_level():
        for grad_on in (True, False):
            with torch.set_grad_enabled(grad_on), pytest.raises(NotImplementedError, match="table: has a tangent"):
                ct.embedding(ids, forward_ad.make_dual(table, torch.ones_like(table)))
