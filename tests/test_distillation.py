"""What the distillation refuses without a GPU: every check is made on the host
before anything is launched."""
import ctypes

import pytest

from helrm_amd.backend import DistillationArgs, load_library

SOME = 1 << 20      # a pointer that is not followed


@pytest.fixture(scope="module")
def lib():
    lib = load_library()
    for name in ("Distillation", "DistillationGrad"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
        getattr(lib, name + "Workspace").argtypes, getattr(lib, name + "Workspace").restype = [ctypes.c_void_p], ctypes.c_long
    return lib


def args(**kw):
    a = DistillationArgs(x=SOME, ldx=8, table=SOME, ldtable=8, ids=SOME, logits=SOME, loss=SOME, lse=SOME, kept=SOME, scores=SOME, probs=SOME, cols=SOME,
                         dloss=SOME, dx=SOME, lddx=8, dtable=SOME, rows=4, width=8, vocab=16, top=3, ignore=-100, temperature=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(lib, call, a, message):
    assert getattr(lib, call)(ctypes.byref(a) if a is not None else None, None) == -1
    assert message in lib.GetLastError().decode(), lib.GetLastError()


@pytest.mark.parametrize("call", ["Distillation", "DistillationGrad"])
def test_refusals_of_the_entry_points(lib, call):
    refused(lib, call, None, "no arguments")
    refused(lib, call, args(type=3), "unknown element type")
    refused(lib, call, args(teacherType=5), "unknown element type")
    for type, teacher in ((0, 1), (0, 2), (1, 2), (2, 1)):
        refused(lib, call, args(type=type, teacherType=teacher), "teacherType")
    for rows in (-1, 1 << 30, 1 << 40):
        refused(lib, call, args(rows=rows), "number of rows")
    for width in (0, 1 << 21):
        refused(lib, call, args(width=width), "width")
    refused(lib, call, args(vocab=0), "table rows")
    for top in (0, -1, 1025):
        refused(lib, call, args(top=top), "teacher's logits")
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-30, 1e30):
        refused(lib, call, args(temperature=t), "temperature")
    refused(lib, call, args(ldx=7), ": x")
    refused(lib, call, args(x=None), ": x")
    refused(lib, call, args(ldtable=7), "table")
    for name in ("lse", "kept", "scores", "probs", "cols"):
        refused(lib, call, args(**{name: None}), name)
    for name in ("ids", "logits", "loss") if call == "Distillation" else ("dx", "dtable", "dloss"):
        refused(lib, call, args(**{name: None}), name)
    size = getattr(lib, call + "Workspace")
    need = size(ctypes.byref(args()))
    assert need > 0 and size(ctypes.byref(args(type=3))) == -1
    assert size(ctypes.byref(args(rows=5000))) > need
    assert size(ctypes.byref(args(rows=500, width=5000))) > size(ctypes.byref(args(rows=500)))
    refused(lib, call, args(workspace=SOME, workspaceBytes=need - 1), "workspace too small")
    refused(lib, call, args(workspace=SOME + 8, workspaceBytes=need), "aligned")


def test_refusals_of_the_tensors():
    torch = pytest.importorskip("torch")
    from torch.autograd import forward_ad

    from helrm_amd import cleartext as ct
    x, table, ids, logits = torch.zeros(9, 5, 4), torch.zeros(7, 4), torch.zeros(9, 5, 3, dtype=torch.int64), torch.zeros(9, 5, 3)
    one = torch.zeros(1, 1)
    for call, message in ((lambda: ct.distillation(x, table, ids, logits), "not on the GPU"),
                          (lambda: ct.distillation(x, table[0], ids, logits), "table: not a matrix"),
                          (lambda: ct.distillation(x, table, ids.view(5, 9, 3), logits), "ids: leading dimensions"),
                          (lambda: ct.distillation(x, table, ids[..., :0], logits[..., :0]), "top from 1 to 1024"),
                          (lambda: ct.distillation(x, table, ids[..., :1].expand(9, 5, 1025), logits), "top from 1 to 1024"),
                          (lambda: ct.distillation(x, table, ids, logits, 0.0), "temperature"),
                          (lambda: ct.distillation(x, table, ids, logits, float("nan")), "temperature"),
                          (lambda: ct.distillation(x, table, ids, logits, -2.0), "temperature"),
                          (lambda: ct.distillation(x, table, ids, logits, ignore_index=1 << 63), "ignore_index"),
                          (lambda: ct.distillation(x, table, ids, logits, reduction="all"), "reduction"),
                          (lambda: ct.distillation(x, table, ids, logits.clone().requires_grad_()), "logits: require a gradient"),
                          (lambda: ct.distillation(one, one.expand(1 << 31, 1), ids[0, :1], logits[0, :1]), "most is"),
                          (lambda: ct.distillation(one.expand(1, 1 << 31), one.expand(1, 1 << 31), ids[0, :1], logits[0, :1]), "most is")):
        with pytest.raises(ValueError, match=message):
            call()
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="x: has a tangent"):
        ct.distillation(forward_ad.make_dual(x, torch.ones_like(x)), table, ids, logits)
