"""What the cleartext operators refuse without a GPU: every check is made on
the host before anything is launched."""
import ctypes

import pytest

from helrm_amd.backend import CrossEntropyArgs, GatedMLPArgs, LayerNormArgs, load_library

SOME = 1 << 20      # a pointer that is not followed


@pytest.fixture(scope="module")
def lib():
    lib = load_library()
    for name in ("LayerNorm", "LayerNormGrad", "GatedMLP", "GatedMLPGrad", "CrossEntropy", "CrossEntropyGrad"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
        if hasattr(lib, name + "Workspace"):
            getattr(lib, name + "Workspace").argtypes, getattr(lib, name + "Workspace").restype = [ctypes.c_void_p], ctypes.c_long
    return lib


def refused(lib, call, args, message):
    assert getattr(lib, call)(ctypes.byref(args) if args is not None else None, None) == -1
    assert message in lib.GetLastError().decode(), lib.GetLastError()


def norm(**kw):
    a = LayerNormArgs(x=SOME, ldx=8, y=SOME, ldy=8, weight=SOME, mean=SOME, rstd=SOME, dy=SOME, lddy=8, dx=SOME, lddx=8, dweight=SOME,
                      rows=4, width=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def mlp(**kw):
    a = GatedMLPArgs(x=SOME, ldx=8, gate=SOME, ldgate=8, up=SOME, ldup=8, down=SOME, lddown=16, y=SOME, ldy=8, g=SOME, u=SOME,
                     dy=SOME, lddy=8, dx=SOME, lddx=8, dgate=SOME, dup=SOME, ddown=SOME, rows=4, width=8, hidden=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def loss(**kw):
    a = CrossEntropyArgs(x=SOME, ldx=8, table=SOME, ldtable=8, target=SOME, loss=SOME, lse=SOME, dloss=SOME, dx=SOME, lddx=8,
                         dtable=SOME, rows=4, width=8, vocab=16, ignore=-100)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("call", ["LayerNorm", "LayerNormGrad", "GatedMLP", "GatedMLPGrad", "CrossEntropy", "CrossEntropyGrad"])
def test_no_arguments(lib, call):
    refused(lib, call, None, "no arguments")


@pytest.mark.parametrize("call,make", [("LayerNorm", norm), ("LayerNormGrad", norm), ("GatedMLP", mlp), ("GatedMLPGrad", mlp),
                                       ("CrossEntropy", loss), ("CrossEntropyGrad", loss)])
def test_shapes_types_and_strides(lib, call, make):
    refused(lib, call, make(type=3), "unknown element type")
    refused(lib, call, make(rows=-1), "number of rows")
    refused(lib, call, make(rows=1 << 40), "number of rows")
    refused(lib, call, make(width=0), "width")
    refused(lib, call, make(ldx=7), ": x")
    refused(lib, call, make(x=None), ": x")


def test_missing_tensors(lib):
    refused(lib, "LayerNorm", norm(weight=None), "weight")
    refused(lib, "LayerNorm", norm(y=None), "y")
    refused(lib, "LayerNorm", norm(paramType=7), "unknown element type")
    refused(lib, "LayerNormGrad", norm(mean=None), "mean and rstd")
    refused(lib, "LayerNormGrad", norm(dweight=None), "weight")
    refused(lib, "LayerNormGrad", norm(lddy=3), "dy")
    for k in ("gate", "up", "down"):
        refused(lib, "GatedMLP", mlp(**{k: None}), k)
        refused(lib, "GatedMLP", mlp(**{"ld" + k: 3}), k)
    refused(lib, "GatedMLP", mlp(u=None), "kept together")
    refused(lib, "GatedMLP", mlp(act=3), "unknown activation")
    refused(lib, "GatedMLP", mlp(hidden=0), "width")
    refused(lib, "GatedMLPGrad", mlp(g=None), "g and u")
    refused(lib, "GatedMLPGrad", mlp(ddown=None), "gradients")
    refused(lib, "CrossEntropy", loss(target=None), "target")
    refused(lib, "CrossEntropy", loss(loss=None), "loss")
    refused(lib, "CrossEntropy", loss(vocab=0), "table rows")
    refused(lib, "CrossEntropy", loss(ldtable=4), "table")
    refused(lib, "CrossEntropyGrad", loss(dtable=None), "dtable")
    refused(lib, "CrossEntropyGrad", loss(dloss=None), "dloss")
    refused(lib, "CrossEntropyGrad", loss(lse=None), "lse")


def test_results_whose_rows_are_too_far_apart(lib):
    """A tile's places in a result are 32-bit offsets from its first one."""
    for ld in (1 << 24, 1 << 40):
        refused(lib, "GatedMLP", mlp(ldy=ld), "GatedMLP: y")
        refused(lib, "GatedMLPGrad", mlp(lddx=ld), "GatedMLPGrad: dx")
    refused(lib, "GatedMLP", mlp(ldy=(1 << 24) - 1), "workspace too small")
    refused(lib, "GatedMLP", mlp(rows=1, ldy=1 << 40), "workspace too small")


def test_workspaces(lib):
    for call, make in (("LayerNormGrad", norm), ("GatedMLP", mlp), ("GatedMLPGrad", mlp), ("CrossEntropy", loss), ("CrossEntropyGrad", loss)):
        size = getattr(lib, call + "Workspace")
        need = size(ctypes.byref(make()))
        assert need > 0
        assert size(ctypes.byref(make(rows=5000))) > need        # rows, width and type lie where the library reads them
        if make is not mlp:                                       # the block's takes the hidden values alone
            assert size(ctypes.byref(make(rows=500, width=5000))) > size(ctypes.byref(make(rows=500)))
        assert size(ctypes.byref(make(type=3))) == -1
        a = make(workspace=SOME, workspaceBytes=need - 1)
        refused(lib, call, a, "workspace too small")
        refused(lib, call, make(workspace=SOME + 8, workspaceBytes=need), "aligned")
    assert lib.GatedMLPWorkspace(ctypes.byref(mlp(hidden=160))) > lib.GatedMLPWorkspace(ctypes.byref(mlp()))
    assert lib.CrossEntropyWorkspace(ctypes.byref(loss(vocab=1 << 20))) > lib.CrossEntropyWorkspace(ctypes.byref(loss()))


def test_tensors_on_the_host():
    torch = pytest.importorskip("torch")
    from helrm_amd import cleartext as ct
    x = torch.zeros(2, 4)
    with pytest.raises(ValueError, match="not on the GPU"):
        ct.layer_norm(x, torch.ones(4))
    with pytest.raises(ValueError, match="not on the GPU"):
        ct.gated_mlp(x, torch.zeros(3, 4), torch.zeros(3, 4), torch.zeros(4, 3))
    with pytest.raises(ValueError, match="not on the GPU"):
        ct.cross_entropy(x, torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))


def test_a_second_hip_runtime_is_refused():
    """The library loaded first brings its own HIP runtime, torch then another one: their streams and pointers mean
    nothing to each other, so the operators refuse to start.  With torch first there is one runtime."""
    import subprocess
    import sys
    pytest.importorskip("torch")
    code = "{}\nfrom helrm_amd import cleartext\ntry:\n    cleartext._library()\n    print('one')\nexcept Exception as e:\n    print(type(e).__name__, e)"
    first = "from helrm_amd.backend import load_library\nload_library()\nimport torch"
    root = __file__.rsplit("/", 2)[0]
    said = [subprocess.run([sys.executable, "-c", code.format(s)], capture_output=True, text=True, cwd=root).stdout for s in (first, "import torch")]
    assert said[1].strip() == "one", said
    assert "two HIP runtimes" in said[0] or said[0].strip() == "one", said     # (one file for both: nothing to refuse)
