"""What the preference loss refuses without a GPU: every check is made on the
host before anything is launched."""
import ctypes

import pytest

from helrm_amd.backend import PreferenceArgs, load_library

SOME = 1 << 20      # a pointer that is not followed


@pytest.fixture(scope="module")
def lib():
    lib = load_library()
    for name in ("Preference", "PreferenceGrad"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    lib.PreferenceWorkspace.argtypes, lib.PreferenceWorkspace.restype = [ctypes.c_void_p], ctypes.c_long
    return lib


def args(**kw):
    a = PreferenceArgs(loss=SOME, ldloss=8, reference=SOME, ldreference=8, target=SOME, ldtarget=8, value=SOME, ratio=SOME, slope=SOME, kept=SOME,
                       dvalue=SOME, dloss=SOME, lddloss=8, pairs=4, length=8, ignore=-100, beta=0.1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(lib, call, a, message):
    assert getattr(lib, call)(ctypes.byref(a) if a is not None else None, None) == -1
    assert message in lib.GetLastError().decode(), lib.GetLastError()


def test_refusals_of_the_entry_points(lib):
    for call in ("Preference", "PreferenceGrad"):
        refused(lib, call, None, "no arguments")
        for pairs in (-1, 1 << 30, 1 << 40):
            refused(lib, call, args(pairs=pairs), "number of pairs")
        for length in (-1, (1 << 40) + 1):
            refused(lib, call, args(length=length, ldloss=1 << 50), "length")
        refused(lib, call, args(kind=2), "unknown kind")
        for bad in (float("nan"), float("inf"), -float("inf")):
            refused(lib, call, args(beta=bad), "finite")
            refused(lib, call, args(margin=bad), "finite")
        for bad in (-0.1, 1.1, float("nan")):
            refused(lib, call, args(smoothing=bad), "smoothing")
        refused(lib, call, args(kind=1, smoothing=0.1), "smoothing")
        refused(lib, call, args(ldtarget=7), "target")
        refused(lib, call, args(slope=None), "slope")
    for name in ("value", "ratio"):
        refused(lib, "Preference", args(**{name: None}), "value, ratio and slope")
    refused(lib, "Preference", args(loss=None), ": loss")
    refused(lib, "Preference", args(loss=None, offsets=SOME), ": loss")
    refused(lib, "Preference", args(ldloss=7), ": loss")
    refused(lib, "Preference", args(ldreference=7), "reference")
    refused(lib, "PreferenceGrad", args(dloss=None), "dloss")
    refused(lib, "PreferenceGrad", args(lddloss=7), "dloss")
    refused(lib, "PreferenceGrad", args(dvalue=None), "dvalue")
    assert lib.PreferenceWorkspace(ctypes.byref(args())) == 0 and lib.PreferenceWorkspace(ctypes.byref(args(kind=2))) == -1
    long = dict(pairs=2, length=1 << 20, ldloss=1 << 20, ldreference=1 << 20, ldtarget=1 << 20)
    need = lib.PreferenceWorkspace(ctypes.byref(args(**long)))
    assert need > 0
    refused(lib, "Preference", args(workspace=SOME, workspaceBytes=need - 1, **long), "workspace too small")
    refused(lib, "Preference", args(workspace=SOME + 8, workspaceBytes=need, **long), "aligned")


def test_refusals_of_the_tensors():
    torch = pytest.importorskip("torch")
    from torch.autograd import forward_ad

    from helrm_amd import cleartext as ct
    losses, line = torch.zeros(3, 2, 5), torch.zeros(12)
    offsets = torch.zeros(5, dtype=torch.int64)
    for call, message in ((lambda: ct.preference(losses), "not on the GPU"),
                          (lambda: ct.preference(line, offsets=offsets), "not on the GPU"),
                          (lambda: ct.preference(losses.bfloat16()), "losses: torch.bfloat16"),
                          (lambda: ct.preference(losses.view(2, 3, 5)), "losses"),
                          (lambda: ct.preference(line), "losses"),
                          (lambda: ct.preference(losses, offsets=offsets), "beside offsets"),
                          (lambda: ct.preference(line, offsets=offsets[:4]), "offsets"),
                          (lambda: ct.preference(line, offsets=offsets.view(1, 5)), "offsets"),
                          (lambda: ct.preference(losses, kind="squared"), "kind"),
                          (lambda: ct.preference(losses, beta=float("nan")), "finite"),
                          (lambda: ct.preference(losses, margin=float("inf")), "finite"),
                          (lambda: ct.preference(losses, smoothing=1.5), "smoothing"),
                          (lambda: ct.preference(losses, kind="hinge", smoothing=0.1), "smoothing"),
                          (lambda: ct.preference(losses, ignore_index=1 << 63), "ignore_index"),
                          (lambda: ct.preference(losses, reduction="all"), "reduction"),
                          (lambda: ct.preference(losses, losses.clone().requires_grad_()), "reference: requires a gradient")):
        with pytest.raises(ValueError, match=message):
            call()
    with forward_ad.dual_level(), pytest.raises((NotImplementedError, ValueError), match="tangent|not on the GPU"):
        ct.preference(forward_ad.make_dual(losses, torch.ones_like(losses)))
