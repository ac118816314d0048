"""Limits of the cleartext operators that show without a GPU: what the entry
points refuse on the host before anything is launched, and the sizes that
their plans come to."""
import ctypes

import pytest

from helrm_amd.backend import LayerNormArgs, load_library

SOME = 1 << 20      # a pointer that is not followed


@pytest.fixture(scope="module")
def lib():
    lib = load_library()
    for name in ("LayerNorm", "LayerNormGrad"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    lib.LayerNormGradWorkspace.argtypes, lib.LayerNormGradWorkspace.restype = [ctypes.c_void_p], ctypes.c_long
    return lib


@pytest.mark.parametrize("type,params", [(0, 1), (0, 2), (1, 2), (2, 1)])
def test_a_norms_parameters_are_of_its_type_or_float32(lib, type, params):
    # read as another type they are misread; as a wider one they are read, and their gradients written, past their end
    a = LayerNormArgs(x=SOME, ldx=8, y=SOME, ldy=8, weight=SOME, mean=SOME, rstd=SOME, dy=SOME, lddy=8, dx=SOME, lddx=8, dweight=SOME,
                      rows=4, width=8, type=type, paramType=params)
    assert lib.LayerNormGradWorkspace(ctypes.byref(a)) == -1
    assert "paramType" in lib.GetLastError().decode()
    for call in (lib.LayerNorm, lib.LayerNormGrad):
        assert call(ctypes.byref(a), None) == -1
        assert "paramType" in lib.GetLastError().decode()
    a.paramType = type
    assert lib.LayerNormGradWorkspace(ctypes.byref(a)) > 0
    a.paramType = 0
    assert lib.LayerNormGradWorkspace(ctypes.byref(a)) > 0
