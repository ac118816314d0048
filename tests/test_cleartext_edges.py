"""Limits of the cleartext operators that show without a GPU: what the entry
points refuse on the host before anything is launched, and the sizes that
their plans come to."""
import ctypes
import os
import subprocess

import pytest

from helrm_amd.backend import LayerNormArgs, LossTotalArgs, load_library

SOME = 1 << 20      # a pointer that is not followed


@pytest.fixture(scope="module")
def lib():
    lib = load_library()
    for name in ("LayerNorm", "LayerNormGrad", "LossTotal"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    for name in ("LayerNormGradWorkspace", "LossTotalWorkspace"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [ctypes.c_void_p], ctypes.c_long
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


# ---- sizes ---------------------------------------------------------------------------


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 5])
def test_sizes_beyond_a_c_int_are_refused(n):
    # (tensors of one element, expanded; with sizes modulo 2^32 a table of 2^32 + 5 rows would be one of 5)
    torch = pytest.importorskip("torch")
    from helrm_amd import cleartext as ct
    one = torch.zeros(1, 1)
    wide, tall, row, target = one.expand(1, n), one.expand(n, 1), one[0].expand(n), torch.zeros(1, dtype=torch.int64)
    for call in (lambda: ct.layer_norm(wide, row), lambda: ct.layer_norm_forward(wide, row), lambda: ct.layer_norm_backward(wide, wide, row, row, row),
                 lambda: ct.gated_mlp(wide, wide, wide, tall), lambda: ct.gated_mlp(one, tall, tall, wide),
                 lambda: ct.gated_mlp_backward(one, one, tall, tall, wide, one), lambda: ct.cross_entropy(one, tall, target),
                 lambda: ct.cross_entropy(wide, wide, target), lambda: ct.cross_entropy_backward(row[:1], one, tall, target, row[:1])):
        with pytest.raises(ValueError, match=f"{n}, the most is"):
            call()
    with pytest.raises(ValueError, match="not on the GPU"):
        ct.layer_norm(one.expand(1, (1 << 31) - 1), one[0].expand((1 << 31) - 1))
    for index in (1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="ignore_index"):
            ct.cross_entropy(one, one, target, ignore_index=index)


def test_norms_so_wide_that_an_index_would_overflow_are_refused(lib):
    # a long row's kernels step past its end by up to 1,024 before they compare
    top = (1 << 31) - 1
    for width in (top, top - 255, top - 1023):
        a = LayerNormArgs(x=SOME, ldx=top, y=SOME, ldy=top, weight=SOME, mean=SOME, rstd=SOME, dy=SOME, lddy=top, dx=SOME, lddx=top, dweight=SOME,
                          rows=1, width=width, type=1, paramType=1)
        assert lib.LayerNormGradWorkspace(ctypes.byref(a)) == -1
        for call in (lib.LayerNorm, lib.LayerNormGrad):
            assert call(ctypes.byref(a), None) == -1
            assert "width" in lib.GetLastError().decode()
    a.width = top - 1024
    assert lib.LayerNormGradWorkspace(ctypes.byref(a)) == 2 * 4 * a.width


def test_tensors_of_the_same_rows_have_them_in_the_same_order():
    torch = pytest.importorskip("torch")
    from helrm_amd import cleartext as ct
    x, m = torch.zeros(9, 5, 4), torch.zeros(4, 4)
    refused = [torch.Size(s) for s in ((5, 9), (3, 15), (5, 3, 3), (1, 5, 9))]
    for s in refused:
        with pytest.raises(ValueError, match="target: leading dimensions"):
            ct.cross_entropy(x, m, torch.zeros(s, dtype=torch.int64))
        with pytest.raises(ValueError, match="target: leading dimensions"):
            ct.cross_entropy_backward(torch.zeros(45), x, m, torch.zeros(s, dtype=torch.int64), torch.zeros(45))
    for s in ((9, 5), (45,), (9, 1, 5), (45, 1), (1, 45)):          # (the next check is the one for the GPU)
        with pytest.raises(ValueError, match="not on the GPU"):
            ct.cross_entropy(x, m, torch.zeros(s, dtype=torch.int64))
        with pytest.raises(ValueError, match="not on the GPU"):
            ct.cross_entropy(x.view(45, 4), m, torch.zeros(s, dtype=torch.int64))


def test_what_a_total_refuses(lib):
    assert lib.LossTotal(None, None) == -1 and "no arguments" in lib.GetLastError().decode()
    for message, change in (("number of rows", dict(rows=-1)), ("number of rows", dict(rows=1 << 30)), (": loss", dict(loss=None)),
                            ("total and factor", dict(factor=None)), ("workspace too small", dict(rows=1 << 20))):
        a = LossTotalArgs(loss=SOME, target=SOME, total=SOME, factor=SOME, rows=100, ignore=-100)
        for k, v in change.items():
            setattr(a, k, v)
        assert lib.LossTotal(ctypes.byref(a), None) == -1
        assert message in lib.GetLastError().decode()
    assert lib.LossTotalWorkspace(ctypes.byref(a)) == 256 * 16


# ---- derivatives that there are not -----------------------------------------------------


def test_tensors_with_a_tangent_are_refused():
    # (the tangent was lost: an output without one is a constant)
    torch = pytest.importorskip("torch")
    from torch.autograd import forward_ad

    from helrm_amd import cleartext as ct
    x, w, m, target = torch.ones(2, 4), torch.ones(4), torch.ones(4, 4), torch.zeros(2, dtype=torch.int64)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: ct.layer_norm(d, w), lambda: ct.layer_norm_forward(d, w), lambda: ct.gated_mlp(d, m, m, m),
                             lambda: ct.cross_entropy(d, m, target), lambda: ct.cross_entropy_forward(d, m, target)):
                    with pytest.raises(NotImplementedError, match="x: has a tangent"):
                        call()
        with pytest.raises(ValueError, match="not on the GPU"):      # none of these has one
            ct.layer_norm(x, w)


# ---- the launches of the loss --------------------------------------------------------

# rows, table rows, width, products a product is made of: small tiles in several launches (few rows; 257 to 384 of float32), a
# short last piece, several launches of large ones, one launch
LOSSES = [(17, (1 << 30) + 300, 8, 1), (65, (1 << 30) + 1, 8, 1), (128, (1 << 31) - 1, 1000, 1), (129, (1 << 31) - 1, 8, 1), (300, (1 << 29) + 300, 8, 6),
          (257, (1 << 30) - 1, 40, 6), (384, (1 << 29) + 1, 8, 6), ((1 << 26) - 256, 57700, 8, 6), (16384, (1 << 24) + 300, 8, 1),
          ((1 << 30) - 1, 1, 1, 1), ((1 << 30) - 1, 700, 1, 6), ((1 << 29) + 1, 257, 300, 1), (65, 300, 8, 6), (8192, 131072, 2048, 1)]


def test_the_pieces_of_all_launches_are_every_piece_once(tmp_path):
    source = tmp_path / "pieces.cpp"
    source.write_text("""
#include <cstdio>
#include "plan.h"
int main() {
  long m, n, k;
  int pairs;
  while (scanf("%ld %ld %ld %d", &m, &n, &k, &pairs) == 4) {
    const clr::SoftmaxPlan s = clr::softmax_plan(m, n, k, pairs);
    printf("%d %ld %d %d\\n", s.parts, s.columns, s.plan.tile(), s.plan.threads());
  }
}
""")
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "helrm_amd", "csrc")
    program = tmp_path / "pieces"
    subprocess.run(["g++", "-std=c++17", "-I", csrc, str(source), "-o", str(program)], check=True)
    said = subprocess.run([str(program)], input="\n".join(" ".join(map(str, s)) for s in LOSSES), capture_output=True, text=True, check=True).stdout
    tiles = set()
    for (rows, vocab, _, _), line in zip(LOSSES, said.splitlines(), strict=True):
        parts, columns, tile, threads = map(int, line.split())
        assert threads == {128: 256, 256: 512}[tile]
        several = columns < vocab
        tiles.add((tile, several))
        assert columns % tile == 0 and 0 < columns < 1 << 31
        at = 0
        for first in range(0, vocab, columns):              # a launch's pieces are its columns' tiles, and lie where they belong
            assert first // tile == at
            here = -(-min(columns, vocab - first) // tile)
            assert -(-rows // tile) * here * threads < 1 << 32
            at += here
        assert at == parts
    assert tiles == {(128, False), (128, True), (256, False), (256, True)}
