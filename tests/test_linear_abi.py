"""CPU checks of the 4-bit linear and expert entry points: struct layout, workspace sizes and the
refusals that come before any device work."""

import ctypes
import subprocess

import pytest

from conftest import ROOT, pkg

INVALID, WORKSPACE = pkg._lib.AM_ERR_INVALID, pkg._lib.AM_ERR_WORKSPACE
PTR = 1 << 20  # a 256-byte aligned address that nothing reads


def weight(n_out=64, n_in=128, experts=1, dtype=1):
    d = pkg._lib.Q4WeightDesc()
    d.codes, d.params, d.row_scale = PTR, PTR, PTR
    d.n_out, d.n_in, d.experts, d.dtype = n_out, n_in, experts, dtype
    return d


def test_weight_layout_matches_header(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text(r'''
#include <stdio.h>
#include <stddef.h>
#include "am_q4.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %zu\n", sizeof(am_q4_weight), offsetof(am_q4_weight, params),
         offsetof(am_q4_weight, row_scale), offsetof(am_q4_weight, n_out),
         offsetof(am_q4_weight, experts), offsetof(am_q4_weight, dtype));
  return 0;
}
''')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    W = pkg._lib.Q4WeightDesc
    assert [int(x) for x in out] == [ctypes.sizeof(W), W.params.offset, W.row_scale.offset, W.n_out.offset,
                                     W.experts.offset, W.dtype.offset]


def test_workspace_sizes():
    """None for a few tokens, else one fp16 row and one float a row of activations."""
    lib = pkg._lib.load()
    w, big = weight(), weight(n_out=14336, n_in=4096)
    r = ctypes.byref
    assert [int(lib.am_q4_linear_workspace_bytes(r(w), None, n)) for n in (0, 1, 8, 9)] == [0, 0, 0, 9 * 260]
    assert int(lib.am_q4_linear_workspace_bytes(r(w), r(w), 8)) == 0
    assert int(lib.am_q4_linear_workspace_bytes(r(big), r(big), 4)) == 0
    assert int(lib.am_q4_linear_workspace_bytes(r(big), r(big), 5)) == 5 * 8196
    e = weight(experts=16)
    assert [int(lib.am_q4_expert_linear_workspace_bytes(r(e), None, n)) for n in (0, 32, 33)] == [0, 0, 33 * 260]
    assert int(lib.am_q4_linear_workspace_bytes(None, None, 100)) == 0


def test_workspace_beyond_the_few_token_kernels_inputs():
    """A few tokens of more inputs than one cluster's shared memory holds go the way of many, and need its
    workspace; up to `linear.FEW_INPUTS` the Python calls need not ask."""
    lib = pkg._lib.load()
    size = lambda n_in, rows, gated=False: int(lib.am_q4_linear_workspace_bytes(  # noqa: E731
        ctypes.byref(weight(n_in=n_in)), ctypes.byref(weight(n_in=n_in)) if gated else None, rows))
    few = pkg.linear.FEW_INPUTS
    assert [size(few, m) for m in range(1, pkg.linear.FEW_TOKENS + 1)] == [0] * pkg.linear.FEW_TOKENS
    assert [size(few, m, True) for m in range(1, pkg.linear.FEW_GATED_TOKENS + 1)] == [0] * pkg.linear.FEW_GATED_TOKENS
    for n_in, rows, gated in ((49408, 5, False), (53248, 8, False), (131072, 4, False), (278528, 1, False),
                              (33024, 5, True), (131072, 3, True)):
        assert size(n_in, rows, gated) == rows * (n_in * 2 + 4), (n_in, rows, gated)
    e = weight(n_in=139264, experts=4)
    assert int(lib.am_q4_expert_linear_workspace_bytes(ctypes.byref(e), None, 8)) == 8 * (139264 * 2 + 4)


@pytest.mark.parametrize("field,value", [("codes", None), ("params", None), ("row_scale", None), ("codes", PTR + 4),
                                         ("n_in", 96), ("n_in", 0), ("n_out", 0), ("n_out", -3), ("experts", 0),
                                         ("dtype", 2), ("dtype", 9)])
def test_a_bad_weight_is_refused(field, value):
    lib = pkg._lib.load()
    w = weight()
    setattr(w, field, value)
    assert lib.am_q4_linear(ctypes.byref(w), None, PTR, 128, 1, PTR, 64, None, 0, None, None) == INVALID
    assert lib.am_q4_expert_linear(ctypes.byref(w), None, PTR, 128, 1, PTR, None, 1, 1, PTR, 64, None, 0, None,
                                   None) == INVALID
    assert lib.am_last_error()


def test_weights_whose_rows_pass_the_kernels_counts_are_refused():
    """Tiles reach up to 512 rows past the last one: row numbers have to stay below 2^31 there too."""
    lib = pkg._lib.load()
    for n_out, experts, want in ((2 ** 31 - 1, 1, INVALID), (2 ** 31 - 1024, 1, INVALID), (2 ** 20, 2048, INVALID),
                                 (2 ** 31 - 1025, 1, WORKSPACE), (2 ** 20, 2047, WORKSPACE)):
        w = weight(n_out=n_out, experts=experts)
        assert lib.am_q4_expert_linear(ctypes.byref(w), None, PTR, 128, 2 ** 13, PTR, None, 1, 2 ** 13, PTR, n_out,
                                       None, 0, None, None) == want, (n_out, experts)


def test_linear_arguments_are_refused():
    lib = pkg._lib.load()
    w, other, grouped = weight(), weight(n_out=32), weight(experts=4)
    r = ctypes.byref
    call = lambda w, up=None, x=PTR, xs=128, rows=1, out=PTR, os=64, ws=None, nb=0: lib.am_q4_linear(  # noqa: E731
        w, up, x, xs, rows, out, os, ws, nb, None, None)
    assert call(None) == INVALID
    assert call(r(w), up=r(other)) == INVALID and b"two weights" in lib.am_last_error()
    assert call(r(grouped)) == INVALID
    assert call(r(w), x=None) == INVALID
    assert call(r(w), x=PTR + 2) == INVALID
    assert call(r(w), xs=64, rows=2) == INVALID
    assert call(r(w), xs=132, rows=2) == INVALID
    assert call(r(w), rows=-1) == INVALID
    assert call(r(w), out=None) == INVALID
    assert call(r(w), os=32, rows=2) == INVALID
    assert call(r(w), rows=9) == WORKSPACE
    assert call(r(w), rows=9, ws=PTR, nb=9 * 260 - 1) == WORKSPACE
    assert call(r(w), rows=9, ws=PTR + 16, nb=9 * 260) == WORKSPACE
    assert call(r(w), rows=0) == pkg._lib.AM_OK


def test_routing_and_combination_arguments_are_refused():
    lib = pkg._lib.load()
    route = lambda lg=PTR, dt=2, st=8, t=1, e=8, k=2, out=PTR: lib.am_route_experts(  # noqa: E731
        lg, dt, st, t, e, k, 1, out, PTR, PTR, PTR, PTR, None)
    assert route(lg=None) == INVALID
    assert route(dt=7) == INVALID
    assert route(e=0) == INVALID and route(e=1025, st=1025) == INVALID
    assert route(k=0) == INVALID and route(k=9) == INVALID and route(e=64, st=64, k=33) == INVALID
    assert route(st=4, t=2) == INVALID
    assert route(t=-1) == INVALID
    assert route(out=None) == INVALID and route(out=PTR + 2) == INVALID and route(lg=PTR + 1) == INVALID
    comb = lambda y=PTR, dt=1, ys=64, w=PTR, out=PTR, t=1, k=2, width=64: lib.am_combine_experts(  # noqa: E731
        y, dt, ys, 4, w, PTR, None, 0, out, 64, t, k, width, None, None)
    assert comb(y=None) == INVALID and comb(w=None) == INVALID and comb(out=None) == INVALID
    assert comb(dt=2) == INVALID
    assert comb(k=0) == INVALID
    assert comb(width=-2) == INVALID
    assert comb(width=0) == pkg._lib.AM_OK  # nothing to write
    assert comb(y=PTR + 1) == INVALID and comb(w=PTR + 2) == INVALID
    assert comb(t=-1) == INVALID
    assert comb(ys=32) == INVALID
