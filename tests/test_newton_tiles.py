"""The sides of the tiles that the Newton-Schulz products take, by their rule
(CPU only): every kernel is one that some sizes run on."""
import ctypes

import pytest

from neuralscript_amd import runtime

i64 = ctypes.c_int64


def sides(n, r, c):
    return tuple(runtime.lib().nsh_test_newton_side(k, i64(n), i64(r), i64(c)) for k in range(4))


# (S, P, X, the last X) of n matrices [r, c]; 0: one workgroup a matrix
@pytest.mark.parametrize("n,r,c,want", [
    (8, 64, 256, (0, 0, 0, 0)), (1, 128, 128, (32, 32, 32, 32)), (3, 1000, 333, (32, 32, 64, 64)),
    (4, 512, 512, (32, 32, 64, 64)), (16, 300, 300, (64, 64, 64, 64)), (64, 200, 333, (128, 32, 128, 128)),
    (1, 2500, 2300, (128, 128, 128, 128)), (64, 1024, 1024, (128, 128, 256, 256)), (16, 1280, 1280, (256, 256, 128, 128)),
    (32768, 1, 8192, (32, 32, 128, 128))])
def test_the_rules_choice(n, r, c, want):
    assert sides(n, r, c) == want


@pytest.mark.parametrize("side", [32, 64, 128, 256])
def test_a_tests_choice_ends_with_it(side):
    lib = runtime.lib()
    before = sides(8, 64, 256)
    try:
        lib.nsh_test_newton_tile(side)
        assert sides(8, 64, 256) == (side,) * 4
        lib.nsh_test_newton_tile(96)  # no such tiles
        assert sides(8, 64, 256) == before
    finally:
        lib.nsh_test_newton_tile(0)
    assert sides(8, 64, 256) == before


def test_sizes_that_are_refused_have_no_tiles():
    assert sides(0, 8, 8) == sides(2, 32769, 32769) == sides(1, 0, 8) == (-1,) * 4
