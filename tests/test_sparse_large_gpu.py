"""Newton-Schulz near its largest sizes: launches of up to 2^32 threads."""
import ctypes

import numpy as np
import pytest

import sparse_oracle as so
from neuralscript_amd import runtime
from sparse_oracle import U, p, put

pytestmark = pytest.mark.gpu


class Plain:
    """Device memory without a host copy."""

    def __init__(self, nbytes, fill=0):
        d = ctypes.c_void_p()
        so.hip("hipMalloc", ctypes.byref(d), ctypes.c_size_t(nbytes))
        self.ptr = d.value
        so.hip("hipMemset", ctypes.c_void_p(self.ptr), fill, ctypes.c_size_t(nbytes))

    def free(self):
        so.hip("hipFree", ctypes.c_void_p(self.ptr))


def room_for(nbytes):
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    so.hip("hipMemGetInfo", ctypes.byref(free), ctypes.byref(total))
    if free.value < nbytes:
        pytest.skip(f"{nbytes >> 30} GiB of device memory wanted")


def test_newton_schulz_of_many_long_rows():
    """2^23 tiles of 32 x 32: 2^32 threads if they were dealt out so."""
    n, c = 32768, 8192
    ws = runtime.lib().nsh_op_newton_schulz_workspace(n, 1, c)
    room_for(ws + (3 << 30))
    rows = np.random.default_rng(0).normal(size=(8, c)).astype(np.float32)
    g = np.tile(rows, (n // 8, 1))
    d, w = put(g), Plain(ws, 0xFF)
    runtime.op("newton_schulz", p(d), p(d), n, 1, c, 5, w.ptr, None)
    so.sync()
    got = d.host((n // 8, 8, c))
    w.free()
    assert np.array_equal(got, np.broadcast_to(got[:1], got.shape))
    for i in range(8):
        want = so.newton_schulz(rows[i:i + 1])[0]
        assert np.linalg.norm(got[0, i] - want) <= 100 * U * np.linalg.norm(want)  # (five steps' roundings)
