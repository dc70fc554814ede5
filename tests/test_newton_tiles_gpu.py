"""Every kernel of the Newton-Schulz products, by its tiles' side, against the
formula in 64 bits: sides that a test asks for at small ragged sizes, and those
that the rule picks at sizes of their own."""
import ctypes

import numpy as np
import pytest

import sparse_oracle as so
from neuralscript_amd import runtime
from sparse_oracle import U, p, put, room
from test_newton_schulz_gpu import close, run_ns

pytestmark = pytest.mark.gpu
i64 = ctypes.c_int64
SIDES = (32, 64, 128, 256)


@pytest.fixture(params=SIDES)
def side(request):
    runtime.lib().nsh_test_newton_tile(request.param)
    yield request.param
    runtime.lib().nsh_test_newton_tile(0)


# one tile and several, ragged by one row and column, both orders, more matrices
# than one, a length of K below a slab's
SHAPES = [(1, 1, 1), (2, 1, 7), (2, 9, 1), (3, 5, 5), (2, 31, 33), (2, 63, 65), (2, 65, 63), (1, 127, 300), (1, 300, 129),
          (2, 255, 257), (1, 257, 255), (3, 100, 333), (1, 520, 300), (1, 300, 520), (1, 513, 513), (1, 40, 1500)]


@pytest.mark.parametrize("n,r,c", SHAPES)
def test_newton_schulz_by_tiles(n, r, c, side):
    print(f"newton_schulz {n} {r} {c} tiles of {side}", flush=True)
    assert all(runtime.lib().nsh_test_newton_side(k, i64(n), i64(r), i64(c)) == side for k in range(4))
    g = np.random.default_rng(n + r + c).normal(size=(n, r, c)).astype(np.float32)
    for steps in (1, 5):
        got = run_ns(g, steps)
        for i in range(n):
            close(got[i], g[i], f"matrix {i}, {steps} steps", steps)
    assert np.array_equal(run_ns(g, in_place=True), got)


@pytest.mark.parametrize("n,r,c", [(2, 70, 130), (2, 130, 70), (1, 260, 300), (1, 300, 260)])
@pytest.mark.parametrize("nesterov", [0, 1])
def test_muon_ns_step_by_tiles(n, r, c, nesterov, side):
    print(f"muon_ns_step {n} {r} {c} {nesterov} tiles of {side}", flush=True)
    rng = np.random.default_rng(r + c)
    w, g, m = (rng.normal(size=(n, r, c)).astype(np.float32) for _ in range(3))
    lr, mu = np.float32(0.02), np.float32(0.9)
    dw, dg, dm = put(w, shift=1), put(g, shift=1), put(m, shift=1)
    ws = room(runtime.lib().nsh_op_newton_schulz_workspace(n, r, c))
    runtime.op("muon_ns_step", p(dw), p(dg), p(dm), n, r, c, float(lr), float(mu), nesterov, 5, p(ws), None)
    so.sync()
    ws.host()
    new = np.float64(mu) * m + g
    assert np.all(np.abs(dm.host(m.shape) - new) <= 2 * U * (np.abs(np.float64(mu) * m) + np.abs(g)))
    u = g + np.float64(mu) * new if nesterov else new
    got = dw.host(w.shape)
    for i in range(n):
        q = so.newton_schulz(u[i])
        step = float(lr) * np.sqrt(min(r, c))
        want = w[i] - step * q - 0.01 * float(lr) * w[i]
        fp32 = np.linalg.norm(so.newton_schulz(u[i].astype(np.float32), 5, np.float32) - q)
        # as in test_muon_ns_step
        allowed = step * (4 * fp32 + 16 * U * np.linalg.norm(q) + 3 * U * 485) + \
            4 * U * np.linalg.norm(np.abs(w[i]) + step * np.abs(q))
        assert np.linalg.norm(got[i] - want) <= allowed


def test_unbounded_matrices_by_tiles(side):
    g = np.random.default_rng(8).normal(size=(5, 150, 130)).astype(np.float32)
    alone = run_ns(g)
    g[1], g[2, 3, 5], g[3, 149, 0] = 0, np.nan, np.inf
    got = run_ns(g)
    assert np.all(got[1] == 0) and np.isnan(got[2]).all() and np.isnan(got[3]).all()
    assert np.array_equal(got[0], alone[0]) and np.array_equal(got[4], alone[4])


# sizes at which the rule picks tiles of 64, 128 and 256 for one product or another
# (test_newton_tiles.py); a few of the matrices are checked
RULE = [(3, 1000, 333), (4, 512, 512), (16, 300, 300), (64, 200, 333), (1, 2500, 2300), (64, 1000, 1020),
        (64, 1020, 1000), (16, 1280, 1280)]


@pytest.mark.parametrize("n,r,c", RULE)
def test_newton_schulz_by_the_rule(n, r, c):
    print(f"newton_schulz {n} {r} {c}", flush=True)
    few = np.random.default_rng(r + c).normal(size=(3, r, c)).astype(np.float32)
    g = np.concatenate([few] + [few[:1]] * (n - 3)) if n > 3 else few[:n]
    out = run_ns(g, 2)
    for i in range(min(n, 2)):
        close(out[i], g[i], f"matrix {i}", 2)
    assert all(np.array_equal(out[i], out[0]) for i in range(3, n))
