"""Every kernel of the Newton-Schulz products, by its tiles' side, against the
formula in 64 bits: sides that a test asks for at small ragged sizes, and those
that the rule picks at sizes of their own."""
import ctypes

import numpy as np
import pytest

import sparse_oracle as so
from neuralscript_amd import runtime
from sparse_oracle import U, p, put, room
from test_moe_branches_gpu import repeated, window
from test_newton_schulz_gpu import close, run_ns
from test_sparse_large_gpu import Plain, room_for

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


def close_by_rows(got, g, what):
    """Each row by itself: four times fp32's error and 16 U, as close() allows, and
    what entries below fp16's normal range lose.  With m <= N and rho the row's share
    of |G|_F: an entry of X or S is off by at most e = 2^-51, of P by 2 e, so a step
    leaves a row's S off by 1.21 e sqrt(N) + e sqrt(m), its P by 2 e sqrt(m) + 10.7 times
    that (4.775 + 2 2.0315 1.21^2 of it), and X by 1.21 times P's and 3.45 e sqrt(N):
    35 e sqrt(N) in all, of a row that starts at rho and that no step makes
    smaller than by 0.68: 5 steps' are below 2^8 e sqrt(N) / rho."""
    want, fp32 = so.newton_schulz(g), so.newton_schulz(g, 5, np.float32)
    size = np.linalg.norm(want, axis=1)
    rho = np.linalg.norm(g.astype(np.float64), axis=1) / np.linalg.norm(g.astype(np.float64))
    off = np.linalg.norm(got - want, axis=1)
    allowed = 4 * np.linalg.norm(fp32 - want, axis=1) + (16 * U + 2.0 ** -43 * np.sqrt(max(g.shape)) / rho) * size
    print(f"  {what}: rows off by {(off / size).max():.3g}, {(off / allowed).max():.3g} of the bound", flush=True)
    assert np.all(off <= allowed), what


def small_rows(r, c, scale, seed):
    g = np.random.default_rng(seed).normal(size=(1, r, c)).astype(np.float32)
    g[:, ::3] *= np.float32(scale)
    return g


@pytest.mark.parametrize("scale", [1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("r,c", [(130, 300), (300, 130), (257, 257)])
def test_small_rows_keep_their_own_accuracy_by_tiles(r, c, scale, side):
    """Rows of an embedding that few tokens read."""
    g = small_rows(r, c, scale, r)
    close_by_rows(run_ns(g)[0], g[0], f"{r} x {c}, {scale:g}, tiles of {side}")


@pytest.mark.parametrize("scale", [1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("r,c", [(64, 256), (256, 64), (90, 90), (512, 2048), (2048, 512)])
def test_small_rows_keep_their_own_accuracy(r, c, scale):
    g = small_rows(r, c, scale, c)
    close_by_rows(run_ns(g)[0], g[0], f"{r} x {c}, {scale:g}")


@pytest.mark.parametrize("r,c,by", [(40, 72, 0), (72, 40, 0), (40, 72, 32), (72, 40, 64), (140, 72, 128), (72, 140, 256)])
@pytest.mark.parametrize("steps", [1, 2, 3, 5])
def test_the_smallest_gradients(r, c, by, steps):
    """A gradient of a few of fp32's smallest values: its norm is far below the 1e-7
    beside it, and a few steps leave X small, but within fp32's normal range.  One
    entry a row and column, so each is scaled by 3.4445^steps / 1e-7 up to rounding:
    16 U, and the 2 U of a norm next to 1e-7."""
    g = np.zeros((1, r, c), np.float32)
    for i in range(3):
        g[0, 7 * i, 11 * i] = (-1) ** i * (i + 3) * 1.4013e-45
    runtime.lib().nsh_test_newton_tile(by)
    try:
        got = run_ns(g, steps)[0].astype(np.float64)
    finally:
        runtime.lib().nsh_test_newton_tile(0)
    want = g[0].astype(np.float64) / 1e-7 * so.NS[0] ** steps
    assert np.abs(want[want != 0]).min() > 1.2e-38
    assert np.all(np.abs(got - want) <= 18 * steps * U * np.abs(want))


def test_matrices_beyond_32_bits():
    """2^31 entries and more, in place: four matrices over and over."""
    n, r, c = 2052, 1024, 1032
    g = np.random.default_rng(3).normal(size=(4, r, c)).astype(np.float32)
    ws = runtime.lib().nsh_op_newton_schulz_workspace(n, r, c)
    assert n * r * c > 1 << 31
    room_for(ws + 4 * n * r * c + (1 << 30))
    d, room_ = repeated(g, n // 4), Plain(ws, 0xFF)
    runtime.op("newton_schulz", d.ptr, d.ptr, n, r, c, 1, room_.ptr, None)
    so.sync()
    first = window(d, 0, g.shape)
    for i in range(2):
        close(first[i], g[i], f"matrix {i}", 1)
    for at in (n // 8 * 4, n - 4):  # (whole periods)
        assert np.array_equal(window(d, at, g.shape), first)
    d.free()
    room_.free()
