"""The operators with K experts a token and the Newton-Schulz update without a
GPU: their argument checks (before any device work), and the 64-bit formulas
that the GPU tests compare with, against differences."""
import ctypes

import numpy as np
import pytest

import sparse_oracle as so
from neuralscript_amd import runtime

BUF = (ctypes.c_float * 64)()
HERE = ctypes.addressof(BUF) // 16 * 16 + 16  # never read: the calls are refused or empty


def refused(name, args):
    lib = runtime.lib()
    assert getattr(lib, "nsh_op_" + name)(*args) == -1, f"{name}{args} was not refused"
    assert name in lib.nsh_last_error().decode()


# logits, bias, active, idx, weight, T, E, K, groups, top_groups, group_best, score, renorm, scale, stream
ROUTE = [HERE, None, None, HERE, HERE, 4, 8, 2, 1, 1, 1, 0, 0, 1.0, None]


@pytest.mark.parametrize("at,value", [(0, None), (3, None), (4, None), (5, -1), (5, (1 << 24) + 1), (6, 0), (6, 1025),
                                      (7, 0), (7, 9), (7, 65), (8, 0), (8, 3), (8, 65), (9, 0), (9, 2), (10, 0),
                                      (10, 3), (11, 2), (11, -1)])
def test_route_refuses(at, value):
    a = list(ROUTE)
    a[at] = value
    refused("moe_route", a)


# dweight, logits, active, idx, dlogits, T, E, K, score, renorm, scale, stream
ROUTE_GRAD = [HERE, HERE, None, HERE, HERE, 4, 8, 2, 0, 0, 1.0, None]


@pytest.mark.parametrize("at,value", [(0, None), (1, None), (3, None), (4, None), (5, -1), (5, (1 << 24) + 1), (6, 0),
                                      (6, 1025), (7, 0), (7, 65), (8, 2)])
def test_route_grad_refuses(at, value):
    a = list(ROUTE_GRAD)
    a[at] = value
    refused("moe_route_grad", a)


# x, idx, weight, W1, W2, y, T, K, D, H, E, act, state, workspace, stream
EXPERTS = [HERE] * 6 + [4, 2, 8, 8, 4, 6, None, HERE, None]
# dy, x, weight, W1, W2, state, dx, dweight, dW1, dW2, T, K, D, H, E, act, workspace, stream
EXPERTS_GRAD = [HERE] * 10 + [4, 2, 8, 8, 4, 6, HERE, None]
SHAPES = [(0, -1), (0, (1 << 24) + 1), (0, 1 << 23), (1, 0), (1, 65), (2, 0), (2, 1 << 26), (3, 0), (3, 1 << 26), (4, 0),
          (4, 1025), (5, -1), (5, 7)]


@pytest.mark.parametrize("at,value", [(i, None) for i in range(6)] + [(6 + i, v) for i, v in SHAPES] +
                         [(12, HERE + 4), (13, None), (13, HERE + 8)])
def test_experts_refuses(at, value):
    a = list(EXPERTS)
    a[at] = value
    if value == 1 << 23:
        a[7] = 4  # T K beyond the slots
    refused("moe_experts", a)


@pytest.mark.parametrize("at,value", [(i, None) for i in range(6)] + [(10 + i, v) for i, v in SHAPES] +
                         [(5, HERE + 4), (16, None), (16, HERE + 8)])
def test_experts_grad_refuses(at, value):
    a = list(EXPERTS_GRAD)
    a[at] = value
    if value == 1 << 23:
        a[11] = 4
    refused("moe_experts_grad", a)


def test_experts_sizes_that_are_refused_need_no_room():
    lib = runtime.lib()
    for shape in ((0, 2, 8, 8, 4), (4, 65, 8, 8, 4), (4, 2, 0, 8, 4), (4, 2, 8, 8, 1025), (-1, 2, 8, 8, 4),
                  (1 << 24, 1, 1 << 14, 8, 4)):
        assert lib.nsh_op_moe_experts_state(*shape) == 0
        assert lib.nsh_op_moe_experts_workspace(*shape, 0) == 0
        assert lib.nsh_op_moe_experts_workspace(*shape, 1) == 0
    a = list(EXPERTS)
    a[6:11] = [1 << 24, 1, 1 << 14, 8, 4]  # more workgroups than a grid holds
    refused("moe_experts", a)


# g, q, n, r, c, steps, workspace, stream
NS = [HERE, HERE, 2, 8, 8, 5, HERE, None]
# w, g, m, n, r, c, lr, mu, nesterov, steps, workspace, stream
MUON = [HERE, HERE, None, 2, 8, 8, 0.1, 0.9, 1, 5, HERE, None]


@pytest.mark.parametrize("at,value", [(0, None), (1, None), (2, -1), (2, 65536), (3, 0), (3, (1 << 22) + 1), (4, 0),
                                      (4, -8), (5, -1), (5, 101), (6, None), (6, HERE + 4)])
def test_newton_schulz_refuses(at, value):
    a = list(NS)
    a[at] = value
    refused("newton_schulz", a)


@pytest.mark.parametrize("at,value", [(0, None), (1, None), (3, -1), (3, 65536), (4, 0), (5, (1 << 22) + 1), (9, -1),
                                      (9, 101), (10, None), (10, HERE + 4)])
def test_muon_ns_step_refuses(at, value):
    a = list(MUON)
    a[at] = value
    refused("muon_ns_step", a)


def test_newton_schulz_refuses_two_large_sides():
    a = list(NS)
    a[3] = a[4] = 32769
    refused("newton_schulz", a)
    assert runtime.lib().nsh_op_newton_schulz_workspace(2, 32769, 32769) == 0
    a[2:5] = [17, 32768, 32768]  # more blocks than a grid holds
    refused("newton_schulz", a)


def test_empty_calls_succeed():
    lib = runtime.lib()
    none = [None] * 5
    assert lib.nsh_op_moe_route(*none, 0, 8, 2, 1, 1, 1, 0, 0, 1.0, None) == 0
    assert lib.nsh_op_moe_route_grad(*none, 0, 8, 2, 0, 0, 1.0, None) == 0
    assert lib.nsh_op_moe_experts(*none, None, 0, 2, 8, 8, 4, 6, None, None, None) == 0
    assert lib.nsh_op_moe_experts_grad(*none, *none, 0, 2, 8, 8, 4, 6, None, None) == 0
    assert lib.nsh_op_newton_schulz(None, None, 0, 8, 8, 5, None, None) == 0
    assert lib.nsh_op_muon_ns_step(None, None, None, 0, 8, 8, 0.1, 0.9, 1, 5, None, None) == 0


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("renorm", [0, 1])
def test_route_gradient_formula_against_differences(score, renorm):
    """Central differences of step h: their truncation is h^2 / 6 times a third
    derivative of order 1, their rounding 1e-16 / h: 1e-9 at h = 1e-5."""
    rng = np.random.default_rng(3)
    T, E, K = 3, 7, 3
    l = rng.normal(size=(T, E))
    active = np.array([1, 1, 0, 1, 1, 1, 1], np.uint8)
    idx, _ = so.route(l, None, active, K, score=score)
    idx[1, 2] = -1
    idx[2, 1] = idx[2, 0]  # the same expert twice
    dw = rng.normal(size=(T, K))
    got, _ = so.route_grad(dw, l, active, idx, score, renorm, 1.7)
    h = 1e-5
    for t in range(T):
        for e in range(E):
            up, down = l.copy(), l.copy()
            up[t, e] += h
            down[t, e] -= h
            d = sum((s * (dw * so.weights_of(v, active, idx, score, renorm, 1.7)).sum()) for s, v in ((1, up), (-1, down)))
            assert abs(d / (2 * h) - got[t, e]) < 1e-8


@pytest.mark.parametrize("code", [0, 3, 4, 5, 6])
def test_experts_gradient_formula_against_differences(code):
    """As above; the activations' constants are the floats that the kernels use
    (2e-9 off), so 1e-7."""
    rng = np.random.default_rng(code)
    T, K, D, H, E = 4, 2, 3, 5, 3
    x, dy = rng.normal(size=(T, D)), rng.normal(size=(T, D))
    W = {"W1": rng.normal(size=(E, D, H)), "W2": rng.normal(size=(E, H, D)), "x": x, "weight": rng.random((T, K))}
    idx = np.array([[0, 1], [1, 1], [-1, 2], [0, 5]])
    out, _ = so.experts(x, idx, W["weight"], W["W1"], W["W2"], code, dy)
    h = 1e-5
    for name, grad in (("x", "dx"), ("weight", "dweight"), ("W1", "dW1"), ("W2", "dW2")):
        for at in np.ndindex(W[name].shape):
            d = 0.0
            for s in (1, -1):
                v = {k: a.copy() for k, a in W.items()}
                v[name][at] += s * h
                d += s * (dy * so.experts(v["x"], idx, v["weight"], v["W1"], v["W2"], code)[0]["y"]).sum()
            assert abs(d / (2 * h) - out[grad][at]) < 1e-7, (name, at)


def test_newton_schulz_drives_the_singular_values():
    """Each step maps a singular value s to a s + b s^3 + c s^5 and keeps the vectors."""
    rng = np.random.default_rng(5)
    g = rng.normal(size=(12, 30))
    u, s, vt = np.linalg.svd(g, full_matrices=False)
    s = s / (np.linalg.norm(g) + 1e-7)
    for _ in range(5):
        s = so.NS[0] * s + so.NS[1] * s ** 3 + so.NS[2] * s ** 5
    assert np.allclose(so.newton_schulz(g), (u * s) @ vt, atol=1e-12)
    assert np.allclose(so.newton_schulz(g.T), so.newton_schulz(g).T, atol=1e-13)


@pytest.mark.parametrize("shape", [(400, 2, 200, 333, 4), (64, 2, 256, 256, 40), (3200, 2, 1024, 1024, 16)])
def test_sizes_of_a_layer_do_not_hang_on_the_environment(shape, monkeypatch):
    """A variable that changes between a sizing call and its launch, or between a
    forward and its gradient, must not change what a buffer has to hold."""
    lib = runtime.lib()
    sizes = lambda: (lib.nsh_op_moe_experts_state(*shape), lib.nsh_op_moe_experts_workspace(*shape, 0),  # noqa: E731
                     lib.nsh_op_moe_experts_workspace(*shape, 1))
    before = sizes()
    for value in ("1", "16", "100000"):
        monkeypatch.setenv("NSHIP_MOE_SPLIT_MIN", value)
        assert sizes() == before


def test_a_tests_choice_of_the_pieces_ends_with_it():
    lib = runtime.lib()
    shape = (400, 2, 200, 333, 4)
    before = lib.nsh_op_moe_experts_state(*shape)
    try:
        lib.nsh_test_moe_split_least(ctypes.c_int64(16))
        assert lib.nsh_op_moe_experts_state(*shape) != before
    finally:
        lib.nsh_test_moe_split_least(ctypes.c_int64(0))
    assert lib.nsh_op_moe_experts_state(*shape) == before
