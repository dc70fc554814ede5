"""Newton-Schulz orthogonalisation and the Muon step on it against the formula
in 64 bits, and a sparse layer's whole training step through the operators."""
import ctypes

import numpy as np
import pytest

import sparse_oracle as so
from neuralscript_amd import runtime
from sparse_oracle import Guarded, U, p, put, room

pytestmark = pytest.mark.gpu


def run_ns(g, steps=5, shift=0, in_place=False, stream=None):
    n, r, c = g.shape
    d = put(g, shift=shift)
    q = d if in_place else Guarded(g.size, shift=shift)
    ws = room(runtime.lib().nsh_op_newton_schulz_workspace(n, r, c))
    runtime.op("newton_schulz", p(d), p(q), n, r, c, steps, p(ws), stream)
    so.sync(stream)
    ws.host()
    return q.host(g.shape)


def close(got, g, what, steps=5):
    """The relative error of a result is at most four times that of the formula
    evaluated in fp32, plus 16 U: its products keep fp32's accuracy (operands to
    2 U instead of U, a product to 4 U), and the steps carry both alike."""
    want = so.newton_schulz(g, steps)
    n = np.linalg.norm(want)
    fp32 = np.linalg.norm(so.newton_schulz(g, steps, np.float32) - want) / n
    err = np.linalg.norm(got - want) / n
    print(f"  {what}: error {err:.3g}, of fp32 {fp32:.3g}", flush=True)
    assert err <= 4 * fp32 + 16 * U, what


# vectors and single values, odd sizes, both orders, sizes around the tiles'
# edges, batches
SHAPES = [(1, 1, 1), (2, 1, 7), (2, 9, 1), (3, 5, 5), (1, 16, 64), (8, 64, 256), (2, 63, 65), (2, 65, 63), (1, 33, 300),
          (1, 128, 128), (2, 129, 130), (3, 100, 333), (1, 257, 100), (2, 512, 200), (1, 300, 700), (1, 1024, 64),
          (1, 2048, 130)]


@pytest.mark.parametrize("n,r,c", SHAPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_newton_schulz(n, r, c, shift):
    print(f"newton_schulz {n} {r} {c} {shift}", flush=True)
    rng = np.random.default_rng(n + r + c)
    g = rng.normal(size=(n, r, c)).astype(np.float32)
    got = run_ns(g, shift=shift)
    for i in range(n):
        close(got[i], g[i], f"matrix {i}")


@pytest.mark.parametrize("steps", [0, 1, 2, 3, 4, 8])
def test_newton_schulz_steps(steps):
    g = np.random.default_rng(steps).normal(size=(2, 70, 90)).astype(np.float32)
    got = run_ns(g, steps)
    for i in range(2):
        close(got[i], g[i], f"{steps} steps", steps)


@pytest.mark.parametrize("scale", [1e-28, 1e-15, 1e20])
def test_newton_schulz_of_any_scale(scale):
    """The norm's 1e-7 counts beside the smallest; squares beyond fp32's range do not."""
    g = (np.random.default_rng(4).normal(size=(2, 40, 72)) * scale).astype(np.float32)
    got = run_ns(g)
    for i in range(2):
        close(got[i], g[i], f"scale {scale}")


@pytest.mark.parametrize("n,r,c", [(2, 200, 150), (1, 64, 256), (1, 700, 130)])
def test_newton_schulz_of_gradients_with_zero_and_small_rows(n, r, c):
    """Rows of an embedding that no token read, rows a million times smaller, a
    gradient of rank 3, one entry alone."""
    rng = np.random.default_rng(r)
    zero = rng.normal(size=(n, r, c)).astype(np.float32)
    zero[:, rng.random(r) < 0.6] = 0
    small = rng.normal(size=(n, r, c)).astype(np.float32)
    small[:, ::3] *= 1e-6
    low = (rng.normal(size=(n, r, 3)) @ rng.normal(size=(n, 3, c))).astype(np.float32)
    single = np.zeros((n, r, c), np.float32)
    single[:, r // 2, c // 3] = -3.0
    for what, g in (("zero rows", zero), ("small rows", small), ("rank 3", low), ("one entry", single)):
        got = run_ns(g)
        for i in range(n):
            close(got[i], g[i], what)
        if what == "zero rows":
            assert np.all(got[g == 0] == 0)


def test_newton_schulz_of_zero_and_unbounded_matrices():
    for r, c in ((48, 80), (200, 130)):
        g = np.random.default_rng(8).normal(size=(5, r, c)).astype(np.float32)
        alone = run_ns(g)
        g[1], g[2, 3, 5], g[3, r - 1, 0] = 0, np.nan, np.inf
        got = run_ns(g)
        assert np.all(got[1] == 0) and np.isnan(got[2]).all() and np.isnan(got[3]).all()
        assert np.array_equal(got[0], alone[0]) and np.array_equal(got[4], alone[4])


@pytest.mark.parametrize("n,r,c", [(2, 64, 256), (1, 333, 100), (3, 150, 150)])
def test_newton_schulz_in_place(n, r, c):
    g = np.random.default_rng(r).normal(size=(n, r, c)).astype(np.float32)
    assert np.array_equal(run_ns(g, in_place=True), run_ns(g))


def test_newton_schulz_equal_calls_give_equal_bits():
    g = np.random.default_rng(2).normal(size=(2, 200, 300)).astype(np.float32)
    assert np.array_equal(run_ns(g), run_ns(g))


@pytest.mark.parametrize("n,r,c", [(1, 1, 5), (8, 64, 256), (2, 100, 33), (2, 130, 260)])
@pytest.mark.parametrize("momentum,nesterov", [(0, 0), (1, 0), (1, 1)])
@pytest.mark.parametrize("shift", [0, 1])
def test_muon_ns_step(n, r, c, momentum, nesterov, shift):
    print(f"muon_ns_step {n} {r} {c} {momentum} {nesterov} {shift}", flush=True)
    rng = np.random.default_rng(r + c)
    w, g, m = (rng.normal(size=(n, r, c)).astype(np.float32) for _ in range(3))
    lr, mu = np.float32(0.02), np.float32(0.9)
    dw, dg, dm = put(w, shift=shift), put(g, shift=shift), put(m, shift=shift) if momentum else None
    ws = room(runtime.lib().nsh_op_newton_schulz_workspace(n, r, c))
    runtime.op("muon_ns_step", p(dw), p(dg), p(dm), n, r, c, float(lr), float(mu), nesterov, 5, p(ws), None)
    so.sync()
    ws.host()
    assert np.array_equal(dg.host(g.shape), g)
    u = g.astype(np.float64)
    if momentum:
        new = np.float64(mu) * m + g
        got = dm.host(m.shape)
        size = np.abs(np.float64(mu) * m) + np.abs(g)
        assert np.all(np.abs(got - new) <= 2 * U * size)  # a product and a sum, or both at once
        u = g + np.float64(mu) * new if nesterov else new
    got = dw.host(w.shape)
    for i in range(n):
        q = so.newton_schulz(u[i])
        step = float(lr) * np.sqrt(min(r, c))
        want = w[i] - step * q - 0.01 * float(lr) * w[i]
        fp32 = np.linalg.norm(so.newton_schulz(u[i].astype(np.float32), 5, np.float32) - q)
        # the update to what close() allows, u rounded twice (carried by at most
        # 3.4445^5 into values whose norm was 1), and the weight's own roundings
        allowed = step * (4 * fp32 + 16 * U * np.linalg.norm(q) + 3 * U * 485) + 4 * U * np.linalg.norm(np.abs(w[i]) + step * np.abs(q))
        assert np.linalg.norm(got[i] - want) <= allowed


# ---- together ---------------------------------------------------------------------

class Layer:
    """A sparse layer's training step on device buffers: route, the experts,
    their gradients, the logits' gradient, Newton-Schulz updates of both
    matrices of every expert."""

    def __init__(self, T, K, D, H, E, seed):
        rng = np.random.default_rng(seed)
        f = lambda *s, scale=1.0: (rng.normal(size=s) * scale).astype(np.float32)  # noqa: E731
        lib = runtime.lib()
        self.size = (T, K, D, H, E)
        self.host = {"x": f(T, D), "logits": f(T, E), "bias": f(E, scale=0.1), "dy": f(T, D),
                     "W1": f(E, D, H, scale=D ** -0.5), "W2": f(E, H, D, scale=H ** -0.5)}
        self.d = {k: put(v) for k, v in self.host.items()}
        self.d["idx"] = Guarded(T * K, np.int32)
        for k, n in (("weight", T * K), ("y", T * D), ("dx", T * D), ("dweight", T * K), ("dlogits", T * E),
                     ("dW1", E * D * H), ("dW2", E * H * D)):
            self.d[k] = Guarded(n)
        self.d["m1"], self.d["m2"] = put(np.zeros(E * D * H)), put(np.zeros(E * H * D))
        self.state = room(lib.nsh_op_moe_experts_state(*self.size))
        self.ws = room(max(lib.nsh_op_moe_experts_workspace(*self.size, 1), lib.nsh_op_newton_schulz_workspace(E, D, H)))

    LR, MU = 0.01, 0.9

    def step(self, stream):
        T, K, D, H, E = self.size
        q = lambda *names: [self.d[n].ptr for n in names]  # noqa: E731
        runtime.op("moe_route", *q("logits", "bias"), None, *q("idx", "weight"), T, E, K, 1, 1, 1, 0, 1, 1.0, stream)
        runtime.op("moe_experts", *q("x", "idx", "weight", "W1", "W2", "y"), *self.size, 6, p(self.state), p(self.ws), stream)
        runtime.op("moe_experts_grad", *q("dy", "x", "weight", "W1", "W2"), p(self.state),
                   *q("dx", "dweight", "dW1", "dW2"), *self.size, 6, p(self.ws), stream)
        runtime.op("moe_route_grad", *q("dweight", "logits"), None, *q("idx", "dlogits"), T, E, K, 0, 1, 1.0, stream)
        runtime.op("muon_ns_step", *q("W1", "dW1", "m1"), E, D, H, self.LR, self.MU, 1, 5, p(self.ws), stream)
        runtime.op("muon_ns_step", *q("W2", "dW2", "m2"), E, H, D, self.LR, self.MU, 1, 5, p(self.ws), stream)

    OUT = ("idx", "weight", "y", "dx", "dweight", "dlogits", "dW1", "dW2", "W1", "W2", "m1", "m2")

    def read(self):
        return {k: self.d[k].host() for k in self.OUT}


def test_a_sparse_layers_training_step():
    T, K, D, H, E = 200, 2, 48, 64, 6
    a = Layer(T, K, D, H, E, 1)
    stream = so.new_stream()
    a.step(stream)
    so.sync(stream)
    got, h = a.read(), a.host
    idx, weight = so.route(h["logits"], h["bias"], None, K, renorm=1)
    assert np.array_equal(got["idx"].reshape(T, K), idx)
    out, off = so.experts(h["x"], idx, weight, h["W1"], h["W2"], 6, h["dy"])
    for k in ("y", "dx", "dweight", "dW1", "dW2"):
        d = np.abs(got[k].reshape(out[k].shape) - out[k])
        assert np.all(d <= 1.01 * off[k] + 4 * U * np.abs(out[k]) + 1e-30), k  # (the weights rounded once more)
    dl, size = so.route_grad(out["dweight"], h["logits"], None, idx, 0, 1, 1.0)
    assert np.linalg.norm(got["dlogits"].reshape(T, E) - dl) <= 1e-5 * np.linalg.norm(size)
    for k, g in (("W1", out["dW1"]), ("W2", out["dW2"])):
        for e in range(E):
            q = so.newton_schulz(g[e] + a.MU * g[e])
            want = h[k][e] - a.LR * np.sqrt(min(D, H)) * q - 0.01 * a.LR * h[k][e]
            d = np.linalg.norm(got[k].reshape(h[k].shape)[e] - want)
            # the gradients' 1e-5 at most, carried by up to 3.4445^5 / |q|
            assert d <= a.LR * np.sqrt(min(D, H)) * 485 * 1e-5, (k, e, d)


@pytest.mark.parametrize("pieces", [False, True])
def test_a_training_step_captured_and_replayed(pieces, monkeypatch):
    """Two layers of different sizes as two graphs, replayed in turn with eager
    steps of a third between them: every replay gives the eager steps' bits."""
    stream = so.new_stream()
    sizes = [(96, 2, 64, 96, 5), (12, 3, 36, 20, 4)]
    if pieces:
        monkeypatch.setenv("NSHIP_MOE_SPLIT_MIN", "16")
        sizes = [(200, 2, 136, 260, 5), (150, 3, 200, 140, 4)]
    eager = []
    for i, s in enumerate(sizes):
        a = Layer(*s, i)
        seen = []
        for _ in range(3):
            a.step(stream)
            so.sync(stream)
            seen.append(a.read())
        eager.append(seen)
    layers = [Layer(*s, i) for i, s in enumerate(sizes)]
    other = Layer(40, 2, 32, 32, 4, 9)
    graphs = [so.capture(stream, lambda a=a: a.step(stream)) for a in layers]
    for n in range(3):
        for x in graphs:
            so.replay(x, stream)
        other.step(stream)
        so.sync(stream)
        for a, seen in zip(layers, eager):
            got = a.read()
            assert all(np.array_equal(got[k], seen[n][k]) for k in a.OUT), n


def test_two_streams_at_once():
    """Steps of two layers with workspaces of their own on two streams."""
    a, b = Layer(96, 2, 64, 96, 5, 0), Layer(300, 2, 32, 64, 4, 1)
    c, d = Layer(96, 2, 64, 96, 5, 0), Layer(300, 2, 32, 64, 4, 1)
    s, t = so.new_stream(), so.new_stream()
    for _ in range(3):
        a.step(s)
        b.step(t)
    so.sync(s)
    so.sync(t)
    for _ in range(3):
        c.step(s)
        d.step(s)
    so.sync(s)
    for x, y in ((a, c), (b, d)):
        p1, p2 = x.read(), y.read()
        assert all(np.array_equal(p1[k], p2[k]) for k in x.OUT)
