"""Routing to K experts a token and the experts' products, forward and
backward, against their 64-bit formulas (sparse_oracle.py)."""
import numpy as np
import pytest

import sparse_oracle as so
from neuralscript_amd import runtime
from sparse_oracle import Guarded, U, p, put, room

pytestmark = pytest.mark.gpu


# ---- routing ----------------------------------------------------------------------

def run_route(l, bias, active, K, groups=1, top=1, best=1, score=0, renorm=0, scale=1.0, shift=0, stream=None):
    T, E = l.shape
    dl, db, da = put(l, shift=shift), put(bias, shift=shift), put(active, np.uint8, shift)
    idx, w = Guarded(T * K, np.int32, shift), Guarded(T * K, shift=shift)
    runtime.op("moe_route", p(dl), p(db), p(da), p(idx), p(w), T, E, K, groups, top, best, score, renorm, scale, stream)
    so.sync(stream)
    return idx.host((T, K)), w.host((T, K))


def check_route(l, bias, active, K, groups=1, top=1, best=1, score=0, renorm=0, scale=1.0, **more):
    idx, w = run_route(l, bias, active, K, groups, top, best, score, renorm, scale, **more)
    want, weight = so.route(l, bias, active, K, groups, top, best, score, renorm, scale)
    assert np.array_equal(idx, want), np.argwhere(idx != want)[:5]
    # 64 bits (a few 1e-16) rounded once
    off = np.abs(w.astype(np.float64) - weight)
    assert np.all(off <= 1.001 * U * np.abs(weight) + 1e-37), off.max()
    return idx, w


# every register layout (up to 64, 128, 256, 512 and 1024 experts) with ragged
# and full counts, one token and odd numbers of them, every K that matters
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 8, 8), (3, 60, 4), (5, 64, 64), (257, 64, 2), (2, 65, 7), (7, 128, 8),
                                   (33, 200, 3), (9, 256, 16), (4, 300, 64), (6, 512, 5), (3, 777, 6), (5, 1024, 64)])
@pytest.mark.parametrize("score", [0, 1])
def test_route(T, E, K, score):
    print(f"route {T} {E} {K} {score}", flush=True)
    rng = np.random.default_rng(T * 1000 + E)
    l = rng.normal(size=(T, E)).astype(np.float32) * 2
    bias = rng.normal(size=E).astype(np.float32) * 0.1
    check_route(l, None, None, K, score=score, renorm=1)
    check_route(l, bias, (rng.random(E) < 0.8).astype(np.uint8), K, score=score, scale=2.5, shift=1)


@pytest.mark.parametrize("E,groups,top,K", [(8, 2, 1, 3), (64, 8, 4, 8), (60, 5, 2, 6), (256, 8, 4, 8), (1024, 64, 3, 20),
                                            (36, 36, 5, 5), (64, 64, 64, 4)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("score", [0, 1])
def test_route_groups(E, groups, top, K, best, score):
    print(f"route groups {E} {groups} {top} {K} {best} {score}", flush=True)
    rng = np.random.default_rng(E + groups)
    l = rng.normal(size=(37, E)).astype(np.float32)
    bias = rng.normal(size=E).astype(np.float32) * 0.2
    active = (rng.random(E) < 0.7).astype(np.uint8)
    check_route(l, bias, None, K, groups, top, best, score, renorm=1)
    check_route(l, bias, active, K, groups, top, best, score, renorm=1)
    active[: E // groups * max(1, groups - 1)] = 0  # one group left, fewer live experts than K
    check_route(l, None, active, K, groups, top, best, score)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("groups,top", [(1, 1), (4, 2)])
def test_route_ties_go_to_the_lower_index(score, groups, top):
    """Logits on a grid of four values, a bias on a grid of two: most places tie."""
    rng = np.random.default_rng(groups)
    l = rng.integers(0, 4, size=(65, 96)).astype(np.float32) / 4
    check_route(l, None, None, 9, groups, top, 2, score, renorm=1)
    check_route(np.zeros((3, 96), np.float32), None, None, 9, groups, top, 2, score)
    check_route(l, rng.integers(0, 2, 96).astype(np.float32), None, 9, groups, top, 1, score)


@pytest.mark.parametrize("score", [0, 1])
def test_route_values_next_to_a_border(score):
    """Logits a last place of fp32 apart: 64 bits tell the choices apart."""
    rng = np.random.default_rng(1)
    base = np.float32(0.7) + np.zeros((64, 128), np.float32)
    step = rng.integers(0, 3, size=base.shape)
    l = (base.view(np.int32) + step.astype(np.int32)).view(np.float32)
    check_route(l, None, None, 6, score=score, renorm=1)
    check_route(l, np.full(128, 0.25, np.float32), None, 6, score=score)


def special_logits(E):
    big = np.float32(3.4028235e38)
    rows = [np.full(E, -np.inf), np.full(E, np.nan), np.full(E, -big), np.full(E, big), np.full(E, np.inf),
            np.where(np.arange(E) % 3 == 0, np.inf, 0.0), np.where(np.arange(E) == E - 2, 0.5, -np.inf),
            np.where(np.arange(E) % 2 == 0, np.nan, np.arange(E) / 7), np.where(np.arange(E) < 2, -big, -np.inf),
            np.where(np.arange(E) == 3, 200.0, -200.0), np.where(np.arange(E) == 3, -1000.0, -1001.0)]
    return np.array(rows, np.float32)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("groups,top", [(1, 1), (4, 2)])
def test_route_masked_and_infinite_logits(score, renorm, groups, top):
    E = 24
    l = special_logits(E)
    idx, w = check_route(l, None, None, 5, groups, top, 2, score, renorm)
    assert np.all(idx[:2] == -1) and np.all(w[:2] == 0) and np.all(np.isfinite(w))
    check_route(l, None, np.zeros(E, np.uint8), 5, groups, top, 2, score, renorm)
    bias = np.zeros(E, np.float32)
    bias[[1, 4]] = np.nan, -np.inf
    idx, _ = check_route(l, bias, None, 5, groups, top, 1, score, renorm)
    assert not np.isin(idx, (1, 4)).any()
    # NaN and infinities under a dead expert are not seen
    active = np.ones(E, np.uint8)
    active[[0, 7]] = 0
    clean = np.random.default_rng(2).normal(size=(4, E)).astype(np.float32)
    dirty = clean.copy()
    dirty[:, 0], dirty[:, 7] = np.nan, np.inf
    a, b = (run_route(v, None, active, 5, groups, top, 2, score, renorm) for v in (clean, dirty))
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


# each rounding of the gradient's terms: exp of a rounded difference (|z| + 2
# places), a sum over E (at most 24 roundings deep) and quotients of each score,
# twice, and the sums over K: 8 (z + 2) + K + 100 of the terms' size
def check_route_grad(l, active, idx, dw, score, renorm, scale, shift=0):
    T, E = l.shape
    K = idx.shape[1]
    d = [put(dw, shift=shift), put(l, shift=shift), put(active, np.uint8, shift), put(idx, np.int32, shift)]
    out = Guarded(T * E, shift=shift)
    runtime.op("moe_route_grad", *(p(b) for b in d), p(out), T, E, K, score, renorm, scale, None)
    so.sync()
    got = out.host((T, E)).astype(np.float64)
    want, size = so.route_grad(dw, l, active, idx, score, renorm, scale)
    live = so.scores(l, active, score)[1]
    z = np.abs(np.where(live & np.isfinite(l), l, 0)).astype(np.float64)
    z = z.max(1, keepdims=True) * (2 if score == 0 else 1)
    off = np.abs(got - want)
    assert np.all(off <= (8 * (z + 2) + K + 100) * U * size + 1e-37), (off / (U * size + 1e-37)).max()
    assert np.all(got[~live] == 0)
    return got


@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 64, 2), (3, 60, 4), (257, 64, 2), (5, 128, 64), (33, 200, 3),
                                   (9, 256, 16), (6, 500, 5), (3, 1024, 8)])
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("renorm", [0, 1])
def test_route_grad(T, E, K, score, renorm):
    print(f"route_grad {T} {E} {K} {score} {renorm}", flush=True)
    rng = np.random.default_rng(T * 1000 + E)
    l = rng.normal(size=(T, E)).astype(np.float32) * 2
    active = (rng.random(E) < 0.8).astype(np.uint8)
    dw = rng.normal(size=(T, K)).astype(np.float32)
    check_route_grad(l, None, so.route(l, None, None, K, score=score)[0], dw, score, renorm, 1.0)
    idx = so.route(l, None, active, K, score=score)[0]
    dw[idx < 0] = np.nan  # not read
    check_route_grad(l, active, idx, dw, score, renorm, 2.5, shift=1)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("renorm", [0, 1])
def test_route_grad_of_any_choice(score, renorm):
    """The same expert twice, experts out of range, dead ones, masked rows."""
    rng = np.random.default_rng(9)
    T, E, K = 40, 20, 6
    l = rng.normal(size=(T, E)).astype(np.float32)
    l[3], l[4, ::2], l[5, 1:] = -np.inf, np.nan, -np.inf
    active = np.ones(E, np.uint8)
    active[7] = 0
    idx = rng.integers(-2, E + 3, size=(T, K)).astype(np.int32)
    idx[0] = 5
    dw = rng.normal(size=(T, K)).astype(np.float32)
    live = so.scores(l, active, score)[1]
    for t in range(T):
        for k, e in enumerate(idx[t]):
            if e < 0 or e >= E or not live[t, e]:
                dw[t, k] = np.nan
    got = check_route_grad(l, active, idx, dw, score, renorm, 1.5)
    assert np.all(got[3] == 0)


@pytest.mark.parametrize("E,K", [(24, 6), (200, 3), (300, 6), (1024, 20)])
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("at", [-600.0, -300.0, -110.0, -60.0, 12.0, 40.0])
def test_route_grad_far_from_zero(E, K, score, renorm, at):
    """Chosen scores that underflow in 32 bits (a bias or a group can choose
    experts far below the best) and sigmoids next to 1, element by element."""
    rng = np.random.default_rng(int(abs(at)) + E)
    T = 7
    l = (at + rng.normal(size=(T, E))).astype(np.float32)
    if score == 0 and at < 0:
        l[:, 0] = 1.0  # the best expert, which no token chose
    idx = np.stack([rng.permutation(np.arange(1, E))[:K] for _ in range(T)]).astype(np.int32)
    dw = rng.normal(size=(T, K)).astype(np.float32)
    out = Guarded(T * E)
    d = [put(dw), put(l), put(idx, np.int32)]
    runtime.op("moe_route_grad", p(d[0]), p(d[1]), None, p(d[2]), p(out), T, E, K, score, renorm, 1.5, None)
    so.sync()
    got = out.host((T, E)).astype(np.float64)
    x, u = np.take_along_axis(l, idx, 1).astype(np.float64), 1.5 * dw.astype(np.float64)
    left = 1 / (1 + np.exp(x)) if score else 1.0  # 1 - s
    want, size = np.zeros((T, E)), np.zeros((T, E))
    if renorm:
        s = np.exp(x - x.max(1, keepdims=True)) * left if score else np.exp(x - x.max(1, keepdims=True))
        w = s / s.sum(1, keepdims=True)
        g = w * (u - (w * u).sum(1, keepdims=True)) * left
        big = w * (np.abs(u) + (w * np.abs(u)).sum(1, keepdims=True)) * left
    elif score:
        g = np.exp(x) * left * left * u
        big = np.abs(g)
    else:
        want, size = so.route_grad(dw, l, None, idx, 0, 0, 1.5)
    if renorm or score:
        np.put_along_axis(want, idx, g, 1)
        np.put_along_axis(size, idx, big, 1)
    # a rounded difference of logits that are within 8 of each other (a whole logit
    # without renorm) in each exponential, twice, and the sums over K
    z = 8 if renorm else np.abs(l).max()
    off = (8 * (z + 2) + K + 100) * U * size + 1e-37
    assert np.all(np.abs(got - want) <= off), (np.abs(got - want) / off).max()


# ---- the experts' products ----------------------------------------------------------

def layer(T, K, D, H, E, seed, empty=0.0, skew=0.0):
    """Inputs of a layer; a share `empty` of the slots has no expert, and their
    weights are NaN; skew: the share of slots that expert 0 holds."""
    rng = np.random.default_rng(seed)
    idx = rng.integers(0, E, size=(T, K)).astype(np.int32)
    idx[rng.random((T, K)) < skew] = 0
    idx[rng.random((T, K)) < empty] = -1
    idx[(rng.random((T, K)) < 0.05) & (idx < 0)] = E + 3
    w = rng.normal(size=(T, K)).astype(np.float32)
    w[(idx < 0) | (idx >= E)] = np.nan
    f = lambda *s, scale=1.0: (rng.normal(size=s) * scale).astype(np.float32)  # noqa: E731
    return {"x": f(T, D), "idx": idx, "weight": w, "W1": f(E, D, H, scale=D ** -0.5), "W2": f(E, H, D, scale=H ** -0.5),
            "dy": f(T, D)}


def within(got, want, off, what):
    d = np.abs(got.astype(np.float64) - want)
    assert np.all(np.isfinite(got)), what
    assert np.all(d <= off + 1e-36), f"{what}: {(d / (off + 1e-36)).max():.3g} of the bound, {d.max():.3g}"
    # far below the bounds, whose terms all err the same way: roundings of a sum
    # of n terms that err at random are sqrt(n) U of it, and two sums follow each other
    n = np.linalg.norm(want)
    if n > 0:
        assert np.linalg.norm(d) <= 1e-5 * n, f"{what}: relative error {np.linalg.norm(d) / n:.3g}"


def run_experts(a, E, act, train, shift=0, grads=("dx", "dweight", "dW1", "dW2"), stream=None):
    T, D = a["x"].shape
    K, H = a["idx"].shape[1], a["W1"].shape[2]
    lib = runtime.lib()
    d = {k: put(v, np.int32 if k == "idx" else np.float32, shift) for k, v in a.items()}
    y = Guarded(T * D, shift=shift)
    state = room(lib.nsh_op_moe_experts_state(T, K, D, H, E)) if train else None
    ws = room(lib.nsh_op_moe_experts_workspace(T, K, D, H, E, int(train)))
    runtime.op("moe_experts", *(p(d[k]) for k in ("x", "idx", "weight", "W1", "W2")), p(y), T, K, D, H, E, act,
               p(state), p(ws), stream)
    so.sync(stream)
    out = {"y": y.host((T, D))}
    ws.host()
    if train:
        state.host()
        sizes = {"dx": (T, D), "dweight": (T, K), "dW1": (E, D, H), "dW2": (E, H, D)}
        g = {k: Guarded(int(np.prod(sizes[k])), shift=shift) if k in grads else None for k in sizes}
        runtime.op("moe_experts_grad", *(p(d[k]) for k in ("dy", "x", "weight", "W1", "W2")), p(state),
                   *(p(g[k]) for k in sizes), T, K, D, H, E, act, p(ws), stream)
        so.sync(stream)
        out.update({k: g[k].host(sizes[k]) for k in sizes if g[k]})
        ws.host()
        state.host()
    return out


# one token to several tiles of 128 rows, odd sizes (no float4), one expert, more
# experts than slots, K = 1, several experts a token, rows without an expert
EXPERTS = [(1, 1, 4, 4, 1, 0.0), (1, 2, 64, 96, 8, 0.0), (1, 2, 1024, 1024, 4, 0.0), (2, 1, 7, 5, 3, 0.3),
           (5, 3, 33, 17, 4, 0.2), (16, 2, 128, 256, 64, 0.0), (37, 2, 256, 192, 40, 0.1), (64, 6, 48, 64, 7, 0.0),
           (130, 1, 64, 256, 2, 0.0), (300, 4, 64, 256, 8, 0.1), (700, 2, 200, 333, 10, 0.0), (1025, 2, 96, 128, 3, 0.5)]


@pytest.mark.parametrize("T,K,D,H,E,empty", EXPERTS)
@pytest.mark.parametrize("shift", [0, 1])
def test_experts(T, K, D, H, E, empty, shift):
    print(f"experts {T} {K} {D} {H} {E} {shift}", flush=True)
    a = layer(T, K, D, H, E, T + D, empty)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 6)
    within(run_experts(a, E, 6, False, shift)["y"], want["y"], off["y"], "y")


@pytest.mark.parametrize("T,K,D,H,E,empty", EXPERTS)
@pytest.mark.parametrize("shift", [0, 1])
def test_experts_grad(T, K, D, H, E, empty, shift):
    print(f"experts_grad {T} {K} {D} {H} {E} {shift}", flush=True)
    a = layer(T, K, D, H, E, T + D, empty)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 6, a["dy"])
    got = run_experts(a, E, 6, True, shift)
    for k in want:
        within(got[k], want[k], off[k], k)
    bad = (a["idx"] < 0) | (a["idx"] >= E)
    assert np.all(got["dweight"][bad] == 0)
    assert np.all(got["y"][bad.all(1)] == 0) and np.all(got["dx"][bad.all(1)] == 0)
    for e in range(E):
        if not (a["idx"] == e).any():
            assert np.all(got["dW1"][e] == 0) and np.all(got["dW2"][e] == 0)


# sizes above 128 with many slots an expert: products of two fp16 pieces (the knob
# lets smaller layers take them).  Odd sizes, sizes around the tiles' 128 and 256, one
# expert, empty ones, slots without an expert
@pytest.fixture
def pieces(monkeypatch):
    monkeypatch.setenv("NSHIP_MOE_SPLIT_MIN", "16")


SPLIT = [(200, 2, 129, 130, 1, 0.0), (400, 1, 256, 132, 1, 0.0), (700, 2, 200, 333, 10, 0.1), (900, 2, 256, 256, 4, 0.0),
         (1000, 2, 264, 140, 5, 0.2), (333, 4, 131, 520, 3, 0.0), (1600, 1, 512, 136, 4, 0.0), (150, 3, 385, 129, 12, 0.0)]


@pytest.mark.parametrize("T,K,D,H,E,empty", SPLIT)
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("skew", [0.0, 0.7])
def test_experts_of_many_slots(T, K, D, H, E, empty, shift, skew, pieces):
    print(f"experts {T} {K} {D} {H} {E} {shift} {skew}", flush=True)
    a = layer(T, K, D, H, E, T + D, empty, skew)
    if E > 2:
        a["idx"][a["idx"] == E - 2] = 0  # an expert without slots
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 6, a["dy"])
    got = run_experts(a, E, 6, True, shift)
    for k in want:
        within(got[k], want[k], off[k], k)
    assert np.array_equal(run_experts(a, E, 6, False, shift)["y"], got["y"])
    bad = (a["idx"] < 0) | (a["idx"] >= E)
    assert np.all(got["dweight"][bad] == 0)
    if E > 2:
        assert np.all(got["dW1"][E - 2] == 0) and np.all(got["dW2"][E - 2] == 0)


def test_experts_of_a_large_layer():
    """Large enough for the pieces without the knob."""
    a = layer(3200, 2, 1024, 1024, 16, 21, 0.02)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 5, a["dy"])
    got = run_experts(a, 16, 5, True)
    for k in want:
        within(got[k], want[k], off[k], k)


@pytest.mark.parametrize("act", [0, 2, 3, 4, 5])
def test_experts_of_many_slots_activations(act, pieces):
    print(f"activation {act}", flush=True)
    a = layer(450, 2, 132, 144, 2, act)
    if act == 2:
        a["W1"] = np.where(np.arange(144) % 2, 1, -1).astype(np.float32) * (np.abs(a["W1"]) + 0.1)
        a["x"] = np.abs(a["x"]) + 0.1
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], act, a["dy"])
    got = run_experts(a, 2, act, True)
    for k in want:
        within(got[k], want[k], off[k], k)


@pytest.mark.parametrize("sx,sw,sd", [(1e-18, 1.0, 1.0), (1e12, 1e-9, 1e-15), (1e3, 1e-3, 1e-25), (1.0, 1e8, 1e10)])
def test_experts_of_many_slots_of_any_scale(sx, sw, sd, pieces):
    """x and dy, the matrices, the slots' weights over many powers of two, other
    ones for every token, expert and column: every operand row is scaled by its own."""
    rng = np.random.default_rng(11)
    a = layer(500, 2, 136, 160, 2, 12)
    p2 = lambda *s: 2.0 ** rng.integers(-6, 7, s)  # noqa: E731
    a["x"] = (a["x"] * sx * p2(500, 1)).astype(np.float32)
    a["dy"] = (a["dy"] * sd * p2(500, 1)).astype(np.float32)
    a["weight"] = (a["weight"] * p2(500, 2)).astype(np.float32)
    a["W1"] = (a["W1"] * sw * p2(2, 1, 160)).astype(np.float32)
    a["W2"] = (a["W2"] * sw * p2(2, 160, 1)).astype(np.float32)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 0, a["dy"])
    got = run_experts(a, 2, 0, True)
    for k in want:
        d = np.abs(got[k].astype(np.float64) - want[k])
        assert np.all(d <= off[k] + 1e-36), k


def test_experts_of_many_slots_with_an_outlier_column(pieces):
    """One column of x 2^12 times the others: their products keep their accuracy."""
    a = layer(500, 2, 136, 160, 2, 13)
    a["x"][:, 7] *= 4096
    a["W1"][:, 7, ::2] = 0  # half of the hidden units do not see it
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 0, a["dy"])
    got = run_experts(a, 2, 0, True)
    for k in want:
        d = np.abs(got[k].astype(np.float64) - want[k])
        assert np.all(d <= off[k] + 1e-36), k


@pytest.mark.parametrize("T", [500, 700])
def test_experts_of_many_slots_keep_infinities_apart(T, pieces):
    a = layer(T, 2, 136, 160, 3, 14)
    a["idx"] %= 2
    a["W1"][2], a["W2"][2] = np.nan, np.inf  # no slot asks for it
    clean = run_experts(a, 3, 6, True)
    assert all(np.isfinite(clean[k]).all() for k in clean)
    only = np.nonzero((a["idx"] == 0).all(1))[0][0]  # a token of expert 0 alone
    a["x"][only, 5], a["dy"][only, 9] = np.inf, np.nan
    got = run_experts(a, 3, 6, True)
    rest = np.arange(T) != only
    assert not np.isfinite(got["y"][only]).any()
    want, off = so.experts(a["x"][rest], a["idx"][rest], a["weight"][rest], a["W1"], a["W2"], 6)
    within(got["y"][rest], want["y"], off["y"], "the other tokens")
    assert np.array_equal(got["y"][rest], clean["y"][rest])
    assert np.array_equal(got["dW1"][1:], clean["dW1"][1:]) and np.array_equal(got["dW2"][1:], clean["dW2"][1:])


@pytest.mark.parametrize("act", [0, 2, 3, 4, 5])
@pytest.mark.parametrize("T", [3, 200])
def test_experts_activations(act, T):
    """(ReLU's and leaky ReLU's derivative jumps at 0: leaky's inputs are kept off it.)"""
    print(f"activation {act} {T}", flush=True)
    a = layer(T, 2, 64, 80, 5, act)
    if act == 2:
        a["W1"] = np.where(np.arange(80) % 2, 1, -1).astype(np.float32) * (np.abs(a["W1"]) + 0.1)
        a["x"] = np.abs(a["x"]) + 0.1
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], act, a["dy"])
    got = run_experts(a, 5, act, True)
    for k in want:
        within(got[k], want[k], off[k], k)
    within(run_experts(a, 5, act, False)["y"], want["y"], off["y"], "y")


def test_experts_relu():
    a = layer(200, 2, 64, 80, 5, 1)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 1)
    within(run_experts(a, 5, 1, False)["y"], want["y"], off["y"], "y")


def test_experts_one_expert_holds_most_slots():
    a = layer(900, 2, 64, 128, 16, 4, skew=0.8)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 6, a["dy"])
    got = run_experts(a, 16, 6, True)
    for k in want:
        within(got[k], want[k], off[k], k)


@pytest.mark.parametrize("T", [4, 150])
def test_experts_no_slot_has_an_expert(T):
    a = layer(T, 2, 64, 32, 4, 1)
    a["idx"][:] = -1
    a["weight"][:] = np.nan
    got = run_experts(a, 4, 6, True)
    assert all(np.all(v == 0) for v in got.values())
    assert np.all(run_experts(a, 4, 6, False)["y"] == 0)


def test_experts_single_gradients():
    """Any of the gradients may be left out; the others keep their bits."""
    a = layer(150, 2, 64, 96, 6, 2, 0.1)
    every = run_experts(a, 6, 6, True)
    for only in (("dx",), ("dweight",), ("dW1",), ("dW2",), ("dx", "dW2"), ()):
        for k, v in run_experts(a, 6, 6, True, grads=only).items():
            assert np.array_equal(v, every[k]), (only, k)


@pytest.mark.parametrize("T,K", [(3, 2), (40, 2), (600, 4)])
def test_experts_equal_calls_give_equal_bits(T, K):
    a = layer(T, K, 64, 256, 8, 3)
    one, two = (run_experts(a, 8, 5, True) for _ in range(2))
    assert all(np.array_equal(one[k], two[k]) for k in one)


@pytest.mark.parametrize("T", [2, 100])
def test_experts_infinities_stay_with_their_token(T):
    """NaN and infinities in one token, or in an expert that no slot asks for."""
    a = layer(T, 2, 64, 32, 4, 6)
    a["idx"] %= 3
    clean = run_experts(a, 4, 6, False)["y"]
    a["W1"][3], a["W2"][3] = np.nan, np.inf
    assert np.array_equal(run_experts(a, 4, 6, False)["y"], clean)
    a["x"][1, 5] = np.inf
    got = run_experts(a, 4, 6, False)["y"]
    assert not np.isfinite(got[1]).any()
    rest = np.arange(T) != 1
    want, off = so.experts(a["x"][rest], a["idx"][rest], a["weight"][rest], a["W1"], a["W2"], 6)
    within(got[rest], want["y"], off["y"], "the other tokens")


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12])
def test_experts_of_very_small_and_large_values(scale):
    """x and the weights of the slots: the products keep their relative accuracy."""
    a = layer(150, 2, 64, 32, 4, 6)
    a["x"] = (a["x"] * scale).astype(np.float32)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 0)
    got = run_experts(a, 4, 0, False)["y"].astype(np.float64)
    assert np.all(np.abs(got - want["y"]) <= off["y"])


@pytest.mark.parametrize("T,D,H", [(3, 64, 96), (3, 33, 17), (400, 132, 260), (401, 131, 129)])
def test_experts_single_gradients_without_a_sort_and_in_pieces(T, D, H, pieces):
    """The other two ways through a layer; the knob sends the many slots to the pieces."""
    a = layer(T, 2, D, H, 6, 2, 0.1)
    every = run_experts(a, 6, 6, True)
    again = run_experts(a, 6, 6, True)
    assert all(np.array_equal(every[k], again[k]) for k in every)
    for only in (("dx",), ("dweight",), ("dW1",), ("dW2",), ("dx", "dW2"), ("dweight", "dW1"), ()):
        for k, v in run_experts(a, 6, 6, True, grads=only).items():
            assert np.array_equal(v, every[k]), (only, k)


@pytest.mark.parametrize("T", [3, 150, 700])
def test_experts_a_token_may_ask_one_expert_twice(T, pieces):
    a = layer(T, 4, 132, 140, 5, 9)
    a["idx"][:, 1] = a["idx"][:, 0]
    a["idx"][::3] = a["idx"][::3, :1]
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 5, a["dy"])
    got = run_experts(a, 5, 5, True)
    for k in want:
        within(got[k], want[k], off[k], k)


# both products in one workgroup: sizes around its 32 rows, 8 columns a step, 32
# columns a block and every division of the second product among eight waves
SMALL = [(60, 2, 4, 4, 2, 0.0), (33, 1, 8, 12, 1, 0.0), (97, 2, 12, 20, 3, 0.1), (64, 1, 36, 28, 2, 0.0),
         (150, 3, 64, 36, 5, 0.2), (128, 2, 68, 100, 4, 0.0), (90, 2, 100, 256, 3, 0.0), (129, 1, 132, 128, 1, 0.0),
         (200, 2, 160, 260, 7, 0.0), (77, 4, 224, 64, 9, 0.3), (161, 1, 256, 512, 4, 0.0), (1024, 2, 256, 132, 3, 0.0)]


@pytest.mark.parametrize("T,K,D,H,E,empty", SMALL)
@pytest.mark.parametrize("act", [1, 5])
def test_experts_of_a_small_layer(T, K, D, H, E, empty, act):
    print(f"experts {T} {K} {D} {H} {E} {act}", flush=True)
    a = layer(T, K, D, H, E, T + D + H, empty, 0.3)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], act, a["dy"])
    got = run_experts(a, E, act, True)
    for k in want:
        within(got[k], want[k], off[k], k)
    assert np.array_equal(run_experts(a, E, act, False)["y"], got["y"])
    bad = (a["idx"] < 0) | (a["idx"] >= E)
    assert np.all(got["dweight"][bad] == 0)
    for only in (("dx",), ("dweight",), ("dW2",)):
        assert np.array_equal(run_experts(a, E, act, True, grads=only)[only[0]], got[only[0]])


def test_experts_of_a_small_layer_keep_infinities_apart():
    a = layer(70, 2, 64, 96, 4, 8)
    a["idx"] %= 3
    a["W1"][3], a["W2"][3] = np.nan, np.inf
    a["x"][5, 3] = np.inf
    a["W2"][a["idx"][5, 0], 2, 3] = np.inf
    got = run_experts(a, 4, 5, True)
    plain = dict(a, x=a["x"].copy())
    plain["x"][5] = 0
    clean = (a["idx"] != a["idx"][5, 0]).all(1) & (np.arange(70) != 5)
    want, off = so.experts(plain["x"][clean], a["idx"][clean], a["weight"][clean], a["W1"][:3], a["W2"][:3], 5,
                           a["dy"][clean])
    for k in ("y", "dx", "dweight"):
        within(got[k][clean], want[k], off[k], k)
    assert not np.isfinite(got["y"][5]).all()


# sorted slots of layers that are neither small nor of many slots: wide ones with one
# side up to 128 (tiles of 128 columns) or above, and a small layer of many slots
SORTED = [(300, 2, 260, 512, 4, 0.0), (500, 2, 512, 264, 16, 0.1), (300, 2, 640, 128, 8, 0.1), (260, 1, 128, 516, 3, 0.0),
          (8300, 2, 128, 256, 8, 0.0)]


@pytest.mark.parametrize("T,K,D,H,E,empty", SORTED)
@pytest.mark.parametrize("act", [2, 6])
def test_experts_of_a_wide_layer(T, K, D, H, E, empty, act):
    print(f"experts {T} {K} {D} {H} {E} {act}", flush=True)
    a = layer(T, K, D, H, E, T + D + H, empty, 0.2)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], act, a["dy"])
    got = run_experts(a, E, act, True)
    for k in want:
        within(got[k], want[k], off[k], k)
    assert np.array_equal(run_experts(a, E, act, False)["y"], got["y"])
    for only in (("dx",), ("dweight",), ("dW1",)):
        assert np.array_equal(run_experts(a, E, act, True, grads=only)[only[0]], got[only[0]])
