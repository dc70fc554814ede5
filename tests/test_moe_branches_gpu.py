"""Ways through the experts' products that sizes of their own take: slots of many
sort blocks and experts, contractions above 1024, several passes over a list,
offsets beyond 32 bits; against the 64-bit formulas (sparse_oracle.py)."""
import ctypes
import threading

import numpy as np
import pytest

import sparse_oracle as so
from neuralscript_amd import runtime
from sparse_oracle import U, p, put
from test_moe_topk_gpu import layer, run_experts, within
from test_newton_schulz_gpu import Layer
from test_sparse_large_gpu import Plain, room_for

pytestmark = pytest.mark.gpu


@pytest.fixture
def pieces():
    """Two fp16 pieces from 16 slots an expert on."""
    runtime.lib().nsh_test_moe_split_least(ctypes.c_int64(16))
    yield
    runtime.lib().nsh_test_moe_split_least(ctypes.c_int64(0))


def check(a, act, shift=0):
    E = a["W1"].shape[0]
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], act, a["dy"])
    got = run_experts(a, E, act, True, shift)
    for k in want:
        within(got[k], want[k], off[k], k)
    bad = (a["idx"] < 0) | (a["idx"] >= E)
    assert np.all(got["dweight"][bad] == 0)
    for e in range(E):
        if not (a["idx"] == e).any():
            assert np.all(got["dW1"][e] == 0) and np.all(got["dW2"][e] == 0)
    assert np.array_equal(run_experts(a, E, act, False, shift)["y"], got["y"])


# more blocks of 1024 slots than the sort has parts for an expert (16 parts of 64
# experts, one of 513 and more), experts in every bit of their index, some empty;
# both products in one kernel (widths of 4) and on grouped products
@pytest.mark.parametrize("T,K,E,skew", [(35001, 2, 64, 0.0), (17500, 4, 33, 0.6), (10000, 2, 1000, 0.1),
                                        (2600, 5, 1024, 0.5), (20001, 1, 513, 0.0), (66000, 1, 2, 0.3)])
@pytest.mark.parametrize("D,H", [(4, 8), (5, 3)])
def test_experts_of_many_sort_blocks(T, K, E, skew, D, H):
    print(f"experts {T} {K} {D} {H} {E} {skew}", flush=True)
    a = layer(T, K, D, H, E, T + E, 0.1, skew)
    a["idx"][a["idx"] % 7 == 3] = E - 1
    check(a, 5)


@pytest.mark.parametrize("E", [300, 1024])
def test_experts_of_many_sort_blocks_on_pieces(E, pieces):
    print(f"experts on pieces, {E}", flush=True)
    a = layer(9 * E, 2, 132, 129, E, E, 0.05, 0.05)
    a["idx"][(a["idx"] % 5 == 2) & (a["idx"] < E)] = 0  # (slots without an expert, whose weights are NaN, stay so)
    check(a, 6)


# contractions longer than what a lane of the layout passes holds (1024), either way
@pytest.mark.parametrize("T,K,D,H,E", [(200, 2, 1100, 260, 2), (200, 2, 260, 1100, 2), (90, 2, 1029, 1031, 2),
                                       (60, 2, 132, 2049, 1)])
@pytest.mark.parametrize("shift", [0, 1])
def test_experts_of_wide_layers_on_pieces(T, K, D, H, E, shift, pieces):
    print(f"experts on pieces {T} {K} {D} {H} {E} {shift}", flush=True)
    check(layer(T, K, D, H, E, D, 0.05), 6, shift)


# features of x, hidden units by either matrix, far smaller than the others
@pytest.mark.parametrize("scale", [1e-4, 1e-6])
@pytest.mark.parametrize("small", ["features", "units by W1", "units by W2", "tokens"])
@pytest.mark.parametrize("act", [0, 6])
def test_small_rows_of_the_weights_gradients_keep_their_own_accuracy(scale, small, act, pieces):
    """Rows and columns of dW1 and dW2 by themselves, within what within() allows a
    whole gradient: one scale serves all positions of an expert there."""
    a = layer(500, 2, 136, 160, 2, 12)
    if small == "features":
        a["x"][:, ::3] *= np.float32(scale)
    elif small == "units by W1":
        a["W1"][:, :, ::3] *= np.float32(scale)
    elif small == "units by W2":
        a["W2"][:, ::3] *= np.float32(scale)
    else:
        a["x"][::3] *= np.float32(scale)
        a["dy"][::3] *= np.float32(scale)
    want, _ = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], act, a["dy"])
    got = run_experts(a, 2, act, True)
    for k in ("dW1", "dW2"):
        for axis in (1, 2):
            err = np.linalg.norm(got[k] - want[k], axis=axis) / np.linalg.norm(want[k], axis=axis)
            print(f"  {k} along {axis}: {err.max():.3g}", flush=True)
            assert np.all(err <= 1e-5), (k, axis)


# without a sort: contractions of several stages (512 forward, 1024 backward), by
# slots and by experts, more than 8 rows an expert, up to 1024 slots
@pytest.mark.parametrize("T,K,D,H,E,skew", [(3, 2, 1030, 2100, 8, 0.0), (8, 2, 1028, 2052, 8, 0.0), (8, 2, 2051, 1025, 4, 0.5),
                                            (150, 2, 36, 1040, 60, 0.95), (1024, 1, 24, 20, 200, 0.7),
                                            (64, 6, 1033, 36, 64, 0.5)])
@pytest.mark.parametrize("shift", [0, 1])
def test_experts_of_wide_layers_without_a_sort(T, K, D, H, E, skew, shift):
    print(f"experts without a sort {T} {K} {D} {H} {E} {skew} {shift}", flush=True)
    check(layer(T, K, D, H, E, D, 0.05, skew), 5, shift)


def test_experts_that_all_tokens_agree_on_without_a_sort():
    """192 tokens, two of 64 experts: 24 passes of 8 rows."""
    a = layer(192, 2, 136, 72, 64, 5)
    a["idx"][:] = [41, 7]
    check(a, 6)


def repeated(rows, times, dtype=np.float32):
    """`rows` as often on the device."""
    rows = np.ascontiguousarray(rows, dtype)
    d = Plain(rows.nbytes * times)
    so.hip("hipMemcpy", ctypes.c_void_p(d.ptr), rows.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(rows.nbytes), 1)
    have = 1
    while have < times:
        n = min(have, times - have)
        so.hip("hipMemcpy", ctypes.c_void_p(d.ptr + have * rows.nbytes), ctypes.c_void_p(d.ptr),
               ctypes.c_size_t(n * rows.nbytes), 3)
        have += n
    return d


def window(d, first, shape, dtype=np.float32):
    out = np.empty(shape, dtype)
    row = out.nbytes // shape[0]
    so.hip("hipMemcpy", out.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(d.ptr + first * row),
           ctypes.c_size_t(out.nbytes), 2)
    return out


# slots times H above 2^31: one kernel for both products, grouped products, pieces
@pytest.mark.parametrize("T,D,H,E", [(1 << 23, 4, 260, 3), (1 << 22, 128, 516, 3), (1 << 22, 132, 520, 3)])
def test_experts_beyond_32_bits(T, D, H, E):
    """2048 tokens over and over: each of them comes out as it does alone, and the
    weights' gradients as often as large."""
    print(f"experts {T} {D} {H} {E}", flush=True)
    lib, P = runtime.lib(), 2048
    sizes = (T, 1, D, H, E)
    assert T * H > 1 << 31
    state, ws = lib.nsh_op_moe_experts_state(*sizes), lib.nsh_op_moe_experts_workspace(*sizes, 1)
    room_for(state + ws + 16 * T * (D + 1) + (1 << 30))
    a = layer(P, 1, D, H, E, D)
    want, off = so.experts(a["x"], a["idx"], a["weight"], a["W1"], a["W2"], 6, a["dy"])
    d = {k: repeated(a[k], T // P, np.int32 if k == "idx" else np.float32) for k in ("x", "idx", "weight", "dy")}
    w = {k: put(a[k]) for k in ("W1", "W2")}
    out = {"y": Plain(4 * T * D, 0x7B), "dx": Plain(4 * T * D, 0x7B), "dweight": Plain(4 * T, 0x7B)}
    dw = {"dW1": put(np.zeros((E, D, H))), "dW2": put(np.zeros((E, H, D)))}
    st, room = Plain(state, 0xFF), Plain(ws, 0xFF)
    runtime.op("moe_experts", *(d[k].ptr for k in ("x", "idx", "weight")), p(w["W1"]), p(w["W2"]), out["y"].ptr, *sizes, 6,
               st.ptr, room.ptr, None)
    runtime.op("moe_experts_grad", *(d[k].ptr for k in ("dy", "x", "weight")), p(w["W1"]), p(w["W2"]), st.ptr,
               out["dx"].ptr, out["dweight"].ptr, p(dw["dW1"]), p(dw["dW2"]), *sizes, 6, room.ptr, None)
    so.sync()
    for first in (0, T // 2, T - P):
        for k, b in out.items():
            within(window(b, first, want[k].shape), want[k], off[k], f"{k} from {first}")
    for k, b in dw.items():  # (sums of T / E terms that err at random)
        total = want[k] * (T // P)
        err = np.linalg.norm(b.host(want[k].shape) - total) / np.linalg.norm(total)
        print(f"  {k}: {err:.3g}", flush=True)
        assert err <= np.sqrt(T / E) * U
    for b in (*d.values(), *out.values(), st, room):
        b.free()


def test_two_host_threads_at_once(pieces):
    """Training steps of layers that go other ways, each from a thread of its own on
    a stream of its own: the bits of the same steps after each other."""
    sizes = [(96, 2, 64, 96, 5), (12, 3, 36, 20, 4), (200, 2, 136, 260, 5)]

    def steps(a, stream):
        for _ in range(20):
            a.step(stream)
        so.sync(stream)

    streams = [so.new_stream() for _ in sizes]
    alone = [Layer(*s, i) for i, s in enumerate(sizes)]
    for a, t in zip(alone, streams):
        steps(a, t)
    both = [Layer(*s, i) for i, s in enumerate(sizes)]
    threads = [threading.Thread(target=steps, args=x) for x in zip(both, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, both):
        x, y = a.read(), b.read()
        assert all(np.array_equal(x[k], y[k]) for k in a.OUT)
