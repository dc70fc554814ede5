"""Plain 64-bit forms of the operators with K experts a token and of the
Newton-Schulz orthogonalisation (include/nship.h), and the device plumbing
that their tests share: buffers with guarded ends, streams and graphs."""
import ctypes
import math

import numpy as np

from neuralscript_amd import runtime
from neuralscript_amd.runtime import DeviceArray as DA

U = 2.0 ** -24  # half a step of fp32, relative
NS = (3.4445, -4.7750, 2.0315)


# ---- formulas -----------------------------------------------------------------

def scores(logits, active, score):
    """s [T, E] and which experts are live, in 64 bits."""
    l = np.asarray(logits, np.float64)
    live = ~np.isnan(l) & (l != -np.inf)
    if active is not None:
        live &= np.asarray(active)[None, :] != 0
    s = np.zeros_like(l)
    for t in range(l.shape[0]):
        v = l[t][live[t]]
        if v.size == 0:
            continue
        if score == 0:
            m = v.max()
            with np.errstate(invalid="ignore"):
                e = np.where(v == m, 1.0, np.exp(v - m))
            s[t][live[t]] = e / e.sum()
        else:
            with np.errstate(over="ignore"):
                s[t][live[t]] = 1.0 / (1.0 + np.exp(-v))
    return s, live


def route(logits, bias, active, K, groups=1, top_groups=1, group_best=1, score=0, renorm=0, scale=1.0):
    T, E = logits.shape
    s, live = scores(logits, active, score)
    idx, weight = np.full((T, K), -1, np.int32), np.zeros((T, K))
    for t in range(T):
        c = s[t] + (0.0 if bias is None else np.asarray(bias, np.float64))
        left = [e for e in range(E) if live[t, e] and not np.isnan(c[e]) and c[e] != -np.inf]
        if top_groups < groups:
            per = E // groups
            value = {}
            for g in range(groups):
                best = sorted((c[e] for e in left if e // per == g), reverse=True)[:group_best]
                if best:
                    value[g] = sum(best)
            keep = sorted(value, key=lambda g: (-value[g], g))[:top_groups]
            left = [e for e in left if e // per in keep]
        left = sorted(left, key=lambda e: (-c[e], e))[:K]
        total = sum(s[t, e] for e in left) if renorm else 1.0
        for k, e in enumerate(left):
            idx[t, k] = e
            weight[t, k] = scale * s[t, e] / total if total > 0 else 0.0
    return idx, weight


def weights_of(logits, active, idx, score, renorm, scale):
    """The routing's weights for a given choice (what the gradient differentiates)."""
    s, live = scores(logits, active, score)
    T, K = idx.shape
    w = np.zeros((T, K))
    for t in range(T):
        ok = [(k, e) for k, e in enumerate(idx[t]) if 0 <= e < s.shape[1] and live[t, e]]
        total = sum(s[t, e] for _, e in ok) if renorm else 1.0
        for k, e in ok:
            w[t, k] = scale * s[t, e] / total if total > 0 else 0.0
    return w


def route_grad(dweight, logits, active, idx, score, renorm, scale):
    """dlogits, and for each the size of what it is summed from."""
    s, live = scores(logits, active, score)
    T, E = s.shape
    dl, size = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        ok = [(k, e) for k, e in enumerate(idx[t]) if 0 <= e < E and live[t, e]]
        total = sum(s[t, e] for _, e in ok)
        if renorm and not total > 0:
            continue
        u = {k: scale * float(dweight[t, k]) for k, _ in ok}
        big = {k: abs(v) for k, v in u.items()}
        if renorm:
            dot, adot = sum(u[k] * s[t, e] for k, e in ok), sum(big[k] * s[t, e] for k, e in ok)
            u = {k: (v - dot / total) / total for k, v in u.items()}
            big = {k: (v + adot / total) / total for k, v in big.items()}
        ds, ads = np.zeros(E), np.zeros(E)
        for k, e in ok:
            ds[e] += u[k]
            ads[e] += big[k]
        if score == 0:
            dl[t] = s[t] * (ds - (s[t] * ds).sum())
            size[t] = s[t] * (ads + (s[t] * ads).sum())
        else:
            dl[t] = s[t] * (1 - s[t]) * ds
            size[t] = s[t] * ads
        dl[t][~live[t]] = 0.0
    return dl, size


_erf = np.vectorize(math.erf, otypes=[np.float64])


def act(u, code):
    with np.errstate(over="ignore"):
        sig = 1.0 / (1.0 + np.exp(-u))
    return {0: lambda: u, 1: lambda: np.maximum(u, 0.0), 2: lambda: np.where(u > 0, u, np.float64(np.float32(0.01)) * u),
            3: lambda: sig, 4: lambda: np.tanh(u), 5: lambda: u * sig,
            6: lambda: 0.5 * u * (1 + _erf(u / np.float64(np.float32(1.41421356))))}[code]()


def act_grad(u, code):
    with np.errstate(over="ignore"):
        sig = 1.0 / (1.0 + np.exp(-u))
    r2 = np.float64(np.float32(1.41421356))
    return {0: lambda: np.ones_like(u), 1: lambda: (u > 0) * 1.0, 2: lambda: np.where(u > 0, 1.0, np.float64(np.float32(0.01))),
            3: lambda: sig * (1 - sig), 4: lambda: 1 - np.tanh(u) ** 2, 5: lambda: sig + u * sig * (1 - sig),
            6: lambda: 0.5 * (1 + _erf(u / r2)) + u * np.exp(-(u / r2) ** 2) / np.float64(np.float32(2.50662827))}[code]()


def experts(x, idx, weight, W1, W2, code, dy=None):
    """y (and dx, dweight, dW1, dW2), each with a bound on what fp32 products
    and sums in any order may be off: every product of K terms within (K + 8) U
    of the sum of its terms' sizes (its roundings, and the two last places that
    a product of pieces may lose), an activation within 16 U of its argument's
    and its value's size, errors of factors carried along."""
    x, W1, W2 = (np.asarray(a, np.float64) for a in (x, W1, W2))
    T, K = idx.shape
    D, (E, _, H) = x.shape[1], W1.shape
    g = lambda n: (n + 8) * U  # noqa: E731
    out = {"y": np.zeros((T, D))}
    off = {"y": np.zeros((T, D))}
    if dy is not None:
        dy = np.asarray(dy, np.float64)
        for n, shape in (("dx", (T, D)), ("dweight", (T, K)), ("dW1", W1.shape), ("dW2", W2.shape)):
            out[n], off[n] = np.zeros(shape), np.zeros(shape)
    for e in range(E):
        t, k = np.nonzero(idx == e)
        if t.size == 0:
            continue
        xe, w = x[t], np.asarray(weight, np.float64)[t, k][:, None]
        u, eu = xe @ W1[e], g(D) * (np.abs(xe) @ np.abs(W1[e]))
        h = act(u, code)
        eh = 1.13 * eu + 16 * U * (np.abs(h) + np.abs(u))
        np.add.at(out["y"], t, w * (h @ W2[e]))
        np.add.at(off["y"], t, np.abs(w) * (g(H + K) * (np.abs(h) @ np.abs(W2[e])) + eh @ np.abs(W2[e])))
        if dy is None:
            continue
        de = dy[t]
        dh, edh = de @ W2[e].T, g(D) * (np.abs(de) @ np.abs(W2[e]).T)
        out["dweight"][t, k] = (h * dh).sum(1)
        off["dweight"][t, k] = (g(H) * np.abs(h * dh) + eh * np.abs(dh) + np.abs(h) * edh).sum(1)
        a = act_grad(u, code)
        ea = 1.0 * eu + 32 * U * (1 + np.abs(u))
        du = w * dh * a
        edu = np.abs(w) * (edh * np.abs(a) + np.abs(dh) * ea) + 4 * U * np.abs(du)
        np.add.at(out["dx"], t, du @ W1[e].T)
        np.add.at(off["dx"], t, g(H + K) * (np.abs(du) @ np.abs(W1[e]).T) + edu @ np.abs(W1[e]).T)
        n = len(t)
        out["dW1"][e], off["dW1"][e] = xe.T @ du, g(n) * (np.abs(xe).T @ np.abs(du)) + np.abs(xe).T @ edu
        wh = w * h
        out["dW2"][e] = wh.T @ de
        off["dW2"][e] = g(n) * (np.abs(wh).T @ np.abs(de)) + (np.abs(w) * eh + 2 * U * np.abs(wh)).T @ np.abs(de)
    return out, off


def newton_schulz(g, steps=5, dtype=np.float64):
    """[r, c] -> its orthogonalisation, computed in `dtype`."""
    a, b, c = (dtype(v) for v in NS)
    g = np.asarray(g, dtype)
    x = (g.astype(np.float64) / (np.sqrt((g.astype(np.float64) ** 2).sum()) + 1e-7)).astype(dtype)
    if x.shape[0] > x.shape[1]:
        x = x.T.copy()
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.T.copy() if g.shape[0] > g.shape[1] else x


# ---- device -----------------------------------------------------------------------

class Guarded:
    """A device buffer of n values whose surroundings must stay as they are;
    `shift` values past the 16-byte boundary."""
    PAD = 64

    def __init__(self, n, dtype=np.float32, shift=0, fill=0x7B, host=None):
        self.n, self.dtype, self.at = int(n), np.dtype(dtype), self.PAD + shift
        raw = np.full((self.n + 2 * self.PAD + shift) * self.dtype.itemsize, fill, np.uint8)
        self.before = raw.copy()
        if host is not None:
            raw.view(self.dtype)[self.at:self.at + self.n] = np.ascontiguousarray(host, self.dtype).ravel()
        self.d = DA.from_host(raw, np.uint8)

    @property
    def ptr(self):
        return self.d.ptr + self.at * self.dtype.itemsize

    def host(self, shape=None):
        raw = self.d.to_host()
        a, b = self.at * self.dtype.itemsize, (self.at + self.n) * self.dtype.itemsize
        assert np.array_equal(raw[:a], self.before[:a]), "written before the buffer"
        assert np.array_equal(raw[b:], self.before[b:]), "written behind the buffer"
        v = raw[a:b].view(self.dtype).copy()
        return v if shape is None else v.reshape(shape)


def put(a, dtype=np.float32, shift=0):
    return None if a is None else Guarded(np.asarray(a).size, dtype, shift, host=a)


def room(nbytes):
    """A workspace of exactly nbytes, filled with NaN patterns."""
    return Guarded(nbytes, np.uint8, fill=0xFF)


def p(b):
    return None if b is None else b.ptr


def hip(name, *args):
    rc = getattr(runtime.lib(), name)(*args)
    assert rc == 0, f"{name}: {rc}"


def new_stream():
    s = ctypes.c_void_p()
    hip("hipStreamCreateWithFlags", ctypes.byref(s), 1)  # not ordered after the null stream
    return s


def sync(stream=None):
    hip("hipStreamSynchronize", stream)


def capture(stream, calls):
    """calls() recorded into a graph on `stream`; returns the executable graph."""
    g, x = ctypes.c_void_p(), ctypes.c_void_p()
    hip("hipStreamBeginCapture", stream, 0)
    try:
        calls()
    finally:
        hip("hipStreamEndCapture", stream, ctypes.byref(g))
    hip("hipGraphInstantiate", ctypes.byref(x), g, None, None, ctypes.c_size_t(0))
    return x


def replay(x, stream):
    hip("hipGraphLaunch", x, stream)
