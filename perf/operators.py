"""The sparse layer's operators as measurable cases: routing of tokens to
experts, the experts' products, and the Newton-Schulz orthogonalisation that
updates their matrices, each forward and backward where it has both.

`run` computes a case with torch's elementary operations (`own` false) or with
the framework's entry points (`own` true); both get the tensors of `prepare`.

  kind        sizes                     what one pass is
  route       T, E, K (groups)          nsh_op_moe_route: experts and weights of T tokens
  route_grad  T, E, K                   nsh_op_moe_route_grad: the logits' gradient
  experts     T, K, D, H, E             nsh_op_moe_experts: the layer's output (serving)
  train       T, K, D, H, E             the same with its state kept, then nsh_op_moe_experts_grad
  ns          n, r, c                   nsh_op_newton_schulz of n matrices
  muon        n, r, c                   nsh_op_muon_ns_step with momentum: weights and momentum updated
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
F32, F64 = torch.float32, torch.float64


def listed():
    return [
        # a decoding step of one token: latency alone
        {"name": "route_one", "kind": "route", "T": 1, "E": 64, "K": 2, "score": 0, "renorm": 1, "groups": 1, "top": 1,
         "best": 1, "bias": 0, "scale": 1.0},
        # a long prompt over many experts, balanced by a bias, the best half of the groups
        {"name": "route_groups", "kind": "route", "T": 16384, "E": 256, "K": 8, "score": 1, "renorm": 1, "groups": 8,
         "top": 4, "best": 2, "bias": 1, "scale": 2.5},
        # the gradient of a ragged batch over a number of experts that is no power of two
        {"name": "route_grad_ragged", "kind": "route_grad", "T": 4099, "E": 60, "K": 4, "score": 1, "renorm": 1,
         "scale": 1.0},
        # the gradient at the benchmark's MoE batch
        {"name": "route_grad_large", "kind": "route_grad", "T": 65536, "E": 64, "K": 2, "score": 0, "renorm": 0,
         "scale": 1.0},
        # one token through two of 64 experts: the weights' bytes and latency
        {"name": "experts_one", "kind": "experts", "T": 1, "K": 2, "D": 1024, "H": 1024, "E": 64, "act": 6},
        # a handful of tokens that reach most experts
        {"name": "experts_few", "kind": "experts", "T": 37, "K": 2, "D": 1024, "H": 1024, "E": 64, "act": 6},
        # the benchmark's MoE batch, two experts a token
        {"name": "experts_large", "kind": "experts", "T": 65536, "K": 2, "D": 1024, "H": 1024, "E": 64, "act": 6},
        # training a small layer on a ragged batch
        {"name": "train_ragged", "kind": "train", "T": 1501, "K": 4, "D": 64, "H": 256, "E": 8, "act": 5},
        # training the benchmark's layer on 16384 tokens
        {"name": "train_large", "kind": "train", "T": 16384, "K": 2, "D": 1024, "H": 1024, "E": 64, "act": 6},
        # the small layer's expert matrices
        {"name": "ns_small", "kind": "ns", "n": 8, "r": 64, "c": 256},
        # odd sizes, taller than wide
        {"name": "ns_ragged", "kind": "ns", "n": 3, "r": 1000, "c": 333},
        # one side of the benchmark layer's 64 experts
        {"name": "muon_experts", "kind": "muon", "n": 64, "r": 1024, "c": 1024},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "route_grad", "experts", "experts", "train", "ns", "muon"])
    if kind in ("route", "route_grad"):
        E = rng.choice([8, 16, 60, 64, 96, 128, 160, 256])
        case = {"kind": kind, "T": _spread(rng, 1, 65536), "E": E, "K": rng.randint(1, 8), "score": rng.randint(0, 1),
                "renorm": rng.randint(0, 1), "scale": rng.choice([1.0, 2.5])}
        if kind == "route":
            groups = rng.choice([1, 1, 4, 8]) if E % 8 == 0 and E >= 64 else 1
            case.update(groups=groups, top=max(1, groups // 2), best=rng.randint(1, 2), bias=rng.randint(0, 1))
        return case
    if kind in ("experts", "train"):
        D, H, E = rng.choice([(1024, 1024, 64), (64, 256, 8), (512, 2048, 16), (200, 333, 10)])
        K = rng.randint(1, min(E, 6))
        most = 131072 if kind == "experts" else 32768
        return {"kind": kind, "T": _spread(rng, 1, most // K), "K": K, "D": D, "H": H, "E": E,
                "act": rng.choice([5, 6])}
    n, r, c = rng.choice([(8, 64, 256), (1, 1024, 64), (4, 512, 512), (1, 512, 2048), (1, 8192, 512),
                          (rng.randint(1, 40), 1024, 1024),
                          (rng.randint(1, 4), _spread(rng, 1, 2500), _spread(rng, 1, 2500))])
    return {"kind": kind, "n": n, "r": r, "c": c}


# ---- inputs ---------------------------------------------------------------------

LR, MU, STEPS = 3e-4, 0.95, 5


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=F32) * std


def _logits(g, T, E):
    """A balanced router's logits: some experts are liked a little more than others."""
    return _normal(g, (T, E), 1.2) + _normal(g, (1, E), 0.1)


def _gradients(g, n, r, c):
    """Gradient-like matrices: a few strong directions over noise."""
    k = max(1, min(r, c) // 16)
    return _normal(g, (n, r, k), 0.3 / math.sqrt(k)) @ _normal(g, (n, k, c)) * 1e-3 + _normal(g, (n, r, c), 1e-3)


def _layer(g, case):
    """x, experts and weights of the tokens' slots, W1, W2."""
    T, K, D, H, E = (case[k] for k in ("T", "K", "D", "H", "E"))
    x = _normal(g, (T, D))
    p, idx = torch.topk(torch.softmax(_logits(g, T, E), 1), K, dim=1)
    w1 = _normal(g, (E, D, H), 1 / math.sqrt(D))
    w2 = _normal(g, (E, H, D), 1 / math.sqrt(H))
    return x, idx.to(torch.int32), p / p.sum(1, keepdim=True), w1, w2


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "route":
        st["logits"] = _logits(g, case["T"], case["E"])
        st["bias"] = _normal(g, (case["E"],), 0.1) if case["bias"] else None
    elif kind == "route_grad":
        st["logits"] = _logits(g, case["T"], case["E"])
        st["idx"] = torch.topk(st["logits"], case["K"], dim=1)[1].to(torch.int32)
        st["dweight"] = _normal(g, (case["T"], case["K"]), 0.1)
    elif kind in ("experts", "train"):
        st["x"], st["idx"], st["weight"], st["w1"], st["w2"] = _layer(g, case)
        if kind == "train":
            st["dy"] = _normal(g, (case["T"], case["D"]), 1e-2)
    else:
        n, r, c = case["n"], case["r"], case["c"]
        st["g"] = _gradients(g, n, r, c)
        if kind == "muon":
            st["w"] = _normal(g, (n, r, c), 0.02)
            st["m"] = _gradients(g, n, r, c)
    return st


# ---- the plain forms --------------------------------------------------------------

def _scores(logits, score):
    return torch.softmax(logits, 1) if score == 0 else torch.sigmoid(logits)


def _top(v, k):
    """Indexes of the k largest of each row, equal ones by index."""
    return torch.sort(v, dim=1, descending=True, stable=True)[1][:, :k]


def _plain_route(case, logits, bias):
    # in 64 bits: two values may lie closer than 32 bits tell apart
    T, E, G = case["T"], case["E"], case["groups"]
    s = _scores(logits.to(F64), case["score"])
    c = s if bias is None else s + bias.to(F64)
    if G > 1:
        group = torch.sort(c.view(T, G, E // G), dim=2, descending=True)[0][:, :, :case["best"]].sum(2)
        keep = torch.zeros((T, G), device=DEV, dtype=torch.bool).scatter_(1, _top(group, case["top"]), True)
        c = torch.where(keep.repeat_interleave(E // G, dim=1), c, -math.inf)
    idx = _top(c, case["K"])
    w = torch.gather(s, 1, idx)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return idx.to(torch.int32), (w * case["scale"]).to(F32)


def _plain_route_grad(case, logits, idx, dweight):
    s = _scores(logits, case["score"])
    i = idx.long()
    u = dweight * case["scale"]
    if case["renorm"]:
        sk = torch.gather(s, 1, i)
        total = sk.sum(1, keepdim=True)
        u = (u - (u * sk).sum(1, keepdim=True) / total) / total
    ds = torch.zeros_like(s).scatter_add_(1, i, u)
    if case["score"] == 0:
        return s * (ds - (s * ds).sum(1, keepdim=True))
    return s * (1 - s) * ds


def _act(u, code):
    return u * torch.sigmoid(u) if code == 5 else 0.5 * u * (1 + torch.erf(u / math.sqrt(2)))


def _act_grad(u, code):
    if code == 5:
        s = torch.sigmoid(u)
        return s + u * s * (1 - s)
    return 0.5 * (1 + torch.erf(u / math.sqrt(2))) + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)


def _sorted(idx, E):
    """The experts in use, their rows padded to the longest: the slot (token and
    choice) of each row, its place among the padded rows, and their number."""
    flat = idx.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    count = torch.bincount(flat, minlength=E)
    used = torch.nonzero(count)[:, 0]
    number = torch.cumsum(count > 0, 0) - 1
    start = torch.cumsum(count, 0) - count
    e = flat[order]
    most = int(count.max())
    at = number[e] * most + torch.arange(len(e), device=DEV) - start[e]
    return used, order, at, most


def _padded(rows, at, used, most):
    out = torch.zeros((len(used) * most, rows.shape[1]), device=DEV, dtype=rows.dtype)
    out[at] = rows
    return out.view(len(used), most, -1)


def _plain_experts(case, st):
    T, K, E, act = case["T"], case["K"], case["E"], case["act"]
    x, weight = st["x"], st["weight"].reshape(-1)
    used, order, at, most = _sorted(st["idx"], E)
    w1, w2 = (st["w1"], st["w2"]) if len(used) == E else (st["w1"][used], st["w2"][used])
    xs = _padded(x[order // K], at, used, most)
    u = xs @ w1
    h = _act(u, act)
    o = (h @ w2).view(-1, case["D"])[at]
    slots = torch.empty_like(o)
    slots[order] = o * weight[order, None]
    y = slots.view(T, K, -1).sum(1)
    if case["kind"] == "experts":
        return y
    dys = _padded(st["dy"][order // K], at, used, most)
    dh = dys @ w2.transpose(1, 2)
    ws = _padded(weight[order, None], at, used, most)
    dweight = torch.empty_like(weight)
    dweight[order] = (h * dh).sum(2).view(-1)[at]
    du = ws * dh * _act_grad(u, act)
    slots[order] = (du @ w1.transpose(1, 2)).view(-1, case["D"])[at]
    dx = slots.view(T, K, -1).sum(1)
    dw1, dw2 = xs.transpose(1, 2) @ du, (h * ws).transpose(1, 2) @ dys
    if len(used) < E:
        dw1 = torch.zeros_like(st["w1"]).index_copy_(0, used, dw1)
        dw2 = torch.zeros_like(st["w2"]).index_copy_(0, used, dw2)
    return y, dx, dweight.view(T, K), dw1, dw2


COEF = (3.4445, -4.7750, 2.0315)


def _plain_ns(g):
    a, b, c = COEF
    x = g / (torch.linalg.vector_norm(g, dim=(1, 2), keepdim=True) + 1e-7)
    tall = g.shape[1] > g.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    for _ in range(STEPS):
        s = x @ x.transpose(1, 2)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(1, 2).contiguous() if tall else x


def _plain_muon(st):
    g, m, w = st["g"], st["m"], st["w"]
    m.mul_(MU).add_(g)
    q = _plain_ns(g + MU * m)
    w.mul_(1 - 0.01 * LR).sub_(q, alpha=LR * math.sqrt(min(g.shape[1:])))
    return w, m


def _plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "route":
        return _plain_route(case, st["logits"], st["bias"])
    if kind == "route_grad":
        return _plain_route_grad(case, st["logits"], st["idx"], st["dweight"])
    if kind in ("experts", "train"):
        return _plain_experts(case, st)
    return _plain_ns(st["g"]) if kind == "ns" else _plain_muon(st)


# ---- the framework's entry points ---------------------------------------------------

def _workspace(nbytes):
    """A workspace of the call's own, on the current device and ordered on the current stream as the
    outputs are: calls on two streams or devices, or captured into two graphs, share none."""
    return torch.empty(nbytes, device=DEV, dtype=torch.uint8)


def _own(st):
    from neuralscript_amd import runtime as rt

    lib = rt.lib()
    case = st["case"]
    kind = case["kind"]
    stream = torch.cuda.current_stream().cuda_stream

    def ptr(t):
        return None if t is None else t.data_ptr()

    if kind == "route":
        T, E, K = case["T"], case["E"], case["K"]
        idx = torch.empty((T, K), device=DEV, dtype=torch.int32)
        weight = torch.empty((T, K), device=DEV, dtype=F32)
        rt.op("moe_route", ptr(st["logits"]), ptr(st["bias"]), None, ptr(idx), ptr(weight), T, E, K, case["groups"],
              case["top"], case["best"], case["score"], case["renorm"], case["scale"], stream)
        return idx, weight
    if kind == "route_grad":
        T, E, K = case["T"], case["E"], case["K"]
        dlogits = torch.empty((T, E), device=DEV, dtype=F32)
        rt.op("moe_route_grad", ptr(st["dweight"]), ptr(st["logits"]), None, ptr(st["idx"]), ptr(dlogits), T, E, K,
              case["score"], case["renorm"], case["scale"], stream)
        return dlogits
    if kind in ("experts", "train"):
        sizes = [case[k] for k in ("T", "K", "D", "H", "E")]
        train = kind == "train"
        ws = _workspace(lib.nsh_op_moe_experts_workspace(*sizes, int(train)))
        y = torch.empty_like(st["x"])
        state = None
        if train:
            state = torch.empty(lib.nsh_op_moe_experts_state(*sizes), device=DEV, dtype=torch.uint8)
        rt.op("moe_experts", ptr(st["x"]), ptr(st["idx"]), ptr(st["weight"]), ptr(st["w1"]), ptr(st["w2"]), ptr(y),
              *sizes, case["act"], ptr(state), ptr(ws), stream)
        if not train:
            return y
        dx, dweight = torch.empty_like(st["x"]), torch.empty_like(st["weight"])
        dw1, dw2 = torch.empty_like(st["w1"]), torch.empty_like(st["w2"])
        rt.op("moe_experts_grad", ptr(st["dy"]), ptr(st["x"]), ptr(st["weight"]), ptr(st["w1"]), ptr(st["w2"]),
              ptr(state), ptr(dx), ptr(dweight), ptr(dw1), ptr(dw2), *sizes, case["act"], ptr(ws), stream)
        return y, dx, dweight, dw1, dw2
    n, r, c = case["n"], case["r"], case["c"]
    ws = _workspace(lib.nsh_op_newton_schulz_workspace(n, r, c))
    if kind == "ns":
        q = torch.empty_like(st["g"])
        rt.op("newton_schulz", ptr(st["g"]), ptr(q), n, r, c, STEPS, ptr(ws), stream)
        return q
    rt.op("muon_ns_step", ptr(st["w"]), ptr(st["g"]), ptr(st["m"]), n, r, c, LR, MU, 1, STEPS, ptr(ws), stream)
    return st["w"], st["m"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- work ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("route", "route_grad"):
        T, E, K = case["T"], case["E"], case["K"]
        # logits in, experts and weights out (the gradient: weights' gradients and experts in, logits' out)
        return {"bytes": 4.0 * T * E * (1 if kind == "route" else 2) + 8.0 * T * K, "flops": 5.0 * T * E}
    if kind in ("experts", "train"):
        T, K, D, H, E = (case[k] for k in ("T", "K", "D", "H", "E"))
        used = min(E, T * K) * 8.0 * D * H
        b, f = used + 8.0 * T * D + 8.0 * T * K, 4.0 * T * K * D * H
        if kind == "train":  # dy in; gradients of x, the weights and every matrix out
            b += 8.0 * T * D + 4.0 * T * K + 8.0 * E * D * H
            f *= 3
        return {"bytes": b, "flops": f}
    n, r, c = case["n"], case["r"], case["c"]
    m, N = min(r, c), max(r, c)
    # the two symmetric products by half
    flops = STEPS * n * (1.0 * m * m * N + 1.0 * m ** 3 + 2.0 * m * m * N)
    return {"bytes": n * r * c * 4.0 * (2 if kind == "ns" else 5), "flops": flops}


# ---- the definition in 64 bits --------------------------------------------------------

def _exact_scores(logits, score):
    l = logits.to(F64)
    if score:
        return 1 / (1 + torch.exp(-l))
    e = torch.exp(l - l.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _rank(v):
    """How many come before each value of a row: the larger ones, and equal ones of a lower index."""
    n = v.shape[1]
    lower = torch.ones((n, n), device=DEV, dtype=torch.bool).tril(-1)  # [i, j]: j < i
    more = v[:, None, :] > v[:, :, None]
    same = (v[:, None, :] == v[:, :, None]) & lower
    return (more | same).sum(2)


def _exact_route(case, logits, bias):
    E, K, G = case["E"], case["K"], case["groups"]
    idx, weight = [], []
    for block in torch.split(logits, max(1, (1 << 26) // (E * E))):
        s = _exact_scores(block, case["score"])
        c = s.clone() if bias is None else s + bias.to(F64)
        if G > 1:
            by = c.view(-1, G, E // G)
            total = by.amax(2)
            if case["best"] == 2:
                total = total + by.kthvalue(E // G - 1, dim=2)[0]
            c[(_rank(total) >= case["top"]).repeat_interleave(E // G, dim=1)] = -math.inf
        rank = _rank(c)
        i = torch.empty((len(c), K), device=DEV, dtype=torch.int64)
        row, e = torch.nonzero(rank < K, as_tuple=True)
        i[row, rank[row, e]] = e
        w = torch.gather(s, 1, i) * case["scale"]
        if case["renorm"]:
            w = w * case["scale"] / w.sum(1, keepdim=True)
        idx.append(i.to(torch.int32))
        weight.append(w)
    return torch.cat(idx), torch.cat(weight)


def _exact_route_grad(case, logits, idx, dweight):
    """Row by row dl = J^T dw, J the weights' derivatives by the scores and the scores' by the logits."""
    s = _exact_scores(logits, case["score"])
    i, dw, scale = idx.long(), dweight.to(F64), case["scale"]
    chosen = torch.gather(s, 1, i)
    if case["renorm"]:
        total = chosen.sum(1, keepdim=True)
        dchosen = scale * (dw * total - (dw * chosen).sum(1, keepdim=True)) / total ** 2
    else:
        dchosen = scale * dw
    if case["score"]:
        return torch.zeros_like(s).scatter_add_(1, i, dchosen * chosen * (1 - chosen))
    out = -s * (dchosen * chosen).sum(1, keepdim=True)
    return out.scatter_add_(1, i, dchosen * chosen)


def _exact_experts(case, st):
    T, K, E = case["T"], case["K"], case["E"]
    train = case["kind"] == "train"
    x, weight = st["x"].to(F64), st["weight"].to(F64)
    y = torch.zeros_like(x)
    if train:
        dy, dx, dweight = st["dy"].to(F64), torch.zeros_like(x), torch.zeros_like(weight)
        dw1, dw2 = (torch.zeros(st[k].shape, device=DEV, dtype=F64) for k in ("w1", "w2"))
    for e in range(E):
        t, k = torch.nonzero(st["idx"] == e, as_tuple=True)
        if len(t) == 0:
            continue
        w1, w2, w = st["w1"][e].to(F64), st["w2"][e].to(F64), weight[t, k][:, None]
        u = x[t] @ w1
        h = _act(u, case["act"])
        y.index_add_(0, t, w * (h @ w2))
        if train:
            dh = dy[t] @ w2.t()
            dweight[t, k] = (dh * h).sum(1)
            du = dh * w * _act_grad(u, case["act"])
            dx.index_add_(0, t, du @ w1.t())
            dw1[e] = x[t].t() @ du
            dw2[e] = (w * h).t() @ dy[t]
    return (y, dx, dweight, dw1, dw2) if train else y


def _exact_ns(g):
    """Matrix by matrix, as a polynomial of the smaller Gram matrix applied once a step."""
    a, b, c = COEF
    out = torch.empty_like(g)
    for i in range(g.shape[0]):
        x = g[i] / (g[i].square().sum().sqrt() + 1e-7)
        eye = torch.eye(min(x.shape), device=DEV, dtype=F64)
        for _ in range(STEPS):
            gram = x.t() @ x if x.shape[0] > x.shape[1] else x @ x.t()
            p = a * eye + gram @ (b * eye + c * gram)
            x = x @ p if x.shape[0] > x.shape[1] else p @ x
        out[i] = x
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _exact_route(case, st["logits"], st["bias"])
    if kind == "route_grad":
        return _exact_route_grad(case, st["logits"], st["idx"], st["dweight"])
    if kind in ("experts", "train"):
        return _exact_experts(case, st)
    g = st["g"].to(F64)
    if kind == "ns":
        return _exact_ns(g)
    m = st["m"].to(F64) * MU + g
    step = LR * math.sqrt(min(case["r"], case["c"]))
    return st["w"].to(F64) * (1 - 0.01 * LR) - step * _exact_ns(g + MU * m), m
