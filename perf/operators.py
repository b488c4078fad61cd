"""Performance cases of the trainable operators around a graph's edges.

diff    TorchGraph.diff_attention / diff_attention_packed: differential
        attention over the edges of a graph prepared once, the difference of two
        softmax maps of 64 dims per head with a learned weight each, values of
        128 dims; alone, or as a training step with all its gradients.
linear  torch_ops.linear: a projection with bias, activation and residual in
        its epilogue; alone, or as a training step.

`own` chooses between the framework's operators and their plain form in torch.
"""
from __future__ import annotations

import math

import torch

own = False

MAP = 64        # dims of one map
D = 2 * MAP     # per head: both maps of q and k side by side, and the values
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _diff(name, n, degree, heads=1, dtype="float16", train=False, packed=False, graph="powerlaw",
          loops=True, gamma=2.2, max_degree=16384, community=4096, p_intra=0.8):
    return {"name": name, "op": "diff", "n": n, "degree": degree, "heads": heads, "dtype": dtype,
            "train": train, "packed": packed, "graph": graph, "loops": loops, "gamma": gamma,
            "max_degree": max_degree, "community": community, "p_intra": p_intra}


def _linear(name, n, K, M, act="none", dtype="float16", bias=True, residual=False, train=False):
    return {"name": name, "op": "linear", "n": n, "K": K, "M": M, "act": act, "dtype": dtype,
            "bias": bias, "residual": residual, "train": train}


def listed():
    return [
        # inference on a citation-sized graph: latency
        _diff("diff_small", 2708, 3.9, gamma=2.5, max_degree=170),
        # full-graph inference on a large graph of random node ids
        _diff("diff_1m", 1_000_000, 16),
        # the same from the output of one projection, communities, three heads,
        # an odd number of nodes, some of them without an edge
        _diff("diff_packed_h3", 150_001, 30, heads=3, dtype="bfloat16", packed=True,
              graph="community", loops=False, community=1000),
        # a training step on a sampled mini-batch
        _diff("diff_train_batch", 20_011, 14, heads=2, train=True, loops=False, packed=True,
              gamma=2.5, max_degree=500),
        # a full-graph training step: communities, many edges per node
        _diff("diff_train_community", 100_000, 40, heads=2, dtype="bfloat16", train=True,
              graph="community"),
        # and on random node ids
        _diff("diff_train_500k", 500_000, 12, train=True),
        # one node's features through a feed-forward product
        _linear("linear_one", 1, 1024, 4096, act="gelu"),
        # a small batch of odd sizes
        _linear("linear_odd", 1003, 100, 301, act="silu", dtype="bfloat16", residual=True),
        # the feed-forward of a full-graph layer: many rows, few inputs
        _linear("linear_up_500k", 500_000, 128, 512, act="gelu"),
        # its way back, with the residual, as a training step
        _linear("linear_down_train", 200_003, 512, 128, residual=True, train=True),
        # a wide model's feed-forward, forward and as a training step
        _linear("linear_wide", 32_768, 1024, 4096, act="relu", dtype="bfloat16"),
        _linear("linear_wide_train", 32_768, 1024, 4096, act="gelu", dtype="bfloat16", train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["float16", "bfloat16"])
    train = rng.random() < 0.5
    if rng.random() < 0.5:
        n = _log(rng, 16, 500_000)
        degree = round(math.exp(rng.uniform(math.log(1.5), math.log(50))), 2)
        heads = rng.choice([1, 1, 2, 3, 4, 6])
        most = 7.5e6 if train else 1.5e7   # edges times heads
        while heads > 1 and n * (degree + 1) * heads > most:
            heads -= 1
        degree = min(degree, max(1.5, round(most / (n * heads) - 1, 2)))
        return {"op": "diff", "n": n, "degree": degree, "heads": heads, "dtype": dtype,
                "train": train, "packed": rng.random() < 0.5,
                "graph": rng.choice(["powerlaw", "community"]), "loops": rng.random() < 0.6,
                "gamma": round(rng.uniform(2.1, 2.9), 2),
                "max_degree": int(min(16384, max(16, n // 16))),
                "community": rng.choice([512, 1000, 4096]),
                "p_intra": round(rng.uniform(0.6, 0.9), 2)}
    n = _log(rng, 1, 500_000)
    K, M = _log(rng, 8, 4096), _log(rng, 8, 4096)
    if rng.random() < 0.6:   # the usual widths
        K, M = -(-K // 64) * 64, -(-M // 64) * 64
    n = max(1, min(n, int(1.3e11 / (K * M)), int(2e8 / (K + M))))
    return {"op": "linear", "n": n, "K": K, "M": M,
            "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "dtype": dtype,
            "bias": rng.random() < 0.7, "residual": rng.random() < 0.5, "train": train}


# ------------------------------------------------------------------ inputs

def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt) % (1 << 62))


def _graph(case, seed):
    """Symmetric CSR (row_ptr, col_idx), int32 CUDA tensors, columns ascending
    and unique in each row: power-law degrees on random node ids, or
    communities of consecutive ids."""
    n, gen = case["n"], _generator(seed, 0)
    pairs = max(1, int(n * case["degree"] / 2))
    if case["graph"] == "powerlaw":
        w = torch.arange(1, n + 1, dtype=torch.float64, device="cuda")
        w = w ** (-1.0 / (case["gamma"] - 1.0))
        w = torch.clamp(w, max=float(w.mean()) * max(2.0, case["max_degree"] / case["degree"]))
        cdf = torch.cumsum(w, 0)
        x = torch.rand(2, pairs, dtype=torch.float64, device="cuda", generator=gen) * cdf[-1]
        ends = torch.searchsorted(cdf, x).clamp_(max=n - 1)
        ends = torch.randperm(n, device="cuda", generator=gen)[ends]   # no order by degree
        u, v = ends[0], ends[1]
    else:
        c = case["community"]
        u = torch.randint(n, (pairs,), device="cuda", generator=gen)
        intra = torch.rand(pairs, device="cuda", generator=gen) < case["p_intra"]
        base = u // c * c
        x = torch.rand(pairs, dtype=torch.float64, device="cuda", generator=gen)
        v = torch.where(intra, base + (x * torch.clamp(n - base, max=c)).long(), (x * n).long())
    keep = u != v
    u, v = u[keep], v[keep]
    keys = [u * n + v, v * n + u]
    if case["loops"]:
        i = torch.arange(n, device="cuda")
        keys.append(i * n + i)
    keys = torch.unique(torch.cat(keys))
    row_ptr = torch.searchsorted(keys, torch.arange(n + 1, device="cuda") * n)
    return row_ptr.to(torch.int32), (keys % n).to(torch.int32)


def _randn(gen, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32).to(dtype)


def _inputs(case, seed):
    gen, dtype = _generator(seed, 1), TYPES[case["dtype"]]
    n = case["n"]
    if case["op"] == "diff":
        H = case["heads"]
        row_ptr, col_idx = _graph(case, seed)
        x = {"row_ptr": row_ptr, "col_idx": col_idx, "qkv": _randn(gen, dtype, n, 3 * H * D),
             # the weights that the learned vectors give: around 0.5
             "lam": 0.5 + 0.2 * torch.randn(H, device="cuda", generator=gen)}
        if not case["packed"]:
            x["q"], x["k"], x["v"] = (t.contiguous() for t in
                                      x.pop("qkv").view(n, 3, H, D).unbind(1))
        if case["train"]:
            x["do"] = _randn(gen, dtype, n, H, D)
        return x
    K, M = case["K"], case["M"]
    x = {"x": _randn(gen, dtype, n, K),
         "w": (torch.randn(M, K, device="cuda", generator=gen) * K ** -0.5).to(dtype)}
    if case["bias"]:
        x["b"] = _randn(gen, dtype, M)
    if case["residual"]:
        x["r"] = _randn(gen, dtype, n, M)
    if case["train"]:
        x["dy"] = _randn(gen, dtype, n, M)
    return x


LEAVES = ("qkv", "q", "k", "v", "lam", "x", "w", "b", "r")


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["train"]:
        for name in LEAVES:
            if name in state:
                state[name].requires_grad_()
    if case["op"] == "diff":
        if own:
            # the prepared graph that a program keeps: tile lists and plan, and
            # for training those of the reversed edges
            from fused3s_amd import torch_ops
            state["graph"] = torch_ops.TorchGraph(state["row_ptr"], state["col_idx"],
                                                  heads=case["heads"])
            if case["train"]:
                state["graph"].prepare_backward()
        else:
            # and here the edges' two ends
            deg = (state["row_ptr"][1:] - state["row_ptr"][:-1]).long()
            state["rows"] = torch.repeat_interleave(torch.arange(case["n"], device="cuda"), deg)
            state["cols"] = state["col_idx"].long()
    return state


# -------------------------------------------------------------- the operators

def run(state):
    case = state["case"]
    if own:
        return _own_diff(state) if case["op"] == "diff" else _own_linear(state)
    with torch.no_grad():
        return _plain_diff(state) if case["op"] == "diff" else _plain_linear(state)


def _own_diff(state):
    case, graph = state["case"], state["graph"]
    if case["packed"]:
        o = graph.diff_attention_packed(state["qkv"], state["lam"], MAP ** -0.5)
        leaves = {"dqkv": state["qkv"], "dlam": state["lam"]}
    else:
        o = graph.diff_attention(state["q"], state["k"], state["v"], state["lam"], MAP ** -0.5)
        leaves = {"dq": state["q"], "dk": state["k"], "dv": state["v"], "dlam": state["lam"]}
    if not case["train"]:
        return {"o": o}
    grads = torch.autograd.grad(o, list(leaves.values()), state["do"])
    return {"o": o.detach(), **dict(zip(leaves, grads))}


def _own_linear(state):
    from fused3s_amd import torch_ops
    case = state["case"]
    y = torch_ops.linear(state["x"], state["w"], state.get("b"),
                         activation=None if case["act"] == "none" else case["act"],
                         residual=state.get("r"))
    if not case["train"]:
        return {"y": y}
    leaves = {"d" + name: state[name] for name in ("x", "w", "b", "r") if name in state}
    grads = torch.autograd.grad(y, list(leaves.values()), state["dy"])
    return {"y": y.detach(), **dict(zip(leaves, grads))}


def _plain_diff(state):
    case = state["case"]
    n, H, dtype, scale = case["n"], case["heads"], TYPES[case["dtype"]], MAP ** -0.5
    rows, cols = state["rows"], state["cols"]
    if case["packed"]:
        q, k, v = state["qkv"].view(n, 3, H, D).float().unbind(1)
    else:
        q, k, v = (state[name].float() for name in ("q", "k", "v"))
    lam = state["lam"]

    def by_row(index, values):
        out = torch.zeros(n, *values.shape[1:], device="cuda")
        return out.index_add_(0, index, values)

    maps = (-1, H, 2, MAP)
    s = (q[rows] * k[cols]).view(maps).sum(-1) * scale
    top = torch.full((n, H, 2), -math.inf, device="cuda")
    top.scatter_reduce_(0, rows[:, None, None].expand_as(s), s, "amax")
    p = torch.exp(s - top[rows])
    p = p / by_row(rows, p)[rows]
    w = p[..., 0] - lam * p[..., 1]
    o = by_row(rows, w[..., None] * v[cols]).to(dtype)
    if not case["train"]:
        return {"o": o}
    do = state["do"].float()
    g = (do[rows] * v[cols]).sum(-1, keepdim=True)
    total = by_row(rows, p * g)
    ds = p * (g - total[rows]) * scale
    ds[..., 1] *= -lam
    ds = ds[..., None]
    dq = by_row(rows, (ds * k[cols].view(maps)).view(-1, H, D)).to(dtype)
    dk = by_row(cols, (ds * q[rows].view(maps)).view(-1, H, D)).to(dtype)
    dv = by_row(cols, w[..., None] * do[rows]).to(dtype)
    dlam = -total[..., 1].double().sum(0).float()
    if case["packed"]:
        return {"o": o, "dqkv": torch.stack([dq, dk, dv], 1).view(n, 3 * H * D), "dlam": dlam}
    return {"o": o, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def _act(act, z):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return (0.5 * z * (1 + t),
                0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z))
    s = 1 / (1 + torch.exp(-z))   # silu
    return z * s, s * (1 + z * (1 - s))


def _plain_linear(state):
    case = state["case"]
    dtype = TYPES[case["dtype"]]
    x, w = state["x"].float(), state["w"].float()
    z = x @ w.t()
    if case["bias"]:
        z = z + state["b"].float()
    a, slope = _act(case["act"], z)
    if case["residual"]:
        a = a + state["r"].float()
    y = a.to(dtype)
    if not case["train"]:
        return {"y": y}
    dz = state["dy"].float() * slope
    out = {"y": y, "dx": (dz @ w).to(dtype), "dw": (dz.t() @ x).to(dtype)}
    if case["bias"]:
        out["db"] = dz.sum(0).to(dtype)
    if case["residual"]:
        out["dr"] = state["dy"]
    return out


# --------------------------------------------------------------------- work

def work(case):
    n = case["n"]
    if case["op"] == "diff":
        H = case["heads"]
        edges = n * (case["degree"] + (1 if case["loops"] else 0))
        lists = 4.0 * (edges + n)
        feature = 2.0 * n * H * D
        if case["train"]:   # q, k, v, do and o, dq, dk, dv; six products of D per edge and head
            return {"bytes": 8 * feature + lists, "flops": 12.0 * D * H * edges}
        return {"bytes": 4 * feature + lists, "flops": 4.0 * D * H * edges}
    K, M = case["K"], case["M"]
    x, w, y = 2.0 * n * K, 2.0 * K * M, 2.0 * n * M
    size = x + w + y + (y if case["residual"] else 0) + (2.0 * M if case["bias"] else 0)
    if case["train"]:   # and dy, dx, dw, db
        return {"bytes": size + y + x + w + (2.0 * M if case["bias"] else 0),
                "flops": 6.0 * n * K * M}
    return {"bytes": size, "flops": 2.0 * n * K * M}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    x = _inputs(case, seed)
    return _exact_diff(case, x) if case["op"] == "diff" else _exact_linear(case, x)


def _exact_diff(case, x):
    """A few rows at a time; gradients by differentiation of the forward pass."""
    n, H, train = case["n"], case["heads"], case["train"]
    if case["packed"]:
        q, k, v = (t.double() for t in x["qkv"].view(n, 3, H, D).unbind(1))
    else:
        q, k, v = (x[name].double() for name in ("q", "k", "v"))
    lam = x["lam"].double()
    o = torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
    grads = [torch.zeros_like(t) for t in (q, k, v, lam)] if train else []
    ptr = x["row_ptr"].long()
    begin = ptr.cpu().tolist()
    r0 = 0
    while r0 < n:
        r1 = r0 + 1
        low, high = r0 + 1, n
        while low <= high:   # the most rows of at most 2^20 edges and heads
            mid = (low + high) // 2
            if (begin[mid] - begin[r0]) * H <= 1 << 20:
                r1, low = max(r1, mid), mid + 1
            else:
                high = mid - 1
        cols = x["col_idx"][begin[r0]:begin[r1]].long()
        if cols.numel():
            lengths = ptr[r0 + 1:r1 + 1] - ptr[r0:r1]
            row = torch.repeat_interleave(torch.arange(r1 - r0, device="cuda"), lengths)
            with torch.set_grad_enabled(train):
                a = [q[r0:r1].clone(), k[cols], v[cols], lam.clone()]
                if train:
                    a = [t.requires_grad_() for t in a]
                qr = a[0][row]
                maps = []
                for c in (0, 1):
                    at = slice(c * MAP, (c + 1) * MAP)
                    s = (qr[..., at] * a[1][..., at]).sum(-1) * MAP ** -0.5
                    e = torch.exp(s - s.detach().max())   # (far from under- and overflow here)
                    total = torch.zeros(r1 - r0, H, dtype=e.dtype, device="cuda")
                    maps.append(e / total.index_add(0, row, e)[row])
                weighted = (maps[0] - a[3] * maps[1])[..., None] * a[2]
                out = torch.zeros(r1 - r0, H, D, dtype=weighted.dtype, device="cuda")
                out = out.index_add(0, row, weighted)
                o[r0:r1] = out.detach()
                if train:
                    g = torch.autograd.grad(out, a, x["do"][r0:r1].double())
                    grads[0][r0:r1] = g[0]
                    grads[1].index_add_(0, cols, g[1])
                    grads[2].index_add_(0, cols, g[2])
                    grads[3] += g[3]
        r0 = r1
    if not train:
        return {"o": o}
    dq, dk, dv, dlam = grads
    if case["packed"]:
        return {"o": o, "dqkv": torch.cat([t.reshape(n, H * D) for t in (dq, dk, dv)], 1),
                "dlam": dlam}
    return {"o": o, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def _exact_linear(case, x):
    a = {name: t.double().requires_grad_(case["train"]) for name, t in x.items() if name != "dy"}
    F = torch.nn.functional
    z = F.linear(a["x"], a["w"], a.get("b"))
    act = {"none": lambda t: t, "relu": F.relu, "gelu": F.gelu, "silu": F.silu,
           "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[case["act"]]
    y = act(z)
    if case["residual"]:
        y = y + a["r"]
    if not case["train"]:
        return {"y": y}
    names = [name for name in ("x", "w", "b", "r") if name in a]
    grads = torch.autograd.grad(y, [a[name] for name in names], x["dy"].double())
    return {"y": y.detach(), **{"d" + name: g for name, g in zip(names, grads)}}
