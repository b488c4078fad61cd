"""Performance cases of the operators that a graph transformer trains with beside
its products: attention over the edges, norms, the loss of its classifier.

attention  TorchGraph.edge_attention / edge_attention_packed: softmax attention
           over the edges of a graph prepared once, 64 dims per head, scores capped
           by a tanh and lowered by the distance of the two nodes; alone, or as a
           training step with all its gradients.
norm       torch_ops.layer_norm: alone, or as a training step.
loss       torch_ops.linear_cross_entropy: the cross entropy of a linear classifier
           over many classes (or entities); alone, or as a training step.

`own` chooses between the framework's operators and their plain form in torch.
"""
from __future__ import annotations

import math

import torch

own = False

D = 64
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def _attention(name, n, degree, heads=1, dtype="float16", train=False, packed=False,
               graph="powerlaw", loops=True, gamma=2.2, max_degree=16384, community=4096,
               p_intra=0.8, cap=0.0, dims=0):
    return {"name": name, "op": "attention", "n": n, "degree": degree, "heads": heads,
            "dtype": dtype, "train": train, "packed": packed, "graph": graph, "loops": loops,
            "gamma": gamma, "max_degree": max_degree, "community": community, "p_intra": p_intra,
            "cap": cap, "dims": dims}


def _norm(name, n, width, dtype="float16", weights="same", bias=True, train=False):
    return {"name": name, "op": "norm", "n": n, "width": width, "dtype": dtype,
            "weights": weights, "bias": bias, "train": train}


def _loss(name, n, K, classes, dtype="bfloat16", bias=True, reduction="mean", ignored=0.1,
          train=False):
    return {"name": name, "op": "loss", "n": n, "K": K, "classes": classes, "dtype": dtype,
            "bias": bias, "reduction": reduction, "ignored": ignored, "train": train}


def listed():
    return [
        # inference on a citation-sized graph, capped scores: latency
        _attention("attention_small", 2708, 3.9, gamma=2.5, max_degree=170, cap=30.0),
        # full-graph inference on random node ids, capped, edges weighted by the nodes' times
        _attention("attention_1m", 1_000_000, 16, cap=50.0, dims=1),
        # points in space in communities, four heads, from one projection's output, an
        # odd number of nodes, some of them without an edge
        _attention("attention_packed_h4", 150_001, 30, heads=4, dtype="bfloat16", packed=True,
                   graph="community", loops=False, community=1000, dims=3),
        # a training step on a sampled mini-batch
        _attention("attention_train_batch", 20_011, 14, heads=2, train=True, loops=False,
                   packed=True, gamma=2.5, max_degree=500, cap=30.0, dims=3),
        # a full-graph training step on random node ids
        _attention("attention_train_500k", 500_000, 12, dtype="bfloat16", train=True, cap=50.0,
                   dims=1),
        # one node's features
        _norm("norm_one", 1, 1024),
        # a small batch of odd sizes, trained
        _norm("norm_odd_train", 1003, 301, dtype="bfloat16", train=True),
        # a full graph's features: inference, and a training step
        _norm("norm_1m", 1_000_000, 128),
        _norm("norm_train_500k", 500_000, 256, dtype="bfloat16", weights="float32", train=True),
        # a few nodes ranked against a vocabulary of entities
        _loss("loss_few", 64, 256, 50_021, dtype="float16", reduction="none", ignored=0.0),
        # a training step of node classification on a full graph
        _loss("loss_nodes_train", 200_003, 128, 47, dtype="float16", ignored=0.4, train=True),
        # a training step of predicting masked entities
        _loss("loss_entities_train", 16_384, 512, 100_003, bias=False, train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    train = rng.random() < 0.5
    op = rng.choice(["attention", "norm", "loss"])
    if op == "attention":
        n = _log(rng, 16, 500_000)
        degree = round(math.exp(rng.uniform(math.log(1.5), math.log(50))), 2)
        heads = rng.choice([1, 1, 2, 3, 4, 8])
        most = 7.5e6 if train else 1.5e7   # edges times heads
        while heads > 1 and n * (degree + 1) * heads > most:
            heads -= 1
        degree = min(degree, max(1.5, round(most / (n * heads) - 1, 2)))
        return {"op": op, "n": n, "degree": degree, "heads": heads,
                "dtype": rng.choice(["float16", "bfloat16"]), "train": train,
                "packed": rng.random() < 0.5, "graph": rng.choice(["powerlaw", "community"]),
                "loops": rng.random() < 0.6, "gamma": round(rng.uniform(2.1, 2.9), 2),
                "max_degree": int(min(16384, max(16, n // 16))),
                "community": rng.choice([512, 1000, 4096]),
                "p_intra": round(rng.uniform(0.6, 0.9), 2),
                "cap": rng.choice([0.0, 20.0, 30.0, 50.0]), "dims": rng.choice([0, 1, 2, 3])}
    if op == "norm":
        width = _log(rng, 8, 16384)
        if rng.random() < 0.6:   # the usual widths
            width = -(-width // 64) * 64
        n = max(1, min(_log(rng, 1, 1_000_000), int(1.28e8 / width)))
        return {"op": op, "n": n, "width": width, "bias": rng.random() < 0.8, "train": train,
                "dtype": rng.choice(["float16", "bfloat16", "float32"]),
                "weights": rng.choice(["same", "float32"])}
    K, classes = _log(rng, 16, 1024), _log(rng, 2, 100_000)
    if rng.random() < 0.7:
        K = -(-K // 64) * 64
    n = max(1, min(_log(rng, 1, 500_000), int(8.3e11 / (K * classes)), int(2e8 / K)))
    dtype, reduction = rng.choice(["float16", "bfloat16"]), rng.choice(["mean", "mean", "sum", "none"])
    if train and reduction != "mean":
        dtype = "bfloat16"   # (sums over all rows leave binary16)
    return {"op": op, "n": n, "K": K, "classes": classes, "dtype": dtype,
            "bias": rng.random() < 0.5, "reduction": reduction,
            "ignored": rng.choice([0.0, 0.1, 0.5]) if n > 8 else 0.0, "train": train}


# ------------------------------------------------------------------ inputs

def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt) % (1 << 62))


def _graph(case, seed):
    """Symmetric CSR (row_ptr, col_idx), int32 CUDA tensors, columns ascending
    and unique in each row: power-law degrees on random node ids, or
    communities of consecutive ids."""
    n, gen = case["n"], _generator(seed, 10)
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


def _inputs(case, seed):
    gen, dtype, n = _generator(seed, 11), TYPES[case["dtype"]], case["n"]

    def randn(*shape, of=dtype, scale=1.0, shift=0.0):
        x = torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32)
        return (x * scale + shift).to(of)

    if case["op"] == "attention":
        H = case["heads"]
        row_ptr, col_idx = _graph(case, seed)
        x = {"row_ptr": row_ptr, "col_idx": col_idx, "qkv": randn(n, 3 * H * D)}
        if not case["packed"]:
            x["q"], x["k"], x["v"] = (t.contiguous() for t in
                                      x.pop("qkv").view(n, 3, H, D).unbind(1))
        if case["dims"]:   # times or points in a box, slopes falling from head to head
            x["positions"] = torch.rand(n, case["dims"], device="cuda", generator=gen) * 8.0
            x["slopes"] = (0.5 ** torch.arange(1, H + 1, device="cuda").float()
                           + 0.02 * torch.randn(H, device="cuda", generator=gen))
        if case["train"]:
            x["do"] = randn(n, H, D)
        return x
    if case["op"] == "norm":
        C = case["width"]
        of = torch.float32 if case["weights"] == "float32" else dtype
        x = {"x": randn(n, C, scale=1.5, shift=0.3), "w": randn(C, of=of, scale=0.2, shift=1.0)}
        if case["bias"]:
            x["b"] = randn(C, of=of, scale=0.2)
        if case["train"]:
            x["dy"] = randn(n, C)
        return x
    K, V = case["K"], case["classes"]
    x = {"x": randn(n, K), "w": randn(V, K, scale=1.5 * K ** -0.5)}
    if case["bias"]:
        x["b"] = randn(V, scale=0.5)
    # some classes are far more frequent than others
    u = torch.rand(n, device="cuda", generator=gen)
    t = (V * u ** 3).long().clamp_(max=V - 1)
    none = torch.rand(n, device="cuda", generator=gen) < case["ignored"]
    none[0] = False
    x["target"] = torch.where(none, -100, t)
    if case["train"]:   # binary16 trains with a scaled loss
        size = 65536.0 if dtype == torch.float16 and case["reduction"] == "mean" else 1.0
        x["dloss"] = (torch.full((), size, device="cuda") if case["reduction"] != "none" else
                      size * (0.5 + torch.rand(n, device="cuda", generator=gen)))
    return x


LEAVES = ("qkv", "q", "k", "v", "slopes", "x", "w", "b")


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["train"]:
        for name in LEAVES:
            if name in state:
                state[name].requires_grad_()
    if case["op"] == "attention":
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
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "norm": _own_norm, "loss": _own_loss}[op](state)
    with torch.no_grad():
        return {"attention": _plain_attention, "norm": _plain_norm, "loss": _plain_loss}[op](state)


def _step(state, out, name, leaves, grad):
    if not state["case"]["train"]:
        return {name: out}
    grads = torch.autograd.grad(out, [state[leaf] for leaf in leaves], state[grad])
    return {name: out.detach(), **{"d" + leaf: g for leaf, g in zip(leaves, grads)}}


def _own_attention(state):
    case, graph = state["case"], state["graph"]
    bias = {"cap": case["cap"] or None, "positions": state.get("positions"),
            "slopes": state.get("slopes")}
    if case["packed"]:
        leaves = ["qkv"]
        o = graph.edge_attention_packed(state["qkv"], D ** -0.5, **bias)
    else:
        leaves = ["q", "k", "v"]
        o = graph.edge_attention(state["q"], state["k"], state["v"], D ** -0.5, **bias)
    return _step(state, o, "o", leaves + (["slopes"] if case["dims"] else []), "do")


def _own_norm(state):
    from fused3s_amd import torch_ops
    y = torch_ops.layer_norm(state["x"], state["w"], state.get("b"), eps=1e-5)
    return _step(state, y, "y", [name for name in ("x", "w", "b") if name in state], "dy")


def _own_loss(state):
    from fused3s_amd import torch_ops
    loss = torch_ops.linear_cross_entropy(state["x"], state["w"], state["target"], state.get("b"),
                                          reduction=state["case"]["reduction"])
    return _step(state, loss, "loss", [name for name in ("x", "w", "b") if name in state], "dloss")


def _plain_attention(state):
    case = state["case"]
    n, H, dtype, scale, cap = (case["n"], case["heads"], TYPES[case["dtype"]], D ** -0.5,
                               case["cap"])
    rows, cols = state["rows"], state["cols"]
    if case["packed"]:
        q, k, v = state["qkv"].view(n, 3, H, D).float().unbind(1)
    else:
        q, k, v = (state[name].float() for name in ("q", "k", "v"))

    def by_row(index, values):
        out = torch.zeros(n, *values.shape[1:], device="cuda")
        return out.index_add_(0, index, values)

    s = (q[rows] * k[cols]).sum(-1) * scale
    if cap:
        t = torch.tanh(s / cap)
        s = cap * t
    if case["dims"]:
        dist = (state["positions"][rows] - state["positions"][cols]).square().sum(-1).sqrt()[:, None]
        s = s - state["slopes"] * dist
    top = torch.full((n, H), -math.inf, device="cuda")
    top.scatter_reduce_(0, rows[:, None].expand_as(s), s, "amax")
    p = torch.exp(s - top[rows])
    p = p / by_row(rows, p)[rows]
    out = {"o": by_row(rows, p[..., None] * v[cols]).to(dtype)}
    if not case["train"]:
        return out
    do = state["do"].float()
    g = (do[rows] * v[cols]).sum(-1)
    ds = p * (g - by_row(rows, p * g)[rows])
    if case["dims"]:
        dslopes = -(ds * dist).double().sum(0).float()
    if cap:
        ds = ds * (1 - t * t)
    ds = (ds * scale)[..., None]
    dq = by_row(rows, ds * k[cols]).to(dtype)
    dk = by_row(cols, ds * q[rows]).to(dtype)
    dv = by_row(cols, p[..., None] * do[rows]).to(dtype)
    if case["packed"]:
        out["dqkv"] = torch.stack([dq, dk, dv], 1).view(n, 3 * H * D)
    else:
        out.update(dq=dq, dk=dk, dv=dv)
    if case["dims"]:
        out["dslopes"] = dslopes
    return out


def _plain_norm(state):
    case = state["case"]
    dtype = TYPES[case["dtype"]]
    x, w = state["x"].float(), state["w"].float()
    x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
    h = x * r
    y = h * w
    if case["bias"]:
        y = y + state["b"].float()
    out = {"y": y.to(dtype)}
    if not case["train"]:
        return out
    dy = state["dy"].float()
    dh = dy * w
    out["dx"] = (r * (dh - dh.mean(-1, keepdim=True)
                      - h * (dh * h).mean(-1, keepdim=True))).to(dtype)
    out["dw"] = (dy * h).sum(0, dtype=torch.float64).to(state["w"].dtype)
    if case["bias"]:
        out["db"] = dy.sum(0, dtype=torch.float64).to(state["b"].dtype)
    return out


def _plain_loss(state):
    """Some rows at a time, so that the logits fit the memory."""
    case = state["case"]
    n, V, dtype, reduction = case["n"], case["classes"], TYPES[case["dtype"]], case["reduction"]
    x, w, target = state["x"], state["w"].float(), state["target"]
    b = state["b"].float() if case["bias"] else None
    counted = target != -100
    many = counted.sum()
    loss = torch.zeros(n, device="cuda")
    if case["train"]:
        g = state["dloss"].expand(n) * counted
        if reduction == "mean":
            g = g / many
        dx = torch.empty(n, case["K"], dtype=dtype, device="cuda")
        dw, db = torch.zeros_like(w), torch.zeros(V, device="cuda")
    per = max(1, (1 << 30) // V)
    for r0 in range(0, n, per):
        at = slice(r0, min(n, r0 + per))
        xf, rows = x[at].float(), torch.arange(at.stop - r0, device="cuda")
        z = xf @ w.t()
        if b is not None:
            z += b
        t = target[at].clamp(min=0)
        top = z.amax(1, keepdim=True)
        zt = z[rows, t]
        e = z.sub_(top).exp_()
        total = e.sum(1, keepdim=True)
        loss[at] = torch.where(counted[at], (top + torch.log(total))[:, 0] - zt, 0.0)
        if case["train"]:
            dz = e.mul_(g[at, None] / total)
            dz[rows, t] -= g[at]
            dx[at] = (dz @ w).to(dtype)
            dw += dz.t() @ xf
            db += dz.sum(0)
    if reduction != "none":
        loss = loss.double().sum()
        loss = (loss / many if reduction == "mean" else loss).float()
    out = {"loss": loss}
    if case["train"]:
        out.update(dx=dx, dw=dw.to(dtype))
        if b is not None:
            out["db"] = db.to(dtype)
    return out


# --------------------------------------------------------------------- work

def work(case):
    n = case["n"]
    size = 4.0 if case["dtype"] == "float32" else 2.0
    if case["op"] == "attention":
        H = case["heads"]
        edges = n * (case["degree"] + (1 if case["loops"] else 0))
        lists = 4.0 * (edges + n) + 4.0 * n * case["dims"]
        feature = 2.0 * n * H * D
        if case["train"]:   # q, k, v, do and o, dq, dk, dv; six products of D per edge and head
            return {"bytes": 8 * feature + lists, "flops": 12.0 * D * H * edges}
        return {"bytes": 4 * feature + lists, "flops": 4.0 * D * H * edges}
    if case["op"] == "norm":
        C = case["width"]
        weights = C * (4.0 if case["weights"] == "float32" else size) * (2 if case["bias"] else 1)
        if case["train"]:
            return {"bytes": 4 * size * n * C + 2 * weights, "flops": 20.0 * n * C}
        return {"bytes": 2 * size * n * C + weights, "flops": 8.0 * n * C}
    K, V = case["K"], case["classes"]
    read = 2.0 * n * K + 2.0 * V * K + 8.0 * n + (2.0 * V if case["bias"] else 0)
    if case["train"]:
        return {"bytes": 2 * read - 8.0 * n, "flops": 6.0 * n * K * V}
    return {"bytes": read, "flops": 2.0 * n * K * V}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    x = _inputs(case, seed)
    return {"attention": _exact_attention, "norm": _exact_norm, "loss": _exact_loss}[case["op"]](
        case, x)


def _exact_attention(case, x):
    """A few rows at a time; gradients by differentiation of the forward pass."""
    n, H, train, cap = case["n"], case["heads"], case["train"], case["cap"]
    if case["packed"]:
        q, k, v = (t.double() for t in x["qkv"].view(n, 3, H, D).unbind(1))
    else:
        q, k, v = (x[name].double() for name in ("q", "k", "v"))
    slopes = x["slopes"].double() if case["dims"] else torch.zeros(H, device="cuda").double()
    o = torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
    grads = [torch.zeros_like(t) for t in (q, k, v, slopes)] if train else []
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
                a = [q[r0:r1].clone(), k[cols], v[cols], slopes.clone()]
                if train:
                    a = [t.requires_grad_() for t in a]
                s = torch.einsum("ehd,ehd->eh", a[0][row], a[1]) * D ** -0.5
                if cap:
                    s = torch.tanh(s / cap) * cap
                if case["dims"]:
                    where = x["positions"].double()
                    s = s - torch.linalg.norm(where[r0 + row] - where[cols], dim=1)[:, None] * a[3]
                e = torch.exp(s - s.detach().max())   # (far from under- and overflow here)
                total = torch.zeros(r1 - r0, H, dtype=e.dtype, device="cuda").index_add(0, row, e)
                weighted = (e / total[row])[..., None] * a[2]
                out = torch.zeros(r1 - r0, H, D, dtype=weighted.dtype, device="cuda")
                out = out.index_add(0, row, weighted)
            o[r0:r1] = out.detach()
            if train:
                g = torch.autograd.grad(out, a, x["do"][r0:r1].double(), allow_unused=True)
                grads[0][r0:r1] = g[0]
                grads[1].index_add_(0, cols, g[1])
                grads[2].index_add_(0, cols, g[2])
                if case["dims"]:
                    grads[3] += g[3]
        r0 = r1
    out = {"o": o}
    if train:
        dq, dk, dv, dslopes = grads
        if case["packed"]:
            out["dqkv"] = torch.cat([t.reshape(n, H * D) for t in (dq, dk, dv)], 1)
        else:
            out.update(dq=dq, dk=dk, dv=dv)
        if case["dims"]:
            out["dslopes"] = dslopes
    return out


def _exact_norm(case, x):
    a = {name: x[name].double().requires_grad_(case["train"]) for name in ("x", "w", "b")
         if name in x}
    y = torch.nn.functional.layer_norm(a["x"], (case["width"],), a["w"], a.get("b"), 1e-5)
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, list(a.values()), x["dy"].double())
    return {"y": y.detach(), **{"d" + name: g for name, g in zip(a, grads)}}


def _exact_loss(case, x):
    """Some rows at a time; torch's own loss and its gradient in 64 bits."""
    n, train, reduction = case["n"], case["train"], case["reduction"]
    w = x["w"].double().requires_grad_(train)
    b = x["b"].double().requires_grad_(train) if case["bias"] else None
    many = int((x["target"] != -100).sum())
    losses, dx, dw, db = [], [], torch.zeros_like(w), None if b is None else torch.zeros_like(b)
    per = max(1, (1 << 28) // case["classes"])
    for r0 in range(0, n, per):
        xr = x["x"][r0:r0 + per].double().requires_grad_(train)
        loss = torch.nn.functional.cross_entropy(
            torch.nn.functional.linear(xr, w, b), x["target"][r0:r0 + per], reduction="none")
        losses.append(loss.detach())
        if train:
            up = x["dloss"].double().expand(n)[r0:r0 + per]
            up = up / many if reduction == "mean" else up
            g = torch.autograd.grad(loss, [xr, w] + ([] if b is None else [b]), up)
            dx.append(g[0])
            dw += g[1]
            if b is not None:
                db += g[2]
    loss = torch.cat(losses)
    if reduction != "none":
        loss = loss.sum() / (many if reduction == "mean" else 1)
    out = {"loss": loss}
    if train:
        out.update(dx=torch.cat(dx), dw=dw.detach())
        if b is not None:
            out["db"] = db.detach()
    return out
