"""Rows moved by ids, as cases that can be timed: embedding lookup with scaling and its gradient by
sorted ids (dense and sparse), and rows sorted by expert (or node type), brought back with weights
applied, and the gradients of both.

A case is a dict of plain values; `listed()` gives the fixed ones, `draw(rng)` one more of the same
ranges.  `run(state)` is one pass: in its plain form, elementary torch operations in 32 bits, or,
with `own` set, through this package.
An id outside its range stands for no row: the -1 of a walker that has died, of padding, of a
choice that found no room.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # the next token of a few sequences that are being generated: scaled rows, latency alone
        {"name": "lookup_4", "kind": "lookup", "rows": 32768, "dim": 2048, "ids": 4, "type": "bf16", "bits": 64,
         "scaled": True, "spread": "skewed", "missing": 0.0},
        # the features of a super-batch's frontier, fetched from a node table that no cache holds
        {"name": "lookup_frontier_600k", "kind": "lookup", "rows": 2_450_000, "dim": 64, "ids": 600_000, "type": "f32",
         "bits": 32, "scaled": False, "spread": "even", "missing": 0.0},
        # a small table learned with few ids a step, odd width: nothing but launches
        {"name": "train_37", "kind": "train", "rows": 1001, "dim": 97, "ids": 37, "type": "f16", "bits": 64,
         "scaled": True, "spread": "skewed", "missing": 0.1},
        # token embeddings in training: frequent tokens many times, padding, gradient of the whole table
        {"name": "train_tokens_16k", "kind": "train", "rows": 32768, "dim": 1024, "ids": 16384, "type": "bf16", "bits": 64,
         "scaled": True, "spread": "skewed", "missing": 0.05},
        # node embeddings of a small graph, whose hubs are in most of the neighbourhoods
        {"name": "train_hubs_400k", "kind": "train", "rows": 1 << 17, "dim": 64, "ids": 400_000, "type": "f32",
         "bits": 32, "scaled": False, "spread": "hubs", "missing": 0.0},
        # skip-gram embeddings on walks over a large graph, some of which end early: gradient of the rows met
        {"name": "train_walks_810k", "kind": "train_sparse", "rows": 4_000_000, "dim": 64, "ids": 810_000, "type": "f32",
         "bits": 32, "scaled": False, "spread": "skewed", "missing": 0.1},
        # a few tokens that are being generated, sent to their experts
        {"name": "dispatch_4x4", "kind": "dispatch", "tokens": 4, "choices": 4, "experts": 64, "dim": 2048,
         "type": "bf16", "bits": 64, "missing": 0.0},
        # the frontier of a heterogeneous graph, its rows brought together by node type
        {"name": "dispatch_types_600k", "kind": "dispatch", "tokens": 600_000, "choices": 1, "experts": 5, "dim": 64,
         "type": "f32", "bits": 32, "missing": 0.0},
        # a long batch of tokens, eight experts each
        {"name": "dispatch_16k_x8", "kind": "dispatch", "tokens": 16384, "choices": 8, "experts": 64, "dim": 2048,
         "type": "bf16", "bits": 64, "missing": 0.0},
        # the same in training with many small experts, some of them full, odd sizes, and its gradient
        {"name": "dispatch_train_5k_x6", "kind": "dispatch_train", "tokens": 5003, "choices": 6, "experts": 160,
         "dim": 1001, "type": "f16", "bits": 64, "missing": 0.05},
        # the experts' results of a few generated tokens, added up by their weights
        {"name": "combine_3x8", "kind": "combine", "tokens": 3, "choices": 8, "experts": 64, "dim": 4096, "type": "f16",
         "bits": 64, "missing": 0.0, "weights": "f32"},
        # few large experts in training: weighted sums, gradients of results and weights
        {"name": "combine_train_8k_x2", "kind": "combine_train", "tokens": 8192, "choices": 2, "experts": 8,
         "dim": 4096, "type": "bf16", "bits": 64, "missing": 0.02, "weights": "f32"},
    ]


_MOST_BYTES = 500_000_000  # of a drawn case; the largest listed one has 839 MB


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["lookup", "train", "train_sparse", "dispatch", "dispatch_train", "combine", "combine_train"])
    case = {"kind": kind, "type": rng.choice(["f32", "bf16", "f16"]), "bits": rng.choice([32, 64]),
            "missing": rng.choice([0.0, 0.02, 0.1, 0.5]), "dim": _between(rng, 8, 4096)}
    if kind in ("lookup", "train", "train_sparse"):
        case.update(rows=_between(rng, 100, 4_000_000), ids=_between(rng, 1, 1_000_000), scaled=rng.random() < 0.5,
                    spread=rng.choice(["even", "skewed", "hubs"]))
        while 4 * case["rows"] * case["dim"] > 1 << 30:
            case["rows"] = max(100, case["rows"] * 2 // 3)
        name = "ids"
    else:
        experts = _between(rng, 2, 256)
        case.update(experts=experts, choices=rng.randint(1, min(8, experts)), tokens=_between(rng, 1, 600_000))
        if kind in ("combine", "combine_train"):
            case["weights"] = rng.choice(["none", "f32", case["type"]])
        name = "tokens"
    while work(case)["bytes"] > _MOST_BYTES:
        if case[name] > 64:
            case[name] = case[name] * 2 // 3
        else:
            case["dim"] = max(8, case["dim"] * 2 // 3)
            case["rows"] = max(100, case.get("rows", 0) * 2 // 3)
    return case


def _row_ids(case, gen):
    n, rows = case["ids"], case["rows"]
    # how often the r-th most frequent row occurs is a case's own, so that as many rows are met whatever
    # the seed; which rows those are, and in which order they come, is the seed's
    own_gen = torch.Generator(device=DEVICE)
    own_gen.manual_seed(n)
    u = torch.rand(n, generator=own_gen, device=DEVICE, dtype=torch.float64)
    if case["spread"] == "even":
        ids = u * rows
    elif case["spread"] == "skewed":  # the r-th most frequent about 1 / r times as often as the first
        ids = (math.log(rows) * u).exp() - 1
    else:  # hubs: a tenth of all on four rows
        ids = torch.where(u < 0.1, u * 40, (u - 0.1) / 0.9 * rows)
    start = torch.randint(rows, (1,), generator=gen, device=DEVICE)
    ids = (ids.long().clamp(0, rows - 1) + start) % rows
    if case["missing"] > 0:
        gone = torch.rand(n, generator=own_gen, device=DEVICE) < case["missing"]
        ids = torch.where(gone, -1, ids)
    ids = ids[torch.randperm(n, generator=gen, device=DEVICE)]
    return ids.to(torch.int32 if case["bits"] == 32 else torch.int64)


def _choices(case, gen):
    """Every token's experts, no two the same, some experts more in demand than others, and how much
    each of them is to count."""
    T, K, E = case["tokens"], case["choices"], case["experts"]
    liking = torch.randn(E, generator=gen, device=DEVICE)
    score, chosen = [], []
    for first in range(0, T, 1 << 16):
        s = torch.randn(min(1 << 16, T - first), E, generator=gen, device=DEVICE) + liking
        top = s.topk(K, dim=1)
        score.append(top.values)
        chosen.append(top.indices)
    score, chosen = torch.cat(score), torch.cat(chosen)
    if case["missing"] > 0:
        gone = torch.rand(T, K, generator=gen, device=DEVICE) < case["missing"]
        chosen = torch.where(gone, -1, chosen)
    return chosen.to(torch.int32 if case["bits"] == 32 else torch.int64), score.softmax(dim=1)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    kind, dt, D = case["kind"], _TYPES[case["type"]], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE).to(dt)

    state = {"kind": kind, "dtype": dt}
    if kind in ("lookup", "train", "train_sparse"):
        state["ids"] = _row_ids(case, gen)
        state["scale"] = math.sqrt(D) if case["scaled"] else 1.0
        state["table"] = normal(case["rows"], D)
        if kind != "lookup":
            state["grad"] = normal(case["ids"], D)
            state["table"].requires_grad_(True)
        return state
    chosen, weights = _choices(case, gen)
    T, K, E = case["tokens"], case["choices"], case["experts"]
    if kind in ("dispatch", "dispatch_train"):
        state.update(chosen=chosen, experts=E, x=normal(T, D))
        if kind == "dispatch_train":
            state["x"].requires_grad_(True)
            state["grad"] = normal(T * K, D)
        return state
    # the experts' results are there, and the order that brought their rows together
    state.update(zip(("order", "place", "offsets"), _sorted(chosen, E)))
    state["y"] = normal(T * K, D)
    state["weights"] = None if case["weights"] == "none" else weights.to(_TYPES[case["weights"]])
    if kind == "combine_train":
        state["grad"] = normal(T, D)
        state["y"].requires_grad_(True)
        if state["weights"] is not None:
            state["weights"].requires_grad_(True)
    return state


# ------------------------------------------------------------------ plain ----
def _found(table, ids, scale):
    """Scaled rows of the table by id, zeros where there is none."""
    ids = ids.long()
    there = (ids >= 0) & (ids < table.shape[0])
    rows = table[torch.where(there, ids, 0)].float() * scale
    return torch.where(there[:, None], rows, 0.0).to(table.dtype)


def _summed(rows, grad, ids, scale, dtype):
    """rows x dim: the scaled sums of the gradients by id; of an id that occurs often, by pieces of 256 first (one
    chain of tens of thousands of 32-bit sums loses digits, and sums in 64 bits take a hundred times as long here)."""
    ids = ids.long()
    key, order = torch.sort(torch.where((ids >= 0) & (ids < rows), ids, rows), stable=True)
    in_run = torch.arange(key.numel(), device=key.device) - torch.searchsorted(key, key)
    piece = (in_run % 256 == 0).cumsum(0) - 1
    pieces = int(piece[-1]) + 1
    part = torch.zeros(pieces, grad.shape[1], device=grad.device).index_add_(0, piece, grad[order].float())
    of = torch.empty(pieces, dtype=torch.int64, device=key.device)
    of[piece] = key
    out = torch.zeros(rows + 1, grad.shape[1], device=grad.device).index_add_(0, of, part)
    return (out[:rows] * scale).to(dtype)


def _sorted(chosen, experts):
    """(order, place, offsets): the items (token, choice) by expert."""
    flat = chosen.reshape(-1).long()
    there = (flat >= 0) & (flat < experts)
    by_expert, order = torch.sort(torch.where(there, flat, experts), stable=True)
    offsets = torch.searchsorted(by_expert, torch.arange(experts + 1, device=flat.device))
    at = torch.arange(flat.numel(), device=flat.device)
    place = torch.empty_like(order)
    place[order] = at
    place = torch.where(there, place, -1).int()
    order = torch.where(at < offsets[-1], order, -1).int()
    return order, place.view(chosen.shape), offsets


def _combined(y, place, weights):
    out = torch.zeros(place.shape[0], y.shape[1], device=y.device)
    for k in range(place.shape[1]):
        at = place[:, k].long()
        rows = y[at.clamp(min=0)].float()
        if weights is not None:
            rows = rows * weights[:, k, None].float()
        out += torch.where(at[:, None] >= 0, rows, 0.0)
    return out.to(y.dtype)


def _plain(s):
    kind = s["kind"]
    with torch.no_grad():
        if kind == "lookup":
            return _found(s["table"], s["ids"], s["scale"])
        if kind == "train":
            out = _found(s["table"], s["ids"], s["scale"])
            return out, _summed(s["table"].shape[0], s["grad"], s["ids"], s["scale"], s["dtype"])
        if kind == "train_sparse":
            out = _found(s["table"], s["ids"], s["scale"])
            ids = s["ids"].long()
            there = (ids >= 0) & (ids < s["table"].shape[0])
            met, which = torch.unique(ids[there], return_inverse=True)
            return out, met, _summed(met.numel(), s["grad"][there], which, s["scale"], s["dtype"])
        if kind in ("dispatch", "dispatch_train"):
            x, K = s["x"], s["chosen"].shape[1]
            order, place, offsets = _sorted(s["chosen"], s["experts"])
            rows = x[order.clamp(min=0).long() // K]
            rows = torch.where(order[:, None] >= 0, rows, torch.zeros((), dtype=x.dtype, device=x.device))
            if kind == "dispatch":
                return rows, order, place, offsets
            return rows, order, place, offsets, _combined(s["grad"], place, None)
        y, place, weights = s["y"], s["place"], s["weights"]
        out = _combined(y, place, weights)
        if kind == "combine":
            return out
        order, dout, K = s["order"].long(), s["grad"].float(), place.shape[1]
        of = order.clamp(min=0)
        dy = dout[of // K]
        if weights is not None:
            dy = dy * weights.reshape(-1)[of, None].float()
        dy = torch.where(order[:, None] >= 0, dy, 0.0).to(y.dtype)
        if weights is None:
            return out, dy
        dw = []
        for k in range(K):
            at = place[:, k].long()
            dots = (y[at.clamp(min=0)].float() * dout).sum(1)
            dw.append(torch.where(at >= 0, dots, 0.0))
        return out, dy, torch.stack(dw, 1).to(weights.dtype)


# -------------------------------------------------------------------- own ----
def _own(s):
    import graph_sampling_amd as gs
    kind = s["kind"]
    if kind == "lookup":
        return gs.ops.embedding(s["table"], s["ids"], s["scale"])
    if kind == "train":
        out = gs.ops.embedding(s["table"], s["ids"], s["scale"])
        grad, = torch.autograd.grad(out, s["table"], s["grad"])
        return out.detach(), grad
    if kind == "train_sparse":
        out = gs.ops.embedding(s["table"], s["ids"], s["scale"], sparse_grad=True)
        grad, = torch.autograd.grad(out, s["table"], s["grad"])
        return out.detach(), grad.indices()[0], grad.values()
    if kind == "dispatch":
        rows, (order, place, offsets) = gs.ops.expert_dispatch(s["x"], s["chosen"], s["experts"])
        return rows, order, place, offsets
    if kind == "dispatch_train":
        rows, (order, place, offsets) = gs.ops.expert_dispatch(s["x"], s["chosen"], s["experts"])
        grad, = torch.autograd.grad(rows, s["x"], s["grad"])
        return rows.detach(), order, place, offsets, grad
    order = gs.ops.ExpertOrder(s["order"], s["place"], s["offsets"])
    out = gs.ops.expert_combine(s["y"], order, s["weights"])
    if kind == "combine":
        return out
    wanted = [t for t in (s["y"], s["weights"]) if t is not None]
    return (out.detach(),) + torch.autograd.grad(out, wanted, s["grad"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    es, b, D = _TYPES[case["type"]].itemsize, case["bits"] // 8, case["dim"]
    kind = case["kind"]
    if kind in ("lookup", "train", "train_sparse"):
        N, V = case["ids"], case["rows"]
        met = min(N, V)
        moved = N * b + (met + N) * D * es
        if kind == "lookup":
            return {"bytes": moved, "flops": N * D}
        written = V * D * es if kind == "train" else met * (8 + D * es)
        return {"bytes": moved + N * D * es + written, "flops": 2 * N * D}
    T, E = case["tokens"], case["experts"]
    n = T * case["choices"]
    if kind in ("dispatch", "dispatch_train"):
        moved = n * b + (T + n) * D * es + n * 8 + (E + 1) * 8
        if kind == "dispatch":
            return {"bytes": moved, "flops": 0}
        return {"bytes": moved + (T + n) * D * es, "flops": n * D}
    wb = 0 if case["weights"] == "none" else _TYPES[case["weights"]].itemsize
    moved = (T + n) * D * es + n * (4 + wb)
    if kind == "combine":
        return {"bytes": moved, "flops": 2 * n * D}
    return {"bytes": moved + (T + n) * D * es + n * wb, "flops": 5 * n * D}


# ------------------------------------------------------------------ exact ----
def _host(t):
    t = t.detach()
    return (t.double() if t.is_floating_point() else t.long()).cpu().numpy()


def exact(case, seed):
    """What `run` returns, in 64 bits on the host: gradients by sorted runs, experts one by one."""
    s = prepare(case, seed)
    kind, D = case["kind"], case["dim"]
    if kind in ("lookup", "train", "train_sparse"):
        ids, V, scale = _host(s["ids"]), case["rows"], s["scale"]
        rows = np.flatnonzero((ids >= 0) & (ids < V))
        out = np.zeros((ids.size, D))
        out[rows] = _host(s["table"][torch.from_numpy(ids[rows]).to(DEVICE)]) * scale
        if kind == "lookup":
            return out
        by_id = rows[np.argsort(ids[rows], kind="stable")]
        keys = ids[by_id]
        heads = np.flatnonzero(np.concatenate([[True], keys[1:] != keys[:-1]])) if keys.size else keys
        sums = np.zeros((heads.size, D))
        if keys.size:
            sums = np.add.reduceat(_host(s["grad"])[by_id], heads, axis=0) * scale
        if kind == "train_sparse":
            return out, keys[heads], sums
        grad = np.zeros((V, D))
        grad[keys[heads]] = sums
        return out, grad
    if kind in ("dispatch", "dispatch_train"):
        E, K, x = case["experts"], case["choices"], _host(s["x"])
        flat = _host(s["chosen"]).reshape(-1)
        of = [np.flatnonzero(flat == e) for e in range(E)]
        offsets = np.cumsum([0] + [len(items) for items in of])
        live = np.concatenate(of)
        order, place = np.full(flat.size, -1), np.full(flat.size, -1)
        order[:live.size] = live
        place[live] = np.arange(live.size)
        rows = np.zeros((flat.size, D))
        rows[:live.size] = x[live // K]
        if kind == "dispatch":
            return rows, order, place.reshape(-1, K), offsets
        dx = np.zeros_like(x)
        drows = _host(s["grad"])
        for k in range(K):
            at = place[k::K]
            dx[at >= 0] += drows[at[at >= 0]]
        return rows, order, place.reshape(-1, K), offsets, dx
    y, order, K = _host(s["y"]), _host(s["order"]), case["choices"]
    live = np.flatnonzero(order >= 0)
    item = order[live]
    weights = np.ones(order.size) if s["weights"] is None else _host(s["weights"]).reshape(-1)
    by_item = np.zeros((order.size, D))
    by_item[item] = y[live] * weights[item, None]
    out = by_item.reshape(-1, K, D).sum(axis=1)
    if kind == "combine":
        return out
    dout = _host(s["grad"])
    dy = np.zeros_like(y)
    dy[live] = dout[item // K] * weights[item, None]
    if s["weights"] is None:
        return out, dy
    dw = np.zeros(order.size)
    dw[item] = np.einsum("nd,nd->n", dout[item // K], y[live])
    return out, dy, dw.reshape(-1, K)
