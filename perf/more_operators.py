"""The work of experts between their rows' going out and coming back, as cases that can be timed: the choice
of experts from a router's logits, the products of rows sorted by expert (or node type) with each
expert's matrix, dropout by counter-based draws, and the gradients of all three.

A case is a dict of plain values; `listed()` gives the fixed ones, `draw(rng)` one more of the same
ranges.  `run(state)` is one pass: in its plain form, elementary torch operations in 32 bits, or,
with `own` set, through this package.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a few tokens that are being generated, four experts each: every row meets a matrix of its own
        {"name": "product_4x4_of_64", "kind": "product", "items": 16, "experts": 64, "inner": 2048, "outer": 1024,
         "type": "bf16", "transposed": False, "missing": 0.0},
        # the same with matrices kept as a linear layer keeps them, [outer, inner]
        {"name": "product_3x8_of_64", "kind": "product", "items": 24, "experts": 64, "inner": 1024, "outer": 4096,
         "type": "f16", "transposed": True, "missing": 0.0},
        # a long batch of tokens, eight experts each
        {"name": "product_16k_x8", "kind": "product", "items": 131072, "experts": 64, "inner": 2048, "outer": 1024,
         "type": "bf16", "transposed": False, "missing": 0.0},
        # the frontier of a heterogeneous graph, a matrix per node type, in training
        {"name": "product_types_600k", "kind": "product_train", "items": 600_000, "experts": 5, "inner": 64,
         "outer": 128, "type": "f32", "transposed": False, "missing": 0.0},
        # many small experts in training, odd sizes, some choices without a place
        {"name": "product_train_5k_x6", "kind": "product_train", "items": 30018, "experts": 160, "inner": 1001,
         "outer": 333, "type": "f16", "transposed": False, "missing": 0.05},
        # few large experts in training
        {"name": "product_train_8k_x2", "kind": "product_train", "items": 16384, "experts": 8, "inner": 4096,
         "outer": 2048, "type": "bf16", "transposed": False, "missing": 0.02},
        # the router of the few tokens: latency alone
        {"name": "choose_4x4_of_64", "kind": "choose", "tokens": 4, "choices": 4, "experts": 64, "type": "bf16",
         "normalize": True, "masked": 0.0},
        # the router of a long batch in training, shares of all experts' sum
        {"name": "choose_train_16k_x8", "kind": "choose_train", "tokens": 16384, "choices": 8, "experts": 256,
         "type": "f32", "normalize": False, "masked": 0.0},
        # many groups of tokens at once, experts that are switched off for some of them, odd sizes
        {"name": "choose_train_100k_x6", "kind": "choose_train", "tokens": 100_003, "choices": 6, "experts": 160,
         "type": "f16", "normalize": True, "masked": 0.1},
        # a small layer's features, odd width: nothing but a launch
        {"name": "dropout_37", "kind": "dropout", "rows": 37, "dim": 97, "type": "f16", "p": 0.1, "residual": False},
        # the features of a super-batch's frontier in training
        {"name": "dropout_train_600k", "kind": "dropout_train", "rows": 600_000, "dim": 64, "type": "f32", "p": 0.5,
         "residual": False},
        # what a layer's experts answered, added to the tokens it began with, in training
        {"name": "dropout_train_16k", "kind": "dropout_train", "rows": 16384, "dim": 2048, "type": "bf16", "p": 0.1,
         "residual": True},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(lo * (hi / lo) ** rng.random())))


_MOST_BYTES = 600_000_000    # of a drawn case; the largest listed one has 1.07 GB
_MOST_FLOPS = 400e9          # the largest listed one has 809 GFLOP
_MOST_WEIGHTS = 60_000_000   # values of all matrices


def draw(rng):
    kind = rng.choice(["product", "product_train", "product", "product_train", "choose", "choose_train", "dropout",
                       "dropout_train"])
    case = {"kind": kind, "type": rng.choice(["f32", "bf16", "f16"])}
    if kind in ("product", "product_train"):
        case.update(experts=_between(rng, 2, 256), items=_between(rng, 1, 600_000), inner=_between(rng, 8, 4096),
                    outer=_between(rng, 8, 4096), transposed=rng.random() < 0.5, missing=rng.choice([0.0, 0.02, 0.1, 0.5]))
        if rng.random() < 0.5:  # widths are multiples of 16 more often than not
            case.update(inner=(case["inner"] + 15) // 16 * 16, outer=(case["outer"] + 15) // 16 * 16)
        while case["experts"] * case["inner"] * case["outer"] > _MOST_WEIGHTS:
            case["experts"] = max(2, case["experts"] * 2 // 3)
        most_flops = _MOST_FLOPS / 8 if case["type"] == "f32" else _MOST_FLOPS
        name = "items"
    elif kind in ("choose", "choose_train"):
        experts = _between(rng, 2, 512)
        case.update(tokens=_between(rng, 1, 600_000), experts=experts, choices=rng.randint(1, min(8, experts)),
                    normalize=rng.random() < 0.5, masked=rng.choice([0.0, 0.1, 0.9]))
        most_flops, name = _MOST_FLOPS, "tokens"
    else:
        case.update(rows=_between(rng, 1, 600_000), dim=_between(rng, 1, 4096), p=rng.choice([0.1, 0.25, 0.5, 0.9]),
                    residual=rng.random() < 0.5)
        most_flops, name = _MOST_FLOPS, "rows"
    while work(case)["bytes"] > _MOST_BYTES or work(case)["flops"] > most_flops:
        if case[name] <= 1:
            break
        case[name] = max(1, case[name] * 2 // 3)
    return case


def _loads(case):
    """How many rows each expert has (and, last, how many items have no expert): some experts are more in
    demand than others; a case's own, whatever the seed."""
    rng = np.random.default_rng([case["items"], case["experts"]])
    share = np.exp(0.5 * rng.standard_normal(case["experts"]))
    share *= (1 - case["missing"]) / share.sum()
    return rng.multinomial(case["items"], np.append(share, max(0.0, 1 - share.sum())))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    kind, dt = case["kind"], _TYPES[case["type"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * by).to(dt)

    state = {"kind": kind, "dtype": dt, "train": kind.endswith("_train")}
    if kind in ("product", "product_train"):
        n, E, D, F = case["items"], case["experts"], case["inner"], case["outer"]
        loads = _loads(case)
        loads[:E] = loads[:E][torch.randperm(E, generator=gen, device=DEVICE).cpu().numpy()]
        live = int(loads[:E].sum())
        # which item went where does not matter to the products; the order is one that a sort could have left
        order = torch.randperm(n, generator=gen, device=DEVICE)
        place = torch.empty_like(order)
        place[order] = torch.arange(n, device=DEVICE)
        state["place"] = torch.where(place < live, place, -1).int()
        state["order"] = torch.where(torch.arange(n, device=DEVICE) < live, order, -1).int()
        state["offsets"] = torch.from_numpy(np.append(0, np.cumsum(loads[:E]))).to(DEVICE)
        state["rows"] = normal(n, D)
        state["rows"][live:] = 0
        if case["transposed"]:
            state["weight"] = normal(E, F, D, by=D ** -0.5).transpose(1, 2)
        else:
            state["weight"] = normal(E, D, F, by=D ** -0.5)
        if state["train"]:
            state["rows"].requires_grad_(True)
            state["weight"] = state["weight"].detach().requires_grad_(True)
            state["grad"] = normal(n, F)
    elif kind in ("choose", "choose_train"):
        T, E = case["tokens"], case["experts"]
        liking = torch.randn(E, generator=gen, device=DEVICE)
        logits = torch.randn(T, E, generator=gen, device=DEVICE) + liking
        if case["masked"] > 0:
            off = torch.rand(T, E, generator=gen, device=DEVICE) < case["masked"]
            logits = torch.where(off, -math.inf, logits)
        state.update(logits=logits.to(dt), choices=case["choices"], normalize=case["normalize"])
        if state["train"]:
            state["logits"].requires_grad_(True)
            state["grad"] = torch.randn(T, case["choices"], generator=gen, device=DEVICE)
    else:
        shape = case["rows"], case["dim"]
        state.update(x=normal(*shape), p=case["p"], residual=normal(*shape) if case["residual"] else None,
                     seed=int(torch.randint(1 << 62, (1,), generator=gen, device=DEVICE)))
        if state["train"]:
            state["x"].requires_grad_(True)
            if case["residual"]:
                state["residual"].requires_grad_(True)
            state["grad"] = normal(*shape)
    return state


# ------------------------------------------------------------------ plain ----
def _products(s):
    """rows of expert e times its matrix, zeros behind the last; with the gradients of both in training."""
    rows, weight, at = s["rows"], s["weight"], s["offsets"].tolist()
    out = torch.zeros(rows.shape[0], weight.shape[2], dtype=s["dtype"], device=rows.device)
    if s["train"]:
        d_rows, d_weight = torch.zeros_like(rows), torch.zeros_like(weight)
    for e in range(weight.shape[0]):
        if at[e] == at[e + 1]:
            continue
        x, w = rows[at[e]:at[e + 1]].float(), weight[e].float()
        out[at[e]:at[e + 1]] = (x @ w).to(s["dtype"])
        if s["train"]:
            g = s["grad"][at[e]:at[e + 1]].float()
            d_rows[at[e]:at[e + 1]] = (g @ w.t()).to(s["dtype"])
            d_weight[e] = (x.t() @ g).to(s["dtype"])
    return (out, d_rows, d_weight) if s["train"] else out


def _choose(s):
    logits, K = s["logits"].float(), s["choices"]
    top, experts = torch.sort(logits, dim=1, descending=True, stable=True)
    top, experts = top[:, :K], experts[:, :K]
    there = top > -math.inf
    most = torch.where(there[:, :1], top[:, :1], 0.0)
    share = torch.exp(top - most)
    total = share.sum(1, keepdim=True) if s["normalize"] else torch.exp(logits - most).sum(1, keepdim=True)
    weights = torch.where(there, share / total, 0.0)
    out = torch.where(there, experts, -1).int(), weights
    if not s["train"]:
        return out
    dot = (weights * s["grad"]).sum(1, keepdim=True)
    if s["normalize"]:
        d_logits = torch.zeros_like(logits)
    else:
        d_logits = torch.where(there[:, :1], -torch.exp(logits - most) / total * dot, 0.0)
        dot = torch.zeros_like(dot)
    d_logits.scatter_add_(1, experts, weights * (s["grad"] - dot))
    return out + (d_logits.to(s["dtype"]),)


def _draws(seed, n, device):
    """A 32-bit number each for positions 0 .. n - 1: word i % 4 of Philox4x32-10's block i / 4 under the
    key `seed` (Salmon et al., SC'11), the block's other counter words 0, 0 and 6."""
    low = 0xFFFFFFFF
    c0 = torch.arange((n + 3) // 4, device=device)
    c3 = ((c0 >> 32) << 8) | 6
    c0, c1, c2 = c0 & low, torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (64 bits, the sign bit as any other)
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]


def _dropped(s):
    x = s["x"]
    kept = _draws(s["seed"], x.numel(), x.device).view(x.shape) >= int(s["p"] * 2 ** 32)
    out = torch.where(kept, x.float() / (1 - s["p"]), 0.0)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    out = out.to(s["dtype"])
    if not s["train"]:
        return out
    dx = torch.where(kept, s["grad"].float() / (1 - s["p"]), 0.0).to(s["dtype"])
    return (out, dx) if s["residual"] is None else (out, dx, s["grad"])


def _plain(s):
    with torch.no_grad():
        if s["kind"].startswith("product"):
            return _products(s)
        return _choose(s) if s["kind"].startswith("choose") else _dropped(s)


# -------------------------------------------------------------------- own ----
def _own(s):
    import graph_sampling_amd as gs
    if s["kind"].startswith("product"):
        order = gs.ops.ExpertOrder(s["order"], s["place"], s["offsets"])
        out = gs.ops.expert_matmul(s["rows"], order, s["weight"])
        leaves = (s["rows"], s["weight"])
        before = ()
    elif s["kind"].startswith("choose"):
        experts, out = gs.ops.expert_choose(s["logits"], s["choices"], s["normalize"])
        leaves = (s["logits"],)
        before = (experts,)
    else:
        out = gs.ops.dropout(s["x"], s["p"], s["seed"], s["residual"])
        leaves = (s["x"],) if s["residual"] is None else (s["x"], s["residual"])
        before = ()
    if not s["train"]:
        return before + (out,) if before else out
    return before + (out.detach(),) + torch.autograd.grad(out, leaves, s["grad"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    es, kind = _TYPES[case["type"]].itemsize, case["kind"]
    if kind in ("product", "product_train"):
        n, E, D, F = case["items"], case["experts"], case["inner"], case["outer"]
        loads = _loads(case)
        live, met = int(loads[:E].sum()), int((loads[:E] > 0).sum())
        once = (live * D + met * D * F + n * F) * es + (E + 1) * 8
        if kind == "product":
            return {"bytes": once, "flops": 2 * live * D * F}
        return {"bytes": once + (live * F + n * D + E * D * F) * es, "flops": 6 * live * D * F}
    if kind in ("choose", "choose_train"):
        T, E, K = case["tokens"], case["experts"], case["choices"]
        moved, flops = T * (E * es + K * 8), T * E * 2
        if kind == "choose":
            return {"bytes": moved, "flops": flops}
        return {"bytes": moved + T * (E * es + K * 4), "flops": 3 * flops}
    n = case["rows"] * case["dim"]
    moved = n * es * (3 if case["residual"] else 2)
    if kind == "dropout":
        return {"bytes": moved, "flops": 2 * n}
    return {"bytes": moved + 2 * n * es, "flops": 3 * n}


# ------------------------------------------------------------------ exact ----
def _exact_products(case, s):
    """In 64 bits, a piece of at most 64 k rows at a time: every row's expert from the offsets."""
    rows, weight, dt = s["rows"].detach(), s["weight"].detach(), torch.float64
    n, E, D, F = case["items"], case["experts"], case["inner"], case["outer"]
    bounds = s["offsets"].cpu().numpy()
    outs = [np.zeros((n, F))]
    if s["train"]:
        outs += [np.zeros((n, D)), np.zeros((E, D, F))]
    for e in np.flatnonzero(np.diff(bounds)):
        w = weight[int(e)].to(dt).contiguous()
        if s["train"]:
            wt, dw = w.t().contiguous(), torch.zeros_like(w)
        for first in range(int(bounds[e]), int(bounds[e + 1]), 1 << 16):
            piece = slice(first, min(first + (1 << 16), int(bounds[e + 1])))
            x = rows[piece].to(dt)
            outs[0][piece] = torch.mm(x, w).cpu().numpy()
            if s["train"]:
                g = s["grad"][piece].to(dt)
                outs[1][piece] = torch.mm(g, wt).cpu().numpy()
                dw += torch.mm(x.t().contiguous(), g)
        if s["train"]:
            outs[2][e] = dw.cpu().numpy()
    return tuple(outs) if s["train"] else outs[0]


def _exact_choice(case, s):
    logits = s["logits"].detach().double().cpu().numpy()
    T, E, K = case["tokens"], case["experts"], case["choices"]
    t = np.arange(T)
    left = logits.copy()
    experts, chosen = np.full((T, K), -1), np.full((T, K), -np.inf)
    for k in range(K):  # the largest that is left, the first of equals
        at = left.argmax(1)
        chosen[:, k] = left[t, at]
        experts[:, k] = np.where(np.isneginf(chosen[:, k]), -1, at)
        left[t, at] = -np.inf
    top = np.where(np.isneginf(chosen[:, 0]), 0.0, chosen[:, 0])[:, None]
    e_all, e_top = np.exp(logits - top), np.exp(chosen - top)
    z = (e_top if s["normalize"] else e_all).sum(1, keepdims=True)
    z[z == 0] = 1.0
    weights = e_top / z
    if not s["train"]:
        return experts, weights
    g = s["grad"].double().cpu().numpy()
    # d w_k / d l_j = w_k (delta_jk - p_j), p_j the share of expert j in the sum
    shares = e_all / z
    if s["normalize"]:
        among = np.zeros((T, E), dtype=bool)
        for k in range(K):
            among[t[experts[:, k] >= 0], experts[experts[:, k] >= 0, k]] = True
        shares = np.where(among, shares, 0.0)
    d = -shares * (weights * g).sum(1, keepdims=True)
    for k in range(K):
        ok = experts[:, k] >= 0
        d[t[ok], experts[ok, k]] += (weights * g)[ok, k]
    return experts, weights, d


def _exact_dropout(case, s):
    n, key = case["rows"] * case["dim"], s["seed"]
    words = np.zeros((4, (n + 3) // 4), dtype=np.uint64)
    words[0] = np.arange(words.shape[1], dtype=np.uint64)
    words[3] = 6
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    keys = [key & 0xFFFFFFFF, key >> 32]
    for _ in range(10):
        a, b = words[0] * np.uint64(0xD2511F53), words[2] * np.uint64(0xCD9E8D57)
        words = np.stack([(b >> half) ^ words[1] ^ np.uint64(keys[0]), b & low,
                          (a >> half) ^ words[3] ^ np.uint64(keys[1]), a & low])
        keys = [(keys[0] + 0x9E3779B9) % 2 ** 32, (keys[1] + 0xBB67AE85) % 2 ** 32]
    dropped = (words.T.reshape(-1)[:n] < math.floor(s["p"] * 2 ** 32)).reshape(case["rows"], case["dim"])

    def thinned(t):
        v = t.detach().double().cpu().numpy() / (1 - s["p"])
        v[dropped] = 0
        return v

    out = thinned(s["x"])
    if case["residual"]:
        out += s["residual"].detach().double().cpu().numpy()
    if not s["train"]:
        return out
    dx = thinned(s["grad"])
    return (out, dx, s["grad"].double().cpu().numpy()) if case["residual"] else (out, dx)


def exact(case, seed):
    """What `run` returns, in 64 bits."""
    s = prepare(case, seed)
    if s["kind"].startswith("product"):
        return _exact_products(case, s)
    return _exact_choice(case, s) if s["kind"].startswith("choose") else _exact_dropout(case, s)
