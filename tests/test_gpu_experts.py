"""gs.ops.expert_* against the formulas in 64 bits.

Tolerances.  Rows sent to experts are copies.  A sum of K products is K fp32 products and additions, each off by 2^-24
of at most the sum S of the magnitudes: 2 * K * 2^-24 * S, then rounded once (eps / 2).  A weight's gradient is a dot product of
D fp32 products, added up along at most D / 4 values a lane and then a tree: (D + 12) * 2^-24 * S at most.  A row's
gradient is one product, rounded once."""
import numpy as np
import pytest
import torch

import graph_sampling_amd as gs
from graph_sampling_amd import capi

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rows(n, dim, dtype, dev, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, dim, generator=g).to(dtype).to(dev)


def experts_of(kind, tokens, choices, num, seed, idt=np.int64):
    rng = np.random.default_rng(seed)
    if kind == "even":
        e = rng.integers(0, max(num, 1), (tokens, choices))
    elif kind == "one":
        e = np.full((tokens, choices), num - 1)
    elif kind == "none":
        e = np.full((tokens, choices), -1)
    elif kind == "outside":
        e = rng.integers(-2, num + 2, (tokens, choices))
        e[rng.random((tokens, choices)) < 0.1] = np.iinfo(idt).max
        e[rng.random((tokens, choices)) < 0.1] = np.iinfo(idt).min
    elif kind == "skewed":
        e = (num ** rng.random((tokens, choices))).astype(np.int64) - 1
        e[rng.random((tokens, choices)) < 0.05] = -1
    return e.astype(idt)


def sorted_items(e, num):
    flat = e.reshape(-1).astype(np.int64)
    there = np.flatnonzero((flat >= 0) & (flat < num))
    live = there[np.argsort(flat[there], kind="stable")]
    order, place = np.full(flat.size, -1), np.full(flat.size, -1)
    order[:live.size] = live
    place[live] = np.arange(live.size)
    offsets = np.searchsorted(flat[live], np.arange(num + 1))
    return order, place.reshape(e.shape), offsets


def check_order(got, e, num):
    order, place, offsets = sorted_items(e, num)
    assert got.order.dtype == got.place.dtype == torch.int32 and got.offsets.dtype == torch.int64
    assert np.array_equal(got.offsets.cpu().numpy(), offsets)
    assert np.array_equal(got.place.cpu().numpy(), place)
    assert np.array_equal(got.order.cpu().numpy(), order)
    return order, place, offsets


def within(got, want, tol, dtype):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape
    assert np.all(np.abs(got - want) <= tol + (np.abs(want) + tol) * half_step(dtype) + smallest(dtype))


CASES = [
    # tokens, choices, experts, width, kind
    (1, 1, 1, 1, "even"), (1, 8, 64, 40, "even"), (3, 2, 5, 7, "outside"), (4, 4, 64, 2048, "even"), (100, 1, 5, 64, "skewed"),
    (128, 8, 255, 33, "skewed"), (513, 8, 256, 20, "even"), (600, 7, 300, 9, "outside"), (1000, 4, 16, 97, "one"),
    (1025, 4, 3, 1001, "none"), (2000, 3, 7, 130, "outside"), (9000, 9, 160, 12, "skewed"), (40000, 1, 5, 64, "skewed"),
    (5000, 2, 70000, 8, "even"), (30, 20, 40, 4096, "skewed"), (5, 11, 4, 1500, "outside"), (0, 3, 4, 8, "even"),
    (7, 0, 4, 8, "even"), (6, 2, 0, 8, "none"), (50, 4, 1000, 16, "outside"), (4096, 1, 256, 4, "even"),
    (1024, 1, 255, 100, "outside"), (205, 5, 17, 100, "skewed"), (140000, 1, 3, 8, "outside"), (270000, 2, 700, 2, "skewed"),
    (3, 3, 5, 70001, "outside"),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,choices,num,dim,kind", CASES)
def test_there_and_back(dev, tokens, choices, num, dim, kind, dtype):
    idt = np.int32 if (tokens + dim) % 2 else np.int64
    e = experts_of(kind, tokens, choices, num, tokens + dim, idt)
    d_e = torch.from_numpy(e).to(dev)
    x = rows(tokens, dim, dtype, dev, 1).requires_grad_(True)
    got_rows, got = gs.ops.expert_dispatch(x, d_e, num)
    order, place, offsets = check_order(got, e, num)
    check_order(gs.ops.expert_sort(d_e, num), e, num)
    live = int(offsets[-1])
    hx = x.detach().double().cpu().numpy()
    want = np.zeros((e.size, dim))
    want[:live] = hx[order[:live] // max(choices, 1)]
    assert got_rows.dtype == dtype and np.array_equal(got_rows.detach().double().cpu().numpy(), want)
    assert torch.equal(gs.ops.expert_gather(x, got), got_rows)
    # gradient: sums of the rows sent
    grad = rows(e.size, dim, dtype, dev, 2)
    hg = grad.double().cpu().numpy()
    at = place.reshape(-1)
    by_item = np.where(at[:, None] >= 0, hg[np.maximum(at, 0)] if e.size else np.zeros((0, dim)), 0).reshape(tokens, choices, dim)
    dx, = torch.autograd.grad(got_rows, x, grad)
    within(dx, by_item.sum(1), 2 * choices * F32 * np.abs(by_item).sum(1), dtype)
    # and back, with weights of either type or none
    for wtype in {None, torch.float32, dtype}:
        y = rows(e.size, dim, dtype, dev, 3).requires_grad_(True)
        w = None
        if wtype is not None:
            w = rows(tokens, choices, wtype, dev, 4).requires_grad_(True)
        hy = y.detach().double().cpu().numpy()
        hw = np.ones(e.shape) if w is None else w.detach().double().cpu().numpy()
        y_of = np.where(at[:, None] >= 0, hy[np.maximum(at, 0)] if e.size else np.zeros((0, dim)), 0).reshape(tokens, choices, dim)
        out = gs.ops.expert_combine(y, got, w)
        assert out.dtype == dtype
        terms = y_of * hw[:, :, None]
        within(out, terms.sum(1), 2 * choices * F32 * np.abs(terms).sum(1), dtype)
        dout = rows(tokens, dim, dtype, dev, 5)
        hd = dout.double().cpu().numpy()
        grads = torch.autograd.grad(out, [y] if w is None else [y, w], dout)
        want_dy = np.zeros((e.size, dim))
        items = order[:live]
        want_dy[:live] = hd[items // max(choices, 1)] * hw.reshape(-1)[items, None]
        within(grads[0], want_dy, np.abs(want_dy) * F32, dtype)
        assert not grads[0][live:].any()
        if w is not None:
            assert grads[1].dtype == wtype
            dots = hd[:, None, :] * y_of
            within(grads[1], dots.sum(2), (dim + 12) * F32 * np.abs(dots).sum(2), wtype)
            only_w, = torch.autograd.grad(gs.ops.expert_combine(y.detach(), got, w), w, dout)
            assert torch.equal(only_w, grads[1])
            only_y, = torch.autograd.grad(gs.ops.expert_combine(y, got, w.detach()), y, dout)
            assert torch.equal(only_y, grads[0])
            both = torch.ops.gs_ops._CAPI_ExpertCombineGrad(dout, y.detach(), got.order, got.place, got.offsets, w.detach())
            assert torch.equal(both[0], grads[0]) and torch.equal(both[1], grads[1])
        # and through the C ABI by itself
        w = None if w is None else w.detach()
        assert torch.equal(capi.expert_combine(y.detach(), got.place, w), out)
        c_dy, c_dw = capi.expert_combine_grad(dout, y.detach(), got.place, got.offsets, w)
        assert torch.equal(c_dy, grads[0]) and (w is None or torch.equal(c_dw, grads[1]))
    assert all(torch.equal(a, b) for a, b in zip(capi.expert_sort(d_e, num), got))
    assert torch.equal(capi.expert_gather(x.detach(), got.place, got.offsets), got_rows)
    assert all(torch.equal(a, b) for a, b in zip(capi.expert_dispatch(x.detach(), d_e, num), (got_rows,) + tuple(got)))


@gpu
@pytest.mark.parametrize("num", [1, 2, 14, 15, 16, 60, 126, 127, 128, 255, 256, 511, 512, 3000, 65536])
def test_sorts_of_every_size_and_number_of_experts(dev, num):
    """Both sides of every size at which the sort changes its tiles or launches, with digits of every width."""
    for n in (1, 255, 1024, 1025, 2048, 4096, 4097, 16384, 16385, 32769, 65537, 131073, 262145, 524289, 1_048_577):
        for kind in ("outside", "skewed"):
            e = experts_of(kind, n, 1, num, n % 1000 + num, np.int32)
            check_order(gs.ops.expert_sort(torch.from_numpy(e).to(dev), num), e, num)


@gpu
@pytest.mark.parametrize("num", [1, 15, 16, 127, 128, 255, 256, 257, 511, 512])
def test_few_items_of_any_number_of_experts(dev, num):
    """Both sides of every number of experts at which the one launch for few items changes its digits, or ends."""
    for tokens, choices, dim in ((1, 1, 3), (1, 8, 4096), (9, 7, 1000), (128, 8, 40), (1024, 1, 17), (1025, 1, 17)):
        for kind in ("outside", "skewed", "none"):
            e = experts_of(kind, tokens, choices, num, tokens + num)
            x = rows(tokens, dim, torch.bfloat16, dev, num)
            got, order = gs.ops.expert_dispatch(x, torch.from_numpy(e).to(dev), num)
            items, _, offsets = check_order(order, e, num)
            live = int(offsets[-1])
            assert torch.equal(got[:live], x[torch.from_numpy(items[:live] // choices).to(dev)]) and not got[live:].any()


@gpu
def test_one_choice_each_without_a_second_dimension(dev):
    """Node types: experts, places and weights of shape [tokens]."""
    e = experts_of("skewed", 777, 1, 6, 6)[:, 0]
    x = rows(777, 24, torch.float32, dev, 7)
    got_rows, order = gs.ops.expert_dispatch(x, torch.from_numpy(e).to(dev), 6)
    check_order(order, e, 6)
    assert order.place.shape == (777,)
    w = torch.rand(777, device=dev)
    out = gs.ops.expert_combine(got_rows, order, w)
    there = torch.from_numpy(e >= 0).to(dev)
    assert torch.equal(out, torch.where(there[:, None], x * w[:, None], 0.0))


@gpu
def test_rows_any_distance_apart(dev):
    for dtype in TYPES:
        base = rows(300, 77, dtype, dev, 8)
        e = experts_of("outside", 100, 3, 9, 9)
        d_e = torch.from_numpy(e).to(dev)
        for view in (base[:100, 1:70], base[::3, 3:35], base[5:105, 7:8], base.t()[:50].t()[:100]):
            x = view.detach().requires_grad_(True)
            got, order = gs.ops.expert_dispatch(x, d_e, 9)
            plain, _ = gs.ops.expert_dispatch(view.contiguous(), d_e, 9)
            assert torch.equal(got, plain)
            wide = rows(300, 2 * view.shape[1] + 1, dtype, dev, 10)
            y = wide[:, 1:view.shape[1] + 1]
            w = rows(3, 100, torch.float32, dev, 11).t()
            assert torch.equal(gs.ops.expert_combine(y, order, w), gs.ops.expert_combine(y.contiguous(), order, w.contiguous()))
            dx, = torch.autograd.grad(got, x, y)
            assert torch.equal(dx, gs.ops.expert_combine(y.contiguous(), order))
            dout = rows(200, 2 * view.shape[1] + 1, dtype, dev, 12)[::2, 1:view.shape[1] + 1]
            y2, w2 = y.detach().requires_grad_(True), w.detach().requires_grad_(True)
            a = torch.autograd.grad(gs.ops.expert_combine(y2, order, w2), (y2, w2), dout)
            y3, w3 = y.contiguous().requires_grad_(True), w.contiguous().requires_grad_(True)
            b = torch.autograd.grad(gs.ops.expert_combine(y3, order, w3), (y3, w3), dout.contiguous())
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        same = rows(1, 16, dtype, dev, 13).expand(100, 16)
        assert torch.equal(gs.ops.expert_gather(same, order), gs.ops.expert_gather(same.contiguous(), order))


@gpu
def test_offsets_beyond_32_bits(dev):
    """More than 2^32 values sent, combined and in the gradients: rows at both ends against the formulas."""
    if torch.cuda.mem_get_info(dev)[0] < 120 << 30:
        pytest.skip("needs about 60 GB of free device memory")
    tokens, choices, num, dim = 2_200_000, 2, 4, 1024
    g = torch.Generator(device=dev)
    g.manual_seed(33)
    e = torch.randint(-1, num, (tokens, choices), generator=g, device=dev, dtype=torch.int32)
    e[-1] = torch.tensor([num - 1, 0], device=dev)
    x = torch.randn(tokens, dim, generator=g, device=dev, dtype=torch.bfloat16)
    got, order = gs.ops.expert_dispatch(x, e, num)
    live = int(order.offsets[-1])
    assert live * dim > 2 ** 31 and got.numel() > 2 ** 32
    some = torch.cat([torch.arange(1000, device=dev), torch.arange(live - 1000, live, device=dev),
                      torch.randint(live, (1000,), generator=g, device=dev)])
    assert torch.equal(got[some], x[order.order[some].long() // choices]) and not got[live:].any()
    w = torch.rand(tokens, choices, generator=g, device=dev)
    out = gs.ops.expert_combine(got, order, w)
    t = torch.cat([torch.arange(500, device=dev), torch.arange(tokens - 500, tokens, device=dev)])
    there = (e[t] >= 0).float()
    within(out[t], (x[t].double() * (w[t] * there).sum(1, keepdim=True).double()).cpu().numpy(),
           6 * F32 * (x[t].abs().double() * w[t].sum(1, keepdim=True).double()).cpu().numpy(), torch.bfloat16)
    dy, dw = torch.ops.gs_ops._CAPI_ExpertCombineGrad(x, got, order.order, order.place, order.offsets, w)
    item = order.order[some].long()
    want = x[item // choices].double() * w.view(-1)[item, None].double()
    within(dy[some], want.cpu().numpy(), want.abs().cpu().numpy() * F32, torch.bfloat16)
    assert not dy[live:].any()
    square = (x[t].double() ** 2).sum(1, keepdim=True)
    within(dw[t], (square * there.double()).cpu().numpy(), ((dim + 12) * F32 * square).cpu().numpy() * np.ones((1, choices)),
           torch.float32)


@gpu
def test_more_lanes_than_one_launch_takes(dev):
    """Sums and gradients of more than 2^32 lanes go in several launches: tokens at both ends and beside the cut."""
    if torch.cuda.mem_get_info(dev)[0] < 120 << 30:
        pytest.skip("needs about 70 GB of free device memory")
    def near(n, cut):
        return torch.cat([torch.arange(1000, device=dev), torch.arange(cut - 1000, cut + 1000, device=dev),
                          torch.arange(n - 1000, n, device=dev)])

    # rows of 17 fp16 values are three lanes each, every token's place the same row
    cut = (2 ** 32 - 1) // 256 * 256 // 3
    tokens = cut + 300_000
    row = torch.arange(1, 18, device=dev).half()
    weights = (torch.arange(tokens, device=dev, dtype=torch.int32) % 64).half().view(tokens, 1)
    place = torch.zeros(tokens, 1, dtype=torch.int32, device=dev)
    at = gs.ops.ExpertOrder(place.view(-1), place, torch.tensor([0, tokens], device=dev))
    out = gs.ops.expert_combine(row.expand(tokens, 17), at, weights)
    t = near(tokens, cut)
    assert torch.equal(out[t], weights[t] * row)  # (whole numbers up to 63 * 17: exact)
    del out, weights, place, at
    # rows of one value have four lanes in the gradient
    cut = (2 ** 32 - 1) // 256 * 64
    tokens = cut + 5000
    weights = (torch.arange(tokens, device=dev, dtype=torch.int32) % 64).half().view(tokens, 1)
    dout = (torch.arange(tokens, device=dev, dtype=torch.int32) % 31).half().view(tokens, 1)
    place = torch.arange(tokens - 1, -1, -1, device=dev, dtype=torch.int32).view(tokens, 1)
    offsets = torch.tensor([0, tokens], device=dev)
    dy, dw = torch.ops.gs_ops._CAPI_ExpertCombineGrad(dout, weights, place.view(-1), place, offsets, weights)
    t = near(tokens, cut)
    back = tokens - 1 - t
    assert torch.equal(dy[back], weights[t] * dout[t]) and torch.equal(dw[t], dout[t] * weights[back])
    assert bool((dy.view(-1).flip(0) == (weights * dout).view(-1)).all())


@gpu
def test_rows_are_kept_for_the_gradient_of_weights_only(dev):
    """Rows that nobody's gradient needs may be overwritten after they were added up."""
    e = torch.randint(-1, 5, (50, 3), device=dev)
    x = rows(50, 24, torch.float32, dev, 3).requires_grad_(True)
    sent, order = gs.ops.expert_dispatch(x, e, 5)
    w = rows(50, 3, torch.float32, dev, 4)
    dout = rows(50, 24, torch.float32, dev, 5)
    want, = torch.autograd.grad(gs.ops.expert_combine(sent, order, w), x, dout, retain_graph=True)
    for weights in (None, w):
        y = sent * 1.0
        out = gs.ops.expert_combine(y, order, weights)
        y.detach().zero_()
        got, = torch.autograd.grad(out, x, dout, retain_graph=True)
        if weights is not None:
            assert torch.equal(got, want)
    kept = w.clone().requires_grad_(True)
    y = sent * 1.0
    out = gs.ops.expert_combine(y, order, kept)
    with torch.no_grad():
        y.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, (x, kept), dout)


@gpu
def test_what_has_no_place_does_not_matter(dev):
    """NaN and infinities in rows and weights of choices that name no expert, and behind the last row."""
    e = np.array([[0, -1], [-1, -1], [5, 1], [1, 0]])
    d_e = torch.from_numpy(e).to(dev)
    order = gs.ops.expert_sort(d_e, 2)
    live = int(order.offsets[-1])
    assert live == 4
    y = rows(8, 20, torch.bfloat16, dev, 14)
    w = torch.rand(4, 2, device=dev)
    there = torch.from_numpy((e >= 0) & (e < 2)).to(dev)
    clean_w = torch.where(there, w, 0.0)
    want = gs.ops.expert_combine(y, order, clean_w)
    y[live:] = float("nan")
    dirty = torch.where(there, w, float("inf")).requires_grad_(True)
    y.requires_grad_(True)
    out = gs.ops.expert_combine(y, order, dirty)
    assert torch.equal(out, want) and torch.equal(out[1], torch.zeros_like(out[1]))
    dout = rows(4, 20, torch.bfloat16, dev, 15)
    dout[1] = float("inf")  # of the token without any expert
    dy, dw = torch.autograd.grad(out, (y, dirty), dout)
    assert dy.isfinite().all() and dw.isfinite().all()
    assert not dy[live:].any() and not dw[~there].any()
    x = rows(4, 20, torch.bfloat16, dev, 16)
    x[1] = float("nan")
    assert gs.ops.expert_gather(x, order).isfinite().all()


@gpu
def test_places_that_lead_nowhere_are_left_out(dev):
    """An order that was not made by a sort: places beyond the rows are neither read nor written."""
    place = torch.tensor([[0, 100], [-7, 2], [2 ** 31 - 1, 1]], dtype=torch.int32, device=dev)
    order = gs.ops.ExpertOrder(torch.zeros(6, dtype=torch.int32, device=dev), place, torch.tensor([0, 3], device=dev))
    x = rows(3, 5, torch.float32, dev, 17)
    got = gs.ops.expert_gather(x, order)
    assert torch.equal(got[:3], x[[0, 2, 1]]) and not got[3:].any()
    assert torch.equal(gs.ops.expert_combine(got, order), x)
    # offsets beyond the rows, and negative ones, clear nothing
    for end in (2 ** 40, -3, 6):
        order = order._replace(offsets=torch.tensor([0, end], device=dev))
        assert torch.equal(gs.ops.expert_gather(x, order)[:3], x[[0, 2, 1]])


@gpu
def test_gradient_against_differences(dev):
    e = torch.tensor([[0, 2], [2, -1], [1, 1]], device=dev)
    order = gs.ops.expert_sort(e, 3)
    y, w = rows(6, 5, torch.float32, dev, 18), rows(3, 2, torch.float32, dev, 19)
    dout = rows(3, 5, torch.float32, dev, 20)
    vy, vw = rows(6, 5, torch.float32, dev, 21), rows(3, 2, torch.float32, dev, 22)
    y.requires_grad_(True), w.requires_grad_(True)
    dy, dw = torch.autograd.grad(gs.ops.expert_combine(y, order, w), (y, w), dout)

    def along(h):
        with torch.no_grad():
            return (gs.ops.expert_combine(y + h * vy, order, w + h * vw).double() * dout.double()).sum().item()

    # bilinear: the central difference is exact but for rounding; values below 4 + 4 h each, h = 1:
    # two evaluations of 15 outputs with sums below 2 * 8 * 8, times gradients below 4, six roundings each
    slope = (dy.double() * vy.double()).sum().item() + (dw.double() * vw.double()).sum().item()
    assert abs((along(1.0) - along(-1.0)) / 2 - slope) < 15 * 128 * 4 * 6 * F32


@gpu
def test_recorded_and_replayed(dev):
    """Sort, rows there and back, and the gradients in one HIP graph, inputs rewritten between replays."""
    for tokens, choices, num, dim in ((6, 4, 16, 40), (3000, 3, 20, 24), (700, 2, 1000, 8)):
        d_e = torch.from_numpy(experts_of("skewed", tokens, choices, num, 23)).to(dev)
        x, w = rows(tokens, dim, torch.float32, dev, 24), rows(tokens, choices, torch.float32, dev, 25)
        dout = rows(tokens, dim, torch.float32, dev, 26)

        def all_of_it():
            got, order = gs.ops.expert_dispatch(x, d_e, num)
            y = got * 2
            out = gs.ops.expert_combine(y, order, w)
            dy, dw = torch.ops.gs_ops._CAPI_ExpertCombineGrad(dout, y, order.order, order.place, order.offsets, w)
            return (got, out, dy, dw, gs.ops.expert_combine(dy, order)) + tuple(order)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            all_of_it()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = all_of_it()
        for rep in range(4):
            d_e.copy_(torch.from_numpy(experts_of("outside" if rep % 2 else "skewed", tokens, choices, num, 30 + rep)))
            x.copy_(rows(tokens, dim, torch.float32, dev, 40 + rep))
            want = all_of_it()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@gpu
def test_recorded_backward_pass(dev):
    """There, back with weights, and the gradients of rows and weights through autograd, recorded."""
    x, w = rows(200, 16, torch.float32, dev, 34).requires_grad_(True), torch.rand(200, 3, device=dev).requires_grad_(True)
    e = torch.from_numpy(experts_of("outside", 200, 3, 7, 35)).to(dev)
    dout = rows(200, 16, torch.float32, dev, 36)

    def step():
        got, order = gs.ops.expert_dispatch(x, e, 7)
        out = gs.ops.expert_combine(torch.tanh(got), order, w)
        return torch.autograd.grad(out, (x, w), dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for rep in range(3):
        e.copy_(torch.from_numpy(experts_of("skewed" if rep % 2 else "outside", 200, 3, 7, 37 + rep)))
        dout.copy_(rows(200, 16, torch.float32, dev, 40 + rep))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_two_threads_at_once(dev):
    import threading
    work = []
    for seed in (43, 44):
        x, e = rows(9000, 24, torch.float32, dev, seed), torch.from_numpy(experts_of("skewed", 9000, 2, 300, seed)).to(dev)
        got, order = gs.ops.expert_dispatch(x, e, 300)
        work.append((x, e, got, order, gs.ops.expert_combine(got, order)))
    torch.cuda.synchronize()
    wrong = []

    def run(x, e, want, want_order, want_out):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got, order = gs.ops.expert_dispatch(x, e, 300)
                same = all(torch.equal(a, b) for a, b in zip((got,) + tuple(order), (want,) + tuple(want_order)))
                if not (same and torch.equal(gs.ops.expert_combine(got, order), want_out)):
                    wrong.append(1)

    threads = [threading.Thread(target=run, args=t) for t in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@gpu
def test_a_layer_of_typed_nodes_end_to_end(dev):
    """Embeddings of a frontier, rows by type, a product per type, back with weights, and the gradients of
    every leaf against the same layer written in 64-bit torch."""
    N, D, H, types = 500, 24, 16, 4
    rng = np.random.default_rng(27)
    ids = torch.from_numpy(rng.integers(-1, N, 900)).to(dev)
    kind = torch.from_numpy(rng.integers(0, types, (900, 2))).to(dev)
    kind[5] = -1
    leaves = [rows(N, D, torch.float32, dev, 28), rows(types * D, H, torch.float32, dev, 29).view(types, D, H) / 5,
              torch.rand(900, 2, device=dev)]
    dout = rows(900, H, torch.float32, dev, 30)
    table, nets, w = (t.clone().requires_grad_(True) for t in leaves)
    h = gs.ops.embedding(table, ids, 0.5)
    got, order = gs.ops.expert_dispatch(h, kind, types)
    at = order.offsets.tolist()
    y = torch.cat([got[at[t]:at[t + 1]] @ nets[t] for t in range(types)] + [got[at[-1]:] @ nets[0]])
    out = gs.ops.expert_combine(y, order, w)
    grads = torch.autograd.grad(out, (table, nets, w), dout)
    table64, nets64, w64 = (t.double().requires_grad_(True) for t in leaves)
    h64 = torch.where((ids >= 0)[:, None], table64[ids.clamp(min=0)] * 0.5, 0.0)
    y64 = (h64[:, None, None, :] @ nets64[kind.clamp(min=0)])[:, :, 0]
    out64 = torch.where((kind >= 0)[:, :, None], y64 * w64[:, :, None], 0.0).sum(1)
    grads64 = torch.autograd.grad(out64, (table64, nets64, w64), dout.double())
    # fp32 chains of at most ~1000 additions (a type's rows) in values of unit size: relative 2^-24 * 1100
    for a, b in zip((out,) + grads, (out64,) + grads64):
        assert (a.double() - b).abs().max() <= 1100 * F32 * b.abs().max()


@gpu
def test_recording_is_refused_where_it_would_end_the_process(dev):
    order = gs.ops.expert_sort(torch.zeros(4, 1, dtype=torch.int64, device=dev), 2)
    x = rows(4, 8, torch.float32, dev, 31).requires_grad_(True)
    w = torch.rand(4, 1, device=dev).requires_grad_(True)
    eager = gs.ops.expert_combine(gs.ops.expert_gather(x, order), order, w)
    torch.cuda.synchronize()
    graph, messages = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        kept = x.detach() * 2
        for call in (lambda: gs.ops.expert_gather(x, order), lambda: gs.ops.expert_combine(x, order),
                     lambda: gs.ops.expert_combine(x.detach(), order, w)):
            try:
                call()
            except RuntimeError as error:
                messages.append(str(error))
    assert len(messages) == 3 and all("eager graph of the same leaf" in m for m in messages)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, x.detach() * 2)
    torch.autograd.grad(eager.sum(), (x, w))


@gpu
def test_sizes_beyond_the_limits_are_refused_before_anything_is_allocated(dev):
    e = torch.zeros(4, dtype=torch.int32, device=dev)
    x = torch.zeros(4, 3, device=dev)
    held = torch.cuda.memory_allocated(dev)
    for num in (1 << 31, 1 << 40, (1 << 63) - 1):
        with pytest.raises(RuntimeError, match="experts are taken"):
            gs.ops.expert_sort(e, num)
        with pytest.raises(RuntimeError, match="experts are taken"):
            gs.ops.expert_dispatch(x, e, num)
        for entry in (torch.ops.gs_ops._CAPI_EmbeddingGrad, torch.ops.gs_ops._CAPI_EmbeddingSparseGrad):
            with pytest.raises(RuntimeError, match="rows are taken"):
                entry(x, e, max(num, 1 << 33), 1.0)
    assert torch.cuda.memory_allocated(dev) == held


@gpu
def test_refusals(dev):
    x, e = rows(5, 4, torch.float32, dev, 32), torch.zeros(5, 2, dtype=torch.int64, device=dev)
    for bad, match in (((x.double(), e, 3), "float32, float16 or bfloat16"), ((x, e.float(), 3), "int64"),
                       ((x[0], e, 3), "two dimensions"), ((x, e[:4], 3), "tokens"), ((x, e[None], 3), "choices"),
                       ((x.cpu(), e, 3), "GPU tensor"), ((x, e.cpu(), 3), "GPU tensor"), ((x, e, -1), "non-negative")):
        with pytest.raises(RuntimeError, match=match):
            gs.ops.expert_dispatch(*bad)
    got, order = gs.ops.expert_dispatch(x, e, 3)
    w = torch.rand(5, 2, device=dev)
    for bad, match in (((got[:9], order), "items"), ((got, order, w[:4]), "shape of place"),
                       ((got.half(), order, w.bfloat16()), "rows' type"), ((got, order, w.cpu()), "GPU tensor"),
                       ((got, order._replace(place=order.place.long())), "int32"),
                       ((got, order._replace(order=order.order[:5])), "order must be"),
                       ((got, order._replace(place=order.place.t())), "contiguous")):
        with pytest.raises(RuntimeError, match=match):
            gs.ops.expert_combine(*bad)
    with pytest.raises(RuntimeError, match="offsets"):
        gs.ops.expert_gather(x, order._replace(offsets=order.offsets[:0]))
    y, w = got.clone().requires_grad_(True), w.requires_grad_(True)
    with pytest.raises(RuntimeError, match="once more"):
        torch.autograd.grad(gs.ops.expert_combine(y, order, w).sum(), y, create_graph=True)
    # what does not depend on anything that is followed needs no second gradient
    torch.autograd.grad(gs.ops.expert_combine(y, order).sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gs.ops.expert_gather(t, order).sum())(x)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("choices,kind", [(1, "outside"), (2, "skewed")])
def test_many_tokens_with_a_part_of_a_workgroup_behind(dev, choices, kind, dtype):
    """Four chunks a lane are taken from 2^20 chunks on: 300 001 rows of 33 values are 2 700 009 in fp32 and 1 500 005 in
    the others, 745 and 869 behind the last whole workgroup of 1024."""
    tokens, dim, num = 300_001, 33, 9
    e = experts_of(kind, tokens, choices, num, choices)
    x = rows(tokens, dim, dtype, dev, 53)
    got, order = gs.ops.expert_dispatch(x, torch.from_numpy(e).to(dev), num)
    items, _, offsets = check_order(order, e, num)
    live = int(offsets[-1])
    assert live < e.size
    assert torch.equal(got[:live], x[torch.from_numpy(items[:live] // choices).to(dev)]) and not got[live:].any()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
# rows of 65, 77, 85, 86 and 129 chunks of four values (fp32) and of eight: both sides of where half a wave a token gives
# way to a whole one, and where either goes around more than once, the last time in part; then tokens too few for that
@pytest.mark.parametrize("tokens,dim", [(4099, 257), (4099, 307), (4099, 339), (4099, 341), (4099, 513), (4099, 611),
                                        (4099, 675), (4099, 681), (4099, 1025), (4096, 340), (130, 300), (130, 511)])
def test_gradients_of_sums_of_long_rows(dev, tokens, dim, dtype):
    choices, num = 3, 9
    e = torch.from_numpy(experts_of("outside", tokens, choices, num, dim)).to(dev)
    order = gs.ops.expert_sort(e, num)
    live = int(order.offsets[-1])
    at = order.place.long()
    there = at >= 0
    assert 0 < live < at.numel()
    dout = rows(tokens, dim, dtype, dev, 55)
    d64 = dout.double()
    for wtype, shift in ((torch.float32, 0), (dtype, 1)):
        y = rows(tokens * choices, dim + shift, dtype, dev, 54)[:, shift:].requires_grad_(True)
        w = rows(tokens, choices, wtype, dev, 56).requires_grad_(True)
        dy, dw = torch.autograd.grad(gs.ops.expert_combine(y, order, w), (y, w), dout)
        want = torch.zeros(tokens * choices, dim, dtype=torch.float64, device=dev)
        want[at[there]] = (d64[:, None, :] * w.detach().double()[:, :, None])[there]
        off = (dy.double() - want).abs()
        assert bool((off <= want.abs() * (F32 + half_step(dtype)) * (1 + F32) + smallest(dtype)).all())
        assert not dy[live:].any()
        terms = torch.where(there[:, :, None], d64[:, None, :] * y.detach().double()[at.clamp(min=0)], 0.0)
        within(dw, terms.sum(2).cpu().numpy(), ((dim + 12) * F32 * terms.abs().sum(2)).cpu().numpy(), wtype)


# ------------------------------------------------------------------ no GPU ----
def test_bad_arguments_are_refused_before_anything_is_launched():
    import ctypes
    lib, i64 = capi.lib(), ctypes.c_int64
    buf = (ctypes.c_int64 * 64)()
    at = ctypes.addressof(buf)

    def fails(status, match):
        assert status < 0 and match in lib.gs_status_string(status), (status, lib.gs_status_string(status))

    def sort(ids=buf, id_bytes=8, n=4, num=3, order=buf, place=buf, offsets=buf, ws=buf, ws_bytes=16):
        return lib.gs_expert_sort(ids, id_bytes, i64(n), i64(num), order, place, offsets, ws, ctypes.c_size_t(ws_bytes), None)

    assert lib.gs_expert_sort_workspace_bytes(i64(4), i64(3)) == 0  # one workgroup's, in LDS
    fails(sort(n=5000), b"workspace")
    fails(sort(n=5, num=300), b"workspace")
    fails(sort(n=-1), b"negative")
    fails(sort(n=1 << 31), b"2^31")
    fails(sort(num=1 << 31), b"experts")
    fails(sort(id_bytes=3), b"id_bytes")
    fails(sort(offsets=None), b"null")
    fails(sort(ids=ctypes.c_void_p(at + 4)), b"aligned")

    def gather(x=buf, stride=8, dim=8, kind=0, place=buf, tokens=2, choices=2, live=buf, out=buf):
        return lib.gs_expert_gather(x, i64(stride), i64(dim), kind, place, i64(tokens), i64(choices), live, out, None)

    assert gather(tokens=0) == gather(choices=0) == gather(dim=0) == 0
    fails(gather(kind=7), b"value type")
    fails(gather(tokens=1 << 20, choices=1 << 20), b"2^31")
    fails(gather(stride=-1), b"stride")
    fails(gather(live=None), b"null")
    fails(gather(x=ctypes.c_void_p(at + 2)), b"aligned")
    fails(lib.gs_expert_combine(buf, i64(8), i64(8), 1, buf, i64(2), i64(2), buf, 2, buf, None), b"weights")
    fails(lib.gs_expert_combine(None, i64(8), i64(8), 1, buf, i64(2), i64(2), buf, 1, buf, None), b"null")
    fails(lib.gs_expert_combine_grad(buf, i64(8), None, i64(8), i64(8), 0, buf, i64(2), i64(2), buf, buf, 0, buf, buf, None),
          b"null")


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU tensor"):
        gs.ops.expert_dispatch(torch.zeros(3, 4), torch.zeros(3, 2, dtype=torch.int64), 4)


def test_the_binding_refuses_weights_in_host_memory(monkeypatch):
    """They would be read, and their gradient written, by a kernel."""
    import ctypes
    monkeypatch.setattr(capi, "_rows", lambda t, name: (ctypes.c_void_p(t.data_ptr()), capi._i64(t.stride(0)),
                                                        capi._i64(t.size(1)), 0))
    monkeypatch.setattr(capi, "_need", lambda t, dtype, name: None)  # (as if the others were on the GPU)
    monkeypatch.setattr(capi, "_stream", lambda device: None)
    y, x, weights = torch.zeros(6, 4), torch.zeros(3, 4), torch.ones(3, 2)
    place, offsets = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(5, dtype=torch.int64)
    monkeypatch.setattr(capi, "lib", lambda: pytest.fail("a library call"))
    with pytest.raises(capi.GsError, match="weights must live on the GPU"):
        capi.expert_combine(y, place, weights)
    with pytest.raises(capi.GsError, match="weights must live on the GPU"):
        capi.expert_combine_grad(x, y, place, offsets, weights)
