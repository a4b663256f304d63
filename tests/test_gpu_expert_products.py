"""gs.ops.expert_matmul and its gradients against the formulas in 64 bits.

Tolerances.  An element is a sum of K products.  Of 16-bit values they are exact in fp32; fp32 products are off by 2^-24
of themselves.  K additions, in whatever order, are off by at most one step (2^-23: the matrix cores' rounding is not
specified) of the sum S of the magnitudes each, pieces of a long sum that are joined by at most 64 more: (K + 72) * 2^-23 * S,
then rounded once (eps / 2).  Small whole numbers (below 2^24 in all sums) are exact, but for the last rounding: there,
results are equal to the formula's, rounded."""
import numpy as np
import pytest
import torch

import graph_sampling_amd as gs
from graph_sampling_amd import capi

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def normal(*shape, dtype, dev, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(dev)


def whole(*shape, dtype, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randint(-3, 4, shape, generator=g, device=dev).to(dtype)


def loads_of(kind, n, experts, seed):
    """Rows of each expert, at most n together."""
    rng = np.random.default_rng(seed)
    if kind == "even":
        return rng.multinomial(n, np.full(experts, 1 / experts)) if experts else np.zeros(0, int)
    if kind == "skewed":  # a part behind the last, experts without rows
        share = rng.random(experts) ** 6
        return rng.multinomial(n, np.append(share / share.sum() * 0.8, 0.2))[:experts]
    if kind == "last":
        return np.append(np.zeros(experts - 1, int), n)
    if kind == "first":
        return np.append(n, np.zeros(experts - 1, int))
    if kind == "none":
        return np.zeros(experts, int)
    raise AssertionError(kind)


def order_of(loads, n, dev):
    at = torch.from_numpy(np.append(0, np.cumsum(loads)).astype(np.int64)).to(dev)
    p = torch.arange(n, device=dev, dtype=torch.int32)
    p = torch.where(p < at[-1], p, -1).int()
    return gs.ops.ExpertOrder(p, p.clone(), at)


def formula(rows, loads, weight, grad=None):
    """(out, d_rows, d_weight) and the sums of the magnitudes of each, in 64 bits."""
    rows, weight = rows.detach().double(), weight.detach().double()
    dev = rows.device
    outs = [torch.zeros(rows.shape[0], weight.shape[2], dtype=torch.float64, device=dev) for _ in range(2)]
    if grad is not None:
        grad = grad.double()
        outs += [torch.zeros_like(rows) for _ in range(2)]
        outs += [torch.zeros(weight.shape, dtype=torch.float64, device=dev) for _ in range(2)]
    first = 0
    for e, load in enumerate(loads):
        if load == 0:
            continue
        of = slice(first, first + int(load))
        first += int(load)
        x, w = rows[of].contiguous(), weight[e].contiguous()
        outs[0][of], outs[1][of] = torch.mm(x, w), torch.mm(x.abs(), w.abs())
        if grad is not None:
            g, wt, xt = grad[of].contiguous(), w.t().contiguous(), x.t().contiguous()
            outs[2][of], outs[3][of] = torch.mm(g, wt), torch.mm(g.abs(), wt.abs())
            outs[4][e], outs[5][e] = torch.mm(xt, g), torch.mm(xt.abs(), g.abs())
    return outs


def within(got, want, size, depth, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    tol = (depth + 72) * 2.0 ** -23 * size
    if not isinstance(depth, int):
        tol = (depth + 72) * 2.0 ** -23 * size
    off = (got.detach().double() - want).abs()
    assert bool((off <= tol + (want.abs() + tol) * half_step(dtype) + smallest(dtype)).all())


def weights_of(make, experts, inner, outer, transposed, **kw):
    return make(experts, outer, inner, **kw).transpose(1, 2) if transposed else make(experts, inner, outer, **kw)


CASES = [
    # rows, experts, inner, outer, kind, transposed
    (1, 1, 1, 1, "even", False), (1, 1, 8, 8, "even", True), (1, 64, 2048, 512, "even", False), (4, 3, 40, 24, "even", True),
    (16, 64, 512, 1024, "even", False), (24, 64, 264, 520, "skewed", True), (33, 5, 17, 9, "skewed", False),
    (100, 7, 31, 33, "skewed", True), (127, 1, 64, 128, "first", False), (129, 2, 65, 127, "last", True),
    (256, 4, 128, 256, "even", False), (257, 3, 96, 257, "skewed", True), (300, 300, 24, 40, "skewed", False),
    (513, 2, 200, 130, "first", True), (1000, 9, 1001, 333, "skewed", False), (1000, 9, 333, 1001, "skewed", True),
    (2000, 16, 320, 448, "even", False), (2048, 3, 256, 512, "skewed", True), (3000, 1, 77, 264, "even", False),
    (5000, 5, 64, 128, "even", False), (5000, 700, 16, 8, "skewed", True), (700, 3, 4096, 256, "even", False),
    (640, 4, 512, 768, "last", False), (9000, 4, 136, 72, "skewed", False), (40, 8, 0, 16, "even", False),
    (40, 8, 16, 0, "even", True), (0, 4, 8, 8, "none", False), (50, 6, 24, 32, "none", False), (70, 0, 8, 16, "none", False),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,experts,inner,outer,kind,transposed", CASES)
def test_products_and_gradients(dev, n, experts, inner, outer, kind, transposed, dtype):
    loads = loads_of(kind, n, experts, n + inner)
    order = order_of(loads, n, dev)
    live = int(sum(loads))
    depth = torch.from_numpy(np.asarray(loads, dtype=np.float64)).to(dev)[:, None, None]
    for make in (whole, normal):
        rows = make(n, inner, dtype=dtype, dev=dev, seed=1).requires_grad_(True)
        weight = weights_of(make, experts, inner, outer, transposed, dtype=dtype, dev=dev, seed=2).detach().requires_grad_(True)
        grad = make(n, outer, dtype=dtype, dev=dev, seed=3)
        out = gs.ops.expert_matmul(rows, order, weight)
        d_rows, d_weight = torch.autograd.grad(out, (rows, weight), grad)
        want = formula(rows, loads, weight, grad)
        if make is whole:
            for a, b in ((out, want[0]), (d_rows, want[2]), (d_weight, want[4])):
                assert a.dtype == dtype and torch.equal(a.detach().double(), b.to(dtype).double())
        else:
            within(out, want[0], want[1], inner, dtype)
            within(d_rows, want[2], want[3], outer, dtype)
            within(d_weight, want[4], want[5], depth, dtype)
        assert not out.detach()[live:].any() and not d_rows[live:].any()
        assert d_weight.stride() == weight.stride() or experts * inner * outer <= 1 or min(inner, outer) <= 1
        # one of the two alone, and through the C ABI by itself
        only, = torch.autograd.grad(gs.ops.expert_matmul(rows, order, weight.detach()), rows, grad)
        assert torch.equal(only, d_rows)
        only, = torch.autograd.grad(gs.ops.expert_matmul(rows.detach(), order, weight), weight, grad)
        assert torch.equal(only, d_weight)
        assert torch.equal(capi.expert_matmul(rows.detach(), order.offsets, weight.detach()), out)
        assert torch.equal(capi.expert_matmul(grad, order.offsets, weight.detach().transpose(1, 2)), d_rows)
        assert torch.equal(torch.ops.gs_ops._CAPI_ExpertMatmulGrad(grad, rows.detach(), order.offsets),
                           capi.expert_matmul_grad(grad, rows.detach(), order.offsets))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("transposed", [False, True])
def test_sizes_around_every_tile(dev, dtype, transposed):
    """Rows, widths and depths on both sides of the sizes of tiles and steps, in whole numbers: equal to the formula."""
    sizes = (1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 191, 192, 193, 255, 256, 257, 383, 384, 385)
    rng = np.random.default_rng(7)
    for i in range(60):
        inner, outer = (int(rng.choice(sizes)) for _ in range(2))
        experts = int(rng.choice((1, 2, 3, 17)))
        loads = rng.choice((0,) + sizes, experts)
        n = int(loads.sum()) + int(rng.choice((0, 1, 300)))
        order = order_of(loads, n, dev)
        rows = whole(n, inner, dtype=dtype, dev=dev, seed=i).requires_grad_(True)
        weight = weights_of(whole, experts, inner, outer, transposed, dtype=dtype, dev=dev, seed=i + 1).detach().requires_grad_(True)
        grad = whole(n, outer, dtype=dtype, dev=dev, seed=i + 2)
        out = gs.ops.expert_matmul(rows, order, weight)
        got = (out,) + torch.autograd.grad(out, (rows, weight), grad)
        for a, b in zip(got, formula(rows, loads, weight, grad)[::2]):
            assert torch.equal(a.detach().double(), b.to(dtype).double()), (i, loads, n, inner, outer)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_of_few_experts(dev, dtype):
    """Node types: the gradients' sums are long, and few of them."""
    for n, experts, inner, outer, kind in ((200_003, 3, 64, 128, "skewed"), (150_000, 1, 24, 17, "first"),
                                           (100_001, 40, 33, 8, "even"), (60_000, 2, 256, 200, "last")):
        loads = loads_of(kind, n, experts, n)
        order = order_of(loads, n, dev)
        rows, grad = (whole(n, d, dtype=dtype, dev=dev, seed=d) for d in (inner, outer))
        weight = whole(experts, inner, outer, dtype=dtype, dev=dev, seed=5)
        want = formula(rows, loads, weight, grad)
        assert float(want[5].max()) < 2 ** 24
        got = (gs.ops.expert_matmul(rows, order, weight), gs.ops.expert_matmul(grad, order, weight.transpose(1, 2)),
               capi.expert_matmul_grad(grad, rows, order.offsets))
        for a, b in zip(got, want[::2]):
            assert torch.equal(a.double(), b.to(dtype).double())
        again = capi.expert_matmul_grad(grad, rows, order.offsets)
        assert torch.equal(got[2], again)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_bits_every_time(dev, dtype):
    """Sums are made in an order that the offsets alone decide."""
    for n, experts, inner, outer in ((12, 32, 1024, 512), (3000, 8, 512, 384), (120_000, 2, 48, 64)):
        loads = loads_of("skewed", n, experts, 1)
        order = order_of(loads, n, dev)
        rows, weight = normal(n, inner, dtype=dtype, dev=dev, seed=1), normal(experts, inner, outer, dtype=dtype, dev=dev, seed=2)
        grad = normal(n, outer, dtype=dtype, dev=dev, seed=3)
        first = capi.expert_matmul(rows, order.offsets, weight), capi.expert_matmul_grad(grad, rows, order.offsets)
        for _ in range(3):
            assert torch.equal(capi.expert_matmul(rows, order.offsets, weight), first[0])
            assert torch.equal(capi.expert_matmul_grad(grad, rows, order.offsets), first[1])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_what_belongs_to_others_does_not_matter(dev, dtype):
    """NaN and infinities in an expert's rows and matrix stay with it, and those behind the last row go nowhere."""
    for n, inner, outer in ((40, 48, 72), (1500, 200, 320), (900, 33, 47)):
        loads = np.array([n // 8, 0, n // 4 + 1, 3, n // 8])
        at = np.append(0, np.cumsum(loads))
        order = order_of(loads, n, dev)
        for transposed in (False, True):
            rows, grad = (normal(n, d, dtype=dtype, dev=dev, seed=d) for d in (inner, outer))
            weight = weights_of(normal, 5, inner, outer, transposed, dtype=dtype, dev=dev, seed=1)
            want = [t.clone() for t in (gs.ops.expert_matmul(rows, order, weight),
                                        gs.ops.expert_matmul(grad, order, weight.transpose(1, 2)),
                                        capi.expert_matmul_grad(grad, rows, order.offsets))]
            rows[at[-1]:], grad[at[-1]:] = float("nan"), float("inf")
            rows[at[3]:at[4]], grad[at[3]:at[4]] = float("nan"), float("inf")
            weight[1], weight[3] = float("nan"), float("inf")
            got = (gs.ops.expert_matmul(rows, order, weight), gs.ops.expert_matmul(grad, order, weight.transpose(1, 2)),
                   capi.expert_matmul_grad(grad, rows, order.offsets))
            for a, b in zip(got[:2], want[:2]):
                assert torch.equal(a[:at[3]], b[:at[3]]) and torch.equal(a[at[4]:], b[at[4]:])
                assert not a[at[3]:at[4]].isfinite().any()
            keep = [0, 1, 2, 4]
            assert torch.equal(got[2][keep], want[2][keep]) and not got[2][3].isfinite().any()
            # an infinity in one row stays there
            rows = normal(n, inner, dtype=dtype, dev=dev, seed=inner)
            weight = weights_of(normal, 5, inner, outer, transposed, dtype=dtype, dev=dev, seed=1)
            rows[1, inner - 1] = float("inf")
            one = gs.ops.expert_matmul(rows, order, weight)
            assert torch.equal(one[2:], want[0][2:]) and torch.equal(one[:1], want[0][:1])
            assert not one[1].isfinite().all()


@gpu
def test_rows_and_matrices_any_distance_apart(dev):
    for dtype in TYPES:
        base = normal(700, 150, dtype=dtype, dev=dev, seed=1)
        for n, view in ((100, base[:100, 1:70]), (230, base[1::3, 3:35][:230]), (100, base[5:105, 7:8]), (300, base[:300, 8:72]),
                        (100, base.t()[:50].t()[:100]), (64, base[:1, :40].expand(64, 40))):
            loads = loads_of("skewed", n, 5, n)
            order = order_of(loads, n, dev)
            inner = view.shape[1]
            big = normal(5, 160, 170, dtype=dtype, dev=dev, seed=2)
            for w in (big[:, :inner, 3:60], big[:, 2:inner + 2, 8:72], big.transpose(1, 2)[:, :inner, :33],
                      big[:, ::2, ::3][:, :inner, :20] if inner <= 80 else big[:, :inner, :20], big[:1, :inner, :40].expand(5, inner, 40),
                      big[::2, :inner, :].repeat(2, 1, 1)[:5, :, 5:6]):
                plain = gs.ops.expert_matmul(view.contiguous(), order, w.contiguous())
                got = gs.ops.expert_matmul(view, order, w)
                want = formula(view, loads, w)
                within(got, want[0], want[1], inner, dtype)
                within(plain, want[0], want[1], inner, dtype)
                wide = normal(n, 2 * w.shape[2] + 1, dtype=dtype, dev=dev, seed=3)
                grad = wide[:, 1:w.shape[2] + 1]
                x2, w2 = view.detach().requires_grad_(True), w.detach().requires_grad_(True)
                a = torch.autograd.grad(gs.ops.expert_matmul(x2, order, w2), (x2, w2), grad)
                want = formula(view, loads, w, grad)
                within(a[0], want[2], want[3], w.shape[2], dtype)
                within(a[1], want[4], want[5], n, dtype)
        # (one value for all: the gradient of a sum)
        x, w = base[:100, :64].detach().requires_grad_(True), normal(5, 64, 24, dtype=dtype, dev=dev, seed=4).requires_grad_(True)
        order = order_of(loads_of("even", 100, 5, 1), 100, dev)
        a = torch.autograd.grad(gs.ops.expert_matmul(x, order, w).sum(), (x, w))
        b = torch.autograd.grad(gs.ops.expert_matmul(x, order, w), (x, w), torch.ones(100, 24, dtype=dtype, device=dev))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@gpu
def test_a_matrix_that_all_experts_share(dev):
    """The gradient of a broadcast matrix is the sum of the experts'."""
    w = normal(1, 24, 16, dtype=torch.float32, dev=dev, seed=1).requires_grad_(True)
    x = normal(90, 24, dtype=torch.float32, dev=dev, seed=2)
    grad = normal(90, 16, dtype=torch.float32, dev=dev, seed=3)
    loads = np.array([30, 0, 25, 35])
    dw, = torch.autograd.grad(gs.ops.expert_matmul(x, order_of(loads, 90, dev), w.expand(4, 24, 16)), w, grad)
    want = x.double().t() @ grad.double()
    assert (dw[0].double() - want).abs().max() <= 100 * 2.0 ** -23 * (x.abs().double().t() @ grad.abs().double()).max()


@gpu
def test_offsets_that_no_sort_left(dev):
    """Offsets beyond the rows, negative ones and ones that descend: nothing outside the results is touched."""
    x, w = whole(300, 24, dtype=torch.bfloat16, dev=dev, seed=1), whole(3, 24, 40, dtype=torch.bfloat16, dev=dev, seed=2)
    grad = whole(300, 40, dtype=torch.bfloat16, dev=dev, seed=3)
    p = torch.arange(300, device=dev, dtype=torch.int32)
    for at in ([0, 2 ** 40, 2 ** 40, 2 ** 62], [-5, 10, 20, 400], [0, 200, 100, 300], [300, 200, 100, 0], [-2 ** 62, -7, -1, -1],
               [0, 300, 0, 300], [-2 ** 63, 2 ** 63 - 1, -2 ** 63, 2 ** 63 - 1]):
        order = gs.ops.ExpertOrder(p, p, torch.tensor(at, device=dev))
        buffers = [torch.full((1 << 20,), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
        assert gs.ops.expert_matmul(x, order, w).shape == (300, 40)
        assert capi.expert_matmul_grad(grad, x, order.offsets).shape == (3, 24, 40)
        assert all(bool((b == 7).all()) for b in buffers)
    # a gap in front counts as no expert's rows but is not written; ascending ones from 0 are the sort's
    order = gs.ops.ExpertOrder(p, p, torch.tensor([0, 100, 100, 260], device=dev))
    got = gs.ops.expert_matmul(x, order, w)
    assert torch.equal(got[:100].float(), (x[:100].float() @ w[0].float()).bfloat16().float()) and not got[260:].any()


@gpu
def test_gradient_against_differences(dev):
    loads = np.array([2, 0, 3])
    order = order_of(loads, 6, dev)
    x, w, grad = (normal(*s, dtype=torch.float32, dev=dev, seed=i) for i, s in enumerate(((6, 5), (3, 5, 4), (6, 4))))
    vx, vw = normal(6, 5, dtype=torch.float32, dev=dev, seed=4), normal(3, 5, 4, dtype=torch.float32, dev=dev, seed=5)
    x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(gs.ops.expert_matmul(x, order, w), (x, w), grad)

    def along(h):
        with torch.no_grad():
            return (gs.ops.expert_matmul(x + h * vx, order, w + h * vw).double() * grad.double()).sum().item()

    # bilinear: the central difference is exact but for rounding; values below 4 + 4 each, five products of at most 64,
    # 24 outputs times gradients below 4, eight roundings each
    slope = (dx.double() * vx.double()).sum().item() + (dw.double() * vw.double()).sum().item()
    assert abs((along(1.0) - along(-1.0)) / 2 - slope) < 24 * 5 * 64 * 4 * 8 * 2.0 ** -24


@gpu
def test_recorded_and_replayed(dev):
    """Products and gradients in one HIP graph, with other offsets and values at each replay."""
    for n, experts, inner, outer, dtype in ((12, 16, 64, 96, torch.bfloat16), (3000, 7, 136, 72, torch.float16),
                                            (70_000, 3, 16, 24, torch.float32)):
        order = order_of(loads_of("even", n, experts, 0), n, dev)
        x, w = whole(n, inner, dtype=dtype, dev=dev, seed=1), whole(experts, inner, outer, dtype=dtype, dev=dev, seed=2)
        x.requires_grad_(True), w.requires_grad_(True)
        grad = whole(n, outer, dtype=dtype, dev=dev, seed=3)

        def step():
            out = gs.ops.expert_matmul(x, order, w)
            return (out.detach(),) + torch.autograd.grad(out, (x, w), grad)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for rep in range(4):
            loads = loads_of("skewed" if rep % 2 else "even", n, experts, rep)
            order.offsets.copy_(torch.from_numpy(np.append(0, np.cumsum(loads))))
            with torch.no_grad():
                x.copy_(whole(n, inner, dtype=dtype, dev=dev, seed=10 + rep))
            want = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b, c in zip(got, want, formula(x, loads, w, grad)[::2]):
                assert torch.equal(a, b) and torch.equal(a.double(), c.to(dtype).double())


@gpu
def test_recording_is_refused_where_it_would_end_the_process(dev):
    order = order_of(np.array([2, 2]), 4, dev)
    x = normal(4, 8, dtype=torch.float32, dev=dev, seed=1).requires_grad_(True)
    w = normal(2, 8, 3, dtype=torch.float32, dev=dev, seed=2).requires_grad_(True)
    eager = gs.ops.expert_matmul(x, order, w)
    torch.cuda.synchronize()
    graph, messages = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        kept = x.detach() * 2
        for call in (lambda: gs.ops.expert_matmul(x, order, w.detach()), lambda: gs.ops.expert_matmul(x.detach(), order, w)):
            try:
                call()
            except RuntimeError as error:
                messages.append(str(error))
    assert len(messages) == 2 and all("eager graph of the same leaf" in m for m in messages)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, x.detach() * 2)
    torch.autograd.grad(eager.sum(), (x, w))


@gpu
def test_two_streams_and_threads_at_once(dev):
    import threading
    work = []
    for seed in (1, 2):
        loads = loads_of("skewed", 40_000, 3, seed)
        order = order_of(loads, 40_000, dev)
        x, g = (whole(40_000, d, dtype=torch.float16, dev=dev, seed=seed + d) for d in (40, 32))
        w = whole(3, 40, 32, dtype=torch.float16, dev=dev, seed=seed)
        work.append((x, g, w, order, [t.to(torch.float16) for t in formula(x, loads, w, g)[::4]]))
    torch.cuda.synchronize()
    wrong = []

    def run(x, g, w, order, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not (torch.equal(gs.ops.expert_matmul(x, order, w), want[0]) and
                        torch.equal(torch.ops.gs_ops._CAPI_ExpertMatmulGrad(g, x, order.offsets), want[1])):
                    wrong.append(1)

    threads = [threading.Thread(target=run, args=t) for t in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@gpu
def test_offsets_beyond_32_bits(dev):
    """More than 2^32 values in rows, results and matrices: both ends against the formula."""
    if torch.cuda.mem_get_info(dev)[0] < 120 << 30:
        pytest.skip("needs about 60 GB of free device memory")
    n, inner, outer = 4_300_000, 1024, 1032
    x = torch.zeros(n, inner, dtype=torch.bfloat16, device=dev)
    some = torch.cat([torch.arange(300, device=dev), torch.arange(n - 400, n, device=dev)])
    x[some] = whole(700, inner, dtype=torch.bfloat16, dev=dev, seed=1)
    w = whole(2, inner, outer, dtype=torch.bfloat16, dev=dev, seed=2)
    p = torch.zeros(n, dtype=torch.int32, device=dev)
    order = gs.ops.ExpertOrder(p, p, torch.tensor([0, n - 399, n - 10], device=dev))
    out = gs.ops.expert_matmul(x, order, w)
    e = torch.where(some < n - 399, 0, 1)
    for k in (0, 1):
        mine = (e == k) & (some < n - 10)
        assert torch.equal(out[some[mine]].double(), torch.mm(x[some[mine]].double(), w[k].double()).bfloat16().double())
    assert not out[n - 10:].any() and not out[300:n - 400:1000].any()
    dw = capi.expert_matmul_grad(out, x, order.offsets)
    want = torch.mm(x[some[e == 0]].double().t().contiguous(), out[some[e == 0]].double())
    size = torch.mm(x[some[e == 0]].double().abs().t().contiguous(), out[some[e == 0]].double().abs())
    within(dw[0], want, size, 701, torch.bfloat16)
    del out, x, dw
    # matrices of 2^32 values together, the last expert's rows
    experts = 4200
    w = torch.zeros(experts, inner, inner, dtype=torch.bfloat16, device=dev)
    w[-1] = whole(inner, inner, dtype=torch.bfloat16, dev=dev, seed=3)
    for rows in (3, 300):
        x = whole(rows, inner, dtype=torch.bfloat16, dev=dev, seed=4)
        at = torch.zeros(experts + 1, dtype=torch.int64, device=dev)
        at[-1] = rows
        order = gs.ops.ExpertOrder(p[:rows], p[:rows], at)
        for weight, m in ((w, w[-1]), (w.transpose(1, 2), w[-1].t())):
            got = gs.ops.expert_matmul(x, order, weight)
            assert torch.equal(got.double(), torch.mm(x.double(), m.double().contiguous()).bfloat16().double())


@gpu
def test_rows_far_apart(dev):
    """Rows and matrices' rows so far apart that a tile's addresses do not fit 32 bits."""
    if torch.cuda.mem_get_info(dev)[0] < 60 << 30:
        pytest.skip("needs about 24 GB of free device memory")
    flat = torch.zeros(5_000_000_000, dtype=torch.bfloat16, device=dev)
    far = flat.as_strided((300, 64), (16_000_000, 1))
    far.copy_(whole(300, 64, dtype=torch.bfloat16, dev=dev, seed=1))
    w = whole(2, 64, 72, dtype=torch.bfloat16, dev=dev, seed=2)
    loads = np.array([140, 150])
    order = order_of(loads, 300, dev)
    grad = whole(300, 72, dtype=torch.bfloat16, dev=dev, seed=3)
    want = formula(far, loads, w, grad)
    assert torch.equal(gs.ops.expert_matmul(far, order, w).double(), want[0].bfloat16().double())
    assert torch.equal(capi.expert_matmul_grad(grad, far, order.offsets).double(), want[4].bfloat16().double())
    x = whole(300, 300, dtype=torch.bfloat16, dev=dev, seed=4)
    wide = flat.as_strided((1, 300, 64), (0, 16_000_000, 1))
    out = gs.ops.expert_matmul(x, order_of(np.array([300]), 300, dev), wide)
    assert torch.equal(out.double(), torch.mm(x.double(), far.double().contiguous()).bfloat16().double())
    out = gs.ops.expert_matmul(whole(300, 64, dtype=torch.bfloat16, dev=dev, seed=5), order_of(np.array([300]), 300, dev),
                               wide.transpose(1, 2))
    want = torch.mm(whole(300, 64, dtype=torch.bfloat16, dev=dev, seed=5).double(), far.double().t().contiguous())
    assert torch.equal(out.double(), want.bfloat16().double())


@gpu
def test_refusals(dev):
    x, w = normal(10, 4, dtype=torch.float32, dev=dev, seed=1), normal(3, 4, 5, dtype=torch.float32, dev=dev, seed=2)
    order = order_of(np.array([3, 3, 4]), 10, dev)
    for bad, match in (((x.double(), order, w), "float32, float16 or bfloat16"), ((x.half(), order, w), "differ in type"),
                       ((x[0], order, w), "two dimensions"), ((x[:9], order, w), "rows of 9"), ((x, order, w[0]), "inner, outer"),
                       ((x, order, w[:2]), "offsets must be"), ((x[:, :3], order, w), "rows of 3 values"),
                       ((x.cpu(), order, w), "GPU tensor"), ((x, order, w.cpu()), "GPU tensor"),
                       ((x, order._replace(offsets=order.offsets.int()), w), "int64"),
                       ((x, order._replace(offsets=order.offsets.cpu()), w), "GPU tensor"),
                       ((x, order._replace(order=order.order[:5]), w), "order must be")):
        with pytest.raises(RuntimeError, match=match):
            gs.ops.expert_matmul(*bad)
    with pytest.raises(RuntimeError, match="gradient of 9 rows"):
        torch.ops.gs_ops._CAPI_ExpertMatmulGrad(normal(9, 5, dtype=torch.float32, dev=dev, seed=1), x, order.offsets)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    for of in (x, w):
        with pytest.raises(RuntimeError, match="once more"):
            torch.autograd.grad(gs.ops.expert_matmul(x, order, w).sum(), of, create_graph=True)
    torch.autograd.grad(gs.ops.expert_matmul(x, order, w.detach()).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gs.ops.expert_matmul(t, order, w.detach()).sum())(x.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y = x * 1.0
        out = gs.ops.expert_matmul(y, order, w)
        y.detach().zero_()
        torch.autograd.grad(out.sum(), w)


@gpu
def test_a_layer_of_experts_end_to_end(dev):
    """A router, rows out, two products with an activation between, back with weights, dropout on the way to the
    tokens: every output and every leaf's gradient against the same layer written in 64-bit torch."""
    T, D, H, E, K = 700, 48, 72, 9, 2
    leaves = [normal(*s, dtype=torch.float32, dev=dev, seed=i) * by for i, (s, by) in enumerate(
        [((T, D), 1.0), ((D, E), 0.3), ((E, D, H), 0.15), ((E, D, H), 0.12)])]
    grad = normal(T, D, dtype=torch.float32, dev=dev, seed=9)
    for normalize in (True, False):
        x, router, w_in, w_out = (t.clone().requires_grad_(True) for t in leaves)
        chosen, weights = gs.ops.expert_choose(x @ router, K, normalize)
        rows, order = gs.ops.expert_dispatch(x, chosen, E)
        h = torch.nn.functional.silu(gs.ops.expert_matmul(rows, order, w_in))
        y = gs.ops.expert_combine(gs.ops.expert_matmul(h, order, w_out.transpose(1, 2)), order, weights)
        out = gs.ops.dropout(y, 0.25, seed=5, residual=x)
        got = (out,) + torch.autograd.grad(out, (x, router, w_in, w_out), grad)

        kept = gs.ops.dropout(torch.ones(T, D, device=dev), 0.25, seed=5) != 0
        x, router, w_in, w_out = (t.double().requires_grad_(True) for t in leaves)
        logits = x @ router
        value = torch.take_along_dim(logits, chosen.long(), 1)
        share = value.softmax(1) if normalize else torch.take_along_dim(logits.softmax(1), chosen.long(), 1)
        h = torch.nn.functional.silu((x[:, None, None, :] @ w_in[chosen.long()])[:, :, 0])
        y = ((h[:, :, None, :] @ w_out.transpose(1, 2)[chosen.long()])[:, :, 0] * share[:, :, None]).sum(1)
        out = torch.where(kept, y / 0.75, 0.0) + x
        want = (out,) + torch.autograd.grad(out, (x, router, w_in, w_out), grad.double())
        # chains of at most T * K additions and 300 operations in values of unit size
        for a, b in zip(got, want):
            assert (a.double() - b).abs().max() <= (T * K + 300) * 2.0 ** -23 * b.abs().max()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_with_small_matrices(dev, dtype):
    """Types of nodes: from 2^18 rows on (fp32 2^19), matrices of a few dozen to a few hundred values a side; whole numbers."""
    n = (1 << (19 if dtype == torch.float32 else 18)) + 77
    for experts, inner, outer, kind, transposed in (
            (5, 100, 128, "skewed", False), (5, 128, 100, "skewed", True), (64, 8, 8, "skewed", False), (16, 8, 8, "skewed", True), (3, 33, 65, "even", True),
            (1, 256, 64, "first", False), (2, 31, 9, "last", False), (4, 64, 127, "skewed", True), (0, 16, 24, "none", False),
            (7, 129, 40, "skewed", True), (3, 40, 333, "skewed", False), (2, 33, 517, "last", False), (9, 64, 200, "skewed", True),
            (2, 9, 15, "none", False), (65, 40, 24, "even", False), (3, 16, 7, "skewed", False)):
        loads = loads_of(kind, n, experts, experts + inner)
        order = order_of(loads, n, dev)
        rows = whole(n, inner, dtype=dtype, dev=dev, seed=inner)
        weight = weights_of(whole, experts, inner, outer, transposed, dtype=dtype, dev=dev, seed=outer)
        want = formula(rows, loads, weight)[0].to(dtype)
        assert torch.equal(gs.ops.expert_matmul(rows, order, weight), want)
        wide = whole(n, inner + 3, dtype=dtype, dev=dev, seed=1)  # rows that lie apart, at odd places
        assert torch.equal(gs.ops.expert_matmul(wide[:, 2:inner + 2], order, weight),
                           gs.ops.expert_matmul(wide[:, 2:inner + 2].contiguous(), order, weight))
        if experts > 1 and loads.min() > 0:  # what is others' does not matter
            at = np.append(0, np.cumsum(loads))
            rows[at[1]:at[2]], weight[1] = float("nan"), float("inf")
            rows[at[-1]:] = float("nan")
            got = gs.ops.expert_matmul(rows, order, weight)
            assert torch.equal(got[:at[1]], want[:at[1]]) and torch.equal(got[at[2]:], want[at[2]:])
            assert not got[at[1]:at[2]].isfinite().any()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_tiles_of_any_alignment(dev, dtype):
    """Widths that end a few values into a tile or a chunk, rows at odd places; whole numbers."""
    for n, experts, inner, outer, kind in ((12_100, 2, 259, 1027, "skewed"), (12_100, 2, 1027, 259, "first"),
                                           (9_001, 3, 1001, 1285, "even"), (6_000, 2, 2049, 1031, "skewed"),
                                           (30_000, 2, 513, 262, "even"), (3_000, 2, 1999, 1543, "last")):
        loads = loads_of(kind, n, experts, inner)
        order = order_of(loads, n, dev)
        for transposed in (False, True):
            rows = whole(n, inner + 2, dtype=dtype, dev=dev, seed=1)[:, 1:inner + 1]
            grad = whole(n, outer + 1, dtype=dtype, dev=dev, seed=2)[:, 1:]
            weight = weights_of(whole, experts, inner, outer, transposed, dtype=dtype, dev=dev, seed=3)
            if dtype == torch.float16:  # (within its range)
                rows, grad = rows.clamp(-1, 1), grad.clamp(-1, 1)
                rows, grad = (torch.cat([t, t[:, :1]], 1)[:, :t.shape[1]] for t in (rows, grad))
            x, w = rows.detach().requires_grad_(True), weight.detach().requires_grad_(True)
            out = gs.ops.expert_matmul(x, order, w)
            got = torch.autograd.grad(out, (x, w), grad)
            want = formula(rows, loads, weight, grad)
            assert torch.equal(out, want[0].to(dtype))
            assert torch.equal(got[0], want[2].to(dtype)) and torch.equal(got[1], want[4].to(dtype))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_few_rows_and_long_depths(dev, dtype):
    """The depth shared out: from one tile of columns to many, depths that end anywhere, whole numbers."""
    for n, experts, inner, outer, kind in ((7, 4, 3497, 70, "skewed"), (160, 4, 3500, 72, "even"), (40, 4, 2053, 1030, "skewed"),
                                           (16, 16, 1001, 333, "even"), (300, 3, 4096, 33, "skewed"), (500, 4, 2048, 1024, "even"),
                                           (33, 2, 777, 31, "last"), (64, 64, 520, 1290, "skewed"), (90, 1, 1600, 9, "first"),
                                           (200, 4, 6400, 2500, "even")):
        loads = loads_of(kind, n, experts, inner)
        order = order_of(loads, n, dev)
        for transposed in (False, True):
            rows = whole(n, inner, dtype=dtype, dev=dev, seed=1)
            weight = weights_of(whole, experts, inner, outer, transposed, dtype=dtype, dev=dev, seed=2)
            got = gs.ops.expert_matmul(rows, order, weight)
            assert torch.equal(got, formula(rows, loads, weight)[0].to(dtype))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_sizes_between_few_and_many(dev, dtype):
    """Every tile and number of steps on the way, with rows behind the last and experts without any; whole numbers."""
    for n, experts, inner, outer, kind in ((6000, 3, 300, 512, "skewed"), (3000, 3, 1152, 896, "even"), (20_000, 2, 512, 512, "skewed"),
                                           (1500, 40, 320, 384, "skewed"), (4000, 4, 1003, 341, "skewed"), (700, 2, 96, 64, "even"),
                                           (9000, 30, 256, 264, "even"), (16_000, 10, 130, 400, "skewed"), (2500, 1, 2000, 200, "first")):
        loads = loads_of(kind, n, experts, inner)
        order = order_of(loads, n, dev)
        for transposed in (False, True):
            rows, grad = (whole(n, d, dtype=dtype, dev=dev, seed=d).clamp(-1, 1) for d in (inner, outer))
            weight = weights_of(whole, experts, inner, outer, transposed, dtype=dtype, dev=dev, seed=3)
            x, w = rows.requires_grad_(True), weight.detach().requires_grad_(True)
            out = gs.ops.expert_matmul(x, order, w)
            got = torch.autograd.grad(out, (x, w), grad)
            want = formula(rows, loads, weight, grad)
            assert torch.equal(out, want[0].to(dtype))
            assert torch.equal(got[0], want[2].to(dtype)) and torch.equal(got[1], want[4].to(dtype))


@gpu
def test_many_rows_and_offsets_that_no_sort_left(dev):
    n = (1 << 18) + 9
    x, w = whole(n, 40, dtype=torch.bfloat16, dev=dev, seed=1), whole(3, 40, 56, dtype=torch.bfloat16, dev=dev, seed=2)
    grad = whole(n, 56, dtype=torch.bfloat16, dev=dev, seed=3)
    p = torch.arange(n, device=dev, dtype=torch.int32)
    for at in ([0, 2 ** 40, 2 ** 40, 2 ** 62], [-5, 10, 20, n + 400], [0, n, 100, 3], [n, 200, 100, 0], [-2 ** 62, -7, -1, -1],
               [0, n, 0, n], [-2 ** 63, 2 ** 63 - 1, -2 ** 63, 2 ** 63 - 1]):
        order = gs.ops.ExpertOrder(p, p, torch.tensor(at, device=dev))
        buffers = [torch.full((1 << 20,), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
        assert gs.ops.expert_matmul(x, order, w).shape == (n, 56)
        assert capi.expert_matmul_grad(grad, x, order.offsets).shape == (3, 40, 56)
        assert all(bool((b == 7).all()) for b in buffers)
    order = gs.ops.ExpertOrder(p, p, torch.tensor([0, 100, 100, 200_000], device=dev))
    got = gs.ops.expert_matmul(x, order, w)
    assert torch.equal(got[:100].float(), (x[:100].float() @ w[0].float()).bfloat16().float())
    assert torch.equal(got[100:200_000].float(), (x[100:200_000].float() @ w[2].float()).bfloat16().float())
    assert not got[200_000:].any()


@gpu
def test_values_below_the_normal_ones(dev):
    """The smallest numbers of a type count like others."""
    for dtype, small, large in ((torch.float16, 2.0 ** -24, 2.0 ** 12), (torch.bfloat16, 2.0 ** -133, 2.0 ** 100),
                                (torch.float32, 2.0 ** -149, 2.0 ** 100)):
        for n, inner, outer in ((20, 64, 72), (700, 200, 136), ((1 << 19) + 5, 32, 24)):
            x = (whole(n, inner, dtype=torch.float64, dev=dev, seed=1) * small).to(dtype)
            w = (whole(2, inner, outer, dtype=torch.float64, dev=dev, seed=2) * large).to(dtype)
            loads = np.array([n // 2, n - n // 2])
            want = formula(x, loads, w)[0]
            assert (want != 0).any()
            assert torch.equal(gs.ops.expert_matmul(x, order_of(loads, n, dev), w), want.to(dtype))


@gpu
def test_as_many_experts_as_there_may_be(dev):
    n, experts = 70_000, 65_536
    loads = loads_of("even", n, experts, 1)
    order = order_of(loads, n, dev)
    rows, weight = (whole(*s, dtype=torch.bfloat16, dev=dev, seed=s[-1]) for s in ((n, 16), (experts, 16, 24)))
    grad = whole(n, 24, dtype=torch.bfloat16, dev=dev, seed=3)
    of = torch.repeat_interleave(torch.arange(experts, device=dev), torch.from_numpy(loads).to(dev))
    want = (rows.float()[:, :, None] * weight.float()[of]).sum(1)
    assert torch.equal(gs.ops.expert_matmul(rows, order, weight).float(), want.bfloat16().float())
    dw = torch.zeros(experts, 16, 24, device=dev).index_add_(0, of, rows.float()[:, :, None] * grad.float()[:, None])
    assert torch.equal(capi.expert_matmul_grad(grad, rows, order.offsets).float(), dw.bfloat16().float())
    too_many = gs.ops.ExpertOrder(order.order, order.place, torch.zeros(experts + 2, dtype=torch.int64, device=dev))
    with pytest.raises(RuntimeError, match="experts"):
        gs.ops.expert_matmul(rows, too_many, weight[:1].expand(experts + 1, 16, 24))


@gpu
def test_more_tiles_than_one_launch_has_workgroups_for(dev):
    """Of as many experts as there may be, wide matrices: more than 2^24 workgroups of 256 threads, or 2^23 of 512.  Whole numbers."""
    if torch.cuda.mem_get_info(dev)[0] < 100 << 30:
        pytest.skip("needs about 40 GB of free device memory")
    n, experts = 70_000, 65_536
    loads = loads_of("even", n - 40, experts, 2)
    order = order_of(loads, n, dev)
    of = torch.repeat_interleave(torch.arange(experts, device=dev), torch.from_numpy(loads).to(dev))
    live = of.numel()
    some = torch.cat([torch.arange(200, device=dev), torch.randint(live, (600,), device=dev), torch.arange(live - 200, live, device=dev)])
    for inner, outer in ((8, 16384), (128, 4096)):  # tiles of 64 x 64; few rows
        rows = whole(n, inner, dtype=torch.float32, dev=dev, seed=inner)
        # (matrices that overlap: each begins a value behind the one before)
        weight = whole(inner * outer + experts, dtype=torch.float32, dev=dev, seed=outer).as_strided((experts, inner, outer), (1, outer, 1))
        out = gs.ops.expert_matmul(rows, order, weight)
        for part in some.split(100):
            want = torch.bmm(rows[part][:, None].double(), weight[of[part]].double())[:, 0]
            assert torch.equal(out[part].double(), want)
        assert torch.equal(out[:live].double().sum(1), (rows[:live].double() * weight.sum(2).double()[of]).sum(1))
        assert not out[live:].any()
        del out, weight
    inner, outer = 4, 16448
    rows, grad = (whole(n, d, dtype=torch.float32, dev=dev, seed=d) for d in (inner, outer))
    dw = capi.expert_matmul_grad(grad, rows, order.offsets)
    want = torch.zeros(experts, inner, device=dev).index_add_(0, of, rows[:live] * grad[:live].sum(1, keepdim=True))
    assert torch.equal(dw.sum(2), want)
    for e in [0, 1, 2, 12_345, 65_534, 65_535]:
        mine = of == e
        assert torch.equal(dw[e], rows[:live][mine].t() @ grad[:live][mine])


# ------------------------------------------------------------------ no GPU ----
def test_bad_arguments_are_refused_before_anything_is_launched():
    import ctypes
    lib, i64 = capi.lib(), ctypes.c_int64
    buf = (ctypes.c_int64 * 64)()
    at = ctypes.addressof(buf)

    def fails(status, match):
        assert status < 0 and match in lib.gs_status_string(status), (status, lib.gs_status_string(status))

    def matmul(rows=buf, stride=8, n=4, inner=8, kind=0, weight=buf, estride=64, wstride=8, transposed=0, num=3, outer=8,
               offsets=buf, out=buf):
        return lib.gs_expert_matmul(rows, i64(stride), i64(n), i64(inner), kind, weight, i64(estride), i64(wstride), transposed,
                                    i64(num), i64(outer), offsets, out, None)

    assert matmul(n=0) == matmul(outer=0) == 0
    for change, match in ((dict(kind=7), b"value type"), (dict(n=-1), b"negative"), (dict(n=1 << 31), b"2^31"),
                          (dict(inner=1 << 24), b"2^24"), (dict(outer=1 << 24), b"2^24"), (dict(num=1 << 31), b"experts"),
                          (dict(stride=-1), b"stride"), (dict(wstride=-1), b"stride"), (dict(offsets=None), b"null"),
                          (dict(rows=None), b"null"), (dict(weight=None), b"null"), (dict(out=None), b"null"),
                          (dict(rows=ctypes.c_void_p(at + 2)), b"aligned"), (dict(weight=ctypes.c_void_p(at + 1)), b"aligned")):
        fails(matmul(**change), match)

    def grad(rows=buf, rstride=8, inner=8, g=buf, gstride=8, outer=8, kind=0, n=4, offsets=buf, num=3, out=buf, ws=buf,
             ws_bytes=256):
        return lib.gs_expert_matmul_grad(rows, i64(rstride), i64(inner), g, i64(gstride), i64(outer), kind, i64(n), offsets,
                                         i64(num), out, ws, ctypes.c_size_t(ws_bytes), None)

    sizes = lib.gs_expert_matmul_grad_workspace_bytes
    assert sizes(i64(100), i64(64), i64(64), i64(4)) == 256
    for bad in ((-1, 64, 64, 4), (1 << 31, 64, 64, 4), (1 << 30, 1 << 24, 64, 4), (1 << 30, 64, 1 << 40, 4), (1 << 30, 64, 64, 1 << 31),
                (1 << 30, 64, 64, -1)):
        assert sizes(*(i64(v) for v in bad)) == 256
    assert sizes(i64(1 << 20), i64(64), i64(128), i64(3)) > 512 * 64 * 128 * 4
    fails(grad(n=1 << 20, num=3), b"workspace")

    assert grad(inner=0) == grad(outer=0) == grad(num=0) == 0
    for change, match in ((dict(kind=7), b"value type"), (dict(n=-1), b"negative"), (dict(n=1 << 31), b"2^31"),
                          (dict(inner=1 << 24), b"2^24"), (dict(num=1 << 31), b"experts"), (dict(gstride=-1), b"stride"),
                          (dict(offsets=None), b"null"), (dict(rows=None), b"null"), (dict(g=None), b"null"),
                          (dict(out=None), b"null"), (dict(g=ctypes.c_void_p(at + 2)), b"aligned")):
        fails(grad(**change), match)


def test_cpu_tensors_are_refused():
    p = torch.zeros(3, dtype=torch.int32)
    order = gs.ops.ExpertOrder(p, p, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        gs.ops.expert_matmul(torch.zeros(3, 4), order, torch.zeros(2, 4, 5))


def test_matrices_that_are_none_are_refused_alike_with_and_without_gradients():
    p = torch.zeros(3, dtype=torch.int32)
    order = gs.ops.ExpertOrder(p, p, torch.zeros(3, dtype=torch.int64))
    for shape in ((4, 5), (4,), (), (2, 4, 5)):
        for followed in (False, True):
            with pytest.raises(RuntimeError, match="GPU tensor"):
                gs.ops.expert_matmul(torch.zeros(3, 4), order, torch.zeros(shape, requires_grad=followed))


@gpu
def test_matrices_of_two_dimensions_are_refused_with_gradients(dev):
    x = normal(10, 4, dtype=torch.float32, dev=dev, seed=1)
    order = order_of(np.array([3, 3, 4]), 10, dev)
    for shape in ((4, 5), (4,)):
        with pytest.raises(RuntimeError, match="inner, outer"):
            gs.ops.expert_matmul(x, order, torch.zeros(shape, device=dev, requires_grad=True))


def test_more_experts_than_are_taken():
    import ctypes
    lib, i64 = capi.lib(), ctypes.c_int64
    buf = (ctypes.c_int64 * 64)()
    rc = lib.gs_expert_matmul(buf, i64(8), i64(4), i64(8), 0, buf, i64(64), i64(8), 0, i64(65537), i64(8), buf, buf, None)
    assert rc < 0 and b"65537 experts" in lib.gs_status_string(rc)
    rc = lib.gs_expert_matmul_grad(buf, i64(8), i64(8), buf, i64(8), i64(8), 0, i64(4), buf, i64(65537), buf, buf,
                                   ctypes.c_size_t(256), None)
    assert rc < 0 and b"65537 experts" in lib.gs_status_string(rc)
    assert lib.gs_expert_matmul_grad_workspace_bytes(i64(1 << 30), i64(8), i64(8), i64(65537)) == 256
