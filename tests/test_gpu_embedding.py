"""gs.ops.embedding against the formulas in 64 bits.

Tolerances.  A looked-up value is one fp32 product (relative error 2^-24) rounded once (eps / 2 of its type).
A gradient is a sum of m fp32 values by sums of sums: at most 32 + 64 * 5 additions lie on any value's way
(tiles of up to 32 positions, then up to 64 entries a level), each off by 2^-24 of a partial sum that is
at most the sum S of the magnitudes, and one product; so it is off by (min(m, 352) + 1) * 2^-24 * scale * S before it
is rounded once."""
import math

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


def smallest(dtype):  # half of the least subnormal: what rounding near zero is off by
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rows(n, dim, dtype, dev, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, dim, generator=g).to(dtype).to(dev)


def ids_of(kind, n, num_rows, seed, idt=np.int64):
    rng = np.random.default_rng(seed)
    if kind == "even":
        ids = rng.integers(0, num_rows, n)
    elif kind == "skewed":
        ids = (num_rows ** rng.random(n)).astype(np.int64) - 1
    elif kind == "one":
        ids = np.full(n, num_rows // 2)
    elif kind == "none":
        ids = np.full(n, -1)
    elif kind == "outside":  # beyond both ends, and as far as the type goes
        ids = rng.integers(-2, num_rows + 2, n)
        ids[rng.random(n) < 0.1] = np.iinfo(idt).max
        ids[rng.random(n) < 0.1] = np.iinfo(idt).min
    elif kind == "sorted":
        ids = np.sort(rng.integers(0, num_rows, n))
    elif kind == "hub":  # half of all on one row, the rest anywhere, a few nowhere
        ids = np.where(rng.random(n) < 0.5, num_rows - 1, rng.integers(0, num_rows, n))
        ids[rng.random(n) < 0.05] = -1
    return ids.astype(idt)


def check_lookup(out, table, ids, scale):
    t = table.double().cpu().numpy()
    there = (ids >= 0) & (ids < t.shape[0])
    want = np.zeros(ids.shape + (t.shape[1],))
    want[there] = t[ids[there]] * float(np.float32(scale))
    got = out.detach().double().cpu().numpy()
    assert got.shape == want.shape
    assert np.all(np.abs(got - want) <= np.abs(want) * (half_step(out.dtype) + 2 * F32) + smallest(out.dtype))
    assert np.all(got[~there] == 0)


def sums_by_id(grad, ids, num_rows, scale):
    """(sums, tolerance before rounding)"""
    g = grad.double().cpu().numpy().reshape(ids.size, grad.shape[-1])
    flat = ids.reshape(-1)
    there = np.flatnonzero((flat >= 0) & (flat < num_rows))
    want = np.zeros((num_rows, g.shape[1]))
    size = np.zeros_like(want)
    np.add.at(want, flat[there], g[there])
    np.add.at(size, flat[there], np.abs(g[there]))
    m = np.bincount(flat[there], minlength=num_rows)[:, None]
    s = abs(float(np.float32(scale)))
    return want * float(np.float32(scale)), (np.minimum(m, 352) + 1) * F32 * s * size


def check_sums(got, want, tol, dtype):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape
    assert np.all(np.abs(got - want) <= tol + (np.abs(want) + tol) * half_step(dtype) + smallest(dtype))


CASES = [
    # rows, width, ids, kind
    (1, 1, 1, "even"), (7, 3, 5, "outside"), (100, 8, 64, "even"), (50, 4, 300, "skewed"), (33, 17, 1000, "outside"),
    (1000, 64, 4096, "hub"), (1000, 64, 4097, "hub"), (3000, 97, 5000, "skewed"), (70000, 16, 9000, "even"),
    (300, 520, 700, "one"), (255, 1001, 333, "none"), (256, 1032, 2000, "sorted"), (257, 130, 50000, "one"),
    (12, 2, 200000, "hub"), (1 << 17, 5, 30000, "even"), (5, 4096, 9, "even"), (20, 8, 0, "even"), (20000000, 1, 5000, "even"),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("num_rows,dim,n,kind", CASES)
def test_lookup_and_gradients(dev, num_rows, dim, n, kind, dtype):
    idt = np.int32 if (n + dim) % 2 else np.int64
    ids = ids_of(kind, n, num_rows, n + dim, idt)
    table = rows(num_rows, dim, dtype, dev, 1).requires_grad_(True)
    d_ids = torch.from_numpy(ids).to(dev)
    scale = math.sqrt(dim) if n % 2 else 1.0
    out = gs.ops.embedding(table, d_ids, scale)
    assert out.dtype == dtype
    check_lookup(out, table.detach(), ids, scale)
    grad = rows(n, dim, dtype, dev, 2)
    want, tol = sums_by_id(grad, ids, num_rows, scale)
    dense, = torch.autograd.grad(out, table, grad)
    assert dense.dtype == dtype and dense.layout == torch.strided
    check_sums(dense, want, tol, dtype)
    again, = torch.autograd.grad(gs.ops.embedding(table, d_ids, scale), table, grad)
    assert torch.equal(dense.view(torch.uint8), again.view(torch.uint8))
    sparse, = torch.autograd.grad(gs.ops.embedding(table, d_ids, scale, sparse_grad=True), table, grad)
    met = np.unique(ids[(ids >= 0) & (ids < num_rows)])
    assert sparse.is_sparse and sparse.is_coalesced() and sparse.shape == table.shape and sparse.dtype == dtype
    assert np.array_equal(sparse.indices()[0].cpu().numpy(), met)
    # the same sums in the same order: the same bits
    assert torch.equal(sparse.values(), dense[sparse.indices()[0]])
    # and through the C ABI by itself
    assert torch.equal(capi.embedding_lookup(table.detach(), d_ids, scale), out)
    assert torch.equal(capi.embedding_grad(grad, d_ids, num_rows, scale), dense)
    c_met, c_values = capi.embedding_sparse_grad(grad, d_ids, num_rows, scale)
    assert torch.equal(c_met, sparse.indices()[0]) and torch.equal(c_values, sparse.values())


@gpu
@pytest.mark.parametrize("num_rows", [1, 200, 255, 256, 65535, 70000, (1 << 18) - 1, 1 << 18, 5_000_000, 140_000_000, 2 ** 32 - 2])
def test_sorts_of_every_size_and_key(dev, num_rows):
    """Both sides of every size at which the sort changes its tiles or launches, with keys of one to four digits of
    eight and nine bits.  Whole numbers, whose sums fp32 holds exactly whatever the order."""
    rng = np.random.default_rng(num_rows % 1000)
    for n in (1, 63, 1024, 1025, 2049, 4096, 4097, 16384, 16385, 65536, 65537, 131072, 131073, 524288, 524289):
        ids = rng.integers(-1, num_rows, n)
        if n > 2000:  # a run that goes through many tiles
            ids[n // 3:n // 2] = num_rows - 1
        grad = rng.integers(-8, 9, (n, 1)).astype(np.float32)
        met, values = torch.ops.gs_ops._CAPI_EmbeddingSparseGrad(torch.from_numpy(grad).to(dev),
                                                                 torch.from_numpy(ids).to(dev), num_rows, 1.0)
        want, which = np.unique(ids[ids >= 0], return_inverse=True)
        assert np.array_equal(met.cpu().numpy(), want)
        assert np.array_equal(values[:, 0].cpu().numpy(), np.bincount(which, grad[ids >= 0, 0], want.size))
        if num_rows <= 5_000_000:
            dense = torch.ops.gs_ops._CAPI_EmbeddingGrad(torch.from_numpy(grad).to(dev), torch.from_numpy(ids).to(dev),
                                                         num_rows, 1.0)
            assert torch.equal(dense[met], values) and int(dense.count_nonzero()) == int(values.count_nonzero())


@gpu
def test_values_near_zero_are_kept(dev):
    """Results below the smallest normal number are rounded, not dropped."""
    for dtype, power in ((torch.float32, -120), (torch.bfloat16, -120), (torch.float16, -12)):
        table = rows(20, 33, dtype, dev, 33).requires_grad_(True)
        ids = ids_of("even", 50, 20, 34)
        scale = 2.0 ** power * 2.0 ** (-9 if dtype != torch.float16 else -4)
        out = gs.ops.embedding(table, torch.from_numpy(ids).to(dev), scale)
        assert (out.detach().abs() < torch.finfo(dtype).smallest_normal).any() and out.detach().count_nonzero() > 0
        check_lookup(out, table.detach(), ids, scale)
        grad = rows(50, 33, dtype, dev, 35)
        got, = torch.autograd.grad(out, table, grad)
        want, tol = sums_by_id(grad, ids, 20, scale)
        check_sums(got, want, tol + smallest(torch.float32), dtype)  # (the product with the scale is fp32 and may be tiny)


@gpu
def test_offsets_beyond_32_bits(dev):
    """Tables, results and gradients of more than 2^32 values, the last rows among those that are named."""
    if torch.cuda.mem_get_info(dev)[0] < 80 << 30:
        pytest.skip("needs about 40 GB of free device memory")
    num_rows, dim = 70_000_000, 64
    table = torch.zeros(num_rows, dim, dtype=torch.float16, device=dev)
    named = torch.tensor([0, 1, 33_554_432, 67_108_863, 67_108_864, num_rows - 1], device=dev)
    table[named] = rows(named.numel(), dim, torch.float16, dev, 36)
    assert torch.equal(gs.ops.embedding(table, named), table[named])
    n = 68_000_000  # ids: the result is as large as the table
    ids = (torch.arange(n, device=dev, dtype=torch.int32) % 1000)
    ids[-3:] = torch.tensor([num_rows - 1, 67_108_864, -1], dtype=torch.int32, device=dev)
    out = gs.ops.embedding(table, ids)
    assert torch.equal(out[-3:-1], table[[num_rows - 1, 67_108_864]]) and not out[-1].any()
    assert torch.equal(out[66_999_000:67_000_000], table[:1000]) and torch.equal(out[:1000], table[:1000])
    # that result as a gradient: 68 k rows for each of a thousand ids, summed to 68 k (or fewer) times the same
    out.fill_(2.0 ** -17)
    met, sums = torch.ops.gs_ops._CAPI_EmbeddingSparseGrad(out, ids, num_rows, 1.0)
    counts = torch.bincount(ids[ids >= 0].long(), minlength=num_rows)
    assert torch.equal(met, counts.nonzero()[:, 0])
    want = counts[met].double() * 2.0 ** -17  # (exact in fp32: counts below 2^24)
    assert (sums.double() - want[:, None]).abs().max() <= want.max() * half_step(torch.float16)
    dense = torch.ops.gs_ops._CAPI_EmbeddingGrad(out, ids, num_rows, 1.0)
    assert torch.equal(dense[met], sums) and int(dense[:, 0].count_nonzero()) == met.numel()


@gpu
def test_two_threads_at_once(dev):
    """Gradients of both kinds by two threads on a stream each: nothing is shared between calls."""
    import threading
    work = []
    for seed in (37, 38):
        grad, ids = rows(30000, 24, torch.float32, dev, seed), torch.from_numpy(ids_of("hub", 30000, 900, seed)).to(dev)
        work.append((grad, ids, torch.ops.gs_ops._CAPI_EmbeddingGrad(grad, ids, 900, 1.0)))
    torch.cuda.synchronize()
    wrong = []

    def run(grad, ids, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                met, values = torch.ops.gs_ops._CAPI_EmbeddingSparseGrad(grad, ids, 900, 1.0)
                dense = torch.ops.gs_ops._CAPI_EmbeddingGrad(grad, ids, 900, 1.0)
                if not (torch.equal(dense, want) and torch.equal(dense[met], values)):
                    wrong.append(1)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@gpu
def test_rows_any_distance_apart_and_off_their_alignment(dev):
    for dtype in TYPES:
        base = rows(400, 61, dtype, dev, 3)
        for view in (base[:, 1:60], base[:, 3:35], base[::3, :40], base[5:, 7:8], base.t()[:50]):
            n = view.shape[0]
            ids = ids_of("outside", 777, n, 4)
            table = view.detach().requires_grad_(True)
            out = gs.ops.embedding(table, torch.from_numpy(ids).to(dev), 1.5)
            check_lookup(out, view, ids, 1.5)
            wide = rows(777, 2 * view.shape[1] + 1, dtype, dev, 5)
            grad = wide[:, 1:view.shape[1] + 1]
            got, = torch.autograd.grad(out, table, grad)
            check_sums(got, *sums_by_id(grad, ids, n, 1.5), dtype)
    # the same gradient row for every id, and one value for all of them
    table = rows(30, 12, torch.float32, dev, 6).requires_grad_(True)
    ids = ids_of("even", 100, 30, 7)
    d_ids = torch.from_numpy(ids).to(dev)
    row = rows(1, 12, torch.float32, dev, 8)
    got, = torch.autograd.grad(gs.ops.embedding(table, d_ids), table, row.expand(100, 12))
    check_sums(got, *sums_by_id(row.expand(100, 12).contiguous(), ids, 30, 1.0), torch.float32)
    got, = torch.autograd.grad(gs.ops.embedding(table, d_ids).sum(), table)
    check_sums(got, *sums_by_id(torch.ones(100, 12), ids, 30, 1.0), torch.float32)


@gpu
def test_ids_of_any_shape_and_order(dev):
    table = rows(40, 6, torch.float32, dev, 9).requires_grad_(True)
    ids = ids_of("even", 60, 40, 10).reshape(4, 5, 3)
    d_ids = torch.from_numpy(ids).to(dev)
    for view, host in ((d_ids, ids), (d_ids.transpose(0, 2), ids.transpose(2, 1, 0)), (d_ids[:, ::2], ids[:, ::2]),
                       (d_ids[1, 2, 0], ids[1, 2, 0]), (d_ids[:0], ids[:0]), (d_ids[0, 0, :1].expand(7), np.repeat(ids[0, 0, :1], 7))):
        host = np.asarray(host)
        out = gs.ops.embedding(table, view, 2.0)
        assert out.shape == host.shape + (6,)
        check_lookup(out, table.detach(), host, 2.0)
        grad = rows(host.size, 6, torch.float32, dev, 11).view(out.shape)
        got, = torch.autograd.grad(out, table, grad)
        check_sums(got, *sums_by_id(grad, host, 40, 2.0), torch.float32)


@gpu
def test_rows_that_no_id_names_do_not_matter(dev):
    """Infinities and NaN in rows of the table, and of the gradient, that stand for nothing."""
    table = rows(10, 20, torch.bfloat16, dev, 12)
    table[3] = float("nan")
    table[4] = float("inf")
    table.requires_grad_(True)
    ids = np.array([1, -1, 2, 10, 9, 1])
    out = gs.ops.embedding(table, torch.from_numpy(ids).to(dev), 0.0)
    assert torch.equal(out, torch.zeros_like(out))  # (a scale of zero, finite rows)
    out = gs.ops.embedding(table, torch.from_numpy(ids).to(dev), 3.0)
    check_lookup(out, torch.nan_to_num(table.detach(), 0, 0, 0), ids, 3.0)
    grad = rows(6, 20, torch.bfloat16, dev, 13)
    grad[1] = float("nan")
    grad[3] = float("inf")
    got, = torch.autograd.grad(out, table, grad)
    clean = grad.clone()
    clean[1] = clean[3] = 0
    check_sums(got, *sums_by_id(clean, ids, 10, 3.0), torch.bfloat16)
    # where they are named, they come through
    out = gs.ops.embedding(table, torch.tensor([3, 4], device=dev), 2.0)
    assert out[0].isnan().all() and out[1].isinf().all()


@gpu
def test_gradient_against_differences(dev):
    table = rows(9, 5, torch.float32, dev, 14)
    ids = torch.tensor([0, 3, 3, 8, -1, 3, 20], device=dev)
    grad, way = rows(7, 5, torch.float32, dev, 15), rows(9, 5, torch.float32, dev, 16)
    table.requires_grad_(True)
    got, = torch.autograd.grad(gs.ops.embedding(table, ids, 0.5), table, grad)
    with torch.no_grad():  # linear: any step will do; powers of two keep the steps exact to rounding
        up = (gs.ops.embedding(table + 4 * way, ids, 0.5).double() * grad.double()).sum()
        down = (gs.ops.embedding(table - 4 * way, ids, 0.5).double() * grad.double()).sum()
    # 14 looked-up rows of values below 32, each off by two roundings, times gradients below 8
    assert abs((up - down).item() / 8 - (got.double() * way.double()).sum().item()) < 35 * 32 * 8 * 2 * F32


@gpu
def test_accumulates_and_steps_like_a_parameter(dev):
    table = torch.nn.Parameter(rows(50, 8, torch.float32, dev, 17))
    ids = ids_of("hub", 40, 50, 18)
    d_ids = torch.from_numpy(ids).to(dev)
    gs.ops.embedding(table, d_ids).sum().backward()
    gs.ops.embedding(table, d_ids).sum().backward()  # twice the same: exactly twice the sums
    once, = torch.autograd.grad(gs.ops.embedding(table, d_ids).sum(), table)
    assert torch.equal(table.grad, 2 * once)
    table.grad = None
    before = table.detach().clone()
    optimizer = torch.optim.SparseAdam([table], lr=0.5)
    gs.ops.embedding(table, d_ids, sparse_grad=True).sum().backward()
    optimizer.step()
    moved = (table.detach() != before).any(1).cpu().numpy()
    assert np.array_equal(np.flatnonzero(moved), np.unique(ids[ids >= 0]))


@gpu
def test_recorded_lookup_and_gradient_follow_their_inputs(dev):
    """Forward and gradient in one HIP graph, ids and values rewritten between replays, eager work between."""
    for n, num_rows, dim in ((50, 30, 16), (6000, 500, 40), (9000, 70000, 8)):
        table = rows(num_rows, dim, torch.float32, dev, 19)
        grad = rows(n, dim, torch.float32, dev, 20)
        ids = torch.from_numpy(ids_of("hub", n, num_rows, 21)).to(dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            gs.ops.embedding(table, ids, 2.0)
            torch.ops.gs_ops._CAPI_EmbeddingGrad(grad, ids, num_rows, 2.0)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = gs.ops.embedding(table, ids, 2.0)
            got = torch.ops.gs_ops._CAPI_EmbeddingGrad(grad, ids, num_rows, 2.0)
        for rep in range(4):
            ids.copy_(torch.from_numpy(ids_of("outside" if rep % 2 else "skewed", n, num_rows, 30 + rep)))
            grad.copy_(rows(n, dim, torch.float32, dev, 40 + rep))
            want = torch.ops.gs_ops._CAPI_EmbeddingGrad(grad, ids, num_rows, 2.0)
            want_out = gs.ops.embedding(table, ids, 2.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want_out) and torch.equal(got, want)


@gpu
def test_recorded_backward_pass(dev):
    """forward + backward through autograd, recorded: no eager graph of the leaf lives."""
    table = rows(300, 24, torch.float32, dev, 22).requires_grad_(True)
    grad = rows(700, 24, torch.float32, dev, 23)
    ids = torch.from_numpy(ids_of("skewed", 700, 300, 24)).to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(gs.ops.embedding(table, ids, 1.5), table, grad)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(gs.ops.embedding(table, ids, 1.5), table, grad)
    for rep in range(3):
        grad.copy_(rows(700, 24, torch.float32, dev, 50 + rep))
        want, = torch.autograd.grad(gs.ops.embedding(table, ids, 1.5), table, grad)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@gpu
def test_recording_is_refused_where_it_would_end_the_process(dev):
    table = rows(30, 8, torch.float32, dev, 25).requires_grad_(True)
    ids = torch.arange(10, device=dev)
    eager = gs.ops.embedding(table, ids)  # lives through the recording, on the default stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    message = None
    with torch.cuda.graph(graph):
        try:
            gs.ops.embedding(table, ids)
        except RuntimeError as error:
            message = str(error)
        plain = gs.ops.embedding(table.detach(), ids)  # nothing flows back: recorded
    assert message and "eager graph of the same leaf" in message
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(plain, eager)
    torch.autograd.grad(eager.sum(), table)


@gpu
def test_recording_with_several_uses_of_a_leaf(dev):
    """Two lookups of one table, and one of a table made inside the recording: their nodes are on the recording
    stream.  A tensor made outside, and followed, is refused."""
    table = rows(40, 8, torch.float32, dev, 44).requires_grad_(True)
    a, b = torch.arange(30, device=dev), torch.arange(5, 25, device=dev)

    def step():
        first, second = gs.ops.embedding(table, a), gs.ops.embedding(table, b, 2.0)
        third = gs.ops.embedding(table * 3, a)
        return torch.autograd.grad((first * first).sum() + second.sum() + third.sum(), table)[0]

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
        with torch.no_grad():
            table.copy_(rows(40, 8, torch.float32, dev, 45 + rep))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    made = table * 2  # outside
    graph, message = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(graph):
        kept = made.detach() + 1
        try:
            gs.ops.embedding(made, a)
        except RuntimeError as error:
            message = str(error)
    assert message and "outside the recording" in message
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, made.detach() + 1)


@gpu
def test_in_a_compiled_sampler(dev):
    """A sampler that hands out its frontier's rows, as written and through jit.compile."""
    from tests.util import rmat_csc_np
    indptr, indices = rmat_csc_np(1 << 12, 1 << 16, seed=1)
    A = gs.Matrix().load_csc(torch.from_numpy(indptr).to(dev), torch.from_numpy(indices).to(dev))
    table = rows(1 << 12, 24, torch.bfloat16, dev, 48)

    def sampler(A, seeds, fanouts, table):
        blocks = []
        for k in fanouts:
            sub = A[:, seeds].columnwise_sampling(k, False)
            seeds = sub.all_indices()
            blocks.insert(0, sub.to_dgl_block())
        return seeds, blocks, gs.ops.embedding(table, seeds, 2.0)

    seeds = torch.randperm(1 << 12, device=dev)[:200]
    compiled = gs.jit.compile(sampler, (A, seeds[:4], [5, 3], table))
    for trial in range(2):
        gs.set_seed(60 + trial)
        nodes, _, h = sampler(A, seeds, [5, 3], table)
        gs.set_seed(60 + trial)
        got_nodes, _, got = compiled(A, seeds, [5, 3], table)
        assert torch.equal(nodes, got_nodes) and torch.equal(h, got)
        assert torch.equal(h, (table[nodes].float() * 2).bfloat16())


@gpu
def test_inference_mode(dev):
    with torch.inference_mode():
        table = rows(40, 8, torch.float32, dev, 47)
        ids = torch.arange(30, device=dev)
        assert torch.equal(gs.ops.embedding(table, ids), table[:30])


@gpu
def test_sparse_gradient_is_not_recorded(dev):
    grad, ids = rows(10, 8, torch.float32, dev, 26), torch.arange(10, device=dev)
    graph = torch.cuda.CUDAGraph()
    message = None
    with torch.cuda.graph(graph):
        kept = grad * 2
        try:
            torch.ops.gs_ops._CAPI_EmbeddingSparseGrad(grad, ids, 30, 1.0)
        except RuntimeError as error:
            message = str(error)
    assert message and "cannot be recorded" in message
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, grad * 2)


@gpu
def test_on_another_stream(dev):
    table = rows(2000, 32, torch.float32, dev, 27).requires_grad_(True)
    ids = torch.from_numpy(ids_of("hub", 20000, 2000, 28)).to(dev)
    grad = rows(20000, 32, torch.float32, dev, 29)
    want, = torch.autograd.grad(gs.ops.embedding(table, ids), table, grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, = torch.autograd.grad(gs.ops.embedding(table, ids), table, grad)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@gpu
def test_refusals(dev):
    table, ids = rows(5, 4, torch.float32, dev, 30), torch.zeros(3, dtype=torch.int64, device=dev)
    for bad, match in (((table.double(), ids), "float32, float16 or bfloat16"), ((table, ids.float()), "int64"),
                       ((table[0], ids), "two dimensions"), ((table.cpu(), ids), "GPU tensor"),
                       ((table, ids.cpu()), "GPU tensor"), ((table.to_sparse(), ids), "dense|subclasses")):
        with pytest.raises(RuntimeError, match=match):
            gs.ops.embedding(*bad)
    with pytest.raises(RuntimeError, match="for 3 ids|shape"):
        torch.ops.gs_ops._CAPI_EmbeddingGrad(rows(4, 4, torch.float32, dev, 31), ids, 5, 1.0)
    with pytest.raises(RuntimeError, match="non-negative"):
        torch.ops.gs_ops._CAPI_EmbeddingGrad(rows(3, 4, torch.float32, dev, 31), ids, -1, 1.0)
    leaf = table.clone().requires_grad_(True)
    out = gs.ops.embedding(leaf, ids)
    dout = rows(3, 4, torch.float32, dev, 32).requires_grad_(True)
    with pytest.raises(RuntimeError, match="once more"):
        torch.autograd.grad(out, leaf, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="once more"):
        torch.ops.gs_ops._CAPI_EmbeddingGrad(dout, ids, 5, 1.0)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gs.ops.embedding(t, ids).sum())(table)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
        gs.ops.embedding(torch.autograd.forward_ad.make_dual(table, table), ids)


@gpu
def test_null_and_empty(dev):
    ids = torch.zeros(4, dtype=torch.int32, device=dev)
    empty = torch.empty(0, 6, device=dev, requires_grad=True)
    out = gs.ops.embedding(empty, ids)
    assert torch.equal(out, torch.zeros(4, 6, device=dev))
    assert torch.autograd.grad(out.sum(), empty)[0].shape == (0, 6)
    sparse, = torch.autograd.grad(gs.ops.embedding(empty, ids, sparse_grad=True).sum(), empty)
    assert sparse.is_sparse and sparse._nnz() == 0
    thin = torch.empty(5, 0, device=dev, requires_grad=True)
    out = gs.ops.embedding(thin, ids)
    assert out.shape == (4, 0)
    assert torch.autograd.grad(out.sum(), thin)[0].shape == (5, 0)
    sparse, = torch.autograd.grad(gs.ops.embedding(thin, ids, sparse_grad=True).sum(), thin)
    assert sparse.indices().tolist() == [[0]] and sparse.values().shape == (1, 0)


# ------------------------------------------------------------------ no GPU ----
def test_bad_arguments_are_refused_before_anything_is_launched():
    import ctypes
    lib, i64 = capi.lib(), ctypes.c_int64
    buf = (ctypes.c_int64 * 64)()
    at = ctypes.addressof(buf)

    def lookup(table=buf, rows=4, stride=8, dim=8, kind=0, ids=buf, id_bytes=8, n=2, out=buf):
        return lib.gs_embedding_lookup(table, i64(rows), i64(stride), i64(dim), kind, ids, id_bytes, i64(n),
                                       ctypes.c_float(1), out, None)

    assert lookup(n=0) == 0 and lookup(dim=0) == 0
    for bad, match in ((dict(kind=3), b"value type"), (dict(id_bytes=2), b"id_bytes"), (dict(n=-1), b"ids"),
                       (dict(n=1 << 31), b"ids"), (dict(rows=(1 << 32) - 1), b"rows"), (dict(dim=1 << 24), b"values"),
                       (dict(stride=-1), b"stride"), (dict(ids=None), b"null"), (dict(out=None), b"null"),
                       (dict(table=None), b"null"), (dict(table=ctypes.c_void_p(at + 2)), b"aligned"),
                       (dict(ids=ctypes.c_void_p(at + 4)), b"aligned"), (dict(kind=1, out=ctypes.c_void_p(at + 1)), b"aligned")):
        status = lookup(**bad)
        assert status < 0 and match in lib.gs_status_string(status), (bad, lib.gs_status_string(status))
    assert lib.gs_embedding_grad_workspace_bytes(i64(1000), i64(64), 0) > 8000  # a word an id
    status = lib.gs_embedding_grad(buf, i64(8), i64(8), 0, buf, 8, i64(2), i64(4), ctypes.c_float(1), buf, buf,
                                   ctypes.c_size_t(16), None)
    assert status == -2 and b"workspace" in lib.gs_status_string(status)
    status = lib.gs_embedding_sparse_grad_count(buf, 8, i64(0), i64(4), i64(8), 0, None, i64(1), buf, ctypes.c_size_t(16),
                                                None)
    assert status == -1 and b"no ids" in lib.gs_status_string(status)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU tensor"):
        gs.ops.embedding(torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))


def test_workspaces_of_sizes_that_no_call_takes():
    """They have no plan: a size comes back all the same, and the call with it refuses."""
    import ctypes
    lib, i64 = capi.lib(), ctypes.c_int64
    buf = (ctypes.c_int64 * 64)()
    sizes = (lib.gs_embedding_grad_workspace_bytes, lib.gs_embedding_sparse_grad_workspace_bytes)
    for dim in (1, 64, 2048, (1 << 24) - 1):
        for kind in (0, 1, 2):
            for size in sizes:
                # the most ids that are taken: a word each at least, and then the launches that join the sums
                assert size(i64((1 << 31) - 1), i64(dim), kind) > 8 << 31
                for n in (1 << 31, 1 << 37, 1 << 45, 1 << 62, (1 << 63) - 1, -1, 0):
                    assert size(i64(n), i64(dim), kind) == 256
    for size in sizes:
        assert size(i64(1000), i64(1 << 24), 0) == size(i64(1000), i64(1 << 62), 0) == size(i64(1000), i64(64), 9) == 256
    for n, dim, kind, match in ((1 << 37, 64, 0, b"ids"), (2, 1 << 24, 0, b"values"), (2, 8, 9, b"value type")):
        status = lib.gs_embedding_grad(buf, i64(8), i64(dim), kind, buf, 8, i64(n), i64(4), ctypes.c_float(1), buf, buf,
                                       ctypes.c_size_t(256), None)
        assert status < 0 and match in lib.gs_status_string(status)
        status = lib.gs_embedding_sparse_grad_count(buf, 8, i64(n), i64(4), i64(dim), kind, None, i64(1), buf,
                                                    ctypes.c_size_t(256), None)
        assert status < 0 and match in lib.gs_status_string(status)


@gpu
def test_more_ids_than_are_taken_are_refused_before_anything_is_allocated(dev):
    ids = torch.zeros(1, dtype=torch.int32, device=dev).expand(1 << 31)
    row, wide = torch.zeros(1, 1, device=dev), torch.zeros(1, 1, device=dev).expand(1, 1 << 24)
    held = torch.cuda.memory_allocated(dev)
    for call in (lambda: gs.ops.embedding(row, ids), lambda: gs.ops.expert_sort(ids, 4),
                 lambda: gs.ops.expert_dispatch(row.expand(1 << 31, 1), ids, 4),
                 lambda: torch.ops.gs_ops._CAPI_EmbeddingGrad(row.expand(1 << 31, 1), ids, 4, 1.0),
                 lambda: torch.ops.gs_ops._CAPI_EmbeddingSparseGrad(row.expand(1 << 31, 1), ids, 4, 1.0)):
        with pytest.raises(RuntimeError, match=r"(ids|experts): at most 2\^31 - 1 are taken"):
            call()
    with pytest.raises(RuntimeError, match=r"at most 2\^24 - 1 values are taken"):
        gs.ops.embedding(wide, ids[:4])
    assert torch.cuda.memory_allocated(dev) == held


class CountingLibrary:
    """Stands in for the kernel library: notes the scratch that every call is given, and what a fill finds in it."""
    def __init__(self):
        self.scratch, self.held = [], None

    def __getattr__(self, name):
        import ctypes
        if name.endswith("_workspace_bytes"):
            return lambda *args: 4096

        def call(*args):
            at = [i for i, a in enumerate(args) if isinstance(a, ctypes.c_size_t)][0] - 1
            self.scratch.append(args[at].value)
            if name == "gs_embedding_sparse_grad_count":
                ctypes.memset(args[at], 7, 4096)
                ctypes.cast(args[6], ctypes.POINTER(ctypes.c_int64))[0] = 2
            elif name == "gs_embedding_sparse_grad_fill":
                self.held = ctypes.string_at(args[at], 4096)
            return 0
        return call


def test_scratch_of_the_binding_is_the_calls_own(monkeypatch):
    """What one call has in its scratch is not written over by another of the binding's calls, by any thread."""
    import ctypes
    import types
    library, cpu, zeros = CountingLibrary(), torch.device("cpu"), torch.zeros
    monkeypatch.setattr(capi, "lib", lambda: library)
    monkeypatch.setattr(capi, "_ws", capi._Workspace())  # (a buffer in host memory is not left for calls on a GPU)
    monkeypatch.setattr(capi, "_ids", lambda t, name: 8)
    monkeypatch.setattr(capi, "_stream", lambda device: None)
    monkeypatch.setattr(capi, "_rows", lambda t, name: (ctypes.c_void_p(t.data_ptr()), capi._i64(t.stride(0)),
                                                        capi._i64(t.size(1)), 0))
    monkeypatch.setattr(torch, "zeros", lambda *args, pin_memory=False, **kw: zeros(*args, **kw))
    grad, ids = torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64)

    def another_call():  # while the first one waits for its stream
        capi.workspace(4096, cpu).fill_(255)
        capi.embedding_grad(grad, ids, 5)
        capi.expert_sort(ids, 4)
        capi.expert_dispatch(grad, ids, 4)

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: types.SimpleNamespace(synchronize=another_call))
    capi.embedding_sparse_grad(grad, ids, 5)
    assert library.held == bytes([7]) * 4096
    count, *others, fill = library.scratch
    assert count == fill and len(others) == 3
    assert capi.workspace(4096, cpu).data_ptr() not in library.scratch


@gpu
def test_two_threads_through_the_binding(dev):
    """Both gradients, sorts and rows sent by two threads on a stream each, through the C ABI's binding."""
    import threading
    work = []
    for seed in (51, 52):
        grad, ids = rows(30000, 24, torch.float32, dev, seed), torch.from_numpy(ids_of("hub", 30000, 900, seed)).to(dev)
        work.append((grad, ids, capi.embedding_grad(grad, ids, 900), capi.expert_dispatch(grad, ids, 900)))
    torch.cuda.synchronize()
    wrong = []

    def run(grad, ids, want, want_sent):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                met, values = capi.embedding_sparse_grad(grad, ids, 900)
                dense = capi.embedding_grad(grad, ids, 900)
                sent = capi.expert_dispatch(grad, ids, 900)
                same = all(torch.equal(a, b) for a, b in zip(sent, want_sent))
                same = same and all(torch.equal(a, b) for a, b in zip(capi.expert_sort(ids, 900), want_sent[1:]))
                if not (same and torch.equal(dense, want) and torch.equal(dense[met], values)):
                    wrong.append(1)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
