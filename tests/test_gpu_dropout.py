"""gs.ops.dropout against the formula, its mask from the oracle's draws.

Tolerances.  The factor 1 / (1 - p) is rounded to fp32, the product and the sum each once (2^-24 of what they are), the
result once more (eps / 2): 3 * 2^-24 of |x| / (1 - p) + |residual|, and half a step of the result.  What is dropped, and
the sums' masks, are exact."""
import numpy as np
import pytest
import torch

import graph_sampling_amd as gs
from graph_sampling_amd import capi
from oracle import oracle as O

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def words(seed, blocks):
    """The four words of each of the blocks under `seed`, by the oracle."""
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    return np.concatenate([np.zeros(0, np.uint32)] + [np.asarray(O.philox4x32_10([b & 0xFFFFFFFF, 0, 0, 6 | ((b >> 32) << 8)], key)) for b in blocks])


def kept_of(seed, n, p):
    return words(seed, range((n + 3) // 4))[:n].astype(np.uint64) >= np.uint64(int(p * 2 ** 32))


def values(shape, dtype, dev, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def check(got, x, r, kept, p, dtype):
    hx, hr = x.detach().double().cpu().numpy(), 0.0 if r is None else r.detach().double().cpu().numpy()
    scaled = np.where(kept, hx / (1 - p) if p < 1 else 0.0, 0.0)
    want = scaled + hr
    tol = 3 * F32 * (np.abs(scaled) + np.abs(hr))
    assert got.dtype == dtype and got.shape == x.shape
    off = np.abs(got.detach().double().cpu().numpy() - want)
    assert np.all(off <= tol + (np.abs(want) + tol) * half_step(dtype) + smallest(dtype))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(), (1,), (3,), (4,), (7, 1), (5, 7), (37, 97), (8, 8), (33, 64), (2, 3, 5, 7), (1025,), (0, 4), (4099,)])
def test_masks_sums_and_gradients(dev, shape, dtype):
    n = int(np.prod(shape))
    for p, seed in ((0.0, 1), (0.1, 7777), (0.5, -3), (0.999, 2 ** 63 - 1), (1.0, 5), (2.0 ** -40, 2 ** 64 - 1), (1 - 2.0 ** -33, 2 ** 33)):
        kept = kept_of(seed, n, p).reshape(shape) if p < 1 else np.zeros(shape, bool)
        x, r = values(shape, dtype, dev, 1).requires_grad_(True), values(shape, dtype, dev, 2).requires_grad_(True)
        grad = values(shape, dtype, dev, 3)
        if 1 - p < 2.0 ** -20 and p < 1 and dtype == torch.float16:
            continue  # (what is kept has no value in fp16)
        out = gs.ops.dropout(x, p, seed)
        check(out, x, None, kept, p, dtype)
        assert not out.detach()[torch.from_numpy(np.asarray(~kept)).to(dev)].any()
        dx, = torch.autograd.grad(out, x, grad)
        check(dx, grad, None, kept, p, dtype)
        out = gs.ops.dropout(x, p, seed, residual=r)
        check(out, x, r, kept, p, dtype)
        both = torch.autograd.grad(out, (x, r), grad)
        assert torch.equal(both[0], dx) and torch.equal(both[1], grad)
        only, = torch.autograd.grad(gs.ops.dropout(x.detach(), p, seed, r), r, grad)
        assert torch.equal(only, grad)
        # the seed in memory, and through the C ABI by itself
        at = torch.tensor([(seed + 2 ** 63) % 2 ** 64 - 2 ** 63], device=dev)
        assert torch.equal(gs.ops.dropout(x, p, at, r), out)
        if n:
            assert torch.equal(capi.dropout(x.detach(), p, seed, r.detach()), out) and torch.equal(capi.dropout(x.detach(), p, at, r.detach()), out)


@gpu
def test_the_type_and_the_cut_do_not_change_the_mask(dev):
    """Positions alone decide: a prefix, another type, another shape and every alignment of the same values draw the same."""
    n = 10_007
    kept = torch.from_numpy(kept_of(9, n, 0.3)).to(dev)
    for dtype in TYPES:
        for shift in range(0, 9):
            x = torch.ones(n + 16, dtype=dtype, device=dev)[shift:shift + n]
            assert torch.equal(gs.ops.dropout(x, 0.3, 9) != 0, kept)
            assert torch.equal(gs.ops.dropout(x[:1003], 0.3, 9) != 0, kept[:1003])
    assert torch.equal(gs.ops.dropout(torch.ones(n // 7, 7, device=dev).t().contiguous().t()[:100], 0.3, 9) != 0, kept[:700].view(100, 7))


@gpu
def test_strides_are_those_of_the_positions(dev):
    for dtype in TYPES:
        base = values((90, 50), dtype, dev, 4)
        for view in (base[:, 3:20], base[::3], base.t(), base[:1].expand(40, 50), base[:, :1].expand(90, 30), base.view(9, 10, 50).transpose(0, 2)):
            x = view.detach().requires_grad_(True)
            r = values(tuple(reversed(view.shape)), dtype, dev, 5).permute(*reversed(range(view.dim())))
            out = gs.ops.dropout(x, 0.4, 11, r)
            assert torch.equal(out, gs.ops.dropout(view.contiguous(), 0.4, 11, r.contiguous()))
            grad = values(tuple(reversed(view.shape)), dtype, dev, 6).permute(*reversed(range(view.dim())))
            dx, = torch.autograd.grad(out, x, grad)
            assert torch.equal(dx, gs.ops.dropout(grad.contiguous(), 0.4, 11))


@gpu
def test_what_is_dropped_leaves_no_trace(dev):
    kept = torch.from_numpy(kept_of(3, 5000, 0.5)).to(dev)
    for dtype in TYPES:
        x = values((5000,), dtype, dev, 7)
        want = gs.ops.dropout(x, 0.5, 3)
        dirty = torch.where(kept, x, torch.tensor([float("nan"), float("inf")], device=dev, dtype=dtype).repeat(2500))
        assert torch.equal(gs.ops.dropout(dirty, 0.5, 3), want)
        assert not gs.ops.dropout(torch.full((999,), float("nan"), dtype=dtype, device=dev), 1.0, 3).any()
        assert gs.ops.dropout(torch.full((999,), float("nan"), dtype=dtype, device=dev), 0.0, 3).isnan().all()


@gpu
def test_shares_and_independence(dev):
    """Of 2^22 draws, p is dropped within six standard deviations; masks of neighbouring seeds and positions agree as
    often as independent ones do, within the same."""
    n = 1 << 22
    ones = torch.ones(n, device=dev)
    for p in (0.1, 0.5):
        a, b = gs.ops.dropout(ones, p, 100) != 0, gs.ops.dropout(ones, p, 101) != 0
        dev6 = 6 * (p * (1 - p) / n) ** 0.5
        assert abs(float(a.double().mean()) - (1 - p)) < dev6
        same = p * p + (1 - p) * (1 - p)
        dev6 = 6 * (same * (1 - same) / n) ** 0.5
        assert abs(float((a == b).double().mean()) - same) < dev6 and abs(float((a[1:] == a[:-1]).double().mean()) - same) < dev6


@gpu
def test_seeds_that_are_counted(dev):
    """Without a seed a call takes the next of the samplers'; its backward pass draws the same mask again."""
    x = torch.ones(3000, device=dev).requires_grad_(True)
    torch.ops.gs_ops._CAPI_SetSeed(500)
    first, second = gs.ops.dropout(x, 0.5), gs.ops.dropout(x, 0.5)
    assert torch.equal(first, gs.ops.dropout(x, 0.5, 500)) and torch.equal(second, gs.ops.dropout(x, 0.5, 501))
    assert not torch.equal(first, second)
    for out in (second, first):
        assert torch.equal(torch.autograd.grad(out, x, torch.ones_like(x))[0], out.detach())
    torch.ops.gs_ops._CAPI_SetSeed(500)
    assert torch.equal(gs.ops.dropout(x, 0.5), first)


@gpu
def test_recorded_and_replayed_with_a_seed_that_changes(dev):
    x, r = values((700, 33), torch.bfloat16, dev, 8).requires_grad_(True), values((700, 33), torch.bfloat16, dev, 9)
    seed = torch.tensor([1], device=dev)
    grad = values((700, 33), torch.bfloat16, dev, 10)

    def step():
        out = gs.ops.dropout(x, 0.25, seed, r)
        return out.detach(), torch.autograd.grad(out, x, grad)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, message = torch.cuda.CUDAGraph(), ""
    with torch.cuda.graph(graph):
        got = step()
        try:
            gs.ops.dropout(x.detach(), 0.25)
        except RuntimeError as error:
            message = str(error)
    assert "needs a seed" in message
    masks = []
    for rep in range(4):
        seed.fill_(2 ** 40 + rep)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(got[0], gs.ops.dropout(x, 0.25, 2 ** 40 + rep, r))
        masks.append(got[1] != 0)
    assert not torch.equal(masks[0], masks[1])
    # a seed that changed between the passes is noticed
    out = gs.ops.dropout(x, 0.25, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, x, grad)


@gpu
def test_recording_is_refused_where_it_would_end_the_process(dev):
    x = values((4, 8), torch.float32, dev, 1).requires_grad_(True)
    eager = gs.ops.dropout(x, 0.5, 1)
    torch.cuda.synchronize()
    graph, messages = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        kept = x.detach() * 2
        for call in (lambda: gs.ops.dropout(x, 0.5, 1), lambda: gs.ops.dropout(x.detach(), 0.5, 1, x)):
            try:
                call()
            except RuntimeError as error:
                messages.append(str(error))
    assert len(messages) == 2 and all("eager graph of the same leaf" in m for m in messages)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, x.detach() * 2)
    torch.autograd.grad(eager.sum(), x)


@gpu
def test_positions_beyond_32_bits(dev):
    """Positions past 2^32, and blocks past 2^32 of those (2^34 positions): the oracle's draws at both ends."""
    if torch.cuda.mem_get_info(dev)[0] < 120 << 30:
        pytest.skip("needs about 70 GB of free device memory")
    n = 2 ** 34 + 1027
    x = torch.ones(n, dtype=torch.bfloat16, device=dev)
    out = gs.ops.dropout(x, 0.5, 21)
    for first in (0, 2 ** 32 - 512, 2 ** 34 - 512, 2 ** 34):
        kept = words(21, range(first // 4, first // 4 + 256)).astype(np.uint64) >= np.uint64(2 ** 31)
        assert np.array_equal((out[first:first + 1024] != 0).cpu().numpy(), kept)
    assert (out[-3:] != 0).tolist() == (words(21, [2 ** 32 + 256])[:3] >= 2 ** 31).tolist()


@gpu
def test_more_values_than_one_launch_has_workgroups_for(dev):
    if torch.cuda.mem_get_info(dev)[0] < 200 << 30:
        pytest.skip("needs about 140 GB of free device memory")
    n = 2 ** 34 + 1027
    out = gs.ops.dropout(torch.ones(n, device=dev), 0.5, 22)
    for first in (0, 2 ** 34 - 2048, 2 ** 34 - 1024, 2 ** 34):
        kept = words(22, range(first // 4, first // 4 + 256)).astype(np.uint64) >= np.uint64(2 ** 31)
        assert np.array_equal(out[first:first + 1024].cpu().numpy(), np.where(kept, 2.0, 0.0))
    assert np.array_equal(out[-3:].cpu().numpy(), np.where(words(22, [2 ** 32 + 256])[:3] >= 2 ** 31, 2.0, 0.0))


@gpu
def test_refusals(dev):
    x = values((6, 5), torch.float32, dev, 1)
    for args, match in (((x.double(), 0.5, 1), "float32, float16 or bfloat16"), ((x, 1.5, 1), "probability"), ((x, -0.1, 1), "probability"),
                        ((x, float("nan"), 1), "probability"), ((x.cpu(), 0.5, 1), "GPU tensor"),
                        ((x, 0.5, torch.tensor([1])), "GPU tensor"), ((x, 0.5, torch.tensor([1, 2], device=dev)), "one int64"),
                        ((x, 0.5, torch.tensor([1], dtype=torch.int32, device=dev)), "int64"), ((x, 0.5, 1, x.half()), "residual"),
                        ((x, 0.5, 1, x[:5]), "residual"), ((x, 0.5, 1, x.cpu()), "residual")):
        with pytest.raises(RuntimeError, match=match):
            gs.ops.dropout(*args)
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="once more"):
        torch.autograd.grad((gs.ops.dropout(x, 0.5, 1) * x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gs.ops.dropout(t, 0.5, 1).sum())(x.detach())


# ------------------------------------------------------------------ no GPU ----
def test_bad_arguments_are_refused_before_anything_is_launched():
    import ctypes
    lib, i64 = capi.lib(), ctypes.c_int64
    buf = (ctypes.c_int64 * 64)()
    at = ctypes.addressof(buf)

    def fails(status, match):
        assert status < 0 and match in lib.gs_status_string(status), (status, lib.gs_status_string(status))

    def dropout(x=buf, r=None, n=8, kind=0, p=0.5, seed_at=None, out=buf):
        return lib.gs_dropout(x, r, i64(n), kind, ctypes.c_double(p), ctypes.c_uint64(1), seed_at, out, None)

    assert dropout(n=0) == 0
    for change, match in ((dict(kind=7), b"value type"), (dict(n=-1), b"negative"), (dict(p=1.5), b"probability"),
                          (dict(p=float("nan")), b"probability"), (dict(x=None), b"null"), (dict(out=None), b"null"),
                          (dict(x=ctypes.c_void_p(at + 2)), b"aligned"), (dict(r=ctypes.c_void_p(at + 1)), b"aligned"),
                          (dict(seed_at=ctypes.c_void_p(at + 4)), b"aligned")):
        fails(dropout(**change), match)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU tensor"):
        gs.ops.dropout(torch.zeros(3, 4), 0.5, 1)
