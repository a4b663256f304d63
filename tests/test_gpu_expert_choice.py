"""gs.ops.expert_choose and its gradient against the formulas in 64 bits.

Tolerances.  A share is exp(l - top) over a sum of E of those: the difference is rounded (2^-24 of itself, which moves the
exponential by |l - top| * 2^-24), the exponential is off by at most 2 steps (2^-23 each), the sum by E additions of 2^-24, the
quotient by 2^-24: relative (|l - top| + E + 12) * 2^-23 in all, and no less than the smallest normal value times 2 per
term.  A gradient adds two products of those with K additions: (K + 8) * 2^-24 more, of the magnitudes' sum."""
import numpy as np
import pytest
import torch

import graph_sampling_amd as gs
from graph_sampling_amd import capi

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
STEP = 2.0 ** -23
TINY = 2.0 ** -125


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def logits_of(kind, tokens, experts, dtype, dev, seed):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(tokens, experts, generator=g)
    if kind == "ties":
        l = torch.randint(-2, 3, (tokens, experts), generator=g).float() * torch.where(torch.rand(tokens, experts, generator=g) < 0.5, 1, -1)
    elif kind == "masked":
        l[torch.rand(tokens, experts, generator=g) < 0.7] = -float("inf")
        l[::5] = -float("inf")
    elif kind == "far":
        l = l * 60
    elif kind == "lowest":
        l[torch.rand(tokens, experts, generator=g) < 0.8] = torch.finfo(dtype).min
        l[::4] = torch.finfo(dtype).min
    return l.to(dtype).to(dev)


def formula(logits, K, normalize, grad):
    l = logits.detach().double().cpu().numpy()
    T, E = l.shape
    order = np.argsort(-l, axis=1, kind="stable")[:, :K]  # (-0.0 and 0.0 are equal)
    value = np.take_along_axis(l, order, 1)
    there = value > -np.inf
    experts = np.where(there, order, -1)
    top = np.where(l.max(1, keepdims=True) > -np.inf, l.max(1, keepdims=True), 0.0) if E else np.zeros((T, 1))
    e_all, e_top = np.exp(l - top), np.exp(value - top)
    z = (e_top if normalize else e_all).sum(1, keepdims=True)
    z = np.where(z > 0, z, 1.0)
    w = e_top / z
    p = e_all / z
    g = grad.double().cpu().numpy()
    dot, size = (w * g).sum(1, keepdims=True), (w * np.abs(g)).sum(1, keepdims=True)
    if normalize:
        among = np.zeros((T, E), dtype=bool)
        np.put_along_axis(among, order, there, 1)
        p = np.where(among, p, 0.0)
    d, d_size = -p * dot, p * size
    add, add_size = np.zeros_like(d), np.zeros_like(d)
    np.put_along_axis(add, order, np.where(there, w * g, 0.0), 1)
    np.put_along_axis(add_size, order, np.where(there, w * np.abs(g), 0.0), 1)
    with np.errstate(invalid="ignore"):
        apart = np.where(l > -np.inf, top - l, 0.0)
    return experts, w, d + add, d_size + add_size, np.minimum(apart, 200.0), np.minimum(np.where(there, top - value, 0.0), 200.0)


CASES = [
    # tokens, experts, choices, kind
    (1, 1, 1, "normal"), (4, 64, 4, "normal"), (3, 2, 2, "ties"), (33, 5, 1, "masked"), (100, 16, 16, "ties"), (17, 17, 3, "normal"),
    (50, 64, 8, "ties"), (50, 65, 8, "far"), (200, 160, 6, "masked"), (513, 256, 8, "ties"), (31, 257, 8, "normal"),
    (9, 100, 17, "ties"), (9, 64, 64, "masked"), (40, 512, 10, "far"), (12, 1000, 64, "ties"), (7, 1024, 5, "lowest"),
    (5, 1025, 7, "masked"), (6, 4096, 64, "ties"), (3, 4095, 1, "far"), (1000, 8, 2, "lowest"), (0, 8, 2, "normal"), (6, 5, 0, "normal"),
    (70001, 3, 2, "masked"),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,num,choices,kind", CASES)
def test_choices_and_gradients(dev, tokens, num, choices, kind, dtype):
    logits = logits_of(kind, tokens, num, dtype, dev, tokens + num).requires_grad_(True)
    grad = torch.randn(tokens, choices, generator=torch.Generator().manual_seed(1)).to(dev)
    for normalize in (True, False):
        experts, weights = gs.ops.expert_choose(logits, choices, normalize)
        w_experts, w_weights, w_d, size, apart, apart_top = formula(logits, choices, normalize, grad)
        assert experts.dtype == torch.int32 and weights.dtype == torch.float32 and experts.shape == weights.shape == (tokens, choices)
        assert np.array_equal(experts.cpu().numpy(), w_experts)
        off = np.abs(weights.detach().double().cpu().numpy() - w_weights)
        assert np.all(off <= (apart_top + num + 12) * STEP * w_weights + TINY)
        assert not weights.detach()[experts < 0].any()
        d, = torch.autograd.grad(weights, logits, grad) if choices else (torch.zeros_like(logits),)
        assert d.dtype == dtype
        tol = (apart + 2 * num + choices + 40) * 2 * STEP * size + TINY * 8
        off = np.abs(d.double().cpu().numpy() - w_d)
        assert np.all(off <= tol + (np.abs(w_d) + tol) * half_step(dtype) + smallest(dtype))
        # through the C ABI by itself
        c_experts, c_weights = capi.expert_choose(logits.detach(), choices, normalize)
        assert torch.equal(c_experts, experts) and torch.equal(c_weights, weights)
        if choices:
            assert torch.equal(capi.expert_choose_grad(grad, logits.detach(), experts, weights.detach(), normalize), d)
            assert torch.equal(torch.ops.gs_ops._CAPI_ExpertChooseGrad(grad, logits.detach(), experts, weights.detach(), normalize), d)


@gpu
def test_every_number_of_experts(dev):
    """Choices of whole numbers, many of them equal, on both sides of every size at which the kernels change."""
    for num in (1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 192, 255, 256, 257, 511, 512, 513, 1023, 1025, 2048, 4096):
        for choices in {1, min(2, num), min(8, num), min(16, num), min(17, num), min(64, num)}:
            for dtype in TYPES:
                logits = torch.randint(-3, 4, (37, num), generator=torch.Generator().manual_seed(num)).to(dtype)
                logits[torch.rand(37, num, generator=torch.Generator().manual_seed(1)) < 0.3] = -float("inf")
                experts, weights = gs.ops.expert_choose(logits.to(dev), choices)
                order = np.argsort(-logits.double().numpy(), axis=1, kind="stable")[:, :choices]
                want = np.where(np.take_along_axis(logits.double().numpy(), order, 1) > -np.inf, order, -1)
                assert np.array_equal(experts.cpu().numpy(), want), (num, choices, dtype)
                total = weights.double().sum(1).cpu().numpy()
                assert np.all(np.abs(total - (want[:, 0] >= 0)) <= (num + 80) * STEP)


@gpu
def test_nan_and_infinities(dev):
    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([[1.0, nan, 3.0, nan], [-inf, -inf, -inf, -inf], [inf, 0.0, -inf, 1.0], [0.0, -0.0, 0.0, -0.0],
                           [-inf, 5.0, -inf, -inf]], device=dev)
    for dtype in TYPES:
        l = logits.to(dtype).requires_grad_(True)
        for normalize in (True, False):
            experts, weights = gs.ops.expert_choose(l, 2, normalize)
            assert experts.tolist() == [[1, 3], [-1, -1], [0, 3], [0, 1], [1, -1]]
            assert weights[0].isnan().all() and not weights[1].any() and weights[2].isnan().any()
            assert weights[3].tolist() == ([0.5, 0.5] if normalize else [0.25, 0.25]) and weights[4].tolist() == [1.0, 0.0]
            d, = torch.autograd.grad(weights, l, torch.tensor([[0, 0], [nan, inf], [0, 0], [1.0, 0.0], [2.0, nan]], device=dev))
            assert not d[1].any() and d[3].tolist() == ([0.25, -0.25, 0, 0] if normalize else [0.1875, -0.0625, -0.0625, -0.0625])
            assert not d[4].any()


@gpu
def test_rows_any_distance_apart(dev):
    for dtype in TYPES:
        base = logits_of("normal", 60, 90, dtype, dev, 1)
        for view in (base[:, 1:70], base[::3, 3:35], base[5:20, 7:8], base.t()[:50], base[:1, :40].expand(30, 40)):
            x = view.detach().requires_grad_(True)
            y = view.contiguous().requires_grad_(True)
            k = min(4, view.shape[1])
            grad = torch.randn(k, view.shape[0], device=dev).t()
            for normalize in (True, False):
                a, b = gs.ops.expert_choose(x, k, normalize), gs.ops.expert_choose(y, k, normalize)
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
                assert torch.equal(torch.autograd.grad(a[1], x, grad)[0], torch.autograd.grad(b[1], y, grad.contiguous())[0])


@gpu
def test_gradient_against_differences(dev):
    l = logits_of("normal", 5, 7, torch.float32, dev, 3).requires_grad_(True)
    grad, v = torch.randn(5, 3, device=dev), torch.randn(5, 7, device=dev)
    for normalize in (True, False):
        experts, weights = gs.ops.expert_choose(l, 3, normalize)
        d, = torch.autograd.grad(weights, l, grad)
        h = 2.0 ** -7

        def along(s):
            moved = gs.ops.expert_choose(l.detach() + s * v, 7, False)  # (all of them, in whatever order)
            share = torch.zeros(5, 7, device=dev, dtype=torch.float64).scatter_(1, moved[0].long(), moved[1].double())
            chosen = torch.take_along_dim(share, experts.long(), 1)
            return ((chosen / chosen.sum(1, keepdim=True) if normalize else chosen) * grad.double()).sum().item()

        # the third derivative of a sum of shares is below 6 |v|^3 a token's term: h^2 / 6 of that, and 2^-23 * 40 / h of rounding
        slope = (d.double() * v.double()).sum().item()
        bound = 5 * 3 * float(grad.abs().max()) * float(v.abs().max()) ** 3 * 8 * h * h + 40 * 2.0 ** -23 / h * 15 * float(grad.abs().max())
        assert abs((along(h) - along(-h)) / (2 * h) - slope) < bound


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_the_sum_of_all_shares_leans_to_no_side(dev, dtype):
    """Of 2^15 tokens, 4095 experts 7.5 to 9 below the first: half of a sum is exponentials of such differences.  An
    exponential that is right to a step, above as often as below, leaves a mean error far below one: 70 roundings of 2^-24, evenly
    spread, are 2.9e-7 a token, six standard deviations of 2^15 tokens' mean 9.6e-9.  An eighth of a step, 2^-26, is allowed; the
    product with log2(e) rounded to fp32, 1.3e-8 of the difference too small, would lean by four times that.

    fp16 has 256 values in that range, so that tokens share their roundings: in the lane that has the first expert's 1, sums are
    multiples of 2^-23, and what an addition loses follows from the term alone.  256 losses spread over 2^-24 either way have a
    mean of 2^-24 / sqrt(3) / 16 = 2.2e-9, 31.5 of them follow the 1, of a sum of 2.17: 3.1e-8, six times that is allowed as well."""
    g = torch.Generator(device=dev).manual_seed(5)
    logits = -7.5 - 1.5 * torch.rand(1 << 15, 4096, generator=g, device=dev)
    first = torch.randint(4096, (1 << 15, 1), generator=g, device=dev)
    logits = logits.scatter_(1, first, 0.0).to(dtype)
    experts, weights = gs.ops.expert_choose(logits, 1, False)
    assert torch.equal(experts.long(), first)
    want = 1.0 / torch.exp(logits.double()).sum(1, keepdim=True)
    assert abs(float((weights.double() / want - 1.0).mean())) < 2.0 ** -26 + (6 * 3.1e-8 if dtype == torch.float16 else 0.0)


@gpu
def test_normalized_shares_keep_no_logits(dev):
    """Their gradient looks at none: the logits may change, and their memory goes back, before the backward pass."""
    for dtype in TYPES:
        x = logits_of("normal", 4096, 1000, dtype, dev, 2).requires_grad_(True)
        grad = torch.randn(4096, 5, device=dev)
        want, = torch.autograd.grad(gs.ops.expert_choose(x * 1.0, 5)[1], x, grad)
        logits = x * 1.0
        weights = gs.ops.expert_choose(logits, 5)[1]
        with torch.no_grad():
            logits.fill_(float("nan"))
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated(dev)
        del logits
        assert before - torch.cuda.memory_allocated(dev) >= 4096 * 1000 * torch.finfo(dtype).bits // 8
        got, = torch.autograd.grad(weights, x, grad)
        assert torch.equal(got, want)
        # over all experts, they are kept, and a change is noticed
        logits = x * 1.0
        weights = gs.ops.expert_choose(logits, 5, False)[1]
        with torch.no_grad():
            logits.fill_(0.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(weights, x, grad)


@gpu
def test_recorded_and_replayed(dev):
    for tokens, num, k in ((4, 64, 4), (900, 160, 6), (30, 600, 20)):
        l = logits_of("normal", tokens, num, torch.bfloat16, dev, 1).requires_grad_(True)
        grad = torch.randn(tokens, k, device=dev)

        def step():
            experts, weights = gs.ops.expert_choose(l, k, False)
            return experts, weights.detach(), torch.autograd.grad(weights, l, grad)[0]

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
            with torch.no_grad():
                l.copy_(logits_of("masked" if rep % 2 else "ties", tokens, num, torch.bfloat16, dev, 10 + rep))
            want = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@gpu
def test_normalized_shares_recorded_and_replayed(dev):
    """Their backward pass, which has no logits, in a graph: other logits at each replay."""
    l = logits_of("normal", 700, 96, torch.float16, dev, 1).requires_grad_(True)
    grad = torch.randn(700, 4, device=dev)

    def step():
        experts, weights = gs.ops.expert_choose(l * 1.0, 4)
        return experts, weights.detach(), torch.autograd.grad(weights, l, grad)[0]

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
        with torch.no_grad():
            l.copy_(logits_of("masked" if rep % 2 else "ties", 700, 96, torch.float16, dev, 20 + rep))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@gpu
def test_offsets_beyond_32_bits(dev):
    if torch.cuda.mem_get_info(dev)[0] < 60 << 30:
        pytest.skip("needs about 20 GB of free device memory")
    tokens, num = 1_100_000, 4096
    l = torch.full((tokens, num), -3.0, dtype=torch.bfloat16, device=dev)
    last = torch.randint(num, (tokens,), device=dev)
    l[torch.arange(tokens, device=dev), last] = 1.0
    experts, weights = gs.ops.expert_choose(l, 1)
    assert torch.equal(experts[:, 0].long(), last) and bool((weights == 1).all())
    d = capi.expert_choose_grad(torch.ones_like(weights), l, experts, weights, False)
    assert torch.equal(d[-1000:].argmax(1), last[-1000:]) and not d[-1000:].isnan().any()


@gpu
def test_as_many_choices_as_there_may_be(dev):
    """2^31 - 1 tokens, of one choice each: more than one launch has workgroups for."""
    if torch.cuda.mem_get_info(dev)[0] < 120 << 30:
        pytest.skip("needs about 60 GB of free device memory")
    n = 2 ** 31 - 1
    l = torch.zeros(n, 2, dtype=torch.bfloat16, device=dev)
    mine = torch.tensor([0, 7, 2 ** 30 - 65, 2 ** 30 - 64, 2 ** 30, 2 ** 30 + 1, n - 2, n - 1], device=dev)
    l[mine, 1] = 1.0
    for normalize in (True, False):
        experts, weights = gs.ops.expert_choose(l, 1, normalize)
        assert experts.shape == (n, 1) and int(experts.sum()) == 8 and bool((experts[mine] == 1).all())
        # (half a step of a sum of two, and the quotient's)
        assert abs(float(weights.min()) - (1.0 if normalize else 0.5)) < 2.0 ** -22
        assert abs(float(weights.max()) - (1.0 if normalize else 1 / (1 + np.exp(-1)))) < 2.0 ** -22
        d = capi.expert_choose_grad(weights, l, experts, weights, normalize)
        if normalize:  # (a share of one is always 1)
            assert not d.any()
        else:
            share = 1 / (1 + np.exp(-1))
            for row, want in ((1, 0.125), (2 ** 30 - 66, 0.125), (2 ** 30 + 2, 0.125), (n - 3, 0.125)):
                assert d[row].tolist() == [want, -want]
            want = share * share * (1 - share)
            off = (d[mine].double() - torch.tensor([-want, want], device=dev, dtype=torch.float64)).abs().max()
            assert float(off) <= want * (half_step(torch.bfloat16) + 2.0 ** -20)
        del experts, weights, d
    with pytest.raises(RuntimeError, match="2\\^31"):
        gs.ops.expert_choose(l[:2 ** 30], 2)


@gpu
def test_recording_is_refused_where_it_would_end_the_process(dev):
    l = logits_of("normal", 4, 8, torch.float32, dev, 1).requires_grad_(True)
    eager = gs.ops.expert_choose(l, 2)[1]
    torch.cuda.synchronize()
    graph, messages = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        kept = l.detach() * 2
        try:
            gs.ops.expert_choose(l, 2)
        except RuntimeError as error:
            messages.append(str(error))
    assert len(messages) == 1 and "eager graph of the same leaf" in messages[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, l.detach() * 2)
    torch.autograd.grad(eager.sum(), l)


@gpu
def test_refusals(dev):
    l = logits_of("normal", 6, 10, torch.float32, dev, 1)
    for bad, match in (((l.double(), 2), "float32, float16 or bfloat16"), ((l[0], 2), "two dimensions"), ((l, 11), "choices"),
                       ((l, -1), "choices"), ((l.cpu(), 2), "GPU tensor"), ((torch.zeros(2, 4097, device=dev), 2), "4096"),
                       ((torch.zeros(2, 100, device=dev), 65), "choices")):
        with pytest.raises(RuntimeError, match=match):
            gs.ops.expert_choose(*bad)
    experts, weights = gs.ops.expert_choose(l, 2)
    grad = torch.ops.gs_ops._CAPI_ExpertChooseGrad
    for bad, match in (((weights[:5], l, experts, weights, True), "shape"), ((weights.half(), l, experts, weights, True), "float32"),
                       ((weights, l, experts.long(), weights, True), "int32"), ((weights, l, experts[:5], weights[:5], True), "int32"),
                       ((weights.cpu(), l, experts, weights, True), "GPU tensor")):
        with pytest.raises(RuntimeError, match=match):
            grad(*bad)
    # experts that are none count for nothing
    outside = torch.tensor([[10, -7], [2 ** 31 - 1, -2 ** 31]] * 3, dtype=torch.int32, device=dev)
    for normalize in (True, False):
        assert not grad(weights, l, outside, weights, normalize).any()
    l.requires_grad_(True)
    with pytest.raises(RuntimeError, match="once more"):
        torch.autograd.grad(gs.ops.expert_choose(l, 2)[1].sum(), l, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gs.ops.expert_choose(t, 2)[1].sum())(l.detach())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_experts_and_choices_around_every_limit(dev, dtype):
    for num in (4, 8, 9, 15, 16, 17, 24, 25, 31, 32, 33, 48, 49, 64, 65, 96, 97, 128, 129, 192, 193, 255, 256, 257, 320, 321, 384,
                385, 511, 512, 513, 768, 769, 1024, 1025, 1536, 1537, 2048, 2049, 4095, 4096):
        for choices in {min(k, num) for k in (1, 4, 5, 8, 9, 16, 17, 32, 33, 64)}:
            tokens = 5 + num % 7
            logits = logits_of("masked" if choices % 2 else "ties", tokens, num, dtype, dev, num + choices)
            for normalize in (True, False):
                x = logits.detach().requires_grad_(True)
                experts, weights = gs.ops.expert_choose(x, choices, normalize)
                grad = torch.randn(tokens, choices, generator=torch.Generator().manual_seed(1)).to(dev)
                dx, = torch.autograd.grad(weights, x, grad)
                want = formula(logits, choices, normalize, grad)
                assert np.array_equal(experts.cpu().numpy(), want[0])
                assert np.allclose(weights.detach().cpu().numpy(), want[1], rtol=(200 + num + 12) * STEP, atol=TINY)
                tol = want[3] * (200 + num + 20) * STEP + np.abs(want[2]) * half_step(dtype) + smallest(dtype)
                assert (np.abs(dx.double().cpu().numpy() - want[2]) <= tol).all()


# ------------------------------------------------------------------ no GPU ----
def test_bad_arguments_are_refused_before_anything_is_launched():
    import ctypes
    lib, i64 = capi.lib(), ctypes.c_int64
    buf = (ctypes.c_int64 * 64)()
    at = ctypes.addressof(buf)

    def fails(status, match):
        assert status < 0 and match in lib.gs_status_string(status), (status, lib.gs_status_string(status))

    def choose(logits=buf, stride=8, kind=0, tokens=2, num=8, k=2, experts=buf, weights=buf):
        return lib.gs_expert_choose(logits, i64(stride), kind, i64(tokens), i64(num), i64(k), 1, experts, weights, None)

    def grad(logits=buf, kind=0, experts=buf, weights=buf, dweights=buf, tokens=2, num=8, k=2, normalize=0, out=buf):
        return lib.gs_expert_choose_grad(logits, i64(8), kind, experts, weights, dweights, i64(tokens), i64(num), i64(k), normalize,
                                         out, None)

    assert choose(tokens=0) == choose(k=0) == grad(tokens=0) == grad(num=0, k=0) == 0
    for change, match in ((dict(kind=7), b"value type"), (dict(tokens=-1), b"negative"), (dict(num=4097), b"4096"),
                          (dict(k=9), b"choices"), (dict(num=100, k=65), b"choices"), (dict(tokens=1 << 31), b"2^31"),
                          (dict(logits=None), b"null"), (dict(experts=None), b"null"), (dict(weights=None), b"null"),
                          (dict(logits=ctypes.c_void_p(at + 2)), b"aligned"), (dict(stride=-1), b"negative")):
        fails(choose(**change), match)
    for change, match in ((dict(kind=7), b"value type"), (dict(num=4097), b"4096"), (dict(out=None), b"null"),
                          (dict(logits=None), b"null"), (dict(experts=None), b"null"), (dict(dweights=None), b"null"),
                          (dict(out=ctypes.c_void_p(at + 2)), b"aligned")):
        fails(grad(**change), match)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU tensor"):
        gs.ops.expert_choose(torch.zeros(3, 4), 2)
