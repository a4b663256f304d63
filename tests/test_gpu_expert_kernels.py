"""Every kernel of gs.ops.expert_matmul and its gradients, in whole numbers: equal to the formulas in 64 bits, with nothing
around their results touched.

Which kernel a call takes is a rule on its sizes, types and alignment.  CASES reach every one that the library holds, of
widths that are odd, and that are not, where it can have both; without a GPU it is checked that they still do, by the library's own
choices, with launches written down instead of made."""
import ctypes
import json
import os
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

import graph_sampling_amd as gs
from graph_sampling_amd import build, capi
from test_gpu_expert_products import formula, loads_of, order_of, weights_of, whole

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
HERE = os.path.dirname(os.path.abspath(__file__))

CASES = [
    # rows, experts, inner, outer, transposed
    (283, 1, 1, 3, True), (1108, 3, 2, 1, False), (2152, 1, 16, 16, True), (2258, 1, 37, 13, False), (1, 1, 16, 16, False),
    (2, 1, 89, 9, True), (101, 28, 3, 309, False), (347, 1, 640, 464, True), (161, 1, 2587, 847, True),
    (5011, 5, 146, 165, True), (4781, 3, 197, 131, True), (715, 1, 2304, 400, False), (530773, 1, 9, 9, False),
    (550407, 5, 9, 10, True), (883, 1, 1731, 311, False), (812, 55, 272, 272, True), (335, 1, 5869, 829, True),
    (1026, 69, 275, 257, False), (24, 287, 360, 3, True), (28410, 1, 129, 135, False), (10188, 66, 416, 112, False),
    (3018, 2, 176, 1840, False), (19886, 8, 549, 343, False), (41415, 2, 23, 420, False), (10772, 2, 27, 1971, False),
    (536808, 5, 9, 68, True), (524610, 1, 13, 67, True), (7255, 2, 270, 1340, False), (276720, 30, 65, 69, False),
    (5, 6, 1773, 8, False), (262264, 1, 80, 80, True), (554688, 3, 43, 67, False), (590895, 2, 36, 73, False),
    (14813, 44, 784, 912, False), (265, 1, 4336, 2624, False), (5073, 6, 69, 3995, True), (262145, 17, 129, 11, False),
    (537116, 9, 33, 35, False), (263786, 15, 140, 8, True), (267336, 40, 142, 10, False), (273736, 3, 141, 9, True),
    (647831, 6, 42, 33, True), (155, 72, 3264, 320, True), (263, 97, 3129, 285, False), (12, 14, 3536, 1872, False),
    (14429, 37, 2183, 343, True), (533602, 11, 65, 37, False), (549449, 13, 71, 34, False),
]


# of experts, and of choices, on both sides of every size at which the kernels of gs.ops.expert_choose change
NUMBERS = (4, 8, 9, 15, 16, 17, 24, 25, 31, 32, 33, 48, 49, 64, 65, 96, 97, 128, 129, 192, 193, 255, 256, 257, 320, 321, 384, 385, 511,
           512, 513, 768, 769, 1024, 1025, 1536, 1537, 2048, 2049, 4095, 4096)
CHOICES = (1, 4, 5, 8, 9, 16, 17, 32, 33, 64)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,experts,inner,outer,transposed", CASES)
def test_every_kernel(dev, n, experts, inner, outer, transposed, dtype):
    """Sums of products of -3 .. 3 are below 2^24 (9 of the longest depth, 647 831), and exact; fp16 results below its largest value
    (by the random signs 3 * 805 * 6, six standard deviations)."""
    for kind in ("even", "skewed"):
        loads = loads_of(kind, n, experts, n + outer)
        order = order_of(loads, n, dev)
        rows, grad = (whole(n, d, dtype=dtype, dev=dev, seed=d) for d in (inner, outer))
        weight = weights_of(whole, experts, inner, outer, transposed, dtype=dtype, dev=dev, seed=3)
        x, w = rows.clone().requires_grad_(True), weight.detach().requires_grad_(True)
        out = gs.ops.expert_matmul(x, order, w)
        got = (out.detach(),) + torch.autograd.grad(out, (x, w), grad)
        for a, b in zip(got, formula(rows, loads, weight, grad)[::2]):
            assert torch.equal(a, b.to(dtype))
        # what belongs to another expert, or to nobody, does not matter
        at = np.append(0, np.cumsum(loads))
        e = int(np.argmax(loads)) // 2
        of = slice(int(at[e]), int(at[e + 1]))
        rows[of], grad[of] = float("nan"), float("inf")
        rows[at[-1]:], grad[at[-1]:] = float("inf"), float("nan")
        weight = weight.clone()
        weight[e] = float("nan")
        for a, b, g in ((gs.ops.expert_matmul(rows, order, weight), got[0], got[0]),
                        (gs.ops.expert_matmul(grad, order, weight.transpose(1, 2)), got[1], got[1])):
            assert torch.equal(a[:of.start], b[:of.start]) and torch.equal(a[of.stop:], b[of.stop:])
            assert not a[of].isfinite().any()
        d = capi.expert_matmul_grad(grad, rows, order.offsets)
        assert torch.equal(d[:e], got[2][:e]) and torch.equal(d[e + 1:], got[2][e + 1:])
        assert loads[e] == 0 or not d[e].isfinite().any()


def guarded(shape, dtype, dev):
    """A tensor in the middle of a larger one full of a value, and whether what lies around it still has that value."""
    size = int(np.prod(shape)) * torch.finfo(dtype).bits // 8
    room = 1 << 16
    whole_of = torch.full((room + (size + 255) // 256 * 256 + room,), 0x5a, dtype=torch.uint8, device=dev)
    mine = whole_of[room:room + size].view(dtype).view(shape)

    def untouched():
        return bool((whole_of[:room] == 0x5a).all()) and bool((whole_of[room + size:] == 0x5a).all())

    return mine, untouched


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,experts,inner,outer", [
    (90, 3, 1001, 333), (24, 3, 3497, 72), (700, 3, 2070, 351),                # few rows
    ((1 << 19) + 9, 3, 40, 56), ((1 << 19) + 9, 3, 33, 67), (9000, 3, 27, 1971),  # small matrices, many rows
    (300, 3, 24, 40), (300, 3, 5, 3), (5011, 3, 146, 165), (14_813, 3, 784, 912), (12_100, 3, 259, 1027),  # tiles
    (100_001, 3, 33, 9), (3018, 3, 176, 1840),                                 # pieces of rows
])
def test_nothing_around_the_results_is_touched_whatever_the_offsets_hold(dev, n, experts, inner, outer, dtype):
    """The C entry points, results and workspace in the middle of memory that is looked at afterwards.  Offsets that ascend once they
    are brought between 0 and n have their rows' results; others leave rows out, or write them twice."""
    lib, i64 = capi.lib(), ctypes.c_int64
    kind = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    rows, grad = (whole(n, d, dtype=dtype, dev=dev, seed=d) for d in (inner, outer))
    for at in ([0, n // 3, n // 2, n], [0, 2 ** 40, 2 ** 40, 2 ** 62], [-5, 10, 20, n + 400], [0, n, n // 3, 3], [n, n // 2, n // 3, 0],
               [-2 ** 62, -7, -1, -1], [0, n, 0, n], [-2 ** 63, 2 ** 63 - 1, -2 ** 63, 2 ** 63 - 1], [7, n // 3, n // 3, n - 9]):
        offsets = torch.tensor(at, device=dev)
        held = np.clip(np.array(at, dtype=object), 0, n).astype(np.int64)
        ascend = bool((np.diff(held) >= 0).all())
        loads = np.append(held[0], np.diff(held))  # (rows before the first offset are nobody's, and not written)
        for transposed in (False, True):
            weight = weights_of(whole, experts, inner, outer, transposed, dtype=dtype, dev=dev, seed=3)
            out, untouched = guarded((n, outer), dtype, dev)
            stride = inner if transposed else outer
            rc = lib.gs_expert_matmul(capi._ptr(rows), i64(inner), i64(n), i64(inner), kind, capi._ptr(weight), i64(inner * outer),
                                      i64(stride), int(transposed), i64(experts), i64(outer), capi._ptr(offsets), capi._ptr(out),
                                      capi._stream(dev))
            assert rc == 0 and untouched()
            if ascend:
                nobody = torch.zeros(1, inner, outer, dtype=dtype, device=dev)
                want = formula(rows, loads, torch.cat([nobody, weight]))[0].to(dtype)
                assert torch.equal(out[held[0]:], want[held[0]:])
        dw, untouched = guarded((experts, inner, outer), dtype, dev)
        size = lib.gs_expert_matmul_grad_workspace_bytes(i64(n), i64(inner), i64(outer), i64(experts))
        ws, ws_untouched = guarded((size // 4,), torch.float32, dev)
        rc = lib.gs_expert_matmul_grad(capi._ptr(rows), i64(inner), i64(inner), capi._ptr(grad), i64(outer), i64(outer), kind, i64(n),
                                       capi._ptr(offsets), i64(experts), capi._ptr(dw), capi._ptr(ws), ctypes.c_size_t(size),
                                       capi._stream(dev))
        assert rc == 0 and untouched() and ws_untouched()
        if ascend:
            want = formula(rows, loads, torch.zeros(experts + 1, inner, outer, dtype=dtype, device=dev), grad)[4][1:]
            assert torch.equal(dw, want.to(dtype))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_around_choices_and_what_dropout_leaves_is_touched(dev, dtype):
    """Numbers of tokens, experts and values that end inside a workgroup, a group of lanes and a chunk."""
    lib, i64 = capi.lib(), ctypes.c_int64
    kind = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    for tokens, num, choices in ((1, 1, 1), (65, 3, 2), (33, 17, 3), (50, 65, 8), (9, 193, 16), (7, 385, 17), (5, 1001, 64), (3, 4095, 5)):
        logits = whole(tokens, num, dtype=dtype, dev=dev, seed=num)
        for normalize in (0, 1):
            weights, w_ok = guarded((tokens, choices), torch.float32, dev)
            experts, e_ok = guarded((tokens, choices), torch.float32, dev)  # (as wide as int32)
            d, d_ok = guarded((tokens, num), dtype, dev)
            assert lib.gs_expert_choose(capi._ptr(logits), i64(num), kind, i64(tokens), i64(num), i64(choices), normalize,
                                        capi._ptr(experts), capi._ptr(weights), capi._stream(dev)) == 0
            assert lib.gs_expert_choose_grad(capi._ptr(logits), i64(num), kind, capi._ptr(experts), capi._ptr(weights),
                                             capi._ptr(weights), i64(tokens), i64(num), i64(choices), normalize, capi._ptr(d),
                                             capi._stream(dev)) == 0
            assert w_ok() and e_ok() and d_ok()
            want = capi.expert_choose(logits, choices, bool(normalize))
            assert torch.equal(experts.view(torch.int32), want[0]) and torch.equal(weights, want[1])
            assert torch.equal(d, capi.expert_choose_grad(weights.clone(), logits, want[0], want[1], bool(normalize)))
    for n in (1, 7, 8, 1023, 2048, 2049, 100_003):
        x = whole(n, dtype=dtype, dev=dev, seed=n)
        out, untouched = guarded((n,), dtype, dev)
        assert lib.gs_dropout(capi._ptr(x), None, i64(n), kind, ctypes.c_double(0.5), ctypes.c_uint64(3), None, capi._ptr(out),
                              capi._stream(dev)) == 0
        assert untouched() and torch.equal(out, capi.dropout(x, 0.5, 3))


# ------------------------------------------------------------------ no GPU ----
_WRITTEN_DOWN = """
import ctypes, json, sys
stand_in = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
stand_in.launches.restype = stand_in.kernels.restype = ctypes.c_char_p
lib.gs_expert_matmul_grad_workspace_bytes.restype = ctypes.c_size_t
i64, at = ctypes.c_int64, [ctypes.c_void_p(1 << k) for k in range(30, 40)]

def launched(status):
    assert status == 0, status
    return [line.split() for line in stand_in.launches().decode().splitlines()]

def matmul(n, num, inner, outer, kind, transposed):
    return launched(lib.gs_expert_matmul(at[0], i64(inner), i64(n), i64(inner), kind, at[1], i64(inner * outer),
                                         i64(inner if transposed else outer), int(transposed), i64(num), i64(outer), at[2], at[3], None))

def grad(n, num, inner, outer, kind):
    size = lib.gs_expert_matmul_grad_workspace_bytes(i64(n), i64(inner), i64(outer), i64(num))
    return launched(lib.gs_expert_matmul_grad(at[0], i64(inner), i64(inner), at[1], i64(outer), i64(outer), kind, i64(n), at[2],
                                              i64(num), at[3], at[4], ctypes.c_size_t(size), None))

def choose(num, choices, kind):
    return (launched(lib.gs_expert_choose(at[0], i64(num), kind, i64(50), i64(num), i64(choices), 1, at[1], at[2], None)) +
            launched(lib.gs_expert_choose_grad(at[0], i64(num), kind, at[1], at[2], at[3], i64(50), i64(num), i64(choices), 1, at[4],
                                               None)))

out = [{"matmul": matmul, "grad": grad, "choose": choose}[call[0]](*call[1:]) for call in json.loads(sys.stdin.read())]
print(json.dumps({"calls": out, "kernels": stand_in.kernels().decode().split()}))
"""


@pytest.fixture(scope="module")
def written_down(tmp_path_factory):
    """calls -> what each would launch, and all kernels that the library holds; in a process of its own, without a GPU."""
    stand_in = str(tmp_path_factory.mktemp("launches") / "launches.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(HERE, "cpp", "launches.cc"), "-o", stand_in],
                   check=True)

    def run(calls):
        done = subprocess.run([sys.executable, "-c", _WRITTEN_DOWN, stand_in, build.KERNEL_LIB], input=json.dumps(calls),
                              capture_output=True, text=True)
        assert done.returncode == 0, done.stderr
        return json.loads(done.stdout)

    return run


def _of_products(name):
    return re.search(r"\d(few_rows|narrow|product|weight_grad|join_pieces)_kernelI", name)


def test_the_cases_reach_every_kernel(written_down):
    calls = [call for n, num, inner, outer, transposed in CASES for kind in range(3) for call in (
        ("matmul", n, num, inner, outer, kind, transposed), ("matmul", n, num, outer, inner, kind, not transposed),
        ("grad", n, num, inner, outer, kind))]
    done = written_down(calls)
    reached = {kernel for launches in done["calls"] for kernel, *_ in launches}
    there = {kernel for kernel in done["kernels"] if _of_products(kernel)}
    assert len(there) > 100 and there - reached == set()


def test_the_numbers_of_experts_and_choices_reach_every_kernel(written_down):
    """Those that test_gpu_expert_choice.py looks at."""
    calls = [("choose", num, min(choices, num), kind) for num in NUMBERS for choices in CHOICES for kind in range(3)]
    done = written_down(calls)
    reached = {kernel for launches in done["calls"] for kernel, *_ in launches}
    there = {kernel for kernel in done["kernels"] if re.search(r"\dchoose(_grad)?_kernelI", kernel)}
    assert len(there) > 80 and there - reached == set()


def test_many_tiles_are_launched_in_turns(written_down):
    """Each launch within what one counts (2^32 threads), every turn but the last a multiple of the dies, all tiles there."""
    of_64, of_16 = ((70_000 // rows + 65_536) for rows in (64, 16))  # tiles of rows that there can be
    for call, tiles in ((("matmul", 1 << 30, 65, 8, 64, 0, False), (1 << 30) // 64),
                        (("matmul", 70_000, 65_536, 8, 16_384, 0, False), of_64 * 256),
                        (("matmul", 70_000, 65_536, 128, 4096, 0, False), of_16 * 128),
                        (("grad", 70_000, 65_536, 4, 16_448, 0), 65_536 * 257), (("matmul", 100, 5, 64, 64, 0, False), 1),
                        (("grad", 1 << 20, 3, 64, 64, 0), 128)):
        launches, = written_down([call])["calls"]
        first = [(int(blocks), int(threads)) for kernel, blocks, threads, _ in launches if kernel == launches[0][0]]
        assert all(blocks * threads < 1 << 32 for blocks, threads in first)
        assert all(blocks % 8 == 0 for blocks, _ in first)
        assert tiles <= sum(blocks for blocks, _ in first) <= tiles * 1.05 + 4096
        assert (len(first) > 1) == (sum(blocks * threads for blocks, threads in first) >= 1 << 32)
