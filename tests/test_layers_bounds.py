"""Plans that are none, and memory that is not there: what the layers' operators read and take then."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import mops_amd
from mops_amd import layers
from tests.test_layers import assert_within, random

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_on_host(tmp_path, text, *arguments):
    """The output of a C++ program over the kernels' own headers, in numbers."""
    source, program = tmp_path / "program.cpp", tmp_path / "program"
    source.write_text(text)
    include = os.path.join(ROOT, "mops_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", include, "-o", str(program), str(source)], check=True)
    done = subprocess.run([str(program), *map(str, arguments)], check=True, capture_output=True, text=True)
    return np.array([[int(x) for x in line.split()] for line in done.stdout.splitlines()], dtype=np.int64)


PLACES = """
#include <cstdio>
#include <cstdlib>
#include "plan_bounds.hpp"
using namespace mops::amd;
// (what overflows is no constant expression: these lines would not compile)
static_assert(places_between(2147483647, 2147483647, 200000).begin == 200000, "");
static_assert(chunks_inside(places_between(2147483647, -2147483647 - 1, 2147418111), 8192).begin == 262136, "");
static_assert(chunks_inside(places_between(-2147483647 - 1, 2147483647, 2147418111), 8192).end == 262135, "");
int main(int n, char** a) {
    for (int i = 1; i + 3 < n; i += 4) {
        const Range places = places_between(atoi(a[i]), atoi(a[i + 1]), atoi(a[i + 2]));
        const Range chunks = chunks_inside(places, atoi(a[i + 3]));
        printf("%d %d %d %d\\n", places.begin, places.end, chunks.begin, chunks.end);
    }
}
"""


def test_offsets_that_are_none_stay_within_the_rows(tmp_path):
    """The places and chunks that the gradient of the embedding and the products count from two neighbouring offsets:
    within the rows for every pair of offsets, near the ends of 32 bits, negative and decreasing ones among them."""
    low, high = np.iinfo(np.int32).min, np.iinfo(np.int32).max
    rng = np.random.default_rng(0)
    points = []
    for n_rows in (0, 1, 63, 64, 257, 200_000, high - 65536):
        near = [low, low + 1, -1, 0, 1, 63, n_rows // 2, n_rows - 1, n_rows, n_rows + 1, high - 8192, high - 1, high]
        near = [int(np.clip(x, low, high)) for x in near] + rng.integers(low, high, 3).tolist()
        points += [(a, b, n_rows, chunk) for a in near for b in near for chunk in (32, 64, 8192)]
    got = np.concatenate(
        [run_on_host(tmp_path, PLACES, *np.ravel(points[i : i + 1000])) for i in range(0, len(points), 1000)]
    )
    a, b, n_rows, chunk = np.array(points, dtype=np.int64).T
    begin = np.clip(a, 0, n_rows)
    end = np.maximum(np.minimum(b, n_rows), begin)
    np.testing.assert_array_equal(got, np.stack([begin, end, -(-begin // chunk), end // chunk], 1))
    # nothing that a workgroup counts past a place leaves 32 bits: 256 teams with eight rows on their way each
    assert (got[:, :2] + 256 * 64).max() <= high and (got * np.array([1, 1, 0, 0])).min() >= 0
    inside = got[:, 2] < got[:, 3]
    assert ((got[:, 3] * chunk)[inside] <= n_rows[inside]).all()


UNITS = """
#include <cstdio>
#include <cstdlib>
#include "plan_bounds.hpp"
using namespace mops::amd;
static_assert(units_to_sum(2147418111, 2147418112) == 1, "");
int main(int n, char** a) {
    const int step = atoi(a[1]);
    long long rows = 0;
    int split = 0;
    for (int i = 2; i < n; i++) { // the groups' sizes
        const int units = units_to_sum(atoi(a[i]), step);
        rows += atoi(a[i]);
        split += units > 1 ? units : 0;
    }
    printf("%d %d\\n", split, most_split_units(int(rows), step));
}
"""


def test_units_of_split_groups_are_few(tmp_path):
    """Room for partial results is for the units of groups of more than one unit: never too little, none where no group
    can have two, and not more for more groups."""
    rng = np.random.default_rng(1)
    reached = 0
    for step, sizes in [
        (256, [447]), (256, [448]), (256, [0, 448, 448, 448, 447]), (64, [112] * 50), (64, [111] * 50), (320, [0] * 100),
        (57344, [256] * 256), (57344, [65536]), (1 << 20, [(1 << 20) * 7 // 4 - 1]),
        *[(64 * int(rng.integers(1, 20)), rng.integers(0, 4000, 40).tolist()) for _ in range(20)],
    ]:  # fmt: skip
        split, most = run_on_host(tmp_path, UNITS, step, *sizes)[0]
        assert split <= most <= 8 * sum(sizes) / (7 * step)
        assert most == 0 or sum(sizes) >= 1.75 * step
        reached += split == most
    assert reached >= 6


GROUPS = {  # sizes of the groups: some of several units in front, between and behind those of one, of more and fewer groups than a wavefront has lanes
    "wide": [700] + [0, 1, 3] * 23 + [900, 2] + [1] * 60 + [2048, 5, 0, 600],
    "narrow": [1, 900, 0, 2, 448, 447, 3000, 0],
    "many": [0] * 300 + [1500] + [1, 0] * 150 + [449, 512],
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64], ids=str)
@pytest.mark.parametrize("columns", [(64, 72), (31, 33)], ids=str)
@pytest.mark.parametrize("sizes", list(GROUPS))
def test_gradients_of_groups_of_several_units(device, sizes, columns, dtype):
    K, L = columns
    sizes = torch.tensor(GROUPS[sizes])
    rows, groups = int(sizes.sum()), len(sizes)
    generator = torch.Generator().manual_seed(rows + K)
    A, grad_output = [random(generator, (rows, width), dtype) for width in (K, L)]
    W = random(generator, (groups, K, L), dtype)
    offsets = torch.zeros(groups + 1, dtype=torch.int32)
    offsets[1:] = sizes.cumsum(0)
    order = torch.randperm(rows, generator=generator).int()
    arguments = [x.to(device) for x in (grad_output, A, W, offsets, order)]
    _, grad_W = mops_amd.grouped_matrix_product_vjp(*arguments, compute_grad_A=False)
    exact, magnitude = torch.zeros(2, groups, K, L, dtype=torch.float64)
    for g in range(groups):
        mine = order[offsets[g] : offsets[g + 1]].long()
        a, c = A[mine].double(), grad_output[mine].double()
        exact[g], magnitude[g] = a.t() @ c, a.abs().t() @ c.abs()
    assert_within(grad_W, exact, magnitude, int(sizes.max()), "grad_W")
    assert torch.equal(mops_amd.grouped_matrix_product_vjp(*arguments)[1], grad_W)


MANY_GROUPS = """
import ctypes
import torch
import mops_amd
from mops_amd._c_lib import device_library

capacity = device_library().cdll.mops_amd_scratch_capacity
capacity.restype = ctypes.c_int64
device = torch.device("cuda:0")
torch.manual_seed(0)
rows, groups, K, L = 1000, 512, 256, 256
A, grad_output = torch.randn(rows, K, device=device), torch.randn(rows, L, device=device)
W = torch.randn(groups, K, L, device=device)
for index in (torch.arange(rows, device=device) % groups, torch.zeros(rows, device=device)):
    order, offsets = mops_amd.order_by_group(index.int(), groups)
    grad_A, grad_W = mops_amd.grouped_matrix_product_vjp(grad_output, A, W, offsets, order)
    exact = torch.zeros(groups, K, L, dtype=torch.float64)
    for row in range(rows):
        exact[int(index[row])] += torch.outer(A[row].cpu().double(), grad_output[row].cpu().double())
    error = (grad_W.cpu().double() - exact).abs().max().item()
    assert error < 0.05, error  # (1016 2^-24 times the magnitudes of 1000 products, which add up to some 640)
    print("ok", capacity(), flush=True)
# the groups that can be split at all, of 256 rows or more, have four units
assert 0 < capacity() <= 4 << 20, capacity()
"""


@pytest.mark.gpu
def test_many_groups_take_no_scratch_memory_each(device):
    """Partial results need room for the groups that are split, not for every group. In a process of its own, whose thread
    has no scratch memory from other calls."""
    done = subprocess.run([sys.executable, "-c", MANY_GROUPS], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout + done.stderr[-3000:]
    assert done.stdout.count("ok ") == 2, done.stdout


THREADS = """
import ctypes, threading
import torch
import mops_amd
from mops_amd._c_lib import device_library

library = device_library().cdll
library.mops_amd_scratch_capacity.restype = ctypes.c_int64
library.mops_amd_reserve_scratch.argtypes = [ctypes.c_int64]
device = torch.device("cuda:0")
end = threading.Event()

def in_a_thread(function):
    \"\"\"The result in a new thread, which lives on and so keeps its scratch memory.\"\"\"
    results, done = [], threading.Event()
    def work():
        try:
            results.append(function())
        except BaseException as error:
            results.append(error)
        done.set()
        end.wait()
    threading.Thread(target=work, daemon=True).start()
    assert done.wait(60)
    if isinstance(results[0], BaseException):
        raise results[0]
    return results[0]

def case(rows, K, L, dtype):
    generator = torch.Generator().manual_seed(K)
    A, W, grad_output = [
        torch.randn(shape, generator=generator, dtype=torch.float32).to(device, dtype)
        for shape in ((rows, K), (1, K, L), (rows, L))
    ]
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=device)
    exact = [A.double() @ W[0].double(), grad_output.double() @ W[0].double().t(), A.double().t() @ grad_output.double()]
    vjp = lambda *wanted: mops_amd.grouped_matrix_product_vjp(grad_output, A, W, offsets, None, *wanted)
    return {
        "product": (lambda: [mops_amd.grouped_matrix_product(A, W, offsets)], exact[:1], K),
        "grad_A": (lambda: [vjp(True, False)[0]], exact[1:2], L),
        "grad_W": (lambda: [vjp(False, True)[1].squeeze(0)], exact[2:], rows),
        "gradients": (lambda: [x.squeeze(0) for x in vjp()], exact[1:], max(L, rows)),
    }

def check(results, exact, unit, terms):
    for result, wanted in zip(results, exact, strict=True):
        # (numbers of size 1: the magnitudes of a sum of n terms add up to less than n)
        error = (result.double() - wanted).abs().max().item()
        assert error <= (terms + 16) * unit[0] * terms + unit[1] * wanted.abs().max().item(), (error, terms)
"""

CAPTURED = THREADS + """
def eager(call):
    results = call()
    torch.cuda.synchronize()
    return results, library.mops_amd_scratch_capacity()

def captured(call, capacity):
    assert library.mops_amd_reserve_scratch(int(capacity / 1.5)) == 0
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        results = call()
    for _ in range(2):
        for result in results:
            result.zero_()
        graph.replay()
        torch.cuda.synchronize()
    return results, library.mops_amd_scratch_capacity()

# the product and grad_A share out a long sum, grad_W the rows of its group
for name, sizes in [
    ("product", (768, 20001, 767)), ("grad_A", (768, 767, 20001)), ("grad_W", (20001, 767, 767)),
    ("gradients", (20001, 767, 767)), ("gradients", (768, 767, 20001)),
]:
    call, exact, terms = case(*sizes, torch.float64)[name]
    results, capacity = in_a_thread(lambda: eager(call))
    check(results, exact, (2.0**-53, 2.0**-53), terms)
    print("eager", name, capacity, flush=True)
    # a block that holds the copies, but not all of the partial results as well (blocks are made half as large again as
    # what is asked for)
    room = capacity / 1.5 - (3 << 20)
    results, got = in_a_thread(lambda: captured(call, room))
    check(results, exact, (2.0**-53, 2.0**-53), terms)
    assert got <= room, (got, room)
    print("ok", name, got, flush=True)
end.set()
"""


@pytest.mark.gpu
def test_a_captured_call_whose_block_holds_the_copies_only(device):
    """Products at odd addresses copy their operands where there is room; during a capture the block has to hold the
    copies and the partial results, or the call does without copies."""
    done = subprocess.run([sys.executable, "-c", CAPTURED], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout + done.stderr[-3000:]
    assert done.stdout.count("ok ") == 5, done.stdout


FULL_DEVICE = THREADS + """
import os
LIMIT = "MOPS_AMD_TEST_SCRATCH_LIMIT"  # what a nearly full device has left for the block
os.environ[LIMIT] = str(200 << 20)

def calls():
    for name, sizes in [
        ("product", (768, 20001, 767)), ("grad_A", (768, 767, 20001)), ("grad_W", (20001, 767, 767)),
        ("gradients", (20001, 767, 767)), ("gradients", (768, 767, 20001)),
    ]:
        call, exact, terms = case(*sizes, torch.float64)[name]
        check(call(), exact, (2.0**-53, 2.0**-53), terms)
        print("ok", name, library.mops_amd_scratch_capacity(), flush=True)
        assert library.mops_amd_scratch_capacity() < 200 << 20
    capacity = library.mops_amd_scratch_capacity()
    assert 0 < capacity
    # memory that a call cannot do without: an error, and no trace of it in the next call
    assert library.mops_amd_reserve_scratch(400 << 20) == 1
    check(call(), exact, (2.0**-53, 2.0**-53), terms)
    # no room for half as much again: what is asked for
    assert library.mops_amd_reserve_scratch(180 << 20) == 0
    assert library.mops_amd_scratch_capacity() == 180 << 20
    check(call(), exact, (2.0**-53, 2.0**-53), terms)
    assert library.mops_amd_scratch_capacity() == 180 << 20
    # memory again
    del os.environ[LIMIT]
    check(call(), exact, (2.0**-53, 2.0**-53), terms)
    assert library.mops_amd_scratch_capacity() > 300 << 20
    print("ok", flush=True)

in_a_thread(calls)
end.set()
"""


@pytest.mark.gpu
def test_products_on_a_device_that_is_nearly_full(device):
    """Copies of operands are memory that a call can do without: where the device has none left, the call runs as it would
    at odd addresses."""
    done = subprocess.run([sys.executable, "-c", FULL_DEVICE], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout + done.stderr[-3000:]
    assert done.stdout.count("ok") == 6, done.stdout


WIDE_INDICES = [
    0, 4, 5, -1, 2, 3, 2**31 - 1, 2**31, 2**31 + 2, 2**32 - 1, 2**32, 2**32 + 3, -(2**31), -(2**31) - 1, -(2**32), 1, 2**33 + 1,
    -(2**32) + 2, -(2**63), -(2**63) + 1, 2**63 - 1, 2**62 + 4, 3,
]  # fmt: skip


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint64, torch.uint32, torch.int16, torch.uint8], ids=str)
def test_wide_indices_in_32_bits(dtype):
    """An index outside of 32 bits is outside of every range: no other index of 32 bits stands for it."""
    low, high = (0, 2 ** (8 * dtype.itemsize)) if "uint" in str(dtype) else [s * 2 ** (8 * dtype.itemsize - 1) for s in (-1, 1)]
    values = [v for v in [*WIDE_INDICES, 2**63, 2**63 + 3, 2**64 - 1, 200] if low <= v < high]
    got = layers._int32(torch.tensor(values, dtype=dtype))
    assert got.dtype == torch.int32
    for value, index in zip(values, got.tolist()):
        assert index == value if 0 <= value < 2**31 - 1 else index < 0 or index == 2**31 - 1, (value, index)


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["package", "operators"])
def test_indices_beyond_32_bits_are_outside(device, where):
    """In every function that takes them, through the package and as an operator."""
    import mops_amd.torch

    ops = mops_amd if where == "package" else torch.ops.mops
    groups, columns = 5, 12
    index = torch.tensor(WIDE_INDICES, device=device)
    inside = (index >= 0) & (index < groups)
    narrow = torch.where(inside, index, -1).int()
    order, offsets = ops.order_by_group(index, groups)
    assert all(torch.equal(x, y) for x, y in zip((order, offsets), mops_amd.order_by_group(narrow, groups)))
    assert offsets[-1].item() == int(inside.sum())
    table = torch.randn(groups, columns, device=device)
    output = ops.scaled_embedding(table, index, 2.0)
    assert torch.equal(output, mops_amd.scaled_embedding(table, narrow, 2.0)) and not output[~inside].any()
    grad_output = torch.randn(len(index), columns, device=device)
    expected = mops_amd.scaled_embedding_vjp(grad_output, table, narrow, 2.0)
    if where == "package":
        assert torch.equal(mops_amd.scaled_embedding_vjp(grad_output, table, index, 2.0), expected)
        assert torch.equal(mops_amd.scaled_embedding_vjp(grad_output, table, index, 2.0, order, offsets), expected)
    else:
        leaf = table.clone().requires_grad_(True)
        ops.scaled_embedding(leaf, index, 2.0).backward(grad_output)
        assert torch.equal(leaf.grad, expected)
