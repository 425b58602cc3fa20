"""The operators of the layers (mops_amd.layers) against their definitions in 64 bits.

Tolerances. A result of n terms that is summed in p bits and rounded once to q bits is off by at most
(n + c) 2^-p times the sum of the terms' magnitudes, plus 2^-q times itself, c for the few further operations on
each term. The sums here come in any order and partly pairwise, for which n is the bound as well. So every element is
held to::

    |actual - exact| <= (n + 16) 2^-p magnitude + 2^-q |exact| + tiny

with p = 24 and q = 24, 8 or 11 for float32, bfloat16 and float16 (p = q = 53 for float64), `magnitude` the same
formula with every term's absolute value, and `tiny` the smallest normal number of the type (below it results lose bits).
Comparisons of whole numbers are exact.
"""
import numpy as np
import pytest
import torch

import mops_amd
from mops_amd import layers

DTYPES = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}
WIDE_BITS = {torch.float32: 24, torch.float64: 53, torch.bfloat16: 24, torch.float16: 24}
BITS = {torch.float32: 24, torch.float64: 53, torch.bfloat16: 8, torch.float16: 11}


def assert_within(actual, exact, magnitude, terms, what):
    dtype = actual.dtype
    assert actual.shape == exact.shape, what
    if actual.numel() == 0:
        return
    actual, exact, magnitude = actual.double().cpu(), exact.cpu(), magnitude.cpu()
    bound = (terms + 16) * 2.0 ** -WIDE_BITS[dtype] * magnitude + 2.0 ** -BITS[dtype] * exact.abs()
    bound = bound + torch.finfo(dtype).tiny
    worst = ((actual - exact).abs() / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound"


def random(generator, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=generator, dtype=torch.float64) * scale).to(dtype)


def generator_of(*values):
    return torch.Generator().manual_seed(hash(tuple(values)) % (1 << 31))


def indices_of(kind, rows, groups, seed=0):
    rng = np.random.default_rng([seed, rows, groups])
    if kind == "uniform":
        index = rng.integers(0, groups, rows)
    elif kind == "one":  # every row in one group, the others empty
        index = np.full(rows, groups // 2)
    elif kind == "padded":  # some rows in no group: negative, or too large
        index = rng.integers(0, groups, rows)
        index[rng.random(rows) < 0.3] = -1
        index[rng.random(rows) < 0.1] = groups
        index[rng.random(rows) < 0.1] = np.iinfo(np.int32).max
        index[rng.random(rows) < 0.1] = np.iinfo(np.int32).min
    elif kind == "nowhere":  # no row in any group
        index = np.full(rows, -1)
    else:  # "frequent": few of them name most rows
        index = np.minimum((groups * rng.random(rows) ** 6).astype(np.int64), groups - 1)
    return torch.from_numpy(index.astype(np.int32))


def plan_of(index, groups):
    key = torch.where((index >= 0) & (index < groups), index.long(), groups)
    order = torch.argsort(key, stable=True)
    offsets = torch.searchsorted(key[order], torch.arange(groups + 1))
    return order.int(), offsets.int()


# -------------------------------------------------------------- the plan ----
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["uniform", "one", "padded", "nowhere", "frequent"])
@pytest.mark.parametrize(
    "rows,groups",
    [(0, 5), (1, 1), (7, 3), (1000, 1), (5000, 94), (4097, 511), (4097, 512), (9000, 5000), (70001, 100003),
     (300000, 7), (200, 3000000), (4096, 511), (4097, 64), (16384, 600), (16385, 600), (3001, 70000), (900, 20)],
)  # fmt: skip
def test_order_by_group(device, rows, groups, kind):
    index = indices_of(kind, rows, groups)
    order, offsets = mops_amd.order_by_group(index.to(device), groups)
    expected_order, expected_offsets = plan_of(index, groups)
    assert order.dtype == torch.int32 and offsets.dtype == torch.int32
    assert torch.equal(order.cpu(), expected_order)
    assert torch.equal(offsets.cpu(), expected_offsets)


@pytest.mark.gpu
def test_order_by_no_group(device):
    order, offsets = mops_amd.order_by_group(torch.tensor([3, -1, 0], dtype=torch.int64, device=device), 0)
    assert order.tolist() == [0, 1, 2] and offsets.tolist() == [0]


# ------------------------------------------------------------- embedding ----
EMBEDDINGS = [
    # rows, table rows, columns, indices
    (0, 5, 8, "uniform"), (1, 1, 1, "uniform"), (3, 4, 7, "padded"), (33, 10, 16, "uniform"), (65, 100, 3, "frequent"),
    (600, 4, 128, "uniform"), (5000, 94, 64, "frequent"), (700, 5000, 513, "frequent"), (129, 3, 2049, "one"),
    (3000, 2, 130, "padded"), (500, 40, 4099, "nowhere"), (20000, 5, 9, "one"), (1500, 7, 5000, "frequent"),
    (200, 3000000, 1, "uniform"), (50000, 60000, 8, "frequent"), (4096, 64, 8, "uniform"), (40000, 30000, 40, "frequent"),
]  # fmt: skip


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,table_rows,columns,kind", EMBEDDINGS)
def test_scaled_embedding(device, rows, table_rows, columns, kind, tag):
    dtype = DTYPES[tag]
    generator = generator_of(rows, table_rows, columns)
    table = random(generator, (table_rows, columns), dtype)
    index = indices_of(kind, rows, table_rows)
    inside = (index >= 0) & (index < table_rows)
    scale = 1.7
    exact = torch.where(inside[:, None], table.double()[torch.where(inside, index, 0).long()] * scale, 0.0)
    output = mops_amd.scaled_embedding(table.to(device), index.to(device), scale)
    assert output.dtype == dtype
    assert_within(output, exact, exact.abs(), 0, "embedding")
    assert not output[~inside.to(device)].any()


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,table_rows,columns,kind", EMBEDDINGS)
def test_scaled_embedding_vjp(device, rows, table_rows, columns, kind, tag):
    dtype = DTYPES[tag]
    generator = generator_of(rows, table_rows, columns, 1)
    table = torch.empty(table_rows, columns, dtype=dtype, device=device)
    index = indices_of(kind, rows, table_rows)
    grad_output = random(generator, (rows, columns), dtype)
    scale = 1.7
    inside = (index >= 0) & (index < table_rows)
    kept, target = grad_output.double()[inside], index[inside].long()
    exact = torch.zeros(table_rows, columns, dtype=torch.float64).index_add_(0, target, kept) * scale
    magnitude = torch.zeros(table_rows, columns, dtype=torch.float64).index_add_(0, target, kept.abs()) * scale
    on_device = grad_output.to(device), table, index.to(device), scale
    grad_table = mops_amd.scaled_embedding_vjp(*on_device)
    terms = torch.bincount(target, minlength=1).max().item() if len(target) else 0
    assert_within(grad_table, exact, magnitude, terms, "grad_table")
    # the caller's plan, and the same bits again
    plan = mops_amd.order_by_group(on_device[2], table_rows)
    assert torch.equal(mops_amd.scaled_embedding_vjp(*on_device, *plan), grad_table)
    assert torch.equal(mops_amd.scaled_embedding_vjp(*on_device), grad_table)


# ------------------------------------------------------ products by group ----
PRODUCTS = [
    # rows, groups, K, L, indices, in an order
    (0, 3, 8, 8, "uniform", True), (1, 1, 1, 1, "uniform", True), (5, 9, 3, 2, "uniform", True),
    (24, 16, 256, 130, "uniform", True), (64, 1, 64, 64, "uniform", False), (65, 2, 65, 63, "uniform", True),
    (600, 4, 128, 128, "frequent", True), (777, 5, 31, 257, "padded", True), (300, 70, 16, 48, "frequent", False),
    (515, 3, 129, 33, "one", True), (100, 4, 40, 24, "nowhere", True), (4000, 3, 8, 8, "frequent", False),
    (1030, 2, 512, 264, "uniform", True), (333, 200, 24, 72, "uniform", True), (2500, 2, 7, 515, "frequent", False),
]  # fmt: skip


# every extent of tiles with rows on 16-byte boundaries and off them, groups that are split into few and into many units,
# more groups than a wavefront has lanes
LARGE_PRODUCTS = [
    (8300, 3, 72, 2056, "padded", True), (8300, 3, 2056, 72, "frequent", True), (5000, 20, 1040, 1032, "frequent", True),
    (5000, 20, 1040, 1032, "uniform", False), (30000, 2, 64, 64, "frequent", False),
    (6000, 130, 70, 90, "frequent", True), (9000, 200, 256, 256, "uniform", True),
    (40000, 2, 130, 514, "padded", True), (4500, 3, 515, 777, "frequent", False), (70000, 3, 5, 3, "uniform", True),
    (7000, 2, 1031, 1029, "padded", True), (9001, 3, 1020, 1101, "uniform", False), (9001, 2, 1101, 1024, "padded", True),
]  # fmt: skip


def product_case(rows, groups, K, L, kind, dtype):
    generator = generator_of(rows, groups, K, L)
    A, W = random(generator, (rows, K), dtype), random(generator, (groups, K, L), dtype)
    grad_output = random(generator, (rows, L), dtype)
    index = indices_of(kind, rows, groups)
    return A, W, grad_output, index


def product_plan(index, groups, ordered):
    """(order or None, offsets, group of every row): in an order, or the rows as they lie, sorted."""
    if ordered:
        return (*plan_of(index, groups), index)
    index = torch.sort(index).values
    return None, plan_of(index, groups)[1], index


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,groups,K,L,kind,ordered", PRODUCTS + LARGE_PRODUCTS)
def test_grouped_matrix_product(device, rows, groups, K, L, kind, ordered, tag):
    A, W, _, index = product_case(rows, groups, K, L, kind, DTYPES[tag])
    order, offsets, index = product_plan(index, groups, ordered)
    output = mops_amd.grouped_matrix_product(
        A.to(device), W.to(device), offsets.to(device), None if order is None else order.to(device)
    )
    exact, magnitude = torch.zeros(rows, L, dtype=torch.float64), torch.zeros(rows, L, dtype=torch.float64)
    for g in range(groups):
        mask = index == g
        exact[mask] = A[mask].double() @ W[g].double()
        magnitude[mask] = A[mask].double().abs() @ W[g].double().abs()
    assert_within(output, exact, magnitude, K, "product")
    outside = ((index < 0) | (index >= groups)).to(device)
    assert not output[outside].any()


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,groups,K,L,kind,ordered", PRODUCTS + LARGE_PRODUCTS)
def test_grouped_matrix_product_vjp(device, rows, groups, K, L, kind, ordered, tag):
    A, W, grad_output, index = product_case(rows, groups, K, L, kind, DTYPES[tag])
    order, offsets, index = product_plan(index, groups, ordered)
    arguments = [t.to(device) for t in (grad_output, A, W, offsets)] + [None if order is None else order.to(device)]
    grad_A, grad_W = mops_amd.grouped_matrix_product_vjp(*arguments)
    exact = torch.zeros(rows, K, dtype=torch.float64), torch.zeros(groups, K, L, dtype=torch.float64)
    magnitude = torch.zeros_like(exact[0]), torch.zeros_like(exact[1])
    most = 0
    for g in range(groups):
        mask = index == g
        most = max(most, int(mask.sum()))
        a, w, c = A[mask].double(), W[g].double(), grad_output[mask].double()
        exact[0][mask], exact[1][g] = c @ w.t(), a.t() @ c
        magnitude[0][mask], magnitude[1][g] = c.abs() @ w.abs().t(), a.abs().t() @ c.abs()
    assert_within(grad_A, exact[0], magnitude[0], L, "grad_A")
    assert_within(grad_W, exact[1], magnitude[1], most, "grad_W")
    outside = ((index < 0) | (index >= groups)).to(device)
    assert not grad_A[outside].any()
    again = mops_amd.grouped_matrix_product_vjp(*arguments, compute_grad_A=False)
    assert again[0] is None and torch.equal(again[1], grad_W)
    again = mops_amd.grouped_matrix_product_vjp(*arguments, compute_grad_W=False)
    assert again[1] is None and torch.equal(again[0], grad_A)


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,K,L", [(70, 40, 72), (9, 513, 300), (300, 33, 20)])
def test_rows_of_other_groups_do_not_matter(device, rows, K, L, tag):
    """Infinities and NaN in rows and matrices of another group, and in rows of none, stay there."""
    dtype = DTYPES[tag]
    A, W, grad_output, _ = product_case(rows, 3, K, L, "uniform", dtype)
    index = torch.arange(rows, dtype=torch.int32) % 4
    index[index == 3] = -1
    order, offsets = plan_of(index, 3)
    plan = offsets.to(device), order.to(device)
    clean = mops_amd.grouped_matrix_product(A.to(device), W.to(device), *plan)
    clean_A, clean_W = mops_amd.grouped_matrix_product_vjp(grad_output.to(device), A.to(device), W.to(device), *plan)
    for poison in (float("nan"), float("inf"), torch.finfo(dtype).min):
        bad_A, bad_W, bad_grad = A.clone(), W.clone(), grad_output.clone()
        other = (index != 0) & (index != 2)
        bad_A[other], bad_grad[other], bad_W[1] = poison, poison, poison
        bad = [t.to(device) for t in (bad_grad, bad_A, bad_W)]
        good = ((index == 0) | (index == 2)).to(device)
        output = mops_amd.grouped_matrix_product(bad[1], bad[2], *plan)
        grad_A, grad_W = mops_amd.grouped_matrix_product_vjp(*bad, *plan)
        assert torch.equal(output[good], clean[good])
        assert torch.equal(grad_A[good], clean_A[good])
        assert torch.equal(grad_W[[0, 2]], clean_W[[0, 2]])
        nowhere = (index == -1).to(device)
        assert not output[nowhere].any() and not grad_A[nowhere].any()


# -------------------------------------------------------- residual update ----
UPDATES = [
    # rows, columns, gate rows
    (0, 8, 1), (1, 1, 1), (3, 2, 1), (2, 3, 2), (5, 7, 5), (9, 15, 1), (50, 33, 50), (300, 64, 1), (17, 129, 1),
    (1000, 384, 1), (700, 513, 700), (8, 1000, 1), (33, 2049, 33), (6, 4096, 6), (5, 8200, 1), (3, 16384, 3),
    (2, 20001, 2), (3, 16385, 1), (2500, 24, 1), (70000, 5, 1),
]  # fmt: skip
SCALE, EPSILON = 0.3, 1e-5


def update_case(rows, columns, gate_rows, dtype):
    generator = generator_of(rows, columns, gate_rows)
    residual, block = random(generator, (rows, columns), dtype), random(generator, (rows, columns), dtype, 0.5)
    gate = random(generator, (gate_rows, columns), dtype)
    weight_block, weight_next = random(generator, (columns,), dtype), random(generator, (columns,), dtype)
    grads = random(generator, (rows, columns), dtype), random(generator, (rows, columns), dtype)
    return [residual, block, gate, weight_block, weight_next], grads


def update_by_definition(residual, block, gate, weight_block, weight_next):
    def norm(x):
        return x / torch.sqrt((x**2).mean(1, keepdim=True) + EPSILON)

    state = residual + SCALE * gate * norm(block) * weight_block
    return state, norm(state) * weight_next


def update_magnitudes(inputs, grads):
    """For every result the same formula with the absolute values of its terms."""
    residual, block, gate, weight_block, weight_next = (t.double() for t in inputs)
    grad_state, grad_next = (g.double().abs() for g in grads)
    columns = max(residual.shape[1], 1)
    rb = 1 / torch.sqrt((block**2).mean(1, keepdim=True) + EPSILON)
    y = block.abs() * rb
    a = SCALE * gate.abs() * y * weight_block.abs()
    t = residual.abs() + a  # (of the state's two terms)
    exact_state = residual + SCALE * gate * block * rb * weight_block
    rt = 1 / torch.sqrt((exact_state**2).mean(1, keepdim=True) + EPSILON)
    state, following = t, t * rt * weight_next.abs() * (1 + (t * exact_state.abs()).mean(1, keepdim=True) * rt**2)
    h = grad_next * weight_next.abs()
    c = rt**2 * (h * t).mean(1, keepdim=True)
    # (rt itself is known to the relative accuracy of a mean of squares of t)
    widen = 1 + (t * exact_state.abs()).mean(1, keepdim=True) * rt**2
    d = grad_state + rt * (h + t * c) * widen**2
    k = SCALE * d * gate.abs() * weight_block.abs()
    mean_ky = (k * y).sum(1, keepdim=True) / columns
    grad_block = rb * (k + y * mean_ky)
    grad_gate = SCALE * d * y * weight_block.abs()
    if gate.shape[0] == 1 and residual.shape[0] != 1:
        grad_gate = grad_gate.sum(0, keepdim=True)
    sums = (SCALE * d * gate.abs() * y).sum(0), (grad_next * t * rt * widen).sum(0)
    return (state, following), (d, grad_block, grad_gate, *sums)


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,columns,gate_rows", UPDATES)
def test_gated_residual_norm(device, rows, columns, gate_rows, tag):
    inputs, grads = update_case(rows, columns, gate_rows, DTYPES[tag])
    results = mops_amd.gated_residual_norm(*[t.to(device) for t in inputs], SCALE, EPSILON)
    exact = update_by_definition(*[t.double() for t in inputs])
    magnitudes, _ = update_magnitudes(inputs, grads)
    for name, actual, expected, magnitude in zip(("state", "next"), results, exact, magnitudes):
        assert actual.dtype == inputs[0].dtype
        assert_within(actual, expected, magnitude, columns, name)


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,columns,gate_rows", UPDATES)
def test_gated_residual_norm_vjp(device, rows, columns, gate_rows, tag):
    inputs, grads = update_case(rows, columns, gate_rows, DTYPES[tag])
    wide = [t.double().requires_grad_(True) for t in inputs]
    exact = torch.autograd.grad(update_by_definition(*wide), wide, [g.double() for g in grads])
    _, magnitudes = update_magnitudes(inputs, grads)
    on_device = [t.to(device) for t in inputs]
    results = mops_amd.gated_residual_norm_vjp(*[g.to(device) for g in grads], *on_device, SCALE, EPSILON)
    names = ("grad_residual", "grad_block", "grad_gate", "grad_weight_block", "grad_weight_next")
    summed = (0, 0, rows if gate_rows == 1 else 0, rows, rows)
    for name, actual, expected, magnitude, n in zip(names, results, exact, magnitudes, summed):
        # (four norms and means over the columns follow each other)
        assert_within(actual, expected, magnitude, 4 * columns + n, name)
    # a subset of the gradients, and only one cotangent
    for index, name in enumerate(names):
        flags = {"compute_" + other: other == name for other in names}
        one = mops_amd.gated_residual_norm_vjp(
            *[g.to(device) for g in grads], *on_device, SCALE, EPSILON, **flags
        )
        assert [r is None for r in one] == [i != index for i in range(5)]
        assert torch.equal(one[index], results[index])
    zero = torch.zeros_like(grads[0])
    for with_none, with_zero in (((grads[0], None), (grads[0], zero)), ((None, grads[1]), (zero, grads[1]))):
        some = mops_amd.gated_residual_norm_vjp(
            *[None if g is None else g.to(device) for g in with_none], *on_device, SCALE, EPSILON
        )
        same = mops_amd.gated_residual_norm_vjp(*[g.to(device) for g in with_zero], *on_device, SCALE, EPSILON)
        for a, b in zip(some, same):
            assert torch.equal(a, b)


# ------------------------------------------------- offsets beyond 32 bits ----
HUGE_ROWS, HUGE_COLUMNS = 70000, 32768  # 2.3e9 numbers


def huge(device, fill):
    tensor = torch.empty(HUGE_ROWS, HUGE_COLUMNS, dtype=torch.bfloat16, device=device)
    return tensor.fill_(fill)


@pytest.mark.gpu
def test_tables_of_more_than_two_to_the_31_numbers(device):
    table = huge(device, 0)
    rows = torch.tensor([HUGE_ROWS - 1, 3, HUGE_ROWS - 1, -1, 65537], dtype=torch.int32, device=device)
    table[-1], table[3], table[65537] = 2.0, 3.0, 5.0
    output = mops_amd.scaled_embedding(table, rows, 0.5)
    assert [output[i].unique().tolist() for i in range(5)] == [[1.0], [1.5], [1.0], [0.0], [2.5]]
    for repeats in (1, 60):  # (without an order in memory, and with one)
        grad = mops_amd.scaled_embedding_vjp(output.repeat(repeats, 1), table, rows.repeat(repeats), 1.0)
        assert [grad[i].unique().tolist() for i in (-1, 3, 65537, 0)] == [[2.0 * repeats], [1.5 * repeats], [2.5 * repeats], [0.0]]
        assert torch.count_nonzero(grad.sum(1)).item() == 3
        del grad


@pytest.mark.gpu
def test_products_of_more_than_two_to_the_31_numbers(device):
    A = huge(device, 0)
    A[-1], A[65537] = 1.0, 2.0
    offsets = torch.tensor([0, 10, HUGE_ROWS], dtype=torch.int32, device=device)
    for width in (8, 3):  # (rows of W on 16-byte boundaries and off them)
        W = torch.full((2, HUGE_COLUMNS, width), 0.5, dtype=torch.bfloat16, device=device)
        output = mops_amd.grouped_matrix_product(A, W, offsets)
        assert output[-1].unique().tolist() == [HUGE_COLUMNS / 2] and output[65537].unique().tolist() == [HUGE_COLUMNS]
        assert torch.count_nonzero(output).item() == 2 * width
        grad_output = torch.zeros(HUGE_ROWS, width, dtype=torch.bfloat16, device=device)
        grad_output[-1], grad_output[65537] = 4.0, 1.0
        grad_A, grad_W = mops_amd.grouped_matrix_product_vjp(grad_output, A, W, offsets)
        assert grad_A[-1].unique().tolist() == [2.0 * width] and grad_A[65537].unique().tolist() == [0.5 * width]
        assert torch.count_nonzero(grad_A[:65537]).item() == 0
        assert grad_W[1].unique().tolist() == [6.0] and not grad_W[0].any()
        del grad_A


@pytest.mark.gpu
def test_updates_of_more_than_two_to_the_31_numbers(device):
    residual, block, gate = huge(device, 1.0), huge(device, 1.0), huge(device, 2.0)
    weight = torch.ones(HUGE_COLUMNS, dtype=torch.bfloat16, device=device)
    residual[-1], gate[-1] = 0.0, 4.0
    state, following = mops_amd.gated_residual_norm(residual, block, gate, weight, weight, 0.5, 0.0)
    # (norm(1) = 1: state = residual + gate / 2)
    assert state[-1].unique().tolist() == [2.0] and state[-2].unique().tolist() == [2.0]
    assert state[0].unique().tolist() == [2.0] and following[-1].unique().tolist() == [1.0]
    del state, following
    grads = mops_amd.gated_residual_norm_vjp(
        gate, None, residual, block, gate, weight, weight, 0.5, 0.0, compute_grad_block=False, compute_grad_gate=False
    )
    assert grads[0][-1].unique().tolist() == [4.0] and grads[0][65537].unique().tolist() == [2.0]


# ---------------------------------------------------------- differences ----
def central_difference(function, inputs, which, direction, cotangents):
    step = 1e-5
    total = 0.0
    for sign in (1, -1):
        moved = list(inputs)
        moved[which] = inputs[which] + sign * step * direction
        outputs = function(*moved)
        outputs = outputs if isinstance(outputs, tuple) else (outputs,)
        total += sign * sum((c * o).sum().item() for c, o in zip(cotangents, outputs))
    return total / (2 * step)


@pytest.mark.gpu
def test_gradients_against_differences(device):
    """In float64: the error of a central difference is h^2 f'''/6, 1e-10 of values of order one, and its rounding
    1e-16 / h = 1e-11; held to 1e-7 of the sum's scale."""
    generator = generator_of(99)

    def rand(*shape):
        return random(generator, shape, torch.float64).to(device)

    index = indices_of("padded", 40, 6).to(device)
    order, offsets = mops_amd.order_by_group(index, 6)
    cases = [
        (lambda table: mops_amd.scaled_embedding(table, index, 1.3), [rand(6, 11)], [rand(40, 11)],
         lambda g, inputs: [mops_amd.scaled_embedding_vjp(*g, *inputs, index, 1.3)]),
        (lambda A, W: mops_amd.grouped_matrix_product(A, W, offsets, order), [rand(40, 9), rand(6, 9, 13)],
         [rand(40, 13)], lambda g, inputs: mops_amd.grouped_matrix_product_vjp(*g, *inputs, offsets, order)),
        (lambda *t: mops_amd.gated_residual_norm(*t, 0.7, 1e-3), [rand(10, 18), rand(10, 18), rand(1, 18), rand(18), rand(18)],
         [rand(10, 18), rand(10, 18)], lambda g, inputs: mops_amd.gated_residual_norm_vjp(*g, *inputs, 0.7, 1e-3)),
    ]  # fmt: skip
    for function, inputs, cotangents, vjp in cases:
        gradients = vjp(cotangents, inputs)
        for which, gradient in enumerate(gradients):
            direction = rand(*inputs[which].shape)
            expected = central_difference(function, inputs, which, direction, cotangents)
            actual = (gradient * direction).sum().item()
            scale = (gradient * direction).abs().sum().item() + 1.0
            assert abs(actual - expected) <= 1e-7 * scale, (which, actual, expected)


# ------------------------------------------------- layouts, streams, calls ----
def all_calls(device, dtype, rows=200, groups=5, columns=70):
    """name -> (function, arguments) of every function, on ordinary tensors."""
    generator = generator_of(rows, groups, columns, 5)

    def rand(*shape):
        return random(generator, shape, dtype).to(device)

    index = indices_of("padded", rows, groups).to(device)
    order, offsets = mops_amd.order_by_group(index, groups)
    table, values, other = rand(groups, columns), rand(rows, columns), rand(rows, 33)
    W = rand(groups, columns, 33)
    update = [rand(rows, columns), rand(rows, columns), rand(1, columns), rand(columns), rand(columns)]
    return {
        "order_by_group": (mops_amd.order_by_group, [index, groups]),
        "scaled_embedding": (mops_amd.scaled_embedding, [table, index, 0.5]),
        "scaled_embedding_vjp": (mops_amd.scaled_embedding_vjp, [values, table, index, 0.5, order, offsets]),
        "grouped_matrix_product": (mops_amd.grouped_matrix_product, [values, W, offsets, order]),
        "grouped_matrix_product_vjp": (mops_amd.grouped_matrix_product_vjp, [other, values, W, offsets, order]),
        "gated_residual_norm": (mops_amd.gated_residual_norm, [*update, 0.5, 1e-6]),
        "gated_residual_norm_vjp": (
            mops_amd.gated_residual_norm_vjp, [rand(rows, columns), rand(rows, columns), *update, 0.5, 1e-6],
        ),
    }  # fmt: skip


FUNCTIONS = list(layers._SIGNATURES)


def as_tuple(result):
    return result if isinstance(result, tuple) else (result,)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(as_tuple(a), as_tuple(b), strict=True))


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("function", FUNCTIONS)
def test_layouts_and_the_way_through_the_interpreter(device, function, tag, monkeypatch):
    """Views with strides, 64-bit indices, data off every boundary, and the ctypes path: the same bits."""
    from mops_amd import _c_lib

    call, arguments = all_calls(device, DTYPES[tag])[function]
    expected = call(*arguments)

    def strided(x):
        if not isinstance(x, torch.Tensor):
            return x
        return x.long() if x.dtype == torch.int32 else torch.stack([x, x], -1)[..., 0]

    def shifted(x):  # contiguous, one element off the boundaries of wide loads
        if not isinstance(x, torch.Tensor):
            return x
        memory = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
        view = memory[1:].view(x.shape)
        view.copy_(x)
        return view

    assert same(call(*[strided(x) for x in arguments]), expected)
    assert same(call(*[shifted(x) for x in arguments]), expected)
    monkeypatch.setattr(layers, "_native", _c_lib._NoFunctions())
    assert same(call(*arguments), expected)
    assert same(call(*[shifted(x) for x in arguments]), expected)


@pytest.mark.gpu
@pytest.mark.parametrize("function", FUNCTIONS)
def test_another_stream_and_a_graph(device, function):
    """On a stream of the caller's, behind work that is still running there; and captured, replayed with other work
    in between: the same bits every time."""
    call, arguments = all_calls(device, torch.float32)[function]
    expected = as_tuple(call(*arguments))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    late = [torch.zeros_like(x) if isinstance(x, torch.Tensor) else x for x in arguments]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work = torch.randn(2000, 2000, device=device)
        for _ in range(5):
            work = work @ work * 1e-3
        for to, x in zip(late, arguments):
            if isinstance(x, torch.Tensor):
                to.copy_(x)
        assert same(call(*late), expected)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = as_tuple(call(*late))
    for repeat in range(4):
        for to, x in zip(late, arguments):
            if isinstance(x, torch.Tensor) and x.is_floating_point():
                to.copy_(x * (1 + repeat % 2))
        graph.replay()
        torch.cuda.synchronize()
        eager = call(*late)
        assert same(captured, eager)
        torch.cuda.synchronize()


# -------------------------------------------------------------- refusals ----
def test_host_tensors_are_refused():
    index = torch.zeros(3, dtype=torch.int32)
    values = torch.zeros(3, 4)
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.order_by_group(index, 2)
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.scaled_embedding(values, index)
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.scaled_embedding_vjp(values, values, index)
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.grouped_matrix_product(values, torch.zeros(1, 4, 2), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.gated_residual_norm(values, values, values, values[0], values[0])


def test_not_arrays():
    with pytest.raises(TypeError, match="`indices` must be an array in order_by_group"):
        mops_amd.order_by_group([0, 1], 2)
    with pytest.raises(ValueError, match="`table` must be a 2D array in scaled_embedding, got a 1D array"):
        mops_amd.scaled_embedding(torch.zeros(3), torch.zeros(3, dtype=torch.int32))


@pytest.mark.gpu
def test_refusals(device):
    def floats(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device=device)

    def integers(*shape):
        return torch.zeros(shape, dtype=torch.int32, device=device)

    with pytest.raises(TypeError, match="Wrong dtype for indices in scaled_embedding"):
        mops_amd.scaled_embedding(floats(3, 4), floats(5))
    with pytest.raises(TypeError, match="Wrong dtype for table in scaled_embedding"):
        mops_amd.scaled_embedding(integers(3, 4), integers(5))
    with pytest.raises(TypeError, match="`scale` must be a scalar"):
        mops_amd.scaled_embedding(floats(3, 4), integers(5), "2")
    with pytest.raises(ValueError, match="`indices` must be a tensor on cuda:0"):
        mops_amd.scaled_embedding(floats(3, 4), torch.zeros(5, dtype=torch.int32))
    with pytest.raises(ValueError, match="must not be negative"):
        mops_amd.order_by_group(integers(4), -1)
    with pytest.raises(ValueError, match="given together"):
        mops_amd.scaled_embedding_vjp(floats(5, 4), floats(3, 4), integers(5), 1.0, integers(5))
    with pytest.raises(mops_amd.MopsError, match="offsets must have 4 elements"):
        mops_amd.scaled_embedding_vjp(floats(5, 4), floats(3, 4), integers(5), 1.0, integers(5), integers(3))
    with pytest.raises(mops_amd.MopsError, match="sizes of order along dimension 0 and indices along dimension 0"):
        mops_amd.scaled_embedding_vjp(floats(5, 4), floats(3, 4), integers(5), 1.0, integers(4), integers(4))
    with pytest.raises(mops_amd.MopsError, match="sizes of grad_output along dimension 1 and grad_table"):
        mops_amd.scaled_embedding_vjp(floats(5, 3), floats(3, 4), integers(5))
    with pytest.raises(TypeError, match="`table` must have the dtype"):
        mops_amd.scaled_embedding_vjp(floats(5, 4), floats(3, 4, dtype=torch.float64), integers(5))
    with pytest.raises(mops_amd.MopsError, match="sizes of A along dimension 1 and W along dimension 1"):
        mops_amd.grouped_matrix_product(floats(5, 3), floats(2, 4, 6), integers(3))
    with pytest.raises(mops_amd.MopsError, match="offsets must have 3 elements"):
        mops_amd.grouped_matrix_product(floats(5, 4), floats(2, 4, 6), integers(2))
    with pytest.raises(mops_amd.MopsError, match="sizes of order along dimension 0 and A along dimension 0"):
        mops_amd.grouped_matrix_product(floats(5, 4), floats(2, 4, 6), integers(3), integers(4))
    with pytest.raises(TypeError, match="Wrong dtype for W in grouped_matrix_product"):
        mops_amd.grouped_matrix_product(floats(5, 4), floats(2, 4, 6, dtype=torch.bfloat16), integers(3))
    with pytest.raises(mops_amd.MopsError, match="sizes of grad_output along dimension 1 and W along dimension 2"):
        mops_amd.grouped_matrix_product_vjp(floats(5, 5), floats(5, 4), floats(2, 4, 6), integers(3))
    rows, row, one = floats(5, 4), floats(4), floats(1, 4)
    with pytest.raises(mops_amd.MopsError, match="gate must have one row or as many rows as residual"):
        mops_amd.gated_residual_norm(rows, rows, floats(2, 4), row, row)
    with pytest.raises(mops_amd.MopsError, match="sizes of block along dimension 0 and residual along dimension 0"):
        mops_amd.gated_residual_norm(rows, floats(4, 4), one, row, row)
    with pytest.raises(mops_amd.MopsError, match="sizes of weight_next along dimension 0 and residual"):
        mops_amd.gated_residual_norm(rows, rows, one, row, floats(3))
    with pytest.raises(mops_amd.MopsError, match="sizes of grad_next along dimension 0 and residual"):
        mops_amd.gated_residual_norm_vjp(rows, floats(4, 4), rows, rows, one, row, row)
    # (a refused call leaves nothing behind: the next one is right)
    assert mops_amd.scaled_embedding(floats(3, 4) + 1, integers(5), 2.0).eq(2).all()


# ------------------------------------------------------ PyTorch operators ----
def operators():
    import mops_amd.torch  # noqa: F401  (registers the operators)

    return torch.ops.mops


SCHEMAS = {
    "order_by_group": "mops::order_by_group(Tensor indices, int n_groups) -> (Tensor, Tensor)",
    "scaled_embedding": "mops::scaled_embedding(Tensor table, Tensor indices, float scale=1.) -> Tensor",
    "grouped_matrix_product": "mops::grouped_matrix_product(Tensor A, Tensor W, Tensor offsets, Tensor? order=None) -> Tensor",
    "gated_residual_norm": "mops::gated_residual_norm(Tensor residual, Tensor block, Tensor gate, Tensor weight_block, Tensor weight_next, float residual_scale=1., float epsilon=9.9999999999999995e-07) -> (Tensor, Tensor)",
}  # fmt: skip


@pytest.mark.parametrize("name", list(SCHEMAS))
def test_operator_schemas(name):
    assert str(getattr(operators(), name).default._schema) == SCHEMAS[name]


def test_operators_refuse_host_tensors():
    index, values = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="device path only"):
        operators().order_by_group(index, 2)
    with pytest.raises(RuntimeError, match="device path only"):
        operators().scaled_embedding(values, index, 1.0)
    with pytest.raises(RuntimeError, match="device path only"):
        operators().grouped_matrix_product(values, torch.zeros(1, 4, 2), index[:2])
    with pytest.raises(RuntimeError, match="device path only"):
        operators().gated_residual_norm(values, values, values, values[0], values[0])


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
def test_operators_with_autograd(device, tag):
    """Values and gradients of the operators: what the functions of the package give, bit for bit."""
    ops, dtype = operators(), DTYPES[tag]
    generator = generator_of(21)

    def rand(*shape):
        return random(generator, shape, dtype).to(device)

    index = indices_of("padded", 50, 4).to(device)
    order, offsets = ops.order_by_group(index.long(), 4)
    assert same((order, offsets), mops_amd.order_by_group(index, 4))
    table, A, W, gate = rand(4, 24), rand(50, 24), rand(4, 24, 10), rand(1, 24)
    rows, weights = [rand(50, 24), rand(50, 24)], [rand(24), rand(24)]
    grad, grads = rand(50, 10), [rand(50, 24), rand(50, 24)]

    leaf = table.clone().requires_grad_(True)
    output = ops.scaled_embedding(leaf, index, 0.7)
    output.backward(grads[0])
    assert same(output.detach(), mops_amd.scaled_embedding(table, index, 0.7))
    assert same(leaf.grad, mops_amd.scaled_embedding_vjp(grads[0], table, index, 0.7))

    leaves = [A.clone().requires_grad_(True), W.clone().requires_grad_(True)]
    output = ops.grouped_matrix_product(*leaves, offsets, order)
    output.backward(grad)
    assert same(output.detach(), mops_amd.grouped_matrix_product(A, W, offsets, order))
    expected = mops_amd.grouped_matrix_product_vjp(grad, A, W, offsets, order)
    assert same(tuple(t.grad for t in leaves), expected)
    # rows that lie in the order of their group already
    in_order = mops_amd.grouped_matrix_product(A, W, offsets)
    assert same(ops.grouped_matrix_product(A, W, offsets), in_order)

    inputs = [*rows, gate, *weights]
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    state, following = ops.gated_residual_norm(*leaves, 0.4, 1e-5)
    assert same((state.detach(), following.detach()), mops_amd.gated_residual_norm(*inputs, 0.4, 1e-5))
    torch.autograd.backward([state, following], grads)
    assert same(tuple(t.grad for t in leaves), mops_amd.gated_residual_norm_vjp(*grads, *inputs, 0.4, 1e-5))
    # only one result used, only some inputs recorded
    block = rows[1].clone().requires_grad_(True)
    ops.gated_residual_norm(rows[0], block, gate, *weights, 0.4, 1e-5)[1].backward(grads[1])
    assert same(block.grad, mops_amd.gated_residual_norm_vjp(None, grads[1], *inputs, 0.4, 1e-5)[1])


@pytest.mark.gpu
def test_operators_registered_from_python():
    """The same tests with the operators of mops_amd/_torch_python_ops.py, in a process of their own."""
    import os
    import subprocess
    import sys

    if os.environ.get("MOPS_AMD_TORCH_PYTHON_OPS", "0") not in ("", "0"):
        pytest.skip("this process already runs them")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run(
        [sys.executable, "-m", "pytest", os.path.join(root, "tests", "test_layers.py"), "-q", "-x", "-k", "operator",
         "-p", "no:cacheprovider"],
        cwd=root, env=dict(os.environ, MOPS_AMD_TORCH_PYTHON_OPS="1"), capture_output=True, text=True,
    )  # fmt: skip
    assert done.returncode == 0, done.stdout[-3000:] + done.stderr[-2000:]
    assert " passed" in done.stdout


# ---------------------------------------------------------------- example ----
class PlainOperators:
    """The operators of the example in elementary torch operations."""

    @staticmethod
    def order_by_group(indices, n_groups):
        order, offsets = plan_of(indices.cpu(), n_groups)
        return order.to(indices.device), offsets.to(indices.device)

    @staticmethod
    def scaled_embedding(table, indices, scale):
        inside = indices >= 0
        return torch.where(inside[:, None], table[torch.where(inside, indices, 0).long()] * scale, 0.0)

    @staticmethod
    def outer_product_scatter_add_with_weights(A, B, W, indices_W, indices_output):
        terms = A[:, :, None] * (B * W[indices_W.long()])[:, None, :]
        zeros = torch.zeros(W.shape[0], A.shape[1], B.shape[1], dtype=A.dtype, device=A.device)
        return zeros.index_add(0, indices_output.long(), terms)

    @staticmethod
    def grouped_matrix_product(A, W, offsets, order):
        output = torch.zeros(A.shape[0], W.shape[2], dtype=A.dtype, device=A.device)
        for g in range(W.shape[0]):
            rows = order[int(offsets[g]) : int(offsets[g + 1])].long()
            output = output.index_add(0, rows, A[rows] @ W[g])
        return output

    @staticmethod
    def gated_residual_norm(residual, block, gate, weight_block, weight_next, scale, epsilon):
        def norm(x):
            return x / torch.sqrt((x**2).mean(1, keepdim=True) + epsilon)

        state = residual + scale * gate * norm(block) * weight_block
        return state, norm(state) * weight_next


@pytest.mark.gpu
def test_example_network(device):
    """The operators together, with the sums over edges: energy and all gradients in float64 against elementary torch
    operations (rounding errors of some 1e4 terms, 1e-16 each, grow through the layers; held to 1e-10 of each gradient's
    largest value), and a loss that falls."""
    import importlib.util
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("element_network", os.path.join(root, "examples", "element_network.py"))
    network = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(network)
    s = network.structure(device, torch.float64)
    results = []
    for ops in (torch.ops.mops, PlainOperators):
        p = network.parameters(device, torch.float64)
        value = network.energy(p, s, ops)
        value.backward()
        results.append((value.detach(), {name: t.grad for name, t in p.items()}))
    assert abs(results[0][0] - results[1][0]) <= 1e-10 * abs(results[1][0])
    for name, gradient in results[0][1].items():
        expected = results[1][1][name]
        assert (gradient - expected).abs().max() <= 1e-10 * expected.abs().max(), name
    losses = network.train(steps=15, device=device)
    assert losses[-1] < 0.2 * losses[0]
