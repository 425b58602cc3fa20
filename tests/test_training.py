"""The operators of networks of layers (mops_amd.training) against their definitions in 64 bits.

Tolerances, with p the bits sums are held in (24, 53 for float64) and q those of the type (8, 11, 24, 53): every result is
held to its rounding, 2^-q of itself, and to what the errors of the sums in front of it can make of it, first order,
written down at each operator. A sum of n terms is off by at most (n + 16) 2^-p times the sum of the terms' magnitudes,
16 for the few operations on each term and for functions that are a few units off (the activations, exp, log).
"""
import ctypes
import math

import pytest
import torch

import mops_amd
from mops_amd import training
from tests.test_layers import (
    BITS,
    DTYPES,
    PRODUCTS,
    WIDE_BITS,
    central_difference,
    generator_of,
    indices_of,
    plan_of,
    product_case,
    product_plan,
    random,
    same,
)
from tests.test_layers_bounds import run_on_host

ACTIVATIONS = ["silu", "gelu", "sigmoid"]


def held_to(actual, exact, bound, what):
    dtype = actual.dtype
    assert actual.shape == exact.shape, what
    if actual.numel() == 0:
        return
    actual, exact, bound = actual.double().cpu(), exact.cpu(), bound.cpu()
    bound = bound + 2.0 ** -BITS[dtype] * exact.abs() + torch.finfo(dtype).tiny
    assert torch.isfinite(actual).all(), what
    worst = ((actual - exact).abs() / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound"


def unit(dtype):
    return 2.0 ** -WIDE_BITS[dtype]


# -------------------------------------------------- gated products by group ----
def activated(name, x):
    """act(x), act'(x) and what bounds |act(x)| for all arguments of that magnitude."""
    if name == "gelu":
        below = torch.special.erfc(x * -math.sqrt(0.5)) / 2  # (torch.special.ndtr is 0 from -8.3 down)
        return x * below, below + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi), x.abs()
    s = torch.sigmoid(x)
    if name == "sigmoid":
        return s, s * (1 - s), torch.ones_like(x)
    return x * s, s * (1 + x * (1 - s)), x.abs()


def gated_by_definition(A, W, index, activation, grad_output, dtype):
    """Per result, exact and bound. With g, u the projections, G, U the sums of their terms' magnitudes, M the bound of
    |act|, |act'| <= 1.2, |act''| <= 0.9 and e = (K + 32) 2^-p: output: e (1.2 G U + M U). The projections' gradients s
    = (c u act', c act) are off by e |c| (1.2 U + 0.9 G U), e |c| (1.2 G + M), and, rounded to the type, by 2^-q |s|; the
    products of s add (n + 16) 2^-p of their terms' magnitudes."""
    rows, groups, K, L = A.shape[0], W.shape[0], A.shape[1], W.shape[2] // 2
    p, q = unit(dtype), 2.0 ** -BITS[dtype]
    e = (K + 32) * p
    output, output_bound = torch.zeros(rows, L, dtype=torch.float64), torch.zeros(rows, L, dtype=torch.float64)
    grad_A, grad_W = torch.zeros(rows, K, dtype=torch.float64), torch.zeros(groups, K, 2 * L, dtype=torch.float64)
    bound_A, bound_W = torch.zeros_like(grad_A), torch.zeros_like(grad_W)
    for k in range(groups):
        mask = index == k
        a, w, c = A[mask].double(), W[k].double(), grad_output[mask].double()
        both, most = a @ w, a.abs() @ w.abs()
        g, u, G, U = both[:, :L], both[:, L:], most[:, :L], most[:, L:]
        value, slope, _ = activated(activation, g)
        M = activated(activation, G)[2]
        output[mask], output_bound[mask] = value * u, e * (1.2 * G * U + M * U)
        s = torch.cat([c * u * slope, c * value], 1)
        off = e * torch.cat([c.abs() * (1.2 * U + 0.9 * G * U), c.abs() * (1.2 * G + M)], 1) + q * s.abs()
        off = off + torch.finfo(dtype).tiny * q
        grad_A[mask], grad_W[k] = s @ w.t(), a.t() @ s
        bound_A[mask] = off @ w.abs().t() + (2 * L + 16) * p * (s.abs() @ w.abs().t())
        bound_W[k] = a.abs().t() @ off + (len(a) + 16) * p * (a.abs().t() @ s.abs())
    return (output, output_bound), (grad_A, bound_A), (grad_W, bound_W)


# every extent of tiles on 16-byte boundaries and off them, shares of k in both directions, operands that are copied
LARGE_GATED = [
    (8300, 3, 72, 1032, "padded", True), (5000, 20, 520, 264, "frequent", True), (4100, 2, 264, 1031, "frequent", True),
    (9000, 2, 50, 299, "uniform", True), (40, 3, 2000, 24, "uniform", True), (30, 2, 1501, 33, "padded", True),
    (2100, 1, 513, 1027, "uniform", False), (6, 2, 3000, 1, "uniform", True), (6, 2, 3000, 16, "uniform", True),
    (30, 2, 1504, 40, "padded", True), (20, 16, 264, 1032, "uniform", True), (7, 0, 16, 8, "nowhere", True),
    (70, 3, 24, 0, "padded", True), (50, 2, 0, 40, "uniform", False),
]  # fmt: skip


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,groups,K,L,kind,ordered", PRODUCTS + LARGE_GATED)
def test_gated_grouped_product(device, rows, groups, K, L, kind, ordered, tag):
    dtype = DTYPES[tag]
    A, W, _, index = product_case(rows, groups, K, 2 * L, kind, dtype)
    grad_output = random(generator_of(rows, L, 17), (rows, L), dtype)
    order, offsets, index = product_plan(index, groups, ordered)
    activation = ACTIVATIONS[(rows + K + L) % 3]
    plan = [offsets.to(device), None if order is None else order.to(device)]
    on_device = [A.to(device), W.to(device), *plan, activation]
    results = gated_by_definition(A, W, index, activation, grad_output, dtype)
    output = mops_amd.gated_grouped_product(*on_device)
    assert output.dtype == dtype
    held_to(output, *results[0], "output")
    grads = mops_amd.gated_grouped_product_vjp(grad_output.to(device), *on_device)
    held_to(grads[0], *results[1], "grad_A")
    held_to(grads[1], *results[2], "grad_W")
    outside = ((index < 0) | (index >= groups)).to(device)
    assert not output[outside].any() and not grads[0][outside].any()
    again = mops_amd.gated_grouped_product_vjp(grad_output.to(device), *on_device, compute_grad_A=False)
    assert again[0] is None and torch.equal(again[1], grads[1])
    again = mops_amd.gated_grouped_product_vjp(grad_output.to(device), *on_device, compute_grad_W=False)
    assert again[1] is None and torch.equal(again[0], grads[0])


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_activations_far_from_zero(device, activation, tag):
    """One number per projection, so that gate and up are what is asked for: the values of the activation where its
    exponential overflows and underflows, and its derivative, to 2^-16 (float64: 2^-40) of themselves (the arguments'
    share, |x| 2^-p times the logarithmic derivative, which is |x| at most, included: 80^2 2^-24 = 2^-11.4 for float32 and
    its likes) and the rounding."""
    dtype = DTYPES[tag]
    x = torch.tensor([-80.0, -30.0, -10.0, -5.5, -3.0, -1.0, -0.25, 0.0, 0.25, 1.0, 3.0, 10.0, 80.0], dtype=dtype)
    A = x[:, None]
    W = torch.ones(1, 1, 2, dtype=dtype)
    W[0, 0, 1] = 0
    ones, offsets = torch.ones(len(x), 1, dtype=dtype), torch.tensor([0, len(x)], dtype=torch.int32)
    value, slope, _ = activated(activation, x.double())
    if activation == "silu":
        value, slope = x.double() * torch.sigmoid(x.double()), torch.sigmoid(x.double()) * (
            1 + x.double() * torch.sigmoid(-x.double())
        )
    if activation == "sigmoid":
        slope = torch.sigmoid(x.double()) * torch.sigmoid(-x.double())
    on_device = [A.to(device), W.to(device), offsets.to(device), None, activation]
    # up = 0: output 0, and s = (0, c act): grad_A = 0 . 1 + act . 0; grad_W holds sums, so the rows go one by one
    off = 2.0**-11 if dtype != torch.float64 else 2.0**-35
    for i in range(len(x)):
        one = [A[i : i + 1].to(device), W.to(device), torch.tensor([0, 1], dtype=torch.int32, device=device), None, activation]
        grad_A, grad_W = mops_amd.gated_grouped_product_vjp(ones[:1].to(device), *one)
        expected = x[i].double() * value[i]  # of W_up: A act
        held_to(grad_W[0, 0, 1], expected, (off + 2.0 ** -BITS[dtype]) * expected.abs(), f"act({x[i]})")
    W[0, 0, 1] = 1
    output = mops_amd.gated_grouped_product(A.to(device), torch.tensor([[[1.0, 0.0]]], dtype=dtype, device=device), *on_device[2:])
    assert not output.any()
    # W_up = 1: up = x, and grad_A = c (x act' + act)
    for i in range(len(x)):
        one = [A[i : i + 1].to(device), W.to(device), torch.tensor([0, 1], dtype=torch.int32, device=device), None, activation]
        grad_A, _ = mops_amd.gated_grouped_product_vjp(ones[:1].to(device), *one)
        terms = x[i].double() * slope[i], value[i]
        bound = (off + 2.0 ** -BITS[dtype]) * (terms[0].abs() + terms[1].abs())
        # (silu and gelu: the derivative is a difference of two numbers, each off by `off` of itself)
        if activation != "sigmoid":
            below = torch.sigmoid(x[i].double()) if activation == "silu" else torch.special.erfc(x[i].double() * -math.sqrt(0.5)) / 2
            bound = bound + off * (2 * below * x[i].abs())
        held_to(grad_A[0, 0], terms[0] + terms[1], bound, f"derivative at {x[i]}")


def activated_far_from_zero(name, x):
    """act(x), act'(x), the magnitudes of the latter's terms and how many units (16 + 2 |x| or 2 x^2) each is held to: the normal
    distribution's integral from an argument in more than 64 bits."""
    import numpy as np

    if name == "gelu":
        exact = np.asarray(x, dtype=np.longdouble) * -np.sqrt(np.longdouble(0.5))
        z = torch.from_numpy(exact.astype(np.float64))
        rest = torch.from_numpy((exact - exact.astype(np.float64)).astype(np.float64))
        below = torch.special.erfc(z) / 2 - torch.exp(-z * z) * rest / math.sqrt(math.pi)
        density = torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
        return x * below, below + x * density, below + x.abs() * density, 16 + 2 * x * x
    s, rest = torch.sigmoid(x), torch.sigmoid(-x)
    if name == "sigmoid":
        return s, s * rest, s * rest, 16 + 2 * x.abs()
    return x * s, s + x * s * rest, s + x.abs() * s * rest, 16 + 2 * x.abs()


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_activations_point_by_point(device, activation, tag):
    """The activation and its derivative at arguments that are exact (one product and a one each), every point to the share that
    the rounding of its own exponent has: (16 + 2 |x|) 2^-p, for GELU (16 + 2 x^2) 2^-p, of the terms, and the result's rounding.
    (Powers below the smallest number of 32 bits are zero.) float64: the oracle's own exponentials are off as much again."""
    dtype = DTYPES[tag]
    x = torch.cat([torch.linspace(-13, 13, 209), torch.tensor([-0.75179, -1.2784, -1e-3, 1e-3, -5.5, 1e-6])])
    if activation != "gelu":
        x = torch.cat([x, torch.linspace(-87, 87, 117), torch.tensor([-88.5, 88.5])])
    x = x.to(dtype)
    n = len(x)
    A = torch.stack([x, torch.ones_like(x)], 1)
    W = torch.eye(2, dtype=dtype).repeat(n, 1, 1)  # gate = x, up = 1, a group for every row
    offsets = torch.arange(n + 1, dtype=torch.int32)
    arguments = [A.to(device), W.to(device), offsets.to(device), None, activation]
    x = x.double()
    value, slope, terms, units = activated_far_from_zero(activation, x)
    share = units * unit(dtype) * (2 if dtype == torch.float64 else 1)
    smallest = torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).tiny * (x.abs() + 1)
    held_to(mops_amd.gated_grouped_product(*arguments)[:, 0], value, share * value.abs() + smallest, "value")
    _, grad_W = mops_amd.gated_grouped_product_vjp(torch.ones(n, 1, dtype=dtype, device=device), *arguments)
    # (of 16-bit types the projections' gradients are rounded, and a sum of one of them is not rounded again)
    held_to(grad_W[:, 1, 0], slope, share * terms + smallest, "slope")
    held_to(grad_W[:, 1, 1], value, share * value.abs() + smallest, "value in the gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,K,L", [(70, 40, 72), (9, 1600, 30), (300, 33, 20), (3000, 64, 520)])
def test_gated_rows_of_other_groups_do_not_matter(device, rows, K, L, tag):
    """Infinities and NaN in rows and matrices of another group, and in rows of none, stay there."""
    dtype = DTYPES[tag]
    A, W, _, _ = product_case(rows, 3, K, 2 * L, "uniform", dtype)
    grad_output = random(generator_of(rows, 3), (rows, L), dtype)
    index = torch.arange(rows, dtype=torch.int32) % 4
    index[index == 3] = -1
    order, offsets = plan_of(index, 3)
    plan = offsets.to(device), order.to(device)
    clean = mops_amd.gated_grouped_product(A.to(device), W.to(device), *plan)
    clean_A, clean_W = mops_amd.gated_grouped_product_vjp(grad_output.to(device), A.to(device), W.to(device), *plan)
    for poison in (float("nan"), float("inf"), torch.finfo(dtype).min):
        bad_A, bad_W, bad_grad = A.clone(), W.clone(), grad_output.clone()
        other = (index != 0) & (index != 2)
        bad_A[other], bad_grad[other], bad_W[1] = poison, poison, poison
        bad = [t.to(device) for t in (bad_grad, bad_A, bad_W)]
        good = ((index == 0) | (index == 2)).to(device)
        output = mops_amd.gated_grouped_product(bad[1], bad[2], *plan)
        grad_A, grad_W = mops_amd.gated_grouped_product_vjp(*bad, *plan)
        assert torch.equal(output[good], clean[good])
        assert torch.equal(grad_A[good], clean_A[good])
        assert torch.equal(grad_W[[0, 2]], clean_W[[0, 2]])
        nowhere = (index == -1).to(device)
        assert not output[nowhere].any() and not grad_A[nowhere].any()


# ----------------------------------------------------------- cross entropy ----
LOSSES = [
    # rows, classes, K, targets
    (0, 5, 8, "uniform"), (1, 1, 1, "uniform"), (3, 2, 7, "padded"), (64, 500, 64, "uniform"), (65, 63, 65, "frequent"),
    (300, 94, 128, "padded"), (40, 3001, 40, "uniform"), (130, 257, 33, "nowhere"), (700, 1000, 24, "one"),
    (33, 90, 1500, "uniform"), (5, 7, 2001, "padded"), (20, 4000, 9, "uniform"), (2000, 40, 72, "padded"),
    (1025, 1030, 64, "frequent"), (513, 2056, 136, "padded"), (17000, 12, 16, "padded"), (4, 0, 6, "nowhere"),
    (90, 31, 0, "uniform"), (2100, 4100, 1033, "uniform"), (64, 33000, 72, "padded"), (40, 33001, 64, "uniform"),
    (20, 40000, 16, "frequent"),
]  # fmt: skip


def loss_case(rows, classes, K, kind, dtype, spread=3.0):
    generator = generator_of(rows, classes, K)
    A = random(generator, (rows, K), dtype)
    W = random(generator, (classes, K), dtype, spread * max(K, 1) ** -0.5)
    targets = indices_of(kind, rows, classes) if classes > 0 else torch.full((rows,), -1, dtype=torch.int32)
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    grads = [random(generator, (rows,), wide, 1 / max(rows, 1)) for _ in range(2)]
    return A, W, targets, grads


def loss_by_definition(A, W, targets, grads, dtype, of_rounding=None):
    """Per result, exact and bound. The logits x are off by E = (K + 32) 2^-p X, X the sum of their terms' magnitudes.
    A power exp(x - m) is off by its argument's error and 2^-p (|x| + |m| + 8) of itself, so the sums' logarithm s by
    S = max(E) + 2^-p (2 max|x| + V + 64 + 4 |s|), a loss by S + E[target] + 4 2^-p (|s| + |loss|). d = a exp(x - s) - g 1
    is off by |a| exp(x - s) (E + S + 2^-p (|x| + |s| + 8)) + 4 2^-p (|a| p + g 1) and, rounded to the type, by 2^-q |d|
    (float16: by its smallest number's half, at the scale at which the largest weight is 2^13 at least: 2^-38 of that); the
    products of d add (n + 16) 2^-p of their terms' magnitudes. `of_rounding`: another part of d than 2^-q."""
    p, q = unit(dtype), 2.0 ** -BITS[dtype] if of_rounding is None else of_rounding
    A, W, (g, h) = A.double(), W.double(), [x.double() for x in grads]
    rows, K, V = A.shape[0], A.shape[1], W.shape[0]
    kept = (targets >= 0) & (targets < V)
    g, h = torch.where(kept, g, 0)[:, None], torch.where(kept, h, 0)[:, None]
    at = torch.where(kept, targets.long(), 0)[:, None]
    if V == 0 or rows == 0:
        none = torch.zeros(rows, dtype=torch.float64, device=A.device)
        zeros = torch.zeros_like(A), torch.zeros_like(W)
        return (none, none), (none, none), (zeros[0], zeros[0]), (zeros[1], zeros[1])
    x, E = A @ W.t().contiguous(), (K + 32) * p * (A.abs() @ W.abs().t().contiguous())
    s = torch.logsumexp(x, 1, keepdim=True)
    S = E.max(1, keepdim=True).values + p * (2 * x.abs().max(1, keepdim=True).values + V + 64 + 4 * s.abs())
    loss = s - x.gather(1, at)
    loss_bound = S + E.gather(1, at) + 4 * p * (s.abs() + loss.abs())
    one = torch.zeros_like(x).scatter_(1, at, 1.0) * g
    power = torch.exp(x - s)
    d = (g + h) * power - one
    off = (g + h).abs() * power * (E + S + p * (x.abs() + s.abs() + 8)) + 4 * p * ((g + h).abs() * power + one.abs())
    off = off + q * d.abs()
    if dtype == torch.float16:
        off = off + 2.0**-38 * torch.maximum(g.abs(), (g + h).abs()).max()
    off = torch.where(kept[:, None], off, 0)
    grad_A, grad_W = d @ W, d.t().contiguous() @ A
    bound_A = off @ W.abs() + (V + 16) * p * (d.abs() @ W.abs())
    bound_W = off.t().contiguous() @ A.abs() + (rows + 16) * p * (d.abs().t().contiguous() @ A.abs())
    clear = lambda t: torch.where(kept, t.squeeze(1), 0)  # noqa: E731
    return (clear(loss), clear(loss_bound)), (clear(s), clear(S)), (grad_A, bound_A), (grad_W, bound_W)


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,classes,K,kind", LOSSES)
def test_linear_cross_entropy(device, rows, classes, K, kind, tag):
    dtype = DTYPES[tag]
    A, W, targets, grads = loss_case(rows, classes, K, kind, dtype)
    results = loss_by_definition(A, W, targets, grads, dtype)
    A, W, targets = A.to(device), W.to(device), targets.to(device)
    grads = [g.to(device) for g in grads]
    losses, log_sums = mops_amd.linear_cross_entropy(A, W, targets)
    assert losses.dtype == log_sums.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
    held_to(losses, *results[0], "losses")
    held_to(log_sums, *results[1], "log_sums")
    grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(*grads, A, W, targets, log_sums)
    held_to(grad_A, *results[2], "grad_A")
    held_to(grad_W, *results[3], "grad_W")
    outside = (targets < 0) | (targets >= classes)
    assert not losses[outside].any() and not log_sums[outside].any() and not grad_A[outside].any()
    again = mops_amd.linear_cross_entropy_vjp(*grads, A, W, targets, log_sums, compute_grad_A=False)
    assert again[0] is None and torch.equal(again[1], grad_W)
    again = mops_amd.linear_cross_entropy_vjp(*grads, A, W, targets, log_sums, compute_grad_W=False)
    assert again[1] is None and torch.equal(again[0], grad_A)
    # either cotangent alone
    zero = torch.zeros_like(grads[0])
    for one, other in (((grads[0], None), (grads[0], zero)), ((None, grads[1]), (zero, grads[1]))):
        assert same(
            mops_amd.linear_cross_entropy_vjp(*one, A, W, targets, log_sums),
            mops_amd.linear_cross_entropy_vjp(*other, A, W, targets, log_sums),
        )


HALVES = ["bf16", "f16"]


@pytest.mark.gpu
@pytest.mark.parametrize("tag", HALVES)
@pytest.mark.parametrize(
    "rows,classes,K,kind",
    [
        (1, 3, 8, "uniform"), (3, 4001, 127, "uniform"), (2, 33001, 64, "uniform"), (9, 95, 200, "padded"),
        (64, 500, 64, "frequent"), (65, 130, 1030, "padded"), (200, 94, 128, "one"), (255, 700, 33, "padded"),
        (256, 1500, 72, "uniform"), (40, 70, 2, "nowhere"), (7, 5, 2001, "padded"),
    ],
)  # fmt: skip
def test_gradients_of_few_rows_are_rounded_once(device, rows, classes, K, kind, tag):
    """d is held in two parts: what the second one's rounding leaves is 2^-q of 2^-q of d (and of a part that is infinite or
    not a number nothing)."""
    dtype = DTYPES[tag]
    A, W, targets, grads = loss_case(rows, classes, K, kind, dtype)
    results = loss_by_definition(A, W, targets, grads, dtype, 2.0 ** (-2 * BITS[dtype]))
    A, W, targets, grads = A.to(device), W.to(device), targets.to(device), [g.to(device) for g in grads]
    _, log_sums = mops_amd.linear_cross_entropy(A, W, targets)
    grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(*grads, A, W, targets, log_sums)
    held_to(grad_A, *results[2], "grad_A")
    held_to(grad_W, *results[3], "grad_W")
    # what rows without a target hold reaches nothing, and an infinite weight everything
    outside = (targets < 0) | (targets >= classes)
    B = A.clone()
    B[outside] = float("nan")
    assert same(mops_amd.linear_cross_entropy_vjp(*grads, B, W, targets, log_sums), (grad_A, grad_W))
    grads[0][0] = float("inf")
    of_infinite = mops_amd.linear_cross_entropy_vjp(*grads, A, W, targets, log_sums)
    assert outside[0] or (not of_infinite[0][0].isfinite().any() and not of_infinite[1].isfinite().any())
    assert torch.equal(of_infinite[0][1:], grad_A[1:]) or tag == "f16"


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,classes,K", [(9, 95, 200), (64, 500, 64), (256, 700, 33), (600, 300, 40), (3000, 94, 128)])
def test_rows_beside_one_of_infinite_weight(device, rows, classes, K, tag):
    """grad_A of all rows but the one whose weight is infinite (or not a number): what it is without that one, to its own bound."""
    dtype = DTYPES[tag]
    A, W, targets, grads = loss_case(rows, classes, K, "padded", dtype)
    on_device = [t.to(device) for t in (A, W, targets)]
    log_sums = mops_amd.linear_cross_entropy(*on_device)[1]
    kept = ((targets >= 0) & (targets < classes)).nonzero().squeeze(1)
    for row in (kept[0].item(), kept[len(kept) // 2].item()):
        without = [g.clone() for g in grads]
        for g in without:
            g[row] = 0
        exact, bound = loss_by_definition(A, W, targets, without, dtype)[2]
        others = torch.arange(rows) != row
        for poison, which in ((math.inf, 0), (-math.inf, 1), (math.nan, 0)):
            bad = [g.clone() for g in grads]
            bad[which][row] = poison
            grad_A, _ = mops_amd.linear_cross_entropy_vjp(*[g.to(device) for g in bad], *on_device, log_sums)
            held_to(grad_A[others.to(device)], exact[others], bound[others], f"beside {poison}")
            assert not grad_A[row].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [100, 600, 2000])
@pytest.mark.parametrize("weight", [1 + 2.0**-8, 1 + 2.0**-11, 1.5 + 2.0**-8 + 2.0**-10])
@pytest.mark.parametrize("tag", HALVES)
def test_gradients_of_a_mean_are_not_off_by_its_weight(device, tag, weight, rows):
    """Rows with one weight g each, of a number that the type rounds, and logits that are zero: the powers are 2^-12 each, d is
    g 2^-12 (of the type, but for g) and g (2^-12 - 1) at the target, which is off by g 2^-12 at most where g is not rounded
    itself (2^-8 g and 2^-11 g). Products add (n + 16) 2^-24 of their terms' magnitudes, powers 64 2^-24."""
    dtype, classes, K = DTYPES[tag], 4096, 16
    generator = generator_of(rows)
    A, W = random(generator, (rows, K), dtype), random(generator, (classes, K), dtype)
    A[:, K // 2 :], W[:, : K // 2] = 0, 0
    targets = indices_of("uniform", rows, classes)
    g = weight / 1024
    d = torch.full((rows, classes), g / classes, dtype=torch.float64)
    at = torch.arange(rows), targets.long()
    d[at] -= g
    off = 80 * 2.0**-24 * d.abs()
    off[at] += g * 2.0**-12
    a, w = A.double(), W.double()
    bound_A = off @ w.abs() + (classes + 16) * 2.0**-24 * (d.abs() @ w.abs())
    bound_W = off.t() @ a.abs() + (rows + 16) * 2.0**-24 * (d.abs().t() @ a.abs())
    A, W, targets = A.to(device), W.to(device), targets.to(device)
    _, log_sums = mops_amd.linear_cross_entropy(A, W, targets)
    grads = torch.full((rows,), g, device=device)
    grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(grads, None, A, W, targets, log_sums)
    held_to(grad_A, d @ w, bound_A, "grad_A")
    held_to(grad_W, d.t() @ a, bound_W, "grad_W")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [100, 600, 2000])
@pytest.mark.parametrize("weight", [1 + 2.0**-8, 1 + 2.0**-11, 1.5 + 2.0**-8 + 2.0**-10])
@pytest.mark.parametrize("tag", HALVES)
def test_gradients_of_log_sums_are_not_off_by_their_weight(device, tag, weight, rows):
    """Likewise for rows whose log_sums have one weight h, with a class each that is certain: logits of 32 and 0, the power of the
    one is 1 - 8e-13 and those of the 63 others 1.3e-14, d is h and h 1.3e-14, off by 80 2^-24 of itself (what h d is held in is
    not rounded: 1; the others are below 2^-38 of the largest in float16)."""
    dtype, classes, extra = DTYPES[tag], 64, 16
    generator = generator_of(rows, 3)
    certain = indices_of("uniform", rows, classes).long()
    A, W = torch.zeros(rows, classes + extra, dtype=dtype), torch.zeros(classes, classes + extra, dtype=dtype)
    A[torch.arange(rows), certain] = 32
    A[:, classes:] = random(generator, (rows, extra), dtype)
    W[torch.arange(classes), torch.arange(classes)] = 1
    h = weight / 1024
    x = A.double() @ W.double().t()
    d = h * torch.softmax(x, 1)
    off = 80 * 2.0**-24 * d + 2.0**-38 * h
    a, w = A.double(), W.double()
    bound_A = off @ w.abs() + (classes + 16) * 2.0**-24 * (d @ w.abs())
    bound_W = off.t() @ a.abs() + (rows + 16) * 2.0**-24 * (d.t() @ a.abs())
    A, W, targets = A.to(device), W.to(device), indices_of("frequent", rows, classes).to(device)
    _, log_sums = mops_amd.linear_cross_entropy(A, W, targets)
    grads = torch.full((rows,), h, device=device)
    grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(None, grads, A, W, targets, log_sums)
    held_to(grad_A, d @ w, bound_A, "grad_A")
    held_to(grad_W, d.t() @ a, bound_W, "grad_W")
    without = mops_amd.linear_cross_entropy_vjp(0 * grads, grads, A, W, targets, log_sums)
    assert same((grad_A, grad_W), without)


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
def test_cross_entropy_in_pieces_of_the_classes(device, tag):
    """More gradients of logits than are held at a time: grad_A is added up over several pieces. (The definition in 64 bits
    on the device, as there are many of them.)"""
    dtype = DTYPES[tag]
    rows, classes, K = {2: (4100, 70001, 40), 4: (4100, 36001, 40), 8: (1030, 70001, 20)}[torch.finfo(dtype).bits // 8]
    A, W, targets, grads = loss_case(rows, classes, K, "padded", dtype)
    on_device = [t.to(device) for t in (A, W, targets)]
    grads = [g.to(device) for g in grads]
    results = loss_by_definition(*on_device, grads, dtype)
    losses, log_sums = mops_amd.linear_cross_entropy(*on_device)
    held_to(losses, *results[0], "losses")
    grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(*grads, *on_device, log_sums)
    held_to(grad_A, *results[2], "grad_A")
    held_to(grad_W, *results[3], "grad_W")
    assert not grad_A[(on_device[2] < 0) | (on_device[2] >= classes)].any()


# every extent of tiles in each of the three products, on 16-byte boundaries and off them, copied and not; several pieces
LARGE_LOSSES = [
    (8200, 2056, 2056), (8200, 520, 33), (8200, 40, 515), (131100, 130, 65), (16500, 17000, 1032), (8200, 9000, 520),
    (4100, 3000, 1027),
]  # fmt: skip


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,classes,K", LARGE_LOSSES)
def test_large_cross_entropy(device, rows, classes, K, tag):
    """(The definition in 64 bits on the device.)"""
    dtype = DTYPES[tag]
    A, W, targets, grads = loss_case(rows, classes, K, "padded", dtype)
    on_device = [t.to(device) for t in (A, W, targets)]
    grads = [g.to(device) for g in grads]
    results = loss_by_definition(*on_device, grads, dtype)
    losses, log_sums = mops_amd.linear_cross_entropy(*on_device)
    held_to(losses, *results[0], "losses")
    held_to(log_sums, *results[1], "log_sums")
    grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(*grads, *on_device, log_sums)
    held_to(grad_A, *results[2], "grad_A")
    held_to(grad_W, *results[3], "grad_W")
    again = mops_amd.linear_cross_entropy_vjp(*grads, *on_device, log_sums, compute_grad_A=False)
    assert again[0] is None and torch.equal(again[1], grad_W)
    again = mops_amd.linear_cross_entropy_vjp(*grads, *on_device, log_sums, compute_grad_W=False)
    assert again[1] is None and torch.equal(again[0], grad_A)


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("rows,classes,K", [(70, 40, 24), (600, 300, 40), (20, 33, 1600), (3000, 512, 64)])
def test_rows_without_a_target_do_not_matter(device, rows, classes, K, tag):
    """Infinities and NaN in the rows of A and the gradients that are padding stay there."""
    dtype = DTYPES[tag]
    A, W, targets, grads = loss_case(rows, classes, K, "padded", dtype)
    padding = (targets < 0) | (targets >= classes)
    on_device = [t.to(device) for t in (A, W, targets)]
    log_sums = mops_amd.linear_cross_entropy(*on_device)[1]
    clean = mops_amd.linear_cross_entropy(*on_device) + mops_amd.linear_cross_entropy_vjp(
        *[g.to(device) for g in grads], *on_device, log_sums
    )
    for poison in (float("nan"), float("inf"), torch.finfo(dtype).min):
        bad, bad_grads = A.clone(), [g.clone() for g in grads]
        bad[padding] = poison
        for g in bad_grads:
            g[padding] = poison
        bad_sums = torch.where(padding.to(device), poison, log_sums)
        arguments = [bad.to(device), *on_device[1:]]
        again = mops_amd.linear_cross_entropy(*arguments) + mops_amd.linear_cross_entropy_vjp(
            *[g.to(device) for g in bad_grads], *arguments, bad_sums
        )
        assert same(again, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_logits_of_any_size(device, dtype):
    """Logits whose powers leave every range: the losses are differences, and probabilities 0 and 1."""
    W = torch.tensor([[1000.0], [0.0], [-1000.0], [999.0]], dtype=dtype, device=device)
    A = torch.tensor([[1.0], [-1.0], [0.0], [64.0]], dtype=dtype, device=device)
    targets = torch.tensor([0, 0, 2, 2], dtype=torch.int32, device=device)
    losses, log_sums = mops_amd.linear_cross_entropy(A, W, targets)
    logits = A.double() @ W.double().t().contiguous()
    exact = torch.logsumexp(logits, 1)
    assert torch.isfinite(losses).all()
    # (numbers up to 1.3e5, whose unit is 2^-7)
    assert (log_sums - exact).abs().max() <= 2.0**-6
    assert (losses - (exact - logits[torch.arange(4), targets.long()])).abs().max() <= 2.0**-6
    grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(torch.ones(4, device=device), None, A, W, targets, log_sums)
    assert torch.isfinite(grad_A).all() and torch.isfinite(grad_W).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
@pytest.mark.parametrize("base", [60.0, 1000.0, -768.0])
@pytest.mark.parametrize("classes,K", [(12, 2), (700, 2), (40, 2048), (9000, 8)])
def test_classes_that_are_all_but_certain(device, classes, K, base, tag):
    """Logits base + t that are exact (the products and sums are), t = 0 for the likeliest class, ten others near it, all further
    ones far away (their powers are 0 in 32 bits, and nothing beside 1 in 64). A power e^(t - ..) is off by (2 |t| + 8) 2^-p of
    itself, which is (2 |t| + 8) e^t <= 8 2^-p of their sum; so a loss, from differences of logits and the logarithm of a sum of 11
    powers, by (11 * 8 + 16 + 4 |loss|) 2^-p, however large the logits. log_sums has its own rounding besides. d = a e^(x - s) - g
    with the s that is handed in: (a p (2 |x - s| + 8) + 4 (a p + g)) 2^-p and the rounding to the type."""
    dtype = DTYPES[tag]
    p = unit(dtype)
    t = torch.cat([torch.tensor([0.0, -11, -13, -14.5, -12, -20, -9.5, -30, -16, -13.25, -11.75], dtype=torch.float64),
                   torch.full((classes - 11,), -2048.0, dtype=torch.float64)])  # fmt: skip
    t = t[torch.randperm(classes, generator=generator_of(classes, K))]
    W = torch.zeros(classes, K, dtype=dtype)
    W[:, 0], W[:, 1] = base, t.to(dtype)
    targets = torch.cat([t.argmax()[None], (t == -13.25).nonzero()[0], (t == -9.5).nonzero()[0]]).int()
    A = torch.zeros(3, K, dtype=dtype)
    A[:, :2] = 1
    x = base + t
    s = torch.logsumexp(t, 0)
    losses, log_sums = mops_amd.linear_cross_entropy(A.to(device), W.to(device), targets.to(device))
    exact = s - t[targets.long()]
    assert ((losses.double().cpu() - exact).abs() <= (11 * 8 + 16 + 4 * exact) * p).all(), losses
    assert ((log_sums.double().cpu() - (base + s)).abs() <= (11 * 8 + 16 + 2 * abs(base)) * p).all(), log_sums
    wide = losses.dtype
    handed = (base + s).to(wide)[None]
    g, h = 0.75, 0.5
    power = torch.exp(x - handed.double())
    for i in range(3):
        row = [A[i : i + 1].to(device), W.to(device), targets[i : i + 1].to(device)]
        for weights in ((g, h), (g, 0.0)):
            grads = [torch.tensor([w], dtype=wide, device=device) for w in weights]
            grad_W = mops_amd.linear_cross_entropy_vjp(*grads, *row, handed.to(device), compute_grad_A=False)[1]
            one = torch.zeros(classes, dtype=torch.float64)
            one[targets[i].item()] = weights[0]
            d = sum(weights) * power - one
            bound = (sum(weights) * power * (2 * (x - handed.double()).abs() + 8) + 4 * (sum(weights) * power + one)) * p
            bound = bound + 2.0 ** (-2 * BITS[dtype]) * d.abs()  # (16 bits: what two parts leave)
            held_to(grad_W[:, 0], d, bound, f"row {i}")


@pytest.mark.gpu
def test_scale_of_float16_gradients(device):
    """Weights of any size, far below the smallest float16 and far apart from row to row: grad_A of a row, divided by its
    weight, is what it is with the weight one (d is rounded to 2^-11 of itself at the scale of the largest weight, and to
    2^-38 of that beside it)."""
    A, W, targets, _ = loss_case(40, 600, 64, "uniform", torch.float16)
    on_device = [t.to(device) for t in (A, W, targets)]
    log_sums = mops_amd.linear_cross_entropy(*on_device)[1]
    x = A.double() @ W.double().t()
    d = torch.softmax(x, 1)
    d[torch.arange(40), targets.long()] -= 1
    for weight in (1.0, 1000.0, 2.0**-12, 0.0):
        weights = torch.full((40,), weight, device=device)
        weights[::3] *= 0.125
        grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(weights, None, *on_device, log_sums)
        scaled = weights.cpu().double()[:, None] * d
        for actual, exact, terms in ((grad_A, scaled @ W.double(), scaled.abs() @ W.double().abs()),
                                     (grad_W, scaled.t() @ A.double(), scaled.abs().t() @ A.double().abs())):  # fmt: skip
            bound = 2.0**-10 * terms + 2.0**-38 * weight * 600 * 4 * 10 + 2.0**-11 * exact.abs() + 2.0**-25
            assert ((actual.double().cpu() - exact).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.skipif("not torch.cuda.is_available() or torch.cuda.mem_get_info()[0] < 60e9")
def test_operands_of_more_than_two_to_the_31_numbers(device):
    """Matrices whose offsets pass 32 bits: the last columns, classes and numbers against 64 bits."""
    generator = torch.Generator(device=device).manual_seed(3)

    def rand(*shape, scale=1.0):
        return torch.randn(shape, generator=generator, device=device, dtype=torch.bfloat16) * scale

    # (of the rows all but the last 50 numbers are zero: sums of 50 terms, exact zeros beside them)
    # gated: a matrix of 2.4e9 numbers
    rows, K, L = 40, 40000, 30000
    A, W, c = rand(rows, K), rand(1, K, 2 * L, scale=0.1), rand(rows, L)
    A[:, :-50] = 0
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=device)
    output = mops_amd.gated_grouped_product(A, W, offsets)
    last = slice(L - 40, L)
    a, w = A[:, -50:].double(), W[0, -50:].double()
    w_gate, w_up = w[:, :L][:, last].contiguous(), w[:, L:][:, last].contiguous()
    gate, up, e = a @ w_gate, a @ w_up, (50 + 32) * 2.0**-24
    G, U = a.abs() @ w_gate.abs(), a.abs() @ w_up.abs()
    held_to(output[:, last], gate * torch.sigmoid(gate) * up, e * 2.2 * G * U, "output")
    grad_W = mops_amd.gated_grouped_product_vjp(c, A, W, offsets, compute_grad_A=False)[1]
    cotangent, value = c[:, last].double(), gate * torch.sigmoid(gate)
    off = cotangent.abs() * (e * 2.2 * G + 2.0**-8 * value.abs())
    exact, turned = a.t().contiguous() @ (cotangent * value), a.abs().t().contiguous()
    bound = turned @ off + (rows + 16) * 2.0**-24 * (turned @ (cotangent * value).abs())
    held_to(grad_W[0, -50:, L:][:, last], exact, bound, "grad_W")
    assert not grad_W[0, :-50].any()
    del W, output, grad_W
    # cross entropy: classes of 2.3e9 numbers
    rows, V, K = 30, 70001, 32768
    A, W = rand(rows, K), rand(V, K, scale=0.1)
    A[:, :-50] = 0
    targets = torch.arange(V - rows, V, dtype=torch.int32, device=device)
    one = torch.ones(rows, device=device)
    losses, log_sums = mops_amd.linear_cross_entropy(A, W, targets)
    grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(one, None, A, W, targets, log_sums)
    results = loss_by_definition(A[:, -50:], W[:, -50:], targets, [one, 0 * one], torch.bfloat16)
    held_to(losses, *results[0], "losses")
    held_to(log_sums, *results[1], "log_sums")
    held_to(grad_A[:, -50:], *results[2], "grad_A")
    held_to(grad_W[:, -50:], *results[3], "grad_W")
    assert not grad_W[:, :-50].any()
    del W, grad_W
    # gradients: one of 2.2e9 numbers, all of them zero but the last
    large = torch.zeros((1 << 31) + 100001, dtype=torch.bfloat16, device=device)
    large[-1] = 4.0
    clipped, norm = mops_amd.clip_gradients([large, torch.full((1,), 3.0, device=device)], 2.5)
    assert norm.item() == 5.0 and clipped[0][-1] == 2.0 and clipped[1].item() == 1.5
    assert clipped[0].count_nonzero() == 1


# --------------------------------------------------------- norm of gradients ----
def gradient_lists():
    f32, f64, bf16, f16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
    return {
        "one number": [((), f32)],
        "nothing in one": [((0,), f32), ((3, 0), bf16), ((5,), f32)],
        "nothing at all": [((0, 4), f16)],
        "odd": [((7,), bf16), ((1,), f32), ((33, 3), f16), ((129,), bf16), ((8191,), f32), ((4097,), f16)],
        "mixed": [((300, 70), bf16), ((300,), f32), ((70,), f64), ((64, 64, 3), f16)],
        "many": [((i % 37 + 1, 5), (f32, bf16, f16)[i % 3]) for i in range(200)],
        "large": [((3000, 4001), bf16), ((1 << 22) + 3, f32), ((2049,), f32), ((5000000,), f16)],
        "double": [((70000,), f64), ((3,), f64)],
    }


def gradients_of(name, device, scale=0.01):
    generator = torch.Generator().manual_seed(len(name))
    shapes = [((shape,) if isinstance(shape, int) else shape, dtype) for shape, dtype in gradient_lists()[name]]
    return [random(generator, shape, dtype, scale).to(device) for shape, dtype in shapes]


def exact_norm(gradients):
    return math.sqrt(sum((g.double() ** 2).sum().item() for g in gradients))


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(gradient_lists()))
def test_gradient_norm(device, name):
    """Squares are exact in 64 bits, their sum is off by n 2^-53 at most, the norm's rounding by 2^-24 (2^-53)."""
    gradients = gradients_of(name, device)
    norm = mops_amd.gradient_norm(gradients)
    wide = any(g.dtype == torch.float64 for g in gradients)
    assert norm.shape == () and norm.dtype == (torch.float64 if wide else torch.float32)
    exact = exact_norm(gradients)
    numbers = sum(g.numel() for g in gradients)
    bound = (numbers * 2.0**-53 + 2.0 ** (-52 if wide else -24)) * exact * 1.01
    assert abs(norm.item() - exact) <= bound
    assert torch.equal(mops_amd.gradient_norm(tuple(gradients)), norm)


@pytest.mark.gpu
@pytest.mark.parametrize("share", [0.3, 1.5, 0.0, math.inf])
@pytest.mark.parametrize("name", list(gradient_lists()))
def test_clip_gradients(device, name, share):
    """A clipped number is off by its rounding, 2^-q of itself, and by the factor's: 2^-24 for 16 bits, where it is held in
    32, and the norm's n 2^-53 and a few 2^-53 for the others."""
    gradients = gradients_of(name, device)
    exact = exact_norm(gradients)
    max_norm = share * exact if exact > 0 else share
    before = [g.clone() for g in gradients]
    clipped, norm = mops_amd.clip_gradients(gradients, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(gradients, before))
    assert torch.equal(norm, mops_amd.gradient_norm(gradients))
    factor = 1.0 if exact <= max_norm else max_norm / exact
    numbers = sum(g.numel() for g in gradients)
    for actual, g in zip(clipped, gradients, strict=True):
        assert actual.dtype == g.dtype and actual.stride() == g.stride()
        off = (2.0**-23 if torch.finfo(g.dtype).bits == 16 else 0) + (numbers + 8) * 2.0**-53
        held_to(actual, g.double().cpu() * factor, off * g.double().cpu().abs() * factor, name)
        if factor == 1.0:
            assert torch.equal(actual, g)
    versions = [g._version for g in gradients]
    assert torch.equal(mops_amd.clip_gradients_(gradients, max_norm), norm)
    assert all(torch.equal(a, b) for a, b in zip(gradients, clipped, strict=True))
    assert all(g._version > version for g, version in zip(gradients, versions))


@pytest.mark.gpu
def test_gradients_of_any_size(device):
    """Numbers whose squares leave 32 bits, and numbers that are none."""
    large = [torch.full((1000,), 1e30, device=device), torch.full((10,), -1e37, dtype=torch.bfloat16, device=device)]
    small = [torch.full((1000,), 1e-30, device=device), torch.full((7,), 2e-38, dtype=torch.bfloat16, device=device)]
    for gradients in (large, small):
        exact = exact_norm(gradients)
        clipped, norm = mops_amd.clip_gradients(gradients, exact / 2)
        assert abs(norm.item() - exact) <= 2.0**-23 * exact
        assert abs(exact_norm(clipped) - exact / 2) <= 2.0**-8 * exact
    ones = torch.ones(5, device=device)
    clipped, norm = mops_amd.clip_gradients([ones, torch.tensor([math.inf, 1.0], device=device)], 1.0)
    assert norm.item() == math.inf and not clipped[0].any() and clipped[1][0].isnan() and clipped[1][1] == 0
    clipped, norm = mops_amd.clip_gradients([ones, torch.tensor([math.nan, 1.0], device=device)], 1.0)
    assert norm.isnan() and clipped[0].isnan().all() and clipped[1].isnan().all()
    zeros = [torch.zeros(9, device=device)]
    assert mops_amd.clip_gradients_(zeros, 0.0).item() == 0 and not zeros[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize(
    "size,max_norm,dtypes",
    [
        (3e38, 1e-3, (torch.bfloat16, torch.float32)), (3e38, 1e-5, (torch.bfloat16,)), (3e38, 1e-30, (torch.bfloat16, torch.float32)),
        (1e150, 1e-200, (torch.float64,)), (1e30, 1e-14, (torch.bfloat16, torch.float64)), (6e4, 1e-2, (torch.float16, torch.float32)),
    ],
)  # fmt: skip
def test_factors_below_every_number_of_the_type(device, size, max_norm, dtypes):
    """max_norm / norm is a number below the smallest one of 32 bits (or 64), a gradient times it is an ordinary number: off by its
    rounding, the factor's digits and the norm's (2^-23 for 16 bits, (n + 8) 2^-53 for the others)."""
    generator = torch.Generator().manual_seed(8)
    gradients = [(torch.rand(shape, generator=generator) * 0.9 + 0.1).double().mul(size).to(dtype).to(device)
                 for dtype in dtypes for shape in ((3001,), (20, 33))]  # fmt: skip
    exact = exact_norm(gradients)
    numbers = sum(g.numel() for g in gradients)
    clipped, _ = mops_amd.clip_gradients(gradients, max_norm)
    for actual, g in zip(clipped, gradients, strict=True):
        expected = g.double().cpu() / exact * max_norm
        off = (2.0**-23 if torch.finfo(g.dtype).bits == 16 else 0) + (numbers + 8) * 2.0**-53
        held_to(actual, expected, off * expected.abs(), str(g.dtype))
    mops_amd.clip_gradients_(gradients, max_norm)
    assert same(tuple(gradients), tuple(clipped))


@pytest.mark.gpu
@pytest.mark.parametrize(
    "sizes", [(1e200,), (1.7e308,), (1e-200,), (1e-308,), (5e-324 * 2.0**20,), (1e150, 1e-160), (1e-150, 1e170), (1e250, 1e-250, 1.0)],
)  # fmt: skip
def test_double_gradients_whose_squares_leave_the_range(device, sizes):
    """Norm and clipped gradients against the same numbers divided by the largest of the sizes (products of numbers of 64 bits
    are off by 2^-53 each, sums of n squares by n 2^-53; beside it smaller sizes are nothing, or as exact)."""
    generator = torch.Generator().manual_seed(9)
    unit_numbers = [torch.rand(shape, generator=generator, dtype=torch.float64) * 0.9 + 0.1 for shape in ((3,), (5001,), (33, 7))]
    largest = max(sizes)
    gradients = [g * size for size in sizes for g in unit_numbers]
    exact = math.sqrt(sum(((g / largest) ** 2).sum().item() for g in gradients))  # times `largest`
    gradients = [g.to(device) for g in gradients] + [torch.full((40,), 1e-38, device=device, dtype=torch.bfloat16)]
    if largest < 1e-38:
        gradients.pop()
    numbers = sum(g.numel() for g in gradients)
    norm = mops_amd.gradient_norm(gradients)
    representable = exact * (largest * 0.001) < 1.7e305
    if representable:
        assert abs(norm.item() / largest - exact) <= (numbers + 8) * 2.0**-53 * exact + 5e-324 / largest
    else:
        assert norm.item() == math.inf
    for max_norm in (0.25 * largest, 1e-3 if largest > 1 else 1e-3 * largest):
        clipped, again = mops_amd.clip_gradients(gradients, max_norm)
        assert torch.equal(again, norm)
        for actual, g in zip(clipped, gradients, strict=True):
            expected = g.double().cpu() / exact * (max_norm / largest)
            off = (2.0**-23 if g.dtype == torch.bfloat16 else 0) + (numbers + 8) * 2.0**-53
            held_to(actual, expected, off * expected.abs(), str(g.dtype))
    unchanged, _ = mops_amd.clip_gradients(gradients, math.inf)
    assert same(tuple(unchanged), tuple(gradients))


@pytest.mark.gpu
def test_layouts_of_gradients(device):
    """Any order of dimensions in place; gaps, expanded numbers and memory off every boundary where nothing is written."""
    generator = torch.Generator().manual_seed(5)
    base = random(generator, (40, 33, 5), torch.float32).to(device)
    turned = base.permute(2, 0, 1)
    gaps, expanded = base[:, ::2], base[:1, :1, :1].expand(3, 4, 5)
    shifted = base.flatten()[1:1000].bfloat16()
    off = torch.empty(1000, dtype=torch.bfloat16, device=device)[1:]
    off.copy_(shifted)
    every = [turned, gaps, expanded, off]
    exact = exact_norm(every)
    assert abs(mops_amd.gradient_norm(every).item() - exact) <= 2.0**-23 * exact
    clipped, _ = mops_amd.clip_gradients(every, exact / 3)
    for actual, g in zip(clipped, every, strict=True):
        assert actual.shape == g.shape
        held_to(actual, g.double().cpu() / 3, 2.0**-22 * g.double().cpu().abs(), "clipped")
    copies = [turned.clone(), off]
    expected, norm = mops_amd.clip_gradients(copies, 0.5)
    assert expected[0].stride() == copies[0].stride()
    memory = copies[0]
    assert torch.equal(mops_amd.clip_gradients_(copies, 0.5), norm)
    assert torch.equal(memory, expected[0]) and torch.equal(off, expected[1])
    for bad in ([gaps], [expanded]):
        with pytest.raises(ValueError, match="without gaps"):
            mops_amd.clip_gradients_(bad, 1.0)
    for bad in ([base, base], [base, base.view(-1)[3:]]):
        with pytest.raises(mops_amd.MopsError, match="must not share memory"):
            mops_amd.clip_gradients_(bad, 1.0)
    # (where nothing is written, the same tensor twice counts twice)
    assert abs(mops_amd.gradient_norm([base, base]).item() - math.sqrt(2) * exact_norm([base])) <= 2.0**-22 * exact_norm([base])


@pytest.mark.gpu
def test_clipped_gradients_of_parameters(device):
    parameter = torch.ones(4, device=device, requires_grad=True)
    with pytest.raises(ValueError, match="requires a gradient itself"):
        mops_amd.clip_gradients_([parameter], 1.0)
    with torch.no_grad():
        assert mops_amd.clip_gradients_([parameter], 1.0).item() == 2.0
    assert parameter.eq(0.5).all()
    (parameter.sum() * 3).backward()
    assert mops_amd.clip_gradients_((p.grad for p in [parameter]), 3.0).item() == 6.0
    assert parameter.grad.eq(1.5).all()


# ------------------------------------------------- layouts, streams, calls ----
def all_calls(device, dtype, rows=200, groups=5, columns=70):
    """name -> (function, arguments) of every function, on ordinary tensors."""
    generator = generator_of(rows, groups, columns, 9)

    def rand(*shape, dtype=dtype):
        return random(generator, shape, dtype).to(device)

    wide = torch.float64 if dtype == torch.float64 else torch.float32
    index = indices_of("padded", rows, groups).to(device)
    order, offsets = mops_amd.order_by_group(index, groups)
    A, W, classes = rand(rows, columns), rand(groups, columns, 66), rand(300, columns)
    targets = indices_of("padded", rows, 300).to(device)
    log_sums = mops_amd.linear_cross_entropy(A, classes, targets)[1]
    return {
        "gated_grouped_product": (mops_amd.gated_grouped_product, [A, W, offsets, order, "gelu"]),
        "gated_grouped_product_vjp": (
            mops_amd.gated_grouped_product_vjp, [rand(rows, 33), A, W, offsets, order, "silu"],
        ),
        "linear_cross_entropy": (mops_amd.linear_cross_entropy, [A, classes, targets]),
        "linear_cross_entropy_vjp": (
            mops_amd.linear_cross_entropy_vjp,
            [rand(rows, dtype=wide), rand(rows, dtype=wide), A, classes, targets, log_sums],
        ),
        "gradient_norm": (lambda *t: mops_amd.gradient_norm(list(t)), [A, W, classes]),
        "clip_gradients": (
            lambda *t: (lambda clipped, norm: (*clipped, norm))(*mops_amd.clip_gradients(list(t), 3.0)), [A, W, classes],
        ),
        "clip_gradients_": (
            lambda *t: (lambda c: (mops_amd.clip_gradients_(c, 3.0), *c))([x.clone() for x in t]), [A, W, classes],
        ),
    }  # fmt: skip


FUNCTIONS = [*training._SIGNATURES, "gradient_norm", "clip_gradients", "clip_gradients_"]


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

    if function != "clip_gradients_":
        assert same(call(*[strided(x) for x in arguments]), expected)
    assert same(call(*[shifted(x) for x in arguments]), expected)
    monkeypatch.setattr(training, "_native", _c_lib._NoFunctions())
    assert same(call(*arguments), expected)
    assert same(call(*[shifted(x) for x in arguments]), expected)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
@pytest.mark.parametrize("function", FUNCTIONS)
def test_another_stream_and_a_graph(device, function, dtype):
    """On a stream of the caller's, behind work that is still running there; and captured, replayed with other work
    in between: the same bits every time."""
    call, arguments = all_calls(device, dtype)[function]
    expected = call(*arguments)
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
        captured = call(*late)
    # (log_sums are those of A and W: of the cross entropy's gradients, the cotangents change)
    changing = 2 if function == "linear_cross_entropy_vjp" else len(late)
    for repeat in range(4):
        for to, x in zip(late[:changing], arguments):
            if isinstance(x, torch.Tensor) and x.is_floating_point():
                to.copy_(x * (1 + repeat % 2))
        graph.replay()
        torch.cuda.synchronize()
        eager = call(*late)
        assert same(captured, eager)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_gradients_against_differences(device):
    """In float64: the error of a central difference is h^2 f'''/6, 1e-10 of values of order one, and its rounding
    1e-16 / h = 1e-11; held to 1e-7 of the sum's scale."""
    generator = generator_of(77)

    def rand(*shape):
        return random(generator, shape, torch.float64).to(device)

    index = indices_of("padded", 40, 6).to(device)
    order, offsets = mops_amd.order_by_group(index, 6)
    targets = indices_of("padded", 40, 23).to(device)

    def loss_vjp(g, inputs):
        return mops_amd.linear_cross_entropy_vjp(*g, *inputs, targets, mops_amd.linear_cross_entropy(*inputs, targets)[1])

    cases = [
        (lambda A, W, which=which: mops_amd.gated_grouped_product(A, W, offsets, order, which),
         [rand(40, 9), rand(6, 9, 26)], [rand(40, 13)],
         lambda g, inputs, which=which: mops_amd.gated_grouped_product_vjp(*g, *inputs, offsets, order, which))
        for which in ACTIVATIONS
    ] + [
        (lambda A, W: mops_amd.linear_cross_entropy(A, W, targets), [rand(40, 9), rand(23, 9)], [rand(40), rand(40)], loss_vjp),
    ]  # fmt: skip
    for function, inputs, cotangents, vjp in cases:
        gradients = vjp(cotangents, inputs)
        for which, gradient in enumerate(gradients):
            direction = rand(*inputs[which].shape)
            expected = central_difference(function, inputs, which, direction, cotangents)
            actual = (gradient * direction).sum().item()
            scale = (gradient * direction).abs().sum().item() + 1.0
            assert abs(actual - expected) <= 1e-7 * scale, (which, actual, expected)


# -------------------------------------------------------------- refusals ----
def test_host_tensors_are_refused():
    index, values = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4)
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.gated_grouped_product(values, torch.zeros(1, 4, 2), index[:2])
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.gated_grouped_product_vjp(values, values, torch.zeros(1, 4, 8), index[:2])
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.linear_cross_entropy(values, values, index)
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.linear_cross_entropy_vjp(values[0], None, values, values, index, values[0])
    for function in (mops_amd.clip_gradients, mops_amd.clip_gradients_):
        with pytest.raises(TypeError, match="device path only"):
            function([values], 1.0)
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.gradient_norm([values])


def test_not_arrays():
    with pytest.raises(TypeError, match="`A` must be an array in linear_cross_entropy"):
        mops_amd.linear_cross_entropy([0.0], torch.zeros(3, 4), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="`W` must be a 3D array in gated_grouped_product, got a 2D array"):
        mops_amd.gated_grouped_product(torch.zeros(3, 4), torch.zeros(3, 4), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="must be a list of tensors in gradient_norm"):
        mops_amd.gradient_norm(torch.zeros(3))
    with pytest.raises(ValueError, match="at least one tensor in clip_gradients"):
        mops_amd.clip_gradients([], 1.0)


@pytest.mark.gpu
def test_refusals(device):
    def floats(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device=device)

    def integers(*shape):
        return torch.zeros(shape, dtype=torch.int32, device=device)

    error, gated, loss = mops_amd.MopsError, mops_amd.gated_grouped_product, mops_amd.linear_cross_entropy
    with pytest.raises(ValueError, match="`activation` must be one of silu, gelu, sigmoid"):
        gated(floats(5, 4), floats(2, 4, 6), integers(3), None, "relu")
    with pytest.raises(error, match="W must have an even number of columns"):
        gated(floats(5, 4), floats(2, 4, 7), integers(3))
    with pytest.raises(error, match="sizes of A along dimension 1 and W along dimension 1"):
        gated(floats(5, 3), floats(2, 4, 6), integers(3))
    with pytest.raises(error, match="offsets must have 3 elements"):
        gated(floats(5, 4), floats(2, 4, 6), integers(2))
    with pytest.raises(error, match="grad_output must have 3 columns"):
        mops_amd.gated_grouped_product_vjp(floats(5, 6), floats(5, 4), floats(2, 4, 6), integers(3))
    with pytest.raises(TypeError, match="Wrong dtype for W in gated_grouped_product"):
        gated(floats(5, 4), floats(2, 4, 6, dtype=torch.float16), integers(3))
    with pytest.raises(error, match="sizes of A along dimension 1 and W along dimension 1"):
        loss(floats(5, 4), floats(6, 3), integers(5))
    with pytest.raises(error, match="sizes of targets along dimension 0 and A along dimension 0"):
        loss(floats(5, 4), floats(6, 4), integers(4))
    with pytest.raises(TypeError, match="Wrong dtype for targets"):
        loss(floats(5, 4), floats(6, 4), floats(5))
    with pytest.raises(TypeError, match="Wrong dtype for grad_losses"):
        half = floats(5, 4, dtype=torch.bfloat16)
        mops_amd.linear_cross_entropy_vjp(half[:, 0], None, half, half, integers(5), floats(5))
    with pytest.raises(error, match="sizes of log_sums along dimension 0"):
        mops_amd.linear_cross_entropy_vjp(None, None, floats(5, 4), floats(6, 4), integers(5), floats(4))
    with pytest.raises(error, match="sizes of grad_log_sums along dimension 0"):
        mops_amd.linear_cross_entropy_vjp(None, floats(6), floats(5, 4), floats(6, 4), integers(5), floats(5))
    for bad in (-1.0, math.nan):
        with pytest.raises(error, match="max_norm must be a number that is not negative"):
            mops_amd.clip_gradients([floats(3)], bad)
    with pytest.raises(TypeError, match="`max_norm` must be a scalar"):
        mops_amd.clip_gradients([floats(3)], "1")
    with pytest.raises(TypeError, match="Wrong dtype or layout"):
        mops_amd.gradient_norm([floats(3), integers(3)])
    with pytest.raises(TypeError, match="device path only"):
        mops_amd.gradient_norm([floats(3), torch.zeros(3)])
    with pytest.raises(TypeError, match=r"`gradients\[1\]` must be a tensor in clip_gradients_"):
        mops_amd.clip_gradients_([floats(3), None], 1.0)
    # (a refused call leaves nothing behind: the next one is right)
    assert mops_amd.gradient_norm([floats(4) + 1]).item() == 2.0


def test_refusals_of_lists(tmp_path):
    """What the C entries for lists refuse before they touch a device."""
    from mops_amd._c_lib import device_library

    library = device_library()
    gradient, norm_type = training._Gradient, training._STRUCTS[(1, "f32")]
    memory = (ctypes.c_float * 64)()
    at = ctypes.addressof(memory)

    def call(outputs, gradients, max_norm=1.0, extent=1, count=None):
        norm = norm_type()
        norm.data = ctypes.cast(ctypes.c_void_p(at), type(norm.data))
        norm.shape[0] = extent
        entry = library.cdll.mops_amd_clip_gradients_f32
        entry.restype = ctypes.c_int
        arrays = [None if x is None else (gradient * len(x))(*[gradient(*y) for y in x]) for x in (outputs, gradients)]
        entry.argtypes = [norm_type, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_double]
        addresses = [None if x is None else ctypes.addressof(x) for x in arrays]
        assert entry(norm, *addresses, len(gradients or []) if count is None else count, max_norm) == 1
        return library.last_error()

    one = [(at, 8, 0)]
    assert "norm must have one element" in call(one, one, extent=2)
    assert "not negative" in call(one, one, max_norm=-0.5)
    assert "there are no gradients" in call(None, None, count=1)
    assert "there are no outputs" in call(None, one)
    assert "does not fit in size_t" in call(one, one, count=-1)
    assert "gradients[0] has no known type" in call(one, [(at, 8, 4)])
    assert "gradients[0] has no memory, or a negative size" in call(one, [(at, -1, 0)])
    assert "gradients[0] has no memory" in call(one, [(None, 8, 0)])
    assert "outputs[0] must have the size and the type" in call([(at, 8, 2)], one)
    assert "outputs[0] must have the size and the type" in call([(at, 7, 0)], one)
    assert "must not share memory with each other" in call([(at, 8, 0), (at + 28, 8, 0)], [(at + 100, 8, 0), (at + 140, 8, 0)])
    assert "share none with any gradient" in call([(at, 8, 0)], [(at + 16, 8, 0)])
    assert "share none with any gradient" in call([(at, 8, 0), (at + 64, 8, 0)], [(at, 8, 0), (at + 8, 8, 0)])


def test_refusals_of_the_memory_of_a_norm():
    """Likewise: a norm without memory, and one that lies in a gradient or an output."""
    from mops_amd._c_lib import device_library

    library = device_library()
    gradient = training._Gradient
    memory = (ctypes.c_double * 64)()
    at = ctypes.addressof(memory)
    for tag, size in (("f32", 4), ("f64", 8)):
        view = training._STRUCTS[(1, tag)]

        def call(name, address, *lists, tag=tag, view=view):
            norm = view()
            norm.data = ctypes.cast(ctypes.c_void_p(address), type(norm.data))
            norm.shape[0] = 1
            entry = getattr(library.cdll, f"mops_amd_{name}_{tag}")
            entry.restype = ctypes.c_int
            entry.argtypes = [view, *[ctypes.POINTER(gradient)] * len(lists), ctypes.c_int64]
            arrays = [(gradient * len(x))(*[gradient(*y) for y in x]) for x in lists]
            arguments = [norm, *arrays, len(lists[0])]
            if name == "clip_gradients":
                entry.argtypes = [*entry.argtypes, ctypes.c_double]
                arguments.append(1.0)
            assert entry(*arguments) == 1
            return library.last_error()

        gradients, outputs = [(at, 8, 0), (at + 64, 8, 0)], [(at + 128, 8, 0), (at + 192, 8, 0)]
        assert "norm has no memory in gradient_norm" in call("gradient_norm", None, gradients)
        assert "norm has no memory in clip_gradients" in call("clip_gradients", None, outputs, gradients)
        inside = [at, at + 96 - size, at + 128, at + 216]
        for address in inside:
            assert "norm must not share memory" in call("clip_gradients", address, outputs, gradients)
        assert "norm must not share memory" in call("clip_gradients", at + 32 - size, gradients, gradients)


TILES = """
#include <cstdio>
#include <vector>
#include "tile_order.hpp"
using namespace mops::amd;
int main() {
    for (int tiles : {0, 1, 7, 8, 9, 63, 64, 65, 901, 4000}) for (int rest : {0, 1, 5, 8, 77, 1328}) {
        std::vector<int> made(tiles + rest, 0);
        const long long workgroups = workgroups_for(tiles + rest);
        for (long long b = 0; b < workgroups; b++) {
            const int tile = tile_of(static_cast<unsigned>(b), tiles, rest);
            if (tile >= tiles + rest) return 1;
            if (tile >= 0) made[tile]++;
        }
        int once = 0, of_first = 0;
        for (int x : made) once += x == 1;
        for (long long b = 0; b < workgroups; b += 8) {
            const int tile = tile_of(static_cast<unsigned>(b), tiles, rest);
            of_first += tile >= 0 && tile < tiles;
        }
        printf("%d %d %d %d %lld\\n", tiles, rest, once, of_first, workgroups);
    }
}
"""


def test_every_tile_is_made_once(tmp_path):
    """Over the kernels' own header: each tile by one workgroup of those there are, however many of the rows are in no group,
    and no XCD has more than its share of the others' tiles."""
    got = run_on_host(tmp_path, TILES)
    tiles, rest, once, of_first, workgroups = got.T
    assert len(got) == 60 and (once == tiles + rest).all()
    assert (of_first <= -(-tiles // 8)).all() and (workgroups <= tiles + rest + 16).all()


FULL_DEVICE = """
import ctypes, os, sys
sys.path.insert(0, os.getcwd())
import torch
import mops_amd
from mops_amd._c_lib import device_library
from tests import test_training as t
os.environ["MOPS_AMD_TEST_SCRATCH_LIMIT"] = str(48 << 20)  # what a nearly full device has left for the block
library = device_library().cdll
library.mops_amd_scratch_capacity.restype = ctypes.c_int64
device = torch.device("cuda:0")
cases = [
    (4100, 9000, 72, torch.bfloat16), (2100, 9001, 65, torch.float32), (4100, 9000, 71, torch.float16),
    (250, 90001, 72, torch.bfloat16), (250, 90001, 40, torch.float16),  # (in two parts, three pieces each)
]
for rows, classes, K, dtype in cases:
    A, W, targets, grads = [
        [x.to(device) for x in y] if isinstance(y, list) else y.to(device)
        for y in t.loss_case(rows, classes, K, "padded", dtype)
    ]
    results = t.loss_by_definition(A, W, targets, grads, dtype, 2.0 ** (-2 * t.BITS[dtype]) if rows == 250 else None)
    losses, log_sums = mops_amd.linear_cross_entropy(A, W, targets)
    t.held_to(losses, *results[0], "losses")
    grad_A, grad_W = mops_amd.linear_cross_entropy_vjp(*grads, A, W, targets, log_sums)
    t.held_to(grad_A, *results[2], "grad_A")
    t.held_to(grad_W, *results[3], "grad_W")
    assert library.mops_amd_scratch_capacity() <= 48 << 20
    print("ok", library.mops_amd_scratch_capacity(), flush=True)
# gated products at odd addresses, without room for copies
generator = torch.Generator().manual_seed(1)
A, W, c = [t.random(generator, shape, torch.float16, scale).to(device)
           for shape, scale in (((5000, 1031), 1.0), ((1, 1031, 2 * 1033), 0.03), ((5000, 1033), 1.0))]
offsets = torch.tensor([0, 5000], dtype=torch.int32, device=device)
index = torch.zeros(5000, dtype=torch.int32)
output = mops_amd.gated_grouped_product(A, W, offsets)
results = t.gated_by_definition(A.cpu(), W.cpu(), index, "silu", c.cpu(), torch.float16)
t.held_to(output, *results[0], "output")
grads = mops_amd.gated_grouped_product_vjp(c, A, W, offsets)
t.held_to(grads[0], *results[1], "grad_A")
t.held_to(grads[1], *results[2], "grad_W")
assert library.mops_amd_scratch_capacity() <= 48 << 20
# memory that a call cannot do without: an error, and no trace of it in the next call
os.environ["MOPS_AMD_TEST_SCRATCH_LIMIT"] = str(1 << 20)
try:
    mops_amd.gated_grouped_product_vjp(c.repeat(4, 1), A.repeat(4, 1), W, offsets * 4)
    raise SystemExit("no error")
except mops_amd.MopsError:
    pass
del os.environ["MOPS_AMD_TEST_SCRATCH_LIMIT"]
assert torch.equal(mops_amd.gated_grouped_product(A[:64], W, torch.tensor([0, 64], dtype=torch.int32, device=device)),
                   mops_amd.gated_grouped_product(A[:64].clone(), W, torch.tensor([0, 64], dtype=torch.int32, device=device)))
print("ok", flush=True)
"""


@pytest.mark.gpu
def test_on_a_device_that_is_nearly_full(device):
    """Copies of operands and large pieces of the classes are memory that a call can do without."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FULL_DEVICE], cwd=root, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout + done.stderr[-3000:]
    assert done.stdout.count("ok") == 6, done.stdout


LOSSES_ON_A_FULL_DEVICE = """
import ctypes, os, sys
sys.path.insert(0, os.getcwd())
import torch
import mops_amd
from mops_amd._c_lib import device_library
from tests import test_training as t
os.environ["MOPS_AMD_TEST_SCRATCH_LIMIT"] = str(3 << 20)
library = device_library().cdll
library.mops_amd_scratch_capacity.restype = ctypes.c_int64
cases = [
    (20000, 9000, 72, torch.bfloat16), (20000, 9000, 71, torch.float16), (20000, 4001, 40, torch.float32),
    (9000, 2003, 33, torch.float64), (20000, 300, 16, torch.bfloat16),
    (200, 500001, 8, torch.float32), (60, 1000003, 8, torch.bfloat16),  # (without a plan; wide tiles)
]
for rows, classes, K, dtype in cases:
    A, W, targets, _ = t.loss_case(rows, classes, K, "padded", dtype)
    A, W, targets = [x.cuda() for x in (A, W, targets)]
    none = torch.zeros(rows, dtype=torch.float64, device="cuda")
    results = t.loss_by_definition(A, W, targets, [none, none], dtype)
    losses, log_sums = mops_amd.linear_cross_entropy(A, W, targets)
    t.held_to(losses, *results[0], "losses")
    t.held_to(log_sums, *results[1], "log_sums")
    again = mops_amd.linear_cross_entropy(A, W, targets)
    assert torch.equal(losses, again[0]) and torch.equal(log_sums, again[1])
    outside = (targets < 0) | (targets >= classes)
    assert outside.any() and not losses[outside].any() and not log_sums[outside].any()
    assert library.mops_amd_scratch_capacity() <= 3 << 20
    print("ok", library.mops_amd_scratch_capacity(), flush=True)
    # captured, in what the block has room for
    stream, graph, fixed = torch.cuda.Stream(), torch.cuda.CUDAGraph(), A.clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        captured = mops_amd.linear_cross_entropy(fixed, W, targets)
    for repeat in range(3):
        fixed.zero_()
        graph.replay()
        torch.cuda.synchronize()
        same = torch.where(outside, 0.0, torch.full_like(losses, classes).log())
        assert (captured[1] - same).abs().max() <= 1e-5
        fixed.copy_(A)
        graph.replay()
        torch.cuda.synchronize()
        t.held_to(captured[0], *results[0], "losses")
        t.held_to(captured[1], *results[1], "log_sums")
        assert torch.equal(mops_amd.linear_cross_entropy(A, W, targets)[0], losses)
"""


@pytest.mark.gpu
def test_losses_on_a_device_that_is_nearly_full(device):
    """The partial sums of all classes at once are memory that a call can do without."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    program = [sys.executable, "-c", LOSSES_ON_A_FULL_DEVICE]
    done = subprocess.run(program, cwd=root, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout + done.stderr[-3000:]
    assert done.stdout.count("ok") == 7, done.stdout


@pytest.mark.gpu
@pytest.mark.skipif("not torch.cuda.is_available() or torch.cuda.mem_get_info()[0] < 60e9")
def test_losses_in_pieces_of_the_classes(device):
    """More partial sums than are held at a time (some rows against the definition in 64 bits)."""
    rows, classes, K = 140000, 128301, 8
    A, W, targets, _ = loss_case(rows, classes, K, "padded", torch.bfloat16)
    some = torch.arange(0, rows, 611)
    none = torch.zeros(len(some), dtype=torch.float64, device=device)
    A, W, targets = A.to(device), W.to(device), targets.to(device)
    results = loss_by_definition(A[some], W, targets[some], [none, none], torch.bfloat16)
    losses, log_sums = mops_amd.linear_cross_entropy(A, W, targets)
    held_to(losses[some], *results[0], "losses")
    held_to(log_sums[some], *results[1], "log_sums")
    outside = (targets < 0) | (targets >= classes)
    assert outside.any() and not losses[outside].any() and not log_sums[outside].any()


# ------------------------------------------------------ PyTorch operators ----
def operators():
    import mops_amd.torch  # noqa: F401  (registers the operators)

    return torch.ops.mops


SCHEMAS = {
    "gated_grouped_product": "mops::gated_grouped_product(Tensor A, Tensor W, Tensor offsets, Tensor? order=None, str activation=\"silu\") -> Tensor",
    "linear_cross_entropy": "mops::linear_cross_entropy(Tensor A, Tensor W, Tensor targets) -> (Tensor, Tensor)",
    "gradient_norm": "mops::gradient_norm(Tensor[] gradients) -> Tensor",
    "clip_gradients": "mops::clip_gradients(Tensor[] gradients, float max_norm) -> (Tensor[], Tensor)",
    "clip_gradients_": "mops::clip_gradients_(Tensor(a!)[] gradients, float max_norm) -> Tensor",
}  # fmt: skip


@pytest.mark.parametrize("name", list(SCHEMAS))
def test_operator_schemas(name):
    assert str(getattr(operators(), name).default._schema) == SCHEMAS[name]


def test_operators_refuse_host_tensors():
    index, values = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="device path only"):
        operators().gated_grouped_product(values, torch.zeros(1, 4, 2), index[:2])
    with pytest.raises(RuntimeError, match="device path only"):
        operators().linear_cross_entropy(values, values, index)
    with pytest.raises(RuntimeError, match="device path only"):
        operators().gradient_norm([values])
    with pytest.raises(RuntimeError, match="device path only"):
        operators().clip_gradients([values], 1.0)
    with pytest.raises(RuntimeError, match="device path only"):
        operators().clip_gradients_([values], 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("tag", list(DTYPES))
def test_operators_with_autograd(device, tag):
    """Values and gradients of the operators: what the functions of the package give, bit for bit."""
    ops, dtype = operators(), DTYPES[tag]
    generator = generator_of(22)

    def rand(*shape, dtype=dtype):
        return random(generator, shape, dtype).to(device)

    wide = torch.float64 if dtype == torch.float64 else torch.float32
    index, targets = indices_of("padded", 50, 4).to(device), indices_of("padded", 50, 31).to(device)
    order, offsets = ops.order_by_group(index, 4)
    A, W, classes, grad = rand(50, 24), rand(4, 24, 20), rand(31, 24), rand(50, 10)
    for activation in ACTIVATIONS:
        leaves = [A.clone().requires_grad_(True), W.clone().requires_grad_(True)]
        output = ops.gated_grouped_product(*leaves, offsets.long(), order, activation)
        output.backward(grad)
        assert same(output.detach(), mops_amd.gated_grouped_product(A, W, offsets, order, activation))
        expected = mops_amd.gated_grouped_product_vjp(grad, A, W, offsets, order, activation)
        assert same(tuple(t.grad for t in leaves), expected)
    # without an order, the default activation, one input recorded
    leaf = W.clone().requires_grad_(True)
    ops.gated_grouped_product(A, leaf, offsets).backward(grad)
    assert same(leaf.grad, mops_amd.gated_grouped_product_vjp(grad, A, W, offsets)[1])

    leaves = [A.clone().requires_grad_(True), classes.clone().requires_grad_(True)]
    losses, log_sums = ops.linear_cross_entropy(*leaves, targets.long())
    assert same((losses.detach(), log_sums.detach()), mops_amd.linear_cross_entropy(A, classes, targets))
    grads = rand(50, dtype=wide), rand(50, dtype=wide)
    torch.autograd.backward([losses, log_sums], grads)
    expected = mops_amd.linear_cross_entropy_vjp(*grads, A, classes, targets, log_sums.detach())
    assert same(tuple(t.grad for t in leaves), expected)
    leaf = classes.clone().requires_grad_(True)
    ops.linear_cross_entropy(A, leaf, targets)[0].sum().backward()  # (the gradient of a sum: expanded, of no strides)
    ones = torch.ones(50, dtype=wide, device=device)
    assert same(leaf.grad, mops_amd.linear_cross_entropy_vjp(ones, None, A, classes, targets, log_sums.detach())[1])

    gradients = [A, W, classes.t(), A[:, ::2]]
    assert same(ops.gradient_norm(gradients), mops_amd.gradient_norm(gradients))
    clipped, norm = ops.clip_gradients(gradients, 2.0)
    expected, expected_norm = mops_amd.clip_gradients(gradients, 2.0)
    assert same((*clipped, norm), (*expected, expected_norm))
    copies = [A.clone(), classes.t().clone()]
    expected, expected_norm = mops_amd.clip_gradients(copies, 2.0)
    versions = [c._version for c in copies]
    assert same((ops.clip_gradients_(copies, 2.0), *copies), (expected_norm, *expected))
    assert all(c._version > version for c, version in zip(copies, versions))


@pytest.mark.gpu
def test_operators_without_derivatives_say_so(device):
    ops, generator = operators(), generator_of(23)

    def rand(*shape):
        return random(generator, shape, torch.float32).to(device).requires_grad_(True)

    index = indices_of("uniform", 20, 3).to(device)
    order, offsets = ops.order_by_group(index, 3)
    A, W, classes = rand(20, 8), rand(3, 8, 10), rand(11, 8)
    (grad,) = torch.autograd.grad(ops.gated_grouped_product(A, W, offsets, order).sum(), A, create_graph=True)
    with pytest.raises(RuntimeError, match="gated_grouped_product: second derivatives are not supported"):
        grad.sum().backward()
    (grad,) = torch.autograd.grad(ops.linear_cross_entropy(A, classes, index)[0].sum(), A, create_graph=True)
    with pytest.raises(RuntimeError, match="linear_cross_entropy: second derivatives are not supported"):
        grad.sum().backward()
    for call in (ops.gradient_norm, lambda g: ops.clip_gradients(g, 1.0), lambda g: ops.clip_gradients_(g, 1.0)):
        with pytest.raises(RuntimeError, match="derivatives are not supported"):
            call([A])
    with pytest.raises((RuntimeError, ValueError), match="activation"):
        ops.gated_grouped_product(A.detach(), W.detach(), offsets, order, "relu")


@pytest.mark.gpu
def test_operators_on_gradients_of_inference_mode(device, monkeypatch):
    """Outside of inference mode they can be read, not changed: an error in front of the launches, on every path; inside they
    can."""
    from mops_amd import _c_lib

    def in_place(gradients):
        return mops_amd.clip_gradients_(gradients, 1.0)

    def by_operator(gradients):
        return operators().clip_gradients_(gradients, 1.0)

    with torch.inference_mode():
        made = torch.full((4,), 2.0, device=device)
    ordinary = torch.full((9,), 3.0, device=device)
    for path in ("native", "ctypes"):
        if path == "ctypes":
            monkeypatch.setattr(training, "_native", _c_lib._NoFunctions())
        for call in (in_place, by_operator):
            for gradients in ([made], [ordinary, made]):
                with pytest.raises((RuntimeError, ValueError), match="made in inference mode"):
                    call(gradients)
            assert made.eq(2).all() and ordinary.eq(3).all() and ordinary._version == 0, path
        clipped, norm = mops_amd.clip_gradients([made, ordinary], 1.0)
        assert abs(norm.item() - math.sqrt(97)) < 1e-5 and abs(exact_norm(clipped) - 1) < 1e-5
        with torch.inference_mode():
            for call in (in_place, by_operator):
                inside, ordinary_inside = made.clone(), ordinary.clone()
                assert abs(call([inside, ordinary_inside]).item() - math.sqrt(97)) < 1e-5
                assert torch.equal(inside, clipped[0]) and torch.equal(ordinary_inside, clipped[1])
    versions = ordinary._version
    in_place([ordinary])
    assert ordinary._version > versions


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
        [sys.executable, "-m", "pytest", os.path.join(root, "tests", "test_training.py"), "-q", "-x", "-k", "operator",
         "-p", "no:cacheprovider"],
        cwd=root, env=dict(os.environ, MOPS_AMD_TORCH_PYTHON_OPS="1"), capture_output=True, text=True,
    )  # fmt: skip
    assert done.returncode == 0, done.stdout[-3000:] + done.stderr[-2000:]
    assert " passed" in done.stdout


# ------------------------------------------------------ a step of training ----
class PlainOperators:
    """The operators of a step in elementary torch operations."""

    @staticmethod
    def scaled_embedding(table, indices, scale):
        inside = indices >= 0
        return torch.where(inside[:, None], table[torch.where(inside, indices, 0).long()] * scale, 0.0)

    @staticmethod
    def grouped_matrix_product(A, W, offsets, order):
        output = torch.zeros(A.shape[0], W.shape[2], dtype=A.dtype, device=A.device)
        for g in range(W.shape[0]):
            rows = order[int(offsets[g]) : int(offsets[g + 1])].long()
            output = output.index_add(0, rows, A[rows] @ W[g])
        return output

    @staticmethod
    def gated_grouped_product(A, W, offsets, order, activation):
        gate, up = PlainOperators.grouped_matrix_product(A, W, offsets, order).chunk(2, 1)
        inside = PlainOperators.grouped_matrix_product(torch.ones_like(A), torch.ones_like(W), offsets, order)[:, :1] != 0
        return torch.where(inside, torch.nn.functional.silu(gate) * up, 0.0)

    @staticmethod
    def gated_residual_norm(residual, block, gate, weight_block, weight_next, scale, epsilon):
        def norm(x):
            return x / torch.sqrt((x**2).mean(1, keepdim=True) + epsilon)

        state = residual + scale * gate * norm(block) * weight_block
        return state, norm(state) * weight_next

    @staticmethod
    def linear_cross_entropy(A, W, targets):
        logits = A @ W.t()
        log_sums = torch.logsumexp(logits, 1)
        kept = (targets >= 0) & (targets < W.shape[0])
        losses = log_sums - logits.gather(1, torch.where(kept, targets, 0).long()[:, None]).squeeze(1)
        return torch.where(kept, losses, 0.0), torch.where(kept, log_sums, 0.0)

    @staticmethod
    def clip_gradients(gradients, max_norm):
        norm = torch.sqrt(sum((g**2).sum() for g in gradients))
        return [g * torch.clamp(max_norm / norm, max=1.0) for g in gradients], norm


def training_step(ops, p, tokens, targets, groups, experts):
    """Loss, gradients and their norm: embedding, two feed-forward blocks by group, the embedding's table as classes."""
    order, offsets = groups
    state = ops.scaled_embedding(p["table"], tokens, 4.0)
    features = state
    for layer in range(2):
        hidden = ops.gated_grouped_product(features, p[f"in{layer}"], offsets, order, "silu")
        block = ops.grouped_matrix_product(hidden, p[f"out{layer}"], offsets, order)
        state, features = ops.gated_residual_norm(
            state, block, p[f"gate{layer}"], p[f"weight_block{layer}"], p[f"weight_next{layer}"], 0.5, 1e-6
        )
    losses, log_sums = ops.linear_cross_entropy(features, p["table"], targets)
    loss = losses.mean() + 1e-3 * (log_sums**2).mean()
    gradients = torch.autograd.grad(loss, list(p.values()))
    clipped, norm = ops.clip_gradients(list(gradients), 0.1)
    return loss.detach(), norm, clipped


@pytest.mark.gpu
def test_a_step_of_training(device):
    """The operators together, in float64 against elementary torch operations (rounding errors of some 1e4 terms, 1e-16
    each, grow through the layers; held to 1e-10 of each result's largest value); eager and captured."""
    rows, tokens_known, width, hidden, experts = 150, 61, 18, 23, 4
    generator = generator_of(31)

    def rand(*shape, scale=1.0, mean=0.0):
        return (random(generator, shape, torch.float64, scale) + mean).to(device).requires_grad_(True)

    p = {"table": rand(tokens_known, width, scale=0.3)}
    for layer in range(2):
        p[f"in{layer}"] = rand(experts, width, 2 * hidden, scale=width**-0.5)
        p[f"out{layer}"] = rand(experts, hidden, width, scale=hidden**-0.5)
        p[f"gate{layer}"] = rand(1, width, scale=0.1, mean=0.5)
        p[f"weight_block{layer}"] = rand(width, scale=0.1, mean=1.0)
        p[f"weight_next{layer}"] = rand(width, scale=0.1, mean=1.0)
    tokens, targets = indices_of("frequent", rows, tokens_known).to(device), indices_of("padded", rows, tokens_known).to(device)
    groups = mops_amd.order_by_group(indices_of("padded", rows, experts, 3).to(device), experts)
    ops = operators()
    actual = training_step(ops, p, tokens, targets, groups, experts)
    expected = training_step(PlainOperators, p, tokens, targets, groups, experts)
    for a, e in zip([*actual[:2], *actual[2]], [*expected[:2], *expected[2]], strict=True):
        assert (a - e).abs().max() <= 1e-10 * e.abs().max()
    # the whole step as a graph, replayed on other tokens with eager work in between
    fixed = tokens.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        training_step(ops, {n: t.detach().clone().requires_grad_(True) for n, t in p.items()}, fixed, targets, groups, experts)
    torch.cuda.synchronize()
    leaves = {n: t.detach().clone().requires_grad_(True) for n, t in p.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = training_step(ops, leaves, fixed, targets, groups, experts)
    for seed in range(4):
        fixed.copy_(indices_of("frequent", rows, tokens_known, seed).to(device))
        graph.replay()
        torch.cuda.synchronize()
        eager = training_step(ops, p, fixed.clone(), targets, groups, experts)
        for a, e in zip(captured[2], eager[2], strict=True):
            assert (a - e).abs().max() <= 1e-12 * e.abs().max()
        torch.cuda.synchronize()
