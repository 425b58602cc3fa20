"""torch.ops.mops.{scaled_embedding, grouped_matrix_product, gated_residual_norm} in networks: arguments left out, and
derivatives of their gradients, which a network that is trained on forces needs."""
import os
import subprocess
import sys

import pytest
import torch

import mops_amd
import mops_amd.torch  # noqa: F401  (registers torch.ops.mops.*)
from tests.test_layers import indices_of, random

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROWS, GROUPS, K, L = 40, 6, 9, 13


class Plain:
    """The same operators in elementary operations."""

    @staticmethod
    def scaled_embedding(table, index, scale=1.0):
        inside = (index >= 0) & (index < len(table))
        return torch.where(inside[:, None], scale * table[index.clamp(0, len(table) - 1).long()], 0)

    @staticmethod
    def grouped_matrix_product(A, W, offsets, order=None):
        order = torch.arange(len(A), device=A.device) if order is None else order.long()
        place = torch.empty_like(order)
        place[order] = torch.arange(len(A), device=A.device)
        group = torch.searchsorted(offsets.long(), place, right=True) - 1
        inside = (group >= 0) & (group < len(W))
        return torch.where(inside[:, None], (A[:, :, None] * W[group.clamp(0, len(W) - 1)]).sum(1), 0)


def case(device, dtype=torch.float64, seed=3):
    generator = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return random(generator, shape, dtype).to(device).requires_grad_(True)

    index = indices_of("padded", ROWS, GROUPS).to(device)
    return rand, index, *mops_amd.order_by_group(index, GROUPS)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_operator_gradients_without_an_order(device, dtype):
    """Rows that lie in the order of their groups: no order, and gradients all the same."""
    rand, _, _, offsets = case(device, dtype)
    A, W, c = rand(ROWS, K), rand(GROUPS, K, L), rand(ROWS, L).detach()
    torch.ops.mops.grouped_matrix_product(A, W, offsets).backward(c)
    expected = mops_amd.grouped_matrix_product_vjp(c, A.detach(), W.detach(), offsets)
    assert torch.equal(A.grad, expected[0]) and torch.equal(W.grad, expected[1])
    (grad_W,) = torch.autograd.grad(torch.ops.mops.grouped_matrix_product(A.detach(), W, offsets, None), W, c)
    assert torch.equal(grad_W, expected[1])


@pytest.mark.gpu
@pytest.mark.parametrize("recorded", ["both", "rows", "matrices"])
def test_operator_second_derivatives(device, recorded):
    """Against differences of the first ones, for every argument that is recorded."""
    rand, index, order, offsets = case(device)
    ops = torch.ops.mops
    if recorded == "both":
        assert torch.autograd.gradgradcheck(lambda t: ops.scaled_embedding(t, index, 1.3), [rand(GROUPS, 11)])
    A, W = rand(ROWS, K), rand(GROUPS, K, L)
    A.requires_grad_(recorded != "matrices")
    W.requires_grad_(recorded != "rows")
    for plan in ((offsets, order), (offsets,)):
        assert torch.autograd.gradgradcheck(lambda a, w: ops.grouped_matrix_product(a, w, *plan), [A, W], fast_mode=True)


def forces(ops, x, table, W, readout, index, offsets, order):
    """A small network whose energy depends on x through a function of its own: the energy, and its gradient for x."""
    features = ops.scaled_embedding(table, index, 1.7) * torch.sin(x)
    hidden = torch.tanh(ops.grouped_matrix_product(features, W, offsets, order))
    energy = ops.grouped_matrix_product(hidden, readout, offsets, order).sum()
    return energy, torch.autograd.grad(energy, x, create_graph=True)[0]


@pytest.mark.gpu
def test_operator_training_on_forces(device):
    """The gradients of a loss on forces, and of a loss on the gradients of that, by plain PyTorch."""
    rand, index, order, offsets = case(device)
    inputs = [rand(ROWS, K), rand(GROUPS, K), rand(GROUPS, K, L), rand(GROUPS, L, 1)]
    results = []
    for ops in (torch.ops.mops, Plain):
        energy, force = forces(ops, *inputs, index, offsets, order)
        first = torch.autograd.grad(energy + (force**2).sum(), inputs, create_graph=True)
        second = torch.autograd.grad(sum((g**2).sum() for g in first), inputs)
        results.append([energy, force, *first, *second])
    for actual, expected in zip(*results):
        # (64 bits on both sides; a few hundred terms of sizes up to the largest)
        assert (actual - expected).abs().max() <= 1e-11 * expected.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_operator_second_derivatives_are_calls_of_the_operators(device, dtype):
    rand, index, order, offsets = case(device, dtype)
    A, W, c, u, v = rand(ROWS, K), rand(GROUPS, K, L), rand(ROWS, L), rand(ROWS, K), rand(GROUPS, K, L)
    output = torch.ops.mops.grouped_matrix_product(A, W, offsets, order)
    grads = torch.autograd.grad(output, [A, W], c, create_graph=True)
    second = torch.autograd.grad(grads, [c, A, W], [u, v])
    with torch.no_grad():
        product, vjp = mops_amd.grouped_matrix_product, mops_amd.grouped_matrix_product_vjp
        assert torch.equal(second[0], product(u, W, offsets, order) + product(A, v, offsets, order))
        assert torch.equal(second[1], vjp(c, A, v, offsets, order)[0])
        assert torch.equal(second[2], vjp(c, u, W, offsets, order)[1])
    table, c, u = rand(GROUPS, K), rand(ROWS, K), rand(GROUPS, K)
    (grad,) = torch.autograd.grad(torch.ops.mops.scaled_embedding(table, index, 0.7), table, c, create_graph=True)
    with torch.no_grad():
        expected = mops_amd.scaled_embedding(u, index, 0.7)
    assert torch.equal(torch.autograd.grad(grad, c, u)[0], expected)


@pytest.mark.gpu
@pytest.mark.parametrize("gate_rows", [1, ROWS])
def test_operator_without_second_derivative_says_so(device, gate_rows):
    """First derivatives of the residual update are the same where they are recorded; derivatives of them are an error,
    not a gradient with terms missing."""
    rand, *_ = case(device)
    inputs = [rand(ROWS, K), rand(ROWS, K), rand(gate_rows, K), rand(K), rand(K)]
    cotangents = [rand(ROWS, K), rand(ROWS, K)]

    def update():
        return torch.ops.mops.gated_residual_norm(*inputs, 0.4, 1e-5)

    plain = torch.autograd.grad(update(), inputs, [x.detach() for x in cotangents])
    recorded = torch.autograd.grad(update(), inputs, cotangents, create_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(plain, recorded, strict=True))
    (of_block,) = torch.autograd.grad(update()[1], inputs[1], cotangents[1].detach(), create_graph=True)
    # the gradient depends on the block as well as on what else is recorded
    for result, wanted in ((of_block, inputs[1]), (recorded[0], cotangents[0]), (recorded[3], inputs[0])):
        with pytest.raises(RuntimeError, match="second derivatives are not supported"):
            torch.autograd.grad(result.sum(), wanted, retain_graph=True)


@pytest.mark.gpu
def test_a_table_may_change_before_its_gradient(device):
    """The gradient of a lookup needs the table's shape only."""
    rand, index, *_ = case(device)
    table, c = rand(GROUPS, K), rand(ROWS, K)
    output = torch.ops.mops.scaled_embedding(table, index, 0.7)
    with torch.no_grad():
        table.zero_()
    (grad,) = torch.autograd.grad(output, table, c.detach())
    assert torch.equal(grad, mops_amd.scaled_embedding_vjp(c.detach(), table.detach(), index, 0.7))


@pytest.mark.gpu
def test_registered_from_python(device):
    """The same with the operators of mops_amd/_torch_python_ops.py, in a process of their own."""
    if os.environ.get("MOPS_AMD_TORCH_PYTHON_OPS", "0") not in ("", "0"):
        pytest.skip("this process already runs them")
    done = subprocess.run(
        [sys.executable, "-m", "pytest", os.path.abspath(__file__), "-q", "-x", "-k", "operator", "-p", "no:cacheprovider"],
        cwd=ROOT, env=dict(os.environ, MOPS_AMD_TORCH_PYTHON_OPS="1"), capture_output=True, text=True, timeout=110,
    )  # fmt: skip
    assert done.returncode == 0, done.stdout[-3000:] + done.stderr[-2000:]
    assert " passed" in done.stdout
