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
