"""Registration of ``torch.ops.mops.*`` from Python, over the C ABI.

Used by ``mops_amd.torch`` when the C++ operators (``mops_amd/csrc/torch_ops.cpp``) have not been
built, or when ``MOPS_AMD_TORCH_PYTHON_OPS=1`` asks for it. Same operators, schemas, gradients and
second derivatives; every call goes through the interpreter (and the backward passes through
``torch.library``'s Python autograd), which costs some hundred microseconds per forward + backward.
"""
import torch

from . import layers as _layers
from . import ops as _ops


_library = torch.library.Library("mops", "DEF")
_library.define("homogeneous_polynomial_evaluation(Tensor A, Tensor C, Tensor indices_A) -> Tensor")
_library.define(
    "outer_product_scatter_add(Tensor A, Tensor B, Tensor indices_output, int output_size) -> Tensor"
)
_library.define(
    "sparse_accumulation_of_products(Tensor A, Tensor B, Tensor C, Tensor indices_A, Tensor indices_B, "
    "Tensor indices_output, int output_size) -> Tensor"
)
_library.define(
    "outer_product_scatter_add_with_weights(Tensor A, Tensor B, Tensor W, Tensor indices_W, "
    "Tensor indices_output) -> Tensor"
)
_library.define(
    "sparse_accumulation_scatter_add_with_weights(Tensor A, Tensor B, Tensor C, Tensor W, Tensor indices_A, "
    "Tensor indices_W_1, Tensor indices_W_2, Tensor indices_output_1, Tensor indices_output_2, "
    "int output_size) -> Tensor"
)
# the vector-Jacobian products, as operators of their own so that the
# backward pass is a dispatcher call as well (bool[] mask: which gradients)
_library.define(
    "homogeneous_polynomial_evaluation_vjp(Tensor grad_output, Tensor A, Tensor C, Tensor indices_A) -> Tensor"
)
_library.define(
    "outer_product_scatter_add_vjp(Tensor grad_output, Tensor A, Tensor B, Tensor indices_output, "
    "bool[2] wanted) -> (Tensor, Tensor)"
)
_library.define(
    "sparse_accumulation_of_products_vjp(Tensor grad_output, Tensor A, Tensor B, Tensor C, Tensor indices_A, "
    "Tensor indices_B, Tensor indices_output, bool[2] wanted) -> (Tensor, Tensor)"
)
_library.define(
    "outer_product_scatter_add_with_weights_vjp(Tensor grad_output, Tensor A, Tensor B, Tensor W, "
    "Tensor indices_W, Tensor indices_output, bool[3] wanted) -> (Tensor, Tensor, Tensor)"
)
_library.define(
    "sparse_accumulation_scatter_add_with_weights_vjp(Tensor grad_output, Tensor A, Tensor B, Tensor C, "
    "Tensor W, Tensor indices_A, Tensor indices_W_1, Tensor indices_W_2, Tensor indices_output_1, "
    "Tensor indices_output_2, bool[3] wanted) -> (Tensor, Tensor, Tensor)"
)
# second order: cotangents of the vjp's outputs in, cotangents of its inputs out;
# `have`: which cotangents are given (the others are empty tensors), `wanted`:
# which of (grad_grad_output, grad_A_2[, grad_B_2]) are computed
_library.define(
    "homogeneous_polynomial_evaluation_vjp_vjp(Tensor grad_grad_A, Tensor grad_output, Tensor A, Tensor C, "
    "Tensor indices_A, bool[2] wanted) -> (Tensor, Tensor)"
)
_library.define(
    "outer_product_scatter_add_vjp_vjp(Tensor grad_grad_A, Tensor grad_grad_B, Tensor grad_output, Tensor A, "
    "Tensor B, Tensor indices_output, bool[2] have, bool[3] wanted) -> (Tensor, Tensor, Tensor)"
)
_library.define(
    "sparse_accumulation_of_products_vjp_vjp(Tensor grad_grad_A, Tensor grad_grad_B, Tensor grad_output, "
    "Tensor A, Tensor B, Tensor C, Tensor indices_A, Tensor indices_B, Tensor indices_output, bool[2] have, "
    "bool[3] wanted) -> (Tensor, Tensor, Tensor)"
)


def _or_empty(gradient, like):
    """Operators cannot return None: a gradient that was not asked for is an empty tensor."""
    return gradient if gradient is not None else like.new_empty((0,))


# ----------------------------------------------------------------- kernels --
def _hpe(A, C, indices_A):
    return _ops.homogeneous_polynomial_evaluation(A, C, indices_A)


def _hpe_vjp(grad_output, A, C, indices_A):
    return _ops.homogeneous_polynomial_evaluation_vjp(grad_output, A, C, indices_A)


def _hpe_vjp_vjp(grad_grad_A, grad_output, A, C, indices_A, wanted):
    grad_grad_output, grad_A_2 = _ops.homogeneous_polynomial_evaluation_vjp_vjp(
        grad_grad_A, grad_output, A, C, indices_A,
        compute_grad_grad_output=wanted[0], compute_grad_A_2=wanted[1],
    )  # fmt: skip
    return _or_empty(grad_grad_output, A), _or_empty(grad_A_2, A)


def _opsa_vjp_vjp(grad_grad_A, grad_grad_B, grad_output, A, B, indices_output, have, wanted):
    grad_grad_output, grad_A_2, grad_B_2 = _ops.outer_product_scatter_add_vjp_vjp(
        grad_grad_A if have[0] else None, grad_grad_B if have[1] else None, grad_output, A, B, indices_output,
        compute_grad_grad_output=wanted[0], compute_grad_A_2=wanted[1], compute_grad_B_2=wanted[2],
    )  # fmt: skip
    return _or_empty(grad_grad_output, A), _or_empty(grad_A_2, A), _or_empty(grad_B_2, B)


def _sap_vjp_vjp(
    grad_grad_A, grad_grad_B, grad_output, A, B, C, indices_A, indices_B, indices_output, have, wanted
):
    grad_grad_output, grad_A_2, grad_B_2 = _ops.sparse_accumulation_of_products_vjp_vjp(
        grad_grad_A if have[0] else None, grad_grad_B if have[1] else None, grad_output, A, B, C,
        indices_A, indices_B, indices_output,
        compute_grad_grad_output=wanted[0], compute_grad_A_2=wanted[1], compute_grad_B_2=wanted[2],
    )  # fmt: skip
    return _or_empty(grad_grad_output, A), _or_empty(grad_A_2, A), _or_empty(grad_B_2, B)


def _opsa(A, B, indices_output, output_size):
    return _ops.outer_product_scatter_add(A, B, indices_output, output_size)


def _opsa_vjp(grad_output, A, B, indices_output, wanted):
    grad_A, grad_B = _ops.outer_product_scatter_add_vjp(
        grad_output, A, B, indices_output, compute_grad_A=wanted[0], compute_grad_B=wanted[1]
    )
    return _or_empty(grad_A, A), _or_empty(grad_B, B)


def _sap(A, B, C, indices_A, indices_B, indices_output, output_size):
    return _ops.sparse_accumulation_of_products(A, B, C, indices_A, indices_B, indices_output, output_size)


def _sap_vjp(grad_output, A, B, C, indices_A, indices_B, indices_output, wanted):
    grad_A, grad_B = _ops.sparse_accumulation_of_products_vjp(
        grad_output, A, B, C, indices_A, indices_B, indices_output,
        compute_grad_A=wanted[0], compute_grad_B=wanted[1],
    )  # fmt: skip
    return _or_empty(grad_A, A), _or_empty(grad_B, B)


def _opsaw(A, B, W, indices_W, indices_output):
    return _ops.outer_product_scatter_add_with_weights(A, B, W, indices_W, indices_output)


def _opsaw_vjp(grad_output, A, B, W, indices_W, indices_output, wanted):
    grad_A, grad_B, grad_W = _ops.outer_product_scatter_add_with_weights_vjp(
        grad_output, A, B, W, indices_W, indices_output,
        compute_grad_A=wanted[0], compute_grad_B=wanted[1], compute_grad_W=wanted[2],
    )  # fmt: skip
    return _or_empty(grad_A, A), _or_empty(grad_B, B), _or_empty(grad_W, W)


def _sasaw(A, B, C, W, indices_A, indices_W_1, indices_W_2, indices_output_1, indices_output_2, output_size):
    return _ops.sparse_accumulation_scatter_add_with_weights(
        A, B, C, W, indices_A, indices_W_1, indices_W_2, indices_output_1, indices_output_2, output_size
    )


def _sasaw_vjp(
    grad_output, A, B, C, W, indices_A, indices_W_1, indices_W_2, indices_output_1, indices_output_2, wanted
):
    grad_A, grad_B, grad_W = _ops.sparse_accumulation_scatter_add_with_weights_vjp(
        grad_output, A, B, C, W, indices_A, indices_W_1, indices_W_2, indices_output_1, indices_output_2,
        compute_grad_A=wanted[0], compute_grad_B=wanted[1], compute_grad_W=wanted[2],
    )  # fmt: skip
    return _or_empty(grad_A, A), _or_empty(grad_B, B), _or_empty(grad_W, W)


for _name, _kernel in [
    ("homogeneous_polynomial_evaluation", _hpe),
    ("homogeneous_polynomial_evaluation_vjp", _hpe_vjp),
    ("outer_product_scatter_add", _opsa),
    ("outer_product_scatter_add_vjp", _opsa_vjp),
    ("sparse_accumulation_of_products", _sap),
    ("sparse_accumulation_of_products_vjp", _sap_vjp),
    ("outer_product_scatter_add_with_weights", _opsaw),
    ("outer_product_scatter_add_with_weights_vjp", _opsaw_vjp),
    ("sparse_accumulation_scatter_add_with_weights", _sasaw),
    ("sparse_accumulation_scatter_add_with_weights_vjp", _sasaw_vjp),
    ("homogeneous_polynomial_evaluation_vjp_vjp", _hpe_vjp_vjp),
    ("outer_product_scatter_add_vjp_vjp", _opsa_vjp_vjp),
    ("sparse_accumulation_of_products_vjp_vjp", _sap_vjp_vjp),
]:
    # ROCm tensors carry the CUDA dispatch key
    _library.impl(_name, _kernel, "CUDA")


def _refuse_host(name):
    def kernel(*args):
        raise RuntimeError(
            f"mops::{name}: tensors must be on a ROCm device; this library implements the device path only"
        )

    return kernel


for _name in [
    "homogeneous_polynomial_evaluation",
    "outer_product_scatter_add",
    "sparse_accumulation_of_products",
    "outer_product_scatter_add_with_weights",
    "sparse_accumulation_scatter_add_with_weights",
]:
    _library.impl(_name, _refuse_host(_name), "CPU")
    _library.impl(_name + "_vjp", _refuse_host(_name + "_vjp"), "CPU")
for _name in [
    "homogeneous_polynomial_evaluation_vjp_vjp",
    "outer_product_scatter_add_vjp_vjp",
    "sparse_accumulation_of_products_vjp_vjp",
]:
    _library.impl(_name, _refuse_host(_name), "CPU")


# ------------------------------------------------------------------ shapes --
# (FakeTensor / torch.compile support: output shapes without running anything)
def _register_fake(name, function):
    torch.library.register_fake(f"mops::{name}", function, lib=_library)


_register_fake("homogeneous_polynomial_evaluation", lambda A, C, indices_A: A.new_empty((A.shape[0],)))
_register_fake(
    "outer_product_scatter_add",
    lambda A, B, indices_output, output_size: A.new_empty((output_size, A.shape[1], B.shape[1])),
)
_register_fake(
    "sparse_accumulation_of_products",
    lambda A, B, C, indices_A, indices_B, indices_output, output_size: A.new_empty((A.shape[0], output_size)),
)
_register_fake(
    "outer_product_scatter_add_with_weights",
    lambda A, B, W, indices_W, indices_output: A.new_empty((W.shape[0], A.shape[1], B.shape[1])),
)
_register_fake(
    "sparse_accumulation_scatter_add_with_weights",
    lambda A, B, C, W, indices_A, indices_W_1, indices_W_2, indices_output_1, indices_output_2, output_size: (
        A.new_empty((W.shape[0], output_size, B.shape[1]))
    ),
)


# ---------------------------------------------------------------- autograd --
def _hpe_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _hpe_backward(ctx, grad_output):
    A, C, indices_A = ctx.saved_tensors
    grad_A = None
    if ctx.needs_input_grad[0]:
        grad_A = torch.ops.mops.homogeneous_polynomial_evaluation_vjp(
            grad_output.contiguous(), A, C, indices_A
        )
    if ctx.needs_input_grad[1]:
        raise RuntimeError("gradients with respect to C are not supported")
    return grad_A, None, None


def _opsa_setup(ctx, inputs, output):
    A, B, indices_output, _ = inputs
    ctx.save_for_backward(A, B, indices_output)


def _opsa_backward(ctx, grad_output):
    A, B, indices_output = ctx.saved_tensors
    wanted = [ctx.needs_input_grad[0], ctx.needs_input_grad[1]]
    grad_A, grad_B = torch.ops.mops.outer_product_scatter_add_vjp(
        grad_output.contiguous(), A, B, indices_output, wanted
    )
    return grad_A if wanted[0] else None, grad_B if wanted[1] else None, None, None


def _sap_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:6])


def _sap_backward(ctx, grad_output):
    A, B, C, indices_A, indices_B, indices_output = ctx.saved_tensors
    if ctx.needs_input_grad[2]:
        raise RuntimeError("gradients with respect to C are not supported")
    wanted = [ctx.needs_input_grad[0], ctx.needs_input_grad[1]]
    grad_A, grad_B = torch.ops.mops.sparse_accumulation_of_products_vjp(
        grad_output.contiguous(), A, B, C, indices_A, indices_B, indices_output, wanted
    )
    return (grad_A if wanted[0] else None, grad_B if wanted[1] else None, None, None, None, None, None)


def _opsaw_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _opsaw_backward(ctx, grad_output):
    A, B, W, indices_W, indices_output = ctx.saved_tensors
    wanted = [ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[2]]
    grad_A, grad_B, grad_W = torch.ops.mops.outer_product_scatter_add_with_weights_vjp(
        grad_output.contiguous(), A, B, W, indices_W, indices_output, wanted
    )
    return (
        grad_A if wanted[0] else None, grad_B if wanted[1] else None, grad_W if wanted[2] else None,
        None, None,
    )  # fmt: skip


def _sasaw_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:9])


def _sasaw_backward(ctx, grad_output):
    A, B, C, W, indices_A, indices_W_1, indices_W_2, indices_output_1, indices_output_2 = ctx.saved_tensors
    if ctx.needs_input_grad[2]:
        raise RuntimeError("gradients with respect to C are not supported")
    wanted = [ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[3]]
    grad_A, grad_B, grad_W = torch.ops.mops.sparse_accumulation_scatter_add_with_weights_vjp(
        grad_output.contiguous(), A, B, C, W, indices_A, indices_W_1, indices_W_2, indices_output_1,
        indices_output_2, wanted,
    )  # fmt: skip
    return (
        grad_A if wanted[0] else None, grad_B if wanted[1] else None, None, grad_W if wanted[2] else None,
        None, None, None, None, None, None,
    )  # fmt: skip


# ---- second order: backward of the *_vjp operators of HPE, OPSA and SAP ----
def _given(cotangent, wanted):
    """A cotangent counts when its output was computed and autograd passes one."""
    return bool(wanted) and cotangent is not None


def _hpe_vjp_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _hpe_vjp_backward(ctx, grad_grad_A):
    grad_output, A, C, indices_A = ctx.saved_tensors
    if ctx.needs_input_grad[2]:
        raise RuntimeError("gradients with respect to C are not supported")
    wanted = [ctx.needs_input_grad[0], ctx.needs_input_grad[1]]
    grad_grad_output, grad_A_2 = torch.ops.mops.homogeneous_polynomial_evaluation_vjp_vjp(
        grad_grad_A.contiguous(), grad_output, A, C, indices_A, wanted
    )
    return grad_grad_output if wanted[0] else None, grad_A_2 if wanted[1] else None, None, None


def _opsa_vjp_setup(ctx, inputs, output):
    grad_output, A, B, indices_output, wanted = inputs
    ctx.save_for_backward(grad_output, A, B, indices_output)
    ctx.computed = list(wanted)


def _opsa_vjp_backward(ctx, grad_grad_A, grad_grad_B):
    grad_output, A, B, indices_output = ctx.saved_tensors
    have = [_given(grad_grad_A, ctx.computed[0]), _given(grad_grad_B, ctx.computed[1])]
    wanted = [ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[2]]
    grad_grad_output, grad_A_2, grad_B_2 = torch.ops.mops.outer_product_scatter_add_vjp_vjp(
        grad_grad_A.contiguous() if have[0] else A.new_empty((0,)),
        grad_grad_B.contiguous() if have[1] else B.new_empty((0,)),
        grad_output, A, B, indices_output, have, wanted,
    )  # fmt: skip
    return (
        grad_grad_output if wanted[0] else None, grad_A_2 if wanted[1] else None,
        grad_B_2 if wanted[2] else None, None, None,
    )  # fmt: skip


def _sap_vjp_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:7])
    ctx.computed = list(inputs[7])


def _sap_vjp_backward(ctx, grad_grad_A, grad_grad_B):
    grad_output, A, B, C, indices_A, indices_B, indices_output = ctx.saved_tensors
    if ctx.needs_input_grad[3]:
        raise RuntimeError("gradients with respect to C are not supported")
    have = [_given(grad_grad_A, ctx.computed[0]), _given(grad_grad_B, ctx.computed[1])]
    wanted = [ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[2]]
    grad_grad_output, grad_A_2, grad_B_2 = torch.ops.mops.sparse_accumulation_of_products_vjp_vjp(
        grad_grad_A.contiguous() if have[0] else A.new_empty((0,)),
        grad_grad_B.contiguous() if have[1] else B.new_empty((0,)),
        grad_output, A, B, C, indices_A, indices_B, indices_output, have, wanted,
    )  # fmt: skip
    return (
        grad_grad_output if wanted[0] else None, grad_A_2 if wanted[1] else None,
        grad_B_2 if wanted[2] else None, None, None, None, None, None,
    )  # fmt: skip


for _name, _backward, _setup in [
    ("homogeneous_polynomial_evaluation_vjp", _hpe_vjp_backward, _hpe_vjp_setup),
    ("outer_product_scatter_add_vjp", _opsa_vjp_backward, _opsa_vjp_setup),
    ("sparse_accumulation_of_products_vjp", _sap_vjp_backward, _sap_vjp_setup),
    ("homogeneous_polynomial_evaluation", _hpe_backward, _hpe_setup),
    ("outer_product_scatter_add", _opsa_backward, _opsa_setup),
    ("sparse_accumulation_of_products", _sap_backward, _sap_setup),
    ("outer_product_scatter_add_with_weights", _opsaw_backward, _opsaw_setup),
    ("sparse_accumulation_scatter_add_with_weights", _sasaw_backward, _sasaw_setup),
]:
    torch.library.register_autograd(f"mops::{_name}", _backward, setup_context=_setup, lib=_library)




# ------------------------------------------------------ layers' operators --
_library.define("order_by_group(Tensor indices, int n_groups) -> (Tensor, Tensor)")
_library.define("scaled_embedding(Tensor table, Tensor indices, float scale=1.) -> Tensor")
_library.define("grouped_matrix_product(Tensor A, Tensor W, Tensor offsets, Tensor? order=None) -> Tensor")
_library.define(
    "gated_residual_norm(Tensor residual, Tensor block, Tensor gate, Tensor weight_block, Tensor weight_next, "
    "float residual_scale=1., float epsilon=1e-06) -> (Tensor, Tensor)"
)
_library.define("scaled_embedding_vjp(Tensor grad_output, Tensor table, Tensor indices, float scale) -> Tensor")
_library.define(
    "grouped_matrix_product_vjp(Tensor grad_output, Tensor A, Tensor W, Tensor offsets, Tensor? order, "
    "bool[2] wanted) -> (Tensor, Tensor)"
)
_library.define(
    "gated_residual_norm_vjp(Tensor? grad_state, Tensor? grad_next, Tensor residual, Tensor block, Tensor gate, "
    "Tensor weight_block, Tensor weight_next, float residual_scale, float epsilon, bool[5] wanted) "
    "-> (Tensor, Tensor, Tensor, Tensor, Tensor)"
)


def _grouped(A, W, offsets, order=None):
    return _layers.grouped_matrix_product(A, W, offsets, order)


def _update(residual, block, gate, weight_block, weight_next, residual_scale=1.0, epsilon=1e-6):
    return _layers.gated_residual_norm(residual, block, gate, weight_block, weight_next, residual_scale, epsilon)


def _grouped_vjp(grad_output, A, W, offsets, order, wanted):
    grad_A, grad_W = _layers.grouped_matrix_product_vjp(grad_output, A, W, offsets, order, *wanted)
    return _or_empty(grad_A, A), _or_empty(grad_W, W)


def _update_vjp(grad_state, grad_next, *arguments):
    *arguments, wanted = arguments
    grads = _layers.gated_residual_norm_vjp(grad_state, grad_next, *arguments, *wanted)
    return tuple(_or_empty(grad, arguments[0]) for grad in grads)


for _name, _kernel in [
    ("order_by_group", _layers.order_by_group),
    ("scaled_embedding", lambda table, indices, scale=1.0: _layers.scaled_embedding(table, indices, scale)),
    ("grouped_matrix_product", _grouped),
    ("gated_residual_norm", _update),
    ("scaled_embedding_vjp", _layers.scaled_embedding_vjp),
    ("grouped_matrix_product_vjp", _grouped_vjp),
    ("gated_residual_norm_vjp", _update_vjp),
]:
    _library.impl(_name, _kernel, "CUDA")
    _library.impl(_name, _refuse_host(_name), "CPU")

_register_fake(
    "order_by_group",
    lambda indices, n_groups: (
        indices.new_empty(indices.shape, dtype=torch.int32), indices.new_empty((n_groups + 1,), dtype=torch.int32),
    ),
)  # fmt: skip
_register_fake(
    "scaled_embedding", lambda table, indices, scale=1.0: table.new_empty((indices.shape[0], table.shape[1]))
)
_register_fake(
    "grouped_matrix_product", lambda A, W, offsets, order=None: A.new_empty((A.shape[0], W.shape[2]))
)
_register_fake(
    "gated_residual_norm",
    lambda residual, block, gate, weight_block, weight_next, residual_scale=1.0, epsilon=1e-6: (
        residual.new_empty(residual.shape), residual.new_empty(residual.shape),
    ),
)  # fmt: skip


def _embedding_setup(ctx, inputs, output):
    table, indices, ctx.scale = inputs
    ctx.save_for_backward(table, indices)


def _embedding_backward(ctx, grad_output):
    table, indices = ctx.saved_tensors
    return torch.ops.mops.scaled_embedding_vjp(grad_output.contiguous(), table, indices, ctx.scale), None, None


def _embedding_vjp_setup(ctx, inputs, output):
    _, _, indices, ctx.scale = inputs
    ctx.save_for_backward(indices)


def _embedding_vjp_backward(ctx, grad_table):
    (indices,) = ctx.saved_tensors
    return torch.ops.mops.scaled_embedding(grad_table.contiguous(), indices, ctx.scale), None, None, None


def _grouped_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _grouped_backward(ctx, grad_output):
    wanted = list(ctx.needs_input_grad[:2])
    grads = torch.ops.mops.grouped_matrix_product_vjp(grad_output.contiguous(), *ctx.saved_tensors, wanted)
    return (*(grad if want else None for grad, want in zip(grads, wanted)), None, None)


def _grouped_vjp_setup(ctx, inputs, output):
    *tensors, ctx.computed = inputs
    ctx.save_for_backward(*tensors)
    ctx.set_materialize_grads(False)


def _grouped_vjp_backward(ctx, u, v):
    """With c = grad_output, by group: grad_A = c W^T and grad_W = A^T c."""
    grad_output, A, W, offsets, order = ctx.saved_tensors
    u, v = [x.contiguous() if _given(x, computed) else None for x, computed in zip((u, v), ctx.computed)]
    product, vjp = torch.ops.mops.grouped_matrix_product, torch.ops.mops.grouped_matrix_product_vjp
    grads = [None, None, None]
    if ctx.needs_input_grad[0]:
        parts = [product(a, w, offsets, order) for a, w in ((u, W), (A, v)) if a is not None and w is not None]
        grads[0] = sum(parts[1:], parts[0]) if parts else None
    if ctx.needs_input_grad[1] and v is not None:
        grads[1] = vjp(grad_output, A, v, offsets, order, [True, False])[0]
    if ctx.needs_input_grad[2] and u is not None:
        grads[2] = vjp(grad_output, u, W, offsets, order, [False, True])[1]
    return (*grads, None, None, None)


def _update_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:5])
    ctx.residual_scale, ctx.epsilon = inputs[5:]
    ctx.set_materialize_grads(False)


def _update_backward(ctx, grad_state, grad_next):
    wanted = list(ctx.needs_input_grad[:5])
    cotangents = [None if grad is None else grad.contiguous() for grad in (grad_state, grad_next)]
    grads = torch.ops.mops.gated_residual_norm_vjp(
        *cotangents, *ctx.saved_tensors, ctx.residual_scale, ctx.epsilon, wanted
    )
    return (*(grad if want else None for grad, want in zip(grads, wanted)), None, None)


def _update_vjp_setup(ctx, inputs, output):
    pass


def _update_vjp_backward(ctx, *grads):
    raise RuntimeError("mops::gated_residual_norm: second derivatives are not supported")


for _name, _backward, _setup in [
    ("scaled_embedding_vjp", _embedding_vjp_backward, _embedding_vjp_setup),
    ("grouped_matrix_product_vjp", _grouped_vjp_backward, _grouped_vjp_setup),
    ("gated_residual_norm_vjp", _update_vjp_backward, _update_vjp_setup),
    ("scaled_embedding", _embedding_backward, _embedding_setup),
    ("grouped_matrix_product", _grouped_backward, _grouped_setup),
    ("gated_residual_norm", _update_backward, _update_setup),
]:
    torch.library.register_autograd(f"mops::{_name}", _backward, setup_context=_setup, lib=_library)
