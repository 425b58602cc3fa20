"""The operators of a network's layers around the sums over edges.

A table looked up by an index, products with a matrix per group of rows, and the residual update around
a block with its two norms and its gate; each with its vector-Jacobian product. None of them exists in
lab-cosmo/mops. What each computes is written down in ``include/mops/layers.h``.

Tensors live on a ROCm device and are ``float32``, ``float64``, ``bfloat16`` or ``float16``, all of a
call of the same type; sums, norms and gradients are computed in 32 bits (64 for ``float64``) and
rounded once. As everywhere in this package inputs are made contiguous, indices are converted to
32 bits, outputs are allocated here, a gradient that is not asked for is ``None``, and the work is
enqueued on the current PyTorch stream without blocking the host.
"""
import ctypes

from . import _dispatch
from ._c_api import _make_struct
from ._c_lib import device_library
from .checks import check_array, check_scalar
from .ops import _native
from .status import MopsError

_TAGS = {"float32": "f32", "float64": "f64", "bfloat16": "bf16", "float16": "f16"}
_ELEMENT = {
    "f32": ctypes.c_float, "f64": ctypes.c_double, "bf16": ctypes.c_uint16, "f16": ctypes.c_uint16,
    "i32": ctypes.c_int32,
}  # fmt: skip
_STRUCTS = {
    (ndim, tag): _make_struct(f"mops_tensor_{ndim}d_{tag}_t", element, ndim)
    for tag, element in _ELEMENT.items()
    for ndim in (1, 2, 3)
}

#: function -> ((dimensions or "double", parameter), ...) in the order of the C prototype; a negative number of
#: dimensions is an index tensor
_SIGNATURES = {
    "order_by_group": ((-1, "order"), (-1, "offsets"), (-1, "indices")),
    "scaled_embedding": ((2, "output"), (2, "table"), (-1, "indices"), ("double", "scale")),
    "scaled_embedding_vjp": (
        (2, "grad_table"), (2, "grad_output"), (-1, "indices"), (-1, "order"), (-1, "offsets"), ("double", "scale"),
    ),
    "grouped_matrix_product": ((2, "output"), (2, "A"), (3, "W"), (-1, "offsets"), (-1, "order")),
    "grouped_matrix_product_vjp": (
        (2, "grad_A"), (3, "grad_W"), (2, "grad_output"), (2, "A"), (3, "W"), (-1, "offsets"), (-1, "order"),
    ),
    "gated_residual_norm": (
        (2, "state"), (2, "next"), (2, "residual"), (2, "block"), (2, "gate"), (1, "weight_block"),
        (1, "weight_next"), ("double", "residual_scale"), ("double", "epsilon"),
    ),
    "gated_residual_norm_vjp": (
        (2, "grad_residual"), (2, "grad_block"), (2, "grad_gate"), (1, "grad_weight_block"), (1, "grad_weight_next"),
        (2, "grad_state"), (2, "grad_next"), (2, "residual"), (2, "block"), (2, "gate"), (1, "weight_block"),
        (1, "weight_next"), ("double", "residual_scale"), ("double", "epsilon"),
    ),
}  # fmt: skip

_functions = {}


def _function(name, tag):
    symbol = f"mops_amd_{name}" if tag is None else f"mops_amd_{name}_{tag}"
    if symbol not in _functions:
        function = getattr(device_library().cdll, symbol)
        function.restype = ctypes.c_int
        function.argtypes = [
            ctypes.c_double if kind == "double" else _STRUCTS[(abs(kind), "i32" if kind < 0 else tag)]
            for kind, _ in _SIGNATURES[name]
        ]
        _functions[symbol] = function
    return _functions[symbol]


def _check_tensors(function, tensors, like):
    """``tensors``: name -> tensor (None: not given). All of them on the device of ``like`` (a name), the
    floating-point ones of its type; first the numbers of dimensions, then types and devices."""
    kinds = {name: kind for kind, name in _SIGNATURES[function]}
    for name, tensor in tensors.items():
        if tensor is not None:
            check_array(tensor, abs(kinds[name]), function, name)
    first = tensors[like]
    if not _dispatch.on_device(first):
        raise TypeError(f"`{like}` must be on a ROCm device in {function}: this library implements the device path only")
    for name, tensor in tensors.items():
        if tensor is None:
            continue
        if kinds[name] < 0:
            correct = _dispatch.is_integer(tensor)
        else:
            correct = _dispatch.dtype_name(tensor) in _TAGS and tensor.dtype == first.dtype
        if not correct:
            raise TypeError(f"Wrong dtype for {name} in {function}: got {_dispatch.dtype_name(tensor)}")
        if not _dispatch.is_torch(tensor) or tensor.device != first.device:
            raise ValueError(
                f"`{name}` must be a tensor on {first.device}, where `{like}` is, in {function}: all tensors must be "
                "on the same device"
            )


def _check_number(function, name, value):
    if not _dispatch.is_scalar(value):
        raise TypeError(f"`{name}` must be a scalar in {function}, got {type(value)}")


def _call(function, like, *arguments):
    """The C function with ``arguments`` in the order of its prototype, on the current stream of ``like``."""
    import torch

    tag = None
    values = []
    for (kind, _), argument in zip(_SIGNATURES[function], arguments):
        if kind == "double":
            values.append(float(argument))
            continue
        if kind > 0:
            tag = _TAGS[_dispatch.dtype_name(like)]
        struct = _STRUCTS[(abs(kind), "i32" if kind < 0 else tag)]()
        if argument is not None:
            element = type(struct.data)
            struct.data = ctypes.cast(ctypes.c_void_p(argument.data_ptr()), element)
            for d, extent in enumerate(argument.shape):
                struct.shape[d] = extent
        values.append(struct)
    library = device_library()
    with torch.cuda.device(like.device):
        library.cdll.mops_amd_set_stream(torch.cuda.current_stream(like.device).cuda_stream)
        library.cdll.mops_amd_set_synchronous(0)
        status = _function(function, tag)(*values)
    if status != 0:
        raise MopsError(library.last_error(), status)


def _values(*tensors):
    return [None if t is None else _dispatch.contiguous(t) for t in tensors]


def _int32(tensor):
    """A number that does not fit 32 bits is outside of every range, and has to stay outside: it becomes -1 or the
    largest one, not what its lower half happens to be."""
    if tensor.dtype.itemsize > 4:
        tensor = tensor.long().clamp(-1, 2**31 - 1)
    return _dispatch.as_int32(tensor)


def _indices(*tensors):
    return [None if t is None else _int32(t) for t in tensors]


def _like(wanted, tensor):
    return _dispatch.empty(tensor.shape, tensor) if wanted else None


# -------------------------------------------------------------- the plan ----
def order_by_group(indices, n_groups):
    """The rows in the order of their group: ``(order, offsets)``, both int32.

    ``order`` is a permutation of the rows, those with ``indices == 0`` first, then those with 1 and so on, rows of
    one group in ascending order; the rows of group ``g`` are ``order[offsets[g]:offsets[g + 1]]``. Rows whose index
    is outside ``[0, n_groups)`` (negative: padding) come last and belong to no group. One plan per batch serves
    ``grouped_matrix_product`` in every layer and the gradient of ``scaled_embedding``.
    """
    result = _native.order_by_group(indices, n_groups)
    if result is not None:
        return result
    function = "order_by_group"
    _check_tensors_index(function, indices)
    check_scalar(n_groups, function, "n_groups")
    if n_groups < 0:
        raise ValueError(f"`n_groups` must not be negative in {function}, got {n_groups}")
    (indices,) = _indices(indices)
    order = _dispatch.empty(indices.shape, indices)
    offsets = _dispatch.empty((n_groups + 1,), indices)
    _call(function, indices, order, offsets, indices)
    return order, offsets


def _check_tensors_index(function, indices):
    check_array(indices, 1, function, "indices")
    if not _dispatch.on_device(indices):
        raise TypeError(
            f"`indices` must be on a ROCm device in {function}: this library implements the device path only"
        )
    if not _dispatch.is_integer(indices):
        raise TypeError(f"Wrong dtype for indices in {function}: got {_dispatch.dtype_name(indices)}")


# ------------------------------------------------------------- embedding ----
def scaled_embedding(table, indices, scale=1.0):
    """``output[i, :] = scale * table[indices[i], :]``; a row of zeros where ``indices[i]`` is outside the table."""
    result = _native.scaled_embedding(table, indices, scale)
    if result is not None:
        return result
    function = "scaled_embedding"
    _check_tensors(function, {"table": table, "indices": indices}, "table")
    _check_number(function, "scale", scale)
    (table,) = _values(table)
    (indices,) = _indices(indices)
    output = _dispatch.empty((indices.shape[0], table.shape[1]), table)
    _call(function, table, output, table, indices, scale)
    return output


def scaled_embedding_vjp(grad_output, table, indices, scale=1.0, order=None, offsets=None):
    """Gradient of ``scaled_embedding`` with respect to ``table`` (of which only the shape is used).

    ``order``, ``offsets``: what ``order_by_group(indices, table.shape[0])`` returned, where the caller has it;
    otherwise the call orders the rows itself. The order of summation depends on the indices only: the same call
    gives the same bits.
    """
    result = _native.scaled_embedding_vjp(grad_output, table, indices, order, offsets, scale)
    if result is not None:
        return result
    function = "scaled_embedding_vjp"
    kinds = {"grad_output": grad_output, "indices": indices, "order": order, "offsets": offsets}
    _check_tensors(function, kinds, "grad_output")
    check_array(table, 2, function, "table")
    if not _dispatch.on_device(table) or table.device != grad_output.device or table.dtype != grad_output.dtype:
        raise TypeError(f"`table` must have the dtype and the device of `grad_output` in {function}")
    _check_number(function, "scale", scale)
    if (order is None) != (offsets is None):
        raise ValueError(f"order and offsets must be given together in {function}")
    (grad_output,) = _values(grad_output)
    indices, order, offsets = _indices(indices, order, offsets)
    grad_table = _dispatch.empty(table.shape, grad_output)
    _call(function, grad_output, grad_table, grad_output, indices, order, offsets, scale)
    return grad_table


# ------------------------------------------------------ products by group ----
def grouped_matrix_product(A, W, offsets, order=None):
    """``output[r, :] = A[r, :] @ W[g]`` for the rows ``r = order[p]`` of group ``g``,
    ``offsets[g] <= p < offsets[g + 1]``.

    ``order``: a permutation of the rows (``order_by_group``), or None where the rows already lie in the order of
    their group. Rows of no group give rows of zeros.
    """
    result = _native.grouped_matrix_product(A, W, offsets, order)
    if result is not None:
        return result
    function = "grouped_matrix_product"
    _check_tensors(function, {"A": A, "W": W, "offsets": offsets, "order": order}, "A")
    A, W = _values(A, W)
    offsets, order = _indices(offsets, order)
    output = _dispatch.empty((A.shape[0], W.shape[2]), A)
    _call(function, A, output, A, W, offsets, order)
    return output


def grouped_matrix_product_vjp(
    grad_output, A, W, offsets, order=None, compute_grad_A=True, compute_grad_W=True
):
    """Gradients of ``grouped_matrix_product`` with respect to ``A`` and ``W``."""
    result = _native.grouped_matrix_product_vjp(grad_output, A, W, offsets, order, compute_grad_A, compute_grad_W)
    if result is not None:
        return result
    function = "grouped_matrix_product_vjp"
    tensors = {"grad_output": grad_output, "A": A, "W": W, "offsets": offsets, "order": order}
    _check_tensors(function, tensors, "grad_output")
    grad_output, A, W = _values(grad_output, A, W)
    offsets, order = _indices(offsets, order)
    grad_A, grad_W = _like(compute_grad_A, A), _like(compute_grad_W, W)
    _call(function, A, grad_A, grad_W, grad_output, A, W, offsets, order)
    return grad_A, grad_W


# -------------------------------------------------------- residual update ----
def gated_residual_norm(residual, block, gate, weight_block, weight_next, residual_scale=1.0, epsilon=1e-6):
    """The residual update around a block; returns ``(state, next)``::

        state = residual + residual_scale * gate * norm(block) * weight_block
        next  = norm(state) * weight_next
        norm(x) = x / sqrt(mean(x**2, over the columns) + epsilon)

    ``gate`` has the shape of ``residual``, or one row for all rows. ``next`` is the input of the next block, made
    from the state before it is rounded.
    """
    result = _native.gated_residual_norm(residual, block, gate, weight_block, weight_next, residual_scale, epsilon)
    if result is not None:
        return result
    function = "gated_residual_norm"
    tensors = {
        "residual": residual, "block": block, "gate": gate, "weight_block": weight_block, "weight_next": weight_next,
    }  # fmt: skip
    _check_tensors(function, tensors, "residual")
    _check_number(function, "residual_scale", residual_scale)
    _check_number(function, "epsilon", epsilon)
    residual, block, gate, weight_block, weight_next = _values(residual, block, gate, weight_block, weight_next)
    state, following = _like(True, residual), _like(True, residual)
    _call(
        function, residual, state, following, residual, block, gate, weight_block, weight_next, residual_scale, epsilon
    )
    return state, following


def gated_residual_norm_vjp(
    grad_state,
    grad_next,
    residual,
    block,
    gate,
    weight_block,
    weight_next,
    residual_scale=1.0,
    epsilon=1e-6,
    compute_grad_residual=True,
    compute_grad_block=True,
    compute_grad_gate=True,
    compute_grad_weight_block=True,
    compute_grad_weight_next=True,
):
    """Gradients of ``gated_residual_norm`` with respect to ``residual``, ``block``, ``gate``, ``weight_block`` and
    ``weight_next``, from those of ``state`` and ``next`` (either may be None: zero)."""
    wanted = (
        compute_grad_residual, compute_grad_block, compute_grad_gate, compute_grad_weight_block,
        compute_grad_weight_next,
    )  # fmt: skip
    result = _native.gated_residual_norm_vjp(
        residual, block, gate, weight_block, weight_next, grad_state, grad_next, residual_scale, epsilon, *wanted
    )
    if result is not None:
        return result
    function = "gated_residual_norm_vjp"
    tensors = {
        "grad_state": grad_state, "grad_next": grad_next, "residual": residual, "block": block, "gate": gate,
        "weight_block": weight_block, "weight_next": weight_next,
    }  # fmt: skip
    _check_tensors(function, tensors, "residual")
    _check_number(function, "residual_scale", residual_scale)
    _check_number(function, "epsilon", epsilon)
    inputs = _values(residual, block, gate, weight_block, weight_next)
    grad_state, grad_next = _values(grad_state, grad_next)
    grads = [_like(want, tensor) for want, tensor in zip(wanted, inputs)]
    _call(function, inputs[0], *grads, grad_state, grad_next, *inputs, residual_scale, epsilon)
    return tuple(grads)
