"""What a network of layers is made of and trained with besides its layers.

The gated half of a feed-forward block by group (beside ``grouped_matrix_product``, which is its other half), the
cross entropy of a linear layer to many classes (the other end of ``scaled_embedding``: its table can be the matrix),
each with its vector-Jacobian product; and the norm of all gradients, by which they are clipped. None of them exists
in lab-cosmo/mops. What each computes is written down in ``include/mops/layers.h``; types, devices, streams and
outputs are those of ``mops_amd.layers``.
"""
import ctypes

from . import _dispatch
from ._c_lib import device_library
from .layers import (
    _STRUCTS,
    _TAGS,
    _call,
    _check_number,
    _check_tensors,
    _indices,
    _like,
    _on_stream,
    _values,
)
from .ops import _native

_ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2}

#: as in ``mops_amd.layers``
_SIGNATURES = {
    "gated_grouped_product": (
        (2, "output"), (2, "A"), (3, "W"), (-1, "offsets"), (-1, "order"), ("int", "activation"),
    ),
    "gated_grouped_product_vjp": (
        (2, "grad_A"), (3, "grad_W"), (2, "grad_output"), (2, "A"), (3, "W"), (-1, "offsets"), (-1, "order"),
        ("int", "activation"),
    ),
    "linear_cross_entropy": (("wide", "losses"), ("wide", "log_sums"), (2, "A"), (2, "W"), (-1, "targets")),
    "linear_cross_entropy_vjp": (
        (2, "grad_A"), (2, "grad_W"), ("wide", "grad_losses"), ("wide", "grad_log_sums"), (2, "A"), (2, "W"),
        (-1, "targets"), ("wide", "log_sums"),
    ),
}  # fmt: skip


# --------------------------------------------- gated products by group ----
def _activation(function, name):
    if name not in _ACTIVATIONS:
        raise ValueError(f"`activation` must be one of {', '.join(_ACTIVATIONS)} in {function}, got {name!r}")
    return _ACTIVATIONS[name]


def gated_grouped_product(A, W, offsets, order=None, activation="silu"):
    """The first half of a gated feed-forward block, for the rows ``r = order[p]`` of group ``g``::

        gate, up = A[r] @ W[g, :, :L], A[r] @ W[g, :, L:]
        output[r] = act(gate) * up

    ``W`` has ``2 * L`` columns. ``activation``: ``"silu"`` (x / (1 + e^-x)), ``"gelu"`` (x times the normal
    distribution's integral up to x) or ``"sigmoid"``. ``order`` and ``offsets`` as in ``grouped_matrix_product``, which
    makes the block's second half; rows of no group give rows of zeros. Both projections, the activation and the
    product are one kernel, and the projections are never rounded.
    """
    result = _native.gated_grouped_product(A, W, offsets, order, activation)
    if result is not None:
        return result
    function = "gated_grouped_product"
    _check_tensors(function, {"A": A, "W": W, "offsets": offsets, "order": order}, "A", _SIGNATURES)
    which = _activation(function, activation)
    A, W = _values(A, W)
    offsets, order = _indices(offsets, order)
    output = _dispatch.empty((A.shape[0], W.shape[2] // 2), A)
    _call(function, A, output, A, W, offsets, order, which, signatures=_SIGNATURES)
    return output


def gated_grouped_product_vjp(
    grad_output, A, W, offsets, order=None, activation="silu", compute_grad_A=True, compute_grad_W=True
):
    """Gradients of ``gated_grouped_product`` with respect to ``A`` and ``W``.

    The projections are computed again. Their gradients, ``2 * L`` numbers per row, are held in the thread's scratch
    memory, rounded to the type of the tensors.
    """
    result = _native.gated_grouped_product_vjp(
        grad_output, A, W, offsets, order, activation, compute_grad_A, compute_grad_W
    )
    if result is not None:
        return result
    function = "gated_grouped_product_vjp"
    tensors = {"grad_output": grad_output, "A": A, "W": W, "offsets": offsets, "order": order}
    _check_tensors(function, tensors, "grad_output", _SIGNATURES)
    which = _activation(function, activation)
    grad_output, A, W = _values(grad_output, A, W)
    offsets, order = _indices(offsets, order)
    grad_A, grad_W = _like(compute_grad_A, A), _like(compute_grad_W, W)
    _call(function, A, grad_A, grad_W, grad_output, A, W, offsets, order, which, signatures=_SIGNATURES)
    return grad_A, grad_W


# ----------------------------------------------------------- cross entropy ----
def _empty_sums(like, rows):
    import torch

    return torch.empty(rows, dtype=torch.float64 if like.dtype == torch.float64 else torch.float32, device=like.device)


def linear_cross_entropy(A, W, targets):
    """The cross entropy of a linear layer to ``W.shape[0]`` classes; returns ``(losses, log_sums)``::

        logits = A @ W.T
        log_sums[r] = log(sum(exp(logits[r])))
        losses[r] = log_sums[r] - logits[r, targets[r]]

    Both are ``float32`` (``float64`` for ``float64``) and zero for a row whose target is outside of the classes
    (negative: padding); what such a row holds does not matter. ``W`` lies like the table of ``scaled_embedding`` and can be
    it. The logits are not rounded and not held in memory. The thread's scratch memory has two numbers per row and tile of
    classes, half a gigabyte at most (then, and where the device has not as much, a piece of the classes at a time).
    """
    result = _native.linear_cross_entropy(A, W, targets)
    if result is not None:
        return result
    function = "linear_cross_entropy"
    _check_tensors(function, {"A": A, "W": W, "targets": targets}, "A", _SIGNATURES)
    A, W = _values(A, W)
    (targets,) = _indices(targets)
    losses, log_sums = _empty_sums(A, A.shape[0]), _empty_sums(A, A.shape[0])
    _call(function, A, losses, log_sums, A, W, targets, signatures=_SIGNATURES)
    return losses, log_sums


def linear_cross_entropy_vjp(
    grad_losses, grad_log_sums, A, W, targets, log_sums, compute_grad_A=True, compute_grad_W=True
):
    """Gradients of ``linear_cross_entropy`` with respect to ``A`` and ``W``, from those of ``losses`` and ``log_sums``
    (either may be None: zero) and the ``log_sums`` it returned.

    The logits are computed again, a piece of the classes at a time; their gradients are held in the thread's scratch
    memory, about half a gigabyte (less where the device has not as much left), rounded to the type of the tensors. The
    order of summation depends on the shapes, on which rows have a target and on that memory only: the same call gives
    the same bits.
    """
    result = _native.linear_cross_entropy_vjp(
        grad_losses, grad_log_sums, A, W, targets, log_sums, compute_grad_A, compute_grad_W
    )
    if result is not None:
        return result
    function = "linear_cross_entropy_vjp"
    tensors = {
        "grad_losses": grad_losses, "grad_log_sums": grad_log_sums, "A": A, "W": W, "targets": targets,
        "log_sums": log_sums,
    }  # fmt: skip
    _check_tensors(function, tensors, "A", _SIGNATURES)
    A, W = _values(A, W)
    grad_losses, grad_log_sums, log_sums = _values(grad_losses, grad_log_sums, log_sums)
    (targets,) = _indices(targets)
    grad_A, grad_W = _like(compute_grad_A, A), _like(compute_grad_W, W)
    _call(function, A, grad_A, grad_W, grad_losses, grad_log_sums, A, W, targets, log_sums, signatures=_SIGNATURES)
    return grad_A, grad_W


# --------------------------------------------------------- norm of gradients ----
class _Gradient(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("size", ctypes.c_int64), ("type", ctypes.c_int32)]


_GRADIENT_TYPES = {"float32": 0, "float64": 1, "bfloat16": 2, "float16": 3}


def _is_dense(tensor):
    """Whether the tensor's numbers fill a piece of memory, in whatever order of dimensions."""
    expected = 1
    for stride, extent in sorted((s, n) for s, n in zip(tensor.stride(), tensor.shape) if n != 1):
        if stride != expected:
            return False
        expected *= extent
    return True


def _check_gradients(function, gradients):
    if _dispatch.is_array(gradients):
        raise TypeError(f"`gradients` must be a list of tensors in {function}, got a single one")
    gradients = list(gradients)
    if not gradients:
        raise ValueError(f"`gradients` must hold at least one tensor in {function}")
    for i, tensor in enumerate(gradients):
        if not _dispatch.is_torch(tensor):
            raise TypeError(f"`gradients[{i}]` must be a tensor in {function}, got {type(tensor)}")
        if not _dispatch.on_device(tensor):
            raise TypeError(
                f"`gradients[{i}]` must be on a ROCm device in {function}: this library implements the device path only"
            )
        if _dispatch.dtype_name(tensor) not in _TAGS or tensor.is_sparse or tensor.is_sparse_csr:
            raise TypeError(f"Wrong dtype or layout for gradients[{i}] in {function}: got {_dispatch.dtype_name(tensor)}")
        if tensor.device != gradients[0].device:
            raise ValueError(f"`gradients[{i}]` must be on {gradients[0].device}, where gradients[0] is, in {function}")
    return gradients


def _empty_norm(gradients):
    import torch

    wide = any(tensor.dtype == torch.float64 for tensor in gradients)
    return torch.empty((), dtype=torch.float64 if wide else torch.float32, device=gradients[0].device)


def _array_of(gradients):
    return (_Gradient * len(gradients))(
        *(_Gradient(t.data_ptr(), t.numel(), _GRADIENT_TYPES[_dispatch.dtype_name(t)]) for t in gradients)
    )


def _call_gradients(function, norm, *arguments):
    tag = _TAGS[_dispatch.dtype_name(norm)]
    view = _STRUCTS[(1, tag)]()
    view.data = ctypes.cast(ctypes.c_void_p(norm.data_ptr()), type(view.data))
    view.shape[0] = 1
    entry = getattr(device_library().cdll, f"mops_amd_{function}_{tag}")
    entry.restype = ctypes.c_int
    arrays = [ctypes.POINTER(_Gradient)] * (len(arguments) - (2 if function == "clip_gradients" else 1))
    entry.argtypes = [type(view), *arrays, ctypes.c_int64]
    if function == "clip_gradients":
        entry.argtypes = [*entry.argtypes, ctypes.c_double]
    _on_stream(norm, entry, [view, *arguments])


def _dense(tensor):
    tensor = tensor.resolve_neg()
    return tensor if _is_dense(tensor) else tensor.contiguous()


def gradient_norm(gradients):
    """The norm of all tensors of a list together, ``sqrt(sum of the squares of all their numbers)``.

    The tensors may have any shapes and any of the types, mixed. Returns a tensor without dimensions, ``float32``, or
    ``float64`` where one of them is. Squares are added up in 64 bits, in an order that depends on the sizes only.
    """
    result = _native.gradient_norm(gradients)
    if result is not None:
        return result
    function = "gradient_norm"
    gradients = [_dense(tensor) for tensor in _check_gradients(function, gradients)]
    norm = _empty_norm(gradients)
    _call_gradients(function, norm, _array_of(gradients), len(gradients))
    return norm


def clip_gradients(gradients, max_norm):
    """``([g * min(1, max_norm / norm) for g in gradients], norm)`` with the ``gradient_norm`` of all of them."""
    result = _native.clip_gradients(gradients, max_norm, False)
    if result is not None:
        return result
    import torch

    function = "clip_gradients"
    gradients = [_dense(tensor) for tensor in _check_gradients(function, gradients)]
    _check_number(function, "max_norm", max_norm)
    outputs = [torch.empty_like(tensor) for tensor in gradients]
    norm = _empty_norm(gradients)
    _call_gradients(function, norm, _array_of(outputs), _array_of(gradients), len(gradients), float(max_norm))
    return outputs, norm


def clip_gradients_(gradients, max_norm):
    """``clip_gradients`` in place; returns the norm they had. Where it is at most ``max_norm``, nothing is written.

    Every tensor must fill its memory (any order of dimensions), and none may share memory with another. One that was made
    in inference mode can be changed there only.
    """
    result = _native.clip_gradients(gradients, max_norm, True)
    if result is not None:
        return result
    import torch

    function = "clip_gradients_"
    gradients = _check_gradients(function, gradients)
    _check_number(function, "max_norm", max_norm)
    for i, tensor in enumerate(gradients):
        if tensor.is_neg() or not _is_dense(tensor):
            raise ValueError(f"`gradients[{i}]` must fill its memory without gaps in {function}")
        if tensor.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"`gradients[{i}]` requires a gradient itself: it cannot be changed in place in {function}")
        if tensor.is_inference() and not torch.is_inference_mode_enabled():
            raise ValueError(
                f"`gradients[{i}]` was made in inference mode and cannot be changed outside of it, in {function}"
            )
    norm = _empty_norm(gradients)
    array = _array_of(gradients)
    _call_gradients("clip_gradients", norm, array, array, len(gradients), float(max_norm))
    for tensor in gradients:
        torch.autograd.graph.increment_version(tensor)
    return norm
