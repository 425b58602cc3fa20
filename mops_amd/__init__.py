"""mops on AMD Instinct MI355X: the five sparse tensor operations of
lab-cosmo/mops and their vector-Jacobian products, as hand-written HIP kernels
for gfx950 behind mops' own C ABI, called here on PyTorch-ROCm tensors; and the
operators of the layers around them (``mops_amd.layers``) and of networks of
such layers (``mops_amd.training``).

The public names are those of the reference's Python package
(``python/mops/src/mops/__init__.py`` of lab-cosmo/mops).
"""
from .layers import (  # noqa: F401
    gated_residual_norm,
    gated_residual_norm_vjp,
    grouped_matrix_product,
    grouped_matrix_product_vjp,
    order_by_group,
    scaled_embedding,
    scaled_embedding_vjp,
)
from .ops import (  # noqa: F401
    accept_unsorted_indices,
    first_occurrences,
    homogeneous_polynomial_evaluation,
    homogeneous_polynomial_evaluation_vjp,
    homogeneous_polynomial_evaluation_vjp_vjp,
    outer_product_scatter_add,
    outer_product_scatter_add_vjp,
    outer_product_scatter_add_vjp_vjp,
    outer_product_scatter_add_with_weights,
    outer_product_scatter_add_with_weights_vjp,
    outer_product_scatter_add_with_weights_vjp_vjp,
    sparse_accumulation_of_products,
    sparse_accumulation_of_products_vjp,
    sparse_accumulation_of_products_vjp_vjp,
    sparse_accumulation_scatter_add_with_weights,
    sparse_accumulation_scatter_add_with_weights_vjp,
    sparse_accumulation_scatter_add_with_weights_vjp_vjp,
)
from .training import (  # noqa: F401
    clip_gradients,
    clip_gradients_,
    gated_grouped_product,
    gated_grouped_product_vjp,
    gradient_norm,
    linear_cross_entropy,
    linear_cross_entropy_vjp,
)
from .status import MopsError  # noqa: F401

__all__ = [name for name in dir() if not name.startswith("_")]
