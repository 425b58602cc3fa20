/* The operators of the layers around the sums over edges: a table looked up by
 * an index, products with a matrix per group of rows, also as gates of each
 * other, the normalised, gated residual update around a block; and what they
 * are trained with: the cross entropy of a linear layer to many classes, and
 * the norm of all gradients, which are clipped by it. None of these exist in
 * lab-cosmo/mops.
 *
 * Device memory only. Conventions as everywhere in this library: contiguous
 * row-major views by value, outputs first and completely overwritten, a
 * gradient whose `data` is NULL is not computed, status 0 / 1 (+ message,
 * mops_get_last_error_message) / 2, the calling thread's stream
 * (mops_amd_set_stream, mops_amd_set_synchronous). Element types: f32, f64,
 * bf16 (bfloat16) and f16 (IEEE half), all floating-point tensors of a call of
 * the same type. Sums, norms and their gradients are computed in 32 bits (in 64
 * for f64) and rounded once, when they are stored. */
#ifndef MOPS_LAYERS_H
#define MOPS_LAYERS_H

#include <stdint.h>

#include "mops/exports.h"
#include "mops/tensor.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Views of 16-bit floating-point data, given by their bits. */
#define MOPS_DEFINE_16_BIT_VIEW(NAME, NDIM)                                                        \
    typedef struct NAME {                                                                          \
        uint16_t* __restrict__ data;                                                               \
        int64_t shape[NDIM];                                                                       \
    } NAME;

MOPS_DEFINE_16_BIT_VIEW(mops_tensor_1d_bf16_t, 1)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_2d_bf16_t, 2)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_3d_bf16_t, 3)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_1d_f16_t, 1)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_2d_f16_t, 2)
MOPS_DEFINE_16_BIT_VIEW(mops_tensor_3d_f16_t, 3)

#undef MOPS_DEFINE_16_BIT_VIEW

/* The rows in the order of their group, and where each group begins.
 *
 * order[p], p = 0 .. N - 1, is a permutation of the rows: those with
 * indices[i] = 0 first, then those with 1, and so on, rows of one group in
 * ascending order; group g has the places offsets[g] .. offsets[g + 1] - 1
 * (offsets.shape[0] = number of groups + 1, offsets[0] = 0). Rows whose index
 * is negative or too large belong to no group and come last, behind
 * offsets[number of groups]: the way to mark rows that are padding. Integer
 * work, bit-exact. */
MOPS_EXPORT int mops_amd_order_by_group(
    mops_tensor_1d_i32_t order, mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t indices
);

/* Activations of mops_amd_gated_grouped_product. */
enum { MOPS_AMD_SILU = 0, MOPS_AMD_GELU = 1, MOPS_AMD_SIGMOID = 2 };

/* A tensor of any of the types among others: `size` numbers that follow each
 * other in memory. */
enum { MOPS_AMD_F32 = 0, MOPS_AMD_F64 = 1, MOPS_AMD_BF16 = 2, MOPS_AMD_F16 = 3 };
typedef struct mops_amd_gradient_t {
    void* data;
    int64_t size;
    int32_t type;
} mops_amd_gradient_t;

/* norm[0] = sqrt(sum of the squares of all numbers of all gradients), added up
 * in 64 bits in an order that depends on the sizes only; no square leaves their
 * range, of 64-bit numbers either. The array is read before the call returns. */
#define MOPS_GRADIENTS_DECLARE(W)                                                                  \
    MOPS_EXPORT int mops_amd_gradient_norm_##W(                                                    \
        mops_tensor_1d_##W##_t norm, const mops_amd_gradient_t* gradients, int64_t n_gradients     \
    );                                                                                             \
    /* And outputs[i] = gradients[i] * min(1, max_norm / norm), of the same size and type. An      \
     * output is its gradient's own memory (in place), or shares none with any gradient; outputs   \
     * share none with each other, and `norm` with none of them. max_norm is not negative. The norm \
     * is not rounded to the type of `norm` in between, nor the factor to that of a gradient. Infinities and not-a-number among   \
     * the gradients make of them what the formula does. */                               \
    MOPS_EXPORT int mops_amd_clip_gradients_##W(                                                   \
        mops_tensor_1d_##W##_t norm, const mops_amd_gradient_t* outputs,                           \
        const mops_amd_gradient_t* gradients, int64_t n_gradients, double max_norm                 \
    );
MOPS_GRADIENTS_DECLARE(f32)
MOPS_GRADIENTS_DECLARE(f64)

#undef MOPS_GRADIENTS_DECLARE

/* For each type S (R: what its sums are held in): */
#define MOPS_LAYERS_DECLARE(S, R)                                                                  \
    /* output[i, :] = scale * table[indices[i], :]; a row of zeros where indices[i] is outside     \
     * the table. */                                                                               \
    MOPS_EXPORT int mops_amd_scaled_embedding_##S(                                                 \
        mops_tensor_2d_##S##_t output, mops_tensor_2d_##S##_t table, mops_tensor_1d_i32_t indices, \
        double scale                                                                               \
    );                                                                                             \
    /* grad_table[v, :] = scale * (sum of grad_output[i, :] over the i with indices[i] = v), added \
     * up in an order that depends on the indices only. order, offsets: what                       \
     * mops_amd_order_by_group gives for indices and grad_table.shape[0] groups, or two NULL views \
     * (the call then orders the rows itself). */                                                  \
    MOPS_EXPORT int mops_amd_scaled_embedding_vjp_##S(                                             \
        mops_tensor_2d_##S##_t grad_table, mops_tensor_2d_##S##_t grad_output,                     \
        mops_tensor_1d_i32_t indices, mops_tensor_1d_i32_t order, mops_tensor_1d_i32_t offsets,    \
        double scale                                                                               \
    );                                                                                             \
    /* output[r, :] = A[r, :] W[g, :, :] for r = order[p], offsets[g] <= p < offsets[g + 1]; a row \
     * of zeros for r = order[p] with p in no group. order: a permutation of the rows, or a NULL   \
     * view where the rows lie in the order of their group already (order[p] = p). offsets is      \
     * non-decreasing. */                                                                          \
    MOPS_EXPORT int mops_amd_grouped_matrix_product_##S(                                           \
        mops_tensor_2d_##S##_t output, mops_tensor_2d_##S##_t A, mops_tensor_3d_##S##_t W,         \
        mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t order                                   \
    );                                                                                             \
    /* grad_A[r, :] = grad_output[r, :] W[g, :, :]^T (zeros for a row in no group), grad_W[g, :, :] \
     * = the sum of A[r, :]^T grad_output[r, :] over the rows of group g (zeros for a group        \
     * without rows). */                                                                           \
    MOPS_EXPORT int mops_amd_grouped_matrix_product_vjp_##S(                                       \
        mops_tensor_2d_##S##_t grad_A, mops_tensor_3d_##S##_t grad_W,                              \
        mops_tensor_2d_##S##_t grad_output, mops_tensor_2d_##S##_t A, mops_tensor_3d_##S##_t W,    \
        mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t order                                   \
    );                                                                                             \
    /* With W = (W_gate, W_up), L columns each, for the rows r of group g as above:                \
     *   output[r, :] = act(A[r, :] W_gate[g, :, :]) * (A[r, :] W_up[g, :, :])                     \
     * W.shape[2] = 2 L is even; a row of zeros for a row in no group. act: MOPS_AMD_SILU          \
     * (x / (1 + e^-x)), MOPS_AMD_GELU (x times the normal distribution's integral up to x),       \
     * MOPS_AMD_SIGMOID. The projections are never rounded. */                                     \
    MOPS_EXPORT int mops_amd_gated_grouped_product_##S(                                            \
        mops_tensor_2d_##S##_t output, mops_tensor_2d_##S##_t A, mops_tensor_3d_##S##_t W,         \
        mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t order, int32_t activation               \
    );                                                                                             \
    /* Its gradients. The gradients of the projections, 2 L numbers per row, are held in scratch   \
     * memory, rounded to the element type. */                                                     \
    MOPS_EXPORT int mops_amd_gated_grouped_product_vjp_##S(                                        \
        mops_tensor_2d_##S##_t grad_A, mops_tensor_3d_##S##_t grad_W,                              \
        mops_tensor_2d_##S##_t grad_output, mops_tensor_2d_##S##_t A, mops_tensor_3d_##S##_t W,    \
        mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t order, int32_t activation               \
    );                                                                                             \
    /* With x[r, v] = A[r, :] . W[v, :] for all classes v (rows of W):                             \
     *   log_sums[r] = log(sum over v of exp(x[r, v]))                                             \
     *   losses[r] = log_sums[r] - x[r, targets[r]]                                                \
     * Both zero for a row whose target is negative or too large: padding, and what it holds does  \
     * not matter. The logits x are not rounded, and not held in memory; two numbers per row and   \
     * tile of classes are, in scratch memory, for a piece of the classes at a time (half a        \
     * gigabyte at most, less where the device has not as much). */                                \
    MOPS_EXPORT int mops_amd_linear_cross_entropy_##S(                                             \
        mops_tensor_1d_##R##_t losses, mops_tensor_1d_##R##_t log_sums, mops_tensor_2d_##S##_t A,  \
        mops_tensor_2d_##S##_t W, mops_tensor_1d_i32_t targets                                     \
    );                                                                                             \
    /* Its gradients, from those of losses and log_sums (either may be a NULL view: zero) and the  \
     * log_sums that the call returned. The gradients of the logits are held in scratch memory for \
     * a piece of the classes at a time (about half a gigabyte), rounded to the element type.      \
     * Zeros for the rows without a target. */                                                     \
    MOPS_EXPORT int mops_amd_linear_cross_entropy_vjp_##S(                                         \
        mops_tensor_2d_##S##_t grad_A, mops_tensor_2d_##S##_t grad_W,                              \
        mops_tensor_1d_##R##_t grad_losses, mops_tensor_1d_##R##_t grad_log_sums,                  \
        mops_tensor_2d_##S##_t A, mops_tensor_2d_##S##_t W, mops_tensor_1d_i32_t targets,          \
        mops_tensor_1d_##R##_t log_sums                                                            \
    );                                                                                             \
    /* With norm(x) = x / sqrt(mean of x^2 over the columns + epsilon), row by row:                \
     *   state = residual + residual_scale * gate * norm(block) * weight_block                     \
     *   next  = norm(state) * weight_next                                                         \
     * gate has as many rows as residual, or one for all of them. next is made from the state      \
     * before it is rounded to the element type. */                                                \
    MOPS_EXPORT int mops_amd_gated_residual_norm_##S(                                              \
        mops_tensor_2d_##S##_t state, mops_tensor_2d_##S##_t next,                                 \
        mops_tensor_2d_##S##_t residual, mops_tensor_2d_##S##_t block,                             \
        mops_tensor_2d_##S##_t gate, mops_tensor_1d_##S##_t weight_block,                          \
        mops_tensor_1d_##S##_t weight_next, double residual_scale, double epsilon                  \
    );                                                                                             \
    /* The gradients of the same, from those of state and next (either may be a NULL view: zero). */ \
    MOPS_EXPORT int mops_amd_gated_residual_norm_vjp_##S(                                          \
        mops_tensor_2d_##S##_t grad_residual, mops_tensor_2d_##S##_t grad_block,                   \
        mops_tensor_2d_##S##_t grad_gate, mops_tensor_1d_##S##_t grad_weight_block,                \
        mops_tensor_1d_##S##_t grad_weight_next, mops_tensor_2d_##S##_t grad_state,                \
        mops_tensor_2d_##S##_t grad_next, mops_tensor_2d_##S##_t residual,                         \
        mops_tensor_2d_##S##_t block, mops_tensor_2d_##S##_t gate,                                 \
        mops_tensor_1d_##S##_t weight_block, mops_tensor_1d_##S##_t weight_next,                   \
        double residual_scale, double epsilon                                                      \
    );

MOPS_LAYERS_DECLARE(f32, f32)
MOPS_LAYERS_DECLARE(f64, f64)
MOPS_LAYERS_DECLARE(bf16, f32)
MOPS_LAYERS_DECLARE(f16, f32)

#undef MOPS_LAYERS_DECLARE

#ifdef __cplusplus
}
#endif

#endif
