/* The operators of the layers around the sums over edges: a table looked up by
 * an index, products with a matrix per group of rows, and the normalised,
 * gated residual update around a block. None of these exist in
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

/* For each type S: */
#define MOPS_LAYERS_DECLARE(S)                                                                     \
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
    /* grad_A[r, :] = grad_output[r, :] W[g, :, :]^T (zeros for a row in no group), grad_W[g, :, :]\
     * = the sum of A[r, :]^T grad_output[r, :] over the rows of group g (zeros for a group        \
     * without rows). */                                                                           \
    MOPS_EXPORT int mops_amd_grouped_matrix_product_vjp_##S(                                       \
        mops_tensor_2d_##S##_t grad_A, mops_tensor_3d_##S##_t grad_W,                              \
        mops_tensor_2d_##S##_t grad_output, mops_tensor_2d_##S##_t A, mops_tensor_3d_##S##_t W,    \
        mops_tensor_1d_i32_t offsets, mops_tensor_1d_i32_t order                                   \
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

MOPS_LAYERS_DECLARE(f32)
MOPS_LAYERS_DECLARE(f64)
MOPS_LAYERS_DECLARE(bf16)
MOPS_LAYERS_DECLARE(f16)

#undef MOPS_LAYERS_DECLARE

#ifdef __cplusplus
}
#endif

#endif
