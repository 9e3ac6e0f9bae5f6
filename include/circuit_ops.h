/*
 * circuit-b200 per-stage operators: the C ABI behind the Python `circuit_cuda`
 * module, one function per op of the reference torch extension
 * (reference native/bindings/torch_extension.cpp:236-257).  Same argument
 * meaning and output semantics as the reference op; tensors are passed as raw
 * device pointers plus sizes, and every call is asynchronous on `stream`
 * (a cudaStream_t; NULL = legacy default stream).
 *
 * These ops evaluate the reference's bound formulas exactly as written there
 * (no rounding margin) so they can be compared element by element with the
 * reference kernels; the fused search of include/circuit.h is the path that
 * inflates every bound by a rigorous fp32 margin.
 *
 * Output buffers are fully written by each op (masks, counts, zero / -1e9
 * fills), so callers may pass uninitialised memory.
 * Like the reference ops, these take the index tables as given: the sizes and
 * pointers are checked on the host, but survivor lists, parent ids and leaf
 * offsets / sizes are used as indices on the device without a range check, so
 * they must describe a valid index (one that circuit_load_index or
 * circuit_index_from_device accepts: those validate every table once).
 * Return value: 0 on success, a negative CIRCUIT_ERR_* code otherwise
 * (description in circuit_last_error()).
 */
#ifndef CIRCUIT_OPS_H
#define CIRCUIT_OPS_H

#include <stdint.h>

#include "circuit.h"

#ifdef __cplusplus
extern "C" {
#endif

/* reference evaluate_root_bounds_cuda (torch_extension.cpp:10-47, root_bounds.cu:11-56):
 * dots[r] = q.c_r; mask[r] = (dots[r] + query_norm * radii[r] >= threshold);
 * indices[0..count) = surviving roots (unspecified order); *count written. */
int circuit_op_evaluate_root_bounds(const float* query, const float* root_centers, const float* root_radii,
                                    float threshold, float query_norm, int num_roots, int dim, int* survivor_mask,
                                    int* survivor_indices, int* num_survivors, float* root_dot_products,
                                    void* stream);

/* reference project_parents_cuda (torch_extension.cpp:49-81, parent_projection.cu:11-65):
 * for each of the first num_survivors entries p of survivor_indices:
 *   projected[p, j] = sum_d q[d] * bases[p, d, j]     (j < rank <= 64)
 *   perp[p] = sqrt(max(query_norm_sq - ||projected[p]||^2, 0))
 * every other row of projected / perp is zero.  No survivor limit (the
 * reference device-count kernel projects at most 512 roots, dispatch.cu:284). */
int circuit_op_project_parents(const float* query, const float* bases, const int* survivor_indices,
                               int num_survivors, int num_bases, int dim, int rank, float query_norm_sq,
                               float* projected_queries, float* perp_norms, void* stream);

/* reference evaluate_child_bounds_cuda (torch_extension.cpp:83-119, child_bounds.cu:11-83):
 * child c of a surviving parent P survives iff
 *   dots[P] + sum_j max(qP_j l_cj, qP_j u_cj) + perp[P] * rho_c >= threshold. */
int circuit_op_evaluate_child_bounds(const float* projected_queries, const float* perp_norms,
                                     const float* root_dot_products, const float* child_intervals_l,
                                     const float* child_intervals_u, const float* child_radii,
                                     const int* child_parent_ids, const int* root_survivor_mask, float threshold,
                                     int num_total_children, int rank, int* child_survivor_mask,
                                     int* child_survivor_indices, int* num_child_survivors, void* stream);

/* reference score_surviving_leaves_cuda (torch_extension.cpp:121-149, dense_score.cu:9-59):
 * vector_scores[0..n) = -1e9, then q.x_v for every row v of the listed children. */
int circuit_op_score_surviving_leaves(const float* query, const float* leaf_vectors, const int* leaf_offsets,
                                      const int* leaf_sizes, const int* child_survivor_indices, int num_survivors,
                                      int64_t n, int dim, float* vector_scores, void* stream);

/* reference flat_exact_score_cuda (torch_extension.cpp:224-234, dense_score.cu:169-212):
 * scores[v] = q.x_v for v < n. */
int circuit_op_flat_exact_score(const float* query, const float* corpus, int64_t n, int dim, float* scores,
                                void* stream);

/* reference hierarchical_search_cuda (torch_extension.cpp:151-222, dispatch.cu:244-307):
 * in place on the caller's workspaces: vector_scores = -1e9, counters = 0, then
 * root bounds -> projection of every surviving root -> child bounds -> scores of
 * every surviving child's rows, with survivor counts read on the device. */
int circuit_op_hierarchical_search(const float* query, const float* root_centers, const float* root_radii,
                                   const float* bases, const float* child_intervals_l,
                                   const float* child_intervals_u, const float* child_radii,
                                   const int* child_parent_ids, const float* leaf_vectors, const int* leaf_offsets,
                                   const int* leaf_sizes, int* survivor_mask, int* survivor_indices,
                                   int* num_survivors, float* root_dot_products, float* projected_queries,
                                   float* perp_norms, int* child_survivor_mask, int* child_survivor_indices,
                                   int* num_child_survivors, float* vector_scores, int num_roots,
                                   int num_total_children, int64_t n, int dim, float threshold, int rank,
                                   float query_norm, void* stream);

/* ---------------------------------------------------------------- rows in 8 bits
 * A row of dim values is kept as dim int8 codes and one fp32 scale; code c stands for c * scale.  These ops run on the
 * device of their pointers, which must be the current one, allocate nothing, and may be captured into a CUDA graph.
 * Strides are in elements of the tensor they belong to (codes: bytes); dim is at most CIRCUIT_INT8_MAX_DIM. */
#define CIRCUIT_INT8_MAX_DIM 16384
#define CIRCUIT_INT8_MAX_QUERIES 65535

/* value types */
#define CIRCUIT_F32 0
#define CIRCUIT_F16 1
#define CIRCUIT_BF16 2

/* norms of circuit_op_quantize_rows */
#define CIRCUIT_NORM_NONE 0 /* scale = max|x| / 127 */
#define CIRCUIT_NORM_RMS 1  /* divided by sqrt(mean(v^2) + eps) */
#define CIRCUIT_NORM_UNIT 2 /* divided by sqrt(sum(v^2) + eps) */

/* Quantises n rows: v = rows (+ residual, rounded once to the rows' type and written to `summed`), u = v * weight,
 * codes = rint(127 u / max|u|) of the real quotient (ties to even), scale = max|u| / 127 over the norm.
 * residual and weight (of the rows' type or fp32, dim values) may be NULL; both need a norm.  A row of zeros gets scale
 * 0; a row with an infinity, a NaN, or a product beyond fp32 gets codes 0 and scale NaN.
 * slots == NULL: row i is written to row i of codes / scales.  Otherwise to row slots[i] (int32 or int64 as slot_bytes
 * says) of the `capacity` rows: a slot outside [0, capacity) writes nothing, of equal slots the last row stays, other
 * rows are left as they are.  `summed` may be `rows` or `residual` itself. */
int circuit_op_quantize_rows(const void* rows, int dtype, int64_t n, int dim, int64_t row_stride,
                             const void* residual, int64_t residual_stride, const void* weight, int weight_dtype,
                             int norm, float eps, void* summed, int64_t summed_stride, const void* slots,
                             int slot_bytes, int64_t capacity, int8_t* codes, int64_t code_stride, float* scales,
                             void* stream);

/* out[i] = codes[id] * scales[id] for id = ids[i] (int32 or int64), or i when ids == NULL, rounded once to dtype.
 * A negative id is an empty place and gives zeros, an id >= rows gives NaN.  With rows == 0 codes and scales may be
 * NULL. */
int circuit_op_dequantize_rows(const int8_t* codes, int64_t code_stride, const float* scales, int64_t rows, int dim,
                               const void* ids, int id_bytes, int64_t n, void* out, int dtype, int64_t out_stride,
                               void* stream);

/* out[i][j] = query_scales[i] * scales[j] * sum_k queries[i][k] codes[j][k] (+ bias[j]).  The sum is exact (32-bit
 * integers); as fp32 it is multiplied with the query's scale (the product has to stay in the range), then with the row's
 * and added to the bias in one operation: up to three fp32 roundings, and one to dtype.  Code rows start on
 * 16 bytes and their strides are multiples of 16; up to 15 bytes past dim are read in each row (the last one's too)
 * and do not count. */
int circuit_op_int8_scores(const int8_t* queries, int64_t query_stride, const float* query_scales, int64_t num_queries,
                           const int8_t* codes, int64_t code_stride, const float* scales, int64_t n, int dim,
                           const float* bias, void* out, int dtype, int64_t out_stride, void* stream);

/* Waits for `stream` and returns CIRCUIT_ERR_TIMEOUT if a bounded wait of circuit_op_int8_scores has given up on the
 * current device since the last call (the results that it would have brought were written as NaN), else 0. */
int circuit_op_int8_status(void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CIRCUIT_OPS_H */
