/* ebr_tokens.h: C ABI of the operators driven by integer ids: the scaled embedding and its gradient, tokens sorted by
 * expert and back, and the distillation loss on a teacher's top logits.
 *
 * Conventions (as include/ebr_attn.h): device pointers, sizes and strides in elements, the caller's stream as void*,
 * nothing allocated, nothing trapped, no host synchronisation. Every function returns EBR_OK (0) or an ebr_status code;
 * ebr_attn_last_error() holds the message. I/O types are EBR_FLOAT32 / EBR_FLOAT16 / EBR_BFLOAT16; sums, softmax
 * statistics and losses are float32 in a fixed order (the same inputs give the same bits), with one rounding to the
 * output's type. Scratch buffers are 16-byte aligned, of at least the bytes that the *_scratch_bytes function gives;
 * other arrays start at a multiple of their elements' size, unless more is said, else EBR_ERR_STRIDE.
 */
#ifndef EBR_TOKENS_H
#define EBR_TOKENS_H

#include <stddef.h>
#include <stdint.h>

#include "ebr_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of an id array. */
typedef enum { EBR_INT32 = 0, EBR_INT64 = 1 } ebr_id_type;

/* out[t, :] = round(scale * W[ids[t], :]) for t in [0, n): W [V, C] of type w_dtype (row stride w_stride, unit column
 * stride), out [n, C] of type out_dtype, contiguous. An id outside [0, V) (a padding id) gives a row of zeros. */
int ebr_scaled_embedding(int w_dtype, int out_dtype, int id_type, int64_t n, int64_t V, int64_t C, double scale,
                         const void* ids, const void* w, int64_t w_stride, void* out, void* stream);

/* Its gradient with respect to the table: dW[v, :] = round(scale * sum over t with ids[t] = v of g[t, :]), g [n, C] of
 * type g_dtype (row stride g_stride, unit column stride), dW [V, C] of type w_dtype, contiguous,
 * 16-byte aligned, every element written.
 * The sum runs over the tokens sorted by id. Ids outside [0, V) contribute nothing. n < 2^30, V < 2^30. */
int ebr_scaled_embedding_grad(int g_dtype, int w_dtype, int id_type, int64_t n, int64_t V, int64_t C, double scale,
                              const void* ids, const void* g, int64_t g_stride, void* dw, void* scratch,
                              size_t scratch_bytes, void* stream);
size_t ebr_scaled_embedding_grad_scratch_bytes(int64_t n, int64_t V, int64_t C);

/* Sorts the T * K slots of an expert choice ids [T, K] (contiguous) by expert, slots of one expert in their own order.
 * offsets [E + 1] (int32): the first sorted position of each expert, counting every slot; offsets[E] = slots with an id
 * in [0, E). capacity = 0: rows = T * K and slot s sits in row row_of[s] = its sorted position. capacity > 0: rows =
 * E * capacity, expert e owns rows [e * capacity, (e + 1) * capacity), and its slots past the capacity are dropped.
 * row_of [T, K] (int32): the slot's row, -1 for a dropped slot or an id outside [0, E); slot_of [rows] (int32): the
 * row's slot, -1 for a row of no slot. 1 <= E <= 1024; T * K < 2^30, E * capacity < 2^30. */
int ebr_expert_route(int id_type, int64_t T, int64_t K, int64_t E, int64_t capacity, const void* ids, int32_t* row_of,
                     int32_t* slot_of, int32_t* offsets, void* scratch, size_t scratch_bytes, void* stream);
size_t ebr_expert_route_scratch_bytes(int64_t T, int64_t K, int64_t E);

/* Tokens to experts: rows_out[row_of[t, k], :] = round(weights[t, k] * x[t, :]) (weights NULL: a copy), rows of no slot
 * zeros; x [T, C] (row stride x_stride, unit column stride), rows_out [rows, C] contiguous. With rows_in [rows, C] and
 * dots [T, K] (both or neither), also dots[t, k] = <x[t, :], rows_in[row_of[t, k], :]> (0 for a dropped slot): with x
 * the gradient of ebr_expert_combine's output, the gradients of its rows and weights. rows_out may be NULL when dots is
 * not. weights and dots have type weight_dtype: EBR_FLOAT32 or dtype. Every row_of value is in [-1, rows). */
int ebr_expert_scatter(int dtype, int weight_dtype, int64_t T, int64_t K, int64_t C, int64_t rows, const void* x,
                       int64_t x_stride, const int32_t* row_of, const int32_t* slot_of, const void* weights,
                       const void* rows_in, void* rows_out, void* dots, void* stream);

/* And back: y[t, :] = round(sum over k of weights[t, k] * rows_in[row_of[t, k], :]) (weights NULL: ones), dropped slots
 * adding nothing (whatever their weights hold); rows_in [rows, C] (row stride rows_stride, unit column stride), y
 * [T, C] contiguous. There is at least one row, and every row_of value is in [-1, rows). */
int ebr_expert_combine(int dtype, int weight_dtype, int64_t T, int64_t K, int64_t C, const void* rows_in,
                       int64_t rows_stride, const int32_t* row_of, const void* weights, void* y, void* stream);

/* Distillation from a teacher's top logits. For each row n of logits [N, V] (row stride logits_stride, unit column
 * stride) the teacher gives K entries (top_ids [N, K], top_logits [N, K], contiguous); an id outside [0, V) is no entry.
 * With p = softmax of the entries' top_logits / tau, q = softmax of the row's logits / tau and w_n = row_weight[n] (1
 * where row_weight is NULL),
 *   losses[n] = w_n * tau^2 * sum over the entries of p_k (log p_k - log q[id_k]),
 *   total = factor * sum over n of losses[n],
 *   grad[n, j] = factor * u_n * w_n * tau * (q_j - sum of p_k with id_k = j),
 * entries with p_k = 0 adding nothing. A row without entries, or with entries of -infinity alone (a teacher's mask that
 * leaves nothing), or with w_n = 0, has loss 0 and gradient 0 whatever its logits hold. 1 <= K <= 1024, 1 <= V <= 2^19,
 * N < 2^31 - 2^16, 2^-126 <= tau <= 1e30.
 *
 * ebr_topk_distill: losses [N] float32; stats [N, 2] float32, 8-byte aligned (each row's largest logit and its sum of
 * exp((s - largest) / tau); 0 and infinity for a row that does not count); total: one float32 (a sum in a fixed order),
 * or NULL; grad [N, V] of type dtype (row stride grad_stride, unit column stride), made with u_n = 1, or NULL.
 * ebr_topk_distill_grad: grad from the forward's stats, u_n = upstream[upstream_stride * n] (stride 0 or 1). With
 * unless_one != 0 and stride 0, nothing is written where upstream[0] is exactly 1: grad was made with it already. */
int ebr_topk_distill(int dtype, int id_type, int top_dtype, int64_t N, int64_t V, int64_t K, double tau, double factor,
                     const void* logits, int64_t logits_stride, const void* top_ids, const void* top_logits,
                     const float* row_weight, float* losses, float* stats, float* total, void* grad, int64_t grad_stride,
                     void* stream);
int ebr_topk_distill_grad(int dtype, int id_type, int top_dtype, int64_t N, int64_t V, int64_t K, double tau,
                          double factor, const void* logits, int64_t logits_stride, const void* top_ids,
                          const void* top_logits, const float* row_weight, const float* stats, const float* upstream,
                          int64_t upstream_stride, int unless_one, void* grad, int64_t grad_stride, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* EBR_TOKENS_H */
