/*
 * cresso_b200_train.h - C ABI of the training operators around the optimizer step.
 *
 * They make the gradients that the step reads: the scaled embedding lookup and
 * its gradient, the norms before and after a block with its gate and residual
 * scale, and the distillation loss from a teacher's top logits.  They have no
 * counterpart in the reference, whose package holds the optimizer only.
 *
 * The conventions are those of cresso_b200.h: raw device pointers aligned to
 * their elements, an int status (the message is read with cresso_last_error),
 * caller-owned scratch (32-byte aligned, not shared by calls that may overlap)
 * whose size is queried first, work ordered on the given stream of the current
 * device, no allocation and no synchronisation.  Several host threads may call
 * them at once, each with a stream of its own.  Outputs overlap inputs only
 * where that is said.  Element types are CRESSO_DTYPE_F32, _F16 and _BF16; sums,
 * statistics and norms are float32 and every output is rounded once.  The same
 * inputs give the same bits in every run.
 */
#ifndef CRESSO_B200_TRAIN_H
#define CRESSO_B200_TRAIN_H

#include "cresso_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bounds of the operators below; larger calls get CRESSO_EUNSUPPORTED. */
enum { CRESSO_TRAIN_MAX_TOP = 1024 };          /* teacher entries of a row            */
enum { CRESSO_TRAIN_MAX_ROWS = 2147483392 };   /* rows of a table, tokens, logit rows */
enum { CRESSO_TRAIN_MAX_EMBEDDING_WIDTH = 4194240 }; /* columns of an embedding gradient */
enum { CRESSO_TRAIN_MAX_NORM_WIDTH = 65536 };  /* columns of a block norm, of at most 2^28 - 32 rows */

/* ------------------------------------------------------------ embedding --- */

/* out[t] = scale * weight[token_t - row0], a row of zeros where token_t - row0
 * is outside [0, rows).  `weight` holds the rows [row0, row0 + rows) of the
 * table (a whole table, or the local block of a row-sharded one), `weight_stride`
 * elements apart; tokens are int32 or int64 (token_bytes 4 or 8); out is
 * contiguous (n, width).  row0 + rows - 1 fits 64 bits. */
CRESSO_API int cresso_embedding_gather(const void* weight, int64_t weight_dtype, int64_t rows, int64_t width,
                                       int64_t weight_stride, const void* tokens, int64_t token_bytes, int64_t n,
                                       int64_t row0, double scale, void* out, int64_t out_dtype,
                                       cresso_stream_t stream);

/* out[r] = scale * sum of grad[t] over the tokens with token_t - row0 = r and
 * token_t != padding, rows without a token zero; with accumulate != 0 the sum is
 * added to out[r] and rows without a token are not touched.  Tokens outside the
 * window take no part.  grad rows lie `grad_stride` elements apart, out is
 * contiguous (rows, width).  has_padding = 0 ignores `padding`. */
CRESSO_API int cresso_embedding_grad_scratch_bytes(int64_t n, int64_t rows, int64_t width, int64_t* bytes);
CRESSO_API int cresso_embedding_grad(const void* grad, int64_t grad_dtype, int64_t n, int64_t width,
                                     int64_t grad_stride, const void* tokens, int64_t token_bytes, int64_t rows,
                                     int64_t row0, int64_t has_padding, int64_t padding, double scale, void* out,
                                     int64_t out_dtype, int64_t accumulate, void* scratch, int64_t scratch_bytes,
                                     cresso_stream_t stream);

/* ----------------------------------------------------------- block norm --- */

/* For each of n rows of `width` elements:
 *   p = x * rsqrt(mean(x^2) + eps) * post_weight     (post_weight NULL: p = x)
 *   h = residual + scale * gate * p                   (gate NULL: 1; x NULL: h = residual)
 *   y = h * rsqrt(mean(h^2) + eps) * pre_weight       (pre_weight NULL: y is not written)
 * residual and h have res_dtype, x and y act_dtype (the same type, or float32
 * with a 16-bit one), the weights weight_dtype.  gate holds gate_rows rows of
 * `width` elements, each for n / gate_rows consecutive rows.  h is not written
 * when x is NULL.  Everything is contiguous. */
CRESSO_API int cresso_block_norm(const void* residual, const void* x, const void* post_weight, const void* pre_weight,
                                 const void* gate, int64_t n, int64_t width, int64_t gate_rows, int64_t res_dtype,
                                 int64_t act_dtype, int64_t weight_dtype, int64_t gate_dtype, double scale, double eps,
                                 void* h, void* y, cresso_stream_t stream);

/* Gradients of cresso_block_norm from its output h, its input x and the
 * gradients d_h of h (NULL: zero) and d_y of y (NULL: zero; needs pre_weight
 * otherwise): d_residual (res_dtype), d_x (act_dtype; NULL when x is NULL),
 * d_post_weight and d_pre_weight (weight_dtype; NULL when the weight is NULL,
 * d_pre_weight also when d_y is NULL) and d_gate (gate_dtype). */
CRESSO_API int cresso_block_norm_grad_scratch_bytes(int64_t n, int64_t width, int64_t gate_rows, int64_t* bytes);
CRESSO_API int cresso_block_norm_grad(const void* h, const void* x, const void* d_h, const void* d_y,
                                      const void* post_weight, const void* pre_weight, const void* gate, int64_t n,
                                      int64_t width, int64_t gate_rows, int64_t res_dtype, int64_t act_dtype,
                                      int64_t weight_dtype, int64_t gate_dtype, double scale, double eps,
                                      void* d_residual, void* d_x, void* d_post_weight, void* d_pre_weight,
                                      void* d_gate, void* scratch, int64_t scratch_bytes, cresso_stream_t stream);

/* --------------------------------------------------------- distillation --- */

/* Row t of the student's logits z (vocab elements, rows logits_stride elements
 * apart) against the k teacher entries (id, u) of that row:
 *   p = softmax over the valid entries of u / temperature,
 *   q = softmax of z / temperature over the whole row,
 *   loss_t = weight_t * temperature^2 * sum_k p_k (log p_k - log q[id_k]),
 *   grad_t[v] = weight_t * temperature * (q[v] - sum of p_k with id_k = v).
 * An entry is valid when 0 <= id < vocab and u is not -inf; an id may occur more
 * than once; temperature is in [1e-6, 1e6].  A row with weight 0 or no valid entry
 * has loss 0 and gradient 0 whatever its logits hold.  A student with a logit of
 * -inf at a teacher entry has loss +inf.  ids and teacher are contiguous (n, k), ids
 * int32 or int64, weight float32 (n) or NULL (1); loss is float32 (n); grad has the logits'
 * type, contiguous (n, vocab), and may be the logits themselves when their rows
 * are contiguous; grad NULL computes the loss only. */
CRESSO_API int cresso_distill(const void* logits, int64_t dtype, int64_t n, int64_t vocab, int64_t logits_stride,
                              const void* ids, int64_t id_bytes, const void* teacher, int64_t teacher_dtype, int64_t k,
                              const float* weight, double temperature, float* loss, void* grad,
                              cresso_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* CRESSO_B200_TRAIN_H */
