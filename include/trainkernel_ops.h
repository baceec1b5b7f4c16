/* C ABI of libtrainkernel_ops.so: language-model operators that stand beside the compiled steps.
 *
 * Token log-probabilities of rows of logits with their gradient, two losses built on them (a clipped
 * policy loss with a KL term, a preference loss over pairs of sequences) and an AdamW update over many
 * tensors with moments in 32 or in 8 bits.  No counterpart in the reference, whose programs end in a
 * mean and whose update is SGD (reference: benchmarks/train_loop.py:35-45).
 *
 * Conventions are those of trainkernel_rt.h: plain pointers and sizes; every function returns 0 on
 * success, otherwise a cudaError_t value or TK_E_ARGUMENT; nothing throws; tk_ops_last_error() describes
 * the most recent failure on the calling thread.  Launches go to `stream` of device `device` (the current
 * device is left as it was found), never synchronise and never allocate, so they may be captured into a
 * CUDA graph.  Pointers are borrowed for the call; workspaces are the caller's, and two calls that can
 * overlap on the GPU need two of them.
 */
#ifndef TRAINKERNEL_OPS_H
#define TRAINKERNEL_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "trainkernel_rt.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { TK_F32 = 0, TK_F16 = 1, TK_BF16 = 2 };
enum { TK_AVERAGE_TOKENS = 0, TK_AVERAGE_SEQUENCES = 1 };

/* A [batch, length] array; strides in elements. */
typedef struct {
    const void* data;
    int64_t stride_batch, stride_token;
} tk_token_array;

/* batch x length rows of `vocab` logits (unit stride inside a row), the token of every row and which rows count.
 * A row whose mask byte is 0 has log-probability 0 and gradient 0, and none of its logits is used.  A target
 * outside [0, vocab) reads nothing and makes the row's results NaN. */
typedef struct {
    const void* logits;
    int64_t stride_batch, stride_token;   /* elements */
    int64_t batch, length, vocab;
    int32_t dtype;                        /* TK_F32 / TK_F16 / TK_BF16 */
    int32_t target_bytes;                 /* 4 or 8 */
    tk_token_array targets;
    tk_token_array mask;                  /* bytes; data may be NULL: every row counts */
} tk_token_rows;

/* Where the gradient of the logits goes and what scales it; data NULL: no gradient.  Rows of the logits' type with unit
 * stride inside a row; rows that do not lie as their logits do relative to 16-byte boundaries are written element by
 * element.  `scale` is multiplied by the FP32 value at `scale_at` when that is not NULL. */
typedef struct {
    void* data;
    int64_t stride_batch, stride_token;   /* elements */
    const float* scale_at;
    float scale;
    int32_t reserved;
} tk_token_grad;

typedef struct {
    tk_token_array old_logprobs, advantages, ref_logprobs;   /* FP32; ref_logprobs.data may be NULL, and is not read when kl_weight is 0 */
    float clip_low, clip_high, kl_weight;
    int32_t average;                                         /* TK_AVERAGE_* */
} tk_policy_terms;

/* Dense FP32 results of [batch, length] rows: `logprobs`, and, where not NULL, `stats` ([rows][2]), which are made for
 * tk_token_logits_grad and handed to it unchanged: the row's largest logit, and the sum of exp(logit - largest) times a
 * factor between 2^-1/256 and 2^1/256 (1 where |largest| is 0 or above 65536) that depends on `largest` alone and that
 * the gradient takes into account.  A log-sum-exp is the target's logit less its logprob, not largest + log(sum). */
int tk_token_logprobs(const tk_token_rows* rows, float* logprobs, float* stats, int device, void* stream);

/* logprobs and grad = scale * d(sum weights * logprobs)/d logits, each logit read from memory once where it fits. */
int tk_token_logprobs_and_grad(const tk_token_rows* rows, const tk_token_array* weights, float* logprobs,
                               const tk_token_grad* grad, int device, void* stream);

/* grad[row] = scale * coefficient[row] * (onehot(target) - softmax(logits)) from saved stats.  The coefficient of row
 * (b, t) is coefficients.data[b * stride_batch + t * stride_token]. */
int tk_token_logits_grad(const tk_token_rows* rows, const tk_token_array* coefficients, const float* stats,
                         const tk_token_grad* grad, int device, void* stream);

/* Clipped policy loss.  `coefficients` (dense, may be NULL) receives d loss / d logprob.  `workspace`:
 * tk_policy_workspace_bytes(batch, length) bytes, 16-byte aligned. */
size_t tk_policy_workspace_bytes(int64_t batch, int64_t length);
int tk_policy_loss(const tk_token_rows* rows, const tk_policy_terms* terms, float* loss, float* logprobs, float* stats,
                   float* coefficients, const tk_token_grad* grad, void* workspace, int device, void* stream);

/* Preference loss over batch / 2 pairs: sequence i against sequence i + batch / 2.  `reference`: FP32, one summed
 * log-probability per sequence, `reference_stride` elements apart.  `sums`: dense [batch].  `coefficients`: dense
 * [batch], receives d loss / d sums. */
size_t tk_preference_workspace_bytes(int64_t batch, int64_t length);
int tk_preference_loss(const tk_token_rows* rows, const float* reference, int64_t reference_stride, float beta,
                       float label_smoothing, float* loss, float* sums, float* stats, float* coefficients,
                       const tk_token_grad* grad, void* workspace, int device, void* stream);

/* One tensor of an AdamW update.  `offset`: where its moments start in the flat state, a multiple of 256. */
typedef struct {
    void* param;
    const void* grad;
    int64_t offset, count;
    float weight_decay;
    int32_t reserved;
} tk_adamw_tensor;

#define TK_ADAMW_BLOCK 256      /* elements that share one scale when moments are held in 8 bits */
#define TK_ADAMW_COUNTERS 4096  /* copies of the step counter, one for each block that may be launched */

typedef struct {
    void* mean;                 /* FP32, or e4m3 codes */
    void* square;               /* FP32, or e4m3 codes of the square root */
    float* mean_scale;          /* 8 bits: one per TK_ADAMW_BLOCK elements; NULL with FP32 moments */
    float* root_scale;
    int64_t* steps;             /* TK_ADAMW_COUNTERS equal values: steps taken so far */
} tk_adamw_state;

typedef struct {
    const float* lr_at;         /* device value used instead of `lr` when not NULL */
    const float* scale_at;      /* device value the gradients are multiplied with when not NULL; not finite: no update */
    double lr, beta1, beta2, eps;
    uint32_t seed;              /* of the stochastic rounding of 8-bit moments */
    int32_t bits;               /* 32 or 8 */
} tk_adamw_options;

/* All tensors share the parameter type and the gradient type.  No parameter overlaps another one, the state, a gradient
 * other than its own (which may be the same memory, element for element) or the values at lr_at and scale_at.
 * `last`: non-zero on the last call of one optimizer step (a step over tensors of several types takes several calls):
 * that call advances the step counters. */
int tk_adamw_update(const tk_adamw_tensor* tensors, int count, int param_dtype, int grad_dtype, const tk_adamw_state* state,
                    const tk_adamw_options* options, int last, int device, void* stream);

const char* tk_ops_last_error(void);
uint64_t tk_ops_launch_count(void);

#ifdef __cplusplus
}
#endif

#endif
