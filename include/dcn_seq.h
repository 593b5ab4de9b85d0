/*
 * dcn_seq.h -- C ABI of the sequence operators of libdcn.so: what follows the clip features of a video network.
 *
 *   gated scan           h_t = a_t h_{t-1} + (1 - a_t) x_t, a_t = 1 / (1 + exp(-gate_t)), per channel over time
 *   gated residual norm  stream = x + scale * s(gate) * rms(block) * post,  normed = rms(stream) * pre
 *   token scores         log-probabilities of given tokens, entropy and the best alternatives of rows of logits
 *   distillation         KL divergence from a teacher's top tokens, with the gradient of the student's logits
 *
 * The reference (lshiwjx/deform_conv3d_pytorch_op) has no counterpart of these.  Conventions as in dcn.h: device pointers on
 * the current device, `stream` a cudaStream_t passed as void*, nothing is allocated and nothing synchronises, no state is kept
 * between calls; every function returns DCN_OK or a negative dcn_status.  Pointers are aligned to their element type; wider
 * loads are used where the pointers and strides allow them.  Strides are in elements, the last axis of every tensor is dense.
 *
 * Element types of activations, logits and their gradients: DCN_SEQ_F32, DCN_SEQ_BF16, DCN_SEQ_F16.  Sums, statistics and states
 * are float32 in every case; a result is rounded once, when it is stored.
 */
#ifndef DCN_SEQ_H_
#define DCN_SEQ_H_

#include "dcn.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { DCN_SEQ_F32 = 0, DCN_SEQ_BF16 = 1, DCN_SEQ_F16 = 2 };

/* ---------------------------------------------------------------------------------------------
 * Gated scan
 * ------------------------------------------------------------------------------------------- */
typedef struct dcn_scan {
    int32_t dtype;                              /* x, gate, y, dy, dx, dgate */
    int64_t batch, steps, channels;             /* any may be 0; batch * ceil(channels / 64) < 2^27 */
    int64_t x_batch, x_step;                    /* strides of x over batch and steps */
    int64_t gate_batch, gate_step;
    int64_t dy_batch, dy_step;                  /* backward only */
} dcn_scan;

/* Bytes of the states that the forward pass leaves for the backward pass: float32 [batch, ceil(steps / 64), channels]. */
size_t dcn_scan_checkpoint_bytes(const dcn_scan* p);

/* y [batch, steps, channels] (dense) and last [batch, channels] (float32): the states after each step and after the last one.
 * `state` [batch, channels] float32, or NULL for zeros.  `lengths` [batch] int64, or NULL: sequence b has lengths[b] steps (taken
 * into [0, steps]); behind them y is zero, and x and gate are not used, whatever they hold.  `checkpoints` NULL where no
 * gradient is wanted.  An infinite state (or x) stays infinite while gates are above zero in float32 (those above -87). */
int dcn_scan_forward(const dcn_scan* p, const void* x, const void* gate, const float* state, const int64_t* lengths, void* y,
                     float* last, float* checkpoints, void* stream);

/* dx, dgate (dense, zero behind a sequence's length) and dstate [batch, channels] (float32, may be NULL) from dy and dlast
 * (float32; either may be NULL for zeros) and the forward pass's checkpoints. */
int dcn_scan_backward(const dcn_scan* p, const void* x, const void* gate, const int64_t* lengths, const float* checkpoints,
                      const void* dy, const float* dlast, void* dx, void* dgate, float* dstate, void* stream);

/* One step of `rows` sequences whose states are rows of a pool: state[slots[r]] advances in place, y[r] is its new value.
 * x and gate [rows, channels] with row strides, y dense; state float32 [pool, channels] dense.  slots int64 [rows] or NULL for
 * 0, 1, ...; a slot outside [0, pool) leaves the pool alone and gives zeros.  No slot may occur twice. */
int dcn_scan_step(int32_t dtype, int64_t rows, int64_t channels, const void* x, int64_t x_row, const void* gate,
                  int64_t gate_row, float* state, int64_t pool, const int64_t* slots, void* y, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Gated residual norm: the norm behind a block, its gate, the scaled residual and the norm before the next block
 *   rms(v) = v / sqrt(mean(v^2) + eps) over the channels
 *   stream = x + scale * s(gate) * rms(block) * post        (gate, scale, post: 1 where NULL)
 *   normed = rms(stream) * pre                              (pre: 1 where NULL; from the unrounded stream)
 * block == NULL: stream is x, and only normed is computed.
 * ------------------------------------------------------------------------------------------- */
typedef struct dcn_norm {
    int32_t dtype;                              /* x, block, gate, stream, normed and their gradients */
    int32_t weight_dtype;                       /* scale, post, pre [channels] and their gradients: float32 or dtype */
    int64_t rows, channels;                     /* rows < 2^31, 1 <= channels <= 8192 */
    int64_t x_row, block_row, gate_row;         /* row strides */
    int64_t dstream_row, dnormed_row;           /* backward only */
    float eps;
} dcn_norm;

/* stream (NULL where block is) and normed [rows, channels] dense; stats float32 [rows, 2]: 1 / sqrt(mean + eps) of block and
 * of stream, for the backward pass, or NULL. */
int dcn_norm_forward(const dcn_norm* p, const void* x, const void* block, const void* gate, const void* scale, const void* post,
                     const void* pre, void* stream_out, void* normed, float* stats, void* stream);

/* Scratch bytes of dcn_norm_backward where a gradient of scale, post or pre is wanted. */
size_t dcn_norm_workspace_bytes(const dcn_norm* p);

/* Gradients (dense; any may be NULL = not wanted) from dstream and dnormed (either may be NULL for zeros).  The sums over the
 * rows of dscale, dpost and dpre are made in a fixed order. */
int dcn_norm_backward(const dcn_norm* p, const void* x, const void* block, const void* gate, const void* scale,
                      const void* post, const void* pre, const float* stats, const void* dstream, const void* dnormed, void* dx,
                      void* dblock, void* dgate, void* dscale, void* dpost, void* dpre, void* workspace,
                      size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Rows of logits.  z = logits / temperature, p = softmax(z) over the row.
 * A logit of -inf stands for a token that cannot come (p = 0).  A row in which nothing is left (all -inf) has log p = -inf
 * everywhere, entropy 0 and a gradient of zeros.  NaN anywhere in a row makes all of its results NaN.
 * ------------------------------------------------------------------------------------------- */
typedef struct dcn_logits {
    int32_t dtype;                              /* logits and dlogits */
    int64_t rows, vocab;                        /* rows < 2^27, 1 <= vocab < 2^31 */
    int64_t row_stride;                         /* of logits; dlogits is dense */
    float temperature;                          /* 1e-3 to 1e3 */
} dcn_logits;

enum { DCN_SCORES_MOST_TOP = 128, DCN_DISTILL_MOST_K = 128, DCN_DISTILL_MOST_VOCAB = 1 << 20, DCN_LOGITS_STATS = 8 };

/* logprob [rows] = log p[tokens], entropy [rows] = -sum p log p, and the `top` tokens of the largest logits with their
 * log p [rows, top], largest first, equal ones by their index, NaN before all others.  A token equal to ignore_index has
 * logprob 0; any other outside [0, vocab) has NaN.  tokens int64 (NULL: logprob may be NULL too); top <= min(128, vocab).
 * stats float32 [rows, DCN_LOGITS_STATS] for the backward pass, or NULL. */
int dcn_scores_forward(const dcn_logits* p, const void* logits, const int64_t* tokens, int64_t ignore_index, int32_t top,
                       float* logprob, float* entropy, float* top_logprobs, int64_t* top_tokens, float* stats, void* stream);

/* dlogits [rows, vocab] from dlogprob, dentropy [rows] and dtop [rows, top] (float32; each may be NULL for zeros). */
int dcn_scores_backward(const dcn_logits* p, const void* logits, const int64_t* tokens, int64_t ignore_index, int32_t top,
                        const int64_t* top_tokens, const float* stats, const float* dlogprob, const float* dentropy,
                        const float* dtop, void* dlogits, void* stream);

/* loss [rows] = temperature^2 KL(teacher || student), the student's p against the teacher's q over its k best tokens:
 * tail = 1: q = exp(teacher_logprobs), and all other tokens together are one more outcome, of q_rest = max(0, 1 - sum q); it is
 *           left out where the student has no mass there (all its other logits are -inf), however much the teacher has: 1 - sum q
 *           is not 0 but of the size of its roundings where the teacher's tokens are all there are;
 * tail = 0: q = softmax(teacher_logprobs), over the k tokens alone.
 * teacher_logprobs are those of teacher logits / temperature, [rows, k] dense, of type teacher_dtype (float32 or dtype);
 * teacher_tokens int64 [rows, k].  A token outside [0, vocab) marks a place that is not used; a row without any has loss 0 and
 * a gradient of zeros.  k <= 128, vocab <= 2^20.  stats float32 [rows, DCN_LOGITS_STATS] for the backward pass, or NULL. */
int dcn_distill_forward(const dcn_logits* p, const void* logits, int32_t k, const void* teacher_logprobs, int32_t teacher_dtype,
                        const int64_t* teacher_tokens, int32_t tail, float* loss, float* stats, void* stream);

/* dlogits [rows, vocab] from dloss [rows] (float32). */
int dcn_distill_backward(const dcn_logits* p, const void* logits, int32_t k, const void* teacher_logprobs, int32_t teacher_dtype,
                         const int64_t* teacher_tokens, int32_t tail, const float* stats, const float* dloss, void* dlogits,
                         void* stream);

#ifdef __cplusplus
}
#endif
#endif /* DCN_SEQ_H_ */
