/*
 * Learner layers on NVIDIA B200 (sm_100a): the operators that follow the
 * learner's input tensors (tb_cuda_prepare_actor_inputs_device) in a learner
 * of stems, a recurrence over trajectories and routed experts.
 *
 *   group norm with an activation, channels last     forward, backward
 *   gated linear recurrence with resets              forward (one step included), backward
 *   routing to experts with slot lists               forward, backward
 *   combining the experts' rows into their tokens    forward, backward
 *
 * Conventions (those of cuda_features.h): device pointers, row-major, the
 * last dimension contiguous; `stream` is a cudaStream_t or NULL for the legacy
 * default stream; calls are asynchronous, allocate nothing, can be captured
 * into a CUDA graph and return 1 if the launches succeeded, 0 on a rejected
 * argument (NULL where it is not allowed, a size of zero or beyond the stated
 * limits, a stride smaller than its row, a pointer not aligned to its
 * element, an output or a workspace at the address of an input or of another
 * output where that is not stated) or a launch error.
 * The recurrence's kernels wait for copies of their own, for a second at most;
 * where that runs out their results are wrong, and tb_cuda_synchronize(stream)
 * (cuda_features.h) says so by returning 0.
 * A descriptor is read during the call only.  Strides are in elements, 0 means
 * dense.  Tensors of `type` may be f32, bf16 or f16; parameters, statistics,
 * states and weights are f32, all sums and states are held in f32, and each
 * result is rounded once.  Every result is the same bits on every run.  The
 * exponentials, reciprocals and square roots in SiLU, in the recurrence's gates
 * and in softmax scores are the special function unit's: within a few units in
 * the last place of f32 (an exponential of -v within v/2 more), 0 below its
 * normal numbers.
 * Workspaces are scratch: at least the stated bytes, 16-byte aligned, contents
 * irrelevant, not shared by calls that may overlap; NULL if 0 bytes are
 * needed.  Any alignment and stride is accepted; rows that start on 16-byte
 * boundaries are fastest.
 */
#ifndef TURBINATOR_CUDA_LEARNER_H
#define TURBINATOR_CUDA_LEARNER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations. */
#define TB_TYPE_F32 0
#define TB_TYPE_BF16 1
#define TB_TYPE_F16 2

/* ---- Group norm with an activation, channels last ---- */

#define TB_ACT_NONE 0
#define TB_ACT_RELU 1
#define TB_ACT_SILU 2
#define TB_ACT_GELU 3 /* u/2 (1 + erf(u/sqrt 2)) */

/* samples * groups < 2^31, channels < 2^31.
 *
 * x [samples, positions, channels]; group i holds channels
 * [i*channels/groups, (i+1)*channels/groups).  Per (sample, group), over its
 * positions*channels/groups values:
 *   mean = E x,  rstd = 1/sqrt(E (x-mean)^2 + epsilon)
 *   u = gamma_c (x-mean) rstd + beta_c,  y = act(u) */
typedef struct tb_group_norm_desc {
    size_t samples, positions, channels, groups; /* groups divides channels */
    size_t x_sample_stride, x_position_stride;   /* of x */
    size_t y_sample_stride, y_position_stride;   /* of y and dy */
    size_t dx_sample_stride, dx_position_stride; /* of dx */
    int type, activation;
    float epsilon;
} tb_group_norm_desc;

/* Bytes of workspace that either direction needs (0 for a bad descriptor). */
size_t tb_cuda_group_norm_workspace(const tb_group_norm_desc *desc);

/* gamma, beta [channels] f32 (NULL: 1 and 0); mean, rstd [samples, groups] f32
 * are written for the backward pass (both NULL: not written).  y may be x
 * (same strides). */
int tb_cuda_group_norm_device(const tb_group_norm_desc *desc, const void *x, const float *gamma,
                              const float *beta, void *y, float *mean, float *rstd, void *workspace,
                              void *stream);

/* dx [samples, positions, channels], dgamma and dbeta [channels] f32 (each NULL: not written), from the
 * forward pass's x, mean, rstd and dy.  dx may be dy or x (same strides). */
int tb_cuda_group_norm_backward_device(const tb_group_norm_desc *desc, const void *x, const float *gamma,
                                       const float *beta, const float *mean, const float *rstd,
                                       const void *dy, void *dx, float *dgamma, float *dbeta,
                                       void *workspace, void *stream);

/* ---- Gated linear recurrence ---- */

/* Steps between two saved states (tb_cuda_gated_recurrence_device). */
#define TB_RECURRENCE_CHECKPOINT 16

/* steps <= 2^31 - 256, sequences * channels < 2^31, sequences *
 * ceil(channels/32) * ceil(steps/8) < 2^31.
 *
 * x, recurrence gate r, input gate i [sequences, steps, channels], per channel
 * a learned decay l, all channels independent:
 *   log a_t = -decay_scale softplus(l) sigmoid(r_t)
 *   h_t = a_t h_(t-1) + sqrt(1 - a_t^2) sigmoid(i_t) x_t
 * A step whose reset flag is set starts anew (a_t = 0: an episode's first
 * step), whatever the state before it, an infinite or NaN one too: where step
 * 0 is one, state_in may be left unset.  Steps at and past a sequence's length change no state; their h and
 * their gradients are written as zero and their inputs (NaN included) are not
 * used. */
typedef struct tb_gated_recurrence_desc {
    size_t sequences, steps, channels;
    size_t in_sequence_stride, in_step_stride;     /* of x and both gates: thirds of one row, say */
    size_t out_sequence_stride, out_step_stride;   /* of h and dh */
    size_t grad_sequence_stride, grad_step_stride; /* of dx and both gates' gradients */
    int type;
    float decay_scale; /* >= 0 */
} tb_gated_recurrence_desc;

/* Bytes of workspace that either direction needs (0 for a bad descriptor). */
size_t tb_cuda_gated_recurrence_workspace(const tb_gated_recurrence_desc *desc);

/* decay [channels] f32; reset [sequences, steps] bytes or NULL; lengths
 * [sequences] int32, taken into [0, steps], or NULL; state_in [sequences,
 * channels] f32 or NULL for zero; state_out likewise (the state after the last
 * step of each sequence) or NULL; it may be state_in, however many the steps,
 * so that a program steps its states in place.  checkpoints [sequences,
 * ceil(steps/16), channels] f32 receives the state before every 16th step for
 * the backward pass, or NULL. */
int tb_cuda_gated_recurrence_device(const tb_gated_recurrence_desc *desc, const void *x,
                                    const void *recurrence_gate, const void *input_gate, const float *decay,
                                    const uint8_t *reset, const int32_t *lengths, const float *state_in,
                                    void *h, float *state_out, float *checkpoints, void *workspace,
                                    void *stream);

/* Gradients of the same from dh and dstate_out (f32, or NULL for zero).
 * ddecay [channels] f32 (NULL: not written), dstate_in [sequences, channels]
 * f32 (NULL: not written); dstate_in may be dstate_out. */
int tb_cuda_gated_recurrence_backward_device(const tb_gated_recurrence_desc *desc, const void *x,
                                             const void *recurrence_gate, const void *input_gate,
                                             const float *decay, const uint8_t *reset,
                                             const int32_t *lengths, const float *checkpoints,
                                             const void *dh, const float *dstate_out, void *dx,
                                             void *drecurrence_gate, void *dinput_gate, float *ddecay,
                                             float *dstate_in, void *workspace, void *stream);

/* ---- Routing to experts ---- */

#define TB_SCORE_SOFTMAX 0
#define TB_SCORE_SIGMOID 1

#define TB_ROUTE_MAX_EXPERTS 1024
#define TB_ROUTE_MAX_TOP_K 32

/* logits [tokens, experts].  An expert whose logit is -inf or NaN is not
 * available to that token.  score = softmax over the available experts, or
 * sigmoid.  Experts are ranked by score + bias in f32 (by the logit itself where
 * there is no bias), ties by the lower index: the score is the kernel's, a
 * sigmoid within 2^-21 of itself, a softmax score within (4 + highest logit -
 * logit) 2^-20 of itself, so that experts nearer to each other than that may
 * change places.  A bias of -inf or NaN takes its expert out.  With groups >
 * 1, a token first keeps its top_groups groups of experts/groups consecutive
 * experts by the sum of each group's group_best (1 or 2) highest ranking
 * values, ties by the lower index (a group with one available expert counts
 * that one; without a bias, group_best 1 ranks by the logit).  The top_k best
 * experts left are the token's slots 0..top_k-1; weight = score (without the
 * bias), divided by the sum of the token's selected scores if renormalise (0
 * where that sum is 0), times weight_scale.  A slot with no available expert
 * left has id -1 and weight 0. */
typedef struct tb_expert_route_desc {
    size_t tokens, experts; /* experts <= TB_ROUTE_MAX_EXPERTS, tokens * top_k < 2^31 */
    size_t logits_stride;   /* of the rows of logits and dlogits */
    int top_k;              /* <= experts, <= TB_ROUTE_MAX_TOP_K */
    int groups, top_groups, group_best;
    int type, score, renormalise;
    float weight_scale;
} tb_expert_route_desc;

/* Bytes of workspace that the forward pass needs (0 for a bad descriptor). */
size_t tb_cuda_route_experts_workspace(const tb_expert_route_desc *desc);

/* bias [experts] f32 or NULL; ids int32 and weights f32 [tokens, top_k].  The
 * slot lists, all NULL or none: the slots (token*top_k + j) that have an
 * expert, sorted by expert and then by slot, in order [tokens*top_k] int32 (-1
 * past their end); expert e's are order[offsets[e] .. offsets[e+1])
 * (offsets [experts+1] int32); position [tokens, top_k] int32 is each slot's
 * place in order (-1 for none). */
int tb_cuda_route_experts_device(const tb_expert_route_desc *desc, const void *logits, const float *bias,
                                 int32_t *ids, float *weights, int32_t *offsets, int32_t *order,
                                 int32_t *position, void *workspace, void *stream);

/* dlogits from the forward pass's logits and ids and dweights [tokens, top_k]
 * (the selection itself has no gradient, nor has the bias). */
int tb_cuda_route_experts_backward_device(const tb_expert_route_desc *desc, const void *logits,
                                          const int32_t *ids, const float *dweights, void *dlogits,
                                          void *stream);

/* ---- Combining the experts' rows ---- */

/* out[t] = sum_j weights[t,j] rows[position[t,j]], summed over j in order; a
 * position outside [0, rows) adds nothing (a slot without an expert has -1).
 * With weights NULL every weight is 1: the gradient of the gather that handed
 * the tokens out. */
typedef struct tb_expert_combine_desc {
    size_t tokens, rows, width;     /* tokens * top_k < 2^31, rows < 2^31 */
    size_t rows_stride, out_stride; /* of rows and drows; of out and dout */
    int top_k;                      /* <= TB_ROUTE_MAX_TOP_K */
    int type;
} tb_expert_combine_desc;

int tb_cuda_combine_experts_device(const tb_expert_combine_desc *desc, const void *rows,
                                   const int32_t *position, const float *weights, void *out, void *stream);

/* drows[position[t,j]] = weights[t,j] dout[t], dweights[t,j] = <dout[t],
 * rows[position[t,j]]> (0 for a slot without a row).  No position may occur
 * twice; rows that none names are not written.  dweights may be NULL (weights
 * without a gradient; rows may then be NULL too).  drows must not overlap
 * rows. */
int tb_cuda_combine_experts_backward_device(const tb_expert_combine_desc *desc, const void *rows,
                                            const int32_t *position, const float *weights,
                                            const void *dout, void *drows, float *dweights, void *stream);

#ifdef __cplusplus
}
#endif

#endif
