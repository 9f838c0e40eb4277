/*
 * A transformer block that is tuned by rewards (no counterpart in the reference): dense layers with bias, activation and
 * residual in one product, the norms between two blocks with the gate and the residual between them, the clipped policy loss, and
 * AdamW over all tensors of a model.  fp32 and fp16 tensors, sums, statistics and moments in fp32 (moments also in 8 bits).
 *
 * Conventions are those of ptl_api.h, which includes this file: blobs describe ONE sample (a token) of `dim` elements,
 * sample n lies at data + n * dim; pointers may be host or device pointers; the calls return 0, 1 after rejecting their
 * arguments (message printed, outputs untouched) or 2 where a HIP call failed, and run on the library's stream.
 * nsamples <= 0 (count <= 0) is an empty batch: nothing is read or written, 0 is returned.  A call takes at most 2^30 samples of at
 * most 2^30 elements (norms: 2^24), a dense layer at most 2^27 inputs and fewer than 2^30 outputs, its backward call tensors of less than
 * 2^31 elements (samples times elements, and the weights), and a product as many outputs as 2^31 threads form (some 4 * 10^9 and more; 33
 * million outputs of a few tokens); larger ones are rejected.  Tensors a call writes must not overlap those it reads or the other ones
 * it writes except where a comment says so.  Blobs of a call whose dims do not fit together are rejected, those that it does not use are not looked
 * at.  A call that gets no memory (status 2) leaves what it reads as it was, also a
 * tensor that its results would have replaced; other outputs may be written in part.  Calls share the library's workspace: graphs
 * captured from them are replayed one after the other, as the calls would run.
 */
#ifndef PTL_TUNING_H
#define PTL_TUNING_H

#include "ptl_structs.h"
#include "ptl_transformer.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Activations of a dense layer: PTL_GATE_SIGMOID .. PTL_GATE_RELU, or none. */
#define PTL_ACT_NONE 4

/* Dense layer with n_in = input->dim, n_out = output->dim:
 *   coeff   n_out x n_in (data and diff);  bias n_out (data and diff), read and written with use_biases == 1
 *   hidden  n_out a sample: h = coeff * x [+ bias]; data is written by the forward call (hidden or its data may be NULL: not
 *           kept) and read by the backward call, diff is written by the backward call
 *   skip    (may be NULL) n_out a sample: the residual; read by the forward call only
 *   forward:  output = act(h) [+ skip], formed from h before it is rounded and rounded once.  output->data may be skip->data.
 *   backward: hidden->diff = output->diff * act'(h) from hidden->data; coeff->diff = hidden->diff^T * input->data (sum over the samples)
 *             and, with use_biases, bias->diff = the sum of hidden->diff, unless skip_wg_grad; input->diff = hidden->diff * coeff
 *             unless skip_in_grad.  hidden->diff is always written and is what the products and sums read, rounded to the tensor type as it
 *             is stored (fp16 calls of up to two samples or fewer than 16384 values: as it was before that, unless
 *             ptl_set_gemm_path() asks for another way); it may be hidden->data (the pre-activations are lost then) or output->diff.
 *             With PTL_ACT_NONE the gradients of the pre-activations are output->diff: hidden is neither read nor written.
 *             The residual's gradient is output->diff. */
struct ActLinear_args {
    struct blob *input;
    struct blob *coeff;
    struct blob *bias;
    struct blob *hidden;
    struct blob *skip;
    struct blob *output;
    int activation;
    int skip_wg_grad;
    int skip_in_grad;
    int use_biases;
};
struct ActLinear_args_fp16 {
    struct blob_fp16 *input;
    struct blob_fp16 *coeff;
    struct blob_fp16 *bias;
    struct blob_fp16 *hidden;
    struct blob_fp16 *skip;
    struct blob_fp16 *output;
    int activation;
    int skip_wg_grad;
    int skip_in_grad;
    int use_biases;
};
int ptl_act_linear_fp32_fw_batched(const struct ActLinear_args *a, int nsamples);
int ptl_act_linear_fp32_bw_batched(const struct ActLinear_args *a, int nsamples);
int ptl_act_linear_fp16_fw_batched(const struct ActLinear_args_fp16 *a, int nsamples);
int ptl_act_linear_fp16_bw_batched(const struct ActLinear_args_fp16 *a, int nsamples);

/* Between two blocks: the norm behind the first, its gate, the residual, and the norm in front of the second.
 *   forward:  u = b / sqrt(mean(b^2) + eps) * coeff_post;  s = skip_scale * x + gate * u;  y = s / sqrt(mean(s^2) + eps) * coeff_pre
 *     input->data b, skip->data x; sum->data receives s, output->data y (coeff_pre NULL: there is no second norm, output is not used).
 *     gate (NULL: 1) holds gates of dim elements one behind the other (gate->dim: of one or of all): sample n has gate n / rows_per_gate; with
 *     rows_per_gate = 0 all samples have the first.  y is formed from s before it is rounded.
 *     With eps = 0 a row whose squares are all 0 in fp32 has 0 in the place of its root's inverse.
 *     sum->data and output->data may be input->data or skip->data (not each other).
 *   backward: ds = sum->diff + the gradient of s by way of output->diff and coeff_pre (either may be missing: sum->diff NULL, coeff_pre
 *     NULL; not both);  reads b from input->data and, with coeff_pre, s from sum->data;
 *     skip->diff = skip_scale * ds, input->diff = the gradient of b, unless skip_in_grad;
 *     gate->diff = sum of ds * u over each gate's samples, coeff_post->diff = sum of gate * ds * b / sqrt(mean(b^2) + eps), coeff_pre->diff =
 *     sum of output->diff * s / sqrt(mean(s^2) + eps), over all samples, unless skip_wg_grad.
 *     input->diff and skip->diff (not each other) may be output->diff, sum->diff or the tensors that b and s are read from. */
struct NormJoin_args {
    struct blob *input;
    struct blob *skip;
    struct blob *gate;
    struct blob *coeff_post;
    struct blob *coeff_pre;
    struct blob *sum;
    struct blob *output;
    float skip_scale;
    float eps;
    int rows_per_gate;
    int skip_wg_grad;
    int skip_in_grad;
};
struct NormJoin_args_fp16 {
    struct blob_fp16 *input;
    struct blob_fp16 *skip;
    struct blob_fp16 *gate;
    struct blob_fp16 *coeff_post;
    struct blob_fp16 *coeff_pre;
    struct blob_fp16 *sum;
    struct blob_fp16 *output;
    float skip_scale;
    float eps;
    int rows_per_gate;
    int skip_wg_grad;
    int skip_in_grad;
};
int ptl_norm_join_fp32_fw_batched(const struct NormJoin_args *a, int nsamples);
int ptl_norm_join_fp32_bw_batched(const struct NormJoin_args *a, int nsamples);
int ptl_norm_join_fp16_fw_batched(const struct NormJoin_args_fp16 *a, int nsamples);
int ptl_norm_join_fp16_bw_batched(const struct NormJoin_args_fp16 *a, int nsamples);

/* Clipped policy loss, a row for each token of an answer.  output holds the logits of dim classes (data; diff receives the gradient),
 * actions the class that was drawn; a row whose action is not in 0 .. dim - 1 (padding) has loss 0, log-probability 0 and gradient 0.
 *   lp = log softmax(output / temperature)[action];  ratio = exp(lp - old_logp);  A = advantages
 *   loss = -min(ratio * A, clip(ratio, 1 - clip_low, 1 + clip_high) * A) + beta * (exp(d) - d - 1),  d = ref_logp - lp
 *   wr_loss[row] = weight * row_weight * loss (written by steps 0 and 2);  wr_logp[row] = lp (may be NULL)
 *   output->diff = weight * row_weight * dloss/dlp / temperature * (1 at the action - softmax(output / temperature)),
 *     dloss/dlp = -ratio * A where ratio * A is not the larger of the two products, else 0, and + beta * (1 - exp(d))
 * ref_logp may be NULL: no such term; row_weight may be NULL: 1.  clip_high may be infinite, clip_low is 0 or more.  Logits of -inf
 * (classes that are masked out) are allowed; an action among them has lp = -inf, a row in which all are has NaN.  temperature: 1e-6 .. 1e6.
 * step: 0 the losses, 1 the gradient, 2 both in one pass.  output->diff may be output->data. */
struct policy_loss_args {
    struct blob *output;
    int *actions;
    float *old_logp;
    float *ref_logp;
    float *advantages;
    float *row_weight;
    float clip_low;
    float clip_high;
    float beta;
    float temperature;
    float weight;
    float *wr_loss;
    float *wr_logp;
};
struct policy_loss_args_fp16 {
    struct blob_fp16 *output;
    int *actions;
    float *old_logp;
    float *ref_logp;
    float *advantages;
    float *row_weight;
    float clip_low;
    float clip_high;
    float beta;
    float temperature;
    float weight;
    float *wr_loss;
    float *wr_logp;
};
int ptl_policy_loss_fp32_batched(const struct policy_loss_args *a, int nsamples, int step);
int ptl_policy_loss_fp16_batched(const struct policy_loss_args_fp16 *a, int nsamples, int step);

/* A step of AdamW over `count` tensors in few launches.  Of each, with g = weights->diff * *grad_factor, t the number of the step:
 *   m = beta1 * m + (1 - beta1) * g;  v = beta2 * v + (1 - beta2) * g^2
 *   w = w - learning_rate * (m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps) + weight_decay * w)
 * state holds the moments before the step (NULL: they are 0 and w is read from weights->data), new_state receives them (NULL: they
 * replace those of state; one of the two is given); updated->data receives the weights (updated NULL: weights->data).  What is given in
 * both may be the same buffer.  state and new_state hold the same form:
 *   m, v            in fp32, weights->dim elements each; or
 *   m_root, v_root  in 8 bits with a scale for every 256 elements (ceil(dim / 256) in m_scale and v_scale): the signed root of m,
 *                   -127 .. 127, and the fourth root of v, 0 .. 255, which the scale multiplies; the scale is the largest root of the
 *                   256 over 127 or 255.  They are rounded to the nearest (ties to even), a v that is not 0 to 1 at least (moments below
 *                   fp32's normal range count as 0).  256 elements with infinities or NaN get a scale that is no finite number.  w is
 *                   formed from m and v before they are rounded.
 *   master          (may be NULL; in both or neither of state and new_state) the weights in fp32: w is read from state->master and
 *                   written to new_state->master, and weights->data is not read; updated->data receives w rounded. */
struct adamw_state {
    float *m;
    float *v;
    int8_t *m_root;
    uint8_t *v_root;
    float *m_scale;
    float *v_scale;
    float *master;
};
struct adamw_args {
    struct blob *weights;
    struct blob *updated;
    struct adamw_state *state;
    struct adamw_state *new_state;
    float learning_rate;
    float weight_decay;
};
struct adamw_args_fp16 {
    struct blob_fp16 *weights;
    struct blob_fp16 *updated;
    struct adamw_state *state;
    struct adamw_state *new_state;
    float learning_rate;
    float weight_decay;
};
/* What the tensors share: beta1 and beta2 in 0 .. 1 (below 1), eps from 1e-30 on.  step is t, from 1 on; step_data (may be NULL: step) a place
 * that holds it when the step runs, so that a captured graph can be replayed with another (learning_rate and weight_decay are what they were at the
 * call: a graph keeps them).  grad_factor (may be NULL: 1) holds a factor
 * of the gradients (the inverse of a loss scale, a clipped norm's); where it is no finite number the step changes nothing that is updated in
 * place, and elsewhere copies what it would have updated (zeros for moments that are 0). */
struct adamw_step {
    float beta1;
    float beta2;
    float eps;
    int step;
    int *step_data;
    float *grad_factor;
};
int ptl_adamw_fp32_multi(const struct adamw_args *list, int count, const struct adamw_step *step);
int ptl_adamw_fp16_multi(const struct adamw_args_fp16 *list, int count, const struct adamw_step *step);

#ifdef __cplusplus
}
#endif
#endif /* PTL_TUNING_H */
