/*
 * The feed-forward half of a transformer block and its training by a teacher (no counterpart in the reference with these
 * arguments): root-mean-square normalisation behind a residual's addition, with an output in 8 bits; gated dense layers;
 * products of 8-bit integers with scales; the loss against a teacher's top logits.  fp32 and fp16 tensors, sums and
 * statistics in fp32.
 *
 * Conventions are those of ptl_api.h, which includes this file: blobs describe ONE sample (a token) of `dim` elements,
 * sample n lies at data + n * dim; pointers may be host or device pointers; the calls return 0, 1 after rejecting their
 * arguments (message printed, outputs untouched) or 2 where a HIP call failed, and run on the library's stream.
 * nsamples <= 0 is an empty batch: nothing is read or written, 0 is returned.  A call takes at most 2^30 samples of at most
 * 2^30 elements, a gated layer at most 2^27 inputs and fewer than 2^29 outputs, its backward call tensors of less than 2^31
 * elements (samples times elements, and the weights), and a product as many outputs as 2^31 threads form (some 4 * 10^9 and
 * more; 33 million outputs of a few tokens); larger ones are rejected.  Tensors a call writes must not overlap those it reads
 * or the other ones it writes except where a comment says so.  A call that gets no memory (status 2) leaves what it reads as
 * it was, also a tensor that its results would have replaced; other outputs may be written in part.  Sums and products in fp32
 * that leave its range count as infinite.
 */
#ifndef PTL_TRANSFORMER_H
#define PTL_TRANSFORMER_H

#include "ptl_structs.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Root-mean-square normalisation of rows, behind a residual's addition.
 *   forward:  s = input [+ skip];  r = 1 / sqrt(mean(s^2) + eps);  y = s * r * coeff
 *     With eps = 0 a row of zeros (one whose squares are all 0 in fp32) has r = 0: y is 0, and backward it takes no part.
 *     sum->data    (needed with skip, else NULL or not read) receives s, rounded to the tensor type
 *     output->data (output or its data may be NULL) receives y
 *     q_data, q_scale (both or neither): y in 8 bits, q = y / scale rounded to the nearest (ties to even), with one scale
 *       per row, the row's largest |y| / 127.  A row of zeros has the scale 0 and zeros; one with infinities or NaN gets a
 *       scale that is no finite number.
 *     At least one of output->data and q_data is given.  y and q are formed from s before it is rounded.
 *     sum->data and output->data may be input->data or skip->data (not each other).
 *   backward: g = output->diff * coeff;  d = r * (g - s * r^2 * mean(g * s)) [+ sum->diff]
 *     reads s from sum->data (with skip; else, where sum is NULL or has no data, from input->data), output->diff,
 *     coeff->data and, where sum and sum->diff are given, the gradient that reaches s from elsewhere;
 *     writes d to input->diff and, where skip and skip->diff are given, to skip->diff (which may be the same buffer), unless
 *     skip_in_grad, and coeff->diff = the sum over the rows of output->diff * s * r unless skip_wg_grad.
 *     input->diff and skip->diff may be output->diff, sum->diff or the tensor that s is read from. */
struct RmsNorm_args {
    struct blob *input;
    struct blob *skip;
    struct blob *sum;
    struct blob *coeff;
    struct blob *output;
    int8_t *q_data;
    float *q_scale;
    float eps;
    int skip_wg_grad;
    int skip_in_grad;
};
struct RmsNorm_args_fp16 {
    struct blob_fp16 *input;
    struct blob_fp16 *skip;
    struct blob_fp16 *sum;
    struct blob_fp16 *coeff;
    struct blob_fp16 *output;
    int8_t *q_data;
    float *q_scale;
    float eps;
    int skip_wg_grad;
    int skip_in_grad;
};
int ptl_rms_norm_fp32_fw_batched(const struct RmsNorm_args *a, int nsamples);
int ptl_rms_norm_fp32_bw_batched(const struct RmsNorm_args *a, int nsamples);
int ptl_rms_norm_fp16_fw_batched(const struct RmsNorm_args_fp16 *a, int nsamples);
int ptl_rms_norm_fp16_bw_batched(const struct RmsNorm_args_fp16 *a, int nsamples);

/* Activation of a gated layer's first half.  Infinities have the activation's and its slope's limits (0 at -inf). */
#define PTL_GATE_SIGMOID 0 /* 1 / (1 + exp(-x)) */
#define PTL_GATE_SILU 1    /* x / (1 + exp(-x)) */
#define PTL_GATE_GELU 2    /* x (1 + tanh(sqrt(2 / pi) (x + 0.044715 x^3))) / 2 */
#define PTL_GATE_RELU 3    /* max(x, 0) */

/* Gated dense layer.  With n_in = input->dim, n_out = output->dim:
 *   coeff   2 n_out x n_in: n_out rows of the gate, then n_out rows of the other projection (data and diff)
 *   bias    2 n_out (data and diff), read and written with use_biases == 1
 *   hidden  2 n_out a sample: h = coeff * x [+ bias]; data is written by the forward call (hidden or its data may be NULL:
 *           not kept) and read by the backward call, diff is written by the backward call
 *   forward:  output = act(h[0 .. n_out)) * h[n_out .. 2 n_out), formed from h before it is rounded
 *   backward: hidden->diff = (output->diff * h_up * act'(h_gate), output->diff * act(h_gate)) from hidden->data;
 *             coeff->diff = hidden->diff^T * input->data (sum over the samples) and, with use_biases, bias->diff = the sum of
 *             hidden->diff, unless skip_wg_grad; input->diff = hidden->diff * coeff unless skip_in_grad.  hidden->diff is
 *             always written and is what the products and sums read, rounded to the tensor type as it is stored (fp16 calls of up
 *             to two samples or fewer than 16384 values: as it was before that, unless ptl_set_gemm_path() asks for another way); it
 *             may be hidden->data (the pre-activations are lost then). */
struct GatedLinear_args {
    struct blob *input;
    struct blob *coeff;
    struct blob *bias;
    struct blob *hidden;
    struct blob *output;
    int activation;
    int skip_wg_grad;
    int skip_in_grad;
    int use_biases;
};
struct GatedLinear_args_fp16 {
    struct blob_fp16 *input;
    struct blob_fp16 *coeff;
    struct blob_fp16 *bias;
    struct blob_fp16 *hidden;
    struct blob_fp16 *output;
    int activation;
    int skip_wg_grad;
    int skip_in_grad;
    int use_biases;
};
int ptl_gated_linear_fp32_fw_batched(const struct GatedLinear_args *a, int nsamples);
int ptl_gated_linear_fp32_bw_batched(const struct GatedLinear_args *a, int nsamples);
int ptl_gated_linear_fp16_fw_batched(const struct GatedLinear_args_fp16 *a, int nsamples);
int ptl_gated_linear_fp16_bw_batched(const struct GatedLinear_args_fp16 *a, int nsamples);

/* Product of 8-bit integers with scales: C[N x M] = A_scale[row] * B_scale[column] * sum_k A[row][k] * B[column][k]
 * [+ bias[column]], A stored N x K and B stored M x K (the weights of a dense layer, one row per output).  The sums are
 * formed in 32-bit integers, exactly: K is at most 131071.  A_scale (N) and B_scale (M) may be NULL: 1.  bias (M) is added
 * with USE_BIASES == 1. */
struct matMul_int8_args {
    int8_t *A;
    int8_t *B;
    float *C;
    float *A_scale;
    float *B_scale;
    float *bias;
    int N;
    int M;
    int K;
    int USE_BIASES;
};
struct matMul_int8_args_fp16 {
    int8_t *A;
    int8_t *B;
    fp16 *C;
    float *A_scale;
    float *B_scale;
    fp16 *bias;
    int N;
    int M;
    int K;
    int USE_BIASES;
};
int ptl_mm_int8_fp32(const struct matMul_int8_args *a);
int ptl_mm_int8_fp16(const struct matMul_int8_args_fp16 *a);

/* Distillation from a teacher's top logits: output holds the logits of dim classes (data; diff receives the gradient),
 * teacher n_top logits a sample (1 .. 2048) and classes the class of each.  An entry whose class is not in 0 .. dim - 1 is
 * left out; a class that is named twice has the sum of both probabilities.
 *   p = softmax over the row's entries of teacher / temperature;  q = softmax over all classes of output / temperature
 *   wr_loss[row] = weight * sum p (log p - log q);   output->diff = weight / temperature * (q * sum p - p)
 * A row without entries (or whose entries are all -inf) has loss 0 and gradient 0.  Logits of -inf (classes that are masked
 * out) are allowed; a row in which all are has no probabilities, and NaN for what an entry asks of it.  temperature: 1e-6 .. 1e6.  step: 0 the losses, 1 the gradient, 2 both in one pass.  output->diff may be output->data. */
struct distill_args {
    struct blob *output;
    float *teacher;
    int *classes;
    int n_top;
    float temperature;
    float weight;
    float *wr_loss;
};
struct distill_args_fp16 {
    struct blob_fp16 *output;
    fp16 *teacher;
    int *classes;
    int n_top;
    float temperature;
    float weight;
    float *wr_loss;
};
int ptl_distill_fp32_batched(const struct distill_args *a, int nsamples, int step);
int ptl_distill_fp16_batched(const struct distill_args_fp16 *a, int nsamples, int step);

#ifdef __cplusplus
}
#endif
#endif /* PTL_TRANSFORMER_H */
