// Dense layers with bias, activation and residual in their product: y = act(x W^T + b) + skip, forward and backward.  The product and what
// follows it are rows_product()'s: the sums go through the wave's share of LDS as they are, in 32 bits, and bias, activation and residual are
// applied in the layout in which the outputs are written, so that residual, hidden values and outputs pass memory in whole 16-byte pieces
// and are rounded once.
#include "ptl_gate_bw.inc"
#include "ptl_rows_mm.inc"
#include "ptl_tuning.h"

namespace ptl {

template <typename T>
int rows_act(RowsArgs &a) {
    return rows_product<T, T, ROWS_ACT>(a);
}

template <typename T, typename Linear, typename Args>
static int act_linear_step(const Args *a, int ns, bool back, const char *fn) {
    if (!a || !a->input || !a->coeff || !a->output) return rows_bad(fn, "null argument structure");
    const int in = a->input->dim, outs = a->output->dim;
    if (in <= 0 || outs <= 0 || in > (1 << 27) || outs >= ROW_MOST) return rows_bad(fn, "invalid tensor geometry");
    if (a->activation < PTL_GATE_SIGMOID || a->activation > PTL_ACT_NONE) return rows_bad(fn, "unknown activation");
    const bool bias = a->use_biases == 1, none = a->activation == PTL_ACT_NONE;
    if (bias && !a->bias) return rows_bad(fn, "use_biases=1 with a null bias blob");
    if (back && !none && !a->hidden) return rows_bad(fn, "null argument structure");
    const bool keeps = back ? !none : blob_data(a->hidden) != nullptr, weights = !back || !a->skip_wg_grad || !a->skip_in_grad;  // (what the call uses)
    const bool fits = (size_t)in * outs > 0x7fffffffu || a->coeff->dim == in * outs;  // (a blob of more has no dim that says so)
    if ((weights && !fits) || (bias && !(back && a->skip_wg_grad) && a->bias->dim != outs) || (keeps && a->hidden->dim != outs) || (!back && a->skip && a->skip->dim != outs))
        return rows_bad(fn, "tensors whose sizes do not fit together");
    if (ns > ROW_MOST) return rows_bad(fn, "more than 2^30 samples");
    if (ns <= 0) return 0;
    auto as = [](auto *p) { return reinterpret_cast<T *>(p); };
    const size_t nx = (size_t)ns * in, ny = (size_t)ns * outs, nw = (size_t)outs * in;
    if (!back) {
        T *h = as(blob_data(a->hidden));
        if (!a->input->data || !a->coeff->data || !a->output->data || (bias && !a->bias->data) || (a->skip && !a->skip->data)) return rows_bad(fn, "null buffer");
        if (!ensure_init()) return 2;
        Stager sg;
        RowsArgs r = {};
        r.x = reinterpret_cast<const char *>(sg.in<T>(as(a->input->data), nx));
        r.w = reinterpret_cast<const char *>(sg.in<T>(as(a->coeff->data), nw));
        if (bias) r.bias = sg.in<T>(as(a->bias->data), (size_t)outs);
        if (a->skip) r.skip = sg.in<T>(as(a->skip->data), ny);
        r.y = sg.out<T>(as(a->output->data), ny);
        if (h) r.hidden = sg.out<T>(h, ny);
        if (sg.failed()) return 2;
        r.row_b = in * (int)sizeof(T);
        r.outs = outs;
        r.tokens = ns;
        r.act = a->activation;
        r.zeros = static_cast<const char *>(state().zeros);
        return sg.finish(rows_act<T>(r));
    }
    const bool wg = !a->skip_wg_grad, ig = !a->skip_in_grad;
    if ((!none && (!a->hidden->data || !a->hidden->diff)) || !a->output->diff ||
        (wg && (!a->input->data || !a->coeff->diff || (bias && !a->bias->diff))) || (ig && (!a->coeff->data || !a->input->diff)))
        return rows_bad(fn, "null buffer");
    if (nx > 0x7fffffffu || ny > 0x7fffffffu || nw > 0x7fffffffu) return rows_bad(fn, "tensor larger than 2^31 elements");
    if (!ensure_init()) return 2;
    ptl_internal_stage_begin();  // the gradients of the pre-activations are the products' input
    return ptl_internal_stage_end(gated_back<T, false, Linear>(a, ns, in, outs, bias, wg, ig));
}

}  // namespace ptl

extern "C" {
int ptl_act_linear_fp32_fw_batched(const struct ActLinear_args *a, int ns) {
    return ptl::act_linear_step<float, ::Linear_args>(a, ns, false, "ptl_act_linear_fp32_fw_batched");
}
int ptl_act_linear_fp32_bw_batched(const struct ActLinear_args *a, int ns) {
    return ptl::act_linear_step<float, ::Linear_args>(a, ns, true, "ptl_act_linear_fp32_bw_batched");
}
int ptl_act_linear_fp16_fw_batched(const struct ActLinear_args_fp16 *a, int ns) {
    return ptl::act_linear_step<ptl::half_t, ::Linear_args_fp16>(a, ns, false, "ptl_act_linear_fp16_fw_batched");
}
int ptl_act_linear_fp16_bw_batched(const struct ActLinear_args_fp16 *a, int ns) {
    return ptl::act_linear_step<ptl::half_t, ::Linear_args_fp16>(a, ns, true, "ptl_act_linear_fp16_bw_batched");
}
}
