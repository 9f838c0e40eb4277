// Products of 8-bit integers with a scale for every token and every row of weights.
#include "ptl_rows_mm.inc"
#include "ptl_transformer.h"

namespace ptl {

template <typename OUT>
int rows_int8(RowsArgs &a) {
    return rows_product<int8_t, OUT, false>(a);
}

template <typename OUT, typename Args>
static int mm_int8_step(const Args *a, const char *fn) {
    if (!a) return rows_bad(fn, "null argument structure");
    if (a->N < 0 || a->N > ROW_MOST || a->M <= 0 || a->K <= 0 || a->M > ROW_MOST) return rows_bad(fn, "invalid matrix geometry");
    if (a->K > 131071) return rows_bad(fn, "sums of more than 131071 products of 8-bit integers do not fit 32 bits");
    const bool bias = a->USE_BIASES == 1;
    if (!a->A || !a->B || !a->C || (bias && !a->bias)) return rows_bad(fn, "null buffer");
    if (a->N == 0) return 0;
    if (!ensure_init()) return 2;
    Stager sg;
    RowsArgs r = {};
    r.x = reinterpret_cast<const char *>(sg.in<int8_t>(a->A, (size_t)a->N * a->K));
    r.w = reinterpret_cast<const char *>(sg.in<int8_t>(a->B, (size_t)a->M * a->K));
    if (a->A_scale) r.x_scale = sg.in<float>(a->A_scale, (size_t)a->N);
    if (a->B_scale) r.w_scale = sg.in<float>(a->B_scale, (size_t)a->M);
    if (bias) r.bias = sg.in(reinterpret_cast<const OUT *>(a->bias), (size_t)a->M);
    r.y = sg.out(reinterpret_cast<OUT *>(a->C), (size_t)a->N * a->M);
    if (sg.failed()) return 2;
    r.row_b = a->K;
    r.outs = a->M;
    r.tokens = a->N;
    r.zeros = static_cast<const char *>(state().zeros);
    return sg.finish(rows_int8<OUT>(r));
}

}  // namespace ptl

extern "C" {
int ptl_mm_int8_fp32(const struct matMul_int8_args *a) { return ptl::mm_int8_step<float>(a, "ptl_mm_int8_fp32"); }
int ptl_mm_int8_fp16(const struct matMul_int8_args_fp16 *a) { return ptl::mm_int8_step<ptl::half_t>(a, "ptl_mm_int8_fp16"); }
}
