// Gated dense layers: y = act(x Wg^T) * (x Wu^T), forward and backward.
#include "ptl_rows_mm.inc"
#include "ptl_internal.h"

namespace ptl {

template <typename T>
int rows_gated(RowsArgs &a) {
    return rows_product<T, T, true>(a);
}

// dh = (dy h_up act'(h_gate), dy act(h_gate)): three values read, two written, nothing else (2048 x 5632 in fp16 21 us, 5.5 TB/s).  dh
// may be h.  part: sums of dh over the rows of a grid row, as it is stored (NULL: not wanted).  copy: dh in rows of `pitch` values, zeros
// behind (NULL: not wanted).
template <typename T>
__global__ __launch_bounds__(256) void gate_back_kernel(const T *h, const T *__restrict__ dy, T *dh, float *__restrict__ part, size_t rows, int outs,
                                                        int act, T *__restrict__ copy, int pitch) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    const int pieces = (outs + VEC - 1) / VEC, p = (int)(blockIdx.x * 256 + threadIdx.x);
    if (p >= pieces) return;
    const Gate gate(act);
    float sum[2][VEC] = {};
    for (size_t row = blockIdx.y; row < rows; row += gridDim.y) {
        Piece g, u, d, og, ou;
        g.fetch(h + row * 2 * outs, p, outs);
        u.fetch(h + row * 2 * outs + outs, p, outs);
        d.fetch(dy + row * outs, p, outs);
        g.trim(p, outs);
        u.trim(p, outs);
        d.trim(p, outs);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float f;
            const float df = gate.back((float)g.e[i], f);
            og.e[i] = (T)((float)d.e[i] * (float)u.e[i] * df);
            ou.e[i] = (T)((float)d.e[i] * f);
        }
        // (the sums are of the values that are stored: formed again for them, with other roundings in between, one in thousands would differ)
        asm volatile("" : "+v"(og.raw), "+v"(ou.raw));
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            sum[0][i] += (float)og.e[i];
            sum[1][i] += (float)ou.e[i];
        }
        og.store(dh + row * 2 * outs, p, outs);
        ou.store(dh + row * 2 * outs + outs, p, outs);
        if (copy) {
            T *to = copy + row * pitch;
            og.store(to, p, outs);
            ou.store(to + outs, p, outs);
            for (int i = 2 * outs + p; p < 8 && i < pitch; i += pieces) to[i] = (T)0.f;
        }
    }
    if (!part) return;
    float *to = part + (size_t)blockIdx.y * 2 * outs;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (p * VEC + i < outs) {
            to[p * VEC + i] = sum[0][i];
            to[outs + p * VEC + i] = sum[1][i];
        }
}

static int linear_bw(const ::Linear_args *l, int ns) { return ptl_linear_fp32_bw_batched(l, ns); }
static int linear_bw(const ::Linear_args_fp16 *l, int ns) { return ptl_linear_fp16_bw_batched(l, ns); }

// Which backward calls have both products made by gated_products().  fp16: from 1.5 GFLOP on (of 60 layers of 64 to 8192 tokens 0.84 to 1.62
// times as fast as a dense layer's call, 1.17 in the mean; below, 64 tokens, 512 -> 1408 and 512 tokens, 256 -> 512, 0.91 and 0.82), from
// 3 where operands have to be copied to rows of whole 16-byte pieces (16 layers 0.93 to 1.99, 1.26 in the mean: 3549 tokens,
// 1748 -> 1216 198 -> 100 us, 2048 tokens, 2047 -> 5631 390 -> 252; 7 layers below 0.69 to 1.0).  fp32: from 5 GFLOP on, and with 16 tokens
// and more where the weights are large (110 layers, copies or not: 52 that qualify 0.9 to 2.1 times as fast, 1.19 in the mean - 111
// tokens, 3300 -> 6400 370 -> 199 us, 32, 2304 -> 2880 65 -> 41 -, the others 0.66 to 1.39).
template <typename T>
static bool own_products(int ns, int in, int outs, bool copied) {
    const bool fits = in < 1 << 23 && outs < 1 << 22;  // (64 rows of the first operand and 128 of the second within 32 bits)
    const double flops = 8.0 * ns * in * outs, weights = (double)in * outs;
    const bool pays = sizeof(T) == 4 ? flops >= 5e9 || (ns >= 16 && weights >= 2.5e6) : flops >= (copied ? 3e9 : 1.5e9);
    return fits && pays && state().gemm_path == 0;
}

template <typename T, typename Linear, typename Args>
static int gated_back(const Args *a, int ns, int in, int outs, bool bias, bool wg, bool ig) {
    auto as = [](auto *p) { return reinterpret_cast<T *>(p); };
    const size_t nx = (size_t)ns * in, ny = (size_t)ns * outs, nw = (size_t)2 * outs * in;
    {
        Stager sg;
        const T *h = sg.in<T>(as(a->hidden->data), 2 * ny), *dy = sg.in<T>(as(a->output->diff), ny);
        T *dh = sg.out<T>(as(a->hidden->diff), 2 * ny);
        if (sg.failed()) return 2;
        const T *x = wg ? sg.in<T>(as(a->input->data), nx) : nullptr, *w = ig ? sg.in<T>(as(a->coeff->data), nw) : nullptr;
        T *dw = wg ? sg.out<T>(as(a->coeff->diff), nw) : nullptr, *dx = ig ? sg.out<T>(as(a->input->diff), nx) : nullptr;
        T *db = wg && bias ? sg.out<T>(as(a->bias->diff), (size_t)2 * outs) : nullptr;
        if (sg.failed()) return 2;
        // rows that are no whole 16-byte pieces are copied to such; dh is written a second time
        constexpr int VEC = RowPiece<T>::VEC;
        const int cols = (in + VEC - 1) / VEC * VEC, pitch = (2 * outs + VEC - 1) / VEC * VEC;
        bool copy_x = ((uintptr_t)x | (uintptr_t)w) % 16 || cols != in, copy_dh = (uintptr_t)dh % 16 || pitch != 2 * outs;
        const bool own = own_products<T>(ns, in, outs, copy_x || copy_dh);
        copy_x = copy_x && own;
        copy_dh = copy_dh && own;
        T *wide_w = nullptr, *wide_x = nullptr, *wide_dh = nullptr;
        if (copy_x || copy_dh) {
            const size_t n_w = copy_x && w ? (size_t)2 * outs * cols : 0, n_x = copy_x && x ? (size_t)ns * cols : 0, n_dh = copy_dh ? (size_t)ns * pitch : 0;
            wide_w = static_cast<T *>(scratch((n_w + n_x + n_dh) * sizeof(T)));
            if (!wide_w) return 2;
            wide_x = wide_w + n_w;
            if (copy_dh) wide_dh = wide_x + n_x;
            if (n_w + n_x) rows_copy(w, w ? 2 * (size_t)outs : 0, x, x ? ns : 0, wide_w, in * (int)sizeof(T), cols * (int)sizeof(T));
        }
        const int wide = ((outs + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC + 255) / 256;
        int high = ns < 65535 ? ns : 65535;
        float *part = nullptr;
        if (own && db) {  // its sums come with the gradients of the pre-activations: eight workgroups a compute unit
            const int most = (8 * state().num_cu + wide - 1) / wide;
            high = high < most ? high : most;
            if (!(part = workspace((size_t)high * 2 * outs * sizeof(float)))) return 2;
        }
        hipLaunchKernelGGL((gate_back_kernel<T>), dim3(wide, high), dim3(256), 0, state().stream, h, dy, dh, part, (size_t)ns, outs, a->activation,
                           wide_dh, pitch);
        if (part) row_shares<T>(part, db, 2 * outs, high);
        int rc = hip_ok(hipGetLastError(), "gated layer launch") ? 0 : 2;
        if (rc == 0 && own && (wg || ig))
            rc = gated_products<T>(copy_x ? wide_x : x, copy_x ? wide_w : w, copy_dh ? wide_dh : dh, dw, dx, ns, in, 2 * outs, cols, pitch);
        rc = sg.finish(rc);
        if (rc || own || !(wg || ig)) return rc;
    }
    auto out = *a->hidden;  // a dense layer of 2 n_out outputs
    out.dim = 2 * outs;
    Linear l = {};
    l.input = a->input;
    l.coeff = a->coeff;
    l.bias = a->bias;
    l.output = &out;
    l.skip_wg_grad = a->skip_wg_grad;
    l.skip_in_grad = a->skip_in_grad;
    l.use_biases = a->use_biases;
    return linear_bw(&l, ns);
}

template <typename T, typename Linear, typename Args>
static int gated_step(const Args *a, int ns, bool back, const char *fn) {
    if (!a || !a->input || !a->coeff || !a->output || (back && !a->hidden)) return rows_bad(fn, "null argument structure");
    const int in = a->input->dim, outs = a->output->dim;
    if (in <= 0 || outs <= 0 || in > (1 << 27) || outs >= ROW_MOST / 2) return rows_bad(fn, "invalid tensor geometry");
    if (a->activation < PTL_GATE_SIGMOID || a->activation > PTL_GATE_RELU) return rows_bad(fn, "unknown activation");
    const bool bias = a->use_biases == 1;
    if (bias && !a->bias) return rows_bad(fn, "use_biases=1 with a null bias blob");
    if (ns > ROW_MOST) return rows_bad(fn, "more than 2^30 samples");
    if (ns <= 0) return 0;
    auto as = [](auto *p) { return reinterpret_cast<T *>(p); };
    const size_t nx = (size_t)ns * in, ny = (size_t)ns * outs, nw = (size_t)2 * outs * in;
    if (!back) {
        T *h = as(blob_data(a->hidden));
        if (!a->input->data || !a->coeff->data || !a->output->data || (bias && !a->bias->data)) return rows_bad(fn, "null buffer");
        if (!ensure_init()) return 2;
        Stager sg;
        RowsArgs r = {};
        r.x = reinterpret_cast<const char *>(sg.in<T>(as(a->input->data), nx));
        r.w = reinterpret_cast<const char *>(sg.in<T>(as(a->coeff->data), nw));
        if (bias) r.bias = sg.in<T>(as(a->bias->data), (size_t)2 * outs);
        r.y = sg.out<T>(as(a->output->data), ny);
        if (h) r.hidden = sg.out<T>(h, 2 * ny);
        if (sg.failed()) return 2;
        r.row_b = in * (int)sizeof(T);
        r.outs = outs;
        r.tokens = ns;
        r.act = a->activation;
        r.zeros = static_cast<const char *>(state().zeros);
        return sg.finish(rows_gated<T>(r));
    }
    const bool wg = !a->skip_wg_grad, ig = !a->skip_in_grad;
    if (!a->hidden->data || !a->hidden->diff || !a->output->diff || (wg && (!a->input->data || !a->coeff->diff || (bias && !a->bias->diff))) ||
        (ig && (!a->coeff->data || !a->input->diff)))
        return rows_bad(fn, "null buffer");
    if (nx > 0x7fffffffu || 2 * ny > 0x7fffffffu || nw > 0x7fffffffu) return rows_bad(fn, "tensor larger than 2^31 elements");
    if (!ensure_init()) return 2;
    ptl_internal_stage_begin();  // the gradients of the pre-activations are the products' input
    return ptl_internal_stage_end(gated_back<T, Linear>(a, ns, in, outs, bias, wg, ig));
}

}  // namespace ptl

extern "C" {
int ptl_gated_linear_fp32_fw_batched(const struct GatedLinear_args *a, int ns) {
    return ptl::gated_step<float, ::Linear_args>(a, ns, false, "ptl_gated_linear_fp32_fw_batched");
}
int ptl_gated_linear_fp32_bw_batched(const struct GatedLinear_args *a, int ns) {
    return ptl::gated_step<float, ::Linear_args>(a, ns, true, "ptl_gated_linear_fp32_bw_batched");
}
int ptl_gated_linear_fp16_fw_batched(const struct GatedLinear_args_fp16 *a, int ns) {
    return ptl::gated_step<ptl::half_t, ::Linear_args_fp16>(a, ns, false, "ptl_gated_linear_fp16_fw_batched");
}
int ptl_gated_linear_fp16_bw_batched(const struct GatedLinear_args_fp16 *a, int ns) {
    return ptl::gated_step<ptl::half_t, ::Linear_args_fp16>(a, ns, true, "ptl_gated_linear_fp16_bw_batched");
}
}
