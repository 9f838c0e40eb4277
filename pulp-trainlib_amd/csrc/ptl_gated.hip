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
// behind (NULL: not wanted).  low: in the same layout, what dh lost by rounding, GRAD_LOW times; the sums are then of dh before it (NULL:
// not wanted).
template <typename T>
__global__ __launch_bounds__(256) void gate_back_kernel(const T *h, const T *__restrict__ dy, T *dh, float *__restrict__ part, size_t rows, int outs,
                                                        int act, T *__restrict__ copy, T *__restrict__ low, int pitch) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    const int pieces = (outs + VEC - 1) / VEC, p = (int)(blockIdx.x * 256 + threadIdx.x);
    if (p >= pieces) return;
    const Gate gate(act);
    float sum[2][VEC] = {};
    for (size_t row = blockIdx.y; row < rows; row += gridDim.y) {
        Piece g, u, d, og, ou;
        float fg[VEC], fu[VEC];
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
            og.e[i] = (T)(fg[i] = (float)d.e[i] * (float)u.e[i] * df);
            ou.e[i] = (T)(fu[i] = (float)d.e[i] * f);
        }
        // (the sums are of the values that are stored: formed again for them, with other roundings in between, one in thousands would differ)
        asm volatile("" : "+v"(og.raw), "+v"(ou.raw));
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            sum[0][i] += low ? fg[i] : (float)og.e[i];
            sum[1][i] += low ? fu[i] : (float)ou.e[i];
        }
        og.store(dh + row * 2 * outs, p, outs);
        ou.store(dh + row * 2 * outs + outs, p, outs);
        if (copy) {
            T *to = copy + row * pitch;
            og.store(to, p, outs);
            ou.store(to + outs, p, outs);
            for (int i = 2 * outs + p; p < 8 && i < pitch; i += pieces) to[i] = (T)0.f;
        }
        if (low) {
            T *to = low + row * pitch;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {  // (nothing is left of what became infinite)
                og.e[i] = (T)(fabsf((float)og.e[i]) < __builtin_inff() ? (fg[i] - (float)og.e[i]) * GRAD_LOW : 0.f);
                ou.e[i] = (T)(fabsf((float)ou.e[i]) < __builtin_inff() ? (fu[i] - (float)ou.e[i]) * GRAD_LOW : 0.f);
            }
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

// The whole backward pass of up to eight tokens.  A workgroup has `high` rows of the weights and 64 pieces of columns; its waves share the
// rows.  It forms dh of its rows for all tokens (in fp32, which is what the products read), passes over the weights once for dx, of which
// every group of rows leaves sums (another launch adds them up), and writes dw.  The weights' bytes, read and written, are all it moves:
// one token, 4096 -> 8000 63 us in fp16 (4.2 TB/s), 106 in fp32 (4.9); small layers 6 to 9 us, two launches.
template <typename T>
struct GateFew {
    const T *h, *dy, *x, *w;
    T *dh, *dw, *dx, *db;  // (dw, dx, db NULL: not wanted)
    float *part;           // of dx: groups of rows x tokens x in (NULL: one group, which writes dx)
    int ns, in, outs, high, act;
};
constexpr int GATE_HIGH = 512;
template <typename T, int NS>
__global__ __launch_bounds__(256) void gate_few_kernel(const GateFew<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC, U = NS > 4 ? 2 : 4;
    __shared__ float g[NS][GATE_HIGH], red[NS * VEC][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), in = a.in, rows = 2 * a.outs;
    const int r0 = (int)blockIdx.y * a.high, n = min(a.high, rows - r0), p = (int)blockIdx.x * 64 + lane, pieces = (in + VEC - 1) / VEC;
    const Gate gate(a.act);
    for (int r = tid; r < n; r += 256) {
        const int o = r0 + r < a.outs ? r0 + r : r0 + r - a.outs;
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < NS; ++t) {
            if (t >= a.ns) {
                g[t][r] = 0.f;
                continue;
            }
            const T *h = a.h + (size_t)t * rows;
            const float up = (float)h[a.outs + o], d = (float)a.dy[(size_t)t * a.outs + o];
            float f;
            const float df = gate.back((float)h[o], f), v = r0 + r < a.outs ? d * up * df : d * f;
            g[t][r] = v;
            sum += v;
            if (blockIdx.x == 0) a.dh[(size_t)t * rows + r0 + r] = (T)v;
        }
        if (a.db && blockIdx.x == 0) a.db[r0 + r] = (T)sum;
    }
    __syncthreads();
    Piece x[NS];
    float s[NS][VEC];
#pragma unroll
    for (int t = 0; t < NS; ++t) {
        if (a.dw && t < a.ns) x[t].template hold<true>(a.x + (size_t)t * in, p, in);
        else x[t].raw = row_u4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[t][i] = 0.f;
    }
    for (int r = wave; r < n; r += 4 * U) {
        Piece w[U];
        if (a.dx) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + 4 * u < n) w[u].template hold<true>(a.w + (size_t)(r0 + r + 4 * u) * in, p, in);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r + 4 * u >= n) break;
            float v[NS];
#pragma unroll
            for (int t = 0; t < NS; ++t) v[t] = g[t][r + 4 * u];
            if (a.dx) {
#pragma unroll
                for (int t = 0; t < NS; ++t)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) s[t][i] = fmaf(v[t], (float)w[u].e[i], s[t][i]);
            }
            if (a.dw) {
                Piece o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float f = v[0] * (float)x[0].e[i];
#pragma unroll
                    for (int t = 1; t < NS; ++t) f = fmaf(v[t], (float)x[t].e[i], f);
                    o.e[i] = row_round<T>(f);
                }
                o.template put<true>(a.dw + (size_t)(r0 + r + 4 * u) * in, p, in);
            }
        }
    }
    if (!a.dx) return;
    for (int k = 0; k < 4; ++k) {  // the waves' sums, in their order
        if (wave == k) {
#pragma unroll
            for (int t = 0; t < NS; ++t)
#pragma unroll
                for (int i = 0; i < VEC; ++i) red[t * VEC + i][lane] = k ? red[t * VEC + i][lane] + s[t][i] : s[t][i];
        }
        __syncthreads();
    }
    if (p >= pieces) return;
    for (int t = wave; t < a.ns; t += 4) {
        const int at = p * VEC - Piece::cut(p, in);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (at + i >= in) break;
            const float v = red[t * VEC + i][lane];
            if (a.part) a.part[((size_t)blockIdx.y * a.ns + t) * in + at + i] = v;
            else a.dx[(size_t)t * in + at + i] = (T)v;
        }
    }
}
template <typename T>
static int gate_few(GateFew<T> a) {
    const size_t n_h = (size_t)a.ns * 2 * a.outs * sizeof(T);
    T *copy = nullptr;  // of h, where dh takes its place: workgroups read what others write over
    if (a.h == a.dh && !(copy = static_cast<T *>(scratch(n_h + 16)))) return 2;
    const int rows = 2 * a.outs, wide = ((a.in + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC + 63) / 64, cu = state().num_cu;
    // four workgroups a compute unit, of sixteen rows and more (2 tokens, 4096 -> 8000 in fp16 with two, four, six 95, 65 and 67 us)
    int high = (int)((long)rows * wide / (4 * cu));
    high = high < 16 ? 16 : high > GATE_HIGH ? GATE_HIGH : high;
    a.high = high;
    const int groups = (rows + high - 1) / high;
    T *dx = a.dx;
    if (dx && groups > 1 && !(a.part = workspace((size_t)groups * a.ns * a.in * sizeof(float)))) return 2;
    if (copy) {
        rows_copy(a.h, 1, nullptr, 0, copy, (int)n_h, (int)((n_h + 15) / 16 * 16));
        a.h = copy;
    }
    const dim3 grid(wide, groups);
    if (a.ns == 1) hipLaunchKernelGGL((gate_few_kernel<T, 1>), grid, dim3(256), 0, state().stream, a);
    else if (a.ns == 2) hipLaunchKernelGGL((gate_few_kernel<T, 2>), grid, dim3(256), 0, state().stream, a);
    else if (a.ns <= 4) hipLaunchKernelGGL((gate_few_kernel<T, 4>), grid, dim3(256), 0, state().stream, a);
    else hipLaunchKernelGGL((gate_few_kernel<T, 8>), grid, dim3(256), 0, state().stream, a);
    if (a.part) row_shares<T>(a.part, dx, a.ns * a.in, groups);
    return hip_ok(hipGetLastError(), "gated layer launch") ? 0 : 2;
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

// fp16: where there are few of them, the products are of the pre-activations' gradients before they are rounded, in two halves.  Rounded
// ones add an error as large as the rounding of the results (both together 1.41 times that); of so few, in a single token of a small
// layer, it can be twice that.  (20 tokens, 100 -> 400 11 us, so 17.)
template <typename T>
static bool few_gradients(int ns, int in, int outs) {
    return sizeof(T) == 2 && in < 1 << 23 && (double)ns * 2 * outs < 16384 && state().gemm_path == 0;
}
// Which calls gate_few() takes: in halves the same 1.1 to 4 times as long; against a dense layer's call one and two tokens 0.92 to 1.37 times
// as fast, in fp32 three and four 0.9 to 1.15 up to 7 million weights of either half (beyond, in rows that are no whole pieces, 0.82 to 0.9;
// in fp16 0.75 to 1.1).
template <typename T>
static bool few_tokens(int ns, int in, int outs) {
    const bool fits = (double)ns * in < ROW_MOST && outs < GATE_HIGH * 32000;  // (columns of a sum of shares, groups of rows)
    const bool pays = ns <= 2 || (sizeof(T) == 4 && ns <= 4 && (double)in * outs <= 7e6) || (ns <= 8 && few_gradients<T>(ns, in, outs));
    return fits && pays && state().gemm_path == 0;
}

// What the sums of a dense layer's backward call take at most: of each product its outputs, in rows of whole pieces whichever operand goes
// first, and the bias' sums for every part of k, none of which is shorter than 256 bytes; or the bias' shares, one for every 128 tokens.
template <typename T>
static size_t dense_workspace(int ns, int in, int out) {
    constexpr size_t KS = 256 / sizeof(T);
    auto parts = [](size_t k) { return (k + KS - 1) / KS; };
    return sizeof(float) * (parts(ns) * ((size_t)out + 8) * ((size_t)in + 16) + parts(out) * ((size_t)ns + 8) * ((size_t)in + 16) + (size_t)(ns / 128 + 1) * out);
}

template <typename T, typename Linear, typename Args>
static int gated_back(const Args *a, int ns, int in, int outs, bool bias, bool wg, bool ig) {
    auto as = [](auto *p) { return reinterpret_cast<T *>(p); };
    const size_t nx = (size_t)ns * in, ny = (size_t)ns * outs, nw = (size_t)2 * outs * in;
    Stager sg;
    const T *h = sg.in<T>(as(a->hidden->data), 2 * ny), *dy = sg.in<T>(as(a->output->diff), ny);
    T *dh = sg.out<T>(as(a->hidden->diff), 2 * ny);
    if (sg.failed()) return 2;
    const T *x = wg ? sg.in<T>(as(a->input->data), nx) : nullptr, *w = ig ? sg.in<T>(as(a->coeff->data), nw) : nullptr;
    T *dw = wg ? sg.out<T>(as(a->coeff->diff), nw) : nullptr, *dx = ig ? sg.out<T>(as(a->input->diff), nx) : nullptr;
    T *db = wg && bias ? sg.out<T>(as(a->bias->diff), (size_t)2 * outs) : nullptr;
    if (sg.failed()) return 2;
    if ((wg || ig) && few_tokens<T>(ns, in, outs)) {
        GateFew<T> k = {};
        k.h = h;
        k.dy = dy;
        k.x = x;
        k.w = w;
        k.dh = dh;
        k.dw = dw;
        k.dx = dx;
        k.db = db;
        k.ns = ns;
        k.in = in;
        k.outs = outs;
        k.act = a->activation;
        return sg.finish(gate_few(k));
    }
    // rows that are no whole 16-byte pieces are copied to such; dh is written a second time
    constexpr int VEC = RowPiece<T>::VEC;
    const int cols = (in + VEC - 1) / VEC * VEC, pitch = (2 * outs + VEC - 1) / VEC * VEC;
    bool copy_x = ((uintptr_t)x | (uintptr_t)w) % 16 || cols != in, copy_dh = (uintptr_t)dh % 16 || pitch != 2 * outs;
    const bool few = few_gradients<T>(ns, in, outs) && (wg || ig), own = few || own_products<T>(ns, in, outs, copy_x || copy_dh);
    copy_x = copy_x && own;
    copy_dh = copy_dh && own;
    // All the memory comes before the first launch: a call that cannot have it leaves the pre-activations as they are, also where the
    // gradients take their place.
    T *wide_w = nullptr, *wide_x = nullptr, *wide_dh = nullptr, *low = nullptr;
    const size_t n_w = copy_x && w ? (size_t)2 * outs * cols : 0, n_x = copy_x && x ? (size_t)ns * cols : 0, n_dh = copy_dh ? (size_t)ns * pitch : 0, n_low = few ? (size_t)ns * pitch : 0;
    if (copy_x || copy_dh || few) {
        wide_w = static_cast<T *>(scratch((n_w + n_x + n_dh + n_low) * sizeof(T)));
        if (!wide_w) return 2;
        wide_x = wide_w + n_w;
        if (copy_dh) wide_dh = wide_x + n_x;
        if (few) low = wide_x + n_x + n_dh;
    }
    const int wide = ((outs + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC + 255) / 256;
    int high = ns < 65535 ? ns : 65535;
    float *part = nullptr, *ws = nullptr;
    GradParts plan = {};
    if (own) {
        size_t need = 0;
        if (db) {  // its sums come with the gradients of the pre-activations: eight workgroups a compute unit
            const int most = (8 * state().num_cu + wide - 1) / wide;
            high = high < most ? high : most;
            need = (size_t)high * 2 * outs * sizeof(float);
        }
        if (int rc = gated_products_plan<T>(plan, wg, ig, few, ns, in, 2 * outs)) return rc;
        // (the parts of the products' sums lie where the bias' were: they are added up by then)
        need = need > plan.bytes ? need : plan.bytes;
        if (need && !(ws = workspace(need))) return 2;
        if (db) part = ws;
    }
    // A dense layer's call asks for its memory itself.  Where the gradients take the pre-activations' place, either there is as much as it
    // can ask for, or it reads them from a place of their own and they are formed again over the pre-activations once it went well (64
    // tokens, 512 -> 1408 in fp16 14.5 and 17.9 us).
    const bool dense = !own && (wg || ig);
    T *to = dh;
    if (dense && h == dh) {
        const size_t most = dense_workspace<T>(ns, in, 2 * outs);
        const bool there = most <= ((size_t)64 << 20) && workspace_if(most);
        if (!there && !(to = static_cast<T *>(scratch(2 * ny * sizeof(T))))) return 2;
    }
    auto gate_back = [&](T *out) {
        hipLaunchKernelGGL((gate_back_kernel<T>), dim3(wide, high), dim3(256), 0, state().stream, h, dy, out, part, (size_t)ns, outs, a->activation,
                           wide_dh, low, pitch);
        if (part) row_shares<T>(part, db, 2 * outs, high);
        return hip_ok(hipGetLastError(), "gated layer launch") ? 0 : 2;
    };
    if (n_w + n_x) rows_copy(w, w ? 2 * (size_t)outs : 0, x, x ? ns : 0, wide_w, in * (int)sizeof(T), cols * (int)sizeof(T));
    int rc = gate_back(to);
    if (rc == 0 && own && (wg || ig))
        rc = gated_products<T>(plan, ws, copy_x ? wide_x : x, copy_x ? wide_w : w, copy_dh ? wide_dh : dh, low, dw, dx, ns, in, 2 * outs, cols, pitch);
    if (to == dh) {
        rc = sg.finish(rc);
        if (rc || !dense) return rc;
    }
    if (rc) return rc;
    auto out = *a->hidden;  // a dense layer of 2 n_out outputs
    out.dim = 2 * outs;
    if (to != dh) out.diff = reinterpret_cast<decltype(out.diff)>(to);
    Linear l = {};
    l.input = a->input;
    l.coeff = a->coeff;
    l.bias = a->bias;
    l.output = &out;
    l.skip_wg_grad = a->skip_wg_grad;
    l.skip_in_grad = a->skip_in_grad;
    l.use_biases = a->use_biases;
    rc = linear_bw(&l, ns);
    if (to == dh) return rc;
    return sg.finish(rc ? rc : gate_back(dh));
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
