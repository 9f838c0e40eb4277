// Root-mean-square normalisation of rows behind a residual's addition: forward (also in 8 bits with a scale per row) and
// backward.
//   s = x [+ skip];  r = 1 / sqrt(mean(s^2) + eps);  y = s r w;  q = y / scale, scale = max|y| / 127
//   g = dy w;  dx = r (g - s r^2 mean(g s)) [+ ds];  dw = sum over rows of dy s r
// Both passes move bytes and nothing else (ten flops an element): a row is read once, into registers, its sums are formed
// over the threads that hold it, and what the pass writes is formed from the same registers.  The statistics are not kept
// for the way back: s is read there anyway, and its sum of squares comes with the other sum of the row.
// A row has a wave of its own where there are rows enough to fill the chip with waves (no barrier, no LDS), else a
// workgroup.  Rows that no workgroup can hold (more than 65536 values in fp16, 32768 in fp32) are read twice.
#include "ptl_rows.hpp"
#include "ptl_transformer.h"

namespace ptl {

template <typename T>
struct NormFw {
    const T *x, *skip, *w;
    T *sum, *y;
    int8_t *q;
    float *scale;
    int rows, dim;
    float eps;
};

// The eight-bit integers of VEC values: one store of VEC bytes where the row has all of them.
template <int VEC>
__device__ inline void put_q(int8_t *row, int p, int dim, const int (&q)[VEC]) {
    const int at = p * VEC;
    if (at + VEC <= dim) {
        unsigned u[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i)
            u[i] = (q[4 * i] & 255) | (q[4 * i + 1] & 255) << 8 | (q[4 * i + 2] & 255) << 16 | (unsigned)q[4 * i + 3] << 24;
        if constexpr (VEC == 8) *reinterpret_cast<row_u2 *>(row + at) = row_u2{u[0], u[1]};
        else *reinterpret_cast<row_u1 *>(row + at) = u[0];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (at + i < dim) row[at + i] = (int8_t)q[i];
    }
}

// NP pieces of a row in each of its TPR threads; NP = 0: the row is walked twice, in the same pieces.
template <typename T, int TPR, int NP, bool Q8>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void rms_norm_fw_kernel(const NormFw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC, HELD = NP ? NP : 1;
    __shared__ float red[16][2];
    const int t = TPR == 64 ? (threadIdx.x & 63) : threadIdx.x;
    const long row = TPR == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= a.rows) return;  // (a whole wave, which has no barrier to meet)
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    const size_t at = (size_t)row * dim;
    float s[HELD][VEC];
    Piece w[HELD];
    float v[2] = {0.f, 0.f};  // sum of squares, largest |s w|
    auto join = [&](Piece x, Piece k, int p, float (&f)[VEC]) {
        x.trim(p, dim);
        if (a.skip) k.trim(p, dim);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = a.skip ? (float)x.e[i] + (float)k.e[i] : (float)x.e[i];
    };
    auto fetch = [&](int p, float (&f)[VEC]) {
        Piece x, k;
        x.fetch(a.x + at, p, dim);
        if (a.skip) k.fetch(a.skip + at, p, dim);
        join(x, k, p, f);
    };
    auto add = [&](const float (&f)[VEC], const Piece &w) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[0] = fmaf(f[i], f[i], v[0]);
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[1] = fmaxf(v[1], fabsf(f[i] * (float)w.e[i]));
        }
    };
    if constexpr (NP > 0) {
        Piece x[HELD], k[HELD];
#pragma unroll
        for (int j = 0; j < NP; ++j) x[j].fetch(a.x + at, j * TPR + t, dim);
#pragma unroll
        for (int j = 0; j < NP; ++j) w[j].fetch(a.w, j * TPR + t, dim);
        if (a.skip) {
#pragma unroll
            for (int j = 0; j < NP; ++j) k[j].fetch(a.skip + at, j * TPR + t, dim);
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            join(x[j], k[j], j * TPR + t, s[j]);  // (pieces behind the end are zeros)
            w[j].trim(j * TPR + t, dim);
            add(s[j], w[j]);
        }
    } else {
        for (int p = t; p < pieces; p += TPR) {
            fetch(p, s[0]);
            w[0].load(a.w, p, dim);
            add(s[0], w[0]);
        }
    }
    row_reduce<TPR, 2, true>(v, red);
    const float r = 1.f / sqrtf(v[0] / (float)dim + a.eps);
    // (a row of zeros: all zeros; otherwise the largest value becomes 127 to within a rounding of the product)
    const float unit = v[1] > 0.f ? 127.f / v[1] : 0.f;
    auto put = [&](int p, const float (&f)[VEC], const Piece &w) {
        if (p >= pieces) return;
        Piece o;
        if (a.skip) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.e[i] = (T)f[i];
            o.store(a.sum + at, p, dim);
        }
        if (a.y) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.e[i] = (T)(f[i] * r * (float)w.e[i]);
            o.store(a.y + at, p, dim);
        }
        if constexpr (Q8) {
            int q[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) q[i] = (int)fminf(fmaxf(rintf(f[i] * (float)w.e[i] * unit), -127.f), 127.f);
            put_q<VEC>(a.q + at, p, dim, q);
        }
    };
    if constexpr (NP > 0) {
#pragma unroll
        for (int j = 0; j < NP; ++j) put(j * TPR + t, s[j], w[j]);
    } else {
        for (int p = t; p < pieces; p += TPR) {
            fetch(p, s[0]);
            w[0].load(a.w, p, dim);
            put(p, s[0], w[0]);
        }
    }
    // infinities and NaN: v[0] is then no finite number, and neither is the scale
    if (Q8 && t == 0) a.scale[row] = v[0] < __builtin_inff() ? v[1] * r / 127.f : __builtin_nanf("");
}

template <typename T, int TPR, int NP>
static void norm_fw_launch(const NormFw<T> &a) {
    const dim3 grid(TPR == 64 ? (a.rows + 3) / 4 : a.rows), block(TPR == 64 ? 256 : TPR);
    if (a.q) hipLaunchKernelGGL((rms_norm_fw_kernel<T, TPR, NP, true>), grid, block, 0, state().stream, a);
    else hipLaunchKernelGGL((rms_norm_fw_kernel<T, TPR, NP, false>), grid, block, 0, state().stream, a);
}

template <typename T>
static void norm_fw(const NormFw<T> &a) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC;
    if (a.rows >= 1024 && pieces <= 512) {
        if (pieces <= 64) return norm_fw_launch<T, 64, 1>(a);
        if (pieces <= 128) return norm_fw_launch<T, 64, 2>(a);
        if (pieces <= 256) return norm_fw_launch<T, 64, 4>(a);
        return norm_fw_launch<T, 64, 8>(a);
    }
    if (pieces <= 64) return norm_fw_launch<T, 64, 1>(a);
    if (pieces <= 256) return norm_fw_launch<T, 256, 1>(a);
    if (pieces <= 512) return norm_fw_launch<T, 256, 2>(a);
    if (pieces <= 1024) return norm_fw_launch<T, 256, 4>(a);
    if (pieces <= 4096) return norm_fw_launch<T, 1024, 4>(a);
    if (pieces <= 8192) return norm_fw_launch<T, 1024, 8>(a);
    norm_fw_launch<T, 1024, 0>(a);
}

template <typename T>
struct NormBw {
    const T *s, *dy, *add, *w;
    T *dx, *dx2;  // (NULL: not wanted)
    float *part;  // of dw: a row for each wave or workgroup (NULL: not wanted)
    float *stat;  // long rows: r and r^3 mean(g s) of each row
    int rows, dim;
    float eps;
};

template <typename T>
__device__ inline float norm_dx(float s, float g, float add, float r, float m) { return fmaf(r, g, fmaf(-m, s, add)); }

// Workgroups walk over rows and keep their share of dw in registers: it is written once, at the end.
template <typename T, int TPR, int NP>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void rms_norm_bw_kernel(const NormBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC, PER = TPR == 64 ? 4 : 1;
    __shared__ float red[2][16][2];
    const int t = TPR == 64 ? (threadIdx.x & 63) : threadIdx.x;
    const int first = TPR == 64 ? (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6) : (int)blockIdx.x;
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    Piece w[NP];
    float dw[NP][VEC];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        w[j].load(a.w, j * TPR + t, dim);
#pragma unroll
        for (int i = 0; i < VEC; ++i) dw[j][i] = 0.f;
    }
    int turn = 0;
    for (long row = first; row < a.rows; row += (long)gridDim.x * PER, turn ^= 1) {
        const size_t at = (size_t)row * dim;
        Piece s[NP], g[NP], d[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            s[j].fetch(a.s + at, j * TPR + t, dim);
            g[j].fetch(a.dy + at, j * TPR + t, dim);
        }
        if (a.add) {
#pragma unroll
            for (int j = 0; j < NP; ++j) d[j].fetch(a.add + at, j * TPR + t, dim);
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            s[j].trim(j * TPR + t, dim);
            g[j].trim(j * TPR + t, dim);
            if (a.add) d[j].trim(j * TPR + t, dim);
        }
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float f = (float)s[j].e[i];
                v[0] = fmaf(f, f, v[0]);
                v[1] = fmaf((float)g[j].e[i] * (float)w[j].e[i], f, v[1]);
            }
        row_reduce<TPR, 2>(v, red[turn]);
        const float r = 1.f / sqrtf(v[0] / (float)dim + a.eps), m = r * r * r * (v[1] / (float)dim);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int p = j * TPR + t;
#pragma unroll
            for (int i = 0; i < VEC; ++i) dw[j][i] = fmaf((float)g[j].e[i], (float)s[j].e[i] * r, dw[j][i]);
            if (!a.dx || p >= pieces) continue;
            Piece o;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                o.e[i] = (T)norm_dx<T>((float)s[j].e[i], (float)g[j].e[i] * (float)w[j].e[i], a.add ? (float)d[j].e[i] : 0.f, r, m);
            o.store(a.dx + at, p, dim);
            if (a.dx2) o.store(a.dx2 + at, p, dim);
        }
    }
    if (!a.part) return;
    float *out = a.part + (size_t)first * dim;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int at = (j * TPR + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (at + i < dim) out[at + i] = dw[j][i];
    }
}

// Rows that no workgroup holds: the statistics of a row, then the columns.
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_stat_kernel(const NormBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    __shared__ float red[16][2];
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    const size_t at = (size_t)blockIdx.x * dim;
    float v[2] = {0.f, 0.f};
    for (int p = threadIdx.x; p < pieces; p += 1024) {
        Piece s, g, w;
        s.load(a.s + at, p, dim);
        g.load(a.dy + at, p, dim);
        w.load(a.w, p, dim);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            v[0] = fmaf((float)s.e[i], (float)s.e[i], v[0]);
            v[1] = fmaf((float)g.e[i] * (float)w.e[i], (float)s.e[i], v[1]);
        }
    }
    row_reduce<1024, 2>(v, red);
    if (threadIdx.x == 0) {
        const float r = 1.f / sqrtf(v[0] / (float)dim + a.eps);
        a.stat[2 * (size_t)blockIdx.x] = r;
        a.stat[2 * (size_t)blockIdx.x + 1] = r * r * r * (v[1] / (float)dim);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void rms_norm_columns_kernel(const NormBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    const int dim = a.dim, p = (int)blockIdx.x * 256 + (int)threadIdx.x;
    if (p * (long)VEC >= dim) return;
    Piece w;
    w.load(a.w, p, dim);
    float dw[VEC] = {};
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const size_t at = (size_t)row * dim;
        const float r = a.stat[2 * row], m = a.stat[2 * row + 1];
        Piece s, g, d, o;
        s.load(a.s + at, p, dim);
        g.load(a.dy + at, p, dim);
        if (a.add) d.load(a.add + at, p, dim);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            dw[i] = fmaf((float)g.e[i], (float)s.e[i] * r, dw[i]);
            o.e[i] = (T)norm_dx<T>((float)s.e[i], (float)g.e[i] * (float)w.e[i], a.add ? (float)d.e[i] : 0.f, r, m);
        }
        if (a.dx) o.store(a.dx + at, p, dim);
        if (a.dx2) o.store(a.dx2 + at, p, dim);
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (p * VEC + i < dim) a.part[(size_t)blockIdx.y * dim + p * VEC + i] = dw[i];
}

template <typename T, int TPR, int NP>
static int norm_bw_launch(NormBw<T> &a, T *dw) {
    constexpr int PER = TPR == 64 ? 4 : 1;
    const int per_cu = TPR == 512 ? 2 : 4;
    const long want = ((long)a.rows + PER - 1) / PER, most = (long)per_cu * state().num_cu;
    const int grid = (int)(want < most ? want : most), shares = grid * PER;
    if (dw && !(a.part = workspace((size_t)shares * a.dim * sizeof(float)))) return 2;
    hipLaunchKernelGGL((rms_norm_bw_kernel<T, TPR, NP>), dim3(grid), dim3(TPR == 64 ? 256 : TPR), 0, state().stream, a);
    if (dw) row_shares<T>(a.part, dw, a.dim, shares);
    return hip_ok(hipGetLastError(), "rms norm launch") ? 0 : 2;
}

template <typename T>
static int norm_bw(NormBw<T> &a, T *dw) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC;
    if (pieces <= 64) return norm_bw_launch<T, 64, 1>(a, dw);
    if (pieces <= 256) return norm_bw_launch<T, 256, 1>(a, dw);
    if (pieces <= 512) return norm_bw_launch<T, 256, 2>(a, dw);
    if (pieces <= 1024) return norm_bw_launch<T, 256, 4>(a, dw);
    if (pieces <= 2048) return norm_bw_launch<T, 512, 4>(a, dw);
    const int shares = a.rows < 64 ? a.rows : 64;
    const size_t stat = (size_t)a.rows * 2;
    float *ws = workspace((stat + (dw ? (size_t)shares * a.dim : 0)) * sizeof(float));
    if (!ws) return 2;
    a.stat = ws;
    a.part = dw ? ws + stat : nullptr;
    hipLaunchKernelGGL((rms_norm_stat_kernel<T>), dim3(a.rows), dim3(1024), 0, state().stream, a);
    hipLaunchKernelGGL((rms_norm_columns_kernel<T>), dim3((pieces + 255) / 256, shares), dim3(256), 0, state().stream, a);
    if (dw) row_shares<T>(a.part, dw, a.dim, shares);
    return hip_ok(hipGetLastError(), "rms norm launch") ? 0 : 2;
}

template <typename T, typename Args>
static int rms_norm_step(const Args *a, int ns, bool back, const char *fn) {
    if (!a || !a->input || !a->coeff || (back && !a->output)) return rows_bad(fn, "null argument structure");
    const int dim = a->input->dim;
    if (dim <= 0 || dim > ROW_MOST) return rows_bad(fn, "invalid tensor geometry");
    if (!(a->eps >= 0.f && a->eps < __builtin_inff())) return rows_bad(fn, "eps is no finite number from 0 on");
    if (ns <= 0) return 0;
    auto as = [](auto *p) { return reinterpret_cast<T *>(p); };
    T *w = as(a->coeff->data), *sum = as(blob_data(a->sum)), *x = as(a->input->data);
    if (!w) return rows_bad(fn, "null buffer");
    if (a->skip && !sum) return rows_bad(fn, "a residual needs a buffer for the sum");
    const size_t n = (size_t)ns * dim;
    int rc;
    if (!back) {
        T *skip = as(blob_data(a->skip)), *y = as(blob_data(a->output));
        if (!x || (a->skip && !skip)) return rows_bad(fn, "null buffer");
        if (!y && !a->q_data) return rows_bad(fn, "no output is wanted");
        if (!a->q_data != !a->q_scale) return rows_bad(fn, "an output in 8 bits needs both q_data and q_scale");
        if (!ensure_init()) return 2;
        Stager sg;
        NormFw<T> k = {};
        k.x = sg.in<T>(x, n);
        k.w = sg.in<T>(w, (size_t)dim);
        if (a->skip) {
            k.skip = sg.in<T>(skip, n);
            k.sum = sg.out<T>(sum, n);
        }
        if (y) k.y = sg.out<T>(y, n);
        if (a->q_data) {
            k.q = sg.out<int8_t>(a->q_data, n);
            k.scale = sg.out<float>(a->q_scale, (size_t)ns);
        }
        if (sg.failed()) return 2;
        k.rows = ns;
        k.dim = dim;
        k.eps = a->eps;
        norm_fw<T>(k);
        rc = hip_ok(hipGetLastError(), "rms norm launch") ? 0 : 2;
        return sg.finish(rc);
    }
    T *s = sum ? sum : x, *dy = as(a->output->diff), *add = as(blob_diff(a->sum));
    T *dx = a->skip_in_grad ? nullptr : as(a->input->diff), *dx2 = a->skip_in_grad ? nullptr : as(blob_diff(a->skip));
    T *dw = a->skip_wg_grad ? nullptr : as(a->coeff->diff);
    if (!s || !dy || (!a->skip_in_grad && !dx) || (!a->skip_wg_grad && !dw)) return rows_bad(fn, "null buffer");
    if (!dx && !dw) return 0;
    if (dx2 == dx) dx2 = nullptr;
    if (!ensure_init()) return 2;
    Stager sg;
    NormBw<T> k = {};
    k.s = sg.in<T>(s, n);
    k.dy = sg.in<T>(dy, n);
    k.w = sg.in<T>(w, (size_t)dim);
    if (add) k.add = sg.in<T>(add, n);
    if (dx) k.dx = sg.out<T>(dx, n);
    if (dx2) k.dx2 = sg.out<T>(dx2, n);
    T *dwd = dw ? sg.out<T>(dw, (size_t)dim) : nullptr;
    if (sg.failed()) return 2;
    k.rows = ns;
    k.dim = dim;
    k.eps = a->eps;
    rc = norm_bw<T>(k, dwd);
    return sg.finish(rc);
}

}  // namespace ptl

extern "C" {
int ptl_rms_norm_fp32_fw_batched(const struct RmsNorm_args *a, int ns) {
    return ptl::rms_norm_step<float>(a, ns, false, "ptl_rms_norm_fp32_fw_batched");
}
int ptl_rms_norm_fp32_bw_batched(const struct RmsNorm_args *a, int ns) {
    return ptl::rms_norm_step<float>(a, ns, true, "ptl_rms_norm_fp32_bw_batched");
}
int ptl_rms_norm_fp16_fw_batched(const struct RmsNorm_args_fp16 *a, int ns) {
    return ptl::rms_norm_step<ptl::half_t>(a, ns, false, "ptl_rms_norm_fp16_fw_batched");
}
int ptl_rms_norm_fp16_bw_batched(const struct RmsNorm_args_fp16 *a, int ns) {
    return ptl::rms_norm_step<ptl::half_t>(a, ns, true, "ptl_rms_norm_fp16_bw_batched");
}
}
