// Root-mean-square normalisation of rows behind a residual's addition: forward (also in 8 bits with a scale per row) and
// backward.
//   s = x [+ skip];  r = 1 / sqrt(mean(s^2) + eps);  y = s r w;  q = y / scale, scale = max|y| / 127
//   g = dy w;  dx = r (g - s r^2 mean(g s)) [+ ds];  dw = sum over rows of dy s r
// Both passes move bytes and nothing else (ten flops an element): a row is read once, into registers, its sums are formed
// over the threads that hold it, and what the pass writes is formed from the same registers.  The statistics are not kept
// for the way back: s is read there anyway, and its sum of squares comes with the other sum of the row.
// A row of up to 2048 bytes (4096 backward, in fp32) has a wave of its own (no barrier), a longer one a workgroup; rows that no workgroup
// holds (more than 4096 pieces of 16 bytes forward, 16384 values backward) are read twice.  Measured, with the residual's addition: 8192 rows of
// 4096 fp16 values forward 45 us, 5.9 TB/s (in 8 bits 42 us), backward with the weights' gradient 62 us, 4.3 TB/s;
// 8192 x 1024 14 and 23 us; a few rows 3.7 us, which is an empty launch, and backward 4 us for one to three,
// 7.3 for the two launches of more.
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
    int first;  // the launch's first row
    float eps;
};

// 1 / sqrt(mean + eps) of a row's sum of squares; 0 where both are 0 (a row of zeros, or of values so small that their squares are, with
// eps = 0): such a row has zeros, and the gradient reaches it along the residual only.
__device__ inline float norm_r(float sum, int dim, float eps) {
    const float q = sum / (float)dim + eps;
    return q == 0.f ? 0.f : 1.f / sqrtf(q);
}

// The eight-bit integers of VEC values, from element `at` on: one store of VEC bytes where the row has all of them (WHOLE: it has).
template <int VEC, bool WHOLE>
__device__ inline void put_q(int8_t *row, int at, int dim, const int (&q)[VEC]) {
    if (WHOLE || at + VEC <= dim) {
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
    constexpr bool SHORT = TPR * NP == 64;  // rows of less than a piece come here too
    __shared__ float red[16][2];
    const int t = TPR == 64 ? (threadIdx.x & 63) : threadIdx.x;
    const long row = a.first + (TPR == 64 ? (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x);
    if (row >= a.rows) return;  // (a whole wave, which has no barrier to meet)
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    const size_t at = (size_t)row * dim;
    auto none = [&](int j) { return j > NP / 2 && j * TPR >= pieces; };  // (pieces that no thread has; half of them someone has)
    float s[HELD][VEC];
    Piece w[HELD];
    float v[2] = {0.f, 0.f};  // sum of squares, largest |s w| (NaN where one is)
    auto join = [&](const Piece &x, const Piece &k, float (&f)[VEC]) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = a.skip ? (float)x.e[i] + (float)k.e[i] : (float)x.e[i];
    };
    auto add = [&](const float (&f)[VEC], const Piece &w, int cut) {
        if (__any(cut)) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[0] = i < cut ? v[0] : fmaf(f[i], f[i], v[0]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[0] = fmaf(f[i], f[i], v[0]);
        }
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[1] = nan_max(v[1], fabsf(f[i] * (float)w.e[i]));
        }
    };
    // (rows that are walked: a thread reads behind the barrier what another may have written over by then, so each has its own elements)
    auto walk = [&](int p, float (&f)[VEC], Piece &w) {
        Piece x, k;
        x.load(a.x + at, p, dim);
        if (a.skip) k.load(a.skip + at, p, dim);
        w.load(a.w, p, dim);
        join(x, k, f);
    };
    if constexpr (NP > 0) {
        Piece x[HELD], k[HELD];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            x[j].template hold<SHORT>(a.x + at, j * TPR + t, dim);
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            w[j].template hold<SHORT>(a.w, j * TPR + t, dim);
        }
        if (a.skip) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                k[j].template hold<SHORT>(a.skip + at, j * TPR + t, dim);
            }
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            join(x[j], k[j], s[j]);
            add(s[j], w[j], Piece::cut(j * TPR + t, dim));
        }
    } else {
        for (int p = t; p < pieces; p += TPR) {
            walk(p, s[0], w[0]);
            add(s[0], w[0], 0);
        }
    }
    row_reduce<TPR, 2, true>(v, red);
    const float r = norm_r(v[0], dim, a.eps);
    // (a row of zeros: all zeros; otherwise the largest value becomes 127 to within a rounding of the product)
    // (fp32: 127 / v[1] is infinite from 3.7e-37 down, and products there lose their bits: such rows are worked on 2^100 times as large)
    const float lift = sizeof(T) == 4 && v[1] < 0x1p-100f ? 0x1p100f : 1.f;
    const float unit = v[1] > 0.f && r > 0.f ? 127.f / (v[1] * lift) : 0.f;
    auto put = [&](int p, const float (&f)[VEC], const Piece &w) {
        if (p >= pieces) return;
        Piece o;
        auto out = [&](T *to) {
            if constexpr (NP > 0) o.template put<SHORT>(to, p, dim);
            else o.store(to, p, dim);
        };
        if (a.skip) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(f[i]);
            out(a.sum + at);
        }
        if (a.y) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(f[i] * r * (float)w.e[i]);
            out(a.y + at);
        }
        if constexpr (Q8) {
            int q[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) q[i] = (int)fminf(fmaxf(rintf((sizeof(T) == 4 ? f[i] * lift : f[i]) * (float)w.e[i] * unit), -127.f), 127.f);
            put_q<VEC, (NP > 0 && !SHORT)>(a.q + at, p * VEC - (NP > 0 ? Piece::cut(p, dim) : 0), dim, q);
        }
    };
    if constexpr (NP > 0) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            put(j * TPR + t, s[j], w[j]);
        }
    } else {
        for (int p = t; p < pieces; p += TPR) {
            walk(p, s[0], w[0]);
            put(p, s[0], w[0]);
        }
    }
    // infinities and NaN: v[0] or (of the weights) v[1] is then no finite number, and neither is the scale
    if (Q8 && t == 0) a.scale[row] = v[0] < __builtin_inff() ? v[1] * r / 127.f : __builtin_nanf("");
}

template <typename T, int TPR, int NP>
static void norm_fw_launch(NormFw<T> a) {
    const int all = a.rows, most = (int)(ROW_THREADS / TPR);
    for (; a.first < all; a.first += most) {
        const int n = all - a.first < most ? all - a.first : most;
        a.rows = a.first + n;
        const dim3 grid(TPR == 64 ? (n + 3) / 4 : n), block(TPR == 64 ? 256 : TPR);
        if (a.q) hipLaunchKernelGGL((rms_norm_fw_kernel<T, TPR, NP, true>), grid, block, 0, state().stream, a);
        else hipLaunchKernelGGL((rms_norm_fw_kernel<T, TPR, NP, false>), grid, block, 0, state().stream, a);
    }
}

template <typename T>
static void norm_fw(const NormFw<T> &a) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC;
    // A wave with four pieces would lose to a workgroup with one where rows are few (300 x 2048 fp16 in 8 bits: 4.1 against 3.9 us) and
    // gain nothing where they are many (8192 x 2048: 24.8 against 25.1); with two it gains (8192 x 1024: 13.8 against 15.2).
    if (pieces <= 64) return norm_fw_launch<T, 64, 1>(a);
    if (pieces <= 128) return norm_fw_launch<T, 64, 2>(a);
    if (pieces <= 256) return norm_fw_launch<T, 256, 1>(a);
    if (pieces <= 512) return norm_fw_launch<T, 256, 2>(a);
    if (pieces <= 1024) return norm_fw_launch<T, 512, 2>(a);
    // (every CU with rows: four waves a row, 2000 x 8192 fp32 48 against 51 us with eight; few rows: eight, 4 x 14144 fp16 3.7 against 4.2)
    if (pieces <= 2048 && a.rows >= state().num_cu) return norm_fw_launch<T, 256, 8>(a);
    if (pieces <= 2048) return norm_fw_launch<T, 512, 4>(a);
    if (pieces <= 4096) return norm_fw_launch<T, 512, 8>(a);
    // (1024 threads with eight pieces each would spill registers: 1000 x 40000 fp16 112 us, in 8 bits 172; read twice 71 and 63)
    norm_fw_launch<T, 1024, 0>(a);
}

template <typename T>
struct NormBw {
    const T *s, *dy, *add, *w;
    T *dx, *dx2;  // (NULL: not wanted)
    T *dw;        // where one workgroup has all the rows (else NULL)
    float *part;  // of dw: a row for each workgroup (NULL: not wanted)
    float *stat;  // long rows: r and r^2 mean(g s) of each row
    int rows, dim;
    int first;  // of the rows whose statistics a launch forms
    float eps;
};

// r (g - s m) + add with m = r^2 mean(g s), formed as r (r mean): each step is of the size of r or of g, where r^3 leaves fp32's range from
// rows of 1e-13 down and from 1e13 up.
__device__ inline float norm_m(float r, float sum, int dim) { return r * (r * (sum / (float)dim)); }
__device__ inline float norm_dx(float s, float g, float add, float r, float m) { return fmaf(r, fmaf(-m, s, g), add); }

// Whether registers hold two rows.
template <typename T, int TPR, int NP>
constexpr bool norm_ahead() { return NP * RowPiece<T>::VEC <= 16 && TPR <= 256; }
// Workgroups walk over rows and keep their share of dw in registers: it is written once, at the end.  The next row is on its way while
// one is worked on, as far as registers go.
template <typename T, int TPR, int NP>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void rms_norm_bw_kernel(const NormBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC, PER = TPR == 64 ? 4 : 1;
    constexpr bool AHEAD = norm_ahead<T, TPR, NP>(), SHORT = TPR * NP == 64;  // (rows of less than a piece come to the latter)
    // 128 registers a thread: the weights and their gradient are in LDS, the gradient along the residual is fetched when the sums are known
    constexpr bool LATE = TPR == 1024;
    __shared__ float red[2][16][2];
    const int t = TPR == 64 ? (threadIdx.x & 63) : threadIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long first = TPR == 64 ? (long)blockIdx.x * 4 + wave : blockIdx.x, stride = (long)gridDim.x * PER;
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    auto none = [&](int j) { return j > NP / 2 && j * TPR >= pieces; };  // (pieces that no thread has; half of them someone has)
    __shared__ row_u4 w_lds[LATE ? NP * TPR : 1];
    __shared__ row_f4 dw_lds[LATE ? NP * TPR : 1];
    Piece w[LATE ? 1 : NP];
    float dw[LATE ? 1 : NP][VEC];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        w[LATE ? 0 : j].template hold<SHORT>(a.w, j * TPR + t, dim);
        if constexpr (LATE) {  // (a thread's own)
            w_lds[j * TPR + t] = w[0].raw;
            dw_lds[j * TPR + t] = row_f4{0.f, 0.f, 0.f, 0.f};
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) dw[j][i] = 0.f;
        }
    }
    auto weights = [&](int j) {
        if constexpr (LATE) w[0].raw = w_lds[j * TPR + t];
        return w[LATE ? 0 : j];
    };
    auto gather = [&](int j) {
        if constexpr (LATE) {
            const row_f4 f = dw_lds[j * TPR + t];
#pragma unroll
            for (int i = 0; i < VEC; ++i) dw[0][i] = f[i];
        }
    };
    struct Row {
        Piece s[NP], g[NP], d[LATE ? 1 : NP];
    };
    // Where a row starts.  With the barrier it is one scalar, not an address for each piece of each tensor that goes along with the rows in
    // registers: 8192 x 4096 fp16 63.2 -> 61.6 us, 8192 x 1024 23.1 -> 21.9; with one piece a thread or four the addresses cost less than
    // what they save (8192 x 2048 35.3 us, 38.2 without them; 5946 x 8243 125 and 132).
    auto start = [&](long row) {
        size_t at = (size_t)row * dim;
        if constexpr (NP == 2 || LATE) asm volatile("" : "+s"(at));
        return at;
    };
    auto fetch = [&](long row, Row &r) {
        const size_t at = start(row);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            r.s[j].template hold<SHORT>(a.s + at, j * TPR + t, dim);
            r.g[j].template hold<SHORT>(a.dy + at, j * TPR + t, dim);
        }
        if (!LATE && a.add) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                r.d[j].template hold<SHORT>(a.add + at, j * TPR + t, dim);
            }
        }
    };
    int turn = 0;
    auto work = [&](long row, Row &x) {
        const size_t at = start(row);
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            const int cut = Piece::cut(j * TPR + t, dim);
            const Piece wj = weights(j);
            auto add = [&](int i) {
                const float f = (float)x.s[j].e[i];
                v[0] = fmaf(f, f, v[0]);
                v[1] = fmaf((float)x.g[j].e[i] * (float)wj.e[i], f, v[1]);
            };
            if (__any(cut)) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (i >= cut) add(i);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) add(i);
            }
        }
        row_reduce<TPR, 2>(v, red[turn]);
        turn ^= 1;
        const float r = norm_r(v[0], dim, a.eps), m = norm_m(r, v[1], dim);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            if constexpr (LATE) __builtin_amdgcn_sched_barrier(0);  // (one piece at a time, for its registers)
            const int p = j * TPR + t;
            gather(j);
#pragma unroll
            for (int i = 0; i < VEC; ++i) dw[LATE ? 0 : j][i] = fmaf((float)x.g[j].e[i], (float)x.s[j].e[i] * r, dw[LATE ? 0 : j][i]);
            if constexpr (LATE) dw_lds[j * TPR + t] = row_f4{dw[0][0], dw[0][1], dw[0][2], dw[0][3]};
            if (!a.dx || p >= pieces) continue;
            if constexpr (LATE) {
                if (a.add) x.d[0].template hold<SHORT>(a.add + at, p, dim);
            }
            const Piece wj = weights(j), &d = x.d[LATE ? 0 : j];
            Piece o;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                o.e[i] = row_round<T>(norm_dx((float)x.s[j].e[i], (float)x.g[j].e[i] * (float)wj.e[i], a.add ? (float)d.e[i] : 0.f, r, m));
            const int cut = LATE ? Piece::cut(p, dim) : 0;
            if (cut) {  // (a.add, read late, may be in the place of dx: another thread's elements are left to it)
#pragma unroll
                for (int i = 1; i < VEC; ++i) {
                    if (i < cut) continue;
                    a.dx[at + p * VEC - cut + i] = o.e[i];
                    if (a.dx2) a.dx2[at + p * VEC - cut + i] = o.e[i];
                }
                continue;
            }
            o.template put<SHORT>(a.dx + at, p, dim);
            if (a.dx2) o.template put<SHORT>(a.dx2 + at, p, dim);
        }
    };
    if constexpr (AHEAD) {
        Row x, y;
        long row = first;
        if (row < a.rows) fetch(row, x);
        for (; row < a.rows; row += 2 * stride) {
            if (row + stride < a.rows) fetch(row + stride, y);
            work(row, x);
            if (row + stride >= a.rows) break;
            if (row + 2 * stride < a.rows) fetch(row + 2 * stride, x);
            work(row + stride, y);
        }
    } else {
        Row x;
        for (long row = first; row < a.rows; row += stride) {
            fetch(row, x);
            work(row, x);
        }
    }
    if (!a.part && !a.dw) return;
    auto out = [&](int c, float v) {
        if (a.dw) a.dw[c] = (T)v;
        else a.part[(size_t)blockIdx.x * dim + c] = v;
    };
    if constexpr (TPR == 64) {  // the four waves' shares as one
        __shared__ float all[4][64 * NP * VEC];
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i >= Piece::cut(j * 64 + t, dim)) all[wave][(j * 64 + t) * VEC - Piece::cut(j * 64 + t, dim) + i] = dw[j][i];
        __syncthreads();
        for (int c = threadIdx.x; c < dim; c += 256) out(c, all[0][c] + all[1][c] + (all[2][c] + all[3][c]));
    } else if (a.dw) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            gather(j);
            Piece o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(dw[LATE ? 0 : j][i]);
            o.template put<SHORT>(a.dw, j * TPR + t, dim);
        }
    } else {
        float *part = a.part + (size_t)blockIdx.x * dim;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int p = j * TPR + t;
            if (p >= pieces) continue;
            gather(j);
#pragma unroll
            for (int i = 0; i < VEC; i += 4)
                *reinterpret_cast<row_u4 *>(part + p * VEC - Piece::cut(p, dim) + i) =
                    __builtin_bit_cast(row_u4, row_f4{dw[LATE ? 0 : j][i], dw[LATE ? 0 : j][i + 1], dw[LATE ? 0 : j][i + 2], dw[LATE ? 0 : j][i + 3]});
        }
    }
}

// Rows that no workgroup holds: the statistics of a row, then the columns.
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_stat_kernel(const NormBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    __shared__ float red[16][2];
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    const size_t row = (size_t)a.first + blockIdx.x, at = row * dim;
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
        const float r = norm_r(v[0], dim, a.eps);
        a.stat[2 * row] = r;
        a.stat[2 * row + 1] = norm_m(r, v[1], dim);
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
            o.e[i] = (T)norm_dx((float)s.e[i], (float)g.e[i] * (float)w.e[i], a.add ? (float)d.e[i] : 0.f, r, m);
        }
        if (a.dx) o.store(a.dx + at, p, dim);
        if (a.dx2) o.store(a.dx2 + at, p, dim);
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (p * VEC + i < dim) a.part[(size_t)blockIdx.y * dim + p * VEC + i] = dw[i];
}

// How many workgroups: the more of them, the faster the rows pass (a workgroup moves about 35 GB/s, up to what memory gives), and the
// more shares of dw are written and read (8 bytes a column and workgroup, at 5 TB/s); the sum of both times is least at
// sqrt(72 rows sizeof(T)).  Measured with 72, 208 and 600: 8192 x 1024 fp16 23.4, 26.4 and 26.5 us, 2000 x 8192 fp16 39.1, 37.9 and 43.5,
// 8192 x 2048 fp32 57.8, 63.5 and 68.1.
template <typename T>
static int norm_groups(int rows, int per) {
    const int groups = (rows + per - 1) / per, best = (int)sqrtf(72.f * (float)rows * sizeof(T));
    return groups < best ? groups : best > 1 ? best : 1;
}
template <typename T, int TPR, int NP>
static int norm_bw_launch(NormBw<T> &a, T *dw) {
    constexpr int per = TPR == 64 ? 4 : 1;
    // Few rows: one workgroup writes dw itself, no second launch (3 x 4096 fp16 5.2 us, with it 7.7; of the longer rows, which wait for
    // memory one by one, only one: 2 x 16384 8.0 us either way, 3 10.8 against 8.0).
    constexpr int few = norm_ahead<T, TPR, NP>() ? 3 : 1;
    const int grid = a.rows <= few * per ? 1 : norm_groups<T>(a.rows, per);
    if (grid == 1) a.dw = dw;
    else if (dw && !(a.part = workspace((size_t)grid * a.dim * sizeof(float)))) return 2;
    hipLaunchKernelGGL((rms_norm_bw_kernel<T, TPR, NP>), dim3(grid), dim3(TPR == 64 ? 256 : TPR), 0, state().stream, a);
    if (a.part) row_shares<T>(a.part, dw, a.dim, grid);
    return hip_ok(hipGetLastError(), "rms norm launch") ? 0 : 2;
}

template <typename T>
static int norm_bw(NormBw<T> &a, T *dw) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC;
    // (a wave for up to 1024 values: 8192 x 1024 fp16 23.4 us, by workgroups of one piece a thread 38.6; fp32 33.3 and 36.1)
    if (pieces <= 64) return norm_bw_launch<T, 64, 1>(a, dw);
    if (pieces <= 128) return norm_bw_launch<T, 64, 2>(a, dw);
    if constexpr (sizeof(T) == 4) {
        if (pieces <= 256) return norm_bw_launch<T, 64, 4>(a, dw);
    }
    if (pieces <= 256) return norm_bw_launch<T, 256, 1>(a, dw);
    if (pieces <= 512) return norm_bw_launch<T, 256, 2>(a, dw);
    if (pieces <= 1024) return norm_bw_launch<T, 256, 4>(a, dw);
    if (pieces <= 2048) return norm_bw_launch<T, 512, 4>(a, dw);
    if constexpr (sizeof(T) == 4) {  // (5946 x 8243 180 us, read twice 314; 300 x 16384 32 and 34)
        if (pieces <= 4096) return norm_bw_launch<T, 1024, 4>(a, dw);
    }
    const int shares = a.rows < 64 ? a.rows : 64;
    const size_t stat = (size_t)a.rows * 2;
    float *ws = workspace((stat + (dw ? (size_t)shares * a.dim : 0)) * sizeof(float));
    if (!ws) return 2;
    a.stat = ws;
    a.part = dw ? ws + stat : nullptr;
    constexpr int most = (int)(ROW_THREADS / 1024);
    for (a.first = 0; a.first < a.rows; a.first += most)
        hipLaunchKernelGGL((rms_norm_stat_kernel<T>), dim3(a.rows - a.first < most ? a.rows - a.first : most), dim3(1024), 0, state().stream, a);
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
    if (ns > ROW_MOST) return rows_bad(fn, "more than 2^30 samples");
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
