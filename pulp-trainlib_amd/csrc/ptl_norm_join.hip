// The norm behind a block, its gate, the residual and the norm in front of the next block, forward and backward.
//   u = b r1 w_post, r1 = 1 / sqrt(mean(b^2) + eps);  s = alpha x + gate u;  y = s r2 w_pre, r2 = 1 / sqrt(mean(s^2) + eps)
//   ds = ds_in + r2 (dy w_pre - s r2^2 mean(dy w_pre s));  dx = alpha ds;  k = gate w_post b
//   db = r1 (gate w_post ds - b r1^2 mean(k ds));  P = sum ds b r1:  dgate = w_post P,  dw_post = gate P;  dw_pre = sum dy s r2
// Both passes move bytes and little else.  A row is read once, into the registers of a wave or a workgroup, which walks over
// neighbouring rows and keeps weights and gates, and backward its share of the three sums over rows.  Backward all of a row's sums come
// from one reduction: mean(k ds) needs r2, but the sums of k ds_in, k dy w_pre and k s do not.
#include "ptl_rows.hpp"
#include "ptl_tuning.h"

namespace ptl {

constexpr int JOIN_MOST = 1 << 24;  // elements of a row

template <typename T>
struct JoinFw {
    const T *b, *x, *gate, *w_post, *w_pre;  // gate, w_pre: NULL where there is none
    T *s, *y;
    int rows, dim, per, chunk;  // per: rows of a gate (all of them: rows); chunk: rows of a walker
    float alpha, eps;
};

// 1 / sqrt(mean + eps) of a row's sum of squares; 0 where both are 0.
__device__ inline float join_r(float sum, int dim, float eps) {
    const float q = sum / (float)dim + eps;
    return q == 0.f ? 0.f : 1.f / sqrtf(q);
}

// NP pieces of a row in each of its TPR threads; NP = 0: the row is walked three times, in the same pieces.
template <typename T, int TPR, int NP>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void join_fw_kernel(const JoinFw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC, HELD = NP ? NP : 1;
    constexpr bool SHORT = TPR * NP == 64;  // rows of less than a piece come here too
    constexpr bool AHEAD = NP > 0 && NP * VEC <= 16;
    __shared__ float red[2][16][1];
    const int t = TPR == 64 ? (threadIdx.x & 63) : threadIdx.x;
    const long walker = TPR == 64 ? (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    const long first = walker * a.chunk, end = min(first + a.chunk, (long)a.rows);
    if (first >= end) return;  // (a whole wave, which has no barrier to meet)
    auto none = [&](int j) { return j > NP / 2 && j * TPR >= pieces; };  // (pieces that no thread has; half of them someone has)
    if constexpr (NP > 0) {
        Piece post[HELD], pre[HELD], gate[HELD];
        int of = -1;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            post[j].template hold<SHORT>(a.w_post, j * TPR + t, dim);
            if (a.w_pre) pre[j].template hold<SHORT>(a.w_pre, j * TPR + t, dim);
        }
        struct Row {
            Piece b[HELD], x[HELD];
        };
        auto fetch = [&](long row, Row &r) {
            const size_t at = (size_t)row * dim;
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                r.b[j].template hold<SHORT>(a.b + at, j * TPR + t, dim);
                r.x[j].template hold<SHORT>(a.x + at, j * TPR + t, dim);
            }
        };
        auto squares = [&](const float (&f)[VEC], int cut, float &v) {
            if (__any(cut)) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v = i < cut ? v : fmaf(f[i], f[i], v);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v = fmaf(f[i], f[i], v);
            }
        };
        auto work = [&](long row, const Row &r) {
            const size_t at = (size_t)row * dim;
            if (a.gate && (int)row / a.per != of) {
                of = (int)row / a.per;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    if (none(j)) break;
                    gate[j].template hold<SHORT>(a.gate + (size_t)of * dim, j * TPR + t, dim);
                }
            }
            float v[1] = {0.f};
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                float f[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = (float)r.b[j].e[i];
                squares(f, Piece::cut(j * TPR + t, dim), v[0]);
            }
            row_reduce<TPR, 1>(v, red[0]);
            const float r1 = join_r(v[0], dim, a.eps);
            float s[HELD][VEC];
            v[0] = 0.f;
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float u = (float)r.b[j].e[i] * r1 * (float)post[j].e[i];
                    s[j][i] = fmaf(a.alpha, (float)r.x[j].e[i], a.gate ? u * (float)gate[j].e[i] : u);
                }
                if (a.w_pre) squares(s[j], Piece::cut(j * TPR + t, dim), v[0]);
            }
            // (behind the second reduction's barrier no wave reads the first one's sums any more, and the other way round)
            if (a.w_pre || TPR > 64) row_reduce<TPR, 1>(v, red[1]);
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                Piece o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(s[j][i]);
                o.template put<SHORT>(a.s + at, j * TPR + t, dim);
            }
            if (!a.w_pre) return;
            const float r2 = join_r(v[0], dim, a.eps);
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                Piece o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(s[j][i] * r2 * (float)pre[j].e[i]);
                o.template put<SHORT>(a.y + at, j * TPR + t, dim);
            }
        };
        if constexpr (AHEAD) {
            Row x, y;
            long row = first;
            fetch(row, x);
            for (; row < end; row += 2) {
                if (row + 1 < end) fetch(row + 1, y);
                work(row, x);
                if (row + 1 >= end) break;
                if (row + 2 < end) fetch(row + 2, x);
                work(row + 1, y);
            }
        } else {
            Row x;
            for (long row = first; row < end; ++row) {
                fetch(row, x);
                work(row, x);
            }
        }
    } else {
        for (long row = first; row < end; ++row) {
            const size_t at = (size_t)row * dim;
            const T *gates = a.gate ? a.gate + (size_t)((int)row / a.per) * dim : nullptr;
            float v[1] = {0.f};
            for (int p = t; p < pieces; p += TPR) {
                Piece b;
                b.load(a.b + at, p, dim);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[0] = fmaf((float)b.e[i], (float)b.e[i], v[0]);
            }
            row_reduce<TPR, 1>(v, red[0]);
            const float r1 = join_r(v[0], dim, a.eps);
            auto join = [&](int p, float (&s)[VEC]) {
                Piece b, x, post, gate;
                b.load(a.b + at, p, dim);
                x.load(a.x + at, p, dim);
                post.load(a.w_post, p, dim);
                if (gates) gate.load(gates, p, dim);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float u = (float)b.e[i] * r1 * (float)post.e[i];
                    s[i] = fmaf(a.alpha, (float)x.e[i], gates ? u * (float)gate.e[i] : u);
                }
            };
            v[0] = 0.f;
            if (a.w_pre) {
                for (int p = t; p < pieces; p += TPR) {
                    float s[VEC];
                    join(p, s);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[0] = fmaf(s[i], s[i], v[0]);
                }
            }
            row_reduce<TPR, 1>(v, red[1]);
            const float r2 = join_r(v[0], dim, a.eps);
            for (int p = t; p < pieces; p += TPR) {  // (each thread writes over its own elements only)
                float s[VEC];
                Piece o, pre;
                join(p, s);
#pragma unroll
                for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(s[i]);
                if (a.w_pre) pre.load(a.w_pre, p, dim);
                o.store(a.s + at, p, dim);
                if (!a.w_pre) continue;
#pragma unroll
                for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(s[i] * r2 * (float)pre.e[i]);
                o.store(a.y + at, p, dim);
            }
        }
    }
}

template <typename T, int TPR, int NP>
static void join_fw_launch(JoinFw<T> a) {
    constexpr int per = TPR == 64 ? 4 : 1, waves = TPR / 64;
    // walkers that fill the chip twice over: 32 waves a compute unit
    const long most = (long)state().num_cu * 32 / waves;
    a.chunk = (int)((a.rows + most - 1) / most);
    const int walkers = (a.rows + a.chunk - 1) / a.chunk;
    hipLaunchKernelGGL((join_fw_kernel<T, TPR, NP>), dim3((walkers + per - 1) / per), dim3(TPR == 64 ? 256 : TPR), 0, state().stream, a);
}

template <typename T>
static void join_fw(const JoinFw<T> &a) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC;
    if (pieces <= 64) return join_fw_launch<T, 64, 1>(a);
    if (pieces <= 128) return join_fw_launch<T, 64, 2>(a);
    if (pieces <= 256) return join_fw_launch<T, 256, 1>(a);
    if (pieces <= 512) return join_fw_launch<T, 256, 2>(a);
    if (pieces <= 1024) return join_fw_launch<T, 512, 2>(a);
    if (pieces <= 2048) return join_fw_launch<T, 512, 4>(a);
    join_fw_launch<T, 1024, 0>(a);
}

// ---- backward --------------------------------------------------------------------------------------------------------

// Walkers (waves or workgroups) have neighbouring rows: with one gate for all `chunk` rows each.  Otherwise a walker has one of
// `parts` parts (of `chunk` rows) of a gate's rows, or, where there are more gates than walkers, `gates` whole ones.
template <typename T>
struct JoinBw {
    const T *b, *s, *dy, *ds, *gate, *w_post, *w_pre;  // s, dy, w_pre NULL: no second norm; ds, gate: may be NULL
    T *dx, *db;                       // (NULL: not wanted)
    T *dgate, *dw_post, *dw_pre;      // what a walker writes itself: gates that it has all rows of; in a grid of one also the weights'
    float *part, *part_gate;          // of the workgroups: sums over rows, P or dw_post and (with the second norm) dw_pre; of the walkers: P of a gate's part
    float *stat;                      // long rows: r1, m1, r2, m2 of each
    int rows, dim, per, chunk, parts, gates, walkers, first;
    float alpha, eps;
    bool sums;
};
struct JoinSpan {
    long first, end;
};
template <typename T>
__device__ inline JoinSpan join_span(const JoinBw<T> &a, long walker, bool groups) {
    JoinSpan s;
    if (groups && a.parts > 1) {
        const long g = walker / a.parts, z = walker - g * a.parts;
        s.first = g * a.per + z * a.chunk;
        s.end = min(min(s.first + a.chunk, (g + 1) * a.per), (long)a.rows);
    } else {
        const long rows = groups ? (long)a.gates * a.per : a.chunk;
        s.first = walker * rows;
        s.end = min(s.first + rows, (long)a.rows);
    }
    return s;
}
// The scalars of a row, from its six sums: s^2, dy w_pre s, b^2, k ds_in, k dy w_pre, k s.  Each step is of the size of r or of a gradient.
struct JoinScalars {
    float r1, m1, r2, m2;
    __device__ inline JoinScalars(const float (&v)[6], int dim, float eps) {
        r2 = join_r(v[0], dim, eps);
        m2 = r2 * (r2 * (v[1] / (float)dim));
        r1 = join_r(v[2], dim, eps);
        m1 = r1 * (r1 * (fmaf(r2, fmaf(-m2, v[5], v[4]), v[3]) / (float)dim));
    }
    __device__ inline JoinScalars(const float4 &v) : r1(v.x), m1(v.y), r2(v.z), m2(v.w) {}
    __device__ inline float ds(float in, float s, float g) const { return fmaf(r2, fmaf(-m2, s, g), in); }
};

// GROUPS: several gates.
template <typename T, int TPR, int NP, bool GROUPS>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void join_bw_kernel(const JoinBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    constexpr bool AHEAD = NP * VEC <= 8, SHORT = TPR * NP == 64;
    __shared__ float red[2][16][6];
    const int t = TPR == 64 ? (threadIdx.x & 63) : threadIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long walker = TPR == 64 ? (long)blockIdx.x * 4 + wave : blockIdx.x;
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    auto none = [&](int j) { return j > NP / 2 && j * TPR >= pieces; };
    const JoinSpan span = join_span(a, walker, GROUPS);
    Piece post[NP], pre[NP], gate[NP];
    float P[NP][VEC], Q[NP][VEC], D[GROUPS ? NP : 1][VEC];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        post[j].template hold<SHORT>(a.w_post, j * TPR + t, dim);
        pre[j].raw = gate[j].raw = row_u4{0, 0, 0, 0};
        if (a.w_pre) pre[j].template hold<SHORT>(a.w_pre, j * TPR + t, dim);
        if (!GROUPS && a.gate) gate[j].template hold<SHORT>(a.gate, j * TPR + t, dim);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            P[j][i] = Q[j][i] = 0.f;
            if constexpr (GROUPS) D[j][i] = 0.f;
        }
    }
    int of = -1;
    // Of a gate whose rows are done: its gradient (or this walker's part of it), and its share of the weights'.
    auto close = [&]() {
        if (!a.sums || (of < 0 && (a.parts == 1 || walker >= a.walkers))) return;  // (a part that no row is left for: zeros)
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            const int p = j * TPR + t;
            if (a.parts == 1) {
                Piece o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(P[j][i] * (float)post[j].e[i]);
                o.template put<SHORT>(a.dgate + (size_t)of * dim, p, dim);
            } else if (p < pieces) {
                float *to = a.part_gate + (size_t)walker * dim;
                const int cut = Piece::cut(p, dim);
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (i >= cut && p * VEC - cut + i < dim) to[p * VEC - cut + i] = P[j][i];
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if constexpr (GROUPS) D[j][i] = fmaf((float)gate[j].e[i], P[j][i], D[j][i]);
                P[j][i] = 0.f;
            }
        }
    };
    struct Row {
        Piece b[NP], s[NP], g[NP], d[NP];
    };
    auto fetch = [&](long row, Row &r) {
        const size_t at = (size_t)row * dim;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            r.b[j].template hold<SHORT>(a.b + at, j * TPR + t, dim);
            r.s[j].raw = r.g[j].raw = r.d[j].raw = row_u4{0, 0, 0, 0};
            if (a.w_pre) {
                r.s[j].template hold<SHORT>(a.s + at, j * TPR + t, dim);
                r.g[j].template hold<SHORT>(a.dy + at, j * TPR + t, dim);
            }
            if (a.ds) r.d[j].template hold<SHORT>(a.ds + at, j * TPR + t, dim);
        }
    };
    int turn = 0;
    auto work = [&](long row, const Row &x) {
        const size_t at = (size_t)row * dim;
        if constexpr (GROUPS) {
            if ((int)row / a.per != of) {
                close();
                of = (int)row / a.per;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    if (none(j)) break;
                    gate[j].template hold<SHORT>(a.gate + (size_t)of * dim, j * TPR + t, dim);
                }
            }
        }
        auto weight = [&](int j, int i) { return a.gate ? (float)post[j].e[i] * (float)gate[j].e[i] : (float)post[j].e[i]; };
        float v[6] = {};
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            const int cut = Piece::cut(j * TPR + t, dim);
            auto add = [&](int i) {
                const float b = (float)x.b[j].e[i], s = (float)x.s[j].e[i], g = (float)x.g[j].e[i] * (float)pre[j].e[i], k = weight(j, i) * b;
                v[0] = fmaf(s, s, v[0]);
                v[1] = fmaf(g, s, v[1]);
                v[2] = fmaf(b, b, v[2]);
                v[3] = fmaf(k, (float)x.d[j].e[i], v[3]);
                v[4] = fmaf(k, g, v[4]);
                v[5] = fmaf(k, s, v[5]);
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
        row_reduce<TPR, 6>(v, red[turn]);
        turn ^= 1;
        const JoinScalars c(v, dim, a.eps);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            const int p = j * TPR + t;
            Piece ox, ob;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float b = (float)x.b[j].e[i], s = (float)x.s[j].e[i], dy = (float)x.g[j].e[i];
                const float ds = c.ds((float)x.d[j].e[i], s, dy * (float)pre[j].e[i]);
                P[j][i] = fmaf(ds, b * c.r1, P[j][i]);
                Q[j][i] = fmaf(dy, s * c.r2, Q[j][i]);
                ox.e[i] = row_round<T>(a.alpha * ds);
                ob.e[i] = row_round<T>(c.r1 * fmaf(-c.m1, b, weight(j, i) * ds));
            }
            if (!a.dx) continue;
            ox.template put<SHORT>(a.dx + at, p, dim);
            ob.template put<SHORT>(a.db + at, p, dim);
        }
    };
    if constexpr (AHEAD) {
        Row x, y;
        long row = span.first;
        if (row < span.end) fetch(row, x);
        for (; row < span.end; row += 2) {
            if (row + 1 < span.end) fetch(row + 1, y);
            work(row, x);
            if (row + 1 >= span.end) break;
            if (row + 2 < span.end) fetch(row + 2, x);
            work(row + 1, y);
        }
    } else {
        Row x;
        for (long row = span.first; row < span.end; ++row) {
            fetch(row, x);
            work(row, x);
        }
    }
    if (!a.sums) return;
    if constexpr (GROUPS) close();
    auto out = [&](int c, float p, float q) {  // (a column's sums over the rows of the workgroup)
        if (a.part) {
            float *part = a.part + (size_t)blockIdx.x * (a.w_pre ? 2 : 1) * dim;
            part[c] = p;
            if (a.w_pre) part[dim + c] = q;
            return;
        }
        if (!GROUPS && a.gate) {
            a.dgate[c] = row_round<T>(p * (float)a.w_post[c]);
            p *= (float)a.gate[c];
        }
        a.dw_post[c] = row_round<T>(p);
        if (a.w_pre) a.dw_pre[c] = row_round<T>(q);
    };
    auto S = [&](int j, int i) { if constexpr (GROUPS) return D[j][i]; else return P[j][i]; };
    if constexpr (TPR == 64) {  // the four waves' shares as one
        __shared__ float all[4][2][64 * NP * VEC];
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int p = j * 64 + t, cut = Piece::cut(p, dim), c = p * VEC - cut + i;
                if (i >= cut && c < dim) {
                    all[wave][0][c] = S(j, i);
                    all[wave][1][c] = Q[j][i];
                }
            }
        __syncthreads();
        for (int c = threadIdx.x; c < dim; c += 256)
            out(c, all[0][0][c] + all[1][0][c] + (all[2][0][c] + all[3][0][c]), all[0][1][c] + all[1][1][c] + (all[2][1][c] + all[3][1][c]));
    } else if (a.part) {
        float *part = a.part + (size_t)blockIdx.x * (a.w_pre ? 2 : 1) * dim;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int p = j * TPR + t;
            if (p >= pieces) continue;
            float *to = part + p * VEC - Piece::cut(p, dim);
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                *reinterpret_cast<row_u4 *>(to + i) = __builtin_bit_cast(row_u4, row_f4{S(j, i), S(j, i + 1), S(j, i + 2), S(j, i + 3)});
                if (a.w_pre) *reinterpret_cast<row_u4 *>(to + dim + i) = __builtin_bit_cast(row_u4, row_f4{Q[j][i], Q[j][i + 1], Q[j][i + 2], Q[j][i + 3]});
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int p = j * TPR + t, cut = Piece::cut(p, dim);
            if (p >= pieces) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i >= cut) out(p * VEC - cut + i, S(j, i), Q[j][i]);
        }
    }
}

// Rows that no workgroup holds: the scalars of a row, then the columns.
template <typename T>
__global__ __launch_bounds__(1024) void join_stat_kernel(const JoinBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    __shared__ float red[16][6];
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    const size_t row = (size_t)a.first + blockIdx.x, at = row * dim;
    const T *gates = a.gate ? a.gate + (row / a.per) * dim : nullptr;
    float v[6] = {};
    for (int p = threadIdx.x; p < pieces; p += 1024) {
        Piece b, s, g, d, post, pre, gate;
        s.raw = g.raw = d.raw = pre.raw = row_u4{0, 0, 0, 0};
        b.load(a.b + at, p, dim);
        post.load(a.w_post, p, dim);
        if (gates) gate.load(gates, p, dim);
        if (a.w_pre) {
            s.load(a.s + at, p, dim);
            g.load(a.dy + at, p, dim);
            pre.load(a.w_pre, p, dim);
        }
        if (a.ds) d.load(a.ds + at, p, dim);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float fb = (float)b.e[i], fs = (float)s.e[i], fg = (float)g.e[i] * (float)pre.e[i];
            const float k = (gates ? (float)post.e[i] * (float)gate.e[i] : (float)post.e[i]) * fb;
            v[0] = fmaf(fs, fs, v[0]);
            v[1] = fmaf(fg, fs, v[1]);
            v[2] = fmaf(fb, fb, v[2]);
            v[3] = fmaf(k, (float)d.e[i], v[3]);
            v[4] = fmaf(k, fg, v[4]);
            v[5] = fmaf(k, fs, v[5]);
        }
    }
    row_reduce<1024, 6>(v, red);
    if (threadIdx.x == 0) {
        const JoinScalars c(v, dim, a.eps);
        reinterpret_cast<float4 *>(a.stat)[row] = make_float4(c.r1, c.m1, c.r2, c.m2);
    }
}
template <typename T, bool GROUPS>
__global__ __launch_bounds__(256) void join_columns_kernel(const JoinBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    const int dim = a.dim, p = (int)blockIdx.x * 256 + (int)threadIdx.x;
    if (p * (long)VEC >= dim) return;
    const JoinSpan span = join_span(a, blockIdx.y, GROUPS);
    Piece post, pre, gate;
    pre.raw = gate.raw = row_u4{0, 0, 0, 0};
    post.load(a.w_post, p, dim);
    if (a.w_pre) pre.load(a.w_pre, p, dim);
    if (!GROUPS && a.gate) gate.load(a.gate, p, dim);
    float P[VEC] = {}, Q[VEC] = {}, D[VEC] = {};
    int of = -1;
    auto close = [&]() {
        if (!a.sums || (of < 0 && a.parts == 1)) return;  // (a part that no row is left for: zeros)
        if (a.parts == 1) {
            Piece o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(P[i] * (float)post.e[i]);
            o.store(a.dgate + (size_t)of * dim, p, dim);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (p * VEC + i < dim) a.part_gate[(size_t)blockIdx.y * dim + p * VEC + i] = P[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            D[i] = fmaf((float)gate.e[i], P[i], D[i]);
            P[i] = 0.f;
        }
    };
    for (long row = span.first; row < span.end; ++row) {
        const size_t at = (size_t)row * dim;
        if (GROUPS && (int)row / a.per != of) {
            close();
            of = (int)row / a.per;
            gate.load(a.gate + (size_t)of * dim, p, dim);
        }
        const JoinScalars c(reinterpret_cast<const float4 *>(a.stat)[row]);
        Piece b, s, g, d, ox, ob;
        s.raw = g.raw = d.raw = row_u4{0, 0, 0, 0};
        b.load(a.b + at, p, dim);
        if (a.w_pre) {
            s.load(a.s + at, p, dim);
            g.load(a.dy + at, p, dim);
        }
        if (a.ds) d.load(a.ds + at, p, dim);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float fb = (float)b.e[i], fs = (float)s.e[i], dy = (float)g.e[i];
            const float ds = c.ds((float)d.e[i], fs, dy * (float)pre.e[i]);
            P[i] = fmaf(ds, fb * c.r1, P[i]);
            Q[i] = fmaf(dy, fs * c.r2, Q[i]);
            ox.e[i] = row_round<T>(a.alpha * ds);
            ob.e[i] = row_round<T>(c.r1 * fmaf(-c.m1, fb, (a.gate ? (float)post.e[i] * (float)gate.e[i] : (float)post.e[i]) * ds));
        }
        if (!a.dx) continue;
        ox.store(a.dx + at, p, dim);
        ob.store(a.db + at, p, dim);
    }
    if (!a.sums) return;
    if (GROUPS) close();
    float *part = a.part + (size_t)blockIdx.y * (a.w_pre ? 2 : 1) * dim;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (p * VEC + i < dim) {
            part[p * VEC + i] = GROUPS ? D[i] : P[i];
            if (a.w_pre) part[dim + p * VEC + i] = Q[i];
        }
}

// Sums over shares: of column c of group z (blockIdx.y) those of part[(z * shares + share) * width + c]; 32 columns (a 128-byte line) a
// workgroup, 32 shares at a time with four loads in flight.
struct JoinSums {
    const float *part;
    int width, shares;
};
template <typename T, typename F>
__device__ inline void join_sums(const JoinSums &a, F put) {
    const int o = threadIdx.x & 31, g = threadIdx.x >> 5, c = (int)blockIdx.x * 32 + o;
    const float *part = a.part + (size_t)blockIdx.y * a.shares * a.width;
    LongSum<T> s;
    s.clear();
    if (c < a.width) {
        int z = g;
        for (; z + 96 < a.shares; z += 128) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = part[(size_t)(z + 32 * u) * a.width + c];
#pragma unroll
            for (int u = 0; u < 4; ++u) s.add(v[u]);
        }
        for (; z < a.shares; z += 32) s.add(part[(size_t)z * a.width + c]);
    }
    __shared__ LongSum<T> red[32][32];
    red[g][o] = s;
    __syncthreads();
    if (g != 0 || c >= a.width) return;
    for (int k = 1; k < 32; ++k) s.add(red[k][o]);
    put(c, s.value());
}
// ... of the weights (and the one gate's, where `gate` is given: its sums are P)
template <typename T>
__global__ __launch_bounds__(1024) void join_weights_kernel(const JoinSums a, const JoinBw<T> b, const T *gate) {
    join_sums<T>(a, [&](int c, float v) {
        if (c >= b.dim) {
            b.dw_pre[c - b.dim] = row_round<T>(v);
            return;
        }
        if (gate) {
            b.dgate[c] = row_round<T>(v * (float)b.w_post[c]);
            v *= (float)gate[c];
        }
        b.dw_post[c] = row_round<T>(v);
    });
}
// ... of gates whose rows several walkers have
template <typename T>
__global__ __launch_bounds__(1024) void join_gates_kernel(const JoinSums a, const JoinBw<T> b) {
    join_sums<T>(a, [&](int c, float v) { b.dgate[(size_t)blockIdx.y * b.dim + c] = row_round<T>(v * (float)b.w_post[c]); });
}

// How the rows are dealt to about `want` walkers; returns how many there are.
template <typename T>
static int join_deal(JoinBw<T> &a, bool groups, int want) {
    a.parts = a.gates = 1;
    if (!groups) {
        a.chunk = (a.rows + want - 1) / want;
        return a.walkers = (a.rows + a.chunk - 1) / a.chunk;
    }
    const int all = (a.rows + a.per - 1) / a.per;
    if (want >= 2 * all) {
        int parts = want / all;
        a.chunk = (a.per + parts - 1) / parts;
        a.parts = (a.per + a.chunk - 1) / a.chunk;
        return a.walkers = all * a.parts;
    }
    a.gates = (all + want - 1) / want;
    return a.walkers = (all + a.gates - 1) / a.gates;
}

template <typename T>
static int join_finish(const JoinBw<T> &a, bool groups, int shares) {
    if (a.part) {
        const JoinSums s = {a.part, a.dim * (a.w_pre ? 2 : 1), shares};
        hipLaunchKernelGGL((join_weights_kernel<T>), dim3((s.width + 31) / 32), dim3(1024), 0, state().stream, s, a, groups ? nullptr : a.gate);
    }
    if (a.part_gate) {
        const JoinSums s = {a.part_gate, a.dim, a.parts};
        hipLaunchKernelGGL((join_gates_kernel<T>), dim3((a.dim + 31) / 32, (a.rows + a.per - 1) / a.per), dim3(1024), 0, state().stream, s, a);
    }
    return hip_ok(hipGetLastError(), "norm launch") ? 0 : 2;
}

template <typename T, int TPR, int NP>
static int join_bw_launch(JoinBw<T> &a, bool groups) {
    constexpr int per = TPR == 64 ? 4 : 1;
    const int best = (int)sqrtf(72.f * (float)a.rows * sizeof(T));
    int want = a.rows <= 3 * per ? per : best * per;
    want = want < a.rows ? want : a.rows;
    const int walkers = join_deal(a, groups, want > 0 ? want : 1), grid = (walkers + per - 1) / per;
    const size_t part = a.sums && (grid > 1) ? (size_t)grid * a.dim * (a.w_pre ? 2 : 1) : 0;
    const size_t part_gate = a.sums && groups && a.parts > 1 ? (size_t)walkers * a.dim : 0;
    if (part + part_gate) {
        float *ws = workspace((part + part_gate) * sizeof(float));
        if (!ws) return 2;
        if (part) a.part = ws;
        if (part_gate) a.part_gate = ws + part;
    }
    const dim3 block(TPR == 64 ? 256 : TPR);
    if (groups) hipLaunchKernelGGL((join_bw_kernel<T, TPR, NP, true>), dim3(grid), block, 0, state().stream, a);
    else hipLaunchKernelGGL((join_bw_kernel<T, TPR, NP, false>), dim3(grid), block, 0, state().stream, a);
    return join_finish(a, groups, grid);
}

template <typename T>
static int join_bw(JoinBw<T> &a, bool groups) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC;
    if (pieces <= 64) return join_bw_launch<T, 64, 1>(a, groups);
    if (pieces <= 128) return join_bw_launch<T, 64, 2>(a, groups);
    if (pieces <= 256) return join_bw_launch<T, 256, 1>(a, groups);
    if (pieces <= 512) return join_bw_launch<T, 512, 1>(a, groups);
    if (pieces <= 1024) return join_bw_launch<T, 512, 2>(a, groups);
    const int walkers = join_deal(a, groups, a.rows < 64 ? a.rows : 64);
    const size_t stat = (size_t)a.rows * 4, part = a.sums ? (size_t)walkers * a.dim * (a.w_pre ? 2 : 1) : 0;
    const size_t part_gate = a.sums && groups && a.parts > 1 ? (size_t)walkers * a.dim : 0;
    float *ws = workspace((stat + part + part_gate) * sizeof(float));
    if (!ws) return 2;
    a.stat = ws;
    a.part = part ? ws + stat : nullptr;
    a.part_gate = part_gate ? ws + stat + part : nullptr;
    constexpr int most = (int)(ROW_THREADS / 1024);
    for (a.first = 0; a.first < a.rows; a.first += most)
        hipLaunchKernelGGL((join_stat_kernel<T>), dim3(a.rows - a.first < most ? a.rows - a.first : most), dim3(1024), 0, state().stream, a);
    const dim3 grid((pieces + 255) / 256, walkers);
    if (groups) hipLaunchKernelGGL((join_columns_kernel<T, true>), grid, dim3(256), 0, state().stream, a);
    else hipLaunchKernelGGL((join_columns_kernel<T, false>), grid, dim3(256), 0, state().stream, a);
    return join_finish(a, groups, walkers);
}

template <typename T, typename Args>
static int norm_join_step(const Args *a, int ns, bool back, const char *fn) {
    if (!a || !a->input || !a->skip || !a->coeff_post || !a->sum || (a->coeff_pre && !a->output)) return rows_bad(fn, "null argument structure");
    const int dim = a->input->dim;
    if (dim <= 0 || dim > JOIN_MOST) return rows_bad(fn, "invalid tensor geometry");
    if (!(a->eps >= 0.f && a->eps < __builtin_inff())) return rows_bad(fn, "eps is no finite number from 0 on");
    if (!(fabsf(a->skip_scale) < __builtin_inff())) return rows_bad(fn, "skip_scale is no finite number");
    if (a->rows_per_gate < 0) return rows_bad(fn, "rows_per_gate is negative");
    if (ns > ROW_MOST) return rows_bad(fn, "more than 2^30 samples");
    if (ns <= 0) return 0;
    auto as = [](auto *p) { return reinterpret_cast<T *>(p); };
    const bool pre = a->coeff_pre;
    T *b = as(a->input->data), *w_post = as(a->coeff_post->data), *w_pre = as(blob_data(a->coeff_pre)), *gate = as(blob_data(a->gate));
    if (!b || !w_post || (pre && !w_pre) || (a->gate && !gate)) return rows_bad(fn, "null buffer");
    const int per = a->rows_per_gate && a->rows_per_gate < ns ? a->rows_per_gate : ns;
    const size_t n = (size_t)ns * dim, n_gate = (size_t)((ns + per - 1) / per) * dim;
    if (!back) {
        if (!a->skip->data || !a->sum->data || (pre && !a->output->data)) return rows_bad(fn, "null buffer");
        if (!ensure_init()) return 2;
        Stager sg;
        JoinFw<T> k = {};
        k.b = sg.in<T>(b, n);
        k.x = sg.in<T>(as(a->skip->data), n);
        k.w_post = sg.in<T>(w_post, (size_t)dim);
        if (pre) k.w_pre = sg.in<T>(w_pre, (size_t)dim);
        if (gate) k.gate = sg.in<T>(gate, n_gate);
        k.s = sg.out<T>(as(a->sum->data), n);
        if (pre) k.y = sg.out<T>(as(a->output->data), n);
        if (sg.failed()) return 2;
        k.rows = ns;
        k.dim = dim;
        k.per = per;
        k.alpha = a->skip_scale;
        k.eps = a->eps;
        join_fw<T>(k);
        return sg.finish(hip_ok(hipGetLastError(), "norm launch") ? 0 : 2);
    }
    const bool wg = !a->skip_wg_grad, ig = !a->skip_in_grad;
    T *s = as(a->sum->data), *ds = as(a->sum->diff), *dy = pre ? as(a->output->diff) : nullptr;
    if ((pre && (!s || !dy)) || (!pre && !ds) || (ig && (!a->input->diff || !a->skip->diff)) ||
        (wg && (!a->coeff_post->diff || (pre && !a->coeff_pre->diff) || (gate && !a->gate->diff))))
        return rows_bad(fn, "null buffer");
    if (!wg && !ig) return 0;
    if (!ensure_init()) return 2;
    Stager sg;
    JoinBw<T> k = {};
    k.b = sg.in<T>(b, n);
    k.w_post = sg.in<T>(w_post, (size_t)dim);
    if (pre) {
        k.s = sg.in<T>(s, n);
        k.dy = sg.in<T>(dy, n);
        k.w_pre = sg.in<T>(w_pre, (size_t)dim);
    }
    if (ds) k.ds = sg.in<T>(ds, n);
    if (gate) k.gate = sg.in<T>(gate, n_gate);
    if (ig) {
        k.dx = sg.out<T>(as(a->skip->diff), n);
        k.db = sg.out<T>(as(a->input->diff), n);
    }
    if (wg) {
        k.dw_post = sg.out<T>(as(a->coeff_post->diff), (size_t)dim);
        if (pre) k.dw_pre = sg.out<T>(as(a->coeff_pre->diff), (size_t)dim);
        if (gate) k.dgate = sg.out<T>(as(a->gate->diff), n_gate);
    }
    if (sg.failed()) return 2;
    k.rows = ns;
    k.dim = dim;
    k.per = per;
    k.alpha = a->skip_scale;
    k.eps = a->eps;
    k.sums = wg;
    return sg.finish(join_bw<T>(k, gate && per < ns));
}

}  // namespace ptl

extern "C" {
int ptl_norm_join_fp32_fw_batched(const struct NormJoin_args *a, int ns) {
    return ptl::norm_join_step<float>(a, ns, false, "ptl_norm_join_fp32_fw_batched");
}
int ptl_norm_join_fp32_bw_batched(const struct NormJoin_args *a, int ns) {
    return ptl::norm_join_step<float>(a, ns, true, "ptl_norm_join_fp32_bw_batched");
}
int ptl_norm_join_fp16_fw_batched(const struct NormJoin_args_fp16 *a, int ns) {
    return ptl::norm_join_step<ptl::half_t>(a, ns, false, "ptl_norm_join_fp16_fw_batched");
}
int ptl_norm_join_fp16_bw_batched(const struct NormJoin_args_fp16 *a, int ns) {
    return ptl::norm_join_step<ptl::half_t>(a, ns, true, "ptl_norm_join_fp16_bw_batched");
}
}
