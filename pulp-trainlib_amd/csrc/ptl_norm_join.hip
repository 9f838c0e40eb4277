// The norm behind a block, its gate, the residual and the norm in front of the next block, forward and backward.
//   u = b r1 w_post, r1 = 1 / sqrt(mean(b^2) + eps);  s = alpha x + gate u;  y = s r2 w_pre, r2 = 1 / sqrt(mean(s^2) + eps)
//   ds = ds_in + r2 (dy w_pre - s r2^2 mean(dy w_pre s));  dx = alpha ds;  k = gate w_post b
//   db = r1 (gate w_post ds - b r1^2 mean(k ds));  P = sum ds b r1:  dgate = w_post P,  dw_post = gate P;  dw_pre = sum dy s r2
// Both passes move bytes and little else.  A row is read once, into the registers of a wave or a workgroup, which walks over
// rows in turn and keeps weights and gates, and backward its share of the sums over rows.  Backward all of a row's sums come
// from one reduction: mean(k ds) needs r2, but the sums of k ds_in, k dy w_pre and k s do not.  What is written, and backward what is read,
// passes by the caches (8192 x 4096 fp16: forward 51.7 -> 48.6 us, backward 90 -> 82; forward the block's output is often still there).
// Measured: 8192 x 4096 fp16 forward 48.6 us (5.5 TB/s), backward with eight gates 82 us (4.9 TB/s), with one 79; 8192 x 1024 12.8 and 28;
// one row 3.4 us, which is an empty launch.  Large copies reach 5.0 TB/s on the same card.
#include "ptl_row_sums.hpp"
#include "ptl_rows.hpp"
#include "ptl_tuning.h"

namespace ptl {

constexpr int JOIN_MOST = 1 << 24;  // elements of a row

template <typename T>
struct JoinFw {
    const T *b, *x, *gate, *w_post, *w_pre;  // gate, w_pre: NULL where there is none
    T *s, *y;
    int rows, dim, per, walkers;  // per: rows of a gate (all of them: rows); walker w has rows w, w + walkers, ...
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
    __shared__ float red[2][ROW_SUMS<TPR, 1>];
    const int t = TPR == 64 ? (threadIdx.x & 63) : threadIdx.x;
    const long walker = TPR == 64 ? (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    const long first = walker, end = a.rows, step = a.walkers;
    if (first >= min(end, step)) return;  // (a whole wave, which has no barrier to meet)
    auto none = [&](int j) { return j > NP / 2 && j * TPR >= pieces; };  // (pieces that no thread has; half of them someone has)
    if constexpr (NP > 0) {
        Piece pre[HELD];
        float w[HELD][VEC];  // w_post times the gate
        int of = -1;
        auto weights = [&](int gate) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                Piece p, g;
                p.template hold<SHORT>(a.w_post, j * TPR + t, dim);
                if (a.gate) g.template hold<SHORT>(a.gate + (size_t)gate * dim, j * TPR + t, dim);
#pragma unroll
                for (int i = 0; i < VEC; ++i) w[j][i] = a.gate ? (float)p.e[i] * (float)g.e[i] : (float)p.e[i];
            }
        };
        if (a.w_pre) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                pre[j].template hold<SHORT>(a.w_pre, j * TPR + t, dim);
            }
        }
        if (!a.gate) weights(0);
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
                weights(of);
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
            row_sums<TPR, 1>(v, red[0]);
            const float r1 = join_r(v[0], dim, a.eps);
            float s[HELD][VEC];
            v[0] = 0.f;
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[j][i] = fmaf(a.alpha, (float)r.x[j].e[i], (float)r.b[j].e[i] * r1 * w[j][i]);
                if (a.w_pre) squares(s[j], Piece::cut(j * TPR + t, dim), v[0]);
            }
            // (behind the second reduction's barrier no wave reads the first one's sums any more, and the other way round)
            if (a.w_pre || TPR > 64) row_sums<TPR, 1>(v, red[1]);
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                Piece o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(s[j][i]);
                o.template put<SHORT, true>(a.s + at, j * TPR + t, dim);
            }
            if (!a.w_pre) return;
            const float r2 = join_r(v[0], dim, a.eps);
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (none(j)) break;
                Piece o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(s[j][i] * r2 * (float)pre[j].e[i]);
                o.template put<SHORT, true>(a.y + at, j * TPR + t, dim);
            }
        };
        Row x;
        for (long row = first; row < end; row += step) {
            fetch(row, x);
            work(row, x);
        }
    } else {
        for (long row = first; row < end; row += step) {
            const size_t at = (size_t)row * dim;
            const T *gates = a.gate ? a.gate + (size_t)((int)row / a.per) * dim : nullptr;
            float v[1] = {0.f};
            for (int p = t; p < pieces; p += TPR) {
                Piece b;
                b.load(a.b + at, p, dim);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[0] = fmaf((float)b.e[i], (float)b.e[i], v[0]);
            }
            row_sums<TPR, 1>(v, red[0]);
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
            row_sums<TPR, 1>(v, red[1]);
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
    // 64 waves a compute unit, twice what it holds: rows of 4096 fp16 values, 8192 of them, 47.8 us; 32 waves 51.7, a workgroup for every row,
    // which reads the weights again for each, 49.9
    const long most = (long)state().num_cu * 64 / waves;
    a.walkers = a.rows < most ? a.rows : (int)most;
    hipLaunchKernelGGL((join_fw_kernel<T, TPR, NP>), dim3((a.walkers + per - 1) / per), dim3(TPR == 64 ? 256 : TPR), 0, state().stream, a);
}

template <typename T>
static void join_fw(const JoinFw<T> &a) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC;
    if (pieces <= 64) return join_fw_launch<T, 64, 1>(a);
    if (pieces <= 128) return join_fw_launch<T, 64, 2>(a);
    if (pieces <= 256) return join_fw_launch<T, 256, 1>(a);
    if (pieces <= 512) return join_fw_launch<T, 256, 2>(a);
    if (pieces <= 1024) return join_fw_launch<T, 512, 2>(a);
    if (pieces <= 2048) return join_fw_launch<T, 1024, 2>(a);
    if (sizeof(T) == 4 && pieces <= 4096) return join_fw_launch<T, 1024, 4>(a);
    join_fw_launch<T, 1024, 0>(a);
}

// ---- backward --------------------------------------------------------------------------------------------------------

// Waves or workgroups ("walkers") take rows in turn, so that what runs together reads neighbouring rows.  With several gates a workgroup has
// every `parts`-th row of one (GATES == 1), or, where there are more gates than workgroups, a walker every `walkers`-th gate's rows (GATES == 2).
template <typename T>
struct JoinBw {
    const T *b, *s, *dy, *ds, *gate, *w_post, *w_pre;  // s, dy, w_pre NULL: no second norm; ds, gate: may be NULL
    T *dx, *db;                   // (NULL: not wanted)
    T *dgate, *dw_post, *dw_pre;  // what a walker writes itself: gates that it has all rows of; in a grid of one also the weights'
    float *part;                  // of the workgroups, sums over their rows: P (GATES == 2: of dw_post) and, with the second norm, of dw_pre
    float *stat;                  // long rows: r1, m1, r2, m2 of each
    int rows, dim, per, parts, walkers, first;
    float alpha, eps;
    bool sums;
};
template <typename T, int GATES>
struct JoinRows {
    int first, end, step, gate;
    const JoinBw<T> &a;
    // Of walker `at` of `of` in workgroup `group`.
    __device__ inline JoinRows(const JoinBw<T> &a, int group, int at, int of) : end(a.rows), gate(0), a(a) {
        const int walker = group * of + at;
        if (GATES == 0) {
            first = walker;
            step = a.walkers;
        } else if (GATES == 1) {
            gate = group / a.parts;
            first = gate * a.per + (group - gate * a.parts) * of + at;
            end = (int)min((long)(gate + 1) * a.per, (long)a.rows);
            step = a.parts * of;
        } else {
            first = walker < a.walkers ? walker * a.per : a.rows;
            step = 1;
        }
    }
    __device__ inline bool has(long row) const { return row < end; }
    __device__ inline long next(long row) const {
        if (GATES == 2) return (int)(row + 1) % a.per == 0 ? row + 1 + (a.walkers - 1) * (long)a.per : row + 1;
        return row + step;
    }
};
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

// A thread's sums over rows, P and Q: in registers, or (KEEP) in its own places of LDS, where those do not suffice.
template <int N, int NT, bool KEEP>
struct JoinSumsOf {
    float v[2][N];
    __device__ inline void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) v[0][i] = v[1][i] = 0.f;
    }
    __device__ inline float get(int k, int i) const { return v[k][i]; }
    __device__ inline void set(int k, int i, float f) { v[k][i] = f; }
};
template <int N, int NT>
struct JoinSumsOf<N, NT, true> {
    __device__ static inline float *at(int k, int i) {
        extern __shared__ __attribute__((aligned(16))) float join_lds[];
        return join_lds + (k * N + i) * NT + threadIdx.x;
    }
    __device__ inline void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) *at(0, i) = *at(1, i) = 0.f;
    }
    __device__ inline float get(int k, int i) const { return *at(k, i); }
    __device__ inline void set(int k, int i, float f) { *at(k, i) = f; }
};

template <typename T, int TPR, int NP, int GATES, bool KEEP>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void join_bw_kernel(const JoinBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC, NT = TPR == 64 ? 256 : TPR;
    constexpr bool AHEAD = NP * VEC <= 8 && TPR < 1024, SHORT = TPR * NP == 64;  // AHEAD: registers hold two rows
    __shared__ float red[2][ROW_SUMS<TPR, 6>];
    const int t = TPR == 64 ? (threadIdx.x & 63) : threadIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int dim = a.dim, pieces = (dim + VEC - 1) / VEC;
    auto none = [&](int j) { return j > NP / 2 && j * TPR >= pieces; };
    const JoinRows<T, GATES> rows(a, blockIdx.x, TPR == 64 ? wave : 0, TPR == 64 ? 4 : 1);
    // w_post times the gate; the sums over rows, of which D, with several gates, only changes where one ends: it is in LDS (a thread's own)
    Piece pre[NP];
    float w[NP][VEC];
    JoinSumsOf<NP * VEC, NT, KEEP> sums;
    __shared__ float D[GATES == 2 ? NP * VEC : 1][NT];
    auto weights = [&](int gate) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            Piece p, g;
            p.template hold<SHORT>(a.w_post, j * TPR + t, dim);
            if (a.gate) g.template hold<SHORT>(a.gate + (size_t)gate * dim, j * TPR + t, dim);
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[j][i] = a.gate ? (float)p.e[i] * (float)g.e[i] : (float)p.e[i];
        }
    };
    sums.clear();
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        pre[j].raw = row_u4{0, 0, 0, 0};
        if (a.w_pre) pre[j].template hold<SHORT>(a.w_pre, j * TPR + t, dim);
        if constexpr (GATES == 2) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) D[j * VEC + i][threadIdx.x] = 0.f;
        }
    }
    if (GATES < 2) weights(rows.gate);
    int of = -1;
    // Of a gate whose rows are done: its gradient, and its share of the weights'.
    auto close = [&]() {
        if (!a.sums || of < 0) return;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            const int p = j * TPR + t;
            Piece gate, o, post;
            gate.template hold<SHORT>(a.gate + (size_t)of * dim, p, dim);
            post.template hold<SHORT>(a.w_post, p, dim);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float P = sums.get(0, j * VEC + i);
                o.e[i] = row_round<T>(P * (float)post.e[i]);
                D[GATES == 2 ? j * VEC + i : 0][threadIdx.x] = fmaf((float)gate.e[i], P, D[GATES == 2 ? j * VEC + i : 0][threadIdx.x]);
                sums.set(0, j * VEC + i, 0.f);
            }
            o.template put<SHORT>(a.dgate + (size_t)of * dim, p, dim);
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
            r.b[j].template hold<SHORT, true>(a.b + at, j * TPR + t, dim);
            r.s[j].raw = r.g[j].raw = r.d[j].raw = row_u4{0, 0, 0, 0};
            if (a.w_pre) {
                r.s[j].template hold<SHORT, true>(a.s + at, j * TPR + t, dim);
                r.g[j].template hold<SHORT, true>(a.dy + at, j * TPR + t, dim);
            }
            if (a.ds) r.d[j].template hold<SHORT, true>(a.ds + at, j * TPR + t, dim);
        }
    };
    int turn = 0;
    auto work = [&](long row, const Row &x) {
        const size_t at = (size_t)row * dim;
        if constexpr (GATES == 2) {
            if ((int)row / a.per != of) {
                close();
                of = (int)row / a.per;
                weights(of);
            }
        }
        float v[6] = {};
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if (none(j)) break;
            const int cut = Piece::cut(j * TPR + t, dim);
            auto add = [&](int i) {
                const float b = (float)x.b[j].e[i], s = (float)x.s[j].e[i], g = (float)x.g[j].e[i] * (float)pre[j].e[i], k = w[j][i] * b;
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
        row_sums<TPR, 6>(v, red[turn]);
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
                sums.set(0, j * VEC + i, fmaf(ds, b * c.r1, sums.get(0, j * VEC + i)));
                sums.set(1, j * VEC + i, fmaf(dy, s * c.r2, sums.get(1, j * VEC + i)));
                ox.e[i] = row_round<T>(a.alpha * ds);
                ob.e[i] = row_round<T>(c.r1 * fmaf(-c.m1, b, w[j][i] * ds));
            }
            if (!a.dx) continue;
            ox.template put<SHORT, true>(a.dx + at, p, dim);
            ob.template put<SHORT, true>(a.db + at, p, dim);
        }
    };
    if constexpr (AHEAD) {
        Row x, y;
        long row = rows.first;
        if (rows.has(row)) fetch(row, x);
        while (rows.has(row)) {
            const long second = rows.next(row), third = rows.next(second);
            if (rows.has(second)) fetch(second, y);
            work(row, x);
            if (!rows.has(second)) break;
            if (rows.has(third)) fetch(third, x);
            work(second, y);
            row = third;
        }
    } else {
        Row x;
        for (long row = rows.first; rows.has(row); row = rows.next(row)) {
            fetch(row, x);
            work(row, x);
        }
    }
    if (!a.sums) return;
    if constexpr (GATES == 2) close();
    auto out = [&](int c, float p, float q) {  // (a column's sums over the rows of the workgroup)
        if (a.part) {
            float *part = a.part + (size_t)blockIdx.x * (a.w_pre ? 2 : 1) * dim;
            part[c] = p;
            if (a.w_pre) part[dim + c] = q;
            return;
        }
        if (GATES == 0 && a.gate) {
            a.dgate[c] = row_round<T>(p * (float)a.w_post[c]);
            p *= (float)a.gate[c];
        }
        a.dw_post[c] = row_round<T>(p);
        if (a.w_pre) a.dw_pre[c] = row_round<T>(q);
    };
    auto S = [&](int j, int i) { return GATES == 2 ? D[GATES == 2 ? j * VEC + i : 0][threadIdx.x] : sums.get(0, j * VEC + i); };
    if constexpr (TPR == 64) {  // the four waves' shares as one
        __shared__ float all[4][2][64 * NP * VEC];
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int p = j * 64 + t, cut = Piece::cut(p, dim), c = p * VEC - cut + i;
                if (i >= cut && c < dim) {
                    all[wave][0][c] = S(j, i);
                    all[wave][1][c] = sums.get(1, j * VEC + i);
                }
            }
        __syncthreads();
        for (int c = threadIdx.x; c < dim; c += 256)
            out(c, all[0][0][c] + all[1][0][c] + (all[2][0][c] + all[3][0][c]), all[0][1][c] + all[1][1][c] + (all[2][1][c] + all[3][1][c]));
    } else {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int p = j * TPR + t, cut = Piece::cut(p, dim);
            if (p >= pieces) continue;
            if (a.part) {
                float *to = a.part + (size_t)blockIdx.x * (a.w_pre ? 2 : 1) * dim + p * VEC - cut;
#pragma unroll
                for (int i = 0; i < VEC; i += 4) {
                    *reinterpret_cast<row_u4 *>(to + i) = __builtin_bit_cast(row_u4, row_f4{S(j, i), S(j, i + 1), S(j, i + 2), S(j, i + 3)});
                    if (a.w_pre)
                        *reinterpret_cast<row_u4 *>(to + dim + i) = __builtin_bit_cast(
                            row_u4, row_f4{sums.get(1, j * VEC + i), sums.get(1, j * VEC + i + 1), sums.get(1, j * VEC + i + 2), sums.get(1, j * VEC + i + 3)});
                }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (i >= cut) out(p * VEC - cut + i, S(j, i), sums.get(1, j * VEC + i));
            }
        }
    }
}

// Rows that no workgroup holds: the scalars of a row, then the columns.
template <typename T>
__global__ __launch_bounds__(1024) void join_stat_kernel(const JoinBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    __shared__ float red[ROW_SUMS<1024, 6>];
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
    row_sums<1024, 6>(v, red);
    if (threadIdx.x == 0) {
        const JoinScalars c(v, dim, a.eps);
        reinterpret_cast<float4 *>(a.stat)[row] = make_float4(c.r1, c.m1, c.r2, c.m2);
    }
}
template <typename T, int GATES>
__global__ __launch_bounds__(256) void join_columns_kernel(const JoinBw<T> a) {
    typedef RowPiece<T> Piece;
    constexpr int VEC = Piece::VEC;
    const int dim = a.dim, p = (int)blockIdx.x * 256 + (int)threadIdx.x;
    if (p * (long)VEC >= dim) return;
    const JoinRows<T, GATES> rows(a, blockIdx.y, 0, 1);
    Piece post, pre, gate;
    pre.raw = row_u4{0, 0, 0, 0};
    post.load(a.w_post, p, dim);
    if (a.w_pre) pre.load(a.w_pre, p, dim);
    if (GATES < 2 && a.gate) gate.load(a.gate + (size_t)rows.gate * dim, p, dim);
    float P[VEC] = {}, Q[VEC] = {}, D[VEC] = {};
    int of = -1;
    auto close = [&]() {
        if (!a.sums || of < 0) return;
        Piece o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            o.e[i] = row_round<T>(P[i] * (float)post.e[i]);
            D[i] = fmaf((float)gate.e[i], P[i], D[i]);
            P[i] = 0.f;
        }
        o.store(a.dgate + (size_t)of * dim, p, dim);
    };
    for (long row = rows.first; rows.has(row); row = rows.next(row)) {
        const size_t at = (size_t)row * dim;
        if (GATES == 2 && (int)row / a.per != of) {
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
    if (GATES == 2) close();
    float *part = a.part + (size_t)blockIdx.y * (a.w_pre ? 2 : 1) * dim;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (p * VEC + i < dim) {
            part[p * VEC + i] = GATES == 2 ? D[i] : P[i];
            if (a.w_pre) part[dim + p * VEC + i] = Q[i];
        }
}

// The workgroups' shares added up, 32 columns (a 128-byte line) a workgroup, 32 shares at a time with four loads in flight: the first
// w_blocks workgroups have the columns of dw_post (GATES == 0: of P, of which dw_post and the one gate's gradient are made; GATES == 1: of P times its
// gate) and behind them those of dw_pre; with GATES == 1 the others have the gates', whose shares lie side by side.
template <typename T, int GATES>
__global__ __launch_bounds__(1024) void join_sums_kernel(const JoinBw<T> a, int shares, int w_blocks) {
    const int o = threadIdx.x & 31, g = threadIdx.x >> 5, width = a.dim * (a.w_pre ? 2 : 1);
    const bool gates = GATES == 1 && (int)blockIdx.x >= w_blocks;
    const int per = (a.dim + 31) / 32, z0 = gates ? ((int)blockIdx.x - w_blocks) / per : 0;
    const int c = (gates ? (int)blockIdx.x - w_blocks - z0 * per : (int)blockIdx.x) * 32 + o, most = gates ? a.dim : width;
    const int first = gates ? z0 * a.parts : 0, end = gates ? first + a.parts : shares;
    const bool scaled = GATES == 1 && !gates && c < a.dim;
    LongSum<T> s;
    s.clear();
    if (c < most) {
        auto value = [&](int z) { return a.part[(size_t)z * width + c] * (scaled ? (float)a.gate[(size_t)(z / a.parts) * a.dim + c] : 1.f); };
        int z = first + g;
        for (; z + 96 < end; z += 128) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = value(z + 32 * u);
#pragma unroll
            for (int u = 0; u < 4; ++u) s.add(v[u]);
        }
        for (; z < end; z += 32) s.add(value(z));
    }
    __shared__ LongSum<T> red[32][32];
    red[g][o] = s;
    __syncthreads();
    if (g != 0 || c >= most) return;
    for (int k = 1; k < 32; ++k) s.add(red[k][o]);
    float v = s.value();
    if (gates) {
        a.dgate[(size_t)z0 * a.dim + c] = row_round<T>(v * (float)a.w_post[c]);
    } else if (c >= a.dim) {
        a.dw_pre[c - a.dim] = row_round<T>(v);
    } else {
        if (GATES == 0 && a.gate) {
            a.dgate[c] = row_round<T>(v * (float)a.w_post[c]);
            v *= (float)a.gate[c];
        }
        a.dw_post[c] = row_round<T>(v);
    }
}

// How the rows are dealt to about `want` workgroups of `of` walkers each: their number, and which kernel (GATES).
template <typename T>
static int join_deal(JoinBw<T> &a, bool groups, int want, int of, int &gates) {
    const int all = (a.rows + a.per - 1) / a.per;
    const bool fits = (long)all * ((a.dim + 31) / 32) <= ROW_THREADS / 2048;  // (workgroups that add up a gate's columns, of 1024 threads)
    a.parts = 1;
    gates = !groups ? 0 : want >= 2 * all && a.per >= 2 * of && fits ? 1 : 2;
    if (gates == 1) {
        const int most = (a.per + of - 1) / of;
        a.parts = want / all < most ? want / all : most;
        return all * a.parts;
    }
    const long units = gates == 0 ? a.rows : all, groups_of = (units + of - 1) / of;
    const int grid = (int)(want < groups_of ? want : groups_of);
    a.walkers = (int)((long)grid * of < units ? (long)grid * of : units);
    return grid;
}

template <typename T>
static int join_finish(const JoinBw<T> &a, int gates, int shares) {
    if (a.part) {
        const int w_blocks = (a.dim * (a.w_pre ? 2 : 1) + 31) / 32, z_blocks = gates == 1 ? (a.dim + 31) / 32 * ((a.rows + a.per - 1) / a.per) : 0;
        const dim3 grid(w_blocks + z_blocks);
        if (gates == 0) hipLaunchKernelGGL((join_sums_kernel<T, 0>), grid, dim3(1024), 0, state().stream, a, shares, w_blocks);
        else if (gates == 1) hipLaunchKernelGGL((join_sums_kernel<T, 1>), grid, dim3(1024), 0, state().stream, a, shares, w_blocks);
        else hipLaunchKernelGGL((join_sums_kernel<T, 2>), grid, dim3(1024), 0, state().stream, a, shares, w_blocks);
    }
    return hip_ok(hipGetLastError(), "norm launch") ? 0 : 2;
}

// Eight waves a compute unit (8192 rows of 4096 fp16 values with eight gates 90 us, with four 108, with twelve 100: the registers hold eight,
// and each workgroup's sums are written and read), fewer where rows are few: a workgroup moves about 35 GB/s, its sums 8 bytes a column.
template <typename T, int TPR>
static int join_want(const JoinBw<T> &a) {
    constexpr int of = TPR == 64 ? 4 : 1, waves = TPR == 64 ? 4 : TPR / 64;
    const int few = (int)sqrtf(72.f * (float)a.rows * sizeof(T)), cu = state().num_cu, full = waves < 8 ? cu * 8 / waves : cu;
    const int want = a.rows <= 3 * of ? 1 : few < full ? few : full;
    return want > 0 ? want : 1;
}
template <typename T, int TPR, int NP, bool KEEP = false>
static int join_bw_launch(JoinBw<T> &a, bool groups) {
    constexpr int of = TPR == 64 ? 4 : 1;
    int gates;
    const int grid = join_deal(a, groups, join_want<T, TPR>(a), of, gates);
    if (a.sums && (grid > 1 || gates == 1) && !(a.part = workspace((size_t)grid * a.dim * (a.w_pre ? 2 : 1) * sizeof(float)))) return 2;
    const dim3 block(TPR == 64 ? 256 : TPR);
    constexpr int lds = KEEP ? 2 * NP * RowPiece<T>::VEC * TPR * 4 : 0;
    if constexpr (KEEP) {
        static bool ready = false;
        if (!ready) {
            for (const void *f : {reinterpret_cast<const void *>(join_bw_kernel<T, TPR, NP, 0, KEEP>), reinterpret_cast<const void *>(join_bw_kernel<T, TPR, NP, 1, KEEP>)})
                if (!hip_ok(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute")) return 2;
            ready = true;
        }
    }
    if (gates == 0) hipLaunchKernelGGL((join_bw_kernel<T, TPR, NP, 0, KEEP>), dim3(grid), block, lds, state().stream, a);
    else if (gates == 1) hipLaunchKernelGGL((join_bw_kernel<T, TPR, NP, 1, KEEP>), dim3(grid), block, lds, state().stream, a);
    else if constexpr (!KEEP) hipLaunchKernelGGL((join_bw_kernel<T, TPR, NP, 2, KEEP>), dim3(grid), block, lds, state().stream, a);
    return join_finish(a, gates, grid);
}

template <typename T>
static int join_bw_columns(JoinBw<T> &a, bool groups) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC;
    int gates;
    const int grid = join_deal(a, groups, a.rows < 64 ? a.rows : 64, 1, gates);
    const size_t stat = (size_t)a.rows * 4, part = a.sums ? (size_t)grid * a.dim * (a.w_pre ? 2 : 1) : 0;
    float *ws = workspace((stat + part) * sizeof(float));
    if (!ws) return 2;
    a.stat = ws;
    a.part = part ? ws + stat : nullptr;
    constexpr int most = (int)(ROW_THREADS / 1024);
    for (a.first = 0; a.first < a.rows; a.first += most)
        hipLaunchKernelGGL((join_stat_kernel<T>), dim3(a.rows - a.first < most ? a.rows - a.first : most), dim3(1024), 0, state().stream, a);
    const dim3 wide((pieces + 255) / 256, grid);
    if (gates == 0) hipLaunchKernelGGL((join_columns_kernel<T, 0>), wide, dim3(256), 0, state().stream, a);
    else if (gates == 1) hipLaunchKernelGGL((join_columns_kernel<T, 1>), wide, dim3(256), 0, state().stream, a);
    else hipLaunchKernelGGL((join_columns_kernel<T, 2>), wide, dim3(256), 0, state().stream, a);
    return join_finish(a, gates, grid);
}

template <typename T>
static int join_bw(JoinBw<T> &a, bool groups) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC;
    if (pieces <= 64) return join_bw_launch<T, 64, 1>(a, groups);
    if (pieces <= 128) return join_bw_launch<T, 64, 2>(a, groups);
    if (pieces <= 256) return join_bw_launch<T, 256, 1>(a, groups);
    if (pieces <= 512) return join_bw_launch<T, 256, 2>(a, groups);
    if constexpr (sizeof(T) == 4) {
        if (pieces <= 1024) return join_bw_launch<T, 512, 2>(a, groups);
        if (pieces <= 2048) return join_bw_launch<T, 1024, 2>(a, groups);
    } else {
        if (pieces <= 1024) return join_bw_launch<T, 1024, 1>(a, groups);
        int gates;
        join_deal(a, groups, join_want<T, 1024>(a), 1, gates);
        if (pieces <= 2048 && gates < 2) return join_bw_launch<T, 1024, 2, true>(a, groups);  // (the sums of several gates do not fit LDS)
    }
    return join_bw_columns(a, groups);
}

template <typename T, typename Args>
static int norm_join_step(const Args *a, int ns, bool back, const char *fn) {
    if (!a || !a->input || !a->skip || !a->coeff_post || !a->sum || (a->coeff_pre && !a->output)) return rows_bad(fn, "null argument structure");
    const int dim = a->input->dim;
    if (dim <= 0 || dim > JOIN_MOST) return rows_bad(fn, "invalid tensor geometry");
    if (!(a->eps >= 0.f && a->eps < __builtin_inff())) return rows_bad(fn, "eps is no finite number from 0 on");
    if (!(fabsf(a->skip_scale) < __builtin_inff())) return rows_bad(fn, "skip_scale is no finite number");
    if (a->rows_per_gate < 0) return rows_bad(fn, "rows_per_gate is negative");
    const bool pre = a->coeff_pre;
    if (((!back || !a->skip_in_grad) && a->skip->dim != dim) || a->sum->dim != dim || a->coeff_post->dim != dim || (pre && (a->coeff_pre->dim != dim || a->output->dim != dim)))
        return rows_bad(fn, "tensors whose sizes do not fit together");
    if (ns > ROW_MOST) return rows_bad(fn, "more than 2^30 samples");
    if (ns <= 0) return 0;
    auto as = [](auto *p) { return reinterpret_cast<T *>(p); };
    T *b = as(a->input->data), *w_post = as(a->coeff_post->data), *w_pre = as(blob_data(a->coeff_pre)), *gate = as(blob_data(a->gate));
    if (!b || !w_post || (pre && !w_pre) || (a->gate && !gate)) return rows_bad(fn, "null buffer");
    const int per = a->rows_per_gate && a->rows_per_gate < ns ? a->rows_per_gate : ns;
    const size_t n = (size_t)ns * dim, n_gate = (size_t)((ns + per - 1) / per) * dim;
    // (a gate's blob has the elements of one, as a sample's has, or of all)
    if (gate && a->gate->dim != dim && n_gate <= 0x7fffffffu && (a->gate->dim % dim != 0 || a->gate->dim < (int)n_gate))
        return rows_bad(fn, "tensors whose sizes do not fit together");
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
