// Loss against a teacher's top logits, and its gradient: with u, z the logits of teacher and student, T the temperature,
//   p = softmax(u / T) over the entries sent,  q = softmax(z / T) over all classes
//   loss = weight * sum p (log p - log q),  dz = weight / T * (q sum p - p)
// A row of logits is read once and its gradient written once; nothing else is of that size.  A workgroup holds the row in
// registers as it was read: its maximum, the sum of its exponentials and the gradient are three walks over registers.  Rows that
// no workgroup holds (more than 16384 pieces of 16 bytes) are read again for the gradient, with maximum and sum found in one walk.  Where the rows are too few to fill the chip, each is cut
// into parts of a workgroup each: one launch leaves every part's maximum and sum, the next one joins them and writes.
// The teacher's entries (tens to hundreds) are worked on by the same workgroup once the row's sum is known: the gradient of
// a class that is named is written a second time, behind a barrier, by the first entry that names it.
// Measured, loss and gradient: 2048 rows of 32000 classes in fp16 60 us (4.4 TB/s), in fp32 111 (4.7); 256 rows of 131072 34 us, in
// fp32 (read twice) 76; 4 rows of 50000 8.7 us in two launches; a few short rows 4 us.
#include "ptl_rows.hpp"
#include "ptl_transformer.h"

namespace ptl {

constexpr int DISTILL_TOP = 2048;  // entries of a row at most: they are kept in LDS, 20 bytes each
constexpr int DISTILL_WAVE_TOP = 512;  // ... where four rows share a workgroup's

struct DistillEntry {
    int to;         // the class, -1 where the entry is left out or another one before names the same class
    float sum;      // of the probabilities of all entries that name it
    float zc;       // the student's logit of the class, which the second launch may not read any more (grad may be z)
    float p, log_p;
    float pad[3];
};
template <typename T>
struct DistillArgs {
    const T *z, *u;
    const int *at;
    T *grad;      // (NULL: not wanted)
    float *loss;  // (NULL: not wanted)
    float2 *part;  // of each part of a row: its largest logit, the sum of exponentials relative to that
    struct DistillEntry *entry;  // of each row, behind those: what the first launch finds out about the teacher's entries
    int rows, first, dim, top, parts, per_part;  // first: the launch's first row; per_part: pieces
    float inv_t, hi, lo, least;  // 1 / T; log2(e) / T as the sum of two floats above 0; z - m from which on exp((z - m) / T) is 0
    float weight, scale;  // scale = weight / T
};

// exp((z - m) / T) of an entry: the exponent as the sum of two floats, the second of which corrects the result.
template <typename T>
__device__ inline float distill_exp(float z, float m, const DistillArgs<T> &a) {
    float d = z - m;
    d = d < a.least ? a.least : d;  // (0 from there on, -inf too; NaN stays)
    const float y = d * a.hi, r = fmaf(d, a.hi, -y) + d * a.lo, e = __builtin_amdgcn_exp2f(y);
    return fmaf(e, r * 0.693147181f, e);
}
// ... and of all the classes.  fp32: the exponent is rounded to 2^-24 of itself, which reaches steps of the result only in classes far
// below the largest (corrected as well: 2048 rows of 32000 124 us, 111 so).  fp16: a fused multiply-add on the value as it was read, less
// m / T rounded to fp32, and what that rounding took away: it is the same for the whole row, but as large as 2^-24 of m / T, and the
// loss and the classes that the teacher names compare the sum with logits relative to m (2048 rows of 32000: 59.7 us, 58.7 without it, 60.7
// with m subtracted first, 75 in the form of fp32; the walks over a row are bound by their instructions).
template <typename T>
struct DistillExp {
    float m, rest;
    const DistillArgs<T> &a;
    __device__ inline DistillExp(float max, const DistillArgs<T> &a) : a(a) {
        if constexpr (sizeof(T) == 4) {
            m = max;
        } else {  // (an infinite maximum gives NaN in every class, as z - m does)
            m = -max * a.hi;
            rest = fmaf(-max, a.hi, -m);
        }
    }
    __device__ inline float operator()(T z) const {
        if constexpr (sizeof(T) == 4) {
            const float d = z - m;
            return __builtin_amdgcn_exp2f(fmaf(d, a.hi, d * a.lo));
        } else {
            return __builtin_amdgcn_exp2f(fmaf((float)z, a.hi, m) + rest);
        }
    }
};

// NT threads have a row: a workgroup, or (64) one wave of a workgroup of four, which needs no barriers.
template <int NT>
__device__ inline int row_thread() { return NT == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x; }
template <int NT>
__device__ inline void row_sync() {
    if constexpr (NT == 64) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}
template <int NT>
__device__ inline void row_sync_wave() {  // where a reduction follows, which is a barrier for a workgroup
    if constexpr (NT == 64) row_sync<NT>();
}
// Two values over them.  `lds` holds two floats per wave and is not written again before another barrier.
template <int NT, bool MAX>
__device__ inline void group_reduce(float (&v)[2], float *lds) {
#pragma unroll
    for (int i = 0; i < 2; ++i) v[i] = MAX ? wave_max(v[i]) : wave_sum(v[i]);
    if constexpr (NT == 64) return;
    if ((threadIdx.x & 63) == 0) *reinterpret_cast<float2 *>(lds + 2 * (threadIdx.x >> 6)) = make_float2(v[0], v[1]);
    __syncthreads();
    const float2 r = *reinterpret_cast<const float2 *>(lds + 2 * (threadIdx.x & (NT / 64 - 1)));
    v[0] = r.x;
    v[1] = r.y;
#pragma unroll
    for (int off = NT / 128; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float o = __shfl_xor(v[i], off);
            v[i] = MAX ? fmaxf(v[i], o) : v[i] + o;
        }
}

// In LDS: room for three reductions, then `top` (in whole fours) each of classes, logits of the teacher (later probabilities) and
// of the student (later gradients).
constexpr int DISTILL_RED = 100;  // (the last four: whether a class is named twice)
inline int distill_room(int top) { return (top + 3) & ~3; }
inline size_t distill_lds(int top) { return sizeof(float) * (DISTILL_RED + 5 * (size_t)distill_room(top)); }
struct DistillTop {
    float *red;
    int *at;
    float *p, *zc, *sum;
    int *to;
    __device__ inline DistillTop(float *lds, int top) : red(lds), at((int *)(lds + DISTILL_RED)) {
        const int room = (top + 3) & ~3;
        p = lds + DISTILL_RED + room;
        zc = p + room;
        sum = zc + room;
        to = at + 4 * room;
    }
};

// The row's entries; a class that is left out becomes -1.  No barrier: a thread reads what it wrote itself.  Returns the largest
// logit of the teacher that the thread has.
template <typename T, int NT>
__device__ inline float distill_fetch(const DistillArgs<T> &a, size_t row, const DistillTop &t) {
    float m = -__builtin_inff();
    for (int i = row_thread<NT>(); i < a.top; i += NT) {
        const int c = a.at[row * a.top + i];
        const bool in = (unsigned)c < (unsigned)a.dim;
        const float u = in ? (float)a.u[row * a.top + i] : -__builtin_inff();
        t.at[i] = in ? c : -1;
        t.p[i] = u;
        t.zc[i] = in ? (float)a.z[row * a.dim + c] : 0.f;
        m = fmaxf(m, u);
    }
    if (row_thread<NT>() < 4 && a.top + row_thread<NT>() < ((a.top + 3) & ~3)) {
        t.at[a.top + row_thread<NT>()] = -1;
        t.p[a.top + row_thread<NT>()] = 0.f;
    }
    const int size = 2 * ((a.top + 3) & ~3);
    int *table = reinterpret_cast<int *>(t.sum);
    for (int i = row_thread<NT>(); i < size; i += NT) table[i] = -1;
    if (row_thread<NT>() == 0) reinterpret_cast<int *>(t.red)[96] = 0;
    return m;
}
// Whether two entries name the same class: each puts its class into a table twice their number, at a place that follows from it or the
// next free one, and finds it there if another one was first.  (Every entry compared with all others took 64 us of 74 for 8192 rows
// of 300 classes with 250 entries.)
template <typename T, int NT>
__device__ inline void distill_insert(const DistillArgs<T> &a, const DistillTop &t) {
    const int size = 2 * ((a.top + 3) & ~3);
    int *table = reinterpret_cast<int *>(t.sum);
    for (int i = row_thread<NT>(); i < a.top; i += NT) {
        const int c = t.at[i];
        if (c < 0) continue;
        int h = (int)__umulhi((unsigned)c * 2654435761u, (unsigned)size);
        for (;;) {
            const int was = atomicCAS(table + h, -1, c);
            if (was == c) reinterpret_cast<int *>(t.red)[96] = 1;
            if (was == c || was == -1) break;
            h = h + 1 == size ? 0 : h + 1;
        }
    }
}
// ... and the thread's sum of exp((u - um) / T); um is the teacher's largest, 0 where it has none (the sum is then 0, or NaN with one).
template <typename T, int NT>
__device__ inline float distill_total(const DistillArgs<T> &a, const DistillTop &t, float &um) {
    if (um == -__builtin_inff()) um = 0.f;
    float s = 0.f;
    for (int i = row_thread<NT>(); i < a.top; i += NT) s += distill_exp(t.p[i], um, a);
    return s;
}

// Probabilities in the place of the logits; f(i, p, u - um) for each of the thread's.
template <typename T, int NT, typename F>
__device__ inline void distill_probabilities(const DistillArgs<T> &a, const DistillTop &t, float um, float total, F f) {
    const float inv_total = total != 0.f ? 1.f / total : 0.f;
    for (int i = row_thread<NT>(); i < a.top; i += NT) {
        const float u = t.p[i], p = distill_exp(u, um, a) * inv_total;
        f(i, p, u - um);
        t.p[i] = p;
    }
}
// Sums of the probabilities of entries that name one class, and which of them is the first.
template <typename T, int NT>
__device__ inline void distill_merge(const DistillArgs<T> &a, const DistillTop &t, bool twice) {
    if (!twice) {
        for (int i = row_thread<NT>(); i < a.top; i += NT) {
            t.to[i] = t.at[i];
            t.sum[i] = t.p[i];
        }
        return;
    }
    row_sync<NT>();  // all probabilities and classes are in LDS
    for (int i = row_thread<NT>(); i < a.top; i += NT) {
        const int c = t.at[i];
        int first = c;
        float p = 0.f;
#pragma unroll 4
        for (int k = 0; k < a.top; k += 4) {  // (the same k in all threads: one read of LDS serves them all)
            const int4 o = *reinterpret_cast<const int4 *>(t.at + k);
            const float4 q = *reinterpret_cast<const float4 *>(t.p + k);
            p += (o.x == c ? q.x : 0.f) + (o.y == c ? q.y : 0.f) + ((o.z == c ? q.z : 0.f) + (o.w == c ? q.w : 0.f));
            const int before = (o.x == c && k < i) | (o.y == c && k + 1 < i) | (o.z == c && k + 2 < i) | (o.w == c && k + 3 < i);
            first = before ? -1 : first;
        }
        t.to[i] = first;
        t.sum[i] = p;
    }
}
// One term of the loss: 0 log 0 = 0.
template <typename T>
__device__ inline float distill_term(float p, float log_p, float zc, float m, float log_sum, const DistillArgs<T> &a) {
    return p != 0.f ? p * (log_p - ((zc - m) * a.inv_t - log_sum)) : 0.f;
}

// NP pieces of logits in each of NT threads, from piece `first` on.  MINE: each piece has its own classes only, and what the row does
// not have is -inf; else a thread may have classes that are another's too (RowPiece::cut), which only the sum has to know.
template <typename T, int NT, int NP, bool MINE>
__device__ inline void distill_hold(RowPiece<T> (&z)[NP], const T *row, int first, int end, int dim) {
    constexpr int VEC = RowPiece<T>::VEC;
    constexpr bool SHORT = NP == 1;  // rows of less than a piece: one piece a thread
    if (!MINE && !(SHORT && dim < VEC)) {
#pragma unroll
        for (int j = 0; j < NP; ++j) z[j].template hold<false>(row, first + j * NT + row_thread<NT>(), dim);
        return;
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) z[j].fetch(row, min(first + j * NT + row_thread<NT>(), end - 1), dim);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int p = first + j * NT + row_thread<NT>();
        z[j].trim(min(p, end - 1), dim);
        if (!__any(p >= end || (p + 1) * VEC > dim)) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (p >= end || p * VEC + i >= dim) z[j].e[i] = (T)-__builtin_inff();
    }
}
// Between two walks over the registers: what one converted is not kept for the next (fp16: twice the registers).
template <typename T, int NP>
__device__ inline void distill_as_read(RowPiece<T> (&z)[NP]) {
#pragma unroll
    for (int j = 0; j < NP; ++j) asm volatile("" : "+v"(z[j].raw));
}
template <typename T, int NP>
__device__ inline float distill_max(const RowPiece<T> (&z)[NP]) {
    if constexpr (sizeof(T) == 2) {  // (two at a time)
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        h2 m = {(T)-__builtin_inff(), (T)-__builtin_inff()};
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const unsigned w[4] = {z[j].raw.x, z[j].raw.y, z[j].raw.z, z[j].raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(h2, w[i]));
        }
        return fmaxf((float)m.x, (float)m.y);
    } else {
        float m = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < RowPiece<T>::VEC; ++i) m = fmaxf(m, (float)z[j].e[i]);
        return m;
    }
}
template <typename T, int NT, int NP, bool MINE>
__device__ inline float distill_sum(const RowPiece<T> (&z)[NP], const DistillExp<T> &e, int dim) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int cut = MINE ? 0 : RowPiece<T>::cut(j * NT + row_thread<NT>(), dim);
        if (!MINE && __any(cut)) {
#pragma unroll
            for (int i = 0; i < RowPiece<T>::VEC; ++i) s += i < cut ? 0.f : e(z[j].e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < RowPiece<T>::VEC; ++i) s += e(z[j].e[i]);
        }
    }
    return s;
}
// The gradient of the classes that are held.
template <typename T, int NT, int NP, bool MINE>
__device__ inline void distill_put(const RowPiece<T> (&z)[NP], T *row, int first, int end, const DistillExp<T> &e, float f, bool some, int dim) {
    int mine = first + row_thread<NT>();
    asm volatile("" : "+v"(mine));  // (the loads' addresses are not kept for the stores)
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int p = mine + j * NT;
        RowPiece<T> o;
        if (some) {
#pragma unroll
            for (int i = 0; i < RowPiece<T>::VEC; ++i) o.e[i] = row_round<T>(e(z[j].e[i]) * f);
        } else {
            o.raw = row_u4{0, 0, 0, 0};
        }
        if (MINE) {
            if (p < end) o.store(row, p, dim);
        } else {
            o.template put<NP == 1>(row, p, dim);
        }
    }
}
// NP = 0: the row is read twice.
template <typename T, int NT, int NP>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void distill_row_kernel(const DistillArgs<T> a) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int wave = NT == 64 ? (int)(threadIdx.x >> 6) : 0;
    const DistillTop t(lds + (size_t)wave * (DISTILL_RED + 5 * ((a.top + 3) & ~3)), a.top);
    const size_t row = a.first + (NT == 64 ? (size_t)blockIdx.x * 4 + wave : blockIdx.x);
    if (NT == 64 && row >= (size_t)a.rows) return;
    constexpr int VEC = RowPiece<T>::VEC, HELD = NP ? NP : 4;
    constexpr bool MINE = NP == 0;  // (the row is read behind what is written, which may be in its place)
    const int pieces = (a.dim + VEC - 1) / VEC;
    const T *zr = a.z + row * a.dim;
    T *gr = a.grad + row * a.dim;
    RowPiece<T> z[HELD];
    float top[2], own = 0.f, sum[2] = {0.f, 0.f};  // of the student, of the teacher
    if constexpr (NP > 0) {
        distill_hold<T, NT, HELD, MINE>(z, zr, 0, pieces, a.dim);
        top[1] = distill_fetch<T, NT>(a, row, t);
        top[0] = distill_max<T>(z);
    } else {
        // maximum and sum in one walk: a thread's sum is to its own largest logit so far
        top[1] = distill_fetch<T, NT>(a, row, t);
        top[0] = -__builtin_inff();
        for (int p = 0; p < pieces; p += NT * HELD) {
            distill_hold<T, NT, HELD, MINE>(z, zr, p, pieces, a.dim);
            const float m = fmaxf(top[0], distill_max<T>(z));
            // (as long as all are -inf: sums of 0, and of NaN, which is no maximum)
            const float part = distill_sum<T, NT, HELD, MINE>(z, DistillExp<T>(m == -__builtin_inff() ? 0.f : m, a), a.dim);
            sum[0] = part + (top[0] == -__builtin_inff() ? sum[0] : sum[0] * distill_exp(top[0], m, a));
            top[0] = m;
        }
        own = top[0];
    }
    row_sync_wave<NT>();
    group_reduce<NT, true>(top, t.red);
    const DistillExp<T> e(top[0], a);
    distill_insert<T, NT>(a, t);
    if constexpr (NP > 0) {
        distill_as_read<T>(z);
        sum[0] = distill_sum<T, NT, HELD, MINE>(z, e, a.dim);
        distill_as_read<T>(z);
    } else {
        if (own != -__builtin_inff()) sum[0] *= distill_exp(own, top[0], a);
    }
    sum[1] = distill_total<T, NT>(a, t, top[1]);
    row_sync_wave<NT>();
    group_reduce<NT, false>(sum, t.red + 32);
    const bool twice = reinterpret_cast<const int *>(t.red)[96] != 0;
    const bool some = sum[1] != 0.f;  // (no entry, or all of them -inf)
    float terms[2] = {0.f, 0.f};
    const float log_total = some ? logf(sum[1]) : 0.f, log_sum = logf(sum[0]);
    distill_probabilities<T, NT>(a, t, top[1], sum[1], [&](int i, float p, float d) {
        terms[0] += distill_term(p, d * a.inv_t - log_total, t.zc[i], top[0], log_sum, a);
    });
    if (a.loss) {
        group_reduce<NT, false>(terms, t.red + 64);
        if (row_thread<NT>() == 0) a.loss[row] = terms[0] * a.weight;
    }
    if (!a.grad) return;
    distill_merge<T, NT>(a, t, twice);
    const float f = a.scale / sum[0];
    if constexpr (NP > 0) {
        distill_put<T, NT, HELD, MINE>(z, gr, 0, pieces, e, f, some, a.dim);
    } else {
        for (int p = 0; p < pieces; p += NT * HELD) {
            distill_hold<T, NT, HELD, MINE>(z, zr, p, pieces, a.dim);
            distill_put<T, NT, HELD, MINE>(z, gr, p, pieces, e, f, some, a.dim);
        }
    }
    row_sync<NT>();  // behind all of those, the classes that the entries name
    for (int i = row_thread<NT>(); i < a.top; i += NT) {
        const int c = t.to[i];
        if (c >= 0) gr[c] = some ? (T)(a.scale * (distill_exp(t.zc[i], top[0], a) / sum[0] - t.sum[i])) : (T)0.f;
    }
}

// A part of a row to a workgroup: its maximum and sum; one more has the teacher's entries ...
constexpr int DISTILL_NT = 256, DISTILL_NP = 4;
template <typename T>
__global__ __launch_bounds__(DISTILL_NT) void distill_part_kernel(const DistillArgs<T> a) {
    constexpr int NT = DISTILL_NT, NP = DISTILL_NP, VEC = RowPiece<T>::VEC;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const DistillTop t(lds, a.top);
    const size_t row = blockIdx.y;
    if (blockIdx.x == 0) {
        float top[2] = {0.f, distill_fetch<T, NT>(a, row, t)}, sum[2] = {0.f, 0.f};
        group_reduce<NT, true>(top, t.red);
        distill_insert<T, NT>(a, t);
        sum[1] = distill_total<T, NT>(a, t, top[1]);
        group_reduce<NT, false>(sum, t.red + 32);
        const bool twice = reinterpret_cast<const int *>(t.red)[96] != 0;
        DistillEntry *e = a.entry + row * a.top;
        const float log_total = sum[1] != 0.f ? logf(sum[1]) : 0.f;
        distill_probabilities<T, NT>(a, t, top[1], sum[1], [&](int i, float p, float d) {
            e[i].p = p;
            e[i].log_p = d * a.inv_t - log_total;
        });
        if (threadIdx.x == 0) a.part[row * (a.parts + 1) + a.parts] = make_float2(sum[1], 0.f);
        distill_merge<T, NT>(a, t, twice);
        for (int i = threadIdx.x; i < a.top; i += NT) {
            e[i].to = t.to[i];
            e[i].sum = t.sum[i];
            e[i].zc = t.zc[i];
        }
        return;
    }
    const int part = (int)blockIdx.x - 1;
    const int pieces = (a.dim + VEC - 1) / VEC, first = part * a.per_part, end = min(first + a.per_part, pieces);
    RowPiece<T> z[NP];
    distill_hold<T, NT, NP, true>(z, a.z + row * a.dim, first, end, a.dim);
    float m[2] = {distill_max<T>(z), 0.f}, s[2] = {0.f, 0.f};
    group_reduce<NT, true>(m, t.red);
    // (a part of nothing but -inf adds nothing to a row that has more; a NaN among them is no maximum, but in the sum)
    const DistillExp<T> e(m[0] == -__builtin_inff() ? 0.f : m[0], a);
    s[0] = distill_sum<T, NT, NP, true>(z, e, a.dim);
    group_reduce<NT, false>(s, t.red + 32);
    if (threadIdx.x == 0) a.part[row * (a.parts + 1) + part] = make_float2(m[0], s[0]);
}
// ... which every workgroup of the row joins before it writes its part's gradient; the first one has the loss.
template <typename T>
__global__ __launch_bounds__(DISTILL_NT) void distill_join_kernel(const DistillArgs<T> a) {
    constexpr int NT = DISTILL_NT, NP = DISTILL_NP, VEC = RowPiece<T>::VEC;
    __shared__ __attribute__((aligned(16))) float red[96];
    const size_t row = blockIdx.y;
    const int pieces = (a.dim + VEC - 1) / VEC, first = (int)blockIdx.x * a.per_part, end = min(first + a.per_part, pieces);
    const float2 *part = a.part + row * (a.parts + 1);
    const DistillEntry *entry = a.entry + row * a.top;
    RowPiece<T> z[NP];
    if (a.grad) distill_hold<T, NT, NP, true>(z, a.z + row * a.dim, first, end, a.dim);
    const bool some = part[a.parts].x != 0.f;
    float top[2] = {-__builtin_inff(), 0.f}, sum[2] = {0.f, 0.f};
    for (int i = threadIdx.x; i < a.parts; i += NT) top[0] = fmaxf(top[0], part[i].x);
    group_reduce<NT, true>(top, red);
    for (int i = threadIdx.x; i < a.parts; i += NT) {
        const float2 v = part[i];
        sum[0] += v.x == -__builtin_inff() ? v.y : v.y * distill_exp(v.x, top[0], a);
    }
    group_reduce<NT, false>(sum, red + 32);
    if (a.loss && blockIdx.x == 0) {
        float terms[2] = {0.f, 0.f};
        const float log_sum = logf(sum[0]);
        for (int i = threadIdx.x; i < a.top; i += NT) terms[0] += distill_term(entry[i].p, entry[i].log_p, entry[i].zc, top[0], log_sum, a);
        group_reduce<NT, false>(terms, red + 64);
        if (threadIdx.x == 0) a.loss[row] = terms[0] * a.weight;
    }
    if (!a.grad) return;
    T *gr = a.grad + row * a.dim;
    distill_put<T, NT, NP, true>(z, gr, first, end, DistillExp<T>(top[0], a), a.scale / sum[0], some, a.dim);
    __syncthreads();  // behind all of those, the classes among them that the entries name
    const int lo = first * VEC, hi = end == pieces ? a.dim : end * VEC;
    for (int i = threadIdx.x; i < a.top; i += NT) {
        const DistillEntry e = entry[i];
        if (e.to >= lo && e.to < hi) gr[e.to] = some ? (T)(a.scale * (distill_exp(e.zc, top[0], a) / sum[0] - e.sum)) : (T)0.f;
    }
}

template <typename T, int NT, int NP>
static void distill_rows(DistillArgs<T> a, int ns) {
    const int most = (int)(ROW_THREADS / NT);
    for (; a.first < ns; a.first += most) {
        const int n = ns - a.first < most ? ns - a.first : most;
        a.rows = a.first + n;
        if (NT == 64) hipLaunchKernelGGL((distill_row_kernel<T, NT, NP>), dim3((n + 3) / 4), dim3(256), 4 * distill_lds(a.top), state().stream, a);
        else hipLaunchKernelGGL((distill_row_kernel<T, NT, NP>), dim3(n), dim3(NT), distill_lds(a.top), state().stream, a);
    }
}

template <typename T>
static int distill_launch(DistillArgs<T> &a, int ns) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC, cu = state().num_cu;
    // Rows in parts: a second launch costs 3 us, so rows have to be long and, where a workgroup holds one easily, few.  In parts and by
    // the row, us: 32 of 24000 in fp16 9.7 and 8.0, of 50000 10.0 and 10.3, 64 10.7 and 11.0, 100 13.1 and 11.3; 100 of 131072 18.8 and
    // 21.0; in fp32 32 of 50000 10.2 and 12.0, 64 13.9 and 13.1, of 131072 21.3 and 30.5, 128 35.5 and 36.3.
    if (pieces > 4096 && (long)ns * (a.dim > 65536 ? 2 : 6) <= cu) {
        const int most = DISTILL_NT * DISTILL_NP;
        int parts = 2 * cu / ns, least = (pieces + most - 1) / most;
        parts = parts < (pieces + DISTILL_NT - 1) / DISTILL_NT ? parts : (pieces + DISTILL_NT - 1) / DISTILL_NT;
        parts = parts > least ? parts : least;
        a.per_part = (pieces + parts - 1) / parts;
        a.parts = (pieces + a.per_part - 1) / a.per_part;
        const size_t entries = sizeof(DistillEntry) * (size_t)ns * a.top;
        char *ws = reinterpret_cast<char *>(workspace(entries + sizeof(float2) * (size_t)ns * (a.parts + 1)));
        if (!ws) return 2;
        a.entry = reinterpret_cast<DistillEntry *>(ws);
        a.part = reinterpret_cast<float2 *>(ws + entries);
        hipLaunchKernelGGL((distill_part_kernel<T>), dim3(a.parts + 1, ns), dim3(DISTILL_NT), distill_lds(a.top), state().stream, a);
        hipLaunchKernelGGL((distill_join_kernel<T>), dim3(a.grad ? a.parts : 1, ns), dim3(DISTILL_NT), 0, state().stream, a);
    } else if (a.top <= DISTILL_WAVE_TOP && ((pieces <= 256 && ns >= 4 * cu) || (pieces <= 512 && ns >= 16 * cu))) {
        // rows by the wave: 8192 of 1000 classes in fp16 30 -> 13 us, 2000 10 -> 6.4; 1000 rows of 2000 6.4 and 6.3, of 4096 7.6 and 8.9
        if (pieces <= 64) distill_rows<T, 64, 1>(a, ns);
        else if (pieces <= 128) distill_rows<T, 64, 2>(a, ns);
        else if (pieces <= 256) distill_rows<T, 64, 4>(a, ns);
        else distill_rows<T, 64, 8>(a, ns);
    } else if (pieces <= 256) {
        distill_rows<T, 256, 1>(a, ns);
    } else if (pieces <= 512) {
        distill_rows<T, 256, 2>(a, ns);
    } else if (pieces <= 1024) {
        distill_rows<T, 256, 4>(a, ns);
    } else if (pieces <= 2048) {
        distill_rows<T, 256, 8>(a, ns);
    } else if (pieces <= 4096) {
        distill_rows<T, 512, 8>(a, ns);
    } else if (pieces <= 8192) {
        distill_rows<T, 1024, 8>(a, ns);
    } else if (pieces <= 12288) {
        distill_rows<T, 1024, 12>(a, ns);
    } else if (pieces <= 16384) {
        distill_rows<T, 1024, 16>(a, ns);
    } else {
        distill_rows<T, 1024, 0>(a, ns);
    }
    return hip_ok(hipGetLastError(), "distillation launch") ? 0 : 2;
}

template <typename T, typename Args>
static int distill_step(const Args *a, int ns, int step, const char *fn) {
    if (!a || !a->output) return rows_bad(fn, "null argument structure");
    const int dim = a->output->dim, top = a->n_top;
    if (dim <= 0 || dim > ROW_MOST) return rows_bad(fn, "invalid tensor geometry");
    if (top < 1 || top > DISTILL_TOP) return rows_bad(fn, "n_top is not in 1 .. 2048");
    if (step < 0 || step > 2) return rows_bad(fn, "step is not 0, 1 or 2");
    if (!(a->temperature >= 1e-6f && a->temperature <= 1e6f)) return rows_bad(fn, "the temperature is not in 1e-6 .. 1e6");
    if (!(fabsf(a->weight) < __builtin_inff())) return rows_bad(fn, "the weight is no finite number");
    const bool loss = step != 1, grad = step != 0;
    if (!a->output->data || !a->teacher || !a->classes || (loss && !a->wr_loss) || (grad && !a->output->diff)) return rows_bad(fn, "null buffer");
    if (ns > ROW_MOST) return rows_bad(fn, "more than 2^30 samples");
    if (ns <= 0) return 0;
    if (!ensure_init()) return 2;
    const size_t n = (size_t)ns * dim, k = (size_t)ns * top;
    Stager sg;
    DistillArgs<T> d = {};
    d.z = sg.in(reinterpret_cast<const T *>(a->output->data), n);
    d.u = sg.in(reinterpret_cast<const T *>(a->teacher), k);
    d.at = sg.in<int>(a->classes, k);
    if (loss) d.loss = sg.out<float>(a->wr_loss, (size_t)ns);
    if (grad) d.grad = sg.out(reinterpret_cast<T *>(a->output->diff), n);
    if (sg.failed()) return 2;
    d.rows = ns;
    d.dim = dim;
    d.top = top;
    const double log2e = 1.4426950408889634074 / a->temperature;
    d.inv_t = 1.f / a->temperature;
    d.hi = (float)log2e;
    if ((double)d.hi >= log2e) d.hi = nextafterf(d.hi, 0.f);
    d.lo = (float)(log2e - (double)d.hi);  // above 0: a difference of -inf gives -inf from both
    d.least = (float)(-150. / log2e);
    d.weight = a->weight;
    d.scale = a->weight / a->temperature;
    return sg.finish(distill_launch<T>(d, ns));
}

}  // namespace ptl

extern "C" {
int ptl_distill_fp32_batched(const struct distill_args *a, int ns, int step) {
    return ptl::distill_step<float>(a, ns, step, "ptl_distill_fp32_batched");
}
int ptl_distill_fp16_batched(const struct distill_args_fp16 *a, int ns, int step) {
    return ptl::distill_step<ptl::half_t>(a, ns, step, "ptl_distill_fp16_batched");
}
}
