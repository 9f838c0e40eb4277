// Loss against a teacher's top logits, and its gradient: with u, z the logits of teacher and student, T the temperature,
//   p = softmax(u / T) over the entries sent,  q = softmax(z / T) over all classes
//   loss = weight * sum p (log p - log q),  dz = weight / T * (q sum p - p)
// A row of logits is read once and its gradient written once; nothing else is of that size.  A workgroup holds the row in
// registers as it was read: its maximum, the sum of its exponentials and the gradient are three walks over registers.  Rows that
// no workgroup holds are read again for the second and third walk.  Where the rows are too few to fill the chip, each is cut
// into parts of a workgroup each: one launch leaves every part's maximum and sum, the next one joins them and writes.
// The teacher's entries (tens to hundreds) are worked on by the same workgroup once the row's sum is known: the gradient of
// a class that is named is written a second time, behind a barrier, by the first entry that names it.
#include "ptl_rows.hpp"
#include "ptl_transformer.h"

namespace ptl {

constexpr int DISTILL_TOP = 2048;  // entries of a row at most: they are kept in LDS

template <typename T>
struct DistillArgs {
    const T *z, *u;
    const int *at;
    T *grad;      // (NULL: not wanted)
    float *loss;  // (NULL: not wanted)
    float2 *part;  // of each part of a row: its largest logit, the sum of exponentials relative to that
    float *zc;     // the student's logits of a row's entries, which the second launch may not read any more (grad may be z)
    int dim, top, parts, per_part;  // per_part: pieces
    float inv_t, hi, lo;  // 1 / T; log2(e) / T as the sum of two floats above 0
    float weight, scale;  // scale = weight / T
};

// exp((z - m) / T): the exponent is formed to 2^-24 of itself, where a product with a rounded constant would be off twice as far.
template <typename T>
__device__ inline float distill_exp(float z, float m, const DistillArgs<T> &a) {
    const float d = z - m;
    return __builtin_amdgcn_exp2f(fmaf(d, a.hi, d * a.lo));
}

// Over a workgroup of NT threads.  `lds` holds a float per wave and is not written again before another barrier.
template <int NT, bool MAX>
__device__ inline float group_reduce(float v, float *lds) {
    v = MAX ? wave_max(v) : wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = lds[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) r = MAX ? fmaxf(r, lds[w]) : r + lds[w];
    return r;
}

// In LDS: 6 x 16 floats for the sums, then `top` each of classes, logits of the teacher (later probabilities) and of the
// student (later gradients).
constexpr int DISTILL_RED = 96;
constexpr size_t distill_lds(int top) { return sizeof(float) * (DISTILL_RED + 3 * (size_t)top); }
struct DistillTop {
    float *red;
    int *at;
    float *p, *zc;
    __device__ inline DistillTop(float *lds, int top) : red(lds), at((int *)(lds + DISTILL_RED)), p(lds + DISTILL_RED + top), zc(p + top) {}
};

// The row's entries; a class that is left out becomes -1.  No barrier: a thread reads what it wrote itself.
template <typename T, int NT>
__device__ inline void distill_fetch(const DistillArgs<T> &a, size_t row, const DistillTop &t) {
    for (int i = threadIdx.x; i < a.top; i += NT) {
        const int c = a.at[row * a.top + i];
        const bool in = (unsigned)c < (unsigned)a.dim;
        t.at[i] = in ? c : -1;
        t.p[i] = in ? (float)a.u[row * a.top + i] : -__builtin_inff();
        t.zc[i] = !in ? 0.f : a.zc ? a.zc[row * a.top + i] : (float)a.z[row * a.dim + c];
    }
}

// Loss of a row, and gradients of its entries' classes (into t.zc; t.at becomes -1 where another entry before names the same
// class).  m, sum: of the student.  Returns whether the row has entries.  Barriers: every thread of the workgroup comes here.
template <typename T, int NT>
__device__ inline bool distill_entries(const DistillArgs<T> &a, size_t row, const DistillTop &t, float m, float sum, bool loss) {
    const int tid = threadIdx.x;
    float um = -__builtin_inff(), total = 0.f;
    for (int i = tid; i < a.top; i += NT) um = fmaxf(um, t.p[i]);
    um = group_reduce<NT, true>(um, t.red + 32);
    if (um == -__builtin_inff()) um = 0.f;  // no entry, or all of them -inf: the sum is 0 (a NaN among them makes it NaN)
    for (int i = tid; i < a.top; i += NT) total += distill_exp(t.p[i], um, a);
    total = group_reduce<NT, false>(total, t.red + 48);
    const bool some = total != 0.f;
    const float inv_total = some ? 1.f / total : 0.f, inv_sum = 1.f / sum;
    const float log_total = some ? logf(total) : 0.f, log_sum = logf(sum);
    float terms = 0.f;
    for (int i = tid; i < a.top; i += NT) {
        const float p = distill_exp(t.p[i], um, a) * inv_total;
        if (p != 0.f) terms += p * ((t.p[i] - um) * a.inv_t - log_total - ((t.zc[i] - m) * a.inv_t - log_sum));  // 0 log 0 = 0
        t.p[i] = p;
    }
    if (loss) {
        terms = group_reduce<NT, false>(terms, t.red + 64);
        if (tid == 0) a.loss[row] = terms * a.weight;
    }
    if (!a.grad) return some;
    __syncthreads();  // all probabilities and classes are in LDS
    int keep[(DISTILL_TOP + NT - 1) / NT];
    int n = 0;
    for (int i = tid; i < a.top; i += NT, ++n) {
        const int c = t.at[i];
        int first = c;
        float p = 0.f;
        for (int k = 0; k < a.top; ++k) {  // (the same k in all threads: one read of LDS serves them all)
            const bool same = t.at[k] == c;
            p += same ? t.p[k] : 0.f;
            if (same && k < i) first = -1;
        }
        t.zc[i] = some ? a.scale * (distill_exp(t.zc[i], m, a) * inv_sum - p) : 0.f;
        keep[n] = first;
    }
    __syncthreads();
    n = 0;
    for (int i = tid; i < a.top; i += NT, ++n) t.at[i] = keep[n];
    return some;
}

// NP pieces of logits in each of NT threads, from piece `first` on; what the row does not have is -inf.
template <typename T, int NT, int NP>
__device__ inline void distill_hold(RowPiece<T> (&z)[NP], const T *row, int first, int end, int dim) {
    constexpr int VEC = RowPiece<T>::VEC;
#pragma unroll
    for (int j = 0; j < NP; ++j) z[j].fetch(row, min(first + j * NT + (int)threadIdx.x, end - 1), dim);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int p = first + j * NT + (int)threadIdx.x;
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
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
        for (int i = 0; i < RowPiece<T>::VEC; ++i) m = fmaxf(m, (float)z[j].e[i]);
    return m;
}
template <typename T, int NP>
__device__ inline float distill_sum(const RowPiece<T> (&z)[NP], float m, const DistillArgs<T> &a) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
        for (int i = 0; i < RowPiece<T>::VEC; ++i) s += distill_exp((float)z[j].e[i], m, a);
    return s;
}
// The gradient of the classes that are held.
template <typename T, int NT, int NP>
__device__ inline void distill_put(const RowPiece<T> (&z)[NP], T *row, int first, int end, float m, float f, bool some, const DistillArgs<T> &a) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int p = first + j * NT + (int)threadIdx.x;
        RowPiece<T> o;
#pragma unroll
        for (int i = 0; i < RowPiece<T>::VEC; ++i) o.e[i] = some ? (T)(distill_exp((float)z[j].e[i], m, a) * f) : (T)0.f;
        if (p < end) o.store(row, p, a.dim);
    }
}
// ... and, behind all of those, of the entries' classes among them.
template <typename T, int NT>
__device__ inline void distill_put_entries(const DistillArgs<T> &a, size_t row, const DistillTop &t, int lo, int hi) {
    __syncthreads();
    for (int i = threadIdx.x; i < a.top; i += NT) {
        const int c = t.at[i];
        if (c >= lo && c < hi) a.grad[row * a.dim + c] = (T)t.zc[i];
    }
}

// A row to a workgroup.  NP = 0: it is read three times.
template <typename T, int NT, int NP>
__global__ __launch_bounds__(NT) void distill_row_kernel(const DistillArgs<T> a) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const DistillTop t(lds, a.top);
    const size_t row = blockIdx.x;
    constexpr int VEC = RowPiece<T>::VEC, HELD = NP ? NP : 4;
    const int pieces = (a.dim + VEC - 1) / VEC;
    const T *zr = a.z + row * a.dim;
    T *gr = a.grad + row * a.dim;
    RowPiece<T> z[HELD];
    float m, s = 0.f;
    if constexpr (NP > 0) {
        distill_hold<T, NT>(z, zr, 0, pieces, a.dim);
        distill_fetch<T, NT>(a, row, t);
        m = group_reduce<NT, true>(distill_max<T>(z), t.red);
        distill_as_read<T>(z);
        s = group_reduce<NT, false>(distill_sum<T>(z, m, a), t.red + 16);
        distill_as_read<T>(z);
    } else {
        distill_fetch<T, NT>(a, row, t);
        m = -__builtin_inff();
        for (int p = 0; p < pieces; p += NT * HELD) {
            distill_hold<T, NT>(z, zr, p, pieces, a.dim);
            m = fmaxf(m, distill_max<T>(z));
        }
        m = group_reduce<NT, true>(m, t.red);
        for (int p = 0; p < pieces; p += NT * HELD) {
            distill_hold<T, NT>(z, zr, p, pieces, a.dim);
            s += distill_sum<T>(z, m, a);
        }
        s = group_reduce<NT, false>(s, t.red + 16);
    }
    const bool some = distill_entries<T, NT>(a, row, t, m, s, a.loss != nullptr);
    if (!a.grad) return;
    const float f = a.scale / s;
    if constexpr (NP > 0) {
        distill_put<T, NT>(z, gr, 0, pieces, m, f, some, a);
    } else {
        for (int p = 0; p < pieces; p += NT * HELD) {
            distill_hold<T, NT>(z, zr, p, pieces, a.dim);
            distill_put<T, NT>(z, gr, p, pieces, m, f, some, a);
        }
    }
    distill_put_entries<T, NT>(a, row, t, 0, a.dim);
}

// A part of a row to a workgroup: its maximum and sum ...
constexpr int DISTILL_NT = 256, DISTILL_NP = 4;
template <typename T>
__global__ __launch_bounds__(DISTILL_NT) void distill_part_kernel(const DistillArgs<T> a) {
    constexpr int NT = DISTILL_NT, NP = DISTILL_NP, VEC = RowPiece<T>::VEC;
    __shared__ float red[32];
    const size_t row = blockIdx.y;
    const int pieces = (a.dim + VEC - 1) / VEC, first = (int)blockIdx.x * a.per_part, end = min(first + a.per_part, pieces);
    RowPiece<T> z[NP];
    distill_hold<T, NT>(z, a.z + row * a.dim, first, end, a.dim);
    const float m = group_reduce<NT, true>(distill_max<T>(z), red);
    // (a part of nothing but -inf adds nothing to a row that has more)
    const float s = group_reduce<NT, false>(m == -__builtin_inff() ? 0.f : distill_sum<T>(z, m, a), red + 16);
    // a NaN among them is no maximum, but in the sum
    if (threadIdx.x == 0) a.part[row * a.parts + blockIdx.x] = make_float2(m, s);
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < a.top; i += NT) {
            const int c = a.at[row * a.top + i];
            a.zc[row * a.top + i] = (unsigned)c < (unsigned)a.dim ? (float)a.z[row * a.dim + c] : 0.f;
        }
    }
}
// ... which every workgroup of the row joins before it writes its part's gradient; the first one has the loss.
template <typename T>
__global__ __launch_bounds__(DISTILL_NT) void distill_join_kernel(const DistillArgs<T> a) {
    constexpr int NT = DISTILL_NT, NP = DISTILL_NP, VEC = RowPiece<T>::VEC;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const DistillTop t(lds, a.top);
    const size_t row = blockIdx.y;
    const int pieces = (a.dim + VEC - 1) / VEC, first = (int)blockIdx.x * a.per_part, end = min(first + a.per_part, pieces);
    RowPiece<T> z[NP];
    if (a.grad) distill_hold<T, NT>(z, a.z + row * a.dim, first, end, a.dim);
    distill_fetch<T, NT>(a, row, t);
    float m = -__builtin_inff(), s = 0.f;
    for (int i = threadIdx.x; i < a.parts; i += NT) m = fmaxf(m, a.part[row * a.parts + i].x);
    m = group_reduce<NT, true>(m, t.red);
    for (int i = threadIdx.x; i < a.parts; i += NT) {
        const float2 v = a.part[row * a.parts + i];
        s += v.x == -__builtin_inff() ? v.y : v.y * distill_exp(v.x, m, a);
    }
    s = group_reduce<NT, false>(s, t.red + 16);
    const bool some = distill_entries<T, NT>(a, row, t, m, s, a.loss && blockIdx.x == 0);
    if (!a.grad) return;
    distill_put<T, NT>(z, a.grad + row * a.dim, first, end, m, a.scale / s, some, a);
    distill_put_entries<T, NT>(a, row, t, first * VEC, end == pieces ? a.dim : end * VEC);
}

template <typename T, int NT, int NP>
static void distill_rows(const DistillArgs<T> &a, int ns) {
    hipLaunchKernelGGL((distill_row_kernel<T, NT, NP>), dim3(ns), dim3(NT), distill_lds(a.top), state().stream, a);
}

template <typename T>
static int distill_launch(DistillArgs<T> &a, int ns) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC, cu = state().num_cu;
    // Too few rows for the chip, each long enough for two workgroups and more.
    if (2L * ns <= cu && pieces > 2 * DISTILL_NT) {
        const int most = DISTILL_NT * DISTILL_NP;
        int parts = 2 * cu / ns, least = (pieces + most - 1) / most;
        parts = parts < (pieces + DISTILL_NT - 1) / DISTILL_NT ? parts : (pieces + DISTILL_NT - 1) / DISTILL_NT;
        parts = parts > least ? parts : least;
        a.per_part = (pieces + parts - 1) / parts;
        a.parts = (pieces + a.per_part - 1) / a.per_part;
        float *ws = workspace(sizeof(float) * ((size_t)ns * a.parts * 2 + (size_t)ns * a.top));
        if (!ws) return 2;
        a.part = reinterpret_cast<float2 *>(ws);
        a.zc = ws + (size_t)ns * a.parts * 2;
        hipLaunchKernelGGL((distill_part_kernel<T>), dim3(a.parts, ns), dim3(DISTILL_NT), 0, state().stream, a);
        hipLaunchKernelGGL((distill_join_kernel<T>), dim3(a.grad ? a.parts : 1, ns), dim3(DISTILL_NT), distill_lds(a.top), state().stream, a);
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
    d.dim = dim;
    d.top = top;
    const double log2e = 1.4426950408889634074 / a->temperature;
    d.inv_t = 1.f / a->temperature;
    d.hi = (float)log2e;
    if ((double)d.hi >= log2e) d.hi = nextafterf(d.hi, 0.f);
    d.lo = (float)(log2e - (double)d.hi);  // above 0: a difference of -inf gives -inf from both
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
