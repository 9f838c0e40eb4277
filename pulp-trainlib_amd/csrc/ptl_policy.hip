// Clipped policy loss with a term that holds the policy near a reference, and its gradient: with z the logits, a the action, T the temperature,
//   lp = (z_a - max z) / T - log sum exp((z - max z) / T);  ratio = exp(lp - old);  d = ref - lp
//   loss = -min(ratio A, clip(ratio) A) + beta (exp(d) - d - 1);  slope = d loss / d lp = -ratio A [not clipped] + beta (1 - exp(d))
//   dz = slope / T (1 at a - softmax(z / T))
// A row of logits is read once, into the registers of a workgroup, and its gradient written once; nothing else is of that size.  What the row's
// scalars need behind its sum is some hundred instructions, which every thread works on by itself: no further barrier.  The thread that has the
// action's class adds to it where it writes.  Rows that no workgroup holds (more than 16384 pieces of 16 bytes) are read twice; where
// the rows are too few to fill the chip each is cut into parts: one launch leaves every part's maximum and sum, the next one joins
// them and writes.  Logits come and gradients go past the caches (2048 rows of 32000 classes in fp16: 54.5 us through them, 51.1 with the stores past
// them, 49.3 with both).
// Measured, loss and gradient: 2048 rows of 32000 classes in fp16 48 us (5.4 TB/s), 1024 in fp32 48 (5.4); 500 of 131072 in fp16 59; 8192 of 1000
// 9; 4 rows of 131072 in fp32 8 to 9 us in two launches.
#include "ptl_soft_rows.hpp"
#include "ptl_tuning.h"

namespace ptl {

template <typename T>
struct PolicyArgs : SoftScale {
    const T *z;
    T *grad;                      // (NULL: not wanted)
    const int *action;
    const float *old, *ref, *adv, *row_weight;  // ref, row_weight: may be NULL
    float *loss, *logp;           // (NULL: not wanted)
    float2 *part;                 // of each part of a row: its largest logit, the sum of exponentials relative to that; behind them the action's logit
    int rows, first, dim, parts, per_part;  // first: the launch's first row; per_part: pieces
    float low, high, beta, weight;  // low, high: the borders of the ratio
};

// What a row is given, on its way while its logits are (2048 rows of 32000 classes in fp16 49.2 us, 48.4 so).
struct PolicyGiven {
    float old, ref, adv, weight;
};
template <typename T>
__device__ inline PolicyGiven policy_given(const PolicyArgs<T> &a, size_t row) {
    return {a.old[row], a.ref ? a.ref[row] : 0.f, a.adv[row], a.row_weight ? a.row_weight[row] : 1.f};
}
// What is left of a row behind its maximum and sum.
struct PolicyRow {
    float slope;  // d loss / d z_a but for the softmax, 0 for rows that are left out
    bool some;
};
// exp(d) - 1 and exp(d) - 1 - d; near 0 the latter from its series, where the difference would cancel.
__device__ inline float policy_away(float d, float &rest) {
    const float e = expm1f(d);
    const float s = d * d * fmaf(d, fmaf(d, fmaf(d, fmaf(d, fmaf(d, 1.f / 5040.f, 1.f / 720.f), 1.f / 120.f), 1.f / 24.f), 1.f / 6.f), 0.5f);
    rest = fabsf(d) < 0.25f ? s : e - d;
    return e;
}
template <typename T>
__device__ inline PolicyRow policy_row(const PolicyArgs<T> &a, const PolicyGiven &given, size_t row, int action, float za, float max, float log_sum, bool mine) {
    PolicyRow r = {0.f, (unsigned)action < (unsigned)a.dim};
    float lp = 0.f, loss = 0.f;
    if (r.some) {
        lp = (za - max) * a.inv_t - log_sum;
        const float ratio = expf(lp - given.old), A = given.adv, w = a.weight * given.weight;
        // (no number: both products are compared in vain)
        const float whole = ratio * A, clipped = fminf(fmaxf(ratio, a.low), a.high) * A;
        loss = whole <= clipped ? -whole : clipped < whole ? -clipped : whole + clipped;
        r.slope = whole <= clipped ? -whole : clipped < whole ? 0.f : whole + clipped;
        if (a.ref) {
            float rest;
            const float e = policy_away(given.ref - lp, rest);
            loss = fmaf(a.beta, rest, loss);
            r.slope = fmaf(-a.beta, e, r.slope);
        }
        loss *= w;
        r.slope *= w * a.inv_t;
    }
    if (mine && a.loss) a.loss[row] = loss;
    if (mine && a.logp) a.logp[row] = lp;
    return r;
}
// The gradient of the classes that are held.
template <typename T, int NT, int NP, bool MINE, typename E>
__device__ inline void policy_put(const RowPiece<T> (&z)[NP], T *row, int first, int end, const E &e, float sum, const PolicyRow &r, int action, int dim) {
    constexpr int VEC = RowPiece<T>::VEC;
    int mine = first + row_thread<NT>();
    asm volatile("" : "+v"(mine));  // (the loads' addresses are not kept for the stores)
    const float f = -r.slope / sum;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int p = mine + j * NT;
        RowPiece<T> o;
        if (r.some) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.e[i] = row_round<T>(e(z[j].e[i]) * f);
            const int at = action - (p * VEC - (MINE ? 0 : RowPiece<T>::cut(p, dim)));  // (a piece that reaches over the end covers the row's last values)
            if (__any((unsigned)at < (unsigned)VEC)) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (at == i) o.e[i] = row_round<T>(fmaf(e(z[j].e[i]), f, r.slope));
            }
        } else {
            o.raw = row_u4{0, 0, 0, 0};
        }
        if (MINE) {
            if (p < end) o.store(row, p, dim);
        } else {
            o.template put<NP == 1, true>(row, p, dim);
        }
    }
}
// The row's action, and its logit, which is read before the gradient takes its place.
template <typename T>
__device__ inline int policy_action(const PolicyArgs<T> &a, size_t row, float &za) {
    const int c = a.action[row];
    za = (unsigned)c < (unsigned)a.dim ? (float)a.z[row * a.dim + c] : 0.f;
    return c;
}

// NP = 0: the row is read twice.  E: the classes' exponentials.
template <typename T, typename E, int NT, int NP>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void policy_row_kernel(const PolicyArgs<T> a) {
    __shared__ __attribute__((aligned(16))) float lds[64];
    const int wave = NT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const size_t row = a.first + (NT == 64 ? (size_t)blockIdx.x * 4 + wave : blockIdx.x);
    if (NT == 64 && row >= (size_t)a.rows) return;
    constexpr int VEC = RowPiece<T>::VEC, HELD = NP ? NP : 4;
    constexpr bool MINE = NP == 0;  // (the row is read behind what is written, which may be in its place)
    const int pieces = (a.dim + VEC - 1) / VEC;
    const T *zr = a.z + row * a.dim;
    RowPiece<T> z[HELD];
    float top[2] = {-__builtin_inff(), 0.f}, sum[2] = {0.f, 0.f}, za;
    if constexpr (NP > 0) {
        soft_hold<T, NT, HELD, MINE, true>(z, zr, 0, pieces, a.dim);
    }
    const int action = policy_action(a, row, za);
    const PolicyGiven given = policy_given(a, row);
    float own = 0.f;
    if constexpr (NP > 0) {
        top[0] = soft_max<T>(z);
    } else {
        // maximum and sum in one walk: a thread's sum is to its own largest logit so far
        for (int p = 0; p < pieces; p += NT * HELD) {
            soft_hold<T, NT, HELD, MINE>(z, zr, p, pieces, a.dim);
            const float m = fmaxf(top[0], soft_max<T>(z));
            // (as long as all are -inf: sums of 0, and of NaN, which is no maximum)
            const float part = soft_sum<T, NT, HELD, MINE>(z, SoftExp<T>(m == -__builtin_inff() ? 0.f : m, a), a.dim);
            sum[0] = part + (top[0] == -__builtin_inff() ? sum[0] : sum[0] * soft_exp(top[0], m, a));
            top[0] = m;
        }
        own = top[0];
    }
    group_reduce<NT, true>(top, lds);
    const E e(top[0], a);
    if constexpr (NP > 0) {
        soft_as_read<T>(z);
        sum[0] = soft_sum<T, NT, HELD, MINE>(z, e, a.dim);
        soft_as_read<T>(z);
    } else {
        if (own != -__builtin_inff()) sum[0] *= soft_exp(own, top[0], a);
        sum[0] = e.unit(sum[0]);  // (the walk's are whole exponentials)
    }
    group_reduce<NT, false>(sum, lds + 32);
    const PolicyRow r = policy_row(a, given, row, action, za, top[0], e.log(sum[0]), row_thread<NT>() == 0);
    if (!a.grad) return;
    T *gr = a.grad + row * a.dim;
    if constexpr (NP > 0) {
        policy_put<T, NT, HELD, MINE>(z, gr, 0, pieces, e, sum[0], r, action, a.dim);
    } else {
        for (int p = 0; p < pieces; p += NT * HELD) {
            soft_hold<T, NT, HELD, MINE>(z, zr, p, pieces, a.dim);
            policy_put<T, NT, HELD, MINE>(z, gr, p, pieces, e, sum[0], r, action, a.dim);
        }
    }
}

// A part of a row to a workgroup: its maximum and sum, the first one also the action's logit, which the second launch may not read any more ...
constexpr int POLICY_NT = 256, POLICY_NP = 4;
template <typename T>
__global__ __launch_bounds__(POLICY_NT) void policy_part_kernel(const PolicyArgs<T> a) {
    constexpr int NT = POLICY_NT, NP = POLICY_NP, VEC = RowPiece<T>::VEC;
    __shared__ __attribute__((aligned(16))) float lds[64];
    const size_t row = blockIdx.y;
    const int pieces = (a.dim + VEC - 1) / VEC, first = (int)blockIdx.x * a.per_part, end = min(first + a.per_part, pieces);
    float2 *part = a.part + row * (a.parts + 1);
    RowPiece<T> z[NP];
    soft_hold<T, NT, NP, true>(z, a.z + row * a.dim, first, end, a.dim);
    float za = 0.f;
    if (blockIdx.x == 0) policy_action(a, row, za);
    float m[2] = {soft_max<T>(z), 0.f}, s[2] = {0.f, 0.f};
    group_reduce<NT, true>(m, lds);
    // (a part of nothing but -inf adds nothing to a row that has more; a NaN among them is no maximum, but in the sum)
    s[0] = soft_sum<T, NT, NP, true>(z, SoftExp<T>(m[0] == -__builtin_inff() ? 0.f : m[0], a), a.dim);
    group_reduce<NT, false>(s, lds + 32);
    if (threadIdx.x != 0) return;
    part[blockIdx.x] = make_float2(m[0], s[0]);
    if (blockIdx.x == 0) part[a.parts] = make_float2(za, 0.f);
}
// ... which every workgroup of the row joins before it writes its part's gradient.
template <typename T, typename E>
__global__ __launch_bounds__(POLICY_NT) void policy_join_kernel(const PolicyArgs<T> a) {
    constexpr int NT = POLICY_NT, NP = POLICY_NP, VEC = RowPiece<T>::VEC;
    __shared__ __attribute__((aligned(16))) float lds[64];
    const size_t row = blockIdx.y;
    const int pieces = (a.dim + VEC - 1) / VEC, first = (int)blockIdx.x * a.per_part, end = min(first + a.per_part, pieces);
    const float2 *part = a.part + row * (a.parts + 1);
    RowPiece<T> z[NP];
    if (a.grad) soft_hold<T, NT, NP, true>(z, a.z + row * a.dim, first, end, a.dim);
    const int action = a.action[row];
    const PolicyGiven given = policy_given(a, row);
    const float za = part[a.parts].x;
    float top[2] = {-__builtin_inff(), 0.f}, sum[2] = {0.f, 0.f};
    float2 mine = threadIdx.x < a.parts ? part[threadIdx.x] : make_float2(-__builtin_inff(), 0.f);  // (most rows have no more than that)
    top[0] = mine.x;
    for (int i = threadIdx.x + NT; i < a.parts; i += NT) top[0] = fmaxf(top[0], part[i].x);
    group_reduce<NT, true>(top, lds);
    for (int i = threadIdx.x;;) {
        sum[0] += mine.x == -__builtin_inff() ? mine.y : mine.y * soft_exp(mine.x, top[0], a);
        i += NT;
        if (i >= a.parts) break;
        mine = part[i];
    }
    group_reduce<NT, false>(sum, lds + 32);
    const E e(top[0], a);
    const PolicyRow r = policy_row(a, given, row, action, za, top[0], logf(sum[0]), blockIdx.x == 0 && threadIdx.x == 0);
    if (!a.grad) return;
    policy_put<T, NT, NP, true>(z, a.grad + row * a.dim, first, end, e, e.unit(sum[0]), r, action, a.dim);
}

template <typename T, typename E, int NT, int NP>
static void policy_rows(PolicyArgs<T> a, int ns) {
    const int most = (int)(ROW_THREADS / NT);
    for (; a.first < ns; a.first += most) {
        const int n = ns - a.first < most ? ns - a.first : most;
        a.rows = a.first + n;
        if (NT == 64) hipLaunchKernelGGL((policy_row_kernel<T, E, NT, NP>), dim3((n + 3) / 4), dim3(256), 0, state().stream, a);
        else hipLaunchKernelGGL((policy_row_kernel<T, E, NT, NP>), dim3(n), dim3(NT), 0, state().stream, a);
    }
}

template <typename T, typename E>
static int policy_launch(PolicyArgs<T> &a, int ns) {
    const int pieces = (a.dim + RowPiece<T>::VEC - 1) / RowPiece<T>::VEC, cu = state().num_cu;
    if (pieces > 4096 && (long)ns * (a.dim > 65536 ? 2 : 6) <= cu) {
        const int most = POLICY_NT * POLICY_NP;
        int parts = 2 * cu / ns, least = (pieces + most - 1) / most;
        parts = parts < (pieces + POLICY_NT - 1) / POLICY_NT ? parts : (pieces + POLICY_NT - 1) / POLICY_NT;
        parts = parts > least ? parts : least;
        a.per_part = (pieces + parts - 1) / parts;
        a.parts = (pieces + a.per_part - 1) / a.per_part;
        a.part = reinterpret_cast<float2 *>(workspace(sizeof(float2) * (size_t)ns * (a.parts + 1)));
        if (!a.part) return 2;
        hipLaunchKernelGGL((policy_part_kernel<T>), dim3(a.parts, ns), dim3(POLICY_NT), 0, state().stream, a);
        hipLaunchKernelGGL((policy_join_kernel<T, E>), dim3(a.grad ? a.parts : 1, ns), dim3(POLICY_NT), 0, state().stream, a);
    } else if ((pieces <= 256 && ns >= 4 * cu) || (pieces <= 512 && ns >= 16 * cu)) {
        if (pieces <= 64) policy_rows<T, E, 64, 1>(a, ns);
        else if (pieces <= 128) policy_rows<T, E, 64, 2>(a, ns);
        else if (pieces <= 256) policy_rows<T, E, 64, 4>(a, ns);
        else policy_rows<T, E, 64, 8>(a, ns);
    } else if (pieces <= 256) {
        policy_rows<T, E, 256, 1>(a, ns);
    } else if (pieces <= 512) {
        policy_rows<T, E, 256, 2>(a, ns);
    } else if (pieces <= 1024) {
        policy_rows<T, E, 256, 4>(a, ns);
    } else if (pieces <= 2048) {
        policy_rows<T, E, 256, 8>(a, ns);
    } else if (pieces <= 4096) {
        policy_rows<T, E, 512, 8>(a, ns);
    } else if (pieces <= 8192) {
        policy_rows<T, E, 1024, 8>(a, ns);
    } else if (pieces <= 12288) {
        policy_rows<T, E, 1024, 12>(a, ns);
    } else if (pieces <= 16384) {
        policy_rows<T, E, 1024, 16>(a, ns);
    } else {
        policy_rows<T, E, 1024, 0>(a, ns);
    }
    return hip_ok(hipGetLastError(), "policy loss launch") ? 0 : 2;
}

template <typename T, typename Args>
static int policy_step(const Args *a, int ns, int step, const char *fn) {
    if (!a || !a->output) return rows_bad(fn, "null argument structure");
    const int dim = a->output->dim;
    if (dim <= 0 || dim > ROW_MOST) return rows_bad(fn, "invalid tensor geometry");
    if (step < 0 || step > 2) return rows_bad(fn, "step is not 0, 1 or 2");
    if (!(a->temperature >= 1e-6f && a->temperature <= 1e6f)) return rows_bad(fn, "the temperature is not in 1e-6 .. 1e6");
    if (!(a->clip_low >= 0.f && a->clip_high >= 0.f)) return rows_bad(fn, "a border of the ratio is no number from 0 on");
    if (!(fabsf(a->beta) < __builtin_inff() && fabsf(a->weight) < __builtin_inff())) return rows_bad(fn, "beta or the weight is no finite number");
    const bool loss = step != 1, grad = step != 0;
    if (!a->output->data || !a->actions || !a->old_logp || !a->advantages || (loss && !a->wr_loss) || (grad && !a->output->diff)) return rows_bad(fn, "null buffer");
    if (ns > ROW_MOST) return rows_bad(fn, "more than 2^30 samples");
    if (ns <= 0) return 0;
    if (!ensure_init()) return 2;
    const size_t n = (size_t)ns * dim, rows = (size_t)ns;
    Stager sg;
    PolicyArgs<T> d = {};
    static_cast<SoftScale &>(d) = SoftScale(a->temperature);
    d.z = sg.in(reinterpret_cast<const T *>(a->output->data), n);
    d.action = sg.in<int>(a->actions, rows);
    d.old = sg.in<float>(a->old_logp, rows);
    d.adv = sg.in<float>(a->advantages, rows);
    if (a->ref_logp && a->beta != 0.f) d.ref = sg.in<float>(a->ref_logp, rows);
    if (a->row_weight) d.row_weight = sg.in<float>(a->row_weight, rows);
    if (loss) d.loss = sg.out<float>(a->wr_loss, rows);
    if (a->wr_logp) d.logp = sg.out<float>(a->wr_logp, rows);
    if (grad) d.grad = sg.out(reinterpret_cast<T *>(a->output->diff), n);
    if (sg.failed()) return 2;
    d.rows = ns;
    d.dim = dim;
    d.low = 1.f - a->clip_low;
    d.high = 1.f + a->clip_high;
    d.beta = a->beta;
    d.weight = a->weight;
    if constexpr (sizeof(T) == 2) {
        if (a->temperature >= SOFT_RATIO_LEAST) return sg.finish(policy_launch<T, SoftRatio>(d, ns));
    }
    return sg.finish(policy_launch<T, SoftExp<T>>(d, ns));
}

}  // namespace ptl

extern "C" {
int ptl_policy_loss_fp32_batched(const struct policy_loss_args *a, int ns, int step) {
    return ptl::policy_step<float>(a, ns, step, "ptl_policy_loss_fp32_batched");
}
int ptl_policy_loss_fp16_batched(const struct policy_loss_args_fp16 *a, int ns, int step) {
    return ptl::policy_step<ptl::half_t>(a, ns, step, "ptl_policy_loss_fp16_batched");
}
}
