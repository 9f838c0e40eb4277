// Rows of logits held in registers: their maximum, the sum of their exponentials and a gradient that is a multiple of the softmax, at a
// temperature T.  Shared by the losses over classes.
#pragma once
#include "ptl_rows.hpp"

namespace ptl {

struct SoftScale {
    float inv_t, hi, lo, least;  // 1 / T; log2(e) / T as the sum of two floats above 0; z - m from which on exp((z - m) / T) is 0
    SoftScale() = default;
    explicit SoftScale(float temperature) {
        const double log2e = 1.4426950408889634074 / temperature;
        inv_t = 1.f / temperature;
        hi = (float)log2e;
        if ((double)hi >= log2e) hi = nextafterf(hi, 0.f);
        lo = (float)(log2e - (double)hi);  // above 0: a difference of -inf gives -inf from both
        least = (float)(-150. / log2e);
    }
};

// exp((z - m) / T) of an entry: the exponent as the sum of two floats, the second of which corrects the result.
__device__ inline float soft_exp(float z, float m, const SoftScale &a) {
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
struct SoftExp {
    float m, rest;
    const SoftScale &a;
    __device__ inline SoftExp(float max, const SoftScale &a) : a(a) {
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
    // The logarithm of a sum of these, and what a sum of whole exponentials is in their unit.
    __device__ inline float log(float sum) const { return logf(sum); }
    __device__ inline float unit(float sum) const { return sum; }
};

// ... of fp16 but for a factor of the whole row, 2^-rest, where only ratios count and the logarithm of the sum is corrected by it: an instruction less
// for each class (the policy loss of 2048 rows of 32000 classes 48.2 us and 48.6 with whole exponentials, 4096 of 8200 29.3 and 31.9, 300 of 32000 11.6 and
// 12.3, 8192 of 1000 and 4 of 131072 the same).  Only where the factor is near 1: `rest` is up to half a step of m / T, and logits of 65504 at a temperature of 2^-7 have
// m / T log2(e) below 2^24, whose half step is 1/2.  (Unbounded it would be 944 at a maximum of 30000 and the smallest temperature, where the
// largest class's exponential is then infinite or 0.)
constexpr float SOFT_RATIO_LEAST = 0x1p-7f;  // the temperature from which on
struct SoftRatio : SoftExp<half_t> {
    __device__ inline SoftRatio(float max, const SoftScale &a) : SoftExp<half_t>(max, a) {}
    __device__ inline float operator()(half_t z) const { return __builtin_amdgcn_exp2f(fmaf((float)z, a.hi, m)); }
    __device__ inline float log(float sum) const { return fmaf(rest, 0.693147181f, logf(sum)); }
    __device__ inline float unit(float sum) const { return sum * __builtin_amdgcn_exp2f(-rest); }
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

// NP pieces of logits in each of NT threads, from piece `first` on.  MINE: each piece has its own classes only, and what the row does
// not have is -inf; else a thread may have classes that are another's too (RowPiece::cut), which only the sum has to know.
template <typename T, int NT, int NP, bool MINE, bool STREAM = false>
__device__ inline void soft_hold(RowPiece<T> (&z)[NP], const T *row, int first, int end, int dim) {
    constexpr int VEC = RowPiece<T>::VEC;
    constexpr bool SHORT = NP == 1;  // rows of less than a piece: one piece a thread
    if (!MINE && !(SHORT && dim < VEC)) {
#pragma unroll
        for (int j = 0; j < NP; ++j) z[j].template hold<false, STREAM>(row, first + j * NT + row_thread<NT>(), dim);
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
__device__ inline void soft_as_read(RowPiece<T> (&z)[NP]) {
#pragma unroll
    for (int j = 0; j < NP; ++j) asm volatile("" : "+v"(z[j].raw));
}
template <typename T, int NP>
__device__ inline float soft_max(const RowPiece<T> (&z)[NP]) {
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
template <typename T, int NT, int NP, bool MINE, typename E>
__device__ inline float soft_sum(const RowPiece<T> (&z)[NP], const E &e, int dim) {
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
__device__ inline void soft_put(const RowPiece<T> (&z)[NP], T *row, int first, int end, const SoftExp<T> &e, float f, bool some, int dim) {
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

}  // namespace ptl
