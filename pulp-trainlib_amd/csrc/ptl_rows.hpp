// Rows of tensors in 16-byte pieces, and sums over the threads of a row: shared by the kernels that give a row to a wave or to
// a workgroup.
#pragma once
#include <stdio.h>

#include <type_traits>

#include "ptl_common.hpp"
#include "ptl_host.hpp"
#include "ptl_sum.hpp"

namespace ptl {

typedef unsigned row_u4 __attribute__((ext_vector_type(4), aligned(1)));  // 16 bytes wherever they start
typedef float row_f4 __attribute__((ext_vector_type(4)));
typedef unsigned row_u2 __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned row_u1 __attribute__((aligned(1)));

template <typename T>
struct RowPiece {
    static constexpr int VEC = 16 / (int)sizeof(T);
    union {
        row_u4 raw;
        T e[VEC];
    };
    // How a thread holds piece p of a row of at least VEC elements where the whole row is in registers before any of it is written:
    // the piece that reaches over the end covers the row's last VEC elements, the first cut() of which are another piece's too
    // (pieces behind the end: all of them).  They are left out of sums and written twice with the same values, so that no load and
    // no store depends on where the row ends: kernels of a few pieces a thread are bound by fetching their own instructions, and
    // values written one by one were most of those (a row of 14144 fp16 values through a gradient: 11 us, 5 so).
    static __device__ inline int cut(int p, int dim) { return p * VEC - min(p * VEC, max(dim - VEC, 0)); }
    // (a row held in registers is far shorter than 4 GB: the row's address plus an unsigned offset is one instruction's operand)
    static __device__ inline unsigned place(int p, int dim) { return (unsigned)min(p * VEC, dim - VEC) * (unsigned)sizeof(T); }
    // STREAM: past the caches, for rows that nothing else of the launch reads.
    template <bool SHORT, bool STREAM = false>
    __device__ inline void hold(const T *row, int p, int dim) {
        if (SHORT && dim < VEC) fetch(row, p, dim);
        else if (STREAM) raw = __builtin_nontemporal_load(reinterpret_cast<const row_u4 *>(reinterpret_cast<const char *>(row) + place(p, dim)));
        else raw = *reinterpret_cast<const row_u4 *>(reinterpret_cast<const char *>(row) + place(p, dim));
    }
    template <bool SHORT, bool STREAM = false>
    __device__ inline void put(T *row, int p, int dim) const {
        if (SHORT && dim < VEC) store(row, p, dim);
        else if (STREAM && p * VEC < dim) __builtin_nontemporal_store(raw, reinterpret_cast<row_u4 *>(reinterpret_cast<char *>(row) + place(p, dim)));
        else if (p * VEC < dim) *reinterpret_cast<row_u4 *>(reinterpret_cast<char *>(row) + place(p, dim)) = raw;
    }
    // Piece p of a row of `dim` elements.  No load depends on where the row ends: a piece that reaches over the end is read so that
    // it ends there, and trim() moves its values down and puts zeros behind them (only the waves that hold such a piece do).  All
    // of a thread's pieces are fetched before the first is trimmed.
    template <bool STREAM = false>
    __device__ inline void fetch(const T *row, int p, int dim) {
        if (dim >= VEC) {
            const row_u4 *from = reinterpret_cast<const row_u4 *>(row + min(p * VEC, dim - VEC));
            raw = STREAM ? __builtin_nontemporal_load(from) : *from;
        } else {
            // (rows shorter than a piece: value by value, the last one first)
            typedef typename std::conditional<sizeof(T) == 4, unsigned, typename std::conditional<sizeof(T) == 2, unsigned short, unsigned char>::type>::type Bits;
            constexpr int B = 8 * (int)sizeof(T);
            unsigned long long lo = 0, hi = 0;
#pragma nounroll
            for (int i = p == 0 ? dim - 1 : -1; i >= 0; --i) {
                hi = hi << B | lo >> (64 - B);
                lo = lo << B | __builtin_bit_cast(Bits, row[i]);
            }
            raw = row_u4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
        }
    }
    __device__ inline void trim(int p, int dim) {
        if (dim < VEC) return;
        const int cut = p * VEC - min(p * VEC, dim - VEC);
        if (!__any(cut)) return;
        unsigned long long lo = (unsigned long long)raw.y << 32 | raw.x, hi = (unsigned long long)raw.w << 32 | raw.z;
        const unsigned bytes = (unsigned)min(cut, VEC) * (unsigned)sizeof(T), bits = (bytes & 7) * 8;
        if (bytes >= 8) {
            lo = hi;
            hi = 0;
        }
        if (bytes == 16) lo = 0;
        lo = lo >> bits | hi << 1 << (63 - bits);
        hi >>= bits;
        raw = row_u4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
    }
    __device__ inline void load(const T *row, int p, int dim) {
        fetch(row, p, dim);
        trim(p, dim);
    }
    __device__ inline void store(T *row, int p, int dim) const {
        const int at = p * VEC;
        if (at + VEC <= dim) {
            *reinterpret_cast<row_u4 *>(row + at) = raw;
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (at + i < dim) row[at + i] = e[i];
        }
    }
};

// A value as it is stored.  It is rounded to fp32 first, in every place alike: left to itself the compiler joins the last operation and the
// rounding to fp16 for some values of a piece and not for others, which gives another value in one of thousands, and the values that
// two pieces share (RowPiece::put) would depend on which is written last.
template <typename T>
__device__ inline T row_round(float f) {
    if constexpr (sizeof(T) == 2) asm("" : "+v"(f));
    return (T)f;
}

constexpr int ROW_MOST = 1 << 30;  // elements of a row, rows of a call
constexpr long ROW_THREADS = 1l << 31;  // of a launch (it takes 2^32 - 1; calls with more rows are several launches)

// Sums (and maxima) of N values over the 64 lanes of a wave, the same in every lane.
__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}
__device__ inline float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
    return v;
}
// The larger value, or NaN where either is none (one instruction takes three of them).
__device__ inline float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ inline float wave_nan_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = nan_max(v, __shfl_xor(v, off));
    return v;
}

// ... over the TPR threads that have a row: one wave, or a workgroup (a float per wave and value in `lds`, which the caller
// does not use again without a barrier).
template <int TPR, int N, bool MAX1 = false>  // MAX1: the second value is a maximum that keeps NaN
__device__ inline void row_reduce(float (&v)[N], float (*lds)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = MAX1 && i == 1 ? wave_nan_max(v[i]) : wave_sum(v[i]);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) lds[wave][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = lds[0][i];
#pragma unroll
            for (int w = 1; w < TPR / 64; ++w) s = MAX1 && i == 1 ? nan_max(s, lds[w][i]) : s + lds[w][i];
            v[i] = s;
        }
    }
}

// out[c] = the sum over the shares of part[share][c]: 32 columns (a 128-byte line) a workgroup, 32 shares at a time with four loads in
// flight, so that a few thousand columns fill the chip (1024 shares of 4096: 18 us with 64 columns and 4 shares at a time, 5 so).
// The columns 32 group .. of a workgroup of NT threads: each of the 32 walks in its order, whichever thread has it.
template <typename T, int NT>
__device__ inline void row_shares_of(const float *__restrict__ part, T *__restrict__ out, int dim, int shares, int group, LongSum<T> (*red)[32]) {
    const int o = threadIdx.x & 31, c = group * 32 + o;
#pragma unroll
    for (int g = threadIdx.x >> 5; g < 32; g += NT / 32) {
        LongSum<T> s;
        s.clear();
        if (c < dim) {
            int z = g;
            for (; z + 96 < shares; z += 128) {
                float v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = part[(size_t)(z + 32 * u) * dim + c];
#pragma unroll
                for (int u = 0; u < 4; ++u) s.add(v[u]);
            }
            for (; z < shares; z += 32) s.add(part[(size_t)z * dim + c]);
        }
        red[g][o] = s;
    }
    __syncthreads();
    if (threadIdx.x >= 32 || c >= dim) return;
    LongSum<T> s = red[0][o];
    for (int k = 1; k < 32; ++k) s.add(red[k][o]);
    out[c] = (T)s.value();
}
template <typename T>
__global__ __launch_bounds__(1024) void row_shares_kernel(const float *__restrict__ part, T *__restrict__ out, int dim, int shares) {
    __shared__ LongSum<T> red[32][32];
    row_shares_of<T, 1024>(part, out, dim, shares, (int)(blockIdx.y * gridDim.x + blockIdx.x), red);
}
template <typename T>
inline void row_shares(const float *part, T *out, int dim, int shares) {
    const int groups = (dim + 31) / 32, most = (int)(ROW_THREADS / 1024);  // (the last of several rows of the grid may reach beyond the end)
    hipLaunchKernelGGL((row_shares_kernel<T>), dim3(groups < most ? groups : most, (groups + most - 1) / most), dim3(1024), 0, state().stream, part, out, dim,
                       shares);
}

// A rejected call: its message, as the other entry points give it.
inline int rows_bad(const char *fn, const char *what) {
    printf("[%s] %s\n", fn, what);
    set_error("%s: %s", fn, what);
    return 1;
}

template <typename Blob>
inline auto *blob_data(const Blob *b) { return b ? b->data : nullptr; }
template <typename Blob>
inline auto *blob_diff(const Blob *b) { return b ? b->diff : nullptr; }

}  // namespace ptl
