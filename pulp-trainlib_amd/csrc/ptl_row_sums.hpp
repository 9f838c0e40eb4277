// Sums of several values over the threads of a row, with exchanges between lanes that do not pass LDS.
#pragma once
#include <hip/hip_runtime.h>

namespace ptl {

// v plus what another lane of the same 16 has: `CTRL` says which.
template <int CTRL>
__device__ inline float lane_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
constexpr int LANE_XOR1 = 0xB1, LANE_XOR2 = 0x4E, LANE_MIRROR8 = 0x141, LANE_MIRROR16 = 0x140, LANE_ROTATE8 = 0x128;
// Rows of 16 lanes: 0 + 1 and 2 + 3; halves of 32 lanes.  (Two copies of v whose odd and even rows change places.)
__device__ inline float lane_add16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned a = r[0], b = r[1];  // (of an element as it stands in the vector the cast takes the first)
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
__device__ inline float lane_add32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned a = r[0], b = r[1];  // (of an element as it stands in the vector the cast takes the first)
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
// The sum over the 64 lanes, in all of them.
__device__ inline float lanes_sum(float v) {
    v = lane_add<LANE_MIRROR16>(lane_add<LANE_MIRROR8>(lane_add<LANE_XOR2>(lane_add<LANE_XOR1>(v))));
    return lane_add32(lane_add16(v));
}

// The largest of the lanes' unsigned integers, as the float that it stands for.
template <int CTRL>
__device__ inline unsigned lane_most(unsigned u) {
    return max(u, (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xf, 0xf, true));
}
__device__ inline float lanes_most(unsigned u) {
    u = lane_most<LANE_MIRROR16>(lane_most<LANE_MIRROR8>(lane_most<LANE_XOR2>(lane_most<LANE_XOR1>(u))));
    auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    u = max((unsigned)r[0], (unsigned)r[1]);
    r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    u = max((unsigned)r[0], (unsigned)r[1]);
    return __builtin_bit_cast(float, u);
}

// ... of N values over the TPR threads that have a row: one wave, or a workgroup.  A workgroup's waves leave their sums in `lds`, ROW_SUMS floats
// that the caller does not use again without a barrier: of one value side by side, of several in eights.  Each wave then reads all of them in
// one or two instructions, a value and wave to a lane, adds up across lanes and has every value as a scalar.  (Each thread reading the sums of
// all waves one by one held 48 registers for six values of eight waves and took a third of a row's time.)
template <int TPR, int N>
constexpr int ROW_SUMS = TPR == 64 ? 1 : (N == 1 ? 1 : 8) * (TPR / 64);
template <int TPR, int N>
__device__ inline void row_sums(float (&v)[N], float *lds) {
    static_assert(TPR == 64 || TPR == 256 || TPR == 512 || TPR == 1024, "waves");
    static_assert(N <= 8, "an eight");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum(v[i]);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64, PER = N == 1 ? 1 : 8;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) lds[wave * PER + i] = v[i];
        }
        __syncthreads();
        if constexpr (N == 1) {
            float s = lane_add<LANE_XOR2>(lane_add<LANE_XOR1>(lds[lane & (W - 1)]));
            if constexpr (W >= 8) s = lane_add<LANE_MIRROR8>(s);
            if constexpr (W == 16) s = lane_add<LANE_MIRROR16>(s);
            v[0] = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, s)));
        } else {
            float s = lds[lane & (8 * W - 1)];
            if constexpr (W == 16) s += lds[64 + lane];
            s = lane_add16(lane_add<LANE_ROTATE8>(s));
            if constexpr (W >= 8) s = lane_add32(s);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), i));
        }
    }
}

}  // namespace ptl
