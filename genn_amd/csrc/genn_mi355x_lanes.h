// Part of libgenn_mi355x.so: exchanges between the lanes of a wavefront without a trip through LDS, shared by the operators' kernels.
#ifndef GENN_MI355X_LANES_H
#define GENN_MI355X_LANES_H

#include <hip/hip_runtime.h>

#include <cstdint>

namespace gennmi_lanes
{
// The value of the lane's partner in the other half of its group of 2 WIDTH lanes.  Lane l's partner is l ^ WIDTH for WIDTH 1, 2, 16 and 32; for 4 and 8
// it is the lane mirrored in the group: for sums and maxima one is as good as the other.
template<int WIDTH> __device__ inline float partner(float x)
{
    const int v = __float_as_int(x);
    if constexpr(WIDTH == 1) { return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true)); }          // quad_perm [1, 0, 3, 2]
    else if constexpr(WIDTH == 2) { return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true)); }     // quad_perm [2, 3, 0, 1]
    else if constexpr(WIDTH == 4) { return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true)); }    // row_half_mirror
    else if constexpr(WIDTH == 8) { return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true)); }    // row_mirror
    else {
        // (swaps the odd rows of 16 lanes, or the upper half, of its first operand with the even ones, or the lower half, of its second)
        const auto s = [&] {
            if constexpr(WIDTH == 16) { return __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false); }
            else { return __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false); }
        }();
        return __int_as_float((int)((threadIdx.x & WIDTH) ? s[0] : s[1]));
    }
}
// Two values become one register: lanes of the lower halves have a's sum with its partner, those of the upper halves b's.
template<int WIDTH> __device__ inline float fold(float a, float b)
{
    if constexpr(WIDTH >= 16) {
        const auto s = [&] {
            if constexpr(WIDTH == 16) { return __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false); }
            else { return __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false); }
        }();
        return __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    else {
        const bool upper = threadIdx.x & WIDTH;
        return (upper ? b : a) + partner<WIDTH>(upper ? a : b);
    }
}
// Of M values a lane, M a power of two, one register is left: lane l has its share of the sum over the lanes of value l / (64 / M), as the 64 / M lanes of that
// value together have all of it.
template<int M, int WIDTH = 32> __device__ inline float shareOfLanes(const float (&v)[M])
{
    if constexpr(M > 1) {
        float half[M / 2];
        #pragma unroll
        for(int i = 0; i < M / 2; i++) { half[i] = fold<WIDTH>(v[i], v[i + M / 2]); }
        return shareOfLanes<M / 2, WIDTH / 2>(half);
    }
    else { return v[0]; }
}
// Of two values' bits, over all lanes: of floats that are not negative the maximum, and not a number where one of them is not.  The halves of the wavefront
// have one value each after the first step.
__device__ inline void maxOfLanes(uint32_t &a, uint32_t &b)
{
    const auto halves = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    uint32_t x = max(halves[0], halves[1]);
    const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(rows[0], rows[1]);
    x = max(x, __float_as_uint(partner<8>(__uint_as_float(x))));
    x = max(x, __float_as_uint(partner<4>(__uint_as_float(x))));
    x = max(x, __float_as_uint(partner<2>(__uint_as_float(x))));
    x = max(x, __float_as_uint(partner<1>(__uint_as_float(x))));
    a = __builtin_amdgcn_readlane(x, 0);
    b = __builtin_amdgcn_readlane(x, 32);
}
}
#endif
