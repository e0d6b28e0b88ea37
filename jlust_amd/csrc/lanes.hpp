// lanes.hpp -- reductions over runs of 2 to 64 lanes of a wave, between vector registers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace jlust {

// v of another lane: of the one whose number differs in bit 0 or 1, of the mirror place
// among 8 or 16.
template <int CTRL, typename A>
__device__ __forceinline__ A from_lane(A v)
{
    if constexpr (sizeof(A) == 4) {
        return __builtin_bit_cast(A, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_mov_dpp((int)u, CTRL, 0xf, 0xf, true);
        const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(u >> 32), CTRL, 0xf, 0xf, true);
        return __builtin_bit_cast(A, (uint64_t)hi << 32 | lo);
    }
}

// f of v here and in the other row of 16 (ROWS 16) or half (32) of the wave.
template <int ROWS, typename A, typename F>
__device__ __forceinline__ A with_other(A v, F &&f)
{
    auto swap = [](uint32_t x) {
        if constexpr (ROWS == 16) return __builtin_amdgcn_permlane16_swap(x, x, false, false);
        else return __builtin_amdgcn_permlane32_swap(x, x, false, false);
    };
    if constexpr (sizeof(A) == 4) {
        const auto r = swap(__builtin_bit_cast(uint32_t, v));
        const uint32_t here = r[0], other = r[1];  // bit_cast of a vector's element takes the first
        return f(__builtin_bit_cast(A, here), __builtin_bit_cast(A, other));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const auto lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
        return f(__builtin_bit_cast(A, (uint64_t)hi[0] << 32 | lo[0]), __builtin_bit_cast(A, (uint64_t)hi[1] << 32 | lo[1]));
    }
}

// f over the first `lanes` (a power of two) lanes of every run of as many, in each of
// them.  Between vector registers: a step by LDS takes some 100 cycles.
template <int LANES, typename A, typename F>
__device__ __forceinline__ A over_lanes(A v, F &&f, int lanes = LANES)
{
    if (LANES >= 2 && lanes >= 2) v = f(v, from_lane<0xB1>(v));
    if (LANES >= 4 && lanes >= 4) v = f(v, from_lane<0x4E>(v));
    if (LANES >= 8 && lanes >= 8) v = f(v, from_lane<0x141>(v));
    if (LANES >= 16 && lanes >= 16) v = f(v, from_lane<0x140>(v));
    if (LANES >= 32 && lanes >= 32) v = with_other<16>(v, f);
    if (LANES >= 64 && lanes >= 64) v = with_other<32>(v, f);
    return v;
}

struct Larger {                                    // of numbers, one instruction
    __device__ __forceinline__ float operator()(float a, float b) const { return __builtin_fmaxf(a, b); }
    __device__ __forceinline__ double operator()(double a, double b) const { return __builtin_fmax(a, b); }
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return b > a ? b : a; }
    __device__ __forceinline__ int operator()(int a, int b) const { return b > a ? b : a; }
};
struct Plus {
    template <typename A>
    __device__ __forceinline__ A operator()(A a, A b) const { return a + b; }
};

}  // namespace jlust
