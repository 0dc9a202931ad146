// lanes.h -- exchanges between the lanes of a wave in vector instructions.  A shuffle through
// LDS (ds_bpermute) answers after some hundred cycles; chains of them, as in sorts and scans
// of one wave, are bound by that.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ds3k {

// v of lane l ^ J.
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v)
{
    static_assert(J == 1 || J == 2 || J == 4 || J == 8 || J == 16 || J == 32, "a lane's distance");
    const int i = (int)v;
    if constexpr (J == 1) return (uint32_t)__builtin_amdgcn_mov_dpp(i, 0xb1, 0xf, 0xf, true);        // lanes 1, 0, 3, 2
    else if constexpr (J == 2) return (uint32_t)__builtin_amdgcn_mov_dpp(i, 0x4e, 0xf, 0xf, true);   // lanes 2, 3, 0, 1
    else if constexpr (J == 4)               // mirrored in 8, then in 4: l ^ 7 ^ 3
        return (uint32_t)__builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(i, 0x141, 0xf, 0xf, true), 0x1b, 0xf, 0xf, true);
    else if constexpr (J == 8) return (uint32_t)__builtin_amdgcn_mov_dpp(i, 0x128, 0xf, 0xf, true);  // turned by 8 in 16
    else if constexpr (J == 16) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? s[0] : s[1];
    } else {
        const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? s[0] : s[1];
    }
}

template <int J>
__device__ __forceinline__ unsigned long long lane_xor(unsigned long long v)
{
    return (unsigned long long)lane_xor<J>((uint32_t)(v >> 32)) << 32 | lane_xor<J>((uint32_t)v);
}

template <int J>
__device__ __forceinline__ float lane_xor(float v) { return __uint_as_float(lane_xor<J>(__float_as_uint(v))); }

template <int J>
__device__ __forceinline__ double lane_xor(double v)
{
    return __builtin_bit_cast(double, lane_xor<J>(__builtin_bit_cast(unsigned long long, v)));
}

template <int J>
__device__ __forceinline__ long long lane_xor(long long v) { return (long long)lane_xor<J>((unsigned long long)v); }

// f over the 16 (UPTO 8) or 64 (32) lanes around each, in every one of them.
template <int UPTO, typename T, typename F>
__device__ __forceinline__ T lanes_join(T v, F f)
{
    v = f(v, lane_xor<1>(v));
    v = f(v, lane_xor<2>(v));
    v = f(v, lane_xor<4>(v));
    v = f(v, lane_xor<8>(v));
    if constexpr (UPTO > 8) {
        v = f(v, lane_xor<16>(v));
        v = f(v, lane_xor<32>(v));
    }
    return v;
}

// v moved by a DPP control, 0 where no lane gives one or ROWS leaves the row out.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t lane_move(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ unsigned long long lane_move(unsigned long long v)
{
    return (unsigned long long)lane_move<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | lane_move<CTRL, ROWS>((uint32_t)v);
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double lane_move(double v)
{
    return __builtin_bit_cast(double, lane_move<CTRL, ROWS>(__builtin_bit_cast(unsigned long long, v)));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ long long lane_move(long long v) { return (long long)lane_move<CTRL, ROWS>((unsigned long long)v); }

// Inclusive sums over 16 lanes each.
template <typename T>
__device__ __forceinline__ T row_scan(T v)
{
    v += lane_move<0x111>(v);
    v += lane_move<0x112>(v);
    v += lane_move<0x114>(v);
    v += lane_move<0x118>(v);
    return v;
}

// Inclusive sums over the wave.
template <typename T>
__device__ __forceinline__ T wave_scan(T v)
{
    v = row_scan(v);
    v += lane_move<0x142, 0xa>(v);           // the last of row 0 to row 1, of row 2 to row 3
    v += lane_move<0x143, 0xc>(v);           // the last of row 1 to rows 2 and 3
    return v;
}

// v of one lane, the same for all.
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ unsigned long long lane_of(unsigned long long v, int lane)
{
    return (unsigned long long)lane_of((uint32_t)(v >> 32), lane) << 32 | lane_of((uint32_t)v, lane);
}
__device__ __forceinline__ double lane_of(double v, int lane)
{
    return __builtin_bit_cast(double, lane_of(__builtin_bit_cast(unsigned long long, v), lane));
}

// One step of a bitonic sort: the pairs J apart, ascending where threadIdx.x & k is 0, or the other way round.
template <int J, typename T>
__device__ __forceinline__ T sort_step(T v, int k, bool down = false)
{
    const T o = lane_xor<J>(v);
    return ((threadIdx.x & J) == 0) == (((threadIdx.x & k) == 0) != down) ? (o < v ? o : v) : (o < v ? v : o);
}

// Merges, from pairs J apart on, two runs of 2 J values in all into one; k, down: as in sort_step.
template <int J, typename T>
__device__ __forceinline__ T sort_merge(T v, int k, bool down = false)
{
    v = sort_step<J>(v, k, down);
    if constexpr (J > 1) v = sort_merge<J / 2>(v, k, down);
    return v;
}

// The lanes' values ascending over UPTO lanes each (16 or 64).
template <int UPTO, typename T>
__device__ __forceinline__ T sort_lanes(T v)
{
    v = sort_merge<1>(v, 2);
    v = sort_merge<2>(v, 4);
    v = sort_merge<4>(v, 8);
    if constexpr (UPTO == 16) return sort_merge<8>(v, 0);
    v = sort_merge<8>(v, 16);
    v = sort_merge<16>(v, 32);
    return sort_merge<32>(v, 0);
}

}  // namespace ds3k
