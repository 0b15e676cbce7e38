// lanes.hpp - exchanges between the four 16-lane groups of a wave without LDS
// (v_permlane16_swap / v_permlane32_swap), and wave reductions built on them.
#pragma once

#include "common.hpp"
#include "wave_ops.hpp"

namespace mimoe {

// groups 1 and 3 of a change places with groups 0 and 2 of b
__device__ __forceinline__ void swap16(uint32_t &a, uint32_t &b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
// lanes 32 .. 63 of a change places with lanes 0 .. 31 of b
__device__ __forceinline__ void swap32(uint32_t &a, uint32_t &b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

// the value of the lane that DPP control CTRL pairs with this one
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)dpp_i<CTRL>((int)(uint32_t)u), hi = (uint32_t)dpp_i<CTRL>((int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// v of this lane and of its partners 16 (32) lanes away, as a pair in the same
// order in both lanes
__device__ __forceinline__ void pair16(double v, double &a, double &b) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    uint32_t l0 = (uint32_t)u, l1 = l0, h0 = (uint32_t)(u >> 32), h1 = h0;
    swap16(l0, l1);
    swap16(h0, h1);
    a = __builtin_bit_cast(double, (uint64_t)h0 << 32 | l0);
    b = __builtin_bit_cast(double, (uint64_t)h1 << 32 | l1);
}
__device__ __forceinline__ void pair32(double v, double &a, double &b) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    uint32_t l0 = (uint32_t)u, l1 = l0, h0 = (uint32_t)(u >> 32), h1 = h0;
    swap32(l0, l1);
    swap32(h0, h1);
    a = __builtin_bit_cast(double, (uint64_t)h0 << 32 | l0);
    b = __builtin_bit_cast(double, (uint64_t)h1 << 32 | l1);
}

// the largest over the wave, in every lane
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max_u(uint32_t m) {
    const uint32_t o = (uint32_t)dpp_i<CTRL>((int)m);
    return o > m ? o : m;
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t m) {
    m = dpp_max_u<0xB1>(m);
    m = dpp_max_u<0x4E>(m);
    m = dpp_max_u<0x141>(m);
    m = dpp_max_u<0x140>(m);
    uint32_t o = m;
    swap16(m, o);
    m = o > m ? o : m;
    o = m;
    swap32(m, o);
    return o > m ? o : m;
}

// sum over the wave, the same bits in every lane
__device__ __forceinline__ double wave_sum_d(double v) {
    v += dpp_d<0xB1>(v);
    v += dpp_d<0x4E>(v);
    v += dpp_d<0x141>(v);
    v += dpp_d<0x140>(v);
    double a, b;
    pair16(v, a, b);
    v = a + b;
    pair32(v, a, b);
    return a + b;
}

}  // namespace mimoe
