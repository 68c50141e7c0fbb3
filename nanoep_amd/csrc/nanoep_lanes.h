// Reductions over 8, 16, 32 or 64 neighbouring lanes of a wavefront, the result in all of them: four steps within a row of 16
// by DPP, two by the row swaps of gfx950, no LDS.  The order of a sum is always the same.
#ifndef NANOEP_LANES_H_
#define NANOEP_LANES_H_

#include "nanoep_device.h"

namespace nanoep {

struct LanesMin {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a < b ? a : b; }
};
struct LanesMax {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
    // (of two values the one that is no NaN)
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct LanesSum {
    template <class T>
    __device__ __forceinline__ T operator()(T a, T b) const {
        return a + b;
    }
};

template <int kControl>
__device__ __forceinline__ uint32_t lanes_moved(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kControl, 0xf, 0xf, true));
}
template <int kControl>
__device__ __forceinline__ int lanes_moved(int v) {
    return __builtin_amdgcn_update_dpp(0, v, kControl, 0xf, 0xf, true);
}
template <int kControl>
__device__ __forceinline__ float lanes_moved(float v) {
    return __uint_as_float(lanes_moved<kControl>(__float_as_uint(v)));
}
template <int kControl>
__device__ __forceinline__ double lanes_moved(double v) {
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(v));
    const uint64_t low = lanes_moved<kControl>(static_cast<uint32_t>(bits)), high = lanes_moved<kControl>(static_cast<uint32_t>(bits >> 32));
    return __longlong_as_double(static_cast<long long>(high << 32 | low));
}

// A value and the one 16 or 32 lanes away, in an order that is the same for both lanes.
template <int kDistance>
__device__ __forceinline__ void lanes_pair(uint32_t v, uint32_t& a, uint32_t& b) {
    const auto both = kDistance == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    a = both[0];
    b = both[1];
}
template <int kDistance>
__device__ __forceinline__ void lanes_pair(int v, int& a, int& b) {
    uint32_t x, y;
    lanes_pair<kDistance>(static_cast<uint32_t>(v), x, y);
    a = static_cast<int>(x);
    b = static_cast<int>(y);
}
template <int kDistance>
__device__ __forceinline__ void lanes_pair(float v, float& a, float& b) {
    uint32_t x, y;
    lanes_pair<kDistance>(__float_as_uint(v), x, y);
    a = __uint_as_float(x);
    b = __uint_as_float(y);
}
template <int kDistance>
__device__ __forceinline__ void lanes_pair(double v, double& a, double& b) {
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(v));
    uint32_t low[2], high[2];
    lanes_pair<kDistance>(static_cast<uint32_t>(bits), low[0], low[1]);
    lanes_pair<kDistance>(static_cast<uint32_t>(bits >> 32), high[0], high[1]);
    a = __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(high[0]) << 32 | low[0]));
    b = __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(high[1]) << 32 | low[1]));
}

template <int kLanes, class T, class Operation>
__device__ __forceinline__ T lanes_reduce(T v, Operation operation) {
    static_assert(kLanes == 8 || kLanes == 16 || kLanes == 32 || kLanes == 64, "8 to 64 lanes");
    v = operation(v, lanes_moved<0xB1>(v));   // quad_perm 1 0 3 2
    v = operation(v, lanes_moved<0x4E>(v));   // quad_perm 2 3 0 1
    v = operation(v, lanes_moved<0x141>(v));  // row_half_mirror
    if constexpr (kLanes >= 16)
        v = operation(v, lanes_moved<0x140>(v));  // row_mirror
    T a, b;
    if constexpr (kLanes >= 32) {
        lanes_pair<16>(v, a, b);
        v = operation(a, b);
    }
    if constexpr (kLanes >= 64) {
        lanes_pair<32>(v, a, b);
        v = operation(a, b);
    }
    return v;
}

template <int kLanes, class T>
__device__ __forceinline__ T lanes_max(T v) {
    return lanes_reduce<kLanes>(v, LanesMax{});
}
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_min(uint32_t v) {
    return lanes_reduce<kLanes>(v, LanesMin{});
}
template <int kLanes, class T>
__device__ __forceinline__ T lanes_sum(T v) {
    return lanes_reduce<kLanes>(v, LanesSum{});
}

// The sum over kLanes lanes with the lanes that are farthest apart added first: whoever has added 64 values down to kLanes of them, those farthest
// apart first as well, has the same sum for any kLanes.
template <int kLanes, class T>
__device__ __forceinline__ T lanes_sum_from_afar(T v) {
    static_assert(kLanes == 8 || kLanes == 16 || kLanes == 32 || kLanes == 64, "8 to 64 lanes");
    T a, b;
    if constexpr (kLanes >= 64) {
        lanes_pair<32>(v, a, b);
        v = a + b;
    }
    if constexpr (kLanes >= 32) {
        lanes_pair<16>(v, a, b);
        v = a + b;
    }
    if constexpr (kLanes >= 16)
        v += lanes_moved<0x128>(v);  // row_ror 8
    v += lanes_moved<0x141>(v);      // row_half_mirror
    v += lanes_moved<0x4E>(v);       // quad_perm 2 3 0 1
    return v + lanes_moved<0xB1>(v);  // quad_perm 1 0 3 2
}

// The lanes of a group of kLanes for which `condition` holds, the group's first lane as bit 0.
template <int kLanes>
__device__ __forceinline__ uint64_t lanes_where(bool condition) {
    const uint64_t all = __ballot(condition);
    if constexpr (kLanes == 64)
        return all;
    return all >> (threadIdx.x % kWave / kLanes * kLanes) & ((uint64_t{1} << kLanes) - 1);
}

// The sum over the lanes of a group of kLanes ahead of this one.
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_before(uint32_t v) {
    static_assert(kLanes >= 16, "whole rows of 16");
    uint32_t up_to = v;
    up_to += lanes_moved<0x111>(up_to);  // row_shr 1, zero at the row's start
    up_to += lanes_moved<0x112>(up_to);
    up_to += lanes_moved<0x114>(up_to);
    up_to += lanes_moved<0x118>(up_to);
    for (int row = 16; row < kLanes; row += 16) {  // a row's end goes into the next one
        const uint32_t ahead = __shfl(up_to, (threadIdx.x % kWave / kLanes) * kLanes + row - 1, kWave);
        up_to += threadIdx.x % kLanes / 16 * 16 == row ? ahead : 0;
    }
    return up_to - v;
}

// The sum over the lanes of a wavefront that are in the same place of their groups of kLanes.
template <int kLanes>
__device__ __forceinline__ float groups_sum(float v) {
    float a, b;
    if constexpr (kLanes <= 8)
        v += lanes_moved<0x128>(v);  // row_ror 8
    if constexpr (kLanes <= 16) {
        lanes_pair<16>(v, a, b);
        v = a + b;
    }
    if constexpr (kLanes <= 32) {
        lanes_pair<32>(v, a, b);
        v = a + b;
    }
    return v;
}

// What a wavefront's lanes wrote to LDS is there for its other lanes (LDS works a wavefront's accesses off in order).
__device__ __forceinline__ void wavefront_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

}  // namespace nanoep

#endif  // NANOEP_LANES_H_
