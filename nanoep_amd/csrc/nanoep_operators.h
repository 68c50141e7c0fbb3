// What the kernels of the expert layer's operators share (nanoep_norm.hip, nanoep_experts.hip,
// nanoep_weighted.hip): 8-bit groups and their scales, bf16 vectors, reductions within a wavefront.
//
// Rows in 8 bits are records: `hidden` e4m3 values, then one fp32 scale for every 128 columns, the whole
// padded to a multiple of 512 bytes, so that nanoep_dispatch moves a record as a bf16 row.  A value stands
// for itself times its group's scale.
#ifndef NANOEP_OPERATORS_H_
#define NANOEP_OPERATORS_H_

#include "nanoep_device.h"

namespace nanoep {

constexpr int kScaleBlock = 128;
constexpr int kRecordAlignment = 512;
constexpr float kLargestFp8 = 448.0f;
// the scale of a group whose values are all smaller than this is this one's: a group of zeros has a finite scale
constexpr float kSmallestAmax = 0x1p-64f;

inline int64_t scale_groups(int64_t columns) { return (columns + kScaleBlock - 1) / kScaleBlock; }
inline int64_t record_bytes_of(int64_t columns) {
    return static_cast<int64_t>(align_up(static_cast<size_t>(columns + 4 * scale_groups(columns)), kRecordAlignment));
}

// A launch of any number of workgroups: an axis of a grid has fewer than 2^32 threads, so more go over two.  The last
// row of such a grid may have workgroups too many, which return.
constexpr int64_t kMostOnAxis = int64_t{1} << 21;  // workgroups, of 1024 threads at most
inline dim3 grid_of(int64_t workgroups) {
    if (workgroups <= kMostOnAxis)
        return dim3(static_cast<unsigned>(workgroups));
    return dim3(static_cast<unsigned>(kMostOnAxis), static_cast<unsigned>((workgroups + kMostOnAxis - 1) / kMostOnAxis));
}
__device__ __forceinline__ int64_t workgroup_number() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

__device__ __forceinline__ float from_bf16_low(uint32_t packed) { return __uint_as_float(packed << 16); }
__device__ __forceinline__ float from_bf16_high(uint32_t packed) { return __uint_as_float(packed & 0xffff0000u); }

// Two values rounded to bf16 (to nearest even, NaN stays one): one instruction on gfx950.
__device__ __forceinline__ uint32_t to_bf16_pair(float low, float high) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 pair = {static_cast<__bf16>(low), static_cast<__bf16>(high)};
    return __builtin_bit_cast(uint32_t, pair);
}

__device__ __forceinline__ void unpack_bf16(const u32x4 v, float (&out)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        out[2 * i] = from_bf16_low(v[i]);
        out[2 * i + 1] = from_bf16_high(v[i]);
    }
}

__device__ __forceinline__ u32x4 pack_bf16(const float (&v)[8]) {
    u32x4 packed;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        packed[i] = to_bf16_pair(v[2 * i], v[2 * i + 1]);
    return packed;
}

// Four values rounded to e4m3 (to nearest even), the first in the lowest byte.  Callers scale by the group's
// largest value, so that nothing exceeds 448 but what was infinite or NaN, and that becomes NaN.
__device__ __forceinline__ uint32_t to_fp8_quad(float a, float b, float c, float d) {
    int packed = 0;
    packed = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, packed, false);
    packed = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, packed, true);
    return static_cast<uint32_t>(packed);
}

// Largest magnitudes are compared as the integers of their bits: the order of non-negative floats, with NaN
// above infinity, so that a NaN in a group is its largest value and makes its scale NaN.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

struct GroupScale {
    float scale;    // what a value is multiplied by to get what it stands for
    float inverse;  // 0 for an infinite scale: finite values become 0 there, infinite ones NaN
};

__device__ __forceinline__ GroupScale group_scale(uint32_t amax_bits) {
    const float amax = __uint_as_float(larger(amax_bits, __float_as_uint(kSmallestAmax)));
    const float scale = amax / kLargestFp8;
    return {scale, 1.0f / scale};
}

// The largest value over the 16 lanes of a row of the wavefront, in all of them.
__device__ __forceinline__ uint32_t largest_of_16(uint32_t v) {
    v = larger(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xf, 0xf, true)));   // quad_perm 1 0 3 2
    v = larger(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xf, 0xf, true)));   // quad_perm 2 3 0 1
    v = larger(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x141, 0xf, 0xf, true)));  // row_half_mirror
    return larger(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x140, 0xf, 0xf, true)));  // row_mirror
}

__device__ __forceinline__ float dpp_add(float v, int moved) { return v + __int_as_float(moved); }

// The sum over a wavefront, in all of its lanes; always in the same order.
__device__ __forceinline__ float wave_sum(float v) {
    v = dpp_add(v, __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, true));
    v = dpp_add(v, __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, true));
    v = dpp_add(v, __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, true));
    v = dpp_add(v, __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, true));
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

}  // namespace nanoep

#endif  // NANOEP_OPERATORS_H_
