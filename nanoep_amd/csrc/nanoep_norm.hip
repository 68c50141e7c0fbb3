// Residual addition and root-mean-square norm of bf16 rows, in 8 bits with a scale for every 128 columns.

#include "nanoep_operators.h"

namespace nanoep {
namespace {

constexpr int kMostNormThreads = 1024;
constexpr int kMostNormVectors = 8;  // 16-byte vectors of a row that a lane holds

// One workgroup a row: s = x + residual, r = 1 / sqrt(mean(s^2) + eps), n = s * r * gamma; then, for every 128
// columns, scale = max |n| / 448 and the values n / scale, rounded to e4m3.  The row stays in registers
// between its sum of squares and its output (kVectors 16-byte vectors a lane, 8 columns each), so that every
// input byte is read once, all of them ahead of anything else; s and n are fp32 throughout, and each output is rounded
// from them once.  16 neighbouring lanes hold the 128 columns of a scale.  HBM-bound: 4096 x 7168 with both bf16 outputs
// (265 MB) 40 to 42 us, 6.5 TB/s, 45.1 a call among others; one token 2.7.  Side by side, back to back: 48.3 us (with plain stores and
// gamma read behind the sum 54.0), 8192 x 2048 24.7; nontemporal loads of the inputs take 44.9 and 27.2 there, but would pass
// over inputs that the last kernel left in the caches.
template <int kVectors>
__global__ void __launch_bounds__(kMostNormThreads) rms_norm_fp8_kernel(const u32x4* __restrict__ x,         // [T][vectors]
                                                                       const u32x4* __restrict__ residual,  // [T][vectors] or null
                                                                       const u32x4* __restrict__ gamma,     // [vectors]
                                                                       char* __restrict__ records,
                                                                       u32x4* __restrict__ residual_out,  // [T][vectors] or null
                                                                       u32x4* __restrict__ normalized,    // [T][vectors] or null
                                                                       int64_t rows,
                                                                       int vectors,
                                                                       int groups,
                                                                       int64_t record_bytes,
                                                                       float columns,
                                                                       float eps) {
    __shared__ float wave_sums[kMostNormThreads / kWave];
    const int64_t row = workgroup_number();
    if (row >= rows)
        return;
    const int threads = blockDim.x;
    const u32x4* row_x = x + row * vectors;
    const u32x4* row_residual = residual + row * vectors;

    float s[kVectors][8];
    float squares = 0.0f;
    u32x4 others[kVectors];
    if (residual != nullptr) {
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const int at = threadIdx.x + v * threads;
            others[v] = at < vectors ? row_residual[at] : u32x4{0u, 0u, 0u, 0u};
        }
    }
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = threadIdx.x + v * threads;
        u32x4 data = {0u, 0u, 0u, 0u};
        if (at < vectors)
            data = row_x[at];
        unpack_bf16(data, s[v]);
    }
    if (residual != nullptr) {
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const int at = threadIdx.x + v * threads;
            float other[8];
            unpack_bf16(others[v], other);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                s[v][i] += other[i];
            if (at < vectors)
                store_vec<true>(residual_out + row * vectors + at, pack_bf16(s[v]));
        }
    }
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            squares = fmaf(s[v][i], s[v][i], squares);
    u32x4 gammas[kVectors];
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = threadIdx.x + v * threads;
        gammas[v] = at < vectors ? gamma[at] : u32x4{0u, 0u, 0u, 0u};
    }
    squares = wave_sum(squares);
    if (threadIdx.x % kWave == 0)
        wave_sums[threadIdx.x / kWave] = squares;
    __syncthreads();
    float total = 0.0f;
    for (int w = 0; w < threads / kWave; ++w)
        total += wave_sums[w];
    const float factor = 1.0f / sqrtf(total / columns + eps);

    char* record = records + row * record_bytes;
    float* scales = reinterpret_cast<float*>(record + static_cast<int64_t>(vectors) * 8);
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = threadIdx.x + v * threads;
        float weight[8];
        unpack_bf16(gammas[v], weight);
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // lanes past the row's end hold zeros, which must stay zeros where the row's factor is infinite or NaN
            s[v][i] = at < vectors ? s[v][i] * factor * weight[i] : 0.0f;
            amax = larger(amax, magnitude_bits(s[v][i]));
        }
        if (normalized != nullptr && at < vectors)
            store_vec<true>(normalized + row * vectors + at, pack_bf16(s[v]));
        const GroupScale group = group_scale(largest_of_16(amax));
        if (at < vectors) {
            uint2 packed;
            packed.x = to_fp8_quad(s[v][0] * group.inverse, s[v][1] * group.inverse, s[v][2] * group.inverse, s[v][3] * group.inverse);
            packed.y = to_fp8_quad(s[v][4] * group.inverse, s[v][5] * group.inverse, s[v][6] * group.inverse, s[v][7] * group.inverse);
            reinterpret_cast<uint2*>(record)[at] = packed;
            if (at % 16 == 0)
                scales[at / 16] = group.scale;
        }
    }
    // the record's padding, so that all of it is defined
    const int used = vectors * 2 + groups;
    for (int word = used + threadIdx.x; word < static_cast<int>(record_bytes / 4); word += threads)
        reinterpret_cast<uint32_t*>(record)[word] = 0u;
}

}  // namespace
}  // namespace nanoep

extern "C" {

int64_t nanoep_fp8_record_bytes(int64_t columns) { return columns > 0 ? nanoep::record_bytes_of(columns) : 0; }

int nanoep_rms_norm_fp8(const void* x, const void* residual, const void* gamma, int64_t num_tokens, int hidden, float eps, void* records,
                        void* residual_out, void* normalized, void* stream) {
    using namespace nanoep;
    if (num_tokens < 0 || num_tokens > 0x7fffffff || hidden <= 0 || hidden % 16 != 0 || hidden > 8 * kMostNormThreads * kMostNormVectors)
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (!(eps >= 0.0f) || (residual == nullptr) != (residual_out == nullptr))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens == 0)
        return NANOEP_OK;
    if (x == nullptr || gamma == nullptr || records == nullptr || !aligned16(x) || !aligned16(residual) || !aligned16(gamma) ||
        !aligned16(records) || !aligned16(residual_out) || !aligned16(normalized))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const int vectors = hidden / 8;
    // one vector a lane up to 1024 lanes while there are few rows; two when the rows alone fill the device (4096 x 7168: one 47.6
    // us, two 48.3, four 49.2; 8192 x 2048: 26.7, 24.7, 27.0)
    const int wanted = num_tokens >= 1024 ? 2 : 1;
    int held = 1;
    while (held < kMostNormVectors && (vectors + held - 1) / held > (held < wanted ? kWave : kMostNormThreads))
        held *= 2;
    const int threads = static_cast<int>(align_up(static_cast<size_t>((vectors + held - 1) / held), kWave));
    const dim3 grid = grid_of(num_tokens);
#define NANOEP_LAUNCH_NORM(HELD)                                                                                                        \
    rms_norm_fp8_kernel<HELD><<<grid, threads, 0, static_cast<hipStream_t>(stream)>>>(                                                  \
        static_cast<const u32x4*>(x), static_cast<const u32x4*>(residual), static_cast<const u32x4*>(gamma), static_cast<char*>(records), \
        static_cast<u32x4*>(residual_out), static_cast<u32x4*>(normalized), num_tokens, vectors, static_cast<int>(scale_groups(hidden)), \
        record_bytes_of(hidden), static_cast<float>(hidden), eps)
    if (held == 1)
        NANOEP_LAUNCH_NORM(1);
    else if (held == 2)
        NANOEP_LAUNCH_NORM(2);
    else if (held == 4)
        NANOEP_LAUNCH_NORM(4);
    else
        NANOEP_LAUNCH_NORM(8);
#undef NANOEP_LAUNCH_NORM
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

}  // extern "C"
