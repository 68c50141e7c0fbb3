// The experts' products: rows in 8 bits, one scale for every 128 columns, times weights in 8 bits, one scale a
// 128 x 128 block, over the expert-major segments that a dispatch leaves.

#include "nanoep_operators.h"

namespace nanoep {
namespace {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kTile = 16;  // rows and columns of one matrix instruction's result

struct Product {
    const char* values;  // rows of e4m3, value_stride bytes apart
    const float* scales;  // rows of `blocks` scales, scale_stride floats apart
    const char* weight;         // [E][columns][inner] e4m3
    const float* weight_scales;  // [E][column_blocks][blocks]
    const int64_t* expert_offsets;  // [E + 1], or null: one expert, all rows
    const int64_t* expert_counts;   // [E], or null
    int64_t rows;
    int64_t value_stride;
    int64_t scale_stride;
    int experts;
    int inner;
    int columns;  // of the weights: a gated product's gate and up columns together
    int blocks;
    int column_blocks;
};

// What one workgroup computes: `live` rows from `row` on that are an expert's, then zeros up to `end`.
struct RowTile {
    int expert;  // -1: nothing
    int64_t row;
    int live;
    int size;
};

// Segment e of the rows: [begin, end), the first `live` of which are the expert's.  The last one (e == experts) is
// what follows the experts' segments.  Whatever the two arrays hold, a segment lies within the rows.
struct Segment {
    int64_t begin;
    int64_t end;
    int64_t live;
};

__device__ __forceinline__ Segment segment_of(const Product& p, int e) {
    if (p.expert_offsets == nullptr)
        return {0, e == 0 ? p.rows : 0, p.rows};
    int64_t begin = p.expert_offsets[e];
    int64_t end = e < p.experts ? p.expert_offsets[e + 1] : p.rows;
    int64_t live = e < p.experts ? p.expert_counts[e] : 0;
    begin = begin < 0 ? 0 : begin > p.rows ? p.rows : begin;
    end = end < begin ? begin : end > p.rows ? p.rows : end;
    live = live < 0 ? 0 : live > end - begin ? end - begin : live;
    return {begin, end, live};
}

// The `index`-th tile of kRows rows, counted over the segments: every wavefront finds it by a prefix sum over the
// segments' tiles, 64 at a time.
template <int kRows>
__device__ __forceinline__ RowTile find_row_tile(const Product& p, int index) {
    const int lane = threadIdx.x % kWave;
    const int segments = p.experts + (p.expert_offsets != nullptr ? 1 : 0);
    int before = 0;
    for (int first = 0; first < segments; first += kWave) {
        Segment segment = {0, 0, 0};
        if (first + lane < segments)
            segment = segment_of(p, first + lane);
        const int tiles = static_cast<int>((segment.end - segment.begin + kRows - 1) / kRows);
        int through = tiles;
#pragma unroll
        for (int step = 1; step < kWave; step *= 2) {
            const int other = __shfl_up(through, step, kWave);
            if (lane >= step)
                through += other;
        }
        const uint64_t behind = __ballot(before + through > index);
        if (behind != 0) {
            const int found = __ffsll(static_cast<long long>(behind)) - 1;
            const int64_t begin = __shfl(segment.begin, found, kWave);
            const int64_t end = __shfl(segment.end, found, kWave);
            const int64_t live = __shfl(segment.live, found, kWave);
            const int64_t skipped = static_cast<int64_t>(index - before - (__shfl(through, found, kWave) - __shfl(tiles, found, kWave))) * kRows;
            const int64_t size = end - begin - skipped, rows_live = live - skipped;
            return {first + found, begin + skipped, static_cast<int>(rows_live < 0 ? 0 : rows_live > kRows ? kRows : rows_live),
                    static_cast<int>(size > kRows ? kRows : size)};
        }
        before += __builtin_amdgcn_readlane(through, kWave - 1);
    }
    return {-1, 0, 0, 0};
}

__device__ __forceinline__ i32x8 operand(const u32x4 low, const u32x4 high) {
    return {static_cast<int>(low.x), static_cast<int>(low.y), static_cast<int>(low.z), static_cast<int>(low.w),
            static_cast<int>(high.x), static_cast<int>(high.y), static_cast<int>(high.z), static_cast<int>(high.w)};
}

// Eight e4m3 values as bf16, which holds them exactly.
__device__ __forceinline__ bf16x8 widened(int low, int high) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, 1.0f, true);
    return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// One block of 128 columns of 16 weight rows times 16 activation rows: lane l gives 32 values of weight row l % 16
// and of activation row l % 16 and gets the products of weight rows 4 * (l / 16) .. + 3 with activation row l % 16.
// Which of the block's columns a lane holds does not matter as long as both operands agree.
//
// The 8-bit matrix instruction adds its products with some 14 bits below the largest of them: on normal
// inputs the sum of a block is off by 1.5e-5 of its deviation, without a bias, however many blocks follow.  Under the bf16
// rounding of a linear product's output (1.7e-3) that does not show.  A gated product's scales are fp32 outputs, where it
// would be the largest error there is, so kExact widens the operands to bf16, whose products and sums the 16-bit
// instruction takes in fp32 (1e-7), at half the rate.
template <bool kExact>
__device__ __forceinline__ f32x4 block_product(const i32x8 weight, const i32x8 row) {
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (kExact) {
#pragma unroll
        for (int part = 0; part < 4; ++part)
            sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(weight[2 * part], weight[2 * part + 1]),
                                                          widened(row[2 * part], row[2 * part + 1]), sum, 0, 0, 0);
        return sum;
    } else {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(weight, row, sum, 0, 0, 0, 0, 0, 0);
    }
}

__device__ __forceinline__ float silu(float v) { return v / (1.0f + __expf(-v)); }

// Products of few rows with much weight: every wavefront streams its weights from memory straight into registers.
// A workgroup computes kColumns * 16 columns of kRows * 16 rows; its four wavefronts take every fourth block of 128
// inner columns, sum the blocks' products, each times its two scales, in fp32 registers, and add their sums through LDS.
// A gated product takes half of its column tiles from the gate and half from the up weights.
template <int kColumns, int kRows, bool kGated, bool kExact>
__global__ void __launch_bounds__(kBlockThreads) experts_stream_kernel(const Product p, void* __restrict__ out, int64_t out_stride) {
    __shared__ f32x4 sums[kWavesPerBlock][kColumns * kRows][kWave];
    const RowTile tile = find_row_tile<kRows * kTile>(p, static_cast<int>(blockIdx.x));
    if (tile.expert < 0)
        return;
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int group = lane / kTile, in_tile = lane % kTile;
    constexpr int kOutTiles = kGated ? kColumns / 2 : kColumns;
    const int out_columns = kGated ? p.columns / 2 : p.columns;
    const int first_column = static_cast<int>(blockIdx.y) * kOutTiles * kTile;

    f32x4 acc[kColumns][kRows];
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            acc[c][r] = {0.0f, 0.0f, 0.0f, 0.0f};

    if (tile.live > 0) {
        // rows and columns past the end are clamped to the last one: what they give is not written
        const char* weight_rows[kColumns];
        const float* weight_scales[kColumns];
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
            const int out_tile = c % kOutTiles;
            const int base = (c / kOutTiles) * out_columns;
            int column = first_column + out_tile * kTile;
            const int block_column = column < out_columns ? column : out_columns - 1;
            column += in_tile;
            column = base + (column < out_columns ? column : out_columns - 1);
            weight_rows[c] = p.weight + (static_cast<int64_t>(tile.expert) * p.columns + column) * p.inner;
            weight_scales[c] = p.weight_scales + (static_cast<int64_t>(tile.expert) * p.column_blocks + (base + block_column) / kScaleBlock) * p.blocks;
        }
        const char* value_rows[kRows];
        const float* row_scales[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int in_live = r * kTile + in_tile;
            const int64_t row = tile.row + (in_live < tile.live ? in_live : tile.live - 1);
            value_rows[r] = p.values + row * p.value_stride;
            row_scales[r] = p.scales + row * p.scale_stride;
        }
        for (int block = wave; block < p.blocks; block += kWavesPerBlock) {
            const int at = block * kScaleBlock + group * 16;
            // the last block may end early: 16 bytes past its end are zeros on both sides
            const bool low_in = at < p.inner, high_in = at + 64 < p.inner;
            const int low_at = low_in ? at : 0, high_at = high_in ? at + 64 : 0;
            const u32x4 zero = {0u, 0u, 0u, 0u};
            i32x8 rows[kRows];
            float scale[kRows];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const u32x4 low = *reinterpret_cast<const u32x4*>(value_rows[r] + low_at);
                const u32x4 high = *reinterpret_cast<const u32x4*>(value_rows[r] + high_at);
                rows[r] = operand(low_in ? low : zero, high_in ? high : zero);
                scale[r] = row_scales[r][block];
            }
#pragma unroll
            for (int c = 0; c < kColumns; ++c) {
                const u32x4 low = *reinterpret_cast<const u32x4*>(weight_rows[c] + low_at);
                const u32x4 high = *reinterpret_cast<const u32x4*>(weight_rows[c] + high_at);
                const i32x8 weight = operand(low_in ? low : zero, high_in ? high : zero);
                const float weight_scale = weight_scales[c][block];
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    const f32x4 product = block_product<kExact>(weight, rows[r]);
                    const float factor = weight_scale * scale[r];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[c][r][i] = fmaf(factor, product[i], acc[c][r][i]);
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            sums[wave][c * kRows + r][lane] = acc[c][r];
    __syncthreads();
    for (int item = wave; item < kOutTiles * kRows; item += kWavesPerBlock) {
        const int c = item / kRows, r = item % kRows;
        f32x4 total = sums[0][c * kRows + r][lane];
#pragma unroll
        for (int w = 1; w < kWavesPerBlock; ++w)
            total += sums[w][c * kRows + r][lane];
        if constexpr (kGated) {
            const int up_at = (c + kOutTiles) * kRows + r;
            f32x4 up = sums[0][up_at][lane];
#pragma unroll
            for (int w = 1; w < kWavesPerBlock; ++w)
                up += sums[w][up_at][lane];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                total[i] = silu(total[i]) * up[i];
        }
        const int in_size = r * kTile + in_tile;
        const int column = first_column + c * kTile + group * 4;
        if (in_size >= tile.size || column >= out_columns)
            continue;
        if (in_size >= tile.live)
            total = {0.0f, 0.0f, 0.0f, 0.0f};
        const int64_t at = (tile.row + in_size) * out_stride + column;
        if constexpr (kGated) {
            *reinterpret_cast<f32x4*>(static_cast<float*>(out) + at) = total;
        } else {
            uint2 packed;
            packed.x = to_bf16_pair(total[0], total[1]);
            packed.y = to_bf16_pair(total[2], total[3]);
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = packed;
        }
    }
}

// fp32 rows in 8 bits with a scale for every 128 columns: a wavefront a row, 16 lanes a group of 128 columns.
__global__ void __launch_bounds__(kBlockThreads) quantize_rows_kernel(const float* __restrict__ rows,
                                                                      char* __restrict__ records,
                                                                      int64_t num_rows,
                                                                      int64_t record_bytes,
                                                                      int columns,
                                                                      int groups) {
    const int lane = threadIdx.x % kWave;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + threadIdx.x / kWave;
    if (row >= num_rows)
        return;
    const float* from = rows + row * columns;
    char* record = records + row * record_bytes;
    float* scales = reinterpret_cast<float*>(record + columns);
    for (int base = 0; base < columns; base += kWave * 8) {
        const int at = base + lane * 8;
        f32x4 low = {0.0f, 0.0f, 0.0f, 0.0f}, high = low;
        if (at < columns) {
            low = *reinterpret_cast<const f32x4*>(from + at);
            high = *reinterpret_cast<const f32x4*>(from + at + 4);
        }
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            amax = larger(amax, larger(magnitude_bits(low[i]), magnitude_bits(high[i])));
        const GroupScale group = group_scale(largest_of_16(amax));
        if (at < columns) {
            uint2 packed;
            packed.x = to_fp8_quad(low[0] * group.inverse, low[1] * group.inverse, low[2] * group.inverse, low[3] * group.inverse);
            packed.y = to_fp8_quad(high[0] * group.inverse, high[1] * group.inverse, high[2] * group.inverse, high[3] * group.inverse);
            *reinterpret_cast<uint2*>(record + at) = packed;
            if (lane % 16 == 0)
                scales[at / kScaleBlock] = group.scale;
        }
    }
    for (int word = columns / 4 + groups + lane; word < static_cast<int>(record_bytes / 4); word += kWave)
        reinterpret_cast<uint32_t*>(record)[word] = 0u;
}

int product_of(const void* values, int64_t value_stride, const float* scales, int64_t scale_stride, const void* weight,
               const float* weight_scales, const int64_t* expert_offsets, const int64_t* expert_counts, int64_t rows, int64_t experts,
               int inner, int columns, int column_multiple, Product& p) {
    if (rows < 0 || rows > 0x7fffffff || experts <= 0 || experts >= (int64_t{1} << 30) || inner <= 0 || inner % 16 != 0 || columns <= 0 ||
        columns % column_multiple != 0 || (expert_offsets == nullptr) != (expert_counts == nullptr))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (expert_offsets == nullptr && experts != 1)
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (rows == 0)
        return NANOEP_OK;
    if (values == nullptr || scales == nullptr || weight == nullptr || weight_scales == nullptr || !aligned16(values) || !aligned16(weight) ||
        value_stride < inner || value_stride % 16 != 0 || scale_stride < scale_groups(inner))
        return NANOEP_ERR_INVALID_ARGUMENT;
    p = {static_cast<const char*>(values), scales, static_cast<const char*>(weight), weight_scales, expert_offsets, expert_counts,
         rows, value_stride, scale_stride, static_cast<int>(experts), inner, columns,
         static_cast<int>(scale_groups(inner)), static_cast<int>(scale_groups(columns))};
    return NANOEP_OK;
}

// Most tiles of kRows rows that the segments can have: each but the full ones ends in one that is not.
int64_t most_row_tiles(const Product& p, int rows) {
    const int64_t segments = p.expert_offsets != nullptr ? p.experts + int64_t{1} : 1;
    return p.rows / rows + (segments < p.rows ? segments : p.rows);
}

template <int kColumns, int kRows, bool kGated, bool kExact>
int launch_stream(const Product& p, void* out, int64_t out_stride, hipStream_t stream) {
    const int out_columns = kGated ? p.columns / 2 : p.columns;
    constexpr int kOutColumns = (kGated ? kColumns / 2 : kColumns) * kTile;
    const int64_t tiles = most_row_tiles(p, kRows * kTile), column_tiles = (out_columns + kOutColumns - 1) / kOutColumns;
    if (tiles > 0x7fffffff || column_tiles > 65535)
        return NANOEP_ERR_INVALID_ARGUMENT;
    experts_stream_kernel<kColumns, kRows, kGated, kExact>
        <<<dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(column_tiles)), kBlockThreads, 0, stream>>>(p, out, out_stride);
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

template <bool kGated, bool kExact>
int launch_product(const Product& p, void* out, int64_t out_stride, hipStream_t stream) {
    const int64_t rows_each = p.rows / p.experts;
    if (rows_each <= 16)
        return launch_stream<2, 1, kGated, kExact>(p, out, out_stride, stream);
    if (rows_each <= 32)
        return launch_stream<2, 2, kGated, kExact>(p, out, out_stride, stream);
    return launch_stream<4, 4, kGated, kExact>(p, out, out_stride, stream);
}

}  // namespace
}  // namespace nanoep

extern "C" {

int nanoep_experts_linear(const void* values, int64_t value_stride, const float* scales, int64_t scale_stride, const void* weight,
                          const float* weight_scales, const int64_t* expert_offsets, const int64_t* expert_counts, int64_t rows,
                          int64_t experts, int inner, int columns, void* out, void* stream) {
    using namespace nanoep;
    Product p{};
    const int status = product_of(values, value_stride, scales, scale_stride, weight, weight_scales, expert_offsets, expert_counts, rows,
                                  experts, inner, columns, 8, p);
    if (status != NANOEP_OK || rows == 0)
        return status;
    if (out == nullptr || !aligned16(out))
        return NANOEP_ERR_INVALID_ARGUMENT;
    // up to 64 inner columns the 16-bit instructions take no longer than the one 128-wide 8-bit one
    if (inner <= kScaleBlock / 2)
        return launch_product<false, true>(p, out, columns, static_cast<hipStream_t>(stream));
    return launch_product<false, false>(p, out, columns, static_cast<hipStream_t>(stream));
}

size_t nanoep_experts_gated_workspace_bytes(int64_t rows, int64_t experts, int inner, int columns) {
    if (rows <= 0 || experts <= 0 || inner <= 0 || columns <= 0)
        return 0;
    return static_cast<size_t>(rows) * static_cast<size_t>(columns / 2) * sizeof(float);
}

int nanoep_experts_gated(const void* values, int64_t value_stride, const float* scales, int64_t scale_stride, const void* weight,
                         const float* weight_scales, const int64_t* expert_offsets, const int64_t* expert_counts, int64_t rows,
                         int64_t experts, int inner, int columns, void* records, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace nanoep;
    Product p{};
    const int status = product_of(values, value_stride, scales, scale_stride, weight, weight_scales, expert_offsets, expert_counts, rows,
                                  experts, inner, columns, 32, p);
    if (status != NANOEP_OK || rows == 0)
        return status;
    if (records == nullptr || !aligned16(records))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const size_t needed = nanoep_experts_gated_workspace_bytes(rows, experts, inner, columns);
    if (workspace_bytes < needed)
        return NANOEP_ERR_WORKSPACE;
    if (needed > 0 && (workspace == nullptr || !aligned16(workspace)))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const auto on = static_cast<hipStream_t>(stream);
    const int launched = launch_product<true, true>(p, workspace, columns / 2, on);
    if (launched != NANOEP_OK)
        return launched;
    const unsigned blocks = static_cast<unsigned>((rows + kWavesPerBlock - 1) / kWavesPerBlock);
    quantize_rows_kernel<<<blocks, kBlockThreads, 0, on>>>(static_cast<const float*>(workspace), static_cast<char*>(records), rows,
                                                           record_bytes_of(columns / 2), columns / 2, static_cast<int>(scale_groups(columns / 2)));
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

}  // extern "C"
