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
constexpr int kUnitRows = 4, kUnitCols = 8;  // neighbouring tiles that one XCD works on at a time

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
            // (row numbers fit 31 bits)
            const int begin = __builtin_amdgcn_readlane(static_cast<int>(segment.begin), found);
            const int end = __builtin_amdgcn_readlane(static_cast<int>(segment.end), found);
            const int live = __builtin_amdgcn_readlane(static_cast<int>(segment.live), found);
            const int skipped = (index - before - __builtin_amdgcn_readlane(through - tiles, found)) * kRows;
            const int size = end - begin - skipped, rows_live = live - skipped;
            return {first + found, begin + skipped, rows_live < 0 ? 0 : rows_live > kRows ? kRows : rows_live, size > kRows ? kRows : size};
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

// ------------------------------------------------------------------ many rows an expert

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)(p)));
}

// Copies 16 (kBytes == 16) or 4 bytes a lane from memory into LDS without registers on the way: lane l's go to
// `to` + l * kBytes.  `to` and `from` are wave-uniform, `offset` is a lane's own.  Nothing waits for it but loads_landed().
template <int kBytes>
__device__ __forceinline__ void load_to_lds(const char* from, uint32_t offset, uint32_t to) {
    if constexpr (kBytes == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(from) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(offset), "s"(from) : "memory");
}

// The same with a whole address of each lane's own.
__device__ __forceinline__ void load_to_lds(const char* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}

// What is read in the place of a piece that lies past its row's end.
__device__ const u32x4 kZeroPiece = {0u, 0u, 0u, 0u};

// Every wavefront's copies into LDS are there, and every wavefront has read what the next ones overwrite.
__device__ __forceinline__ void loads_landed() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The products of a tile of 16 * kRowTiles * kRowWaves rows and 16 * kColTiles * kColWaves weight rows, one workgroup.
template <int kRowTiles, int kColTiles, int kRowWaves, int kColWaves>
struct TileShape {
    static constexpr int kWaves = kRowWaves * kColWaves;
    static constexpr int kThreads = kWaves * kWave;
    static constexpr int kRows = kTile * kRowTiles * kRowWaves;
    static constexpr int kCols = kTile * kColTiles * kColWaves;
    static constexpr int kStageRows = kRows + kCols;  // 128-byte rows of one stage: the weights', then the activations'
    static constexpr int kLoads = kStageRows / 8 / kWaves;
    static_assert(kCols % (8 * kWaves) == 0 && kRows % (8 * kWaves) == 0 && kRows % kWave == 0 && kRows / kWave <= kWaves);
};

template <int kRowTiles, int kColTiles, int kRowWaves, int kColWaves, bool kGated>
__global__ void __launch_bounds__(kRowWaves * kColWaves * kWave)
    experts_tile_kernel(const Product p, char* __restrict__ out, int64_t out_stride, int column_tiles, int column_groups, XcdMap xcd) {
    using Shape = TileShape<kRowTiles, kColTiles, kRowWaves, kColWaves>;
    constexpr int kStageBytes = Shape::kStageRows * kScaleBlock;
    __shared__ __attribute__((aligned(1024))) char stages[2][kStageBytes];
    __shared__ float row_scales[2][Shape::kRows];
    __shared__ uint32_t group_amax[kGated ? Shape::kRows : 1][kColWaves];

    // units of kUnitRows x kUnitCols neighbouring tiles, which share their rows and weights in one XCD's L2, go round the XCDs
    const uint32_t turn = fast_divide(blockIdx.x, xcd.magic, xcd.shift);
    const uint32_t on_xcd = blockIdx.x - turn * xcd.count;
    const uint32_t unit = turn / (kUnitRows * kUnitCols) * xcd.count + on_xcd;
    const uint32_t in_unit = turn % (kUnitRows * kUnitCols);
    const int row_group = static_cast<int>(unit / column_groups), column_group = static_cast<int>(unit % column_groups);
    const int column_tile = column_group * kUnitCols + static_cast<int>(in_unit / kUnitRows);
    if (column_tile >= column_tiles)
        return;
    const RowTile tile = find_row_tile<Shape::kRows>(p, row_group * kUnitRows + static_cast<int>(in_unit % kUnitRows));
    if (tile.expert < 0)
        return;

    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col_wave = wave % kColWaves, row_wave = wave / kColWaves;
    const int group = lane / kTile, in_tile = lane % kTile;
    constexpr int kOutTiles = kGated ? kColTiles / 2 : kColTiles;  // column tiles of the output a wavefront makes
    constexpr int kOutCols = kGated ? Shape::kCols / 2 : Shape::kCols;
    const int out_columns = kGated ? p.columns / 2 : p.columns;
    const int first_column = column_tile * kOutCols;

    f32x4 acc[kColTiles][kRowTiles];
#pragma unroll
    for (int c = 0; c < kColTiles; ++c)
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r)
            acc[c][r] = {0.0f, 0.0f, 0.0f, 0.0f};

    if (tile.live > 0) {
        // This lane's part of a stage: load i brings in row 8 * (i * kWaves + wave) + lane / 8 of it, eight lanes a row.  Within its
        // row the 16-byte piece that the lane fetches, and so where that piece lies in LDS, is turned by the row, so
        // that eight rows' same piece, which a matrix operand reads at once, lie in different banks.
        const int piece = (lane % 8) ^ (lane / 8);
        const char* weight = p.weight + static_cast<int64_t>(tile.expert) * p.columns * p.inner;
        const char* values = p.values + tile.row * p.value_stride;
        constexpr int kWeightLoads = Shape::kCols / (8 * Shape::kWaves);
        uint32_t row_offset[Shape::kLoads];
#pragma unroll
        for (int i = 0; i < Shape::kLoads; ++i) {
            const int first = 8 * (i * Shape::kWaves + wave);
            const int row = first + lane / 8;
            if (i < kWeightLoads) {
                int column;
                if constexpr (kGated) {
                    const int in_wave = row % (kTile * kColTiles), half = in_wave / (kTile * kOutTiles);
                    column = first_column + row / (kTile * kColTiles) * (kTile * kOutTiles) + in_wave % (kTile * kOutTiles);
                    column = (column < out_columns ? column : out_columns - 1) + half * out_columns;
                } else {
                    column = first_column + row;
                    column = column < out_columns ? column : out_columns - 1;
                }
                row_offset[i] = static_cast<uint32_t>(column) * static_cast<uint32_t>(p.inner);
            } else {
                const int in_rows = row - Shape::kCols;
                row_offset[i] = static_cast<uint32_t>(in_rows < tile.live ? in_rows : tile.live - 1) * static_cast<uint32_t>(p.value_stride);
            }
        }
        const int scale_row = wave * kWave + lane < tile.live ? wave * kWave + lane : tile.live - 1;
        const uint32_t scale_offset = static_cast<uint32_t>(scale_row) * static_cast<uint32_t>(p.scale_stride) * 4u;
        const char* scales = reinterpret_cast<const char*>(p.scales + tile.row * p.scale_stride);
        const uint32_t stages_at = lds_address(stages), scales_at = lds_address(row_scales);

        const auto fetch = [&](int block) {
            const int64_t at = static_cast<int64_t>(block) * kScaleBlock;
            const bool whole = at + kScaleBlock <= p.inner, in_row = at + piece * 16 < p.inner;
            const uint32_t to = stages_at + (block & 1) * kStageBytes + static_cast<uint32_t>(wave) * 8 * kScaleBlock;
            constexpr uint32_t kStep = Shape::kWaves * 8 * kScaleBlock;
            if (whole) {
#pragma unroll
                for (int i = 0; i < Shape::kLoads; ++i)
                    load_to_lds<16>((i < kWeightLoads ? weight : values) + at, row_offset[i] + piece * 16, to + i * kStep);
            } else {
#pragma unroll
                for (int i = 0; i < Shape::kLoads; ++i)
                    load_to_lds(in_row ? (i < kWeightLoads ? weight : values) + at + row_offset[i] + piece * 16 : reinterpret_cast<const char*>(&kZeroPiece),
                                to + i * kStep);
            }
            if (wave < Shape::kRows / kWave)
                load_to_lds<4>(scales + static_cast<int64_t>(block) * 4, scale_offset, scales_at + ((block & 1) * Shape::kRows + static_cast<uint32_t>(wave * kWave)) * 4u);
        };

        // the scales' blocks of this wavefront's column tiles: one block where they are neighbours within 128 columns
        constexpr int kScales = kGated ? kColTiles : 1;
        static_assert(kGated || kScaleBlock % (kColTiles * kTile) == 0);
        const float* weight_scales[kScales];
#pragma unroll
        for (int c = 0; c < kScales; ++c) {
            int column = first_column + (col_wave * kOutTiles + c % kOutTiles) * kTile;
            column = (column < out_columns ? column : out_columns - 1) + (c / kOutTiles) * out_columns;
            weight_scales[c] = p.weight_scales + (static_cast<int64_t>(tile.expert) * p.column_blocks + column / kScaleBlock) * p.blocks;
        }

        fetch(0);
        float next_scale[kScales];
#pragma unroll
        for (int c = 0; c < kScales; ++c)
            next_scale[c] = uniform_load(weight_scales[c]);
        for (int block = 0; block < p.blocks; ++block) {
            loads_landed();
            if (block + 1 < p.blocks)
                fetch(block + 1);
            const char* stage = stages[block & 1];
            const int turned = (group ^ (lane & 7)) * 16;
            const char* weight_at = stage + (col_wave * kColTiles * kTile + in_tile) * kScaleBlock;
            const char* value_at = stage + (Shape::kCols + row_wave * kRowTiles * kTile + in_tile) * kScaleBlock;
            float column_scale[kScales];
#pragma unroll
            for (int c = 0; c < kScales; ++c)
                column_scale[c] = next_scale[c];
            const int next_block = block + 1 < p.blocks ? block + 1 : block;
#pragma unroll
            for (int c = 0; c < kScales; ++c)
                next_scale[c] = uniform_load(weight_scales[c] + next_block);
            i32x8 weights[kColTiles];
#pragma unroll
            for (int c = 0; c < kColTiles; ++c)
                weights[c] = operand(*reinterpret_cast<const u32x4*>(weight_at + c * kTile * kScaleBlock + turned),
                                     *reinterpret_cast<const u32x4*>(weight_at + c * kTile * kScaleBlock + (turned ^ 64)));
            const auto row_operand = [&](int r) {
                return operand(*reinterpret_cast<const u32x4*>(value_at + r * kTile * kScaleBlock + turned),
                               *reinterpret_cast<const u32x4*>(value_at + r * kTile * kScaleBlock + (turned ^ 64)));
            };
            const float* scale_at = &row_scales[block & 1][row_wave * kRowTiles * kTile + in_tile];
            i32x8 rows[2];
            rows[0] = row_operand(0);
            float scale[2] = {scale_at[0], 0.0f};
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) {
                // a step's operand is read during the step ahead of it, and not earlier: there are no registers for more
                __builtin_amdgcn_sched_barrier(0);
                if (r + 1 < kRowTiles) {
                    rows[(r + 1) & 1] = row_operand(r + 1);
                    scale[(r + 1) & 1] = scale_at[(r + 1) * kTile];
                }
                f32x4 product[kColTiles];
#pragma unroll
                for (int c = 0; c < kColTiles; ++c)
                    product[c] = block_product<kGated>(weights[c], rows[r & 1]);
#pragma unroll
                for (int c = 0; c < kColTiles; ++c) {
                    const float factor = column_scale[c % kScales] * scale[r & 1];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[c][r][i] = fmaf(factor, product[c][i], acc[c][r][i]);
                }
            }
        }
    }

    const int first_row = row_wave * kRowTiles * kTile + in_tile;
    if constexpr (!kGated) {
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) {
            const int in_rows = first_row + r * kTile;
            if (in_rows >= tile.size)
                continue;
            uint16_t* row = reinterpret_cast<uint16_t*>(out) + (tile.row + in_rows) * out_stride;
#pragma unroll
            for (int c = 0; c < kColTiles; ++c) {
                const int column = first_column + (col_wave * kColTiles + c) * kTile + group * 4;
                if (column >= out_columns)
                    continue;
                const f32x4 v = in_rows < tile.live ? acc[c][r] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                uint2 packed;
                packed.x = to_bf16_pair(v[0], v[1]);
                packed.y = to_bf16_pair(v[2], v[3]);
                *reinterpret_cast<uint2*>(row + column) = packed;
            }
        }
    } else {
        // the tile's output columns are one group of 128: its largest value is found over the wavefronts through LDS
        static_assert(!kGated || kOutCols == kScaleBlock);
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) {
            uint32_t amax = 0;
            const bool live = first_row + r * kTile < tile.live;
#pragma unroll
            for (int c = 0; c < kOutTiles; ++c) {
                const int column = first_column + (col_wave * kOutTiles + c) * kTile + group * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float act = live && column < out_columns ? silu(acc[c][r][i]) * acc[c + kOutTiles][r][i] : 0.0f;
                    acc[c][r][i] = act;
                    amax = larger(amax, magnitude_bits(act));
                }
            }
            amax = larger(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 16, kWave)));
            amax = larger(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 32, kWave)));
            if (group == 0)
                group_amax[first_row + r * kTile][col_wave] = amax;
        }
        __syncthreads();
        const int groups = (out_columns + kScaleBlock - 1) / kScaleBlock;
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) {
            const int in_rows = first_row + r * kTile;
            uint32_t amax = group_amax[in_rows][0];
#pragma unroll
            for (int w = 1; w < kColWaves; ++w)
                amax = larger(amax, group_amax[in_rows][w]);
            const GroupScale scale = group_scale(amax);
            if (in_rows >= tile.size)
                continue;
            char* record = out + (tile.row + in_rows) * out_stride;
#pragma unroll
            for (int c = 0; c < kOutTiles; ++c) {
                const int column = first_column + (col_wave * kOutTiles + c) * kTile + group * 4;
                if (column < out_columns)
                    *reinterpret_cast<uint32_t*>(record + column) = to_fp8_quad(acc[c][r][0] * scale.inverse, acc[c][r][1] * scale.inverse,
                                                                               acc[c][r][2] * scale.inverse, acc[c][r][3] * scale.inverse);
            }
            if (col_wave == 0 && group == 0)
                reinterpret_cast<float*>(record + out_columns)[column_tile] = scale.scale;
            // the record's padding goes with its last group
            if (column_tile == column_tiles - 1 && col_wave == kColWaves - 1)
                for (int word = out_columns / 4 + groups + group; word < static_cast<int>(out_stride / 4); word += 4)
                    reinterpret_cast<uint32_t*>(record)[word] = 0u;
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

template <int kRowTiles, int kColTiles, int kRowWaves, int kColWaves, bool kGated>
int launch_tiles(const Product& p, void* out, int64_t out_stride, hipStream_t stream) {
    using Shape = TileShape<kRowTiles, kColTiles, kRowWaves, kColWaves>;
    constexpr int kOutCols = kGated ? Shape::kCols / 2 : Shape::kCols;
    const int out_columns = kGated ? p.columns / 2 : p.columns;
    const XcdMap xcd = make_xcd_map(current_topology(current_tuning()).xcds);
    const int column_tiles = (out_columns + kOutCols - 1) / kOutCols;
    const int column_groups = (column_tiles + kUnitCols - 1) / kUnitCols;
    const int64_t row_groups = (most_row_tiles(p, Shape::kRows) + kUnitRows - 1) / kUnitRows;
    const int64_t units = (row_groups * column_groups + xcd.count - 1) / xcd.count * xcd.count;
    if (units * kUnitRows * kUnitCols > 0x7fffffff)
        return NANOEP_ERR_INVALID_ARGUMENT;
    experts_tile_kernel<kRowTiles, kColTiles, kRowWaves, kColWaves, kGated>
        <<<dim3(static_cast<unsigned>(units * kUnitRows * kUnitCols)), Shape::kThreads, 0, stream>>>(p, static_cast<char*>(out), out_stride,
                                                                                                    column_tiles, column_groups, xcd);
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

// Whether the tile kernel takes a product: enough rows an expert, and an expert's weight and a tile's rows within the 32-bit
// offsets it addresses them with.
bool takes_tiles(int64_t rows, int64_t experts, int inner, int columns, int64_t value_stride, int64_t scale_stride) {
    constexpr int64_t kMost = int64_t{1} << 32;
    return rows / experts > 64 && static_cast<int64_t>(columns) * inner <= kMost && value_stride <= kMost / 256 && scale_stride <= kMost / 1024;
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
    if (inner > kScaleBlock / 2 && takes_tiles(rows, experts, inner, columns, value_stride, scale_stride))
        return launch_tiles<8, 4, 2, 4, false>(p, out, columns, static_cast<hipStream_t>(stream));
    if (inner <= kScaleBlock / 2)
        return launch_product<false, true>(p, out, columns, static_cast<hipStream_t>(stream));
    return launch_product<false, false>(p, out, columns, static_cast<hipStream_t>(stream));
}

size_t nanoep_experts_gated_workspace_bytes(int64_t rows, int64_t experts, int inner, int columns, int64_t value_stride,
                                            int64_t scale_stride) {
    if (rows <= 0 || experts <= 0 || inner <= 0 || columns <= 0 ||
        nanoep::takes_tiles(rows, experts, inner, columns, value_stride, scale_stride))
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
    const size_t needed = nanoep_experts_gated_workspace_bytes(rows, experts, inner, columns, value_stride, scale_stride);
    if (workspace_bytes < needed)
        return NANOEP_ERR_WORKSPACE;
    if (needed > 0 && (workspace == nullptr || !aligned16(workspace)))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const auto on = static_cast<hipStream_t>(stream);
    if (takes_tiles(rows, experts, inner, columns, value_stride, scale_stride))
        return launch_tiles<8, 4, 2, 4, true>(p, records, record_bytes_of(columns / 2), on);
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
