// The experts' products: rows in 8 bits, one scale for every 128 columns, times weights in 8 bits, one scale a
// 128 x 128 block, over the expert-major segments that a dispatch leaves.

#include <algorithm>

#include "nanoep_operators.h"

namespace nanoep {
namespace {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kTile = 16;  // rows and columns of one matrix instruction's result
constexpr int kUnitRows = 4, kUnitCols = 8;  // neighbouring tiles that an XCD works on together

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

// What one workgroup computes: `live` rows from `row` on that are an expert's.
struct RowTile {
    int expert;  // -1: nothing
    int64_t row;
    int live;
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

// The `index`-th tile of kRows rows, counted over the experts' rows: every wavefront finds it by a prefix sum over the
// experts' tiles, 64 at a time.
template <int kRows>
__device__ __forceinline__ RowTile find_row_tile(const Product& p, int index) {
    const int lane = threadIdx.x % kWave;
    int before = 0;
    for (int first = 0; first < p.experts; first += kWave) {
        Segment segment = {0, 0, 0};
        if (first + lane < p.experts)
            segment = segment_of(p, first + lane);
        const int tiles = static_cast<int>((segment.live + kRows - 1) / kRows);
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
            const int live = __builtin_amdgcn_readlane(static_cast<int>(segment.live), found);
            const int skipped = (index - before - __builtin_amdgcn_readlane(through - tiles, found)) * kRows;
            const int left = live - skipped;
            return {first + found, begin + skipped, left > kRows ? kRows : left};
        }
        before += __builtin_amdgcn_readlane(through, kWave - 1);
    }
    return {-1, 0, 0};
}

// The rows of no expert, behind every expert's and behind the last segment, in kGapParts parts each: `part` of all
// (experts + 1) * kGapParts, as rows [begin, end).
constexpr int kGapParts = 8;
struct RowRange {
    int64_t begin;
    int64_t end;
};
__device__ __forceinline__ RowRange gap_part(const Product& p, int64_t part) {
    const Segment segment = segment_of(p, static_cast<int>(part / kGapParts));
    const int64_t begin = segment.begin + segment.live, rows = segment.end - begin;
    return {begin + rows * (part % kGapParts) / kGapParts, begin + rows * (part % kGapParts + 1) / kGapParts};
}

// What a product's output holds in the rows [begin, end) of no expert: zeros, and in records the scale of a group of zeros.
template <bool kRecords, int kThreads, int kValueBytes = 2>
__device__ __forceinline__ void clear_rows(char* out, int64_t stride, int columns, RowRange rows) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    const int groups = (columns + kScaleBlock - 1) / kScaleBlock;
    const float scale = group_scale(0).scale;
    for (int64_t row = rows.begin; row < rows.end; ++row) {
        char* at = out + row * stride;
        if constexpr (kRecords) {
            // (a record is a multiple of 512 bytes; its scales are words of it)
            for (int word = threadIdx.x; word < static_cast<int>(stride / 4); word += kThreads)
                reinterpret_cast<uint32_t*>(at)[word] = word >= columns / 4 && word < columns / 4 + groups ? __float_as_uint(scale) : 0u;
        } else {
            for (int vector = threadIdx.x; vector < columns / (16 / kValueBytes); vector += kThreads)
                reinterpret_cast<u32x4*>(at)[vector] = zero;
        }
    }
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
// The operands are widened to bf16, whose products and sums the 16-bit instruction takes in fp32 (off by 1e-7 of a block's
// deviation).  The 8-bit instruction has twice the rate, but adds its products with some 14 bits below the largest of them:
// 1.5e-5 on normal inputs, and where large products cancel, small ones beside them are lost.
__device__ __forceinline__ f32x4 block_product(const i32x8 weight, const i32x8 row) {
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int part = 0; part < 4; ++part)
        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(weight[2 * part], weight[2 * part + 1]),
                                                      widened(row[2 * part], row[2 * part + 1]), sum, 0, 0, 0);
    return sum;
}

__device__ __forceinline__ float silu(float v) { return v / (1.0f + __expf(-v)); }

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)(p)));
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// Copies 16 (kBytes == 16) or 4 bytes a lane from memory into LDS without registers on the way: lane l's go to
// `to` + l * kBytes.  `to` and `from` are wave-uniform, `offset` is a lane's own.  Waits are the caller's, by counting.
// m0 is named as overwritten, so that the compiler takes nothing it has put there to be there still; that it warns of a
// register of its own on that list is switched off.
template <int kBytes>
__device__ __forceinline__ void load_to_lds(const char* from, uint32_t offset, uint32_t to) {
    if constexpr (kBytes == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(from) : "m0", "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(offset), "s"(from) : "m0", "memory");
}

// The same with a whole address of each lane's own.
template <int kBytes>
__device__ __forceinline__ void load_to_lds(const char* from, uint32_t to) {
    if constexpr (kBytes == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "m0", "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "m0", "memory");
}

#pragma clang diagnostic pop

// What is read in the place of a piece that lies past its row's end.
__device__ const u32x4 kZeroPiece = {0u, 0u, 0u, 0u};

// The odd groups of 16 lanes of `a` and the even ones of `b` change places.
__device__ __forceinline__ u32x2 swapped(uint32_t a, uint32_t b) {
    const auto both = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    return {both[0], both[1]};
}

// Waits until all but the newest kNewer of this wavefront's loads are done, and its reads of LDS.
template <int kNewer>
__device__ __forceinline__ void loaded_but_newest() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kNewer) : "memory");
}

// ------------------------------------------------------------------ few rows an expert

// Products of few rows with much weight: what counts is that HBM is kept busy.  A workgroup computes kColumns * 16 columns of
// kRows * 16 rows; its four wavefronts take every fourth block of 128 inner columns, sum the blocks' products, each
// times its two scales, in fp32 registers, and add their sums through LDS.  Each wavefront has a ring of kDepth blocks' operands in
// LDS of its own, filled straight from memory, whole 128-byte lines at a time, and needs no barrier to read it: kDepth - 1
// blocks are on their way.  A gated product takes half of its column tiles from the gate and half from the up weights,
// and leaves fp32 rows to quantize_rows_kernel, since no workgroup has the 128 columns of a scale.
//
// Measured: one token's eight experts, gated, 7168 -> 2 x 2048 (223 MB of weights): 40 to 47 us, 5.0 TB/s, and 4 for the
// scales' launch.  What is left is the workgroups' start and their sums.  Two blocks' operands in registers, loaded there in
// their layout, took the same time; eight wavefronts that have a whole group's columns and need no second launch 53 us
// against 50 for both, and up to 2.8 times as long at smaller sizes.
template <int kColumns, int kRows, int kDepth, bool kGated>
__global__ void __launch_bounds__(kBlockThreads)
    experts_stream_kernel(const Product p, void* __restrict__ out, int64_t out_stride, int first_row_tile, int row_tiles, int first_column_tile) {
    constexpr int kTileBytes = kTile * kScaleBlock;
    constexpr int kScalesAt = (kColumns + kRows) * kTileBytes, kBlockBytes = kScalesAt + kWave * 4;
    constexpr int kLoads = 2 * (kColumns + kRows) + 1;  // of a block
    constexpr int kSumBytes = kColumns * kRows * kWave * 16;
    constexpr int kWaveBytes = kDepth * kBlockBytes > kSumBytes ? kDepth * kBlockBytes : kSumBytes;
    static_assert(kRows * kTile <= kWave && (kDepth - 1) * kLoads < 64);
    __shared__ __attribute__((aligned(1024))) char memory[kWavesPerBlock][kWaveBytes];
    constexpr int kOutTiles = kGated ? kColumns / 2 : kColumns;
    const int out_columns = kGated ? p.columns / 2 : p.columns;
    if (static_cast<int>(blockIdx.x) >= row_tiles) {
        // workgroups of their own for the rows of no expert
        constexpr int kValueBytes = kGated ? 4 : 2;
        const int64_t workgroups = static_cast<int64_t>(gridDim.x - row_tiles) * gridDim.y;
        for (int64_t part = static_cast<int64_t>(blockIdx.x - row_tiles) * gridDim.y + blockIdx.y; part < (p.experts + int64_t{1}) * kGapParts;
             part += workgroups)
            clear_rows<false, kBlockThreads, kValueBytes>(static_cast<char*>(out), out_stride * kValueBytes, out_columns, gap_part(p, part));
        return;
    }
    const RowTile tile = find_row_tile<kRows * kTile>(p, first_row_tile + static_cast<int>(blockIdx.x));
    if (tile.expert < 0)
        return;
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int group = lane / kTile, in_tile = lane % kTile;
    const int first_column = (first_column_tile + static_cast<int>(blockIdx.y)) * kOutTiles * kTile;

    f32x4 acc[kColumns][kRows];
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            acc[c][r] = {0.0f, 0.0f, 0.0f, 0.0f};

    {
        // A lane's part of a load: row lane / 8 of its eight and, of that row, a 16-byte piece that is turned by the row, and with
        // it its place in LDS, so that the same piece of eight rows, which an operand reads at once, lies in different banks.
        // Rows and columns past the end are the last one again: what they give is not written.
        const int piece = (lane % 8) ^ (lane / 8);
        const char* weight = p.weight + static_cast<int64_t>(tile.expert) * p.columns * p.inner;
        const char* values = p.values + tile.row * p.value_stride;
        const char* scales = reinterpret_cast<const char*>(p.scales + tile.row * p.scale_stride);
        const char* weight_rows[kColumns][2];
        const char* value_rows[kRows][2];
        const float* weight_scales[kColumns];
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
            const int base = (c / kOutTiles) * out_columns;
            const int column = first_column + c % kOutTiles * kTile;
            weight_scales[c] = p.weight_scales +
                               (static_cast<int64_t>(tile.expert) * p.column_blocks + (base + (column < out_columns ? column : out_columns - 1)) / kScaleBlock) * p.blocks;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = column + half * 8 + lane / 8;
                weight_rows[c][half] = weight + static_cast<int64_t>(base + (row < out_columns ? row : out_columns - 1)) * p.inner;
            }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = r * kTile + half * 8 + lane / 8;
                value_rows[r][half] = values + (row < tile.live ? row : tile.live - 1) * p.value_stride;
            }
        const char* scale_row = scales + (lane < tile.live ? lane : tile.live - 1) * p.scale_stride * 4;
        const uint32_t ring = lds_address(memory[wave]);

        const auto fetch = [&](int block, int slot) {
            const int at = block * kScaleBlock + piece * 16;
            const uint32_t to = ring + slot * kBlockBytes;
#pragma unroll
            for (int c = 0; c < kColumns; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    load_to_lds<16>(at < p.inner ? weight_rows[c][half] + at : reinterpret_cast<const char*>(&kZeroPiece),
                                    to + c * kTileBytes + half * (kTileBytes / 2));
#pragma unroll
            for (int r = 0; r < kRows; ++r)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    load_to_lds<16>(at < p.inner ? value_rows[r][half] + at : reinterpret_cast<const char*>(&kZeroPiece),
                                    to + (kColumns + r) * kTileBytes + half * (kTileBytes / 2));
            load_to_lds<4>(scale_row + block * 4, to + kScalesAt);
        };
        const int turned = in_tile * kScaleBlock + (group ^ (lane & 7)) * 16;
        const auto multiply = [&](int block, int slot) {
            const char* from = memory[wave] + slot * kBlockBytes;
            const auto operand_at = [&](int at) {
                return operand(*reinterpret_cast<const u32x4*>(from + at + turned), *reinterpret_cast<const u32x4*>(from + at + (turned ^ 64)));
            };
            i32x8 weights[kColumns];
            float weight_scale[kColumns];
#pragma unroll
            for (int c = 0; c < kColumns; ++c) {
                weights[c] = operand_at(c * kTileBytes);
                weight_scale[c] = uniform_load(weight_scales[c] + block);
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const i32x8 row = operand_at((kColumns + r) * kTileBytes);
                const float row_scale = reinterpret_cast<const float*>(from + kScalesAt)[r * kTile + in_tile];
#pragma unroll
                for (int c = 0; c < kColumns; ++c) {
                    const f32x4 product = block_product(weights[c], row);
                    const float factor = weight_scale[c] * row_scale;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[c][r][i] = fmaf(factor, product[i], acc[c][r][i]);
                }
            }
        };
        // this wavefront's blocks: wave, wave + 4, ...
        const int count = (p.blocks - wave + kWavesPerBlock - 1) / kWavesPerBlock;
#pragma unroll
        for (int n = 0; n < kDepth - 1; ++n)
            if (n < count)
                fetch(wave + n * kWavesPerBlock, n);
        int slot = 0;
        for (int n = 0; n < count; ++n) {
            // (the slot that is filled is the one the last turn read: its reads are done)
            if (n + kDepth - 1 < count) {
                loaded_but_newest<(kDepth - 2) * kLoads>();
                fetch(wave + (n + kDepth - 1) * kWavesPerBlock, slot == 0 ? kDepth - 1 : slot - 1);
            } else {
                loaded_but_newest<0>();
            }
            multiply(wave + n * kWavesPerBlock, slot);
            slot = slot + 1 == kDepth ? 0 : slot + 1;
        }
    }
    // the ring's memory takes the sums
    f32x4* const sums = reinterpret_cast<f32x4*>(memory[0]);
    constexpr int kWaveSums = kWaveBytes / 16;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            sums[wave * kWaveSums + (c * kRows + r) * kWave + lane] = acc[c][r];
    __syncthreads();
    for (int item = wave; item < kOutTiles * kRows; item += kWavesPerBlock) {
        const int c = item / kRows, r = item % kRows;
        f32x4 total = sums[(c * kRows + r) * kWave + lane];
#pragma unroll
        for (int w = 1; w < kWavesPerBlock; ++w)
            total += sums[w * kWaveSums + (c * kRows + r) * kWave + lane];
        if constexpr (kGated) {
            const int up_at = (c + kOutTiles) * kRows + r;
            f32x4 up = sums[up_at * kWave + lane];
#pragma unroll
            for (int w = 1; w < kWavesPerBlock; ++w)
                up += sums[w * kWaveSums + up_at * kWave + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                total[i] = silu(total[i]) * up[i];
        }
        const int in_size = r * kTile + in_tile;
        const int column = first_column + c * kTile + group * 4;
        if (in_size >= tile.live || column >= out_columns)
            continue;
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

// The same number, which the compiler takes for another: what is computed from it is computed where it is
// needed, and holds no registers over the loops around that place.
__device__ __forceinline__ int afresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Waits until all but the newest kNewer of this wavefront's loads and stores are done, and its reads of LDS, and
// then for the other wavefronts to say the same.
template <int kNewer>
__device__ __forceinline__ void all_but_newest() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kNewer) : "memory");
}

// Waits for this wavefront's reads and writes of LDS, and for the other wavefronts'.
__device__ __forceinline__ void lds_settled() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The products of a tile of 16 * kRowTiles * kRowWaves rows and 16 * kColTiles * kColWaves weight rows, one workgroup.
template <int kRowTiles, int kColTiles, int kRowWaves, int kColWaves, bool kGated>
struct TileShape {
    static constexpr int kWaves = kRowWaves * kColWaves;
    static constexpr int kThreads = kWaves * kWave;
    static constexpr int kRows = kTile * kRowTiles * kRowWaves;
    static constexpr int kCols = kTile * kColTiles * kColWaves;
    static constexpr int kOutCols = kGated ? kCols / 2 : kCols;
    static constexpr int kRowLoads = kRows / 8 / kWaves;     // loads of a wavefront that bring in a block of the rows
    static constexpr int kWeightLoads = kCols / 8 / kWaves;  // ... and of the weights
    // blocks in LDS: as many as fit beside the lists
    static constexpr int kStages = (kRows + kCols) * kScaleBlock * 3 <= (148 << 10) ? 3 : 2;
    // stores of a wavefront that write a tile's output
    static constexpr int kStores = kGated ? kRowTiles * kColTiles / 4 : kRowTiles * kColTiles / 2;
    static_assert(kRows % (8 * kWaves) == 0 && kCols % (8 * kWaves) == 0 && kRows % kWave == 0);
};

// One tile of the list that a workgroup works through.
struct Item {
    int expert;
    int row;
    int live;  // rows, at most the tile's
    int column_tile;
};

constexpr int kMostItems = 256;        // tiles of a list; a workgroup with more makes several
constexpr int kMostSegments = 1 << 14;  // segments whose prefix sums fit the memory the list is made in

// Fills `items` with this workgroup's tiles from its `first`-th on and returns how many there are.  All tiles, of which
// every workgroup counts the same number, are numbered so that kUnit neighbours are kUnitRows row tiles by
// as many column tiles: these share rows and weights, and go to one XCD's workgroups at a time.  `before` has room
// for the segments' prefix sums, `wave_sums` for one number a wavefront.
template <int kRows, int kThreads>
__device__ __forceinline__ int list_tiles(const Product& p, int column_tiles, uint32_t xcd, uint32_t on_xcd, uint32_t xcds, uint32_t unit, int first,
                                          int* before, int* wave_sums, Item* items) {
    const int segments = p.experts;
    const int each = (segments + kThreads - 1) / kThreads;
    const int from = static_cast<int>(threadIdx.x) * each;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int mine = 0;
    for (int e = from; e < from + each && e < segments; ++e) {
        const Segment segment = segment_of(p, e);
        mine += static_cast<int>((segment.live + kRows - 1) / kRows);
    }
    int through = mine;
#pragma unroll
    for (int step = 1; step < kWave; step *= 2) {
        const int other = __shfl_up(through, step, kWave);
        if (lane >= step)
            through += other;
    }
    if (lane == kWave - 1)
        wave_sums[wave] = through;
    lds_settled();
    int at = through - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) {
        at += w < wave ? wave_sums[w] : 0;
        total += wave_sums[w];
    }
    // no more than segments behind one another can have: a layout whose segments lie over one another ends as soon
    const int most = static_cast<int>(p.rows / kRows) + static_cast<int>(p.experts < p.rows ? p.experts : p.rows);
    total = __builtin_amdgcn_readfirstlane(total < 0 || total > most ? most : total);
    for (int e = from; e < from + each && e < segments; ++e) {
        const Segment segment = segment_of(p, e);
        before[e] = at;
        at += static_cast<int>((segment.live + kRows - 1) / kRows);
    }
    lds_settled();
    const uint32_t tiles = static_cast<uint32_t>(total) * static_cast<uint32_t>(column_tiles);
    for (int i = threadIdx.x; i < kMostItems; i += kThreads) {
        const uint64_t number = (static_cast<uint64_t>(first + i) * xcds + xcd) * unit + on_xcd;
        if (number >= tiles)
            continue;
        const uint32_t group_tiles = kUnitRows * static_cast<uint32_t>(column_tiles);
        const uint32_t group = static_cast<uint32_t>(number) / group_tiles, in_group = static_cast<uint32_t>(number) - group * group_tiles;
        const uint32_t left = static_cast<uint32_t>(total) - group * kUnitRows, group_rows = left < kUnitRows ? left : kUnitRows;
        const int row_tile = static_cast<int>(group * kUnitRows + in_group % group_rows);
        // the segment that holds it: the last one that begins at or before it (those behind begin later, or are empty)
        int low = 0, high = segments;
        while (high - low > 1) {
            const int middle = (low + high) / 2;
            if (before[middle] <= row_tile)
                low = middle;
            else
                high = middle;
        }
        const Segment segment = segment_of(p, low);
        const int skipped = (row_tile - before[low]) * kRows;
        const int live = static_cast<int>(segment.live) - skipped;
        // (segments that lie over one another may have more tiles than fit an int: one row then, of some expert's)
        items[i] = skipped < 0 || live <= 0 ? Item{0, 0, 1, 0}
                                            : Item{low, static_cast<int>(segment.begin) + skipped, live > kRows ? kRows : live, static_cast<int>(in_group / group_rows)};
    }
    lds_settled();
    const uint64_t start = (static_cast<uint64_t>(first) * xcds + xcd) * unit + on_xcd;
    const uint64_t stride = static_cast<uint64_t>(xcds) * unit;
    const uint64_t count = start < tiles ? (tiles - start + stride - 1) / stride : 0;
    return static_cast<int>(count > kMostItems ? kMostItems : count);
}

// Products of many rows an expert.  As many workgroups as compute units work through their lists of tiles, 256 rows by 256
// weight rows (a gated product's: 128 of the gate's and the same 128 of the up projection's, so that its 128 output
// columns are one group of the output's scales).  A block of 128 inner columns of both lies in LDS, brought there
// straight from memory; eight wavefronts of 64 weight rows x 128 rows each read their operands from it.
//
// What the order below is about is keeping loads and matrix instructions going.  A wavefront reads a block's weights into
// registers while it works on the last row tile of the block before; half a block on, when all have, their place takes
// the weights of the block after next.  Those come from HBM, all at once for an XCD's workgroups, and have 1.5 blocks'
// time for it.  Rows mostly come from L2 and have one block's.  The two cursors run on into the next tile, whose first
// operands so arrive while this one's output is written.
//
// A lane's four columns of a tile are 8 bytes of bf16: neighbouring column tiles swap halves first, so that half as many
// stores write twice as much each (60 experts, 1424 -> 2816: 140 us against 149).
//
// Measured (32 experts, 29500 rows): 2048 -> 7168 812 to 836 us, 1.04 PFLOP/s; gated 7168 -> 2 x 2048 1650 to 1710 us, 1.04 PFLOP/s:
// 81 % of what a large library product reaches in bf16, matrix instructions busy for 49 and 48 % of the clocks at 2.35 GHz.
// 64 experts of 28 rows, gated, 4096 -> 2 x 2048, 64-row tiles: 200 us, 5.4 TB/s.  The loads of a block of a 256-row tile
// alone take 1.36 us (64 KB that L2 hands out in 64-byte requests), the whole block 3.5; with one block's time ahead for the
// weights the loads alone took 1.76 us.  The 256-row tile spills 19 registers, outside its loop over the blocks.
template <int kRowTiles, int kColTiles, int kRowWaves, int kColWaves, bool kGated>
__global__ void __launch_bounds__(kRowWaves * kColWaves * kWave, 2)
    experts_tile_kernel(const Product p, char* __restrict__ out, int64_t out_stride, int column_tiles, XcdMap xcds) {
    using Shape = TileShape<kRowTiles, kColTiles, kRowWaves, kColWaves, kGated>;
    constexpr int kStages = Shape::kStages;
    constexpr bool kSkips = kRowTiles <= 4;
    constexpr int kRowStep = kRowWaves * kTile;  // the row wavefronts' row tiles alternate
    constexpr int kWeightBytes = Shape::kCols * kScaleBlock, kRowBytes = Shape::kRows * kScaleBlock;
    // accesses of a wavefront that are newer than the next block's operands when it asks for those
    constexpr int kNewer = (kStages - 1) * Shape::kWeightLoads + (kStages - 2) * (Shape::kRowLoads + 1);
    const auto after = [](int slot) { return slot + 1 == kStages ? 0 : slot + 1; };
    __shared__ __attribute__((aligned(1024))) char weight_blocks[kStages][kWeightBytes];
    __shared__ __attribute__((aligned(1024))) char row_blocks[kStages][kRowBytes];
    __shared__ float row_scales[kStages][Shape::kRows];
    __shared__ uint32_t group_amax[kGated ? Shape::kRows : 1][kColWaves];
    __shared__ int wave_sums[Shape::kWaves];
    __shared__ Item items[kMostItems];
    static_assert(sizeof(weight_blocks) >= kMostSegments * sizeof(int));

    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col_wave = wave % kColWaves, row_wave = wave / kColWaves;
    const int group = lane / kTile, in_tile = lane % kTile;
    constexpr int kOutTiles = kGated ? kColTiles / 2 : kColTiles;  // column tiles of the output that a wavefront makes
    const int out_columns = kGated ? p.columns / 2 : p.columns;
    const uint32_t on_xcd = fast_divide(blockIdx.x, xcds.magic, xcds.shift);
    const uint32_t xcd = blockIdx.x - on_xcd * xcds.count;
    const uint32_t unit = fast_divide(gridDim.x, xcds.magic, xcds.shift);

    // A lane's part of a load: row lane / 8 of the load's eight and, of that row, a 16-byte piece that is turned by the row,
    // and with it the piece's place in LDS, so that the same piece of eight rows, which a matrix operand reads at
    // once, lies in different banks.
    const int piece = (lane % 8) ^ (lane / 8);
    const uint32_t weights_at = lds_address(weight_blocks) + wave * 8 * kScaleBlock, rows_at = lds_address(row_blocks) + wave * 8 * kScaleBlock;
    const uint32_t scales_at = lds_address(row_scales) + (wave * kWave % Shape::kRows) * 4;
    constexpr uint32_t kStep = Shape::kWaves * 8 * kScaleBlock;

    for (int listed = 0;; listed += kMostItems) {
        const int count = list_tiles<Shape::kRows, Shape::kThreads>(p, column_tiles, xcd, on_xcd, xcds.count, unit, listed,
                                                                    reinterpret_cast<int*>(weight_blocks), wave_sums, items);
        const auto item_at = [&](int i) -> Item {
            const Item item = items[i];
            return {__builtin_amdgcn_readfirstlane(item.expert), __builtin_amdgcn_readfirstlane(item.row),
                    __builtin_amdgcn_readfirstlane(item.live), __builtin_amdgcn_readfirstlane(item.column_tile)};
        };

        // Tiles begin at different blocks and go round.  All of a block's weights are a weight row's length apart, which for a
        // length like 4096 is on a few of the memory's channels; with all workgroups at the same block, the 256-token decode step
        // took 279 us, so 228.  Tiles that one XCD works on together share their rows, and so begin together.
        const auto first_block = [&](const Item& item) {
            const uint32_t turned = static_cast<uint32_t>(item.expert) * 7 + static_cast<uint32_t>(item.column_tile / kUnitCols) * 5;
            return static_cast<int>(turned % static_cast<uint32_t>(p.blocks));
        };
        // the weights' cursor
        int weight_item = 0, weight_block = 0, weight_left = 0, weight_slot = 0;
        const char* weight = nullptr;
        uint32_t weight_offset[Shape::kWeightLoads];
        const auto aim_weights = [&]() {
            const Item item = item_at(weight_item);
            weight = p.weight + static_cast<int64_t>(item.expert) * p.columns * p.inner;
            weight_block = first_block(item);
            weight_left = p.blocks;
            const int first_column = item.column_tile * Shape::kOutCols;
            const int row_in_load = afresh(lane) / 8;
#pragma unroll
            for (int i = 0; i < Shape::kWeightLoads; ++i) {
                const int row = 8 * (i * Shape::kWaves + wave) + row_in_load;
                int column;
                if constexpr (kGated) {
                    // a wavefront's weight rows: its tiles of the gate, then the same ones of the up projection
                    const int in_wave = row % (kTile * kColTiles), half = in_wave / (kTile * kOutTiles);
                    column = first_column + row / (kTile * kColTiles) * (kTile * kOutTiles) + in_wave % (kTile * kOutTiles);
                    column = (column < out_columns ? column : out_columns - 1) + half * out_columns;
                } else {
                    column = first_column + row;
                    column = column < out_columns ? column : out_columns - 1;
                }
                weight_offset[i] = static_cast<uint32_t>(column) * static_cast<uint32_t>(p.inner);
            }
        };
        // brings in the cursor's block; whether there was one
        const auto fetch_weights = [&]() {
            if (weight_item >= count)
                return false;
            const int64_t at = static_cast<int64_t>(weight_block) * kScaleBlock;
            const uint32_t to = weights_at + weight_slot * kWeightBytes;
            if (at + kScaleBlock <= p.inner) {
#pragma unroll
                for (int i = 0; i < Shape::kWeightLoads; ++i)
                    load_to_lds<16>(weight + at, weight_offset[i] + piece * 16, to + i * kStep);
            } else {
                // (whole addresses, made from the offsets here: kept over the loops they would cost the registers of twice as many)
#pragma unroll
                for (int i = 0; i < Shape::kWeightLoads; ++i) {
                    const uint32_t offset = static_cast<uint32_t>(afresh(static_cast<int>(weight_offset[i])));
                    load_to_lds<16>(at + piece * 16 < p.inner ? weight + at + offset + piece * 16 : reinterpret_cast<const char*>(&kZeroPiece),
                                    to + i * kStep);
                }
            }
            weight_slot = after(weight_slot);
            if (++weight_block == p.blocks)
                weight_block = 0;
            if (--weight_left == 0) {
                ++weight_item;
                if (weight_item < count)
                    aim_weights();
            }
            return true;
        };

        // the rows' cursor; rows past the live ones are the last one again, and what they give is not written
        int row_item = weight_item, row_block = 0, row_left = 0, row_slot = 0;
        const char *values = nullptr, *scales = nullptr;
        uint32_t row_offset[Shape::kRowLoads], scale_offset = 0;
        const auto aim_rows = [&]() {
            const Item item = item_at(row_item);
            const int live = item.live;
            row_block = first_block(item);
            row_left = p.blocks;
            values = p.values + static_cast<int64_t>(item.row) * p.value_stride;
            scales = reinterpret_cast<const char*>(p.scales + static_cast<int64_t>(item.row) * p.scale_stride);
            const int row_in_load = afresh(lane) / 8;
#pragma unroll
            for (int i = 0; i < Shape::kRowLoads; ++i) {
                const int row = 8 * (i * Shape::kWaves + wave) + row_in_load;
                row_offset[i] = static_cast<uint32_t>(row < live ? row : live - 1) * static_cast<uint32_t>(p.value_stride);
            }
            const int scaled = wave * kWave % Shape::kRows + afresh(lane);
            scale_offset = static_cast<uint32_t>(scaled < live ? scaled : live - 1) * static_cast<uint32_t>(p.scale_stride) * 4u;
        };
        const auto fetch_rows = [&]() {
            if (row_item >= count)
                return;
            const int64_t at = static_cast<int64_t>(row_block) * kScaleBlock;
            const uint32_t to = rows_at + row_slot * kRowBytes;
            if (at + kScaleBlock <= p.inner) {
#pragma unroll
                for (int i = 0; i < Shape::kRowLoads; ++i)
                    load_to_lds<16>(values + at, row_offset[i] + piece * 16, to + i * kStep);
            } else {
#pragma unroll
                for (int i = 0; i < Shape::kRowLoads; ++i) {
                    const uint32_t offset = static_cast<uint32_t>(afresh(static_cast<int>(row_offset[i])));
                    load_to_lds<16>(at + piece * 16 < p.inner ? values + at + offset + piece * 16 : reinterpret_cast<const char*>(&kZeroPiece),
                                    to + i * kStep);
                }
            }
            // (where there are more wavefronts than 64 rows, some bring in the same scales)
            load_to_lds<4>(scales + static_cast<int64_t>(row_block) * 4, scale_offset, scales_at + row_slot * Shape::kRows * 4);
            row_slot = after(row_slot);
            if (++row_block == p.blocks)
                row_block = 0;
            if (--row_left == 0) {
                ++row_item;
                if (row_item < count)
                    aim_rows();
            }
        };

        int slot = 0;
        const int turned = (group ^ (lane & 7)) * 16;
        const int weight_at = (col_wave * kColTiles * kTile + in_tile) * kScaleBlock, row_at = (row_wave * kTile + in_tile) * kScaleBlock;
        const int scale_at = row_wave * kTile + in_tile;
        // a lane's two pieces of a row: columns group * 16 on of the block, and 64 further
        const auto weight_piece = [&](int in_slot, int c, int half) {
            return *reinterpret_cast<const u32x4*>(weight_blocks[in_slot] + weight_at + c * kTile * kScaleBlock + (turned ^ half * 64));
        };
        const auto row_piece = [&](int in_slot, int r, int half) {
            return *reinterpret_cast<const u32x4*>(row_blocks[in_slot] + row_at + r * kRowStep * kScaleBlock + (turned ^ half * 64));
        };
        bf16x8 wide_weights[kColTiles][4];
        const auto read_weights = [&](int in_slot, int c) {
            const u32x4 low = weight_piece(in_slot, c, 0), high = weight_piece(in_slot, c, 1);
            wide_weights[c][0] = widened(low.x, low.y);
            wide_weights[c][1] = widened(low.z, low.w);
            wide_weights[c][2] = widened(high.x, high.y);
            wide_weights[c][3] = widened(high.z, high.w);
        };
        u32x4 rows[2][2];
        float scale[2];
        const auto read_rows = [&](int in_slot, int r, int to) {
            rows[to][0] = row_piece(in_slot, r, 0);
            rows[to][1] = row_piece(in_slot, r, 1);
            scale[to] = row_scales[in_slot][scale_at + r * kRowStep];
        };
        bool weights_ahead = false;  // whether the newest fetch of weights was one
        if (weight_item < count) {
            aim_weights();
            aim_rows();
#pragma unroll
            for (int stage = 0; stage < kStages; ++stage) {
                weights_ahead = fetch_weights();
                fetch_rows();
            }
            if (weights_ahead)
                all_but_newest<(kStages - 1) * (Shape::kWeightLoads + Shape::kRowLoads + 1)>();
            else
                all_but_newest<0>();
#pragma unroll
            for (int c = 0; c < kColTiles; ++c)
                read_weights(0, c);
            read_rows(0, 0, 0);
        }
        // the rows of no expert, while the first operands are on their way
        if (listed == 0 && p.expert_offsets != nullptr)
            for (int part = static_cast<int>(blockIdx.x); part < (p.experts + 1) * kGapParts; part += static_cast<int>(gridDim.x))
                clear_rows<kGated, Shape::kThreads>(out, out_stride, out_columns, gap_part(p, part));
        int stored = 0;  // blocks whose operands are older than the last tile's stores
        for (int i = 0; i < count; ++i) {
            const Item item = item_at(i);
            const int live = item.live;
            const int first_column = item.column_tile * Shape::kOutCols;
            f32x4 acc[kColTiles][kRowTiles];
#pragma unroll
            for (int c = 0; c < kColTiles; ++c)
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r)
                    acc[c][r] = {0.0f, 0.0f, 0.0f, 0.0f};

            {
                // the scales of this wavefront's column tiles: one where they are neighbours within 128 columns
                constexpr int kScales = kGated ? kColTiles : 1;
                static_assert(kGated || kScaleBlock % (kColTiles * kTile) == 0);
                static_assert(kRowTiles % 2 == 0);  // a step's place of the two that hold row operands goes by its number
                constexpr int kRefill = kRowTiles / 2 - 1;
                const float* weight_scales[kScales];
                float next_scale[kScales];
#pragma unroll
                for (int c = 0; c < kScales; ++c) {
                    int column = first_column + (col_wave * kOutTiles + c % kOutTiles) * kTile;
                    column = (column < out_columns ? column : out_columns - 1) + (c / kOutTiles) * out_columns;
                    weight_scales[c] = p.weight_scales + (static_cast<int64_t>(item.expert) * p.column_blocks + column / kScaleBlock) * p.blocks;
                    next_scale[c] = uniform_load(weight_scales[c] + first_block(item));
                }
                // Row tiles without a live row are left out of small tiles, whose few rows an expert the matrix instructions take
                // longer with than the weights' way from memory: gated, 32 experts of 16 rows 188 us against 238; linear,
                // 128 experts of 1 row 30.6 against 35.7.  A 256-row tile has no registers for it (gated 1690 us would be 2000), nor
                // for one branch over its other half where it is half full (linear, 2048 -> 7168 828 us would be 982).
                const int live_tiles = kSkips ? __builtin_amdgcn_readfirstlane((static_cast<int>(live) - row_wave * kTile + kRowStep - 1) / kRowStep) : kRowTiles;
                int block = first_block(item);
                for (int turn = 0; turn < p.blocks; ++turn) {
                    float column_scale[kScales];
                    block = block + 1 < p.blocks ? block + 1 : 0;
                    const int next_block = block;
#pragma unroll
                    for (int c = 0; c < kScales; ++c) {
                        column_scale[c] = next_scale[c];
                        next_scale[c] = uniform_load(weight_scales[c] + next_block);
                    }
#pragma unroll
                    for (int r = 0; r < kRowTiles; ++r) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (r == kRefill) {
                            // every wavefront has read the block's weights: the next but one's may come
                            lds_settled();
                            weights_ahead = fetch_weights();
                        }
                        if (r + 1 < kRowTiles) {
                            read_rows(slot, r + 1, (r + 1) & 1);
                        } else {
                            // The next block's operands are there, and every wavefront has read this block's last row tile. The
                            // matrix instructions of that tile hide the first reads of the next block.
                            if (!weights_ahead)
                                all_but_newest<0>();
                            else if (stored > 0)
                                all_but_newest<kNewer + Shape::kStores>();
                            else
                                all_but_newest<kNewer>();
                            --stored;
                            fetch_rows();
                            read_rows(after(slot), 0, 0);
                        }
                        float linear_factor = 0.0f;  // (a gated product has no registers for its four ahead of their use)
                        if constexpr (!kGated)
                            linear_factor = column_scale[0] * scale[r & 1];
                        f32x4 product[kColTiles];
#pragma unroll
                        for (int c = 0; c < kColTiles; ++c)
                            product[c] = {0.0f, 0.0f, 0.0f, 0.0f};
                        if (!kSkips || r < live_tiles) {
#pragma unroll
                            for (int part = 0; part < 4; ++part) {
                                const u32x4 raw = rows[r & 1][part / 2];
                                const bf16x8 wide = part % 2 == 0 ? widened(raw.x, raw.y) : widened(raw.z, raw.w);
#pragma unroll
                                for (int c = 0; c < kColTiles; ++c)
                                    product[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wide_weights[c][part], wide, product[c], 0, 0, 0);
                            }
                        }
                        if (r + 1 == kRowTiles) {
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                            for (int c = 0; c < kColTiles; ++c)
                                read_weights(after(slot), c);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        if (!kSkips || r < live_tiles) {
#pragma unroll
                            for (int c = 0; c < kColTiles; ++c) {
                                const float factor = kGated ? column_scale[c % kScales] * scale[r & 1] : linear_factor;
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    acc[c][r][j] = fmaf(factor, product[c][j], acc[c][r][j]);
                            }
                        }
                        // (done here, not where the sums are next used, with all products kept until then)
                        static_assert(kColTiles == 4);
                        asm volatile("" : "+v"(acc[0][r]), "+v"(acc[1][r]), "+v"(acc[2][r]), "+v"(acc[3][r]));
                    }
                    slot = after(slot);
                }
            }

            // Stores past the tile's rows or columns are dropped by the buffer's bounds, not branched around: a wavefront's
            // number of them is always the same, which the count of newest accesses above relies on.
            const int out_lane = afresh(lane), in_group = out_lane / kTile;
            const int first_row = row_wave * kTile + out_lane % kTile;
            constexpr uint32_t kNowhere = 0xffffffffu;
            char* tile_out = out + item.row * out_stride;
            const __amdgpu_buffer_rsrc_t tile_rows = __builtin_amdgcn_make_buffer_rsrc(tile_out, 0, static_cast<int>(live * out_stride), 0x00020000);
            if constexpr (!kGated) {
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) {
                    const int in_rows = first_row + r * kRowStep;
                    const uint32_t row = static_cast<uint32_t>(in_rows) * static_cast<uint32_t>(out_stride);
#pragma unroll
                    for (int c = 0; c < kColTiles; c += 2) {
                        // two neighbouring column tiles: lanes of even groups get eight columns of the first, of odd ones of the second
                        const f32x4 v = acc[c][r], w = acc[c + 1][r];
                        const u32x2 low = swapped(to_bf16_pair(v[0], v[1]), to_bf16_pair(w[0], w[1]));
                        const u32x2 high = swapped(to_bf16_pair(v[2], v[3]), to_bf16_pair(w[2], w[3]));
                        const int column = first_column + (col_wave * kColTiles + c + in_group % 2) * kTile + in_group / 2 * 8;
                        __builtin_amdgcn_raw_buffer_store_b128(u32x4{low.x, high.x, low.y, high.y}, tile_rows,
                                                               column < out_columns ? row + column * 2 : kNowhere, 0, 0);
                    }
                }
            } else {
                // the tile's output columns are one group of 128: its largest value is found over the wavefronts through LDS
                static_assert(!kGated || Shape::kOutCols == kScaleBlock);
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) {
                    uint32_t amax = 0;
                    const bool is_live = first_row + r * kRowStep < live;
#pragma unroll
                    for (int c = 0; c < kOutTiles; ++c) {
                        const int column = first_column + (col_wave * kOutTiles + c) * kTile + in_group * 4;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float act = is_live && column < out_columns ? silu(acc[c][r][j]) * acc[c + kOutTiles][r][j] : 0.0f;
                            acc[c][r][j] = act;
                            amax = larger(amax, magnitude_bits(act));
                        }
                    }
                    amax = larger(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 16, kWave)));
                    amax = larger(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 32, kWave)));
                    if (in_group == 0)
                        group_amax[first_row + r * kRowStep][col_wave] = amax;
                }
                lds_settled();
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) {
                    const int in_rows = first_row + r * kRowStep;
                    uint32_t amax = group_amax[in_rows][0];
#pragma unroll
                    for (int w = 1; w < kColWaves; ++w)
                        amax = larger(amax, group_amax[in_rows][w]);
                    const GroupScale scale = group_scale(amax);
                    const uint32_t row = static_cast<uint32_t>(in_rows) * static_cast<uint32_t>(out_stride);
                    // the scale, and the record's padding with its last group
                    if (col_wave == 0 && in_group == 0 && in_rows < live)
                        reinterpret_cast<float*>(tile_out + row + out_columns)[item.column_tile] = scale.scale;
                    if (item.column_tile == column_tiles - 1 && col_wave == kColWaves - 1 && in_rows < live)
                        for (int word = out_columns / 4 + column_tiles + in_group; word < static_cast<int>(out_stride / 4); word += 4)
                            reinterpret_cast<uint32_t*>(tile_out + row)[word] = 0u;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int c = 0; c < kOutTiles; ++c)
                            acc[c][r][j] *= scale.inverse;
                }
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) {
                    const uint32_t row = static_cast<uint32_t>(first_row + r * kRowStep) * static_cast<uint32_t>(out_stride);
                    static_assert(kOutTiles % 2 == 0 || !kGated);
#pragma unroll
                    for (int c = 0; c < kOutTiles; c += 2) {
                        const u32x2 both = swapped(to_fp8_quad(acc[c][r][0], acc[c][r][1], acc[c][r][2], acc[c][r][3]),
                                                   to_fp8_quad(acc[c + 1][r][0], acc[c + 1][r][1], acc[c + 1][r][2], acc[c + 1][r][3]));
                        const int column = first_column + (col_wave * kOutTiles + c + in_group % 2) * kTile + in_group / 2 * 8;
                        __builtin_amdgcn_raw_buffer_store_b64(both, tile_rows, column < out_columns ? row + column : kNowhere, 0, 0);
                    }
                }
            }
            stored = kStages - 1;
        }
        // (the list's memory is the weights': nothing may still be on its way there)
        if (count < kMostItems)
            return;
        all_but_newest<0>();
    }
}

// fp32 rows in 8 bits with a scale for every 128 columns: a wavefront a row, 16 lanes a group of 128 columns.  Few rows
// behind a product of few rows, so that its time is a launch's: eight rows of 2048 4.1 us.
__global__ void __launch_bounds__(kBlockThreads) quantize_rows_kernel(const float* __restrict__ rows,
                                                                      char* __restrict__ records,
                                                                      int64_t num_rows,
                                                                      int64_t record_bytes,
                                                                      int columns,
                                                                      int groups) {
    const int lane = threadIdx.x % kWave;
    const int64_t row = workgroup_number() * kWavesPerBlock + threadIdx.x / kWave;
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

constexpr int kMostColumns = 1 << 24;

int product_of(const void* values, int64_t value_stride, const float* scales, int64_t scale_stride, const void* weight,
               const float* weight_scales, const int64_t* expert_offsets, const int64_t* expert_counts, int64_t rows, int64_t experts,
               int inner, int columns, int column_multiple, Product& p) {
    if (rows < 0 || rows > 0x7fffffff || experts <= 0 || experts >= (int64_t{1} << 30) || inner <= 0 || inner % 16 != 0 || columns <= 0 ||
        columns > kMostColumns || columns % column_multiple != 0 || (expert_offsets == nullptr) != (expert_counts == nullptr))
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

// Most tiles of kRows rows that the experts' rows can have: each expert's but the full ones end in one that is not.
int64_t most_row_tiles(const Product& p, int rows) { return p.rows / rows + (p.experts < p.rows ? p.experts : p.rows); }

constexpr int kMostGridSteps = 65535;  // of a launch's second axis

template <int kColumns, int kRows, int kDepth, bool kGated>
int launch_stream(const Product& p, void* out, int64_t out_stride, hipStream_t stream) {
    const int out_columns = kGated ? p.columns / 2 : p.columns;
    constexpr int kOutColumns = (kGated ? kColumns / 2 : kColumns) * kTile;
    const int64_t tiles = most_row_tiles(p, kRows * kTile), column_tiles = (out_columns + kOutColumns - 1) / kOutColumns;
    // as many rows and columns at a time as the axes of a grid have steps; the first launch clears the rows of no expert
    for (int64_t first_row = 0; first_row < tiles; first_row += kMostOnAxis)
        for (int64_t first = 0; first < column_tiles; first += kMostGridSteps) {
            const int64_t rows = std::min(tiles - first_row, kMostOnAxis), columns = std::min<int64_t>(column_tiles - first, kMostGridSteps);
            const bool clears = p.expert_offsets != nullptr && first_row == 0 && first == 0;
            const int64_t gaps = clears ? std::min(((p.experts + int64_t{1}) * kGapParts + columns - 1) / columns, kMostOnAxis) : 0;
            experts_stream_kernel<kColumns, kRows, kDepth, kGated>
                <<<dim3(static_cast<unsigned>(rows + gaps), static_cast<unsigned>(columns)), kBlockThreads, 0, stream>>>(
                    p, out, out_stride, static_cast<int>(first_row), static_cast<int>(rows), static_cast<int>(first));
            NANOEP_HIP_TRY(hipGetLastError());
        }
    return NANOEP_OK;
}

template <int kRowTiles, int kColTiles, int kRowWaves, int kColWaves, bool kGated>
int launch_tiles(const Product& p, void* out, int64_t out_stride, hipStream_t stream) {
    using Shape = TileShape<kRowTiles, kColTiles, kRowWaves, kColWaves, kGated>;
    const Topology topology = current_topology(current_tuning());
    const XcdMap xcds = make_xcd_map(topology.xcds);
    const int out_columns = kGated ? p.columns / 2 : p.columns;
    const int column_tiles = (out_columns + Shape::kOutCols - 1) / Shape::kOutCols;
    if (most_row_tiles(p, Shape::kRows) * column_tiles > 0x7fffffff)
        return NANOEP_ERR_INVALID_ARGUMENT;
    // a workgroup a compute unit, the same number on every XCD
    const unsigned workgroups = xcds.count * std::max(1u, static_cast<unsigned>(topology.cus) / xcds.count);
    experts_tile_kernel<kRowTiles, kColTiles, kRowWaves, kColWaves, kGated>
        <<<dim3(workgroups), Shape::kThreads, 0, stream>>>(p, static_cast<char*>(out), out_stride, column_tiles, xcds);
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

// Rows of the tile kernel's tiles for a product, 0 for the stream kernel.
//   The tile follows the rows an expert has on average.  Of 32 experts, 2048 -> 7168 (gated, 7168 -> 2 x 2048):
//       rows each                   43         58        115        130        172         460
//       64-row tiles, us     107 (192)  129 (274)  193 (428)  233        260        663 (1403)
//       128-row tiles        116 (210)  122 (229)  153 (370)  202 (500)  246 (530)  491 (1042)
//       256-row tiles        225        225 (445)  228 (457)  230 (458)  234 (457)  428 (895)
//   With most rows at a few experts the two larger ones change order a little later: 172 rows each, 266 (619) and 287 us (617).
//   Smaller tiles, where the larger ones do not go round the compute units.
//   The stream kernel, whose wavefronts share out the inner columns, where the smallest do not either: one token's eight experts,
//   gated, 7168 -> 2048, 47 us against 93; 768 -> 2048, 7.4 us against 15.1; 115 rows of 128 experts of these 43 us, 31 with 64-row tiles.
//   And for addresses beyond the tile kernel's: an expert's weight and a tile's rows, in and out, lie within 32-bit offsets, its list
//   of tiles is made from at most kMostSegments experts.
int tile_rows(int64_t rows, int64_t experts, int inner, int columns, int out_columns_each, int out_columns, int64_t value_stride, int64_t scale_stride) {
    constexpr int64_t kMost = int64_t{1} << 32;
    if (experts >= kMostSegments || columns > 1 << 21 || static_cast<int64_t>(columns) * inner > kMost || value_stride > kMost / 256 ||
        scale_stride > kMost / 1024)
        return 0;
    const Tuning tuning = current_tuning();
    if (tuning.experts_tile != 0)
        return tuning.experts_tile == 64 || tuning.experts_tile == 128 || tuning.experts_tile == 256 ? tuning.experts_tile : 0;
    const int64_t cus = current_topology(tuning).cus;
    const int64_t each = rows / experts, column_tiles = (out_columns + out_columns_each - 1) / out_columns_each;
    const int64_t owners = experts < rows ? experts : rows;
    for (const int tile : {256, 128, 64}) {
        const bool suits = tile == 64 || each > (tile == 256 ? 128 : 48);
        if (suits && (rows / tile > owners ? rows / tile : owners) * column_tiles >= cus)
            return tile;
    }
    return 0;
}

template <bool kGated>
int launch_product(const Product& p, void* out, int64_t out_stride, int tile, hipStream_t stream) {
    if (tile == 256)
        return launch_tiles<8, 4, 2, 4, kGated>(p, out, out_stride, stream);
    if (tile == 128)
        return launch_tiles<4, 4, 2, 4, kGated>(p, out, out_stride, stream);
    return launch_tiles<2, 4, 2, 4, kGated>(p, out, out_stride, stream);
}

// `out_stride` in values: bf16 ones, or a gated product's fp32 ones.
template <bool kGated>
int launch_streams(const Product& p, void* out, int64_t out_stride, hipStream_t stream) {
    if (p.rows / p.experts <= 16)
        return launch_stream<2, 1, 3, kGated>(p, out, out_stride, stream);
    return launch_stream<2, 4, 2, kGated>(p, out, out_stride, stream);
}

int linear_tile_rows(const Product& p) {
    return tile_rows(p.rows, p.experts, p.inner, p.columns, TileShape<8, 4, 2, 4, false>::kOutCols, p.columns, p.value_stride, p.scale_stride);
}

int gated_tile_rows(int64_t rows, int64_t experts, int inner, int columns, int64_t value_stride, int64_t scale_stride) {
    return tile_rows(rows, experts, inner, columns, TileShape<8, 4, 2, 4, true>::kOutCols, columns / 2, value_stride, scale_stride);
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
    const auto on = static_cast<hipStream_t>(stream);
    if (const int tile = linear_tile_rows(p))
        return launch_product<false>(p, out, static_cast<int64_t>(columns) * 2, tile, on);
    return launch_streams<false>(p, out, columns, on);
}

size_t nanoep_experts_gated_workspace_bytes(int64_t rows, int64_t experts, int inner, int columns, int64_t value_stride,
                                            int64_t scale_stride) {
    if (rows <= 0 || experts <= 0 || inner <= 0 || columns <= 0 ||
        nanoep::gated_tile_rows(rows, experts, inner, columns, value_stride, scale_stride) != 0)
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
    if (const int tile = gated_tile_rows(rows, experts, inner, columns, value_stride, scale_stride))
        return launch_product<true>(p, records, record_bytes_of(columns / 2), tile, on);
    const int launched = launch_streams<true>(p, workspace, columns / 2, on);
    if (launched != NANOEP_OK)
        return launched;
    quantize_rows_kernel<<<grid_of((rows + kWavesPerBlock - 1) / kWavesPerBlock), kBlockThreads, 0, on>>>(
        static_cast<const float*>(workspace), static_cast<char*>(records), rows, record_bytes_of(columns / 2), columns / 2,
        static_cast<int>(scale_groups(columns / 2)));
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

}  // extern "C"
