// Combine with the gate weights applied, and its gradient.

#include <algorithm>

#include "nanoep_operators.h"

namespace nanoep {
namespace {

constexpr int kWeightedRows = 8;  // rows of a token that are fetched at a time

// out[t] = bias[t] + sum over valid k, ascending, of weights[t][k] * y[slot[t][k]], in fp32, rounded to bf16 once.
// One wavefront a 512-column chunk of a token's row, four to a workgroup: lane k fetches the token's k-th slot and
// weight, which are broadcast to scalars; up to eight rows are fetched back to back (a masked choice is not fetched).
// HBM-bound: 4096 tokens of 7168, eight choices and a bias (540 MB) 85.3 us, 6.3 TB/s, what plain streams reach.  Chunks, not
// rows, because a few hundred tokens fill the device with them: 256 tokens of 4096 (17 MB) 5.3 us, a launch and the chain of slot,
// row and store.
__global__ void __launch_bounds__(kBlockThreads) combine_weighted_kernel(const u32x4* __restrict__ y,             // [C][vectors]
                                                                         const int32_t* __restrict__ token_slots,  // [T][K]
                                                                         const float* __restrict__ weights,       // [T][K]
                                                                         const u32x4* __restrict__ bias,          // [T][vectors] or null
                                                                         u32x4* __restrict__ out,                 // [T][vectors]
                                                                         int64_t y_rows,
                                                                         int64_t work_items,
                                                                         int vectors,
                                                                         int chunks,
                                                                         int num_topk) {
    const int lane = threadIdx.x % kWave;
    const int64_t item = workgroup_number() * kWavesPerBlock + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (item >= work_items)
        return;
    const int64_t token = item / chunks;
    const int chunk = static_cast<int>(item - token * chunks);
    const int vector = chunk * kWave + lane;
    const int load_vector = vector < vectors ? vector : 0;

    int slot = -1;
    float weight = 0.0f;
    if (lane < num_topk) {
        slot = token_slots[token * num_topk + lane];
        weight = weights[token * num_topk + lane];
    }
    const uint64_t valid = __ballot(slot >= 0 && slot < y_rows);
    float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int base = 0; base < num_topk; base += kWeightedRows) {
        u32x4 data[kWeightedRows];
#pragma unroll
        for (int k = 0; k < kWeightedRows; ++k)
            if ((valid >> (base + k)) & 1)
                data[k] = load_vec<true>(y + static_cast<int64_t>(__builtin_amdgcn_readlane(slot, base + k)) * vectors + load_vector);
#pragma unroll
        for (int k = 0; k < kWeightedRows; ++k)
            if ((valid >> (base + k)) & 1) {
                const float factor = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), base + k));
                float values[8];
                unpack_bf16(data[k], values);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    acc[i] = fmaf(factor, values[i], acc[i]);
            }
    }
    if (vector < vectors) {
        if (bias != nullptr) {
            float values[8];
            unpack_bf16(bias[token * vectors + vector], values);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                acc[i] += values[i];
        }
        store_vec<true>(out + token * vectors + vector, pack_bf16(acc));
    }
}

// Zeros in a part of the rows of grad_y that no choice refers to: behind every expert's rows, and behind the last expert's
// segment, each in kGapParts parts, at most kMostGapBlocks at a time.
constexpr int kGapParts = 8;
constexpr int64_t kMostGapBlocks = int64_t{1} << 20;
constexpr int64_t kGapBytesApart = int64_t{32} << 20;
__device__ __forceinline__ void clear_gap(const int64_t* expert_offsets, const int64_t* expert_counts, u32x4* rows, int64_t num_rows,
                                          int64_t num_experts, int vectors, int64_t part) {
    const int64_t expert = part / kGapParts;
    int64_t begin = expert_offsets[expert], end = num_rows;
    if (expert < num_experts) {
        begin += expert_counts[expert];
        end = expert_offsets[expert + 1];
    }
    begin = begin < 0 ? 0 : begin;
    end = end > num_rows ? num_rows : end;
    if (begin >= end)
        return;
    const int64_t gap = (end - begin) * vectors, each = (gap + kGapParts - 1) / kGapParts;
    const int64_t from = part % kGapParts * each, to = from + each < gap ? from + each : gap;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int64_t at = from + threadIdx.x; at < to; at += kBlockThreads)
        store_vec<true>(rows + begin * vectors + at, zero);
}

// The gradient: grad_y[slot[t][k]] = weights[t][k] * grad[t], grad_weights[t][k] = <y[slot[t][k]], grad[t]>.
// One wavefront a (token, choice) walks the row once: it reads both rows, writes the third and keeps the product's
// sum in its lanes, which are added in a fixed order at the end.  A token's choices are neighbours, so that its
// gradient row comes from the caches for all but one of them.  Workgroups ahead of theirs clear the rows of no expert.
// No atomics: the order of every sum is fixed.  HBM-bound: 4096 tokens of 7168, eight choices (1.14 GB with 16200 padding rows)
// 169 to 171 us and 22 for the padding, 5.9 TB/s; 1537 of 2816, six choices (115 MB) 20 to 23 us, 5.2 TB/s.
__global__ void __launch_bounds__(kBlockThreads) combine_weighted_backward_kernel(const u32x4* __restrict__ grad,  // [T][vectors]
                                                                                  const u32x4* __restrict__ y,     // [C][vectors]
                                                                                  const int32_t* __restrict__ token_slots,
                                                                                  const float* __restrict__ weights,
                                                                                  u32x4* __restrict__ grad_y,
                                                                                  float* __restrict__ grad_weights,
                                                                                  const int64_t* __restrict__ expert_offsets,  // null: all cleared before
                                                                                  const int64_t* __restrict__ expert_counts,
                                                                                  int64_t num_experts,
                                                                                  int64_t y_rows,
                                                                                  int64_t pairs,
                                                                                  int64_t gap_blocks,
                                                                                  int vectors,
                                                                                  int num_topk) {
    const int64_t block = workgroup_number();
    if (block < gap_blocks) {
        for (int64_t part = block; part < (num_experts + 1) * kGapParts; part += gap_blocks)
            clear_gap(expert_offsets, expert_counts, grad_y, y_rows, num_experts, vectors, part);
        return;
    }
    const int lane = threadIdx.x % kWave;
    const int64_t pair = (block - gap_blocks) * kWavesPerBlock + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (pair >= pairs)
        return;
    const int64_t slot = token_slots[pair];
    if (slot < 0 || slot >= y_rows) {
        if (lane == 0)
            grad_weights[pair] = 0.0f;
        return;
    }
    const float weight = weights[pair];
    const u32x4* grad_row = grad + pair / num_topk * vectors;
    const u32x4* y_row = y + slot * vectors;
    u32x4* out_row = grad_y + slot * vectors;
    float product = 0.0f;
#pragma unroll 4
    for (int at = lane; at < vectors; at += kWave) {
        float g[8], v[8];
        unpack_bf16(grad_row[at], g);
        unpack_bf16(load_vec<true>(y_row + at), v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            product = fmaf(v[i], g[i], product);
            g[i] *= weight;
        }
        store_vec<true>(out_row + at, pack_bf16(g));
    }
    product = wave_sum(product);
    if (lane == 0)
        grad_weights[pair] = product;
}

__global__ void __launch_bounds__(kBlockThreads) zero_rows_kernel(u32x4* __restrict__ rows, int64_t vectors) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x; at < vectors;
         at += static_cast<int64_t>(gridDim.x) * kBlockThreads)
        store_vec<true>(rows + at, zero);
}

bool weighted_sizes_fit(int64_t y_rows, int64_t num_tokens, int hidden, int num_topk) {
    return y_rows >= 0 && num_tokens >= 0 && hidden > 0 && hidden % 8 == 0 && num_topk >= 1 && num_topk <= kMaxTopk &&
           num_tokens <= 0x7fffffff / kMaxTopk && y_rows <= 0x7fffffff;
}

}  // namespace
}  // namespace nanoep

extern "C" {

int nanoep_combine_weighted(const void* y, int64_t y_rows, const int32_t* token_slots, const float* weights, const void* bias,
                            int64_t num_tokens, int hidden, int num_topk, void* out, void* stream) {
    using namespace nanoep;
    if (!weighted_sizes_fit(y_rows, num_tokens, hidden, num_topk))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens == 0)
        return NANOEP_OK;
    if ((y == nullptr && y_rows > 0) || token_slots == nullptr || weights == nullptr || out == nullptr || !aligned16(y) || !aligned16(bias) ||
        !aligned16(out))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const int vectors = hidden / 8;
    const int chunks = (vectors + kWave - 1) / kWave;
    const int64_t items = num_tokens * chunks;
    const int64_t blocks = (items + kWavesPerBlock - 1) / kWavesPerBlock;
    combine_weighted_kernel<<<grid_of(blocks), kBlockThreads, 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const u32x4*>(y), token_slots, weights, static_cast<const u32x4*>(bias), static_cast<u32x4*>(out), y_rows, items, vectors,
        chunks, num_topk);
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

int nanoep_combine_weighted_backward(const void* grad, const void* y, int64_t y_rows, const int32_t* token_slots, const float* weights,
                                     const int64_t* expert_offsets, const int64_t* expert_counts, int64_t num_local_experts,
                                     int64_t num_tokens, int hidden, int num_topk, void* grad_y, float* grad_weights, void* stream) {
    using namespace nanoep;
    if (!weighted_sizes_fit(y_rows, num_tokens, hidden, num_topk) || (expert_offsets == nullptr) != (expert_counts == nullptr))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (expert_offsets != nullptr && (num_local_experts <= 0 || num_local_experts >= 0x7fffffff))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if ((y_rows > 0 && (y == nullptr || grad_y == nullptr)) || !aligned16(grad) || !aligned16(y) || !aligned16(grad_y))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens > 0 && (grad == nullptr || token_slots == nullptr || weights == nullptr || grad_weights == nullptr))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens == 0 && y_rows == 0)
        return NANOEP_OK;
    const int vectors = hidden / 8;
    const auto on = static_cast<hipStream_t>(stream);
    if (y_rows > 0 && expert_offsets == nullptr) {
        zero_rows_kernel<<<2048, kBlockThreads, 0, on>>>(static_cast<u32x4*>(grad_y), y_rows * vectors);
        NANOEP_HIP_TRY(hipGetLastError());
    }
    const int64_t pairs = num_tokens * num_topk, pair_blocks = (pairs + kWavesPerBlock - 1) / kWavesPerBlock;
    const int64_t gap_blocks = y_rows > 0 && expert_offsets != nullptr ? std::min((num_local_experts + 1) * kGapParts, kMostGapBlocks) : 0;
    // Few rows to clear ride in the gradient's launch (9222 choices, 450 padding rows of 2816: 23.0 us, in a launch of their own
    // 28.8); many have one ahead of it, because writes alone and the gradient's mix go faster one after the other (29500
    // choices, 16200 padding rows of 7168: 197 us, beside one another 204).
    const bool apart = (y_rows - pairs) * hidden * 2 > kGapBytesApart;
    const auto launch = [&](int64_t gaps, int64_t blocks) {
        if (blocks > 0)
            combine_weighted_backward_kernel<<<grid_of(blocks), kBlockThreads, 0, on>>>(
                static_cast<const u32x4*>(grad), static_cast<const u32x4*>(y), token_slots, weights, static_cast<u32x4*>(grad_y), grad_weights,
                expert_offsets, expert_counts, num_local_experts, y_rows, pairs, gaps, vectors, num_topk);
    };
    if (apart)
        launch(gap_blocks, gap_blocks);
    launch(apart ? 0 : gap_blocks, (apart ? 0 : gap_blocks) + pair_blocks);
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

}  // extern "C"
