// The router's choice of experts with its gate weights, the loss that balances the experts, and their gradients.
//
// Scores of a token's logits l over the experts: softmax e^l_e / sum e^l, or sigmoid 1 / (1 + e^-l_e).
// Values that are not rounded the same way everywhere must not decide which expert is chosen: the choice goes by the logits
// themselves, which are in the order of their scores, or, where a bias is added or groups are compared, by scores
// in 64 bits.  Weights, losses and gradients are fp32.

#include <algorithm>

#include "nanoep_lanes.h"
#include "nanoep_operators.h"

namespace nanoep {
namespace {

constexpr int kMostExperts = 4096;
constexpr int kMostGroups = 64;

struct Logits {
    const void* data;
    int64_t stride;  // elements from a token to the next
    bool wide;       // fp32, else bf16
    bool quads;      // four neighbours from a multiple of four on are aligned, and all of them are experts or none
};

__device__ __forceinline__ float load_logit(const Logits& logits, int64_t token, int expert) {
    const int64_t at = token * logits.stride + expert;
    if (logits.wide)
        return static_cast<const float*>(logits.data)[at];
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(logits.data)[at]) << 16);
}

// kEach neighbours of a token's logits from `first` on, -infinity behind the last expert.
template <int kEach>
__device__ __forceinline__ void load_neighbours(const Logits& logits, int64_t token, int first, int experts, float (&out)[kEach]) {
    if (kEach % 4 == 0 && logits.quads) {
        const int64_t base = token * logits.stride + first;
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
            const bool in = first + i < experts;
            if (logits.wide) {
                u32x4 data = {0u, 0u, 0u, 0u};
                if (in)
                    data = *reinterpret_cast<const u32x4*>(static_cast<const float*>(logits.data) + base + i);
#pragma unroll
                for (int j = 0; j < 4 && i + j < kEach; ++j)
                    out[i + j] = in ? __uint_as_float(data[j]) : -INFINITY;
            } else {
                uint2 data = {0u, 0u};
                if (in)
                    data = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(logits.data) + base + i);
                const float four[4] = {from_bf16_low(data.x), from_bf16_high(data.x), from_bf16_low(data.y), from_bf16_high(data.y)};
#pragma unroll
                for (int j = 0; j < 4 && i + j < kEach; ++j)
                    out[i + j] = in ? four[j] : -INFINITY;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        out[i] = first + i < experts ? load_logit(logits, token, first + i) : -INFINITY;
}

// Values as unsigned integers in the same order: 0 for -infinity, which stands for an expert that cannot be chosen, NaN above
// everything, both zeros alike.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    if (v != v)
        return 0xffffffffu;
    if (bits == 0xff800000u)
        return 0u;
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(double v) {
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    if (v != v)
        return ~uint64_t{0};
    if (bits == 0xfff0000000000000u)
        return 0u;
    return bits >> 63 ? ~bits : bits | uint64_t{1} << 63;
}
__device__ __forceinline__ double value_of(uint64_t key) {
    if (key == 0)
        return -INFINITY;
    return __longlong_as_double(static_cast<long long>(key >> 63 ? key & ~(uint64_t{1} << 63) : ~key));  // all ones: a NaN
}

// The largest key over the lanes that share a token, in all of them.
template <int kLanes>
__device__ __forceinline__ uint32_t largest_key(uint32_t key) {
    return lanes_max<kLanes>(key);
}
template <int kLanes>
__device__ __forceinline__ uint64_t largest_key(uint64_t key) {
    const uint32_t high = lanes_max<kLanes>(static_cast<uint32_t>(key >> 32));
    const uint32_t low = lanes_max<kLanes>(static_cast<uint32_t>(key >> 32) == high ? static_cast<uint32_t>(key) : 0u);
    return static_cast<uint64_t>(high) << 32 | low;
}

// What a wavefront's lanes wrote to LDS is there for its other lanes (LDS works a wavefront's accesses off in order).
__device__ __forceinline__ void wavefront_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The lanes of this token for which `condition` holds, the token's first lane as bit 0.
template <int kLanes>
__device__ __forceinline__ uint64_t lanes_where(bool condition) {
    const uint64_t all = __ballot(condition);
    if constexpr (kLanes == 64)
        return all;
    return all >> (threadIdx.x % kWave / kLanes * kLanes) & ((uint64_t{1} << kLanes) - 1);
}

struct Route {
    Logits logits;
    const float* bias;    // [E] or null
    const uint8_t* mask;  // [T] or null: zero for tokens that go nowhere
    int64_t* ids;         // [T][K]
    float* weights;       // [T][K]
    int64_t tokens;
    int experts, topk, groups, topk_groups;
    bool sigmoid, normalize;
    float scale;
};

struct Choice {
    int expert;
    float logit;
};

// kLanes neighbouring lanes a token, kEach neighbouring experts a lane.  K rounds: the largest key of all, the lowest lane
// that has it, the lowest of its experts that has it; that lane notes the choice in LDS and strikes the expert out.  Then
// lane k has choice k, and the weights come from the chosen logits (and the sums over all of them, for a softmax that is not
// normalized over the choices).
// kExact: keys are scores (plus bias) in 64 bits.  Groups of neighbouring experts are then compared by the sum of their two
// largest values, by groups of lanes that read the keys from LDS, and the experts of all but the best are struck out first.
template <int kLanes, int kEach, bool kExact>
__global__ void __launch_bounds__(kBlockThreads) route_topk_kernel(const Route a) {
    using Key = std::conditional_t<kExact, uint64_t, uint32_t>;
    __shared__ Choice choices[kBlockThreads / kLanes][kMaxTopk];
    extern __shared__ uint64_t all_keys[];  // [wavefronts][kLanes * kEach], for groups
    const int lane = threadIdx.x % kLanes, place = threadIdx.x / kLanes;
    const int64_t token = workgroup_number() * (blockDim.x / kLanes) + place;
    const bool here = token < a.tokens;
    const bool routed = here && (a.mask == nullptr || a.mask[token] != 0);
    const int first = lane * kEach;

    float logit[kEach];
    load_neighbours<kEach>(a.logits, routed ? token : 0, first, routed ? a.experts : 0, logit);

    // the softmax over all experts
    float largest = -INFINITY, total = 0.0f;
    bool broken = false;  // a NaN or an infinity among them: all of their scores are NaN
    if (!a.sigmoid && (kExact || !a.normalize)) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            largest = fmaxf(largest, logit[i]);
        largest = lanes_max<kLanes>(largest);
        if (largest == -INFINITY)
            largest = 0.0f;  // no expert: sums are 0, nothing is chosen
    }
    if (!a.sigmoid && !a.normalize) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            total += expf(logit[i] - largest);
        total = lanes_sum<kLanes>(total);
    }

    Key key[kEach];
    if constexpr (kExact) {
        double value[kEach], sum = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            value[i] = exp(a.sigmoid ? -static_cast<double>(logit[i]) : static_cast<double>(logit[i]) - largest);
            sum += value[i];
        }
        if (!a.sigmoid)
            sum = lanes_sum<kLanes>(sum);
        broken = !a.sigmoid && sum != sum;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            value[i] = a.sigmoid ? 1.0 / (1.0 + value[i]) : value[i] / sum;
            if (a.bias != nullptr && first + i < a.experts)
                value[i] += a.bias[first + i];
            key[i] = logit[i] == -INFINITY ? 0 : key_of(value[i]);
        }
        if (a.groups > 1) {
            uint64_t* keys = all_keys + static_cast<int64_t>(place) * kLanes * kEach;
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                keys[first + i] = key[i];
            wavefront_sync();
            // (a whole wavefront a token) its lanes are shared out among the groups, a power of two each
            const int size = a.experts / a.groups;
            int sharing = 1;
            while (2 * sharing * a.groups <= kLanes)
                sharing *= 2;
            const int group = lane / sharing;
            uint64_t best = 0, second = 0;
            if (group < a.groups)
                for (int at = lane % sharing; at < size; at += sharing) {
                    const uint64_t other = keys[group * size + at];
                    second = other > best ? best : other > second ? other : second;
                    best = other > best ? other : best;
                }
            for (int distance = 1; distance < sharing; distance *= 2) {
                const uint64_t other_best = __shfl_xor(static_cast<unsigned long long>(best), distance, kWave);
                const uint64_t other_second = __shfl_xor(static_cast<unsigned long long>(second), distance, kWave);
                const uint64_t lower = best < other_best ? best : other_best, higher = second > other_second ? second : other_second;
                best = best > other_best ? best : other_best;
                second = lower > higher ? lower : higher;
            }
            uint64_t of_group = 0;
            if (group < a.groups && lane % sharing == 0 && best != 0)
                of_group = second == 0 ? best : key_of(value_of(best) + value_of(second));
            uint64_t open = 0;  // bit `group * sharing` for the best groups
            for (int round = 0; round < a.topk_groups; ++round) {
                const uint64_t top = largest_key<kLanes>(of_group);
                const uint64_t having = __ballot(of_group == top && top != 0);
                const uint64_t winner = having & (~having + 1);
                open |= winner;
                if (winner >> lane & 1)
                    of_group = 0;
            }
            int of = first / size, left = size - (first - of * size);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                if (left == 0) {
                    ++of;
                    left = size;
                }
                if (of >= a.groups || !(open >> (of * sharing) & 1))
                    key[i] = 0;
                --left;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            key[i] = key_of(logit[i]);
    }

    for (int round = 0; round < a.topk; ++round) {
        Key best = key[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i)
            best = key[i] > best ? key[i] : best;
        const Key top = largest_key<kLanes>(best);
        const bool match = best == top && top != 0;
        const uint64_t having = lanes_where<kLanes>(match);
        if (match && (having & ((uint64_t{1} << lane) - 1)) == 0) {
            int at = kEach;
            float value = 0.0f;
#pragma unroll
            for (int i = kEach - 1; i >= 0; --i)
                if (key[i] == top) {
                    at = i;
                    value = logit[i];
                }
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                key[i] = i == at ? 0 : key[i];
            choices[place][round] = {first + at, value};
        } else if (having == 0 && lane == 0) {
            choices[place][round] = {-1, 0.0f};
        }
    }
    wavefront_sync();

    Choice choice = {-1, 0.0f};
    if (lane < a.topk)
        choice = choices[place][lane];
    const bool valid = choice.expert >= 0;
    float weight;
    if (a.sigmoid) {
        // numerators and denominators times e^-shift, so that their sum is not lost where all scores are tiny
        const float shift = a.normalize ? fminf(lanes_max<kLanes>(valid ? choice.logit : -INFINITY), 0.0f) : 0.0f;
        weight = expf(fminf(choice.logit, 0.0f) - shift) / (1.0f + expf(-fabsf(choice.logit)));
        if (choice.logit != choice.logit)
            weight = choice.logit;
    } else {
        if (a.normalize)
            largest = lanes_max<kLanes>(valid ? choice.logit : -INFINITY);
        weight = broken ? NAN : expf(choice.logit - largest);
    }
    weight = valid ? weight : 0.0f;
    if (a.normalize)
        total = lanes_sum<kLanes>(weight);
    if (a.normalize || !a.sigmoid)
        weight = valid ? weight / total : 0.0f;
    if (here && lane < a.topk) {
        a.ids[token * a.topk + lane] = choice.expert;
        a.weights[token * a.topk + lane] = weight * a.scale;
    }
}

// ------------------------------------------------------------------ gradients of a token's scores

// What a wavefront has of a token's logits: expert i * 64 + lane in place i, -infinity behind the last.
template <int kEach>
__device__ __forceinline__ void load_spread(const Logits& logits, int64_t token, int experts, float (&out)[kEach]) {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int expert = i * kWave + lane;
        out[i] = expert < experts ? load_logit(logits, token, expert) : -INFINITY;
    }
}

template <int kEach>
__device__ __forceinline__ void store_spread(void* out, bool wide, int64_t token, int experts, const float (&v)[kEach]) {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int expert = i * kWave + lane;
        if (expert >= experts)
            continue;
        if (wide)
            static_cast<float*>(out)[token * experts + expert] = v[i];
        else
            static_cast<uint16_t*>(out)[token * experts + expert] = static_cast<uint16_t>(to_bf16_pair(v[i], 0.0f));
    }
}

// Every expert's share of its token: softmax, or sigmoid over its sum.  rest: what is left of its sigmoid to one (softmax: 1).
// Experts at -infinity have none; a token of nothing else has no shares.
template <int kEach>
__device__ __forceinline__ void shares_of(const float (&logit)[kEach], bool sigmoid, float (&share)[kEach], float (&rest)[kEach]) {
    float largest = -INFINITY, total = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        largest = fmaxf(largest, logit[i]);
    largest = lanes_max<kWave>(largest);
    const float shift = largest == -INFINITY ? 0.0f : sigmoid ? fminf(largest, 0.0f) : largest;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (sigmoid) {
            // e^-shift * sigmoid: the sum is not lost where all of them are tiny
            const float tail = expf(-fabsf(logit[i]));
            const float inverse = 1.0f / (1.0f + tail);
            share[i] = logit[i] != logit[i] ? logit[i] : expf(fminf(logit[i], 0.0f) - shift) * inverse;
            rest[i] = logit[i] >= 0.0f ? tail * inverse : inverse;
        } else {
            share[i] = expf(logit[i] - shift);
            rest[i] = 1.0f;
        }
        total += share[i];
    }
    total = lanes_sum<kWave>(total);
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        share[i] *= inverse;
}

struct RouteBackward {
    Logits logits;
    const float* grad;   // [T][K]
    const int64_t* ids;  // [T][K]
    void* grad_logits;   // [T][E], as wide as the logits
    int64_t tokens;
    int experts, topk;
    bool sigmoid, normalize;
    float scale;
};

// A wavefront a token.  With the gradients g_k of the weights w_k, c = scale:
//   softmax over the choices          dl_k = w_k (g_k - sum_j g_j w_j / c)
//   softmax over all experts          dl_e = p_e ([e is chosen] c g_e - sum_j c g_j p_j)
//   sigmoids over the choices' sum    dl_k = w_k (1 - s_k) (g_k - sum_j g_j w_j / c)
//   sigmoids                          dl_k = c g_k s_k (1 - s_k)
// and zero for every other expert.  Only the second reads more than the chosen logits.  An expert that is named twice has both
// gradients.
template <int kEach>
__global__ void __launch_bounds__(kBlockThreads) route_topk_backward_kernel(const RouteBackward a) {
    const int lane = threadIdx.x % kWave;
    const int64_t token = workgroup_number() * kWavesPerBlock + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (token >= a.tokens)
        return;
    int64_t named = -1;
    float g = 0.0f, logit = -INFINITY;
    if (lane < a.topk) {
        named = a.ids[token * a.topk + lane];
        g = a.grad[token * a.topk + lane];
    }
    const bool valid = named >= 0 && named < a.experts;
    const int expert = valid ? static_cast<int>(named) : -1;
    if (valid)
        logit = load_logit(a.logits, token, expert);
    g = valid ? g * a.scale : 0.0f;

    float out[kEach];
    float each = 0.0f;  // the gradient of this lane's choice
    if (a.normalize) {
        const float largest = lanes_max<kWave>(logit);
        float score = 0.0f, rest = 1.0f;
        if (a.sigmoid) {
            const float tail = expf(-fabsf(logit)), inverse = 1.0f / (1.0f + tail);
            score = logit != logit ? logit : expf(fminf(logit, 0.0f) - fminf(largest, 0.0f)) * inverse;
            rest = logit >= 0.0f ? tail * inverse : inverse;
        } else {
            score = expf(logit - largest);
        }
        score = valid ? score : 0.0f;
        const float total = lanes_sum<kWave>(score);
        score = valid ? score / total : 0.0f;
        const float mean = lanes_sum<kWave>(score * g);
        each = score * rest * (g - mean);
    } else if (a.sigmoid) {
        const float tail = expf(-fabsf(logit)), inverse = 1.0f / (1.0f + tail);
        each = g * tail * inverse * inverse;
    } else {
        float rest[kEach], all[kEach];
        load_spread<kEach>(a.logits, token, a.experts, all);
        shares_of<kEach>(all, false, out, rest);
        // the chosen ones' shares from the same sums: where they are in `out`
        float along = 0.0f;
        for (int k = 0; k < a.topk; ++k) {
            const int at = __builtin_amdgcn_readlane(expert, k);
            const float gk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), k));
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (i * kWave + lane == at)
                    along = fmaf(gk, out[i], along);
        }
        along = lanes_sum<kWave>(along);
        float wide[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            wide[i] = 0.0f;
        for (int k = 0; k < a.topk; ++k) {
            const int at = __builtin_amdgcn_readlane(expert, k);
            const float gk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), k));
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                wide[i] += i * kWave + lane == at ? gk : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] *= wide[i] - along;
        store_spread<kEach>(a.grad_logits, a.logits.wide, token, a.experts, out);
        return;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        out[i] = 0.0f;
    for (int k = 0; k < a.topk; ++k) {
        const int at = __builtin_amdgcn_readlane(expert, k);
        const float gk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(each), k));
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] += i * kWave + lane == at ? gk : 0.0f;
    }
    store_spread<kEach>(a.grad_logits, a.logits.wide, token, a.experts, out);
}

// ------------------------------------------------------------------ the balance loss

struct Balance {
    Logits logits;
    const int64_t* ids;      // [T][K]
    const int64_t* offsets;  // [S + 1], null: all tokens are one sequence
    int64_t tokens, sequences;
    int experts, topk, parts;  // workgroups a sequence
    bool sigmoid;
};

// The tokens of a part of a sequence, within the batch whatever the offsets say.
__device__ __forceinline__ void part_of(const Balance& a, int64_t sequence, int part, int64_t& from, int64_t& to) {
    int64_t begin = 0, end = a.tokens;
    if (a.offsets != nullptr) {
        begin = a.offsets[sequence];
        end = a.offsets[sequence + 1];
        begin = begin < 0 ? 0 : begin;
        end = end > a.tokens ? a.tokens : end;
    }
    const int64_t length = end > begin ? end - begin : 0, each = (length + a.parts - 1) / a.parts;
    from = begin + (part * each < length ? part * each : length);
    to = from + each < begin + length ? from + each : begin + length;
}

// A choice of a token in lane k, and whether the token has any.
__device__ __forceinline__ int choice_of(const Balance& a, int64_t token, bool& live) {
    const int lane = threadIdx.x % kWave;
    int64_t named = -1;
    if (lane < a.topk)
        named = a.ids[token * a.topk + lane];
    const bool valid = named >= 0 && named < a.experts;
    live = __ballot(valid) != 0;
    return valid ? static_cast<int>(named) : -1;
}

__device__ __forceinline__ float workgroup_sum(float v, float* place) {
    v = lanes_sum<kWave>(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0)
        place[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < static_cast<int>(blockDim.x) / kWave; ++w)
        v += place[w];
    return v;
}

// counts, tokens and loss of a sequence from the sums over its tokens: loss = E / (C T') * sum over e of c_e * sum of shares.
// Each thread has the experts from threadIdx.x on, blockDim.x apart.
__device__ __forceinline__ void finish_sequence(int64_t sequence, int experts, const float* shares, const int* chosen, int live, float* loss,
                                                int64_t* counts, int64_t* tokens, float* place) {
    float sum = 0.0f, number = 0.0f;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {
        counts[sequence * experts + e] = chosen[e];
        sum = fmaf(static_cast<float>(chosen[e]), shares[e], sum);
        number += static_cast<float>(chosen[e]);
    }
    sum = workgroup_sum(sum, place);
    number = workgroup_sum(number, place);
    if (threadIdx.x == 0) {
        tokens[sequence] = live;
        loss[sequence] = live > 0 ? sum * static_cast<float>(experts) / number / static_cast<float>(live) : 0.0f;
    }
}

// Wavefronts of a workgroup, by the experts a lane has (registers, and LDS: half of the wavefronts' sums and the counts).
constexpr int kMostBalanceWaves = 16;
constexpr int balance_waves(int each) { return each <= 16 ? kMostBalanceWaves : 4; }

// A workgroup a part of a sequence: a wavefront a token at a time, its lanes keep their experts' sums of shares in registers;
// choices are counted in LDS (whole numbers: any order gives the same).  The wavefronts' sums are added in a fixed order.  A sequence
// of one part is finished here, others leave a row of sums to balance_finish_kernel.
template <int kEach>
__global__ void __launch_bounds__(balance_waves(kEach) * kWave) balance_loss_kernel(const Balance a, float* __restrict__ part_shares,  // [S * parts][E]
                                                                                int* __restrict__ part_counts,  // [S * parts][E + 1]
                                                                                float* __restrict__ loss, int64_t* __restrict__ counts,
                                                                                int64_t* __restrict__ tokens) {
    extern __shared__ float lds[];  // [waves / 2][kEach * 64] sums, then [kEach * 64] counts
    __shared__ float place[kMostBalanceWaves];
    __shared__ int live_tokens;
    constexpr int kWidth = kEach * kWave;
    const int64_t block = workgroup_number();
    if (block >= a.sequences * a.parts)
        return;
    const int64_t sequence = block / a.parts;
    const int waves = blockDim.x / kWave, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    int* chosen = reinterpret_cast<int*>(lds + waves / 2 * kWidth);
    for (int e = threadIdx.x; e < kWidth; e += blockDim.x)
        chosen[e] = 0;
    if (threadIdx.x == 0)
        live_tokens = 0;
    __syncthreads();

    int64_t from, to;
    part_of(a, sequence, static_cast<int>(block - sequence * a.parts), from, to);
    float sums[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        sums[i] = 0.0f;
    int number = 0;
    for (int64_t token = from + wave; token < to; token += waves) {
        bool live;
        const int expert = choice_of(a, token, live);
        float logit[kEach], share[kEach], rest[kEach];
        load_spread<kEach>(a.logits, token, a.experts, logit);
        if (expert >= 0)
            atomicAdd(&chosen[expert], 1);
        if (live) {
            ++number;
            shares_of<kEach>(logit, a.sigmoid, share, rest);
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                sums[i] += share[i];
        }
    }
    if (lane == 0 && number > 0)
        atomicAdd(&live_tokens, number);
    for (int half = waves / 2; half > 0; half /= 2) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                lds[(wave - half) * kWidth + i * kWave + lane] = sums[i];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                sums[i] += lds[wave * kWidth + i * kWave + lane];
        __syncthreads();
    }
    if (a.parts > 1) {
        if (wave == 0)
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (i * kWave + lane < a.experts)
                    part_shares[block * a.experts + i * kWave + lane] = sums[i];
        for (int e = threadIdx.x; e < a.experts; e += blockDim.x)
            part_counts[block * (a.experts + 1) + e] = chosen[e];
        if (threadIdx.x == 0)
            part_counts[block * (a.experts + 1) + a.experts] = live_tokens;
        return;
    }
    if (wave == 0)
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            lds[i * kWave + lane] = sums[i];
    __syncthreads();
    finish_sequence(sequence, a.experts, lds, chosen, live_tokens, loss, counts, tokens, place);
}

constexpr int kFinishThreads = 1024;

// One workgroup a sequence adds up the rows of its parts, every expert's in the order of the parts (shared out among groups of threads).
__global__ void __launch_bounds__(kFinishThreads) balance_finish_kernel(int64_t sequences, int experts, int parts, int width,  // a power of two, at most 1024
                                                                        const float* __restrict__ part_shares, const int* __restrict__ part_counts,
                                                                        float* __restrict__ loss, int64_t* __restrict__ counts,
                                                                        int64_t* __restrict__ tokens) {
    __shared__ float shares[kMostExperts];
    __shared__ int chosen[kMostExperts];
    __shared__ float group_shares[kFinishThreads];
    __shared__ int group_counts[kFinishThreads];
    __shared__ float place[kFinishThreads / kWave];
    __shared__ int live_tokens;
    const int64_t sequence = workgroup_number();
    if (sequence >= sequences)
        return;
    const int groups = kFinishThreads / width, group = threadIdx.x / width, column = threadIdx.x % width;
    const int64_t first = sequence * parts;
    if (threadIdx.x == 0)
        live_tokens = 0;
    __syncthreads();
    for (int base = 0; base < experts; base += width) {
        const int e = base + column;
        float share = 0.0f;
        int count = 0;
        if (e < experts)
#pragma unroll 8
            for (int part = group; part < parts; part += groups) {
                share += part_shares[(first + part) * experts + e];
                count += part_counts[(first + part) * (experts + 1) + e];
            }
        group_shares[threadIdx.x] = share;
        group_counts[threadIdx.x] = count;
        __syncthreads();
        if (group == 0 && e < experts) {
            for (int other = 1; other < groups; ++other) {
                share += group_shares[other * width + column];
                count += group_counts[other * width + column];
            }
            shares[e] = share;
            chosen[e] = count;
        }
        __syncthreads();
    }
    int live = 0;
    for (int part = threadIdx.x; part < parts; part += kFinishThreads)
        live += part_counts[(first + part) * (experts + 1) + experts];
    if (live > 0)
        atomicAdd(&live_tokens, live);
    __syncthreads();
    finish_sequence(sequence, experts, shares, chosen, live_tokens, loss, counts, tokens, place);
}

// The gradient: with F_e = g E c_e / (C T') of the token's sequence, p_e (F_e - sum of F p) (times 1 - s_e for sigmoids); zero for
// tokens without a choice and for those of no sequence, which the workgroups behind the last sequence's clear.
template <int kEach>
__global__ void __launch_bounds__(kBlockThreads) balance_loss_backward_kernel(const Balance a, const float* __restrict__ grad,  // [S]
                                                                              const int64_t* __restrict__ counts, const int64_t* __restrict__ tokens,
                                                                              void* __restrict__ grad_logits) {
    const int64_t block = workgroup_number();
    const int64_t sequence = block / a.parts;
    const int part = static_cast<int>(block - sequence * a.parts);
    const int waves = blockDim.x / kWave, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    float factor[kEach], out[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        out[i] = 0.0f;
    if (sequence >= a.sequences) {
        if (sequence > a.sequences || a.offsets == nullptr)
            return;
        const int64_t begin = a.offsets[0], end = a.offsets[a.sequences];
        for (int64_t token = static_cast<int64_t>(part) * waves + wave; token < a.tokens; token += static_cast<int64_t>(a.parts) * waves)
            if (token < begin || token >= end)
                store_spread<kEach>(grad_logits, a.logits.wide, token, a.experts, out);
        return;
    }
    int64_t from, to;
    part_of(a, sequence, part, from, to);
    if (from + wave >= to)
        return;
    float number = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int expert = i * kWave + lane;
        factor[i] = expert < a.experts ? static_cast<float>(counts[sequence * a.experts + expert]) : 0.0f;
        number += factor[i];
    }
    number = lanes_sum<kWave>(number);
    const int64_t live_tokens = tokens[sequence];
    const float each = live_tokens > 0 && number > 0.0f ? grad[sequence] * static_cast<float>(a.experts) / number / static_cast<float>(live_tokens) : 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        factor[i] *= each;
    for (int64_t token = from + wave; token < to; token += waves) {
        bool live;
        choice_of(a, token, live);
        float logit[kEach], share[kEach], rest[kEach], along = 0.0f;
        load_spread<kEach>(a.logits, token, a.experts, logit);
        if (live) {
            shares_of<kEach>(logit, a.sigmoid, share, rest);
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                along = fmaf(factor[i], share[i], along);
            along = lanes_sum<kWave>(along);
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] = live ? share[i] * rest[i] * (factor[i] - along) : 0.0f;
        store_spread<kEach>(grad_logits, a.logits.wide, token, a.experts, out);
    }
}

// ------------------------------------------------------------------ launches

// Experts a lane when a wavefront has a token.
int each_of(int experts) {
    int each = 1;
    while (each * kWave < experts)
        each *= 2;
    return each;
}

#define NANOEP_BY_EACH(EACH, CALL) \
    switch (EACH) {                \
        case 1:                    \
            CALL(1);               \
            break;                 \
        case 2:                    \
            CALL(2);               \
            break;                 \
        case 4:                    \
            CALL(4);               \
            break;                 \
        case 8:                    \
            CALL(8);               \
            break;                 \
        case 16:                   \
            CALL(16);              \
            break;                 \
        case 32:                   \
            CALL(32);              \
            break;                 \
        default:                   \
            CALL(64);              \
            break;                 \
    }

bool router_sizes_fit(int64_t stride, int logits_type, int64_t num_tokens, int experts, int topk, int scoring) {
    return num_tokens >= 0 && num_tokens <= 0x7fffffff / kMaxTopk && experts >= 1 && experts <= kMostExperts && topk >= 1 && topk <= kMaxTopk &&
           stride >= experts && stride <= int64_t{1} << 31 && (logits_type == NANOEP_BF16 || logits_type == NANOEP_FP32) &&
           (scoring == NANOEP_SOFTMAX || scoring == NANOEP_SIGMOID);
}

Logits logits_of(const void* data, int64_t stride, int type, int experts) {
    const size_t quad = type == NANOEP_FP32 ? 16 : 8;
    return {data, stride, type == NANOEP_FP32, experts % 4 == 0 && stride % 4 == 0 && reinterpret_cast<uintptr_t>(data) % quad == 0};
}

// Parts of a sequence: one for every 64 tokens of an average one, at most 256 (balance_finish_kernel reads them all).
constexpr int64_t kPartTokens = 64;
constexpr int64_t kMostParts = 256;
int parts_of(int64_t num_tokens, int64_t sequences) {
    const int64_t average = (num_tokens + sequences - 1) / sequences;
    return static_cast<int>(std::min(kMostParts, std::max<int64_t>(1, (average + kPartTokens - 1) / kPartTokens)));
}

}  // namespace
}  // namespace nanoep

extern "C" {

int nanoep_route_topk(const void* logits, int64_t logits_stride, int logits_type, const float* bias, const uint8_t* mask, int64_t num_tokens,
                      int num_experts, int num_topk, int groups, int topk_groups, int scoring, int normalize, float scale, int64_t* ids,
                      float* weights, void* stream) {
    using namespace nanoep;
    if (!router_sizes_fit(logits_stride, logits_type, num_tokens, num_experts, num_topk, scoring) || num_topk > num_experts)
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (groups < 1 || groups > kMostGroups || num_experts % groups != 0 || topk_groups < 1 || topk_groups > groups ||
        num_topk > topk_groups * (num_experts / groups))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens == 0)
        return NANOEP_OK;
    if (logits == nullptr || ids == nullptr || weights == nullptr)
        return NANOEP_ERR_INVALID_ARGUMENT;
    const Route arguments = {logits_of(logits, logits_stride, logits_type, num_experts), bias, mask, ids, weights, num_tokens, num_experts, num_topk,
                             topk_groups < groups ? groups : 1, topk_groups, scoring == NANOEP_SIGMOID, normalize != 0, scale};
    const bool exact = bias != nullptr || arguments.groups > 1;
    const int each = each_of(num_experts);
    const int waves = arguments.groups > 1 && each > 16 ? 1 : kWavesPerBlock;  // (LDS: 8 bytes an expert for groups)
    const size_t lds = arguments.groups > 1 ? static_cast<size_t>(waves) * each * kWave * sizeof(uint64_t) : 0;
    const dim3 grid = grid_of((num_tokens + waves - 1) / waves);
    const auto on = static_cast<hipStream_t>(stream);
#define NANOEP_LAUNCH_ROUTE(EACH)                                                          \
    if (exact)                                                                             \
        route_topk_kernel<kWave, EACH, true><<<grid, waves * kWave, lds, on>>>(arguments); \
    else                                                                                   \
        route_topk_kernel<kWave, EACH, false><<<grid, waves * kWave, lds, on>>>(arguments)
    NANOEP_BY_EACH(each, NANOEP_LAUNCH_ROUTE)
#undef NANOEP_LAUNCH_ROUTE
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

int nanoep_route_topk_backward(const float* grad, const void* logits, int64_t logits_stride, int logits_type, const int64_t* ids,
                               int64_t num_tokens, int num_experts, int num_topk, int scoring, int normalize, float scale, void* grad_logits,
                               void* stream) {
    using namespace nanoep;
    if (!router_sizes_fit(logits_stride, logits_type, num_tokens, num_experts, num_topk, scoring))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens == 0)
        return NANOEP_OK;
    if (grad == nullptr || logits == nullptr || ids == nullptr || grad_logits == nullptr)
        return NANOEP_ERR_INVALID_ARGUMENT;
    const RouteBackward arguments = {logits_of(logits, logits_stride, logits_type, num_experts), grad, ids, grad_logits, num_tokens, num_experts,
                                     num_topk, scoring == NANOEP_SIGMOID, normalize != 0, scale};
    const dim3 grid = grid_of((num_tokens + kWavesPerBlock - 1) / kWavesPerBlock);
    const auto on = static_cast<hipStream_t>(stream);
#define NANOEP_LAUNCH_ROUTE_BACKWARD(EACH) route_topk_backward_kernel<EACH><<<grid, kBlockThreads, 0, on>>>(arguments)
    NANOEP_BY_EACH(each_of(num_experts), NANOEP_LAUNCH_ROUTE_BACKWARD)
#undef NANOEP_LAUNCH_ROUTE_BACKWARD
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

size_t nanoep_balance_loss_workspace_bytes(int64_t num_tokens, int num_experts, int64_t sequences) {
    using namespace nanoep;
    if (num_tokens < 0 || num_experts < 1 || num_experts > kMostExperts || sequences < 1 || sequences > 0x7fffffff)
        return 0;
    const int parts = parts_of(num_tokens, sequences);
    return parts == 1 ? 0 : static_cast<size_t>(sequences) * parts * (2 * static_cast<size_t>(num_experts) + 1) * sizeof(float);
}

int nanoep_balance_loss(const void* logits, int64_t logits_stride, int logits_type, const int64_t* ids, const int64_t* sequence_offsets,
                        int64_t num_tokens, int num_experts, int num_topk, int64_t sequences, int scoring, float* loss, int64_t* counts,
                        int64_t* tokens, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace nanoep;
    if (!router_sizes_fit(logits_stride, logits_type, num_tokens, num_experts, num_topk, scoring) || sequences < 1 || sequences > 0x7fffffff ||
        (sequence_offsets == nullptr && sequences != 1))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (loss == nullptr || counts == nullptr || tokens == nullptr || (num_tokens > 0 && (logits == nullptr || ids == nullptr)))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < nanoep_balance_loss_workspace_bytes(num_tokens, num_experts, sequences))
        return NANOEP_ERR_WORKSPACE;
    const Balance arguments = {logits_of(logits, logits_stride, logits_type, num_experts), ids, sequence_offsets, num_tokens, sequences, num_experts,
                               num_topk, parts_of(num_tokens, sequences), scoring == NANOEP_SIGMOID};
    if (arguments.parts > 1 && (workspace == nullptr || !aligned16(workspace)))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const int each = each_of(num_experts);
    const int waves = balance_waves(each);
    const size_t lds = (static_cast<size_t>(waves / 2) + 1) * each * kWave * sizeof(float);
    const int64_t blocks = sequences * arguments.parts;
    auto* part_shares = static_cast<float*>(workspace);
    auto* part_counts = static_cast<int*>(workspace) + (arguments.parts > 1 ? blocks * num_experts : 0);
    const auto on = static_cast<hipStream_t>(stream);
#define NANOEP_LAUNCH_BALANCE(EACH) \
    balance_loss_kernel<EACH><<<grid_of(blocks), waves * kWave, lds, on>>>(arguments, part_shares, part_counts, loss, counts, tokens)
    NANOEP_BY_EACH(each, NANOEP_LAUNCH_BALANCE)
#undef NANOEP_LAUNCH_BALANCE
    NANOEP_HIP_TRY(hipGetLastError());
    if (arguments.parts > 1) {
        int width = kWave;
        while (width < num_experts && width < kFinishThreads)
            width *= 2;
        balance_finish_kernel<<<grid_of(sequences), kFinishThreads, 0, on>>>(sequences, num_experts, arguments.parts, width, part_shares, part_counts,
                                                                           loss, counts, tokens);
        NANOEP_HIP_TRY(hipGetLastError());
    }
    return NANOEP_OK;
}

int nanoep_balance_loss_backward(const float* grad, const void* logits, int64_t logits_stride, int logits_type, const int64_t* ids,
                                 const int64_t* counts, const int64_t* tokens, const int64_t* sequence_offsets, int64_t num_tokens,
                                 int num_experts, int num_topk, int64_t sequences, int scoring, void* grad_logits, void* stream) {
    using namespace nanoep;
    if (!router_sizes_fit(logits_stride, logits_type, num_tokens, num_experts, num_topk, scoring) || sequences < 1 || sequences > 0x7fffffff ||
        (sequence_offsets == nullptr && sequences != 1))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens == 0)
        return NANOEP_OK;
    if (grad == nullptr || logits == nullptr || ids == nullptr || counts == nullptr || tokens == nullptr || grad_logits == nullptr)
        return NANOEP_ERR_INVALID_ARGUMENT;
    Balance arguments = {logits_of(logits, logits_stride, logits_type, num_experts), ids, sequence_offsets, num_tokens, sequences, num_experts,
                         num_topk, 1, scoring == NANOEP_SIGMOID};
    // a token a wavefront until the sequences alone fill the device, four later
    const int64_t average = (num_tokens + sequences - 1) / sequences;
    arguments.parts = static_cast<int>(std::min<int64_t>(4096, (average + kWavesPerBlock - 1) / kWavesPerBlock));
    const int64_t blocks = (sequences + (sequence_offsets != nullptr ? 1 : 0)) * arguments.parts;
    const auto on = static_cast<hipStream_t>(stream);
#define NANOEP_LAUNCH_BALANCE_BACKWARD(EACH) \
    balance_loss_backward_kernel<EACH><<<grid_of(blocks), kBlockThreads, 0, on>>>(arguments, grad, counts, tokens, grad_logits)
    NANOEP_BY_EACH(each_of(num_experts), NANOEP_LAUNCH_BALANCE_BACKWARD)
#undef NANOEP_LAUNCH_BALANCE_BACKWARD
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

}  // extern "C"
