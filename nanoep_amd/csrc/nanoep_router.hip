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
constexpr uint32_t kNoExpert = 0xffffffffu;

struct Logits {
    const void* data;
    int64_t stride;  // elements from a token to the next
    bool wide;       // fp32, else bf16
};

__device__ __forceinline__ float load_logit(const Logits& logits, int64_t token, int expert) {
    const int64_t at = token * logits.stride + expert;
    if (logits.wide)
        return static_cast<const float*>(logits.data)[at];
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(logits.data)[at]) << 16);
}

// A token's logits over the kLanes lanes that share it: expert i * kLanes + lane in place i, -infinity behind the last expert and
// where there is no token.  Neighbouring lanes read neighbours, whatever the rows' alignment.  All loads are on their way before any is
// looked at: lanes without an expert read the first one's, of a token that there is.
template <int kLanes, int kEach>
__device__ __forceinline__ void load_spread(const Logits& logits, int64_t token, bool here, int experts, float (&out)[kEach]) {
    const int lane = threadIdx.x % kLanes;
    const int64_t row = here ? token * logits.stride : 0;
    if (logits.wide) {
        const float* from = static_cast<const float*>(logits.data) + row;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] = from[i * kLanes + lane < experts ? i * kLanes + lane : 0];
    } else {
        const uint16_t* from = static_cast<const uint16_t*>(logits.data) + row;
        uint16_t narrow[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            narrow[i] = from[i * kLanes + lane < experts ? i * kLanes + lane : 0];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] = __uint_as_float(static_cast<uint32_t>(narrow[i]) << 16);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        out[i] = here && i * kLanes + lane < experts ? out[i] : -INFINITY;
}

template <int kLanes, int kEach>
__device__ __forceinline__ void store_spread(void* out, bool wide, int64_t token, bool here, int experts, const float (&v)[kEach]) {
    const int lane = threadIdx.x % kLanes, mine = here ? experts : 0;
    const int64_t row = here ? token * experts : 0;
    if (wide) {
        float* to = static_cast<float*>(out) + row;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i * kLanes + lane < mine)
                to[i * kLanes + lane] = v[i];
    } else {
        uint16_t* to = static_cast<uint16_t*>(out) + row;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i * kLanes + lane < mine)
                to[i * kLanes + lane] = static_cast<uint16_t>(to_bf16_pair(v[i], 0.0f));
    }
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
__device__ __forceinline__ float value_of(uint32_t key) {
    if (key == 0)
        return -INFINITY;
    return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);  // all ones: a NaN
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

// K rounds over a token's keys: the largest of all, the lowest expert that has it.  chosen_expert, chosen_key: the token's in LDS.
template <int kLanes, int kEach, class Key>
__device__ __forceinline__ void choose_in_turn(Key (&key)[kEach], int rounds, uint32_t* chosen_expert, Key* chosen_key) {
    const uint32_t lane = threadIdx.x % kLanes;
    for (int round = 0; round < rounds; ++round) {
        Key best = key[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i)
            best = key[i] > best ? key[i] : best;
        const Key top = largest_key<kLanes>(best);
        uint32_t expert = kNoExpert;
        if (best == top) {
#pragma unroll
            for (int i = kEach - 1; i >= 0; --i)
                expert = key[i] == top ? i * kLanes + lane : expert;
        }
        // more lanes than tokens have theirs: equal keys
        uint32_t winner = expert;
        if (__popcll(__ballot(best == top)) > kWave / kLanes)
            winner = lanes_min<kLanes>(expert);
        if (expert == winner && best == top) {
            chosen_expert[round] = top != 0 ? expert : kNoExpert;
            chosen_key[round] = top;
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                key[i] = i * kLanes + lane == expert ? 0 : key[i];
        }
    }
    wavefront_sync();
}

// Of the largest keys of the lanes that share a token, the K-th largest: a bound that K keys reach, and few more (spread over 16 lanes,
// K = 8: 11 on average); 0 if fewer lanes have any.  maxima: LDS of the token.
template <int kLanes, int kEach>
__device__ __forceinline__ uint32_t bound_of(const uint32_t (&key)[kEach], int topk, uint32_t* maxima) {
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < kEach; ++i)
        best = key[i] > best ? key[i] : best;
    maxima[threadIdx.x % kLanes] = best;
    wavefront_sync();
    int ahead = 0;
#pragma unroll
    for (int j = 0; j < kLanes; ++j)
        ahead += maxima[j] > best ? 1 : 0;
    return lanes_min<kLanes>(ahead < topk ? best : 0xffffffffu);
}

// Hands every expert whose key reaches the bound to `put`, with places from 0 on that go up lane by lane; others get the place `none`.
// Returns their number; nothing is handed out where some token of the wavefront has more than `none` of them.
template <int kLanes, int kEach, class Put>
__device__ __forceinline__ uint32_t list_candidates(const uint32_t (&key)[kEach], uint32_t bound, uint32_t none, uint32_t& most, Put put) {
    bound = bound > 0 ? bound : 1;
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        mine += key[i] >= bound ? 1 : 0;
    uint32_t at = lanes_before<kLanes>(mine);
    const uint32_t number = lanes_max<kLanes>(at + mine);
    most = __builtin_amdgcn_readfirstlane(lanes_max<kWave>(number));
    if (most <= none) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const bool in = key[i] >= bound;
            put(in ? at : none, i);
            at += in ? 1 : 0;
        }
        wavefront_sync();
    }
    return number;
}

// Strikes out the experts of all groups but the best ones, a group being as good as the sum of its two largest values.  The keys go
// through LDS ([kLanes * kEach] of the token), where lanes share out every group to find the two; the groups' sums go through it too, and
// every group counts how many are ahead of it.  Returns how far the last group that was kept is above the first that was not.
template <int kLanes, int kEach, class Key>
__device__ __forceinline__ auto keep_groups(Key (&key)[kEach], const Route& a, Key* keys) {
    const int lane = threadIdx.x % kLanes, groups = a.groups, size = a.experts / groups;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        keys[i * kLanes + lane] = key[i];
    wavefront_sync();
    int width = 1;  // lanes from a part of a group to the next: a power of two
    while (width < groups)
        width *= 2;
    const int group = lane % width, parts = kLanes / width;
    Key best = 0, second = 0;
    if (group < groups)
#pragma unroll 8
        for (int at = lane / width; at < size; at += parts) {
            const Key other = keys[group * size + at];
            const Key lower = other < best ? other : best;
            second = lower > second ? lower : second;
            best = other > best ? other : best;
        }
    for (int distance = width; distance < kLanes; distance *= 2) {
        const Key other_best = __shfl_xor(best, distance, kWave), other_second = __shfl_xor(second, distance, kWave);
        const Key lower = best < other_best ? best : other_best, higher = second > other_second ? second : other_second;
        best = best > other_best ? best : other_best;
        second = lower > higher ? lower : higher;
    }
    wavefront_sync();
    Key of_group = 0;
    if (lane < groups && best != 0)
        of_group = second == 0 ? best : key_of(value_of(best) + value_of(second));
    if (lane < groups)
        keys[lane] = of_group;
    wavefront_sync();
    int ahead = 0;
#pragma unroll 8
    for (int other = 0; other < groups; ++other) {
        const Key against = keys[other];
        ahead += against > of_group || (against == of_group && other < lane) ? 1 : 0;
    }
    const bool kept = lane < groups && ahead < a.topk_groups;
    const uint64_t open = lanes_where<kLanes>(kept && of_group != 0);
    const Key last = ~largest_key<kLanes>(kept ? ~of_group : Key{0}), first_out = largest_key<kLanes>(lane < groups && !kept ? of_group : Key{0});
    // (a quotient of the middle of an expert's place: never near a whole number)
    const float per_group = 1.0f / static_cast<float>(size);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int expert = i * kLanes + lane;
        const int of = static_cast<int>((static_cast<float>(expert) + 0.5f) * per_group);
        const bool stays = kLanes == kWave ? open >> (of & 63) & 1 : static_cast<uint32_t>(open) >> (of & 31) & 1;
        key[i] = stays && expert < a.experts ? key[i] : 0;
    }
    return value_of(last) - value_of(first_out);
}

// Weights of the choices, lane k with choice k, and both to memory.  largest, total: of the softmax over all experts, if the weights
// are that; broken: it has a NaN or an infinity, so that all of them are NaN.
template <int kLanes>
__device__ __forceinline__ void store_choices(const Route& a, int64_t token, uint32_t expert, float logit, float largest, float total, bool broken) {
    const int lane = threadIdx.x % kLanes;
    const bool valid = expert != kNoExpert;
    float weight;
    if (a.sigmoid) {
        // numerators and denominators times e^-shift, so that their sum is not lost where all scores are tiny
        const float shift = a.normalize ? fminf(lanes_max<kLanes>(valid ? logit : -INFINITY), 0.0f) : 0.0f;
        weight = expf(fminf(logit, 0.0f) - shift) / (1.0f + expf(-fabsf(logit)));
        if (logit != logit)
            weight = logit;
    } else {
        if (a.normalize)
            largest = lanes_max<kLanes>(valid ? logit : -INFINITY);
        weight = broken ? NAN : expf(logit - largest);
    }
    weight = valid ? weight : 0.0f;
    if (a.normalize)
        total = lanes_sum<kLanes>(weight);
    if (a.normalize || !a.sigmoid)
        weight = valid ? weight / total : 0.0f;
    if (token < a.tokens && lane < a.topk) {
        a.ids[token * a.topk + lane] = valid ? static_cast<int64_t>(expert) : -1;
        a.weights[token * a.topk + lane] = weight * a.scale;
    }
}

// The largest logit (0 where there is none), and the sum of e^(logit - largest).
template <int kLanes, int kEach>
__device__ __forceinline__ void softmax_of(const float (&logit)[kEach], float (&exponential)[kEach], float& largest, float& total) {
    largest = -INFINITY;
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        largest = fmaxf(largest, logit[i]);
    largest = lanes_max<kLanes>(largest);
    largest = largest == -INFINITY ? 0.0f : largest;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        exponential[i] = expf(logit[i] - largest);
        total += exponential[i];
    }
    total = lanes_sum<kLanes>(total);
}

// Experts by their logits; kLanes neighbouring lanes a token, its experts spread over them.  With few experts a lane in K rounds; else
// those that reach a bound that K of them reach go to a list, and each counts how many of the list are ahead of it.
template <int kLanes, int kEach>
__global__ void __launch_bounds__(kBlockThreads) route_topk_kernel(const Route a) {
    constexpr int kTokens = kBlockThreads / kLanes, kListed = 2 * kLanes;
    constexpr bool kList = kEach >= 8;
    __shared__ uint32_t all_experts[kTokens][kLanes], all_keys[kTokens][kLanes];
    __shared__ uint64_t all_lists[kTokens][kList ? kListed + 1 : 1];  // key, then its expert's complement: larger is earlier
    const int lane = threadIdx.x % kLanes, place = threadIdx.x / kLanes;
    const int64_t token = workgroup_number() * (blockDim.x / kLanes) + place;
    const bool routed = token < a.tokens && (a.mask == nullptr || a.mask[token] != 0);
    uint32_t *experts = all_experts[place], *keys = all_keys[place];

    float logit[kEach], largest = 0.0f, total = 0.0f;
    load_spread<kLanes, kEach>(a.logits, token, routed, a.experts, logit);
    if (!a.sigmoid && !a.normalize) {
        float exponential[kEach];
        softmax_of<kLanes, kEach>(logit, exponential, largest, total);
    }
    uint32_t key[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        key[i] = key_of(logit[i]);
    bool listed = false;
    if constexpr (kList) {
        uint64_t* list = all_lists[place];
        list[lane] = list[kLanes + lane] = 0;
        const uint32_t bound = bound_of<kLanes, kEach>(key, a.topk, keys);
        uint32_t most;
        const uint32_t number = list_candidates<kLanes, kEach>(key, bound, kListed, most, [&](uint32_t at, int i) {
            list[at] = static_cast<uint64_t>(key[i]) << 32 | ~static_cast<uint32_t>(i * kLanes + lane);
        });
        listed = most <= kListed;
        if (listed) {
            const uint64_t one = list[lane], other = list[kLanes + lane];
            int ahead = 0, other_ahead = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < most; ++j) {
                const uint64_t against = list[j];
                ahead += against > one ? 1 : 0;
                other_ahead += against > other ? 1 : 0;
            }
            if (lane >= static_cast<int>(number))
                experts[lane] = kNoExpert;
            if (one != 0 && ahead < a.topk) {
                experts[ahead] = ~static_cast<uint32_t>(one);
                keys[ahead] = static_cast<uint32_t>(one >> 32);
            }
            if (other != 0 && other_ahead < a.topk) {
                experts[other_ahead] = ~static_cast<uint32_t>(other);
                keys[other_ahead] = static_cast<uint32_t>(other >> 32);
            }
            wavefront_sync();
        }
    }
    if (!listed)  // (or many equal keys, or all of the largest in a few lanes)
        choose_in_turn<kLanes, kEach>(key, a.topk, experts, keys);
    uint32_t expert = kNoExpert;
    float chosen = 0.0f;
    if (lane < a.topk)
        expert = experts[lane];
    if (expert != kNoExpert)
        chosen = value_of(keys[lane]);
    store_choices<kLanes>(a, token, expert, chosen, largest, total, false);
}

// An expert's value in 64 bits.
__device__ __forceinline__ double value_of_expert(const Route& a, float logit, float bias, float largest, double total) {
    double value = exp(a.sigmoid ? -static_cast<double>(logit) : static_cast<double>(logit) - largest);
    if (a.sigmoid)
        value = 1.0 / (1.0 + value);
    else if (a.bias != nullptr)  // (without one the sum is nothing but a common factor)
        value /= total;
    return value + bias;
}

// A token's choice by values in 64 bits throughout, by a whole wavefront; the choices and their logits go to LDS.
template <int kEach>
__device__ __forceinline__ void choose_by_value(const Route& a, int64_t token, uint32_t* experts, float* logits, uint64_t* keys) {
    const int lane = threadIdx.x % kWave;
    __shared__ uint64_t all_chosen[kWavesPerBlock][kMaxTopk];
    float logit[kEach], largest = -INFINITY;
    load_spread<kWave, kEach>(a.logits, token, true, a.experts, logit);
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        largest = fmaxf(largest, logit[i]);
    largest = lanes_max<kWave>(largest);
    largest = largest == -INFINITY ? 0.0f : largest;
    double total = 0.0;
    if (!a.sigmoid && a.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            total += exp(static_cast<double>(logit[i]) - largest);
        total = lanes_sum<kWave>(total);
    }
    uint64_t key[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int expert = i * kWave + lane;
        const float bias = a.bias != nullptr && expert < a.experts ? a.bias[expert] : 0.0f;
        key[i] = logit[i] == -INFINITY ? 0 : key_of(value_of_expert(a, logit[i], bias, largest, total));
    }
    if (a.groups > 1)
        keep_groups<kWave, kEach>(key, a, keys);
    choose_in_turn<kWave, kEach>(key, a.topk, experts, all_chosen[threadIdx.x / kWave]);
    if (lane < a.topk && experts[lane] != kNoExpert)
        logits[lane] = load_logit(a.logits, token, experts[lane]);
    wavefront_sync();
}

// 32-bit words of LDS that a wavefront has for the keys of its tokens, or for one token's of 64 bits.
constexpr int key_words(int lanes, int each) { return kWave * (lanes == kWave ? 2 * each : each > 2 ? each : 2); }

// Experts by their values: scores plus bias, and groups.  Values in fp32, with a bound on their error, find the groups and list
// those experts that can be among the first K; the values of the list, one or two a lane, are then computed in 64 bits, and each
// counts how many are ahead of it.  A token whose groups fp32 cannot tell apart, or whose list is too long (all values equal), is done
// again in 64 bits throughout, by its whole wavefront.
template <int kLanes, int kEach>
__global__ void __launch_bounds__(kBlockThreads) route_values_kernel(const Route a) {
    constexpr int kTokens = kBlockThreads / kLanes, kListed = 2 * kLanes;
    struct alignas(16) Candidate {
        uint64_t key;
        uint32_t expert;
        float logit;
    };
    __shared__ uint32_t all_experts[kTokens][kLanes], all_maxima[kTokens][kLanes];
    __shared__ float all_logits[kTokens][kLanes];
    __shared__ Candidate all_lists[kTokens][kListed + 1];
    extern __shared__ uint64_t all_keys[];  // key_words of every wavefront, for groups
    const int lane = threadIdx.x % kLanes, place = threadIdx.x / kLanes;
    uint32_t* keys = reinterpret_cast<uint32_t*>(all_keys) + threadIdx.x / kWave * key_words(kLanes, kEach);
    const int64_t token = workgroup_number() * (blockDim.x / kLanes) + place;
    const bool routed = token < a.tokens && (a.mask == nullptr || a.mask[token] != 0);
    uint32_t* experts = all_experts[place];
    float* logits = all_logits[place];
    Candidate* list = all_lists[place];

    float logit[kEach], bias[kEach], value[kEach], largest = 0.0f, total = 0.0f;
    if (a.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            bias[i] = a.bias[i * kLanes + lane < a.experts ? i * kLanes + lane : 0];
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            bias[i] = 0.0f;
    }
    load_spread<kLanes, kEach>(a.logits, token, routed, a.experts, logit);

    // What a value is off by: `off`, and `part` of itself.  A sigmoid's argument is rounded by 1.5 l 2^-24, of which s (1 - s) is left; with the
    // exponential, a sum and a reciprocal that is 5 * 2^-24 at most.  A softmax's share: 2^-17 of the largest (the sum's terms have
    // arguments that are rounded by (1 + log E) 2^-24 on average, and go through 70 additions).  The sum with the bias is rounded.
    // Without a bias, where a softmax is compared by its numerators: parts of themselves, with arguments of up to 88.
    float off = 0.0f, part = 0x1p-16f;
    if (a.sigmoid)
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            value[i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(logit[i] * -1.44269504f));
    else
        softmax_of<kLanes, kEach>(logit, value, largest, total);
    if (a.bias != nullptr) {
        const float factor = a.sigmoid ? 1.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            value[i] = fmaf(value[i], factor, bias[i]);
        off = a.sigmoid ? 0x1.4p-22f : 0x1p-17f * factor;
        part = 0x1p-22f;
    }
    uint32_t key[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        key[i] = logit[i] == -INFINITY ? 0 : key_of(value[i]);
    bool again = false;
    if (a.groups > 1) {
        float size = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            size = fmaxf(size, key[i] != 0 ? fabsf(value[i]) : 0.0f);
        size = lanes_max<kLanes>(size);
        const float margin = keep_groups<kLanes, kEach>(key, a, keys + place % (kWave / kLanes) * kLanes * kEach);
        // Two sums of two, rounded.  Without a bias no value is off by more than the largest one is.
        const float each = a.bias != nullptr ? off : size * (0x1.4p-22f - 0x1.8p-24f * fminf(__log2f(size), 0.0f));
        again = !(margin > 4.0f * each + 0x1p-21f * size);
    }
    uint32_t bound = bound_of<kLanes, kEach>(key, a.topk, all_maxima[place]);
    const float least = value_of(bound);
    if (fabsf(least) < INFINITY)
        bound = key_of(least - 2.0f * off - 4.0f * part * fabsf(least));
    list[lane].key = list[kLanes + lane].key = 0;
    wavefront_sync();
    uint32_t most;
    const uint32_t number = list_candidates<kLanes, kEach>(key, bound, kListed, most, [&](uint32_t at, int i) {
        list[at] = {1 + static_cast<uint64_t>(__float_as_uint(bias[i])), static_cast<uint32_t>(i * kLanes + lane), logit[i]};
    });
    again = again || number > kListed;
    double wide_total = 0.0;
    if (!a.sigmoid && a.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            wide_total += exp(static_cast<double>(logit[i]) - largest);
        wide_total = lanes_sum<kLanes>(wide_total);
    }
    if (most <= kListed) {
        Candidate own[2] = {list[lane], list[kLanes + lane]};
        wavefront_sync();
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            if (which == 1 && most <= kLanes)
                break;
            if (own[which].key != 0) {
                own[which].key = key_of(value_of_expert(a, own[which].logit, __uint_as_float(static_cast<uint32_t>(own[which].key - 1)), largest, wide_total));
                list[which * kLanes + lane].key = own[which].key;
            }
        }
        wavefront_sync();
        int ahead[2] = {0, 0};
#pragma unroll 4
        for (uint32_t j = 0; j < most; ++j) {
            const Candidate against = list[j];
#pragma unroll
            for (int which = 0; which < 2; ++which)
                ahead[which] += against.key > own[which].key || (against.key == own[which].key && against.expert < own[which].expert) ? 1 : 0;
        }
        if (lane >= static_cast<int>(number))
            experts[lane] = kNoExpert;
#pragma unroll
        for (int which = 0; which < 2; ++which)
            if (own[which].key != 0 && ahead[which] < a.topk) {
                experts[ahead[which]] = own[which].expert;
                logits[ahead[which]] = own[which].logit;
            }
        wavefront_sync();
    } else {
        again = true;
    }
    for (uint64_t todo = __ballot(again && routed && lane == 0); todo != 0; todo &= todo - 1) {
        const int first = __ffsll(static_cast<unsigned long long>(todo)) - 1, other = threadIdx.x / kWave * (kWave / kLanes) + first / kLanes;
        choose_by_value<(kLanes * kEach + kWave - 1) / kWave>(a, workgroup_number() * (blockDim.x / kLanes) + other, all_experts[other], all_logits[other],
                                                             reinterpret_cast<uint64_t*>(keys));
    }
    uint32_t expert = kNoExpert;
    float chosen = 0.0f;
    if (routed && lane < a.topk)
        expert = experts[lane];
    if (expert != kNoExpert)
        chosen = logits[lane];
    store_choices<kLanes>(a, token, expert, chosen, largest, total, total != total);
}

// ------------------------------------------------------------------ gradients of a token's scores

// Every expert's share of its token: softmax, or sigmoid over its sum.  rest: what is left of its sigmoid to one (softmax: 1).
// Experts at -infinity have none; a token of nothing else has no shares.
template <int kLanes, int kEach>
__device__ __forceinline__ void shares_of(const float (&logit)[kEach], bool sigmoid, float (&share)[kEach], float (&rest)[kEach]) {
    float largest = -INFINITY, total = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        largest = fmaxf(largest, logit[i]);
    largest = lanes_max<kLanes>(largest);
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
    total = lanes_sum<kLanes>(total);
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

// kLanes neighbouring lanes a token, lane k with its choice k.  With the gradients g_k of the weights w_k, c = scale:
//   softmax over the choices          dl_k = w_k (g_k - sum_j g_j w_j / c)
//   softmax over all experts          dl_e = p_e ([e is chosen] c g_e - sum_j c g_j p_j)
//   sigmoids over the choices' sum    dl_k = w_k (1 - s_k) (g_k - sum_j g_j w_j / c)
//   sigmoids                          dl_k = c g_k s_k (1 - s_k)
// and zero for every other expert.  Only the second reads more than the chosen logits.  An expert that is named twice has both
// gradients: its first choice adds them up, in their order.  Choices become experts' through a row in LDS.
template <int kLanes, int kEach>
__global__ void __launch_bounds__(kBlockThreads) route_topk_backward_kernel(const RouteBackward a) {
    __shared__ float2 all_choices[kBlockThreads / kLanes][kLanes];  // expert's bits, gradient
    extern __shared__ float rows[];                                // [tokens][kLanes * kEach]
    const int lane = threadIdx.x % kLanes, place = threadIdx.x / kLanes;
    const int64_t token = workgroup_number() * (blockDim.x / kLanes) + place;
    const bool here = token < a.tokens;
    const bool over_all = !a.sigmoid && !a.normalize;
    float* row = rows + static_cast<int64_t>(place) * kLanes * kEach;
    int64_t named = -1;
    float g = 0.0f, logit = -INFINITY;
    if (here && lane < a.topk) {
        named = a.ids[token * a.topk + lane];
        g = a.grad[token * a.topk + lane];
    }
    const bool valid = named >= 0 && named < a.experts;
    const int expert = valid ? static_cast<int>(named) : -1;
    if (valid && !over_all)
        logit = load_logit(a.logits, token, expert);
    g = valid ? g * a.scale : 0.0f;

    float share[kEach], out[kEach];
    if (over_all) {
        float rest[kEach];
        load_spread<kLanes, kEach>(a.logits, token, here, a.experts, out);
        shares_of<kLanes, kEach>(out, false, share, rest);
    } else if (a.normalize) {
        const float largest = lanes_max<kLanes>(logit);
        float score = 0.0f, rest = 1.0f;
        if (a.sigmoid) {
            const float tail = expf(-fabsf(logit)), inverse = 1.0f / (1.0f + tail);
            score = logit != logit ? logit : expf(fminf(logit, 0.0f) - fminf(largest, 0.0f)) * inverse;
            rest = logit >= 0.0f ? tail * inverse : inverse;
        } else {
            score = expf(logit - largest);
        }
        score = valid ? score : 0.0f;
        const float total = lanes_sum<kLanes>(score);
        score = valid ? score / total : 0.0f;
        g = score * rest * (g - lanes_sum<kLanes>(score * g));
    } else {
        const float tail = expf(-fabsf(logit)), inverse = 1.0f / (1.0f + tail);
        g = g * tail * inverse * inverse;
    }
    all_choices[place][lane] = make_float2(__int_as_float(expert), g);
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        row[i * kLanes + lane] = 0.0f;
    wavefront_sync();
    float sum = 0.0f;
    bool first = true;
    for (int k = 0; k < a.topk; ++k) {
        const float2 other = all_choices[place][k];
        const bool same = __float_as_int(other.x) == expert;
        sum += same ? other.y : 0.0f;
        first = first && !(same && k < lane);
    }
    if (valid && first)
        row[expert] = sum;
    wavefront_sync();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        out[i] = row[i * kLanes + lane];
    if (over_all) {
        float along = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            along = fmaf(out[i], share[i], along);
        along = lanes_sum<kLanes>(along);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] = share[i] * (out[i] - along);
    }
    store_spread<kLanes, kEach>(a.grad_logits, a.logits.wide, token, here, a.experts, out);
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

// Whether the token that kLanes lanes share has a choice; each one is given to `count`, once.
template <int kLanes, class Count>
__device__ __forceinline__ bool has_choice(const Balance& a, int64_t token, bool here, Count count) {
    bool any = false;
    for (int k = threadIdx.x % kLanes; k < a.topk; k += kLanes) {
        const int64_t named = here ? a.ids[token * a.topk + k] : -1;
        if (named >= 0 && named < a.experts) {
            any = true;
            count(static_cast<int>(named));
        }
    }
    return lanes_where<kLanes>(any) != 0;
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

// A workgroup a part of a sequence: kLanes lanes a token at a time, which keep their experts' sums of shares in registers;
// choices are counted in LDS (whole numbers: any order gives the same).  The sums of a wavefront's tokens, then those of the wavefronts
// are added in a fixed order.  A sequence of one part is finished here, others leave a row of sums to balance_finish_kernel.
template <int kLanes, int kEach>
__global__ void __launch_bounds__(balance_waves(kEach) * kWave) balance_loss_kernel(const Balance a, float* __restrict__ part_shares,  // [S * parts][E]
                                                                                    int* __restrict__ part_counts,  // [S * parts][E + 1]
                                                                                    float* __restrict__ loss, int64_t* __restrict__ counts,
                                                                                    int64_t* __restrict__ tokens) {
    constexpr int kWidth = kLanes * kEach, kWaves = balance_waves(kEach);
    __shared__ float sums[kWaves / 2 * kWidth];
    __shared__ int chosen[kWidth];
    __shared__ float place[kWaves];
    __shared__ int live_tokens;
    const int64_t block = workgroup_number();
    if (block >= a.sequences * a.parts)
        return;
    const int64_t sequence = block / a.parts;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kLanes;
    for (int e = threadIdx.x; e < kWidth; e += kWaves * kWave)
        chosen[e] = 0;
    if (threadIdx.x == 0)
        live_tokens = 0;
    __syncthreads();

    int64_t from, to;
    part_of(a, sequence, static_cast<int>(block - sequence * a.parts), from, to);
    float own[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        own[i] = 0.0f;
    int number = 0;
    constexpr int kTokens = kWaves * kWave / kLanes;
    for (int64_t first = from; first < to; first += kTokens) {
        const int64_t token = first + threadIdx.x / kLanes;
        const bool here = token < to;
        float logit[kEach], share[kEach], rest[kEach];
        load_spread<kLanes, kEach>(a.logits, token, here, a.experts, logit);
        const bool live = has_choice<kLanes>(a, token, here, [&](int expert) { atomicAdd(&chosen[expert], 1); });
        number += live ? 1 : 0;
        shares_of<kLanes, kEach>(logit, a.sigmoid, share, rest);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            own[i] += live ? share[i] : 0.0f;
    }
    if (lane == 0 && number > 0)
        atomicAdd(&live_tokens, number);
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        own[i] = groups_sum<kLanes>(own[i]);
    const bool writes = threadIdx.x % kWave < kLanes;
    for (int half = kWaves / 2; half > 0; half /= 2) {
        if (wave >= half && wave < 2 * half && writes)
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                sums[(wave - half) * kWidth + i * kLanes + lane] = own[i];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                own[i] += sums[wave * kWidth + i * kLanes + lane];
        __syncthreads();
    }
    if (wave == 0 && writes)
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            sums[i * kLanes + lane] = own[i];
    __syncthreads();
    if (a.parts > 1) {
        for (int e = threadIdx.x; e < a.experts; e += kWaves * kWave) {
            part_shares[block * a.experts + e] = sums[e];
            part_counts[block * (a.experts + 1) + e] = chosen[e];
        }
        if (threadIdx.x == 0)
            part_counts[block * (a.experts + 1) + a.experts] = live_tokens;
        return;
    }
    finish_sequence(sequence, a.experts, sums, chosen, live_tokens, loss, counts, tokens, place);
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
template <int kLanes, int kEach>
__global__ void __launch_bounds__(kBlockThreads) balance_loss_backward_kernel(const Balance a, const float* __restrict__ grad,  // [S]
                                                                              const int64_t* __restrict__ counts, const int64_t* __restrict__ tokens,
                                                                              void* __restrict__ grad_logits) {
    constexpr int kTokens = kBlockThreads / kLanes;
    const int64_t block = workgroup_number();
    const int64_t sequence = block / a.parts;
    const int part = static_cast<int>(block - sequence * a.parts);
    const int lane = threadIdx.x % kLanes, place = threadIdx.x / kLanes;
    float factor[kEach], out[kEach];
    if (sequence >= a.sequences) {
        if (sequence > a.sequences || a.offsets == nullptr)
            return;
        const int64_t begin = a.offsets[0], end = a.offsets[a.sequences];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] = 0.0f;
        for (int64_t token = static_cast<int64_t>(part) * kTokens + place; token < a.tokens; token += static_cast<int64_t>(a.parts) * kTokens)
            store_spread<kLanes, kEach>(grad_logits, a.logits.wide, token, token < begin || token >= end, a.experts, out);
        return;
    }
    int64_t from, to;
    part_of(a, sequence, part, from, to);
    if (from >= to)
        return;
    float number = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int expert = i * kLanes + lane;
        factor[i] = expert < a.experts ? static_cast<float>(counts[sequence * a.experts + expert]) : 0.0f;
        number += factor[i];
    }
    number = lanes_sum<kLanes>(number);
    const int64_t live_tokens = tokens[sequence];
    const float each = live_tokens > 0 && number > 0.0f ? grad[sequence] * static_cast<float>(a.experts) / number / static_cast<float>(live_tokens) : 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        factor[i] *= each;
    for (int64_t first = from; first < to; first += kTokens) {
        const int64_t token = first + place;
        const bool here = token < to;
        float logit[kEach], share[kEach], rest[kEach], along = 0.0f;
        load_spread<kLanes, kEach>(a.logits, token, here, a.experts, logit);
        const bool live = has_choice<kLanes>(a, token, here, [](int) {});
        shares_of<kLanes, kEach>(logit, a.sigmoid, share, rest);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            along = fmaf(factor[i], share[i], along);
        along = lanes_sum<kLanes>(along);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] = live ? share[i] * rest[i] * (factor[i] - along) : 0.0f;
        store_spread<kLanes, kEach>(grad_logits, a.logits.wide, token, here, a.experts, out);
    }
}

// ------------------------------------------------------------------ launches

// Lanes a token, and experts a lane.
struct Spread {
    int lanes, each;
};
// At least `needed` lanes, 16 experts a lane at most as long as that leaves a wavefront several tokens.
Spread spread_of(int experts, int needed) {
    Spread spread = {8, 1};
    while (spread.lanes < needed)
        spread.lanes *= 2;
    while (spread.lanes * spread.each < experts) {
        const int most = spread.lanes == 8 ? 4 : 16;
        if (spread.each < most || spread.lanes == kWave)
            spread.each *= 2;
        else
            spread.lanes *= 2, spread.each /= 2;
    }
    return spread;
}

// For the router's choices: a lane for each of them, and 32 while that is no more than four wavefronts a SIMD, which have little work each
// then (us with 16, 32 and 64 lanes of 256 experts, a bias: 1 token 5.7, 4.8, 4.4; 4096 tokens 8.4, 6.9, 7.8; 32768 tokens 19.2, 22.4, 41.6).
Spread spread_for_choices(int64_t num_tokens, int experts, int needed) {
    return spread_of(experts, std::max(needed, num_tokens <= int64_t{32} * current_topology(current_tuning()).cus ? 32 : 1));
}

// CALL(lanes, experts a lane) for a Spread of 8 lanes or more, of 16 or more, and of whatever number suits the experts.
#define NANOEP_BY_SPREAD(SPREAD, CALL)              \
    switch ((SPREAD).lanes * 100 + (SPREAD).each) { \
        case 801:                                   \
            CALL(8, 1);                             \
            break;                                  \
        case 802:                                   \
            CALL(8, 2);                             \
            break;                                  \
        case 804:                                   \
            CALL(8, 4);                             \
            break;                                  \
        case 1601:                                  \
            CALL(16, 1);                            \
            break;                                  \
        case 1602:                                  \
            CALL(16, 2);                            \
            break;                                  \
        case 1604:                                  \
            CALL(16, 4);                            \
            break;                                  \
        case 1608:                                  \
            CALL(16, 8);                            \
            break;                                  \
        case 1616:                                  \
            CALL(16, 16);                           \
            break;                                  \
        case 3201:                                  \
            CALL(32, 1);                            \
            break;                                  \
        case 3202:                                  \
            CALL(32, 2);                            \
            break;                                  \
        case 3204:                                  \
            CALL(32, 4);                            \
            break;                                  \
        case 3208:                                  \
            CALL(32, 8);                            \
            break;                                  \
        case 3216:                                  \
            CALL(32, 16);                           \
            break;                                  \
        case 6401:                                  \
            CALL(64, 1);                            \
            break;                                  \
        case 6402:                                  \
            CALL(64, 2);                            \
            break;                                  \
        case 6404:                                  \
            CALL(64, 4);                            \
            break;                                  \
        case 6408:                                  \
            CALL(64, 8);                            \
            break;                                  \
        case 6416:                                  \
            CALL(64, 16);                           \
            break;                                  \
        case 6432:                                  \
            CALL(64, 32);                           \
            break;                                  \
        default:                                    \
            CALL(64, 64);                           \
            break;                                  \
    }
#define NANOEP_BY_SPREAD_FROM_16(SPREAD, CALL)      \
    switch ((SPREAD).lanes * 100 + (SPREAD).each) { \
        case 1601:                                  \
            CALL(16, 1);                            \
            break;                                  \
        case 1602:                                  \
            CALL(16, 2);                            \
            break;                                  \
        case 1604:                                  \
            CALL(16, 4);                            \
            break;                                  \
        case 1608:                                  \
            CALL(16, 8);                            \
            break;                                  \
        case 1616:                                  \
            CALL(16, 16);                           \
            break;                                  \
        case 3201:                                  \
            CALL(32, 1);                            \
            break;                                  \
        case 3202:                                  \
            CALL(32, 2);                            \
            break;                                  \
        case 3204:                                  \
            CALL(32, 4);                            \
            break;                                  \
        case 3208:                                  \
            CALL(32, 8);                            \
            break;                                  \
        case 3216:                                  \
            CALL(32, 16);                           \
            break;                                  \
        case 6401:                                  \
            CALL(64, 1);                            \
            break;                                  \
        case 6402:                                  \
            CALL(64, 2);                            \
            break;                                  \
        case 6404:                                  \
            CALL(64, 4);                            \
            break;                                  \
        case 6408:                                  \
            CALL(64, 8);                            \
            break;                                  \
        case 6416:                                  \
            CALL(64, 16);                           \
            break;                                  \
        case 6432:                                  \
            CALL(64, 32);                           \
            break;                                  \
        default:                                    \
            CALL(64, 64);                           \
            break;                                  \
    }
#define NANOEP_BY_FREE_SPREAD(SPREAD, CALL)         \
    switch ((SPREAD).lanes * 100 + (SPREAD).each) { \
        case 801:                                   \
            CALL(8, 1);                             \
            break;                                  \
        case 802:                                   \
            CALL(8, 2);                             \
            break;                                  \
        case 804:                                   \
            CALL(8, 4);                             \
            break;                                  \
        case 1604:                                  \
            CALL(16, 4);                            \
            break;                                  \
        case 1608:                                  \
            CALL(16, 8);                            \
            break;                                  \
        case 1616:                                  \
            CALL(16, 16);                           \
            break;                                  \
        case 3216:                                  \
            CALL(32, 16);                           \
            break;                                  \
        case 6416:                                  \
            CALL(64, 16);                           \
            break;                                  \
        case 6432:                                  \
            CALL(64, 32);                           \
            break;                                  \
        default:                                    \
            CALL(64, 64);                           \
            break;                                  \
    }

bool router_sizes_fit(int64_t stride, int logits_type, int64_t num_tokens, int experts, int topk, int scoring) {
    return num_tokens >= 0 && num_tokens <= 0x7fffffff / kMaxTopk && experts >= 1 && experts <= kMostExperts && topk >= 1 && topk <= kMaxTopk &&
           stride >= experts && stride <= int64_t{1} << 31 && (logits_type == NANOEP_BF16 || logits_type == NANOEP_FP32) &&
           (scoring == NANOEP_SOFTMAX || scoring == NANOEP_SIGMOID);
}

Logits logits_of(const void* data, int64_t stride, int type) { return {data, stride, type == NANOEP_FP32}; }

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
    const Route arguments = {logits_of(logits, logits_stride, logits_type), bias, mask, ids, weights, num_tokens, num_experts, num_topk,
                             topk_groups < groups ? groups : 1, topk_groups, scoring == NANOEP_SIGMOID, normalize != 0, scale};
    const bool by_value = bias != nullptr || arguments.groups > 1;
    const Spread spread = spread_for_choices(num_tokens, num_experts, std::max({num_topk, arguments.groups, by_value ? 16 : 1}));
    const int threads = spread.each > 16 ? kWave : kBlockThreads;  // (LDS)
    const size_t lds = arguments.groups > 1 ? static_cast<size_t>(threads / kWave) * key_words(spread.lanes, spread.each) * sizeof(uint32_t) : 0;
    const int tokens = threads / spread.lanes;
    const dim3 grid = grid_of((num_tokens + tokens - 1) / tokens);
    const auto on = static_cast<hipStream_t>(stream);
#define NANOEP_LAUNCH_ROUTE(LANES, EACH) route_topk_kernel<LANES, EACH><<<grid, threads, 0, on>>>(arguments)
#define NANOEP_LAUNCH_VALUES(LANES, EACH) route_values_kernel<LANES, EACH><<<grid, threads, lds, on>>>(arguments)
    if (by_value)
        NANOEP_BY_SPREAD_FROM_16(spread, NANOEP_LAUNCH_VALUES)
    else
        NANOEP_BY_SPREAD(spread, NANOEP_LAUNCH_ROUTE)
#undef NANOEP_LAUNCH_ROUTE
#undef NANOEP_LAUNCH_VALUES
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
    const RouteBackward arguments = {logits_of(logits, logits_stride, logits_type), grad, ids, grad_logits, num_tokens, num_experts,
                                     num_topk, scoring == NANOEP_SIGMOID, normalize != 0, scale};
    const Spread spread = spread_for_choices(num_tokens, num_experts, num_topk);
    const int threads = spread.each > 16 ? kWave : kBlockThreads;  // (LDS: 4 bytes an expert)
    const size_t lds = static_cast<size_t>(threads) * spread.each * sizeof(float);
    const int tokens = threads / spread.lanes;
    const dim3 grid = grid_of((num_tokens + tokens - 1) / tokens);
    const auto on = static_cast<hipStream_t>(stream);
#define NANOEP_LAUNCH_ROUTE_BACKWARD(LANES, EACH) route_topk_backward_kernel<LANES, EACH><<<grid, threads, lds, on>>>(arguments)
    NANOEP_BY_SPREAD(spread, NANOEP_LAUNCH_ROUTE_BACKWARD)
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
    const Balance arguments = {logits_of(logits, logits_stride, logits_type), ids, sequence_offsets, num_tokens, sequences, num_experts,
                               num_topk, parts_of(num_tokens, sequences), scoring == NANOEP_SIGMOID};
    if (arguments.parts > 1 && (workspace == nullptr || !aligned16(workspace)))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const Spread spread = spread_of(num_experts, 1);
    const int64_t blocks = sequences * arguments.parts;
    auto* part_shares = static_cast<float*>(workspace);
    auto* part_counts = static_cast<int*>(workspace) + (arguments.parts > 1 ? blocks * num_experts : 0);
    const auto on = static_cast<hipStream_t>(stream);
#define NANOEP_LAUNCH_BALANCE(LANES, EACH)                                                                                        \
    balance_loss_kernel<LANES, EACH><<<grid_of(blocks), balance_waves(EACH) * kWave, 0, on>>>(arguments, part_shares, part_counts, loss, \
                                                                                             counts, tokens)
    NANOEP_BY_FREE_SPREAD(spread, NANOEP_LAUNCH_BALANCE)
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
    Balance arguments = {logits_of(logits, logits_stride, logits_type), ids, sequence_offsets, num_tokens, sequences, num_experts,
                         num_topk, 1, scoring == NANOEP_SIGMOID};
    // two rounds of tokens a workgroup
    const Spread spread = spread_of(num_experts, 1);
    const int64_t average = (num_tokens + sequences - 1) / sequences, each = 2 * kBlockThreads / spread.lanes;
    arguments.parts = static_cast<int>(std::min<int64_t>(4096, (average + each - 1) / each));
    const int64_t blocks = (sequences + (sequence_offsets != nullptr ? 1 : 0)) * arguments.parts;
    const auto on = static_cast<hipStream_t>(stream);
#define NANOEP_LAUNCH_BALANCE_BACKWARD(LANES, EACH) \
    balance_loss_backward_kernel<LANES, EACH><<<grid_of(blocks), kBlockThreads, 0, on>>>(arguments, grad, counts, tokens, grad_logits)
    NANOEP_BY_FREE_SPREAD(spread, NANOEP_LAUNCH_BALANCE_BACKWARD)
#undef NANOEP_LAUNCH_BALANCE_BACKWARD
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

}  // extern "C"
