// The router's choice of experts with its gate weights, the loss that balances the experts, and their gradients.
//
// Scores of a token's logits l over the experts: softmax e^l_e / sum e^l, or sigmoid 1 / (1 + e^-l_e).
// Values that are not rounded the same way everywhere must not decide which expert is chosen: the choice goes by the logits
// themselves, which are in the order of their scores, or, where a bias is added or groups are compared, by scores
// in 64 bits.  Weights, losses and gradients are fp32.

#include <algorithm>
#include <type_traits>

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

// A token's logits over the kLanes lanes that share it: expert i * kLanes + lane in place i.  Neighbouring lanes read neighbours, whatever
// the rows' alignment.  All loads are on their way before any is looked at: lanes without an expert read the first one's, of a token that
// there is.  Rows that fill their lanes, as most do, need neither that nor an address for each place.
template <int kLanes, int kEach, class T>
__device__ __forceinline__ void load_row(const T* from, int experts, uint32_t (&out)[kEach]) {
    const int lane = threadIdx.x % kLanes;
    if (experts == kLanes * kEach) {
        from += lane;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] = from[i * kLanes];
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            out[i] = from[i * kLanes + lane < experts ? i * kLanes + lane : 0];
    }
}
template <int kLanes, int kEach>
__device__ __forceinline__ void load_raw(const Logits& logits, int64_t token, bool here, int experts, uint32_t (&out)[kEach]) {
    const int64_t row = here ? token * logits.stride : 0;
    if (logits.wide)
        load_row<kLanes, kEach>(static_cast<const uint32_t*>(logits.data) + row, experts, out);
    else
        load_row<kLanes, kEach>(static_cast<const uint16_t*>(logits.data) + row, experts, out);
}

// Their values: -infinity behind the last expert and where there is no token.
template <int kLanes, int kEach>
__device__ __forceinline__ void logits_of_raw(const Logits& logits, const uint32_t (&raw)[kEach], bool here, int experts, float (&out)[kEach]) {
    const int lane = threadIdx.x % kLanes, shift = logits.wide ? 0 : 16;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        out[i] = here && i * kLanes + lane < experts ? __uint_as_float(raw[i] << shift) : -INFINITY;
}

template <int kLanes, int kEach>
__device__ __forceinline__ void load_spread(const Logits& logits, int64_t token, bool here, int experts, float (&out)[kEach]) {
    uint32_t raw[kEach];
    load_raw<kLanes, kEach>(logits, token, here, experts, raw);
    logits_of_raw<kLanes, kEach>(logits, raw, here, experts, out);
}

template <int kLanes, int kEach, class Put>
__device__ __forceinline__ void store_row(bool here, int experts, Put put) {
    const int lane = threadIdx.x % kLanes;
    if (experts == kLanes * kEach) {
        if (here)
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                put(i);
    } else {
        const int mine = here ? experts : 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i * kLanes + lane < mine)
                put(i);
    }
}
template <int kLanes, int kEach>
__device__ __forceinline__ void store_spread(void* out, bool wide, int64_t token, bool here, int experts, const float (&v)[kEach]) {
    const int64_t row = (here ? token * experts : 0) + threadIdx.x % kLanes;
    if (wide) {
        float* to = static_cast<float*>(out) + row;
        store_row<kLanes, kEach>(here, experts, [&](int i) { to[i * kLanes] = v[i]; });
    } else {
        uint16_t* to = static_cast<uint16_t*>(out) + row;
        store_row<kLanes, kEach>(here, experts, [&](int i) { to[i * kLanes] = static_cast<uint16_t>(to_bf16_pair(v[i], 0.0f)); });
    }
}

// e^x for x <= 0, good to 2^-22: 2^n times 2 to the rest of x log2 e, with log2 e in two parts.
__device__ __forceinline__ float exp_below(float x) {
    x = x < -200.0f ? -200.0f : x;  // (a NaN stays one)
    const float whole = rintf(x * 0x1.715476p+0f);
    const float rest = fmaf(x, 0x1.4ae0cp-26f, fmaf(x, 0x1.715476p+0f, -whole));
    return ldexpf(__builtin_amdgcn_exp2f(rest), static_cast<int>(whole));
}

// Values as unsigned integers in the same order: 0 for -infinity, which stands for an expert that cannot be chosen, NaN above
// everything, both zeros alike.
constexpr uint32_t kLowestKey = 0x007fffffu;  // of -infinity, ahead of its subtraction
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    const uint32_t key = bits ^ (static_cast<uint32_t>(static_cast<int>(bits) >> 31) | 0x80000000u);
    return v != v ? 0xffffffffu : key - kLowestKey;
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
    const uint32_t bits = key + (key == 0xffffffffu ? 0u : kLowestKey);
    return __uint_as_float(bits >> 31 ? bits & 0x7fffffffu : ~bits);  // all ones: a NaN
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
    int group_size, group_bits;  // experts of a group; the groups' number is 2^group_bits at most
    float per_group;             // 1 / group_size
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

// The same for few keys a lane, which are sorted first, so that a round looks at a lane's first one and moves the others up: with four
// of them, eight rounds and the sort are 150 vector instructions where eight rounds over all are 250.
template <int kLanes, int kEach>
__device__ __forceinline__ void choose_sorted(uint32_t (&key)[kEach], int rounds, uint32_t* chosen_expert, uint32_t* chosen_key) {
    uint32_t expert[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        expert[i] = i * kLanes + threadIdx.x % kLanes;
#pragma unroll
    for (int last = kEach - 1; last > 0; --last)
#pragma unroll
        for (int i = 0; i < last; ++i) {  // neighbours only, so that equal ones stay in their order
            const uint32_t one = key[i], other = key[i + 1], expert_of_one = expert[i], expert_of_other = expert[i + 1];
            key[i] = other > one ? other : one;
            key[i + 1] = other > one ? one : other;
            expert[i] = other > one ? expert_of_other : expert_of_one;
            expert[i + 1] = other > one ? expert_of_one : expert_of_other;
        }
    for (int round = 0; round < rounds; ++round) {
        const uint32_t top = lanes_max<kLanes>(key[0]);
        bool wins = key[0] == top;
        if (__popcll(__ballot(wins)) > kWave / kLanes) {  // more lanes than tokens have theirs: equal keys
            const uint32_t lowest = lanes_min<kLanes>(wins ? expert[0] : kNoExpert);
            wins = wins && expert[0] == lowest;
        }
        if (wins) {
            chosen_expert[round] = top != 0 ? expert[0] : kNoExpert;
            chosen_key[round] = top;
#pragma unroll
            for (int i = 0; i + 1 < kEach; ++i) {
                key[i] = key[i + 1];
                expert[i] = expert[i + 1];
            }
            key[kEach - 1] = 0;
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

// How good a group is, from its two largest values' keys: their sum.
template <class Key>
__device__ __forceinline__ Key key_of_group(Key best, Key second) {
    return best == 0 || second == 0 ? best : key_of(value_of(best) + value_of(second));
}

// The best groups as bits; lane g has group g's key.  Every group counts how many are ahead of it.  keys: LDS of the token, a key a group.
template <int kLanes, class Key>
__device__ __forceinline__ uint64_t best_groups(const Route& a, Key of_group, Key* keys, bool& kept) {
    const int lane = threadIdx.x % kLanes, groups = a.groups;
    if (lane < groups)
        keys[lane] = of_group;
    wavefront_sync();
    int ahead = 0;
#pragma unroll 8
    for (int other = 0; other < groups; ++other) {
        const Key against = keys[other];
        ahead += against > of_group || (against == of_group && other < lane) ? 1 : 0;
    }
    kept = lane < groups && ahead < a.topk_groups;
    return lanes_where<kLanes>(kept && of_group != 0);
}

// A lane's experts' groups: (expert + 1/2) / (experts of a group), rounded down.  (A quotient of the middle of an expert's place is never
// near a whole number.)
template <int kLanes>
struct GroupOf {
    float per_group, first;
    __device__ __forceinline__ explicit GroupOf(const Route& a)
        : per_group(a.per_group), first((static_cast<float>(threadIdx.x % kLanes) + 0.5f) * per_group) {}
    __device__ __forceinline__ uint32_t of_place(int i) const { return static_cast<uint32_t>(fmaf(static_cast<float>(i * kLanes), per_group, first)); }
    __device__ __forceinline__ int of_expert(uint32_t expert) const { return static_cast<int>((static_cast<float>(expert) + 0.5f) * per_group); }
};

// Strikes out the experts of all groups but the open ones.
template <int kLanes, int kEach, class Key>
__device__ __forceinline__ void strike_out(Key (&key)[kEach], const Route& a, uint64_t open) {
    const GroupOf<kLanes> group(a);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if constexpr (kLanes == kWave)
            key[i] = open >> (group.of_place(i) & 63) & 1 ? key[i] : 0;
        else
            key[i] &= static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(open), group.of_place(i), 1));  // (a bit, as all of a word)
    }
}

// The best groups as bits, a group being as good as the sum of its two largest values.  The keys go through LDS ([kLanes * kEach] of the
// token), where lanes share out every group to find the two (lane g then has the second of group g); the groups' sums go through it too.
// margin: how far the last group that was kept is above the first that was not.
template <int kLanes, int kEach, class Key, class Value>
__device__ __forceinline__ uint64_t find_groups(const Key (&key)[kEach], const Route& a, Key* keys, Key& second, Value& margin) {
    const int lane = threadIdx.x % kLanes, groups = a.groups, size = a.group_size;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        keys[i * kLanes + lane] = key[i];
    wavefront_sync();
    const int width = 1 << a.group_bits, group = lane & (width - 1), parts = kLanes >> a.group_bits;  // width: from a part of a group to the next
    Key best = 0;
    second = 0;
    if (group < groups)
#pragma unroll 8
        for (int at = lane >> a.group_bits; at < size; at += parts) {
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
    const Key of_group = lane < groups ? key_of_group(best, second) : 0;
    bool kept;
    const uint64_t open = best_groups<kLanes>(a, of_group, keys, kept);
    const Key last = ~largest_key<kLanes>(kept ? ~of_group : Key{0}), first_out = largest_key<kLanes>(lane < groups && !kept ? of_group : Key{0});
    margin = value_of(last) - value_of(first_out);
    return open;
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
        weight = exp_below(fminf(logit, 0.0f) - shift) / (1.0f + exp_below(-fabsf(logit)));
        if (logit != logit)
            weight = logit;
    } else {
        if (a.normalize)
            largest = lanes_max<kLanes>(valid ? logit : -INFINITY);
        weight = broken ? NAN : exp_below(logit - largest);
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

// The sum over a token's experts of `of` their places, in an order that goes by the experts alone, so that a token has the same sum however many
// lanes it is spread over: every 64th expert in turn, then those of the 64 sums that are farthest apart.
template <int kLanes, int kEach, class Of>
__device__ __forceinline__ auto experts_sum(Of of) {
    constexpr int kHeld = kWave / kLanes < kEach ? kWave / kLanes : kEach;  // of the 64, in a lane
    decltype(of(0)) sum[kHeld];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        sum[i % kHeld] = i < kHeld ? of(i) : sum[i % kHeld] + of(i);
#pragma unroll
    for (int half = kHeld / 2; half > 0; half /= 2)
#pragma unroll
        for (int i = 0; i < half; ++i)
            sum[i] += sum[i + half];
    return lanes_sum_from_afar<kLanes>(sum[0]);
}

// The largest logit (0 where there is none), and the sum of e^(logit - largest).
template <int kLanes, int kEach>
__device__ __forceinline__ void softmax_of(const float (&logit)[kEach], float (&exponential)[kEach], float& largest, float& total) {
    largest = -INFINITY;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        largest = fmaxf(largest, logit[i]);
    largest = lanes_max<kLanes>(largest);
    largest = largest == -INFINITY ? 0.0f : largest;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        exponential[i] = exp_below(logit[i] - largest);
    total = experts_sum<kLanes, kEach>([&](int i) { return exponential[i]; });
}

// Experts by their logits; kLanes neighbouring lanes a token, its experts spread over them.  With few experts a lane in K rounds; else
// those that reach a bound that K of them reach go to a list, and each counts how many of the list are ahead of it.
// Vector instructions and latencies, not bytes: 32768 tokens of 64 experts (12 MB) 6.7 us (350 vector instructions a wavefront of
// four tokens: 90 % of its time), of 256 experts 10.4 (K rounds 16.0; a whole wavefront a token and K rounds 22.2); 4096 of 256 4.2; one
// token 2.8, a launch.
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
            if (lane >= static_cast<int>(number))
                experts[lane] = kNoExpert;
            const auto choose = [&](auto listed_each) {  // one or two of the list a lane
                constexpr int kListedEach = decltype(listed_each)::value;
                uint64_t own[kListedEach];
                int ahead[kListedEach] = {};
#pragma unroll
                for (int which = 0; which < kListedEach; ++which)
                    own[which] = list[which * kLanes + lane];
#pragma unroll 4
                for (uint32_t j = 0; j < most; ++j) {
                    const uint64_t against = list[j];
#pragma unroll
                    for (int which = 0; which < kListedEach; ++which)
                        ahead[which] += against > own[which] ? 1 : 0;
                }
#pragma unroll
                for (int which = 0; which < kListedEach; ++which)
                    if (own[which] != 0 && ahead[which] < a.topk) {
                        experts[ahead[which]] = ~static_cast<uint32_t>(own[which]);
                        keys[ahead[which]] = static_cast<uint32_t>(own[which] >> 32);
                    }
            };
            if (most <= kLanes)
                choose(std::integral_constant<int, 1>{});
            else
                choose(std::integral_constant<int, 2>{});
            wavefront_sync();
        }
    }
    if constexpr (kEach <= 4)
        choose_sorted<kLanes, kEach>(key, a.topk, experts, keys);
    else if (!listed)  // (many equal keys, or all of the largest in a few lanes)
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
    if (!a.sigmoid && a.bias != nullptr)
        total = experts_sum<kWave, kEach>([&](int i) { return exp(static_cast<double>(logit[i]) - largest); });
    uint64_t key[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int expert = i * kWave + lane;
        const float bias = a.bias != nullptr && expert < a.experts ? a.bias[expert] : 0.0f;
        key[i] = logit[i] == -INFINITY ? 0 : key_of(value_of_expert(a, logit[i], bias, largest, total));
    }
    if (a.groups > 1) {
        uint64_t second;
        double margin;
        strike_out<kWave, kEach>(key, a, find_groups<kWave, kEach>(key, a, keys, second, margin));
    }
    choose_in_turn<kWave, kEach>(key, a.topk, experts, all_chosen[threadIdx.x / kWave]);
    if (lane < a.topk && experts[lane] != kNoExpert)
        logits[lane] = load_logit(a.logits, token, experts[lane]);
    wavefront_sync();
}

// 32-bit words of LDS that a wavefront has for the keys of its tokens, or for one token's of 64 bits.
constexpr int key_words(int lanes, int each) { return kWave * (lanes == kWave ? 2 * each : each > 2 ? each : 2); }

// Experts by their values: scores plus bias, and groups.  Values in fp32, with a bound on their error, find the groups and list
// those experts that can be among the first K; the values of the list, one or two a lane, are then computed in 64 bits, and each
// counts how many are ahead of it.  Groups that fp32 cannot tell apart (one token in ten thousand) are found in the same way from a list of
// those that can be among their two largest.  A token whose list is too long (all values equal) is done again in 64 bits throughout, by
// its whole wavefront.
// 4096 tokens of 256 experts, bias, four of eight groups: 7.9 us (all values in 64 bits: 11.6), half of the time instructions (980 vector
// instructions a wavefront of two tokens, 200 of them for the groups), half waits for LDS and memory; without groups 6.4, 32768
// tokens 17; one token 5.7, without groups 4.5.  Groups in 64 bits add 2 us to a launch (with the whole wavefront's second go: 5).
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
    // Without a bias, where a softmax is compared by its numerators: parts of themselves, with arguments of up to 88, and all of
    // those below 2^-126, where exponentials overflow and results lose their digits or are zero.
    float off = 0x1p-126f, part = 0x1p-16f;
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
    double wide_total = 0.0;
    if (!a.sigmoid && a.bias != nullptr)
        wide_total = experts_sum<kLanes, kEach>([&](int i) { return exp(static_cast<double>(logit[i]) - largest); });
    // Candidates go to the list with their bias and logit, then those of a lane, one or two, have their values in 64 bits as keys.
    uint32_t most, number;
    const auto list_those = [&](const uint32_t (&of)[kEach], uint32_t from) {
        list[lane].key = list[kLanes + lane].key = 0;
        wavefront_sync();
        number = list_candidates<kLanes, kEach>(of, from, kListed, most, [&](uint32_t at, int i) {
            list[at] = {uint64_t{1} << 32 | __float_as_uint(bias[i]), static_cast<uint32_t>(i * kLanes + lane), logit[i]};
        });
    };
    const auto key_of_listed = [&](Candidate (&own)[2]) {
        own[0] = list[lane];
        own[1] = list[kLanes + lane];
        wavefront_sync();
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            if (which == 1 && most <= kLanes)
                break;
            if (own[which].key != 0) {
                own[which].key = key_of(value_of_expert(a, own[which].logit, __uint_as_float(static_cast<uint32_t>(own[which].key)), largest, wide_total));
                list[which * kLanes + lane].key = own[which].key;
            }
        }
        wavefront_sync();
    };
    bool again = false;
    if (a.groups > 1) {
        uint32_t* own_keys = keys + place % (kWave / kLanes) * key_words(kLanes, kEach) / (kWave / kLanes);
        float size = 0.0f, margin;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            size = fmaxf(size, key[i] != 0 ? fabsf(value[i]) : 0.0f);
        size = lanes_max<kLanes>(size);
        uint32_t second;
        uint64_t open = find_groups<kLanes, kEach>(key, a, own_keys, second, margin);
        // Two sums of two, rounded.  Without a bias no value is off by more than the largest one is (which may be zero, as of sigmoids
        // below e^-89 or next to an infinite logit: all are told apart in 64 bits then).
        const float each = a.bias != nullptr ? off : fmaf(size, 0x1.4p-22f - 0x1.8p-24f * fminf(__log2f(fmaxf(size, 0x1p-126f)), 0.0f), off);
        const float unsure = 4.0f * each + 0x1p-21f * size;
        const bool close = !(margin > unsure) && routed;
        if (__any(close)) {
            // Again from values in 64 bits of all that can be among a group's two largest, two or three a group.
            const GroupOf<kLanes> group(a);
            const float least = value_of(second);
            wavefront_sync();
            if (lane < a.groups)
                own_keys[lane] = fabsf(least) < INFINITY ? key_of(least - 0.5f * unsure) : second;
            wavefront_sync();
            uint32_t among[kEach];
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                among[i] = key[i] != 0 && key[i] >= own_keys[group.of_place(i)] ? key[i] : 0;
            list_those(among, 1);
            if (most <= kListed) {
                Candidate own[2];
                key_of_listed(own);
                uint64_t first = 0, next = 0;
                for (uint32_t j = 0; j < number; ++j) {
                    const Candidate other = list[j];
                    if (group.of_expert(other.expert) == lane) {
                        const uint64_t lower = other.key < first ? other.key : first;
                        next = lower > next ? lower : next;
                        first = other.key > first ? other.key : first;
                    }
                }
                bool kept;
                open = best_groups<kLanes>(a, key_of_group(first, next), reinterpret_cast<uint64_t*>(own_keys), kept);
            } else {
                again = close;
            }
        }
        strike_out<kLanes, kEach>(key, a, open);
    }
    uint32_t bound = bound_of<kLanes, kEach>(key, a.topk, all_maxima[place]);
    const float least = value_of(bound);
    if (fabsf(least) < INFINITY)
        bound = key_of(least - 2.0f * off - 4.0f * part * fabsf(least));
    list_those(key, bound);
    again = again || number > kListed;
    if (most <= kListed) {
        Candidate own[2];
        key_of_listed(own);
        if (lane >= static_cast<int>(number))
            experts[lane] = kNoExpert;
        const auto choose = [&](auto listed_each) {  // one or two of the list a lane
            constexpr int kListedEach = decltype(listed_each)::value;
            int ahead[kListedEach] = {};
#pragma unroll 4
            for (uint32_t j = 0; j < most; ++j) {
                const Candidate against = list[j];
#pragma unroll
                for (int which = 0; which < kListedEach; ++which)
                    ahead[which] += against.key > own[which].key || (against.key == own[which].key && against.expert < own[which].expert) ? 1 : 0;
            }
#pragma unroll
            for (int which = 0; which < kListedEach; ++which)
                if (own[which].key != 0 && ahead[which] < a.topk) {
                    experts[ahead[which]] = own[which].expert;
                    logits[ahead[which]] = own[which].logit;
                }
        };
        if (most <= kLanes)
            choose(std::integral_constant<int, 1>{});
        else
            choose(std::integral_constant<int, 2>{});
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
    if (sigmoid) {
        // times e^-shift, so that the sum is not lost where all of them are tiny; mostly there is a logit above 0
        const float shift = largest == -INFINITY ? 0.0f : fminf(largest, 0.0f);
        const bool shifted = __any(shift < 0.0f);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float tail = exp_below(-fabsf(logit[i])), inverse = __builtin_amdgcn_rcpf(1.0f + tail);
            share[i] = logit[i] >= 0.0f ? inverse : tail * inverse;
            rest[i] = logit[i] >= 0.0f ? tail * inverse : inverse;
        }
        if (shifted) {
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (logit[i] < 0.0f)
                    share[i] = exp_below(logit[i] - shift) * __builtin_amdgcn_rcpf(1.0f + exp_below(logit[i]));
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            total += share[i];
    } else {
        const float shift = largest == -INFINITY ? 0.0f : largest;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            share[i] = exp_below(logit[i] - shift);
            rest[i] = 1.0f;
            total += share[i];
        }
    }
    total = lanes_sum<kLanes>(total);
    const float inverse = total == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(total);  // (half of the largest share at least: no tiny one)
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
// 8192 tokens of 128 experts, softmax over all (9 MB) 4.2 us, 32768 of 64 (19 MB) 6.0, 1537 of 60 3.0: a launch and the bytes.
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
        float largest = lanes_max<kLanes>(logit);
        largest = largest == -INFINITY ? 0.0f : largest;  // (nothing but experts that cannot be chosen: no weights)
        float score = 0.0f, rest = 1.0f;
        if (a.sigmoid) {
            const float tail = exp_below(-fabsf(logit)), inverse = 1.0f / (1.0f + tail);
            score = logit != logit ? logit : exp_below(fminf(logit, 0.0f) - fminf(largest, 0.0f)) * inverse;
            rest = logit >= 0.0f ? tail * inverse : inverse;
        } else {
            score = exp_below(logit - largest);
        }
        score = valid ? score : 0.0f;
        const float total = lanes_sum<kLanes>(score);
        score = valid && total != 0.0f ? score / total : 0.0f;
        g = score * rest * (g - lanes_sum<kLanes>(score * g));
    } else {
        const float tail = exp_below(-fabsf(logit)), inverse = 1.0f / (1.0f + tail);
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
    int chunk_bits;  // a workgroup (the gradient: a wavefront) has 2^chunk_bits tokens, wherever sequences begin
    int experts, topk;
    bool sigmoid;
};

// The tokens of a sequence that are in [from, to).
__device__ __forceinline__ void clip(const Balance& a, int64_t sequence, int64_t& from, int64_t& to) {
    if (a.offsets == nullptr)
        return;
    const int64_t begin = uniform_load(a.offsets + sequence), end = uniform_load(a.offsets + sequence + 1);
    from = begin > from ? begin : from;
    to = end < to ? end : to;
}

// The sequences that end at or ahead of a token, and so the first that can have it: a search with 64 probes at a time.
__device__ __forceinline__ int64_t sequences_ahead(const Balance& a, int64_t token) {
    if (a.offsets == nullptr)
        return 0;
    int64_t low = 0, high = a.sequences;
    while (low < high) {
        const int64_t apart = (high - low + kWave - 1) / kWave, probe = low + threadIdx.x % kWave * apart;
        const int ended = __popcll(__ballot(probe < high && a.offsets[probe + 1] <= token));
        if (ended == 0)
            return low;
        const int64_t last = low + (ended - 1) * apart;
        low = last + 1;
        high = last + apart < high ? last + apart : high;
    }
    return low;
}

// A token of each group of kLanes lanes: its logits as they lie in memory, and choice k in lane k.
template <int kEach>
struct BalanceToken {
    uint32_t logit[kEach];
    int64_t named;
    bool here;
};
template <int kLanes, int kEach>
__device__ __forceinline__ void load_token(const Balance& a, int64_t token, bool here, BalanceToken<kEach>& out) {
    const int lane = threadIdx.x % kLanes;
    out.here = here;
    out.named = -1;
    if (here && lane < a.topk)
        out.named = a.ids[token * a.topk + lane];
    load_raw<kLanes, kEach>(a.logits, token, here, a.experts, out.logit);
}

// (a count of 64 bits in three instructions: its halves are whole numbers, the larger one rounded once more where there is one)
__device__ __forceinline__ float float_of(int64_t count) {
    return fmaf(static_cast<float>(static_cast<uint32_t>(count >> 32)), 0x1p32f, static_cast<float>(static_cast<uint32_t>(count)));
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

// loss = E / (C T') * sum over e of c_e * its sum of shares.
__device__ __forceinline__ float loss_of(int experts, float sum, float number, int live) {
    return live > 0 ? sum * static_cast<float>(experts) / number / static_cast<float>(live) : 0.0f;
}

// A workgroup has a chunk of tokens, whatever sequences they are of: kLanes lanes a token at a time, which keep their experts' sums of shares in
// registers, the next token's inputs on their way; choices are counted in LDS (whole numbers: any order gives the same).  The sums of a
// wavefront's tokens, then those of the wavefronts are added in a fixed order.  Chunk c leaves its part of sequence s in row c + s of
// `rows` (from one to the next either c or s goes up by one), shares, then counts, as wide as the lanes' experts, for
// balance_finish_kernel, whose count of workgroups that have arrived the first one clears.  One sequence of one chunk is finished here.
// 32768 tokens of 64 experts (10 MB) 6.3 us, 8192 of 128 in 17 sequences 6.4: half of a wavefront's time is waiting for its offsets, then its
// tokens.  (A workgroup a part of a sequence, a wavefront a token: 11.6 and 16.4.)
template <int kLanes, int kEach>
__global__ void __launch_bounds__(kBlockThreads) balance_loss_kernel(const Balance a, uint32_t* __restrict__ rows,  // null: finished here
                                                                     int* __restrict__ live_of_rows, int* __restrict__ arrived,
                                                                     float* __restrict__ loss, int64_t* __restrict__ counts,
                                                                     int64_t* __restrict__ tokens) {
    constexpr int kWidth = kLanes * kEach, kWaves = kWavesPerBlock, kTokens = kBlockThreads / kLanes;
    __shared__ float sums[kWaves / 2 * kWidth];
    __shared__ int chosen[kWidth];
    __shared__ float place[kWaves];
    __shared__ int live_tokens;
    const int64_t chunk = workgroup_number(), begin = chunk << a.chunk_bits, length = int64_t{1} << a.chunk_bits;
    if (begin >= a.tokens)
        return;
    if (arrived != nullptr && chunk == 0 && threadIdx.x == 0)
        *arrived = 0;
    const int64_t end = begin + length < a.tokens ? begin + length : a.tokens;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    for (int64_t sequence = rows == nullptr ? 0 : sequences_ahead(a, begin); sequence < a.sequences; ++sequence) {
        int64_t from = begin, to = end;
        clip(a, sequence, from, to);
        if (from >= end && rows != nullptr)  // (the one sequence that is finished here may have none of the tokens)
            break;
        BalanceToken<kEach> next;
        load_token<kLanes, kEach>(a, from + group, from + group < to, next);
        __syncthreads();  // (the last sequence's are read)
        for (int e = threadIdx.x; e < kWidth; e += kWaves * kWave)
            chosen[e] = 0;
        if (threadIdx.x == 0)
            live_tokens = 0;
        __syncthreads();
        float own[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            own[i] = 0.0f;
        int number = 0;
        for (int64_t first = from; first < to; first += kTokens) {
            const BalanceToken<kEach> token = next;
            load_token<kLanes, kEach>(a, first + kTokens + group, first + kTokens + group < to, next);
            const bool valid = token.named >= 0 && token.named < a.experts;
            if (valid)
                atomicAdd(&chosen[token.named], 1);
            const bool live = lanes_where<kLanes>(valid) != 0;
            number += live ? 1 : 0;
            float logit[kEach], share[kEach], rest[kEach];
            logits_of_raw<kLanes, kEach>(a.logits, token.logit, token.here, a.experts, logit);
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
        if (rows != nullptr) {
            uint32_t* row = rows + (chunk + sequence) * 2 * kWidth;
            if (wave == 0 && writes)
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    row[i * kLanes + lane] = __float_as_uint(own[i]);
            for (int e = threadIdx.x; e < kWidth; e += kWaves * kWave)
                row[kWidth + e] = static_cast<uint32_t>(chosen[e]);
            if (threadIdx.x == 0)
                live_of_rows[chunk + sequence] = live_tokens;
            continue;
        }
        if (wave == 0 && writes)
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                sums[i * kLanes + lane] = own[i];
        __syncthreads();
        float sum = 0.0f, all = 0.0f;
        for (int e = threadIdx.x; e < a.experts; e += kBlockThreads) {
            counts[e] = chosen[e];
            sum = fmaf(static_cast<float>(chosen[e]), sums[e], sum);
            all += static_cast<float>(chosen[e]);
        }
        sum = workgroup_sum(sum, place);
        all = workgroup_sum(all, place);
        if (threadIdx.x == 0) {
            *tokens = live_tokens;
            *loss = loss_of(a.experts, sum, all, live_tokens);
        }
    }
}

// A sequence's rows are added up by 2^slice_bits workgroups, each for its part of the experts: four columns a thread, neighbouring threads
// neighbouring columns, the rows shared out among groups of threads, whose sums are then added in a fixed order.  Each leaves its part
// of sum c_e * share_e and of C; the one that arrives last adds those up, in their order as well.  (Several slices only for one sequence:
// rows are many then.)  A chain of latencies (offsets, rows, the slices' arrival), not of bytes: 512 rows of 64 experts 6.3 us, 17 sequences of
// some 31 rows of 128 5.0.  Neighbouring threads on neighbouring rows instead: 9.2 and 11.2.
constexpr int kMostSlices = 16, kRowsAtOnce = 8, kFinishThreads = 1024;
__global__ void __launch_bounds__(kFinishThreads) balance_finish_kernel(const Balance a, int width,  // columns of a row's half: 8 to 4096
                                                                       int slice_bits, const u32x4* __restrict__ rows,
                                                                       const int* __restrict__ live_of_rows, int* __restrict__ arrived,
                                                                       uint64_t* __restrict__ parts_of_loss,  // [slices]: sum's bits, C's above them
                                                                       float* __restrict__ loss, int64_t* __restrict__ counts,
                                                                       int64_t* __restrict__ tokens) {
    __shared__ float share_parts[4 * kFinishThreads];
    __shared__ uint32_t count_parts[4 * kFinishThreads];
    __shared__ float place[kFinishThreads / kWave][2];
    __shared__ int live_place[kFinishThreads / kWave];
    const int64_t sequence = workgroup_number() >> slice_bits;
    const int slices = 1 << slice_bits, slice = static_cast<int>(workgroup_number()) & (slices - 1);
    if (sequence >= a.sequences)
        return;
    int64_t from = 0, to = a.tokens;
    clip(a, sequence, from, to);
    const int64_t first = (from >> a.chunk_bits) + sequence, end = to > from ? ((to - 1) >> a.chunk_bits) + sequence + 1 : first;
    const int threads = blockDim.x;
    int live = 0;
    for (int64_t row = first + threadIdx.x; row < end; row += threads)
        live += live_of_rows[row];
    const int quads = width / 4 >> slice_bits;  // of this slice's columns
    const int across = quads < threads ? quads : threads, groups = threads / across;
    const int group = threadIdx.x / across, lane = threadIdx.x % across;
    float sum = 0.0f, number = 0.0f;
    for (int some = 0; some < quads; some += across) {
        const int at = slice * quads + some;
        float share[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        u32x4 count = {0u, 0u, 0u, 0u};
        for (int64_t base = first + group; base < end; base += kRowsAtOnce * groups) {
            u32x4 other[kRowsAtOnce], more[kRowsAtOnce];
#pragma unroll
            for (int r = 0; r < kRowsAtOnce; ++r) {
                const int64_t row = base + r * groups < end ? base + r * groups : base;
                other[r] = rows[row * (width / 2) + at + lane];
                more[r] = rows[row * (width / 2) + width / 4 + at + lane];
            }
#pragma unroll
            for (int r = 0; r < kRowsAtOnce; ++r)
                if (base + r * groups < end) {
                    count += more[r];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        share[i] += __uint_as_float(other[r][i]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            share_parts[(group * across + lane) * 4 + i] = share[i];
            count_parts[(group * across + lane) * 4 + i] = count[i];
        }
        __syncthreads();
        for (int column = threadIdx.x; column < across * 4; column += threads) {
            float shares = 0.0f;
            uint32_t chosen = 0;
#pragma unroll 8
            for (int part = 0; part < groups; ++part) {
                shares += share_parts[part * across * 4 + column];
                chosen += count_parts[part * across * 4 + column];
            }
            if (at * 4 + column < a.experts) {
                counts[sequence * a.experts + at * 4 + column] = chosen;
                sum = fmaf(static_cast<float>(chosen), shares, sum);
                number += static_cast<float>(chosen);
            }
        }
        __syncthreads();
    }
    sum = lanes_sum<kWave>(sum);
    number = lanes_sum<kWave>(number);
    live = lanes_sum<kWave>(live);
    if (threadIdx.x % kWave == 0) {
        place[threadIdx.x / kWave][0] = sum;
        place[threadIdx.x / kWave][1] = number;
        live_place[threadIdx.x / kWave] = live;
    }
    __syncthreads();
    if (threadIdx.x > 0)
        return;
    sum = number = 0.0f;
    live = 0;
    for (int w = 0; w < threads / kWave; ++w) {
        sum += place[w][0];
        number += place[w][1];
        live += live_place[w];
    }
    if (slices > 1) {
        // The exchange has been done where every workgroup sees it when it comes back; only then is this slice counted.
        const uint64_t both = static_cast<uint64_t>(__float_as_uint(number)) << 32 | __float_as_uint(sum);
        const uint64_t old = __hip_atomic_exchange(parts_of_loss + slice, both, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        int one = 1;
        asm volatile("" : "+v"(one) : "v"(old) : "memory");
        if (__hip_atomic_fetch_add(arrived, one, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != slices - 1)
            return;
        uint64_t all[kMostSlices];
#pragma unroll
        for (int other = 0; other < kMostSlices; ++other)
            all[other] = other < slices ? __hip_atomic_load(parts_of_loss + other, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
        sum = number = 0.0f;
#pragma unroll
        for (int other = 0; other < kMostSlices; ++other) {
            sum += __uint_as_float(static_cast<uint32_t>(all[other]));
            number += __uint_as_float(static_cast<uint32_t>(all[other] >> 32));
        }
    }
    tokens[sequence] = live;
    loss[sequence] = loss_of(a.experts, sum, number, live);
}

// The gradient: with F_e = g E c_e / (C T') of the token's sequence, p_e (F_e - sum of F p) (times 1 - s_e for sigmoids); zero for
// tokens without a choice and for those of no sequence.  A wavefront has a chunk of tokens, whatever sequences they are of; the next
// tokens' inputs are on their way.  32768 tokens of 64 experts (19 MB) 7.0 us, 8192 of 128 in 17 sequences 6.6, 14681 of 211 (25 MB) 10.4.
template <int kLanes, int kEach>
__global__ void __launch_bounds__(kBlockThreads) balance_loss_backward_kernel(const Balance a, const float* __restrict__ grad,  // [S]
                                                                              const int64_t* __restrict__ counts, const int64_t* __restrict__ tokens,
                                                                              void* __restrict__ grad_logits) {
    constexpr int kTokens = kWave / kLanes;
    const int64_t begin = (workgroup_number() * kWavesPerBlock + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)) << a.chunk_bits;
    const int64_t length = int64_t{1} << a.chunk_bits;
    if (begin >= a.tokens)
        return;
    const int64_t end = begin + length < a.tokens ? begin + length : a.tokens;
    const int lane = threadIdx.x % kLanes, group = threadIdx.x % kWave / kLanes;
    for (int64_t sequence = sequences_ahead(a, begin); sequence < a.sequences; ++sequence) {
        int64_t from = begin, to = end;
        clip(a, sequence, from, to);
        if (from >= end)
            break;
        BalanceToken<kEach> next;
        load_token<kLanes, kEach>(a, from + group, from + group < to, next);
        int64_t count[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            count[i] = counts[sequence * a.experts + (i * kLanes + lane < a.experts ? i * kLanes + lane : 0)];
        const int64_t live_tokens = tokens[sequence];
        const float of_loss = grad[sequence];
        __builtin_amdgcn_sched_barrier(0);  // (a conversion behind every load would wait for each of them)
        float factor[kEach], number = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            factor[i] = i * kLanes + lane < a.experts ? float_of(count[i]) : 0.0f;
            number += factor[i];
        }
        number = lanes_sum<kLanes>(number);
        const float each = live_tokens > 0 && number > 0.0f ? of_loss * static_cast<float>(a.experts) / number / float_of(live_tokens) : 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            factor[i] *= each;
        for (int64_t first = from; first < to; first += kTokens) {
            const BalanceToken<kEach> token = next;
            load_token<kLanes, kEach>(a, first + kTokens + group, first + kTokens + group < to, next);
            const bool live = lanes_where<kLanes>(token.named >= 0 && token.named < a.experts) != 0;
            float logit[kEach], share[kEach], rest[kEach], out[kEach], along = 0.0f;
            logits_of_raw<kLanes, kEach>(a.logits, token.logit, token.here, a.experts, logit);
            shares_of<kLanes, kEach>(logit, a.sigmoid, share, rest);
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                along = fmaf(factor[i], share[i], along);
            along = lanes_sum<kLanes>(along);
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                out[i] = live ? share[i] * rest[i] * (factor[i] - along) : 0.0f;
            store_spread<kLanes, kEach>(grad_logits, a.logits.wide, first + group, token.here, a.experts, out);
        }
    }
    if (a.offsets != nullptr) {
        const int64_t behind = a.offsets[a.sequences], ahead = a.offsets[0];
        float zero[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            zero[i] = 0.0f;
        if (begin < ahead || end > behind)
            for (int64_t token = begin + group; token < end; token += kTokens)
                store_spread<kLanes, kEach>(grad_logits, a.logits.wide, token, token < ahead || token >= behind, a.experts, zero);
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
// then (us a call with 16, 32 and 64 lanes, 256 experts, a bias: 1 token 5.6, 5.2, 5.1; 4096 tokens 6.6, 5.9, 7.2; 8192 tokens 7.2, 7.5, 11.9;
// 32768 tokens 16.6, 23.0, 40.3).
Spread spread_for_choices(int64_t num_tokens, int experts, int needed) {
    return spread_of(experts, std::max(needed, num_tokens <= int64_t{32} * current_topology(current_tuning()).cus ? 32 : 1));
}

// For the loss, the same, and 32 lanes for more than 128 experts, because twice as many experts a lane leave a SIMD half of its
// wavefronts (the gradient of 14681 tokens of 211 experts: 16 lanes 12.2 us, 32 lanes 9.7).
Spread spread_for_balance(int64_t num_tokens, int experts, int topk) {
    return spread_for_choices(num_tokens, experts, experts > 128 ? std::max(topk, 32) : topk);
}

// CALL(lanes, experts a lane) for a Spread: those that every kernel meets, and MORE that some do: 8 lanes, for up to 32 experts that are not chosen by
// value; 16 lanes with 16 experts each, which the loss spreads over 32; whole wavefronts for fewer than 513 experts, with more than 32 groups.
#define NANOEP_SPREAD(LANES, EACH, CALL) \
    case (LANES) * 100 + (EACH):         \
        CALL(LANES, EACH);               \
        break;
#define NANOEP_SPREADS_OF_8(CALL) NANOEP_SPREAD(8, 1, CALL) NANOEP_SPREAD(8, 2, CALL) NANOEP_SPREAD(8, 4, CALL)
#define NANOEP_SPREAD_16_16(CALL) NANOEP_SPREAD(16, 16, CALL)
#define NANOEP_SPREADS_OF_MANY_GROUPS(CALL) \
    NANOEP_SPREAD(64, 1, CALL) NANOEP_SPREAD(64, 2, CALL) NANOEP_SPREAD(64, 4, CALL) NANOEP_SPREAD(64, 8, CALL)
#define NANOEP_BY_SPREAD(SPREAD, CALL, MORE)                                                                                          \
    switch ((SPREAD).lanes * 100 + (SPREAD).each) {                                                                                   \
        NANOEP_SPREAD(16, 1, CALL) NANOEP_SPREAD(16, 2, CALL) NANOEP_SPREAD(16, 4, CALL) NANOEP_SPREAD(16, 8, CALL)                    \
        NANOEP_SPREAD(32, 1, CALL) NANOEP_SPREAD(32, 2, CALL) NANOEP_SPREAD(32, 4, CALL) NANOEP_SPREAD(32, 8, CALL)                    \
        NANOEP_SPREAD(32, 16, CALL) NANOEP_SPREAD(64, 16, CALL) NANOEP_SPREAD(64, 32, CALL) NANOEP_SPREAD(64, 64, CALL)                \
        MORE                                                                                                                          \
        default:                                                                                                                      \
            return NANOEP_ERR_INVALID_ARGUMENT;                                                                                       \
    }

bool router_sizes_fit(int64_t stride, int logits_type, int64_t num_tokens, int experts, int topk, int scoring) {
    return num_tokens >= 0 && num_tokens <= 0x7fffffff / kMaxTopk && experts >= 1 && experts <= kMostExperts && topk >= 1 && topk <= kMaxTopk &&
           stride >= experts && stride <= int64_t{1} << 31 && (logits_type == NANOEP_BF16 || logits_type == NANOEP_FP32) &&
           (scoring == NANOEP_SOFTMAX || scoring == NANOEP_SIGMOID);
}

Logits logits_of(const void* data, int64_t stride, int type) { return {data, stride, type == NANOEP_FP32}; }

int bits_of(int64_t least) {
    int bits = 0;
    while ((int64_t{1} << bits) < least)
        ++bits;
    return bits;
}

// How the loss's tokens are dealt out: a workgroup has one round of tokens, more (but no more than a sequence's) where that would be more
// than two workgroups a compute unit, or a few rounds of one sequence, which then take one launch.  Each leaves rows of sums, which several
// workgroups add up for one sequence, and one each for several.
struct BalancePlan {
    Spread spread;
    int chunk_bits, slice_bits;
    int64_t chunks, rows;  // rows of sums: 0 where none are needed
};
BalancePlan plan_balance(int64_t num_tokens, int experts, int topk, int64_t sequences) {
    BalancePlan plan;
    plan.spread = spread_for_balance(num_tokens, experts, topk);
    const int64_t round = kBlockThreads / plan.spread.lanes, most = int64_t{2} * current_topology(current_tuning()).cus;
    const int64_t average = (num_tokens + sequences - 1) / sequences;
    plan.chunk_bits = bits_of(sequences == 1 && num_tokens <= 4 * round ? 4 * round : std::max(round, std::min(average, (num_tokens + most - 1) / most)));
    plan.chunks = (num_tokens + (int64_t{1} << plan.chunk_bits) - 1) >> plan.chunk_bits;
    plan.rows = sequences == 1 && plan.chunks == 1 ? 0 : plan.chunks + sequences;
    // (256 bytes of a row a slice: loss and gradient of 32768 tokens of 256 experts 33.6 us, with 512 or 1024 bytes 36.0, 40.8; of 64 experts
    // 19.0, with 128 bytes 20.7)
    plan.slice_bits = sequences == 1 ? std::min(bits_of(kMostSlices), bits_of((plan.spread.lanes * plan.spread.each + 63) / 64)) : 0;
    return plan;
}
// The slices' parts of the loss, rows, their numbers of tokens, the number of slices that are done.
size_t balance_workspace(const BalancePlan& plan) {
    const size_t row = 2 * static_cast<size_t>(plan.spread.lanes) * plan.spread.each * sizeof(uint32_t);
    return plan.rows == 0 ? 0 : kMostSlices * sizeof(uint64_t) + static_cast<size_t>(plan.rows) * (row + sizeof(int)) + sizeof(int);
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
                             topk_groups < groups ? groups : 1, topk_groups, scoring == NANOEP_SIGMOID, normalize != 0, scale,
                             num_experts / groups, bits_of(groups), static_cast<float>(groups) / static_cast<float>(num_experts)};
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
        NANOEP_BY_SPREAD(spread, NANOEP_LAUNCH_VALUES, NANOEP_SPREAD_16_16(NANOEP_LAUNCH_VALUES) NANOEP_SPREADS_OF_MANY_GROUPS(NANOEP_LAUNCH_VALUES))
    else
        NANOEP_BY_SPREAD(spread, NANOEP_LAUNCH_ROUTE, NANOEP_SPREADS_OF_8(NANOEP_LAUNCH_ROUTE) NANOEP_SPREAD_16_16(NANOEP_LAUNCH_ROUTE))
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
    NANOEP_BY_SPREAD(spread, NANOEP_LAUNCH_ROUTE_BACKWARD, NANOEP_SPREADS_OF_8(NANOEP_LAUNCH_ROUTE_BACKWARD) NANOEP_SPREAD_16_16(NANOEP_LAUNCH_ROUTE_BACKWARD))
#undef NANOEP_LAUNCH_ROUTE_BACKWARD
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

size_t nanoep_balance_loss_workspace_bytes(int64_t num_tokens, int num_experts, int num_topk, int64_t sequences) {
    using namespace nanoep;
    if (!router_sizes_fit(num_experts, NANOEP_FP32, num_tokens, num_experts, num_topk, NANOEP_SOFTMAX) || sequences < 1 || sequences > 0x7fffffff)
        return 0;
    return balance_workspace(plan_balance(num_tokens, num_experts, num_topk, sequences));
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
    const BalancePlan plan = plan_balance(num_tokens, num_experts, num_topk, sequences);
    if (workspace_bytes < balance_workspace(plan))
        return NANOEP_ERR_WORKSPACE;
    if (plan.rows > 0 && (workspace == nullptr || !aligned16(workspace)))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const Balance arguments = {logits_of(logits, logits_stride, logits_type), ids, sequence_offsets, num_tokens, sequences, plan.chunk_bits, num_experts,
                               num_topk, scoring == NANOEP_SIGMOID};
    const int width = plan.spread.lanes * plan.spread.each;
    uint64_t* parts_of_loss = nullptr;
    uint32_t* rows = nullptr;
    int *live_of_rows = nullptr, *arrived = nullptr;
    if (plan.rows > 0) {
        parts_of_loss = static_cast<uint64_t*>(workspace);
        rows = reinterpret_cast<uint32_t*>(parts_of_loss + kMostSlices);
        live_of_rows = reinterpret_cast<int*>(rows + plan.rows * 2 * width);
        arrived = live_of_rows + plan.rows;
    }
    const auto on = static_cast<hipStream_t>(stream);
    if (plan.chunks > 0) {
#define NANOEP_LAUNCH_BALANCE(LANES, EACH)                                                                                                   \
    balance_loss_kernel<LANES, EACH><<<grid_of(plan.chunks), kBlockThreads, 0, on>>>(arguments, rows, live_of_rows, arrived, loss, counts, tokens)
        NANOEP_BY_SPREAD(plan.spread, NANOEP_LAUNCH_BALANCE, NANOEP_SPREADS_OF_8(NANOEP_LAUNCH_BALANCE))
#undef NANOEP_LAUNCH_BALANCE
        NANOEP_HIP_TRY(hipGetLastError());
    }
    if (plan.rows > 0) {
        const int slice_bits = plan.chunks > 0 ? plan.slice_bits : 0;  // (without tokens nobody cleared the number of those done)
        // (several sequences: 14681 tokens of 211 experts in 17 of them, loss and gradient, with 256, 512 and 1024 threads 27.4, 25.9, 26.5 us)
        balance_finish_kernel<<<grid_of(sequences << slice_bits), sequences == 1 ? kFinishThreads : kFinishThreads / 2, 0, on>>>(
            arguments, width, slice_bits, reinterpret_cast<const u32x4*>(rows), live_of_rows, arrived, parts_of_loss, loss, counts, tokens);
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
    // a wavefront one round of tokens, more where that would be more than 16 wavefronts a compute unit (us with 4, 8, 16, 32 of them: 32768
    // tokens of 64 experts 9.0, 6.8, 6.7, 7.1; of 128, 64 sequences, 15.0, 11.6, 11.0, 12.6)
    const Spread spread = spread_for_balance(num_tokens, num_experts, num_topk);
    const int64_t held = int64_t{16} * current_topology(current_tuning()).cus;
    const int chunk_bits = bits_of(std::max<int64_t>(kWave / spread.lanes, (num_tokens + held - 1) / held));
    const Balance arguments = {logits_of(logits, logits_stride, logits_type), ids, sequence_offsets, num_tokens, sequences, chunk_bits, num_experts, num_topk,
                               scoring == NANOEP_SIGMOID};
    const int64_t chunks = (num_tokens + (int64_t{1} << chunk_bits) - 1) >> chunk_bits, blocks = (chunks + kWavesPerBlock - 1) / kWavesPerBlock;
    const auto on = static_cast<hipStream_t>(stream);
#define NANOEP_LAUNCH_BALANCE_BACKWARD(LANES, EACH) \
    balance_loss_backward_kernel<LANES, EACH><<<grid_of(blocks), kBlockThreads, 0, on>>>(arguments, grad, counts, tokens, grad_logits)
    NANOEP_BY_SPREAD(spread, NANOEP_LAUNCH_BALANCE_BACKWARD, NANOEP_SPREADS_OF_8(NANOEP_LAUNCH_BALANCE_BACKWARD))
#undef NANOEP_LAUNCH_BALANCE_BACKWARD
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

}  // extern "C"
