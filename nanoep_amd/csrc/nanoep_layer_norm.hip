// Layer norm and root-mean-square norm of rows, with a residual added first, and their gradients.
//
//   s = x + residual, rounded to the rows' type (it goes on as the residual stream, and is what the norm sees)
//   mean = sum(s) / H (0 for the root-mean-square norm), r = 1 / sqrt(sum((s - mean)^2) / H + eps)
//   y = (s - mean) * r * gamma + beta
// and for a gradient g of y, with z = (s - mean) * r and u = g * gamma:
//   dx = r * (u - mean(u) - z * mean(u * z)) + the gradient of s itself,  dgamma = sum over rows of g * z,  dbeta = that of g
//   (the root-mean-square norm: without mean(u), beta)
// All of it in fp32, every output rounded once.

#include <algorithm>
#include <type_traits>

#include "nanoep_lanes.h"
#include "nanoep_operators.h"

namespace nanoep {
namespace {

constexpr int kMostThreads = 1024;
constexpr int kBackwardThreads = 512;  // two wavefronts a SIMD: 256 registers a lane
constexpr int kMostRowWaves = kMostThreads / kWave;
constexpr int kMostHidden = 16384;
constexpr int kWaitForLoads = 0x0f70;    // an operand of s_waitcnt: no vector memory access is left
constexpr int kRawBuffer = 0x00020000;  // the last word of a buffer of plain 32-bit data

struct Bf16 {};  // two bytes a value
struct Fp32 {};

// One 16-byte vector of a row: kColumns values.
template <class T>
struct RowType;
template <>
struct RowType<Bf16> {
    static constexpr int kColumns = 8;
    static __device__ __forceinline__ void unpack(const u32x4 v, float (&out)[8]) { unpack_bf16(v, out); }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[8]) { return pack_bf16(v); }
};
template <>
struct RowType<Fp32> {
    static constexpr int kColumns = 4;
    static __device__ __forceinline__ void unpack(const u32x4 v, float (&out)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            out[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[4]) {
        return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    }
};

// The parameters of a lane's vectors, kept as narrow as they lie in memory.
template <class P, int kColumns>
struct HeldParameters {
    u32x4 data[kColumns / RowType<P>::kColumns];
    __device__ __forceinline__ void load(const u32x4* parameters, int at) {
#pragma unroll
        for (int part = 0; part < kColumns / RowType<P>::kColumns; ++part)
            data[part] = parameters[at * (kColumns / RowType<P>::kColumns) + part];
    }
    __device__ __forceinline__ void unpack(float (&out)[kColumns]) const {
        if constexpr (RowType<P>::kColumns == 8) {
            unpack_bf16(data[0], out);
        } else {
#pragma unroll
            for (int i = 0; i < kColumns; ++i)
                out[i] = __uint_as_float(data[i / 4][i % 4]);
        }
    }
};

// A store to the row's vector `at`, dropped where that is behind its `size` bytes, without a branch around it: where a store may be
// skipped, a wait for the loads ahead of it is a wait for it as well, since both are counted together, in their order.
template <bool kNonTemporal, class V>
__device__ __forceinline__ void store_within(void* row, int size, int at, const V v) {
    const __amdgpu_buffer_rsrc_t within = __builtin_amdgcn_make_buffer_rsrc(row, 0, size, kRawBuffer);
    constexpr int kCache = kNonTemporal ? 2 : 0;
    if constexpr (sizeof(V) == 16)
        __builtin_amdgcn_raw_buffer_store_b128(v, within, at * 16, 0, kCache);
    else
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), within, at * 4, 0, kCache);
}

// What the wavefronts of a row left in LDS, one in each of 16 neighbouring lanes; nothing behind the last.
__device__ __forceinline__ float2 of_wavefront(const float2* places, int waves) {
    const int lane = threadIdx.x % kMostRowWaves;
    return lane < waves ? places[lane] : make_float2(0.0f, 0.0f);
}

// A workgroup works through rows (`teams` at a time, those of a turn neighbours over all workgroups), blockDim.x lanes a row, with the
// parameters in registers; a row stays there (kVectors 16-byte vectors a lane) between its sums and its output, so that every input
// byte is read once, and the next row's inputs are on their way meanwhile.
// One barrier a row: every wavefront has the mean and the squares about it of its own part, and the parts are put together as
// mean = sum n_w m_w / H, squares = sum (squares_w + n_w (m_w - mean)^2), as good as squares about the row's mean.
// kPastCache: the call's rows do not fit the last-level cache; then loads are the nontemporal ones, else the stores.
// HBM-bound: 4096 x 7168 with a residual (235 MB) 38 to 40 us, 6 TB/s, 8192 x 2048 (134 MB) 21.2; fp32, 4096 x 4096 (268 MB) 42.8; one token 3.2, a
// launch.  (A workgroup a row, two barriers, the parameters from L2 for every row: 43.8.)
template <class T, class P, int kVectors, bool kPastCache>
__global__ void __launch_bounds__(kMostThreads) layer_norm_kernel(const u32x4* __restrict__ x,         // [T][vectors]
                                                                  const u32x4* __restrict__ residual,  // [T][vectors] or null
                                                                  const u32x4* __restrict__ gamma,
                                                                  const u32x4* __restrict__ beta,  // null: none
                                                                  u32x4* __restrict__ total,       // [T][vectors], null exactly when residual is
                                                                  u32x4* __restrict__ normalized,
                                                                  float* __restrict__ means,  // [T], null: the root-mean-square norm
                                                                  float* __restrict__ rstds,  // [T]
                                                                  int64_t rows,
                                                                  int64_t groups,
                                                                  int vectors,
                                                                  float columns,
                                                                  float eps) {
    using Row = RowType<T>;
    constexpr int kColumns = Row::kColumns;
    __shared__ float2 places[2][kMostRowWaves];  // of a wavefront: squares, mean
    // (a wavefront is one team's: what goes by the row is scalar)
    const int waves = blockDim.x / kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int teams = blockDim.y, team = __builtin_amdgcn_readfirstlane(threadIdx.y), first_wave = team * waves;
    const int64_t group = workgroup_number();
    const bool centred = means != nullptr;

    HeldParameters<P, kColumns> factors[kVectors], shifts[kVectors];
    bool in_row[kVectors];
    uint32_t place[kVectors];  // of a lane's vector in its row; lanes beside the row read the first one and count nothing
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = threadIdx.x + v * blockDim.x;
        in_row[v] = at < vectors;
        place[v] = in_row[v] ? at : 0;
    }
    // columns of the row that wavefront w has
    const auto part_of = [&](int w) {
        int held = 0;
#pragma unroll
        for (int v = 0; v < kVectors && w < waves; ++v) {
            const int left = vectors - w * kWave - v * static_cast<int>(blockDim.x);
            held += left < 0 ? 0 : left > kWave ? kWave : left;
        }
        return static_cast<float>(held * kColumns);
    };
    const float own_part = part_of(wave), part = part_of(threadIdx.x % kMostRowWaves);
    const float per_part = own_part > 0.0f ? 1.0f / own_part : 0.0f, per_column = 1.0f / columns;
    u32x4 next[kVectors], next_added[kVectors];
    const auto load = [&](int64_t row) {
        row = row < rows ? row : rows - 1;  // (rows past the end are the last one again, and leave nothing)
        const u32x4* row_x = x + row * vectors;
        if (residual != nullptr) {
            const u32x4* row_residual = residual + row * vectors;
#pragma unroll
            for (int v = 0; v < kVectors; ++v)
                next_added[v] = load_vec<kPastCache>(row_residual + place[v]);
        }
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
            next[v] = load_vec<kPastCache>(row_x + place[v]);
    };
    const int64_t apart = groups * teams;
    load(group * teams + team);
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        factors[v].load(gamma, place[v]);
        if (beta != nullptr)
            shifts[v].load(beta, place[v]);
    }
    int turn = 0;
    __builtin_amdgcn_s_waitcnt(kWaitForLoads);  // (in the loop, a wait that suits the first row as well would be one for the last row's stores)
    for (int64_t first = group * teams; first < rows; first += apart, turn ^= 1) {
        const int64_t row = first + team;
        const bool here = row < rows;
        const int64_t base = here ? row * vectors : 0;
        const int size = here ? vectors * 16 : 0;
        float s[kVectors][kColumns];
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            Row::unpack(next[v], s[v]);
            if (residual != nullptr) {
                float added[kColumns];
                Row::unpack(next_added[v], added);
#pragma unroll
                for (int i = 0; i < kColumns; ++i)
                    s[v][i] += added[i];
                const u32x4 packed = Row::pack(s[v]);
                store_within<!kPastCache>(total + base, size, threadIdx.x + v * blockDim.x, packed);
                Row::unpack(packed, s[v]);
            }
        }
        load(row + apart);
        float mean = 0.0f, squares = 0.0f;
        if (centred) {
#pragma unroll
            for (int v = 0; v < kVectors; ++v) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < kColumns; ++i)
                    sum += s[v][i];
                mean += in_row[v] ? sum : 0.0f;
            }
            mean = lanes_sum<kWave>(mean) * per_part;
        }
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kColumns; ++i)
                sum = fmaf(s[v][i] - mean, s[v][i] - mean, sum);
            squares += in_row[v] ? sum : 0.0f;
        }
        squares = lanes_sum<kWave>(squares);
        if (waves > 1) {
            if (threadIdx.x % kWave == 0)
                places[turn][first_wave + wave] = make_float2(squares, mean);
            __syncthreads();
            const float2 other = of_wavefront(places[turn] + first_wave, waves);
            squares = other.x;
            if (centred) {
                mean = lanes_sum<kMostRowWaves>(part * other.y) * per_column;
                squares = fmaf(part * (other.y - mean), other.y - mean, squares);
            }
            squares = lanes_sum<kMostRowWaves>(squares);
        }
        const float rstd = 1.0f / sqrtf(fmaf(squares, per_column, eps));
        store_within<false>(rstds + (here ? row : 0), here ? 4 : 0, threadIdx.x, rstd);
        if (centred)
            store_within<false>(means + (here ? row : 0), here ? 4 : 0, threadIdx.x, mean);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            float factor[kColumns];
            factors[v].unpack(factor);
#pragma unroll
            for (int i = 0; i < kColumns; ++i)
                s[v][i] = (s[v][i] - mean) * rstd * factor[i];
            if (beta != nullptr) {
                float shift[kColumns];
                shifts[v].unpack(shift);
#pragma unroll
                for (int i = 0; i < kColumns; ++i)
                    s[v][i] += shift[i];
            }
            store_within<!kPastCache>(normalized + base, size, threadIdx.x + v * blockDim.x, Row::pack(s[v]));
        }
    }
}

// The gradient.  A workgroup works through rows (those of a turn are neighbours over all workgroups; `teams` of them at a time in a
// workgroup) and keeps the two sums over rows in registers; at its end it writes them, added over its teams, to its row of `sums`
// ([workgroups][2][columns] fp32), which parameter_gradient_kernel adds up in a fixed order.  No atomics.
// z and u stay in registers between a row's sums and its output; the next row's inputs are on their way meanwhile.
// HBM-bound up to the sums: 4096 x 7168 with grad_residual (235 MB) 45.0 us, without the parameters' gradients 41.1 (5.7 TB/s; a library's
// addition of two such arrays into a third 5.5); 15 MB of sums at the end and parameter_gradient_kernel's 4.8 are the rest of a call.
// fp32 rows, 4096 x 4096 (268 MB) 48.1.  1537 x 2816 with fp32 parameters 8.2 + 3.2 (on a box where it was 8.0: three teams instead of two 8.2,
// five 9.0).  A workgroup's rows next to one another: 54 a call instead of 50; two workgroups a compute unit, so twice the sums: 59; fourteen
// wavefronts a row instead of seven: 55; two teams of seven: 47 instead of 45; two rows ahead: the same.
template <class T, class P, int kVectors, bool kAdded, bool kInput>
__global__ void __launch_bounds__(kBackwardThreads) layer_norm_backward_kernel(const u32x4* __restrict__ grad,   // [T][vectors]
                                                                               const u32x4* __restrict__ total,  // [T][vectors]
                                                                               const u32x4* __restrict__ gamma,
                                                                               const float* __restrict__ means,  // null: the root-mean-square norm
                                                                               const float* __restrict__ rstds,
                                                                               const u32x4* __restrict__ grad_residual,  // [T][vectors], if kAdded
                                                                               u32x4* __restrict__ grad_x,               // [T][vectors], if kInput
                                                                               u32x4* __restrict__ sums,                 // null: not wanted
                                                                               int64_t rows,
                                                                               int64_t groups,
                                                                               int vectors,
                                                                               float columns) {
    using Row = RowType<T>;
    constexpr int kColumns = Row::kColumns;
    __shared__ float2 places[2][kBackwardThreads / kWave];
    extern __shared__ u32x4 team_sums[];  // [teams][columns / 4], if there are several
    // (a wavefront is one team's: what goes by the row is scalar)
    const int waves = blockDim.x / kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int teams = blockDim.y, team = __builtin_amdgcn_readfirstlane(threadIdx.y), first_wave = team * waves;
    const int64_t group = blockIdx.x;

    HeldParameters<P, kColumns> held[kVectors];
    float sum_z[kVectors][kColumns], sum_g[kVectors][kColumns];
    bool in_row[kVectors];
    uint32_t place[kVectors];  // of a lane's vector in its row; lanes beside the row read the first one and count nothing
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = threadIdx.x + v * blockDim.x;
        in_row[v] = at < vectors;
        place[v] = in_row[v] ? at : 0;
        held[v].load(gamma, place[v]);
#pragma unroll
        for (int i = 0; i < kColumns; ++i)
            sum_z[v][i] = sum_g[v][i] = 0.0f;
    }
    struct Inputs {
        u32x4 total[kVectors], grad[kVectors], added[kVectors];
        float mean, rstd;
    };
    // rows past the end are the last one again, and count nothing
    const auto load = [&](int64_t row, Inputs& in) {
        row = row < rows ? row : rows - 1;
        const u32x4 *row_total = total + row * vectors, *row_grad = grad + row * vectors;
        in.rstd = rstds[row];
        in.mean = means != nullptr ? means[row] : 0.0f;
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            in.total[v] = row_total[place[v]];
            in.grad[v] = row_grad[place[v]];
        }
        if (kAdded) {
            const u32x4* row_added = grad_residual + row * vectors;
#pragma unroll
            for (int v = 0; v < kVectors; ++v)
                in.added[v] = row_added[place[v]];
        }
    };
    const float per_column = 1.0f / columns;
    Inputs next;
    const int64_t apart = groups * teams;
    load(group * teams + team, next);
    int turn = 0;
    __builtin_amdgcn_s_waitcnt(kWaitForLoads);  // (in the loop, a wait that suits the first row as well would be one for the last row's stores)
    for (int64_t first = group * teams; first < rows; first += apart, turn ^= 1) {
        const int64_t row = first + team;
        const bool here = row < rows;
        const float mean = next.mean, rstd = next.rstd;
        float z[kVectors][kColumns], u[kVectors][kColumns], both[2] = {0.0f, 0.0f};
        u32x4 added[kVectors];
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            float factor[kColumns];
            Row::unpack(next.total[v], z[v]);
            Row::unpack(next.grad[v], u[v]);
            held[v].unpack(factor);
            if (kAdded)
                added[v] = next.added[v];
            if (here && in_row[v]) {
#pragma unroll
                for (int i = 0; i < kColumns; ++i) {
                    const float g = u[v][i];
                    z[v][i] = (z[v][i] - mean) * rstd;
                    u[v][i] *= factor[i];
                    sum_g[v][i] += g;
                    sum_z[v][i] = fmaf(g, z[v][i], sum_z[v][i]);
                    both[0] += u[v][i];
                    both[1] = fmaf(u[v][i], z[v][i], both[1]);
                }
            }
        }
        load(row + apart, next);
        if (kInput) {
            both[0] = lanes_sum<kWave>(both[0]);
            both[1] = lanes_sum<kWave>(both[1]);
            if (waves > 1) {
                if (threadIdx.x % kWave == 0)
                    places[turn][first_wave + wave] = make_float2(both[0], both[1]);
                __syncthreads();
                const float2 other = of_wavefront(places[turn] + first_wave, waves);
                both[0] = lanes_sum<kMostRowWaves>(other.x);
                both[1] = lanes_sum<kMostRowWaves>(other.y);
            }
            const float across = means != nullptr ? both[0] * per_column * -rstd : 0.0f, along = both[1] * per_column * -rstd;
#pragma unroll
            for (int v = 0; v < kVectors; ++v) {
#pragma unroll
                for (int i = 0; i < kColumns; ++i)
                    u[v][i] = fmaf(u[v][i], rstd, fmaf(z[v][i], along, across));
                if (kAdded) {
                    float more[kColumns];
                    Row::unpack(added[v], more);
#pragma unroll
                    for (int i = 0; i < kColumns; ++i)
                        u[v][i] += more[i];
                }
                store_within<true>(grad_x + (here ? row * vectors : 0), here ? vectors * 16 : 0, threadIdx.x + v * blockDim.x, Row::pack(u[v]));
            }
        }
    }
    if (sums == nullptr)
        return;
    // first of g * z, then of g; those of several teams in the order of the teams, four columns a thread of all of them
    constexpr int kQuads = kColumns / 4;  // of a vector
    const int quads = vectors * kQuads;
    u32x4* to = sums + 2 * group * quads;
#pragma unroll
    for (int which = 0; which < 2; ++which, to += quads) {
        if (which == 1 && means == nullptr)
            break;
        const auto& own = which == 0 ? sum_z : sum_g;
        const auto put = [&](u32x4* into) {
#pragma unroll
            for (int v = 0; v < kVectors; ++v) {
                const int at = threadIdx.x + v * blockDim.x;
                if (at < vectors)
#pragma unroll
                    for (int q = 0; q < kQuads; ++q)
                        into[at * kQuads + q] = RowType<Fp32>::pack({own[v][4 * q], own[v][4 * q + 1], own[v][4 * q + 2], own[v][4 * q + 3]});
            }
        };
        if (teams == 1) {
            put(to);
            continue;
        }
        __syncthreads();  // (the last sums are read)
        put(team_sums + team * quads);
        __syncthreads();
        for (int at = team * blockDim.x + threadIdx.x; at < quads; at += teams * blockDim.x) {
            float sum[4], more[4];
            RowType<Fp32>::unpack(team_sums[at], sum);
#pragma unroll 4
            for (int other = 1; other < teams; ++other) {
                RowType<Fp32>::unpack(team_sums[other * quads + at], more);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sum[i] += more[i];
            }
            to[at] = RowType<Fp32>::pack(sum);
        }
    }
}

// dgamma and dbeta from the workgroups' sums: 64 columns a workgroup, its 16 groups of 16 lanes share out the rows of sums, all loads of
// 16 rows on their way at once; then a thread a column adds up the groups'.  256 rows of 2 x 7168 (15 MB, from the last-level cache) 4.9 us.
constexpr int kSumLanes = 16, kSumGroups = 16, kSumRows = 16;
template <class P>
__global__ void __launch_bounds__(kSumLanes * kSumGroups) parameter_gradient_kernel(const u32x4* __restrict__ sums,  // [groups][2][columns / 4]
                                                                                    void* __restrict__ grad_gamma,
                                                                                    void* __restrict__ grad_beta,
                                                                                    int64_t groups,
                                                                                    int quads) {
    __shared__ float parts[kSumGroups][kSumLanes * 4];
    const int lane = threadIdx.x % kSumLanes, part = threadIdx.x / kSumLanes;
    const int at = blockIdx.x * kSumLanes + lane, from = at < quads ? at : 0;
    const int which = blockIdx.y;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t base = part; base < groups; base += kSumGroups * kSumRows) {
        u32x4 data[kSumRows];
#pragma unroll
        for (int r = 0; r < kSumRows; ++r) {
            const int64_t group = base + r * kSumGroups;
            data[r] = sums[(2 * (group < groups ? group : base) + which) * quads + from];
        }
#pragma unroll
        for (int r = 0; r < kSumRows; ++r)
            if (base + r * kSumGroups < groups)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sum[i] += __uint_as_float(data[r][i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        parts[part][lane * 4 + i] = sum[i];
    __syncthreads();
    const int column = blockIdx.x * kSumLanes * 4 + threadIdx.x;
    if (threadIdx.x >= kSumLanes * 4 || column >= quads * 4)
        return;
    float all = 0.0f;
#pragma unroll
    for (int other = 0; other < kSumGroups; ++other)
        all += parts[other][threadIdx.x];
    void* out = which == 0 ? grad_gamma : grad_beta;
    if constexpr (RowType<P>::kColumns == 8)
        static_cast<uint16_t*>(out)[column] = static_cast<uint16_t>(to_bf16_pair(all, 0.0f));
    else
        static_cast<float*>(out)[column] = all;
}

// Lanes and vectors a lane for rows of `vectors` vectors: two vectors a lane, more only where `most` lanes would not do.  By the
// row's length alone, so that a row's result is the same in any batch.
struct RowShape {
    int held;     // 1, 2, 4 or 8
    int threads;  // a multiple of 64
};
RowShape shape_of(int vectors, int most) {
    int held = vectors > kWave ? 2 : 1;
    while ((vectors + held - 1) / held > most)
        held *= 2;
    return {held, static_cast<int>(align_up(static_cast<size_t>((vectors + held - 1) / held), kWave))};
}

// Rows of a workgroup of the norm: several where a row takes few lanes.
int teams_of(int threads) { return std::max(1, kBlockThreads / threads); }

bool types_fit(int rows_type, int parameters_type) {
    return (rows_type == NANOEP_BF16 && (parameters_type == NANOEP_BF16 || parameters_type == NANOEP_FP32)) ||
           (rows_type == NANOEP_FP32 && parameters_type == NANOEP_FP32);
}

bool norm_sizes_fit(int64_t num_tokens, int hidden, int rows_type, int parameters_type) {
    return num_tokens >= 0 && num_tokens <= 0x7fffffff && hidden > 0 && hidden % 8 == 0 && hidden <= kMostHidden &&
           types_fit(rows_type, parameters_type);
}

// One workgroup a compute unit (or less), so that there are few rows of sums to write and to add up again.
struct BackwardPlan {
    RowShape shape;
    int vectors, teams;
    int64_t groups;
};
BackwardPlan plan_backward(int64_t num_tokens, int hidden, int rows_type, const Topology& topology) {
    BackwardPlan plan;
    plan.vectors = hidden / (rows_type == NANOEP_BF16 ? 8 : 4);
    plan.shape = shape_of(plan.vectors, kBackwardThreads);
    const int64_t most = topology.cus, rows_each = std::max<int64_t>(1, (num_tokens + most - 1) / most);
    plan.teams = static_cast<int>(std::min<int64_t>(kBackwardThreads / plan.shape.threads, rows_each));
    plan.groups = std::min(most, (num_tokens + plan.teams - 1) / plan.teams);
    return plan;
}

template <class T, class P>
int launch_norm(const void* x, const void* residual, const void* gamma, const void* beta, int64_t num_tokens, int hidden, float eps, void* total,
                void* normalized, float* mean, float* rstd, hipStream_t stream) {
    const int vectors = hidden / RowType<T>::kColumns;
    const RowShape shape = shape_of(vectors, kMostThreads);
    const int teams = teams_of(shape.threads);
    // 16 wavefronts a compute unit, the rows dealt out evenly (4096 x 7168 with a residual, two workgroups of seven: 37.6 us, one 39.4,
    // three 41.9, a row a workgroup 41.5)
    const int64_t most = int64_t{current_topology(current_tuning()).cus} * std::max(1, kMostRowWaves / (shape.threads / kWave * teams));
    const int64_t turns = (num_tokens + most * teams - 1) / (most * teams);
    const int64_t groups = (num_tokens + turns * teams - 1) / (turns * teams);
    const dim3 grid = grid_of(groups), block(shape.threads, teams);
    const auto launch = [&](auto kernel) {
        kernel<<<grid, block, 0, stream>>>(static_cast<const u32x4*>(x), static_cast<const u32x4*>(residual), static_cast<const u32x4*>(gamma),
                                           static_cast<const u32x4*>(beta), static_cast<u32x4*>(total), static_cast<u32x4*>(normalized), mean,
                                           rstd, num_tokens, groups, vectors, static_cast<float>(hidden), eps);
    };
    // Nontemporal loads or stores, by the bytes of all rows (us; nontemporal loads, nontemporal stores): 235 MB 38.2, 42.0; 196 MB
    // 32.1, 32.3; 134 MB 23.3, 21.2; 82 MB 15.9, 13.9.
    const int64_t bytes = num_tokens * vectors * 16 * (residual != nullptr ? 4 : 2);
    const bool past_cache = bytes > kLastLevelCacheBytes / 4 * 3;
    const auto pick = [&](auto near, auto far) { past_cache ? launch(far) : launch(near); };
    if (shape.held == 1)
        pick(layer_norm_kernel<T, P, 1, false>, layer_norm_kernel<T, P, 1, true>);
    else if (shape.held == 2)
        pick(layer_norm_kernel<T, P, 2, false>, layer_norm_kernel<T, P, 2, true>);
    else if constexpr (RowType<T>::kColumns == 4)  // (the longest rows in bf16 are two vectors a lane)
        pick(layer_norm_kernel<T, P, 4, false>, layer_norm_kernel<T, P, 4, true>);
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

template <class T, class P>
int launch_backward(const BackwardPlan& plan, const void* grad, const void* total, const void* gamma, const float* mean, const float* rstd,
                    const void* grad_residual, int64_t num_tokens, int hidden, void* grad_x, void* grad_gamma, void* grad_beta, void* workspace,
                    hipStream_t stream) {
    if (plan.groups > 0) {
        const size_t lds = grad_gamma != nullptr && plan.teams > 1 ? static_cast<size_t>(plan.teams) * hidden * sizeof(float) : 0;
        const dim3 grid(static_cast<unsigned>(plan.groups)), block(plan.shape.threads, plan.teams);
        const auto launch = [&](auto kernel) {
            kernel<<<grid, block, lds, stream>>>(static_cast<const u32x4*>(grad), static_cast<const u32x4*>(total),
                                                 static_cast<const u32x4*>(gamma), mean, rstd, static_cast<const u32x4*>(grad_residual),
                                                 static_cast<u32x4*>(grad_x), grad_gamma != nullptr ? static_cast<u32x4*>(workspace) : nullptr,
                                                 num_tokens, plan.groups, plan.vectors, static_cast<float>(hidden));
        };
        const auto pick = [&](auto vectors_held) {
            constexpr int kHeld = decltype(vectors_held)::value;
            if (grad_x == nullptr)
                launch(layer_norm_backward_kernel<T, P, kHeld, false, false>);
            else if (grad_residual == nullptr)
                launch(layer_norm_backward_kernel<T, P, kHeld, false, true>);
            else
                launch(layer_norm_backward_kernel<T, P, kHeld, true, true>);
        };
        if (plan.shape.held == 1)
            pick(std::integral_constant<int, 1>{});
        else if (plan.shape.held == 2)
            pick(std::integral_constant<int, 2>{});
        else if (plan.shape.held == 4)
            pick(std::integral_constant<int, 4>{});
        else if constexpr (RowType<T>::kColumns == 4)
            pick(std::integral_constant<int, 8>{});
        NANOEP_HIP_TRY(hipGetLastError());
    }
    if (grad_gamma != nullptr) {
        const int quads = hidden / 4;
        parameter_gradient_kernel<P><<<dim3((quads + kSumLanes - 1) / kSumLanes, grad_beta != nullptr ? 2 : 1), kSumLanes * kSumGroups, 0, stream>>>(
            static_cast<const u32x4*>(workspace), grad_gamma, grad_beta, plan.groups, quads);
        NANOEP_HIP_TRY(hipGetLastError());
    }
    return NANOEP_OK;
}

}  // namespace
}  // namespace nanoep

extern "C" {

int nanoep_layer_norm(const void* x, const void* residual, const void* gamma, const void* beta, int64_t num_tokens, int hidden, float eps,
                      int rows_type, int parameters_type, void* total, void* normalized, float* mean, float* rstd, void* stream) {
    using namespace nanoep;
    if (!norm_sizes_fit(num_tokens, hidden, rows_type, parameters_type) || !(eps >= 0.0f))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens == 0)  // (and the arrays of no rows may be NULL)
        return NANOEP_OK;
    if ((residual == nullptr) != (total == nullptr) || (mean == nullptr && beta != nullptr))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (x == nullptr || gamma == nullptr || normalized == nullptr || rstd == nullptr || !aligned16(x) || !aligned16(residual) ||
        !aligned16(gamma) || !aligned16(beta) || !aligned16(total) || !aligned16(normalized))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const auto on = static_cast<hipStream_t>(stream);
    const auto launch = rows_type == NANOEP_FP32         ? launch_norm<Fp32, Fp32>
                        : parameters_type == NANOEP_FP32 ? launch_norm<Bf16, Fp32>
                                                         : launch_norm<Bf16, Bf16>;
    return launch(x, residual, gamma, beta, num_tokens, hidden, eps, total, normalized, mean, rstd, on);
}

size_t nanoep_layer_norm_backward_workspace_bytes(int64_t num_tokens, int hidden, int rows_type) {
    using namespace nanoep;
    if (!norm_sizes_fit(num_tokens, hidden, rows_type, NANOEP_FP32))
        return 0;
    return static_cast<size_t>(plan_backward(num_tokens, hidden, rows_type, current_topology(current_tuning())).groups) * 2 * hidden * sizeof(float);
}

int nanoep_layer_norm_backward(const void* grad, const void* total, const void* gamma, const float* mean, const float* rstd,
                               const void* grad_residual, int64_t num_tokens, int hidden, int rows_type, int parameters_type, void* grad_x,
                               void* grad_gamma, void* grad_beta, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace nanoep;
    if (!norm_sizes_fit(num_tokens, hidden, rows_type, parameters_type) || (grad_beta != nullptr && grad_gamma == nullptr))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens > 0 && ((grad_x == nullptr && grad_gamma == nullptr) || (grad_beta != nullptr) != (grad_gamma != nullptr && mean != nullptr)))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (!aligned16(grad) || !aligned16(total) || !aligned16(gamma) || !aligned16(grad_residual) || !aligned16(grad_x) || !aligned16(grad_gamma) ||
        !aligned16(grad_beta) || !aligned16(workspace))
        return NANOEP_ERR_INVALID_ARGUMENT;
    if (num_tokens > 0 && (grad == nullptr || total == nullptr || gamma == nullptr || rstd == nullptr))
        return NANOEP_ERR_INVALID_ARGUMENT;
    const BackwardPlan plan = plan_backward(num_tokens, hidden, rows_type, current_topology(current_tuning()));
    if (grad_gamma != nullptr && plan.groups > 0) {
        if (workspace_bytes < static_cast<size_t>(plan.groups) * 2 * hidden * sizeof(float))
            return NANOEP_ERR_WORKSPACE;
        if (workspace == nullptr)
            return NANOEP_ERR_INVALID_ARGUMENT;
    }
    const auto on = static_cast<hipStream_t>(stream);
    const auto launch = rows_type == NANOEP_FP32         ? launch_backward<Fp32, Fp32>
                        : parameters_type == NANOEP_FP32 ? launch_backward<Bf16, Fp32>
                                                         : launch_backward<Bf16, Bf16>;
    return launch(plan, grad, total, gamma, mean, rstd, grad_residual, num_tokens, hidden, grad_x, grad_gamma, grad_beta, workspace, on);
}

}  // extern "C"
