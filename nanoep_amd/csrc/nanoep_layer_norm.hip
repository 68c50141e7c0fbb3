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

#include "nanoep_lanes.h"
#include "nanoep_operators.h"

namespace nanoep {
namespace {

constexpr int kMostThreads = 1024;
constexpr int kMostHidden = 16384;

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

// The parameters beside a row's vector `at`: as wide as its values, or fp32 beside bf16.
template <class P, int kColumns>
__device__ __forceinline__ void load_parameters(const u32x4* parameters, int at, float (&out)[kColumns]) {
    if constexpr (RowType<P>::kColumns == kColumns) {
        RowType<P>::unpack(parameters[at], out);
    } else {
        static_assert(kColumns == 8 && RowType<P>::kColumns == 4, "fp32 beside bf16");
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const u32x4 data = parameters[2 * at + half];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                out[4 * half + i] = __uint_as_float(data[i]);
        }
    }
}

// The sums over the wavefronts that share a row, in all of them.  One barrier; `place` is not used again before the next one.
template <int kValues>
__device__ __forceinline__ void row_sums(float (&v)[kValues], float (*place)[kValues], int first_wave, int wave, int waves) {
#pragma unroll
    for (int i = 0; i < kValues; ++i)
        v[i] = lanes_sum<kWave>(v[i]);
    if (waves == 1)
        return;
    if (threadIdx.x % kWave == 0)
#pragma unroll
        for (int i = 0; i < kValues; ++i)
            place[first_wave + wave][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kValues; ++i)
        v[i] = 0.0f;
    for (int w = 0; w < waves; ++w)
#pragma unroll
        for (int i = 0; i < kValues; ++i)
            v[i] += place[first_wave + w][i];
}

// blockDim.x lanes a row, blockDim.y rows; the row stays in registers (kVectors 16-byte vectors a lane) between its two
// sums and its output, so that every input byte is read once.
template <class T, class P, int kVectors>
__global__ void __launch_bounds__(kMostThreads) layer_norm_kernel(const u32x4* __restrict__ x,         // [T][vectors]
                                                                  const u32x4* __restrict__ residual,  // [T][vectors] or null
                                                                  const u32x4* __restrict__ gamma,
                                                                  const u32x4* __restrict__ beta,  // null: none
                                                                  u32x4* __restrict__ total,       // [T][vectors], null exactly when residual is
                                                                  u32x4* __restrict__ normalized,
                                                                  float* __restrict__ means,  // [T], null: the root-mean-square norm
                                                                  float* __restrict__ rstds,  // [T]
                                                                  int64_t rows,
                                                                  int vectors,
                                                                  float columns,
                                                                  float eps) {
    using Row = RowType<T>;
    constexpr int kColumns = Row::kColumns;
    __shared__ float places[2][kMostThreads / kWave][1];
    const int waves = blockDim.x / kWave, wave = threadIdx.x / kWave, first_wave = threadIdx.y * waves;
    const int64_t row = workgroup_number() * blockDim.y + threadIdx.y;
    const bool here = row < rows;
    const int64_t base = here ? row * vectors : 0;
    const int mine = here ? vectors : 0;  // (a row past the end has no vectors, but stays for the barriers)

    float s[kVectors][kColumns];
    u32x4 data[kVectors], other[kVectors];
    if (residual != nullptr) {
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const int at = threadIdx.x + v * blockDim.x;
            other[v] = at < mine ? residual[base + at] : u32x4{0u, 0u, 0u, 0u};
        }
    }
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = threadIdx.x + v * blockDim.x;
        data[v] = at < mine ? x[base + at] : u32x4{0u, 0u, 0u, 0u};
    }
    float factor[kVectors][kColumns], shift[kVectors][kColumns];
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = threadIdx.x + v * blockDim.x;
        const int from = at < vectors ? at : 0;
        load_parameters<P>(gamma, from, factor[v]);
        if (beta != nullptr)
            load_parameters<P>(beta, from, shift[v]);
    }
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        Row::unpack(data[v], s[v]);
        if (residual != nullptr) {
            const int at = threadIdx.x + v * blockDim.x;
            float added[kColumns];
            Row::unpack(other[v], added);
#pragma unroll
            for (int i = 0; i < kColumns; ++i)
                s[v][i] += added[i];
            const u32x4 packed = Row::pack(s[v]);
            if (at < mine)
                store_vec<true>(total + base + at, packed);
            Row::unpack(packed, s[v]);
        }
    }
    float mean = 0.0f;
    if (means != nullptr) {
        float sum[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
#pragma unroll
            for (int i = 0; i < kColumns; ++i)
                sum[0] += s[v][i];
        row_sums<1>(sum, places[0], first_wave, wave, waves);
        mean = sum[0] / columns;
    }
    float squares[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const bool in_row = static_cast<int>(threadIdx.x + v * blockDim.x) < mine;
#pragma unroll
        for (int i = 0; i < kColumns; ++i) {
            s[v][i] = in_row ? s[v][i] - mean : 0.0f;
            squares[0] = fmaf(s[v][i], s[v][i], squares[0]);
        }
    }
    row_sums<1>(squares, places[1], first_wave, wave, waves);
    const float rstd = 1.0f / sqrtf(squares[0] / columns + eps);
    if (threadIdx.x == 0 && here) {
        rstds[row] = rstd;
        if (means != nullptr)
            means[row] = mean;
    }
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = threadIdx.x + v * blockDim.x;
        if (at < mine) {
            float y[kColumns];
#pragma unroll
            for (int i = 0; i < kColumns; ++i) {
                y[i] = s[v][i] * rstd * factor[v][i];
                if (beta != nullptr)
                    y[i] += shift[v][i];
            }
            store_vec<true>(normalized + base + at, Row::pack(y));
        }
    }
}

// The gradient.  A workgroup works through rows of its own (`per_team` rows a team of blockDim.x lanes) and keeps the two sums
// over rows in registers; at its end it writes them, added over its teams, to its row of `sums` ([workgroups][2][columns] fp32),
// which parameter_gradient_kernel adds up in a fixed order.  No atomics.
template <class T, class P, int kVectors>
__global__ void __launch_bounds__(kMostThreads) layer_norm_backward_kernel(const u32x4* __restrict__ grad,   // [T][vectors]
                                                                           const u32x4* __restrict__ total,  // [T][vectors]
                                                                           const u32x4* __restrict__ gamma,
                                                                           const float* __restrict__ means,  // null: the root-mean-square norm
                                                                           const float* __restrict__ rstds,
                                                                           const u32x4* __restrict__ grad_residual,  // [T][vectors] or null
                                                                           u32x4* __restrict__ grad_x,               // [T][vectors] or null
                                                                           float* __restrict__ sums,                 // null: not wanted
                                                                           int64_t rows,
                                                                           int64_t per_team,
                                                                           int vectors,
                                                                           float columns) {
    using Row = RowType<T>;
    constexpr int kColumns = Row::kColumns;
    __shared__ float places[2][kMostThreads / kWave][2];
    extern __shared__ float team_sums[];  // [blockDim.y - 1][columns], if there are several teams
    const int waves = blockDim.x / kWave, wave = threadIdx.x / kWave, first_wave = threadIdx.y * waves;
    const int teams = blockDim.y;
    const int64_t group = workgroup_number();

    float factor[kVectors][kColumns], sum_z[kVectors][kColumns], sum_g[kVectors][kColumns];
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int at = threadIdx.x + v * blockDim.x;
        load_parameters<P>(gamma, at < vectors ? at : 0, factor[v]);
#pragma unroll
        for (int i = 0; i < kColumns; ++i)
            sum_z[v][i] = sum_g[v][i] = 0.0f;
    }
    for (int64_t turn = 0; turn < per_team; ++turn) {
        const int64_t row = (group * per_team + turn) * teams + threadIdx.y;
        const bool here = row < rows;
        const int64_t base = here ? row * vectors : 0;
        const int mine = here ? vectors : 0;
        u32x4 data[kVectors], grads[kVectors], added[kVectors];
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const int at = threadIdx.x + v * blockDim.x;
            data[v] = at < mine ? load_vec<true>(total + base + at) : u32x4{0u, 0u, 0u, 0u};
            grads[v] = at < mine ? load_vec<true>(grad + base + at) : u32x4{0u, 0u, 0u, 0u};
            if (grad_residual != nullptr)
                added[v] = at < mine ? load_vec<true>(grad_residual + base + at) : u32x4{0u, 0u, 0u, 0u};
        }
        const float rstd = here ? rstds[row] : 0.0f, mean = here && means != nullptr ? means[row] : 0.0f;
        float z[kVectors][kColumns], u[kVectors][kColumns], both[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const bool in_row = static_cast<int>(threadIdx.x + v * blockDim.x) < mine;
            Row::unpack(data[v], z[v]);
            Row::unpack(grads[v], u[v]);
#pragma unroll
            for (int i = 0; i < kColumns; ++i) {
                const float g = u[v][i];
                z[v][i] = in_row ? (z[v][i] - mean) * rstd : 0.0f;
                u[v][i] = in_row ? g * factor[v][i] : 0.0f;
                sum_g[v][i] += g;
                sum_z[v][i] = fmaf(g, z[v][i], sum_z[v][i]);
                both[0] += u[v][i];
                both[1] = fmaf(u[v][i], z[v][i], both[1]);
            }
        }
        if (grad_x != nullptr) {
            row_sums<2>(both, places[turn % 2], first_wave, wave, waves);
            const float across = means != nullptr ? both[0] / columns : 0.0f, along = both[1] / columns;
#pragma unroll
            for (int v = 0; v < kVectors; ++v) {
                const int at = threadIdx.x + v * blockDim.x;
                if (at < mine) {
                    float out[kColumns], more[kColumns];
                    if (grad_residual != nullptr)
                        Row::unpack(added[v], more);
#pragma unroll
                    for (int i = 0; i < kColumns; ++i) {
                        out[i] = (u[v][i] - across - z[v][i] * along) * rstd;
                        if (grad_residual != nullptr)
                            out[i] += more[i];
                    }
                    store_vec<true>(grad_x + base + at, Row::pack(out));
                }
            }
        }
    }
    if (sums == nullptr)
        return;
    // the teams' sums in the order of the teams, first of g * z, then of g
    const int64_t width = static_cast<int64_t>(vectors) * kColumns;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (which == 1 && means == nullptr)
            break;
        auto& own = which == 0 ? sum_z : sum_g;
        if (teams > 1) {
            __syncthreads();
            if (threadIdx.y > 0)
#pragma unroll
                for (int v = 0; v < kVectors; ++v) {
                    const int at = threadIdx.x + v * blockDim.x;
                    if (at < vectors)
#pragma unroll
                        for (int i = 0; i < kColumns; ++i)
                            team_sums[(threadIdx.y - 1) * width + at * kColumns + i] = own[v][i];
                }
            __syncthreads();
        }
        if (threadIdx.y == 0)
#pragma unroll
            for (int v = 0; v < kVectors; ++v) {
                const int at = threadIdx.x + v * blockDim.x;
                if (at >= vectors)
                    continue;
                for (int team = 1; team < teams; ++team)
#pragma unroll
                    for (int i = 0; i < kColumns; ++i)
                        own[v][i] += team_sums[(team - 1) * width + at * kColumns + i];
                float* to = sums + (2 * group + which) * width + static_cast<int64_t>(at) * kColumns;
#pragma unroll
                for (int i = 0; i < kColumns; i += 4)
                    *reinterpret_cast<u32x4*>(to + i) = RowType<Fp32>::pack({own[v][i], own[v][i + 1], own[v][i + 2], own[v][i + 3]});
            }
    }
}

// dgamma and dbeta from the workgroups' sums: 64 columns a workgroup, its 16 groups of 16 lanes share out the rows of sums.
constexpr int kSumLanes = 16, kSumGroups = 16;
template <class P>
__global__ void __launch_bounds__(kSumLanes * kSumGroups) parameter_gradient_kernel(const u32x4* __restrict__ sums,  // [groups][2][columns / 4]
                                                                                    void* __restrict__ grad_gamma,
                                                                                    void* __restrict__ grad_beta,
                                                                                    int64_t groups,
                                                                                    int quads) {
    __shared__ float parts[kSumGroups][kSumLanes][4];
    const int lane = threadIdx.x % kSumLanes, part = threadIdx.x / kSumLanes;
    const int at = blockIdx.x * kSumLanes + lane;
    const int which = blockIdx.y;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (at < quads) {
#pragma unroll 8
        for (int64_t group = part; group < groups; group += kSumGroups) {
            const u32x4 data = sums[(2 * group + which) * quads + at];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sum[i] += __uint_as_float(data[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        parts[part][lane][i] = sum[i];
    __syncthreads();
    if (part > 0 || at >= quads)
        return;
    for (int other = 1; other < kSumGroups; ++other)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            sum[i] += parts[other][lane][i];
    void* out = which == 0 ? grad_gamma : grad_beta;
    if constexpr (RowType<P>::kColumns == 8)
        static_cast<uint2*>(out)[at] = make_uint2(to_bf16_pair(sum[0], sum[1]), to_bf16_pair(sum[2], sum[3]));
    else
        static_cast<u32x4*>(out)[at] = RowType<Fp32>::pack(sum);
}

// Lanes and vectors a lane for rows of `vectors` vectors: two vectors a lane, more only where 1024 lanes would not do.  By the
// row's length alone, so that a row's result is the same in any batch.
struct RowShape {
    int held;     // 1, 2 or 4
    int threads;  // a multiple of 64
};
RowShape shape_of(int vectors) {
    int held = vectors > kWave ? 2 : 1;
    while ((vectors + held - 1) / held > kMostThreads)
        held *= 2;
    return {held, static_cast<int>(align_up(static_cast<size_t>((vectors + held - 1) / held), kWave))};
}

// Rows of a workgroup: several where a row takes few lanes.
int teams_of(int threads) { return std::max(1, kBlockThreads / threads); }

bool types_fit(int rows_type, int parameters_type) {
    return (rows_type == NANOEP_BF16 && (parameters_type == NANOEP_BF16 || parameters_type == NANOEP_FP32)) ||
           (rows_type == NANOEP_FP32 && parameters_type == NANOEP_FP32);
}

bool norm_sizes_fit(int64_t num_tokens, int hidden, int rows_type, int parameters_type) {
    return num_tokens >= 0 && num_tokens <= 0x7fffffff && hidden > 0 && hidden % 8 == 0 && hidden <= kMostHidden &&
           types_fit(rows_type, parameters_type);
}

struct BackwardPlan {
    RowShape shape;
    int vectors, teams;
    int64_t per_team, groups;
};
BackwardPlan plan_backward(int64_t num_tokens, int hidden, int rows_type, const Topology& topology) {
    BackwardPlan plan;
    plan.vectors = hidden / (rows_type == NANOEP_BF16 ? 8 : 4);
    plan.shape = shape_of(plan.vectors);
    plan.teams = teams_of(plan.shape.threads);
    const int64_t most = 2 * int64_t{topology.cus};
    plan.per_team = std::max<int64_t>(1, (num_tokens + most * plan.teams - 1) / (most * plan.teams));
    plan.groups = (num_tokens + plan.per_team * plan.teams - 1) / (plan.per_team * plan.teams);
    return plan;
}

template <class T, class P>
int launch_norm(const void* x, const void* residual, const void* gamma, const void* beta, int64_t num_tokens, int hidden, float eps, void* total,
                void* normalized, float* mean, float* rstd, hipStream_t stream) {
    const int vectors = hidden / RowType<T>::kColumns;
    const RowShape shape = shape_of(vectors);
    const int teams = teams_of(shape.threads);
    const dim3 grid = grid_of((num_tokens + teams - 1) / teams), block(shape.threads, teams);
    const auto launch = [&](auto kernel) {
        kernel<<<grid, block, 0, stream>>>(static_cast<const u32x4*>(x), static_cast<const u32x4*>(residual), static_cast<const u32x4*>(gamma),
                                           static_cast<const u32x4*>(beta), static_cast<u32x4*>(total), static_cast<u32x4*>(normalized), mean,
                                           rstd, num_tokens, vectors, static_cast<float>(hidden), eps);
    };
    if (shape.held == 1)
        launch(layer_norm_kernel<T, P, 1>);
    else if (shape.held == 2)
        launch(layer_norm_kernel<T, P, 2>);
    else if constexpr (RowType<T>::kColumns == 4)  // (the longest rows in bf16 are two vectors a lane)
        launch(layer_norm_kernel<T, P, 4>);
    NANOEP_HIP_TRY(hipGetLastError());
    return NANOEP_OK;
}

template <class T, class P>
int launch_backward(const BackwardPlan& plan, const void* grad, const void* total, const void* gamma, const float* mean, const float* rstd,
                    const void* grad_residual, int64_t num_tokens, int hidden, void* grad_x, void* grad_gamma, void* grad_beta, void* workspace,
                    hipStream_t stream) {
    if (plan.groups > 0) {
        const size_t lds = grad_gamma != nullptr ? static_cast<size_t>(plan.teams - 1) * hidden * sizeof(float) : 0;
        const dim3 grid = grid_of(plan.groups), block(plan.shape.threads, plan.teams);
        const auto launch = [&](auto kernel) {
            kernel<<<grid, block, lds, stream>>>(static_cast<const u32x4*>(grad), static_cast<const u32x4*>(total),
                                                 static_cast<const u32x4*>(gamma), mean, rstd, static_cast<const u32x4*>(grad_residual),
                                                 static_cast<u32x4*>(grad_x), grad_gamma != nullptr ? static_cast<float*>(workspace) : nullptr,
                                                 num_tokens, plan.per_team, plan.vectors, static_cast<float>(hidden));
        };
        if (plan.shape.held == 1)
            launch(layer_norm_backward_kernel<T, P, 1>);
        else if (plan.shape.held == 2)
            launch(layer_norm_backward_kernel<T, P, 2>);
        else if constexpr (RowType<T>::kColumns == 4)
            launch(layer_norm_backward_kernel<T, P, 4>);
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
