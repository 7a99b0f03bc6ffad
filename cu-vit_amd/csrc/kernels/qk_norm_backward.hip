// The gradients of rotate_heads with a norm. For a head x with u = x (less its
// mean with kLayer), s = 1 / sqrt(mean(u^2) + epsilon) and n = u s, and the
// output's gradient turned back, d = rotation^-1(dy):
//   dgamma += d n,  dbeta += d,  g = d gamma,
//   dx = s (g - n mean(g n))            (kRms)
//   dx = s (g - mean(g) - n mean(g n))  (kLayer)
// Nothing of the forward is kept: x is read anyway, and s costs less than a load.
//
// Bound: HBM (x and dy read, dx written). A workgroup takes the query heads or
// the key heads (grid y) of groups of tokens, so that a lane's values keep one
// gamma, and their sums for dgamma and dbeta stay in registers over all its
// groups. At its end the teams' sums are added in LDS and written to the
// workspace, [part][gamma, beta][workgroup][head_dim]; a second launch adds
// those of the workgroups. Both orders are fixed by the sizes, no atomics.
#include "rotary_common.hpp"

#include <type_traits>

namespace cuvit::detail {
namespace rotary {
namespace {

/// Workgroups of a part: two for each CU, which the parts together double.
constexpr int kMaxGroups = 512;

struct KernelArgs {
    int rows;
    int tokens;
    int heads[3]; // of queries, of keys, of values
    int skip[3];  // heads before them
    int head_dim;
    int block_tokens[3];
    int log_team;
    float per_head[2]; // 1 / heads
    float inverse_dim;
    float epsilon;
    bool copy_whole;
    std::int64_t pitch; // elements from token to token
    Rotation rotation;
    const float* gamma[2];
    float* partial; // null: no gradient of gamma or beta is wanted
};

template <typename T, int U, bool Vector, HeadNorm Norm, bool Adjacent>
__global__ __launch_bounds__(kThreads) void rotate_heads_backward_kernel(const T* in, const T* grad_out, T* grad_in,
                                                                         KernelArgs args) {
    extern __shared__ float4 lds_floats[];
    float* const lds = reinterpret_cast<float*>(lds_floats);
    const int part = static_cast<int>(blockIdx.y);
    const int block_tokens = args.block_tokens[part];
    const int heads = args.heads[part];
    const std::int64_t skip = static_cast<std::int64_t>(args.skip[part]) * args.head_dim;
    const int stride = static_cast<int>(gridDim.x);
    const int groups = (args.rows + block_tokens - 1) / block_tokens;
    if (part == 2) {
        for (int g = static_cast<int>(blockIdx.x); g < groups; g += stride) {
            const int row0 = g * block_tokens;
            copy_tokens(grad_out, grad_in, args.pitch, skip, heads * args.head_dim, row0,
                        min(block_tokens, args.rows - row0), args.copy_whole);
        }
        return;
    }
    const int thread = static_cast<int>(threadIdx.x);
    const int team = thread >> args.log_team;
    const int teams = kThreads >> args.log_team;
    const int lane = thread & ((1 << args.log_team) - 1);
    const Place place = place_of<U, Vector, Adjacent>(lane, args.head_dim, args.rotation.pairs);
    float gamma[2][U];
    float sum_gamma[2][U];
    float sum_beta[2][U];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const bool given = args.gamma[part] != nullptr && i < place.count[r];
            gamma[r][i] = given ? args.gamma[part][place.at[r] + i] : 1.0F;
            sum_gamma[r][i] = 0.0F;
            sum_beta[r][i] = 0.0F;
        }

    for (int g = static_cast<int>(blockIdx.x); g < groups; g += stride) {
        const int row0 = g * block_tokens;
        const int tokens = min(block_tokens, args.rows - row0);
        const int items = tokens * heads;
        bool filled = false;
        for (int base = 0; base < items; base += teams) {
            const int item = base + team;
            const int token = static_cast<int>((static_cast<float>(item) + 0.5F) * args.per_head[part]);
            const std::int64_t at =
                (row0 + token) * args.pitch + skip + static_cast<std::int64_t>(item - token * heads) * args.head_dim;
            Run<T, U> x_runs[2], d_runs[2];
            if (item < items) {
                read_runs<T, U, Vector>(in + at, place, x_runs);
                read_runs<T, U, Vector>(grad_out + at, place, d_runs);
            }
            if (!filled && args.rotation.pairs > 0) { // (the same for the whole workgroup)
                __syncthreads();                      // the last group's turns are used
                fill_table(lds, args.rotation, row0, tokens, args.tokens, -1.0F);
                __syncthreads();
            }
            filled = true;
            if (item >= items) {
                continue;
            }
            float n[2][U], d[2][U];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                widen<T, U>(x_runs[r], n[r]);
                widen<T, U>(d_runs[r], d[r]);
            }
            const float scale = normalise<Norm>(n[0], n[1], place, args.log_team, args.inverse_dim, args.epsilon);
            if (args.rotation.pairs > 0) {
                turn_runs<U, Vector, Adjacent>(d[0], d[1], lds + 2 * token * table_pitch(args.rotation.pairs), place,
                                               args.rotation.pairs);
            }
            float along = 0.0F; // sum of g n
            float sum = 0.0F;   // sum of g
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    n[r][i] *= scale;
                    sum_gamma[r][i] = fmaf(d[r][i], n[r][i], sum_gamma[r][i]);
                    sum_beta[r][i] += d[r][i];
                    d[r][i] *= gamma[r][i];
                    along = fmaf(d[r][i], n[r][i], along);
                    sum += d[r][i];
                }
            along = team_sum(along, args.log_team) * args.inverse_dim;
            if constexpr (Norm == HeadNorm::kLayer) {
                sum = team_sum(sum, args.log_team) * args.inverse_dim;
            } else {
                sum = 0.0F;
            }
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int i = 0; i < U; ++i)
                    d[r][i] = scale * (d[r][i] - fmaf(n[r][i], along, sum));
            write_runs<T, U, Vector>(grad_in + at, place, d[0], d[1]);
        }
    }
    if (args.partial == nullptr) {
        return;
    }
    // The teams' sums, one row of head_dim a team, added by column.
    float* const rows = lds;
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (i < place.count[r]) {
                    rows[team * args.head_dim + place.at[r] + i] = kind == 0 ? sum_gamma[r][i] : sum_beta[r][i];
                }
        __syncthreads();
        float* const to = args.partial + (static_cast<std::int64_t>(2 * part + kind) * kMaxGroups + blockIdx.x) *
                                             args.head_dim;
        for (int column = thread; column < args.head_dim; column += kThreads) {
            float total = 0.0F;
            for (int t = 0; t < teams; ++t)
                total += rows[t * args.head_dim + column];
            to[column] = total;
        }
    }
}

/// Sixteen columns of one gradient: sixteen threads a column, each over every
/// sixteenth workgroup's sums.
__global__ __launch_bounds__(kThreads) void join_partials_kernel(const float* partial, HeadGradients gradients,
                                                                 int head_dim, int groups) {
    const int which = static_cast<int>(blockIdx.y); // 2 part + (0 gamma, 1 beta)
    float* const to = (which & 1) != 0 ? gradients.beta[which >> 1] : gradients.gamma[which >> 1];
    if (to == nullptr) {
        return;
    }
    __shared__ float sums[16][17];
    const int column = static_cast<int>(threadIdx.x) & 15;
    const int row = static_cast<int>(threadIdx.x) >> 4;
    const int at = static_cast<int>(blockIdx.x) * 16 + column;
    float total = 0.0F;
    if (at < head_dim) {
        const float* const from = partial + static_cast<std::int64_t>(which) * kMaxGroups * head_dim + at;
#pragma unroll 8
        for (int g = row; g < groups; g += 16)
            total += from[static_cast<std::int64_t>(g) * head_dim];
    }
    sums[row][column] = total;
    __syncthreads();
    if (row == 0 && at < head_dim) {
        for (int r = 1; r < 16; ++r)
            total += sums[r][column];
        to[at] = total;
    }
}

template <typename T, int U, bool Vector>
hipError_t launch(const T* input, const T* grad_output, T* grad_input, const HeadGradients& gradients,
                  const HeadArgs& a, hipStream_t stream) {
    KernelArgs args{};
    args.rows = a.images * a.tokens;
    args.tokens = a.tokens;
    args.heads[0] = a.q_heads;
    args.heads[1] = a.heads - a.q_heads;
    args.heads[2] = a.copied;
    args.skip[1] = a.q_heads;
    args.skip[2] = a.heads;
    args.head_dim = a.head_dim;
    args.log_team = log_team_of(lanes_of_head(U, a.rotation.adjacent, a.head_dim, a.rotation.pairs));
    args.inverse_dim = 1.0F / static_cast<float>(a.head_dim);
    args.epsilon = a.epsilon;
    args.pitch = a.input.token;
    args.rotation = a.rotation;
    const int teams = kThreads >> args.log_team;
    const int spread = args.rows / kMaxGroups + 1;
    int groups = 0;
    for (int part = 0; part < 3; ++part) {
        const int full = teams / args.heads[part] > 0 ? teams / args.heads[part] : 1;
        args.block_tokens[part] = full < spread ? full : spread;
        const int of_part = (args.rows + args.block_tokens[part] - 1) / args.block_tokens[part];
        groups = groups < of_part ? of_part : groups;
        if (part < 2) {
            args.per_head[part] = 1.0F / static_cast<float>(args.heads[part]);
            args.gamma[part] = a.gamma[part];
        }
    }
    groups = groups < kMaxGroups ? groups : kMaxGroups;
    const bool summed = gradients.gamma[0] != nullptr || gradients.gamma[1] != nullptr ||
                        gradients.beta[0] != nullptr || gradients.beta[1] != nullptr;
    args.partial = summed ? gradients.workspace : nullptr;
    constexpr int kPerVec = Elem<T>::kPerVec;
    args.copy_whole = a.copied * a.head_dim % kPerVec == 0 && a.heads * a.head_dim % kPerVec == 0 &&
                      args.pitch % kPerVec == 0 && aligned16(grad_output) && aligned16(grad_input);
    const int most = args.block_tokens[0] > args.block_tokens[1] ? args.block_tokens[0] : args.block_tokens[1];
    const std::size_t table = table_floats(most, a.rotation.pairs);
    const std::size_t sums = summed ? static_cast<std::size_t>(teams) * a.head_dim : 0;
    const std::size_t lds = 4 * (table > sums ? table : sums);
    const dim3 grid(static_cast<unsigned int>(groups), grad_input == grad_output ? 2U : 3U);
    auto run = [&](auto kernel) -> hipError_t {
        if (const hipError_t opted = allow_lds<decltype(kernel)::kValue>(lds); opted != hipSuccess) {
            return opted;
        }
        decltype(kernel)::kValue<<<grid, kThreads, lds, stream>>>(input, grad_output, grad_input, args);
        return hipGetLastError();
    };
    auto with_norm = [&](auto adjacent) -> hipError_t {
        constexpr bool kAdjacent = decltype(adjacent)::value;
        return a.norm == HeadNorm::kRms
                   ? run(KernelConstant<rotate_heads_backward_kernel<T, U, Vector, HeadNorm::kRms, kAdjacent>>{})
                   : run(KernelConstant<rotate_heads_backward_kernel<T, U, Vector, HeadNorm::kLayer, kAdjacent>>{});
    };
    const hipError_t launched = a.rotation.adjacent ? with_norm(std::true_type{}) : with_norm(std::false_type{});
    if (launched != hipSuccess || !summed) {
        return launched;
    }
    join_partials_kernel<<<dim3(static_cast<unsigned int>((a.head_dim + 15) / 16), 4), kThreads, 0, stream>>>(
        gradients.workspace, gradients, a.head_dim, groups);
    return hipGetLastError();
}

template <typename T>
hipError_t pick(const T* input, const T* grad_output, T* grad_input, const HeadGradients& gradients,
                const HeadArgs& a, hipStream_t stream) {
    const std::uintptr_t addresses = reinterpret_cast<std::uintptr_t>(input) |
                                     reinterpret_cast<std::uintptr_t>(grad_output) |
                                     reinterpret_cast<std::uintptr_t>(grad_input);
    auto whole = [&](int unit) {
        return whole_runs(unit, sizeof(T), addresses, a.head_dim, a.head_dim, a.rotation.pairs, a.rotation.adjacent);
    };
    constexpr int kUnit = Elem<T>::kPerVec;
    if (whole(kUnit)) {
        return launch<T, kUnit, true>(input, grad_output, grad_input, gradients, a, stream);
    }
    if constexpr (sizeof(T) == 2) {
        if (whole(4)) {
            return launch<T, 4, true>(input, grad_output, grad_input, gradients, a, stream);
        }
    }
    return launch<T, 8, false>(input, grad_output, grad_input, gradients, a, stream);
}

} // namespace
} // namespace rotary

std::int64_t rotate_heads_workspace(int head_dim) {
    return static_cast<std::int64_t>(4) * rotary::kMaxGroups * head_dim * 4;
}

hipError_t rotate_heads_no_tokens(const HeadGradients& gradients, int head_dim, hipStream_t stream) {
    rotary::join_partials_kernel<<<dim3(static_cast<unsigned int>((head_dim + 15) / 16), 4), rotary::kThreads, 0,
                                   stream>>>(gradients.workspace, gradients, head_dim, 0);
    return hipGetLastError();
}

hipError_t rotate_heads_backward(const float* input, const float* grad_output, float* grad_input,
                                 const HeadGradients& gradients, const HeadArgs& args, hipStream_t stream) {
    return rotary::pick(input, grad_output, grad_input, gradients, args, stream);
}

hipError_t rotate_heads_backward(const std::uint16_t* input, const std::uint16_t* grad_output,
                                 std::uint16_t* grad_input, const HeadGradients& gradients, const HeadArgs& args,
                                 hipStream_t stream) {
    return rotary::pick(input, grad_output, grad_input, gradients, args, stream);
}

} // namespace cuvit::detail
