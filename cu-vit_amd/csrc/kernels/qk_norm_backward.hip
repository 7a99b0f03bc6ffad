// The gradients of rotate_heads with a norm. For a head x with u = x (less its
// mean with kLayer), s = 1 / sqrt(mean(u^2) + epsilon) and n = u s, and the
// output's gradient turned back, d = rotation^-1(dy):
//   dgamma += d n,  dbeta += d,  g = d gamma,
//   dx = s (g - n mean(g n))            (kRms)
//   dx = s (g - mean(g) - n mean(g n))  (kLayer)
// Nothing of the forward is kept: x is read anyway, and s costs less than a load.
//
// Bound: HBM (x and dy read, dx written). A workgroup takes the query heads or the
// key heads (grid y) of consecutive tokens, so that a lane's values keep one gamma,
// and their sums for dgamma and dbeta stay in registers all along; the turns of all
// its tokens are computed at once, where a step of its own for each round of heads
// put a barrier and a load of positions in front of it (16 x 197 tokens of 12 heads
// in bf16: 15.1 us so, 12.6 now). At its end the teams' sums are added in LDS and
// written to the workspace, [part][gamma, beta][workgroup][head_dim]; a second
// launch adds those of the workgroups. Both orders are fixed by the sizes, no
// atomics.
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
    int block_tokens; // of a workgroup
    int chunk_tokens; // whose turns it holds at a time
    int log_team;
    float per_head[2]; // 1 / heads
    float inverse_dim;
    float epsilon;
    bool copy_whole;
    std::int64_t pitch; // elements from token to token
    Rotation rotation;
    const float* gamma[2];
    float* partial; // null: no gradient of gamma or beta is wanted
    bool wanted[2][2]; // of the query's and the key's: gamma's, beta's
};

template <typename T, int U, bool Vector, HeadNorm Norm, bool Adjacent>
__global__ __launch_bounds__(kThreads) void rotate_heads_backward_kernel(const T* in, const T* grad_out, T* grad_in,
                                                                         KernelArgs args) {
    extern __shared__ float4 lds_floats[];
    float* const lds = reinterpret_cast<float*>(lds_floats);
    const int part = static_cast<int>(blockIdx.y);
    const int heads = args.heads[part];
    const std::int64_t skip = static_cast<std::int64_t>(args.skip[part]) * args.head_dim;
    const int row_lo = static_cast<int>(blockIdx.x) * args.block_tokens;
    const int rows = min(args.block_tokens, args.rows - row_lo);
    if (part == 2) {
        copy_tokens(grad_out, grad_in, args.pitch, skip, heads * args.head_dim, row_lo, rows, args.copy_whole);
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

    // A step is a round of the teams' items of one chunk of tokens; the next
    // step's operands are on their way while one is computed.
    const int rounds = (args.chunk_tokens * heads + teams - 1) / teams;
    const int chunks = (rows + args.chunk_tokens - 1) / args.chunk_tokens;
    struct Step {
        std::int64_t at;
        int token; // of the chunk; -1: nothing for this team
        Run<T, U> x[2];
        Run<T, U> d[2];
    };
    auto chunk_rows = [&](int chunk) { return min(args.chunk_tokens, rows - chunk * args.chunk_tokens); };
    auto read = [&](int chunk, int round, Step& step) {
        const int item = round * teams + team;
        const int token = static_cast<int>((static_cast<float>(item) + 0.5F) * args.per_head[part]);
        step.token = item < chunk_rows(chunk) * heads ? token : -1;
        if (step.token >= 0) {
            step.at = (row_lo + chunk * args.chunk_tokens + token) * args.pitch + skip +
                      static_cast<std::int64_t>(item - token * heads) * args.head_dim;
            read_runs<T, U, Vector>(in + step.at, place, step.x);
            read_runs<T, U, Vector>(grad_out + step.at, place, step.d);
        }
    };
    auto process = [&](const Step& step) {
        if (step.token < 0) {
            return;
        }
        float n[2][U], d[2][U];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            widen<T, U>(step.x[r], n[r]);
            widen<T, U>(step.d[r], d[r]);
        }
        const float scale = normalise<Norm, Vector>(n[0], n[1], place, args.log_team, args.inverse_dim, args.epsilon);
        if (args.rotation.pairs > 0) {
            Turns<U> turns;
            read_turns<U, Vector, Adjacent>(lds + 2 * step.token * table_pitch(args.rotation.pairs), place,
                                            args.rotation.pairs, turns);
            turn_runs<U, Vector, Adjacent>(d[0], d[1], turns, place, args.rotation.pairs);
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
        write_runs<T, U, Vector, Vector>(grad_in + step.at, place, d[0], d[1]);
    };
    Step now, next;
    read(0, 0, now);
    for (int chunk = 0; chunk < chunks; ++chunk) {
        if (args.rotation.pairs > 0) {
            __syncthreads(); // the last chunk's turns are used
            fill_table(lds, args.rotation, row_lo + chunk * args.chunk_tokens, chunk_rows(chunk), args.tokens, -1.0F);
            __syncthreads();
        }
        for (int round = 0; round < rounds; ++round) {
            if (round + 1 < rounds) {
                read(chunk, round + 1, next);
            } else if (chunk + 1 < chunks) {
                read(chunk + 1, 0, next);
            }
            process(now);
            now = next;
        }
    }
    if (args.partial == nullptr) {
        return;
    }
    // The teams' sums, one row of head_dim a team, added by column.
    float* const sums = lds;
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
        if (!args.wanted[part][kind]) {
            continue;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (i < place.count[r]) {
                    sums[team * args.head_dim + place.at[r] + i] = kind == 0 ? sum_gamma[r][i] : sum_beta[r][i];
                }
        __syncthreads();
        float* const to = args.partial + (static_cast<std::int64_t>(2 * part + kind) * kMaxGroups + blockIdx.x) *
                                             args.head_dim;
        for (int column = thread; column < args.head_dim; column += kThreads) {
            float total = 0.0F;
#pragma unroll 8
            for (int t = 0; t < teams; ++t)
                total += sums[t * args.head_dim + column];
            to[column] = total;
        }
    }
}

/// Sixteen columns of one gradient: 64 threads a column, each over every 64th
/// workgroup's sums, all their loads in flight at once.
constexpr int kJoinRows = 64;
__global__ __launch_bounds__(16 * kJoinRows) void join_partials_kernel(const float* partial, HeadGradients gradients,
                                                                       int head_dim, int groups) {
    const int which = static_cast<int>(blockIdx.y); // 2 part + (0 gamma, 1 beta)
    float* const to = (which & 1) != 0 ? gradients.beta[which >> 1] : gradients.gamma[which >> 1];
    if (to == nullptr) {
        return;
    }
    __shared__ float sums[kJoinRows][17];
    const int column = static_cast<int>(threadIdx.x) & 15;
    const int row = static_cast<int>(threadIdx.x) >> 4;
    const int at = static_cast<int>(blockIdx.x) * 16 + column;
    const float* const from = partial + static_cast<std::int64_t>(which) * kMaxGroups * head_dim + at;
    float total = 0.0F;
#pragma unroll
    for (int i = 0; i < kMaxGroups / kJoinRows; ++i) {
        const int g = row + i * kJoinRows;
        total += at < head_dim && g < groups ? from[static_cast<std::int64_t>(g) * head_dim] : 0.0F;
    }
    sums[row][column] = total;
    __syncthreads();
    if (row < 16) { // threads 16 r .. + 15, a DPP row, add up column r
        total = 0.0F;
#pragma unroll
        for (int r = 0; r < kJoinRows / 16; ++r)
            total += sums[column + 16 * r][row];
        total = row16_allreduce(total, Sum{});
        if (column == 0 && static_cast<int>(blockIdx.x) * 16 + row < head_dim) {
            to[static_cast<int>(blockIdx.x) * 16 + row] = total;
        }
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
    // Workgroups of a part: kMaxGroups of them, or fewer with one full round each.
    const int most = a.q_heads > args.heads[1] ? a.q_heads : args.heads[1];
    const int round = teams / most > 0 ? teams / most : 1;
    const int share = (args.rows - 1) / kMaxGroups + 1;
    args.block_tokens = share > round ? share : round;
    const int groups = (args.rows - 1) / args.block_tokens + 1;
    // Their turns at a time: within 16 KiB, and 2^20 items (the kernel divides an
    // item by the heads in fp32, exact as far as that).
    const int by_table = a.rotation.pairs > 0 ? 2048 / table_pitch(a.rotation.pairs) : 64;
    const int by_items = (1 << 20) / most;
    const int held = by_table < by_items ? by_table : by_items;
    args.chunk_tokens = args.block_tokens < held ? args.block_tokens : held;
    for (int part = 0; part < 2; ++part) {
        args.per_head[part] = 1.0F / static_cast<float>(args.heads[part]);
        args.gamma[part] = a.gamma[part];
        args.wanted[part][0] = gradients.gamma[part] != nullptr;
        args.wanted[part][1] = gradients.beta[part] != nullptr;
    }
    const bool summed = gradients.gamma[0] != nullptr || gradients.gamma[1] != nullptr ||
                        gradients.beta[0] != nullptr || gradients.beta[1] != nullptr;
    args.partial = summed ? gradients.workspace : nullptr;
    constexpr int kPerVec = Elem<T>::kPerVec;
    args.copy_whole = a.copied * a.head_dim % kPerVec == 0 && a.heads * a.head_dim % kPerVec == 0 &&
                      args.pitch % kPerVec == 0 && aligned16(grad_output) && aligned16(grad_input);
    const std::size_t table = table_floats(args.chunk_tokens, a.rotation.pairs);
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
    join_partials_kernel<<<dim3(static_cast<unsigned int>((a.head_dim + 15) / 16), 4), 16 * kJoinRows, 0, stream>>>(
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
    // Runs of four in either type: of eight, a lane's sums and operands take 140
    // registers and leave three wavefronts a SIMD.
    if (whole(4)) {
        return launch<T, 4, true>(input, grad_output, grad_input, gradients, a, stream);
    }
    return loose_runs_of_four(a) ? launch<T, 4, false>(input, grad_output, grad_input, gradients, a, stream)
                                 : launch<T, 8, false>(input, grad_output, grad_input, gradients, a, stream);
}

} // namespace
} // namespace rotary

std::int64_t rotate_heads_workspace(int head_dim) {
    return static_cast<std::int64_t>(4) * rotary::kMaxGroups * head_dim * 4;
}

hipError_t rotate_heads_no_tokens(const HeadGradients& gradients, int head_dim, hipStream_t stream) {
    rotary::join_partials_kernel<<<dim3(static_cast<unsigned int>((head_dim + 15) / 16), 4), 16 * rotary::kJoinRows, 0,
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
