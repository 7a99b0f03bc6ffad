// Heads rotated by their tokens' positions, after a norm of each head if asked
// for: out = rotation(norm(x) gamma + beta), heads of any strides.
//
// Bound: HBM. Each value is read once and written once; a value takes about 7
// instructions with a norm, 3 without.
//
// Results go out non-temporally (64 x 197 tokens of 24 heads of 64 in bf16, with
// their values copied: 26.0 -> 20.8 us, a plain copy of the same bytes 23.3; 4 x 3136
// of 12, rotated, 9.5 -> 8.3, a copy 6.8), but in place, where the lines are in the
// caches and what reads them comes next. With attention reading the result at once
// the two calls take as long either way: in bf16, with plain stores in brackets, 51.0
// (50.8) at 64 x 197, 17.8 (18.3) at 16 x 197, 11.8 (11.5) at one image; in fp32 158
// (155) at 64 x 197. In place they take 43.6 at 64 x 197 in bf16, 144 in fp32.
//
// A workgroup takes whole tokens with all their heads, as many as its teams have
// items for, so that the turns of a token are computed once for all its heads and
// a token's heads, which lie side by side, are read side by side.
#include "rotary_common.hpp"

#include <type_traits>

namespace cuvit::detail {
namespace rotary {
namespace {

struct KernelArgs {
    int rows;         // images * tokens
    int tokens;
    int heads;
    int q_heads;
    int copied;
    int head_dim;
    int block_tokens; // of a workgroup
    int log_team;
    float per_head;   // 1 / heads
    float inverse_dim;
    float epsilon;
    bool flat_input;  // images follow one another like tokens
    bool flat_output;
    bool copy_whole;  // copied heads in 16-byte pieces
    HeadStrides input;
    HeadStrides output;
    Rotation rotation;
    const float* gamma[2];
    const float* beta[2];
};

/// (in and out may be the same memory: a lane reads its values before it writes them.)
template <typename T, int U, bool Vector, HeadNorm Norm, bool Adjacent, bool Streaming>
__global__ __launch_bounds__(kThreads) void rotate_heads_kernel(const T* in, T* out, KernelArgs args) {
    extern __shared__ float4 lds_floats[];
    const int row0 = static_cast<int>(blockIdx.x) * args.block_tokens;
    const int tokens = min(args.block_tokens, args.rows - row0);
    if (blockIdx.y != 0) {
        copy_tokens(in, out, args.input.token, args.heads * args.input.head, args.copied * args.head_dim, row0, tokens,
                    args.copy_whole);
        return;
    }
    // LDS: gamma and beta of the query and of the key heads, then the turns.
    constexpr bool kNorm = Norm != HeadNorm::kNone;
    const int width = (args.head_dim + 3) / 4 * 4;
    float* const weights = reinterpret_cast<float*>(lds_floats);
    float* const table = weights + (kNorm ? 4 * width : 0);
    const bool with_beta = kNorm && (args.beta[0] != nullptr || args.beta[1] != nullptr);

    const int thread = static_cast<int>(threadIdx.x);
    const int team = thread >> args.log_team;
    const int teams = kThreads >> args.log_team;
    const int lane = thread & ((1 << args.log_team) - 1);
    const Place place = place_of<U, Vector, Adjacent>(lane, args.head_dim, args.rotation.pairs);
    const int items = tokens * args.heads;

    constexpr int kTogether = 2;
    Run<T, U> raw[kTogether][2];
    int token[kTogether], head[kTogether];
    auto read = [&](int base) {
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            const int item = base + k * teams + team;
            // item / heads: exact, as items stay far below 2^20.
            token[k] = static_cast<int>((static_cast<float>(item) + 0.5F) * args.per_head);
            head[k] = item - token[k] * args.heads;
            if (item < items) {
                const T* const from =
                    in + token_offset(args.input, args.flat_input, row0 + token[k], args.tokens) + head[k] * args.input.head;
                read_runs<T, U, Vector>(from, place, raw[k]);
            }
        }
    };
    read(0);

    if (args.rotation.pairs > 0) {
        fill_table(table, args.rotation, row0, tokens, args.tokens, args.rotation.inverse ? -1.0F : 1.0F);
    }
    if constexpr (kNorm) {
        for (int i = thread; i < 2 * args.head_dim; i += kThreads) {
            const int part = i >= args.head_dim ? 1 : 0;
            const int column = i - part * args.head_dim;
            weights[2 * part * width + column] = args.gamma[part] != nullptr ? args.gamma[part][column] : 1.0F;
            weights[(2 * part + 1) * width + column] = args.beta[part] != nullptr ? args.beta[part][column] : 0.0F;
        }
    }
    __syncthreads();

    for (int base = 0; base < items; base += kTogether * teams) {
        if (base > 0) {
            read(base);
        }
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            if (base + k * teams + team >= items) {
                continue;
            }
            float first[U], second[U];
            widen<T, U>(raw[k][0], first);
            widen<T, U>(raw[k][1], second);
            if constexpr (kNorm) {
                const float scale =
                    normalise<Norm, Vector>(first, second, place, args.log_team, args.inverse_dim, args.epsilon);
                const float* const gamma = weights + (head[k] < args.q_heads ? 0 : 2 * width);
                auto scaled = [&](float(&v)[U], int r) {
                    float g[U], b[U];
                    read_floats<U, Vector>(gamma + place.at[r], g);
                    if (with_beta) {
                        read_floats<U, Vector>(gamma + width + place.at[r], b);
#pragma unroll
                        for (int i = 0; i < U; ++i)
                            v[i] = fmaf(v[i], scale * g[i], b[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < U; ++i)
                            v[i] *= scale * g[i];
                    }
                };
                scaled(first, 0);
                scaled(second, 1);
            }
            if (args.rotation.pairs > 0) {
                Turns<U> turns;
                read_turns<U, Vector, Adjacent>(table + 2 * token[k] * table_pitch(args.rotation.pairs), place,
                                                args.rotation.pairs, turns);
                turn_runs<U, Vector, Adjacent>(first, second, turns, place, args.rotation.pairs);
            }
            T* const to = out + token_offset(args.output, args.flat_output, row0 + token[k], args.tokens) +
                          head[k] * args.output.head;
            write_runs<T, U, Vector, Streaming>(to, place, first, second);
        }
    }
}

template <typename T, int U, bool Vector>
hipError_t launch(const T* input, T* output, const HeadArgs& a, hipStream_t stream) {
    const Rotation& rotation = a.rotation;
    KernelArgs args{};
    args.rows = a.images * a.tokens;
    args.tokens = a.tokens;
    args.heads = a.heads;
    args.q_heads = a.q_heads;
    args.copied = input == output ? 0 : a.copied;
    args.head_dim = a.head_dim;
    args.log_team = log_team_of(lanes_of_head(U, rotation.adjacent, a.head_dim, rotation.pairs));
    args.per_head = 1.0F / static_cast<float>(a.heads);
    args.inverse_dim = 1.0F / static_cast<float>(a.head_dim);
    args.epsilon = a.epsilon;
    args.flat_input = a.images == 1 || a.input.image == a.tokens * a.input.token;
    args.flat_output = a.images == 1 || a.output.image == a.tokens * a.output.token;
    args.input = a.input;
    args.output = a.output;
    args.rotation = rotation;
    for (int part = 0; part < 2; ++part) {
        args.gamma[part] = a.gamma[part];
        args.beta[part] = a.beta[part];
    }
    if (args.copied > 0) {
        constexpr int kPerVec = Elem<T>::kPerVec;
        args.copy_whole = a.copied * a.head_dim % kPerVec == 0 && a.heads * a.input.head % kPerVec == 0 &&
                          a.input.token % kPerVec == 0 && aligned16(input) && aligned16(output);
    }
    // Tokens for two rounds of a workgroup's teams, fewer while the chip has
    // workgroups to spare, and no more than 2^23 workgroups, whose threads HIP
    // counts in 32 bits.
    const int teams = kThreads >> args.log_team;
    const int full = 2 * teams / a.heads > 0 ? 2 * teams / a.heads : 1;
    const int spread = args.rows / (4 * compute_units()) + 1;
    const int least = (args.rows >> 23) + 1;
    args.block_tokens = full < spread ? full : spread;
    args.block_tokens = args.block_tokens > least ? args.block_tokens : least;
    const std::size_t lds =
        4 * (table_floats(args.block_tokens, rotation.pairs) +
             (a.norm != HeadNorm::kNone ? static_cast<std::size_t>(4) * ((a.head_dim + 3) / 4 * 4) + 8 : 0));
    const dim3 grid(static_cast<unsigned int>((args.rows - 1) / args.block_tokens + 1), // (rows reach 2^31 - 1)
                    args.copied > 0 ? 2U : 1U);
    auto run = [&](auto kernel) -> hipError_t {
        if (const hipError_t opted = allow_lds<decltype(kernel)::kValue>(lds); opted != hipSuccess) {
            return opted;
        }
        decltype(kernel)::kValue<<<grid, kThreads, lds, stream>>>(input, output, args);
        return hipGetLastError();
    };
    auto with_norm = [&](auto adjacent, auto streaming) -> hipError_t {
        constexpr bool kAdjacent = decltype(adjacent)::value;
        constexpr bool kStreaming = decltype(streaming)::value;
        switch (a.norm) {
        case HeadNorm::kNone:
            return run(KernelConstant<rotate_heads_kernel<T, U, Vector, HeadNorm::kNone, kAdjacent, kStreaming>>{});
        case HeadNorm::kRms:
            return run(KernelConstant<rotate_heads_kernel<T, U, Vector, HeadNorm::kRms, kAdjacent, kStreaming>>{});
        default:
            return run(KernelConstant<rotate_heads_kernel<T, U, Vector, HeadNorm::kLayer, kAdjacent, kStreaming>>{});
        }
    };
    auto with_stores = [&](auto adjacent) -> hipError_t {
        if constexpr (Vector) {
            if (input != output) {
                return with_norm(adjacent, std::true_type{});
            }
        }
        return with_norm(adjacent, std::false_type{});
    };
    return rotation.adjacent ? with_stores(std::true_type{}) : with_stores(std::false_type{});
}

template <typename T> hipError_t pick(const T* input, T* output, const HeadArgs& a, hipStream_t stream) {
    const std::uintptr_t addresses = reinterpret_cast<std::uintptr_t>(input) | reinterpret_cast<std::uintptr_t>(output);
    const std::int64_t strides = a.input.image | a.input.token | a.input.head | a.output.image | a.output.token |
                                 a.output.head;
    auto whole = [&](int unit) {
        return whole_runs(unit, sizeof(T), addresses, strides, a.head_dim, a.rotation.pairs, a.rotation.adjacent);
    };
    constexpr int kUnit = Elem<T>::kPerVec;
    if (whole(kUnit)) {
        return launch<T, kUnit, true>(input, output, a, stream);
    }
    if constexpr (sizeof(T) == 2) {
        if (whole(4)) {
            return launch<T, 4, true>(input, output, a, stream);
        }
    }
    return loose_runs_of_four(a) ? launch<T, 4, false>(input, output, a, stream)
                                 : launch<T, 8, false>(input, output, a, stream);
}

} // namespace
} // namespace rotary

hipError_t rotate_heads(const float* input, float* output, const HeadArgs& args, hipStream_t stream) {
    return rotary::pick(input, output, args, stream);
}

hipError_t rotate_heads(const std::uint16_t* input, std::uint16_t* output, const HeadArgs& args, hipStream_t stream) {
    return rotary::pick(input, output, args, stream);
}

} // namespace cuvit::detail
