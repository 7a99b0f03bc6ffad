// The gradients of attention over packed sequences. With p = exp(scale q.k - lse) the
// weights, anew from the kept log-sum-exp, d the result's gradient and
// delta = sum(d out) = sum(p (d.v)) of a row:
//   ds = p (d.v - delta),  grad_q = scale ds.k,  grad_k = scale ds^T.q,  grad_v = p^T.d.
//
// Two launches. The first takes tiles of rows, as the forward does, and walks the keys:
// delta, kept for the second, and grad_q. The second takes tiles of keys and walks the
// rows that see them, one query head of the group after another: grad_k and grad_v. So
// every gradient is summed in registers by one wavefront, in an order that sizes alone
// fix, at the cost of computing logits and d.v twice (7 products for 5); sums across
// workgroups would need atomics, whose order changes results, or fp32 copies of grad_q.
//
// Weights, slopes and sums are fp32; in bf16 weights and slopes are rounded once, for the
// matrix units that multiply them, whose fp32 rate is an eighth (2^-8 of each: gradients
// 2.4e-3 off, 1.7e-3 with fp32 ones).
#include "packed.hpp"
#include "packed_choice.hpp"

namespace cuvit::detail {
namespace packed {
namespace {

/// How a workgroup's wavefronts divide its work: Shared of them take the same rows (or
/// keys), each its own part of every block, and add up at the end, so that tiles are
/// smaller and more where they would not fill the chip.
template <typename T, int D, int Shared> struct Division {
    using R = Rows<T, D>;
    static constexpr int kShared = Shared;
    static constexpr int kTile = R::kE * kWaves / Shared;
    static constexpr int kCount = kBlockRows<T, D> > R::kE * Shared ? kBlockRows<T, D> : R::kE * Shared; // of a block
    static constexpr int kTiles = kCount / R::kE / Shared; // of a block, a wavefront's
    using Loads = Stage<T, D, kCount>;
    static constexpr int kBlocks = 4 * Loads::kBytes; // two operands, two buffers
    static_assert(kBlocks <= 128 * 1024, "two blocks of two operands");
};
template <typename T, int D> constexpr int kMostShared = Rows<T, D>::kPitch <= 256 * static_cast<int>(sizeof(T)) / 2 ? 4 : 2;

/// Adds the accumulators of the wavefronts that share a tile, in their order, in the
/// first one of them; false for the others, which are done.
template <typename T, int D, int Shared>
__device__ __forceinline__ bool add_up(float* lds, int wave, int lane,
                                       typename Mma<T>::Acc (&acc)[Rows<T, D>::kTiles]) {
    if constexpr (Shared > 1) {
        constexpr int kSums = Rows<T, D>::kTiles * kRegisters<T>;
        static_assert(kWaves / Shared * (Shared - 1) * kSums * kWave * 4 <= Division<T, D, Shared>::kBlocks,
                      "the blocks' LDS holds them");
        float* const sums = lds + wave / Shared * (Shared - 1) * kSums * kWave + lane;
        const int share = wave % Shared;
        __syncthreads();
        if (share > 0) {
#pragma unroll
            for (int t = 0; t < Rows<T, D>::kTiles; ++t) {
#pragma unroll
                for (int i = 0; i < kRegisters<T>; ++i) {
                    sums[((share - 1) * kSums + t * kRegisters<T> + i) * kWave] = acc[t][i];
                }
            }
        }
        __syncthreads();
        if (share == 0) {
#pragma unroll
            for (int o = 0; o < Shared - 1; ++o) {
#pragma unroll
                for (int t = 0; t < Rows<T, D>::kTiles; ++t) {
#pragma unroll
                    for (int i = 0; i < kRegisters<T>; ++i) {
                        acc[t][i] += sums[(o * kSums + t * kRegisters<T> + i) * kWave];
                    }
                }
            }
        }
        return share == 0;
    }
    return true;
}

/// Wavefronts that share a SIMD (packed_attention.hip).
template <int D> constexpr int kShareQueries = D <= 128 ? 2 : 1;
template <int D> constexpr int kShareKeys = D <= 96 ? 2 : 1;

template <typename T, int D, typename S>
__global__ __launch_bounds__(kThreads, kShareQueries<D>) void query_gradient_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                                  const T* __restrict__ v,
                                                                  PackedGradients<T> gradients, PackedArgs args,
                                                                  int slots) {
    using R = Rows<T, D>;
    using Acc = typename Mma<T>::Acc;
    constexpr int E = R::kE;
    constexpr int K = S::kCount;
    constexpr int kTile = S::kTile;
    using Loads = typename S::Loads;
    extern __shared__ Vec16 lds_vectors[];
    unsigned char* const lds = reinterpret_cast<unsigned char*>(lds_vectors);
    const Item item = item_of(blockIdx.x, slots, args.kv_heads, args.causal);
    if (item.head < 0) {
        return; // the whole workgroup, before any barrier (so below)
    }
    const Spot spot = find(args.starts, args.sequences, args.tokens, args.group, kTile, item.slot);
    if (spot.sequence < 0) {
        return;
    }
    const Span span = span_of(args, spot.sequence);
    const int rows = span.queries * args.group;
    const int first_row = spot.tile * kTile;
    if (first_row >= rows) {
        return;
    }
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const unsigned int lds_base = __builtin_amdgcn_readfirstlane(lds_address(lds));
    const int share = wave % S::kShared; // which keys of a block are this wavefront's
    const int wave_row = first_row + wave / S::kShared * E;
    const int row = wave_row + lane % E;
    const bool there = row < rows;
    const int query = row / args.group;
    const int head = item.head * args.group + row % args.group;
    const int behind = span.keys - span.queries;
    const auto sees = [&](int r) {
        return args.causal ? min(max(min(r, rows - 1) / args.group + 1 + behind, 0), span.keys) : span.keys;
    };
    const int seen = there ? sees(row) : 0;
    const int wave_least = __builtin_amdgcn_readfirstlane(sees(wave_row));
    const int wave_most = wave_row < rows ? __builtin_amdgcn_readfirstlane(sees(wave_row + E - 1)) : 0;
    const int most = __builtin_amdgcn_readfirstlane(sees(first_row + kTile - 1));

    const Loads k_loads(k + span.first_key * args.k.token + item.head * args.k.head, args.k.token, args.head_dim, wave,
                        lane);
    const Loads v_loads(v + span.first_key * args.v.token + item.head * args.v.head, args.v.token, args.head_dim, wave,
                        lane);
    auto issue = [&](int first, int buffer) {
        const unsigned int to = lds_base + static_cast<unsigned int>(buffer * 2 * Loads::kBytes);
        k_loads.issue(first, span.keys - first, to, wave);
        v_loads.issue(first, span.keys - first, to + Loads::kBytes, wave);
    };
    if (most > 0) {
        issue(0, 0);
    }
    const std::int64_t token = static_cast<std::int64_t>(span.first_query) + query;
    const std::int64_t place = token * args.out.token + head * args.out.head;
    Vec16 qf[R::kBlocks], df[R::kBlocks];
    load_rows<T, D>(there ? q + token * args.q.token + head * args.q.head : nullptr, args.head_dim, lane, qf);
    load_rows<T, D>(there ? gradients.grad_out + place : nullptr, args.head_dim, lane, df);
    float delta = 0.F;
    {
        Vec16 of[R::kBlocks];
        load_rows<T, D>(there ? gradients.out + place : nullptr, args.head_dim, lane, of);
#pragma unroll
        for (int b = 0; b < R::kBlocks; ++b) {
#pragma unroll
            for (int e = 0; e < R::kV; ++e) {
                delta = fmaf(Elem<T>::get(df[b], e), Elem<T>::get(of[b], e), delta);
            }
        }
    }
    delta = combine_column<T>(delta, Sum{});
    const float shift = there ? -gradients.lse[token * args.heads + head] * kLog2e : 0.F;
    const float c = args.scale * kLog2e;
    // A tile of keys, its first being @p first of which @p keys and @p values are the
    // rows: weights in x and d.v in y, both 0 for keys that the row does not see.
    auto weigh = [&](int first, const unsigned char* keys, const unsigned char* values, Acc& x, Acc& y) {
        x = Acc{};
        y = Acc{};
#pragma unroll
        for (int b = 0; b < R::kBlocks; ++b) {
            Mma<T>::run(x, R::along(keys, lane % E, b, lane), qf[b]);
            Mma<T>::run(y, R::along(values, lane % E, b, lane), df[b]);
        }
#pragma unroll
        for (int i = 0; i < kRegisters<T>; ++i) {
            x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c, shift));
        }
        if (first + E > wave_least) {
            const int left = seen - first - row_of<T>(lane, 0); // compared with constants
#pragma unroll
            for (int i = 0; i < kRegisters<T>; ++i) {
                x[i] = row_of<T>(0, i) < left ? x[i] : 0.F;
            }
        }
    };
    if constexpr (sizeof(T) == 2) {
        // Over few keys a rounded result leaves its rounding in delta where exact weights
        // would cancel: there it is summed from the weights (gradients of sequences of 2
        // tokens 3.8e-3 off -> 2.4e-3, the plain form 1.7e-3).
        if (most > 0 && most <= K) {
            landed();
            delta = 0.F;
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
                const int first = (share * S::kTiles + t) * E;
                if (first < wave_most) {
                    const unsigned char* const keys = lds + first * R::kPitch;
                    Acc x, y;
                    weigh(first, keys, keys + Loads::kBytes, x, y);
#pragma unroll
                    for (int i = 0; i < kRegisters<T>; ++i) {
                        delta = fmaf(x[i], y[i], delta);
                    }
                }
            }
            delta = combine_column<T>(delta, Sum{});
            if constexpr (S::kShared > 1) {
                float* const parts = reinterpret_cast<float*>(lds + 2 * Loads::kBytes); // the other buffer
                parts[wave * E + lane % E] = delta;
                __syncthreads();
                delta = 0.F;
#pragma unroll
                for (int w = 0; w < S::kShared; ++w) {
                    delta += parts[(wave / S::kShared * S::kShared + w) * E + lane % E];
                }
            }
        }
    }
    if (there && lane < E && share == 0) {
        static_cast<float*>(gradients.workspace)[token * args.heads + head] = delta;
    }
    Acc acc[R::kTiles];
#pragma unroll
    for (int t = 0; t < R::kTiles; ++t) {
        acc[t] = Acc{};
    }
    int buffer = 0;
    for (int block = 0; block < most; block += K) {
        landed(); // and every wavefront is done with the other buffer
        if (block + K < most) {
            issue(block + K, buffer ^ 1);
        }
        const int first = block + share * S::kTiles * E; // this wavefront's first key
        const unsigned char* const keys = lds + buffer * 2 * Loads::kBytes + share * S::kTiles * E * R::kPitch;
        const unsigned char* const values = keys + Loads::kBytes;
        buffer ^= 1;
        if (first >= wave_most) {
            continue;
        }
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
            const unsigned char* const rows_of_tile = keys + t * E * R::kPitch;
            Acc x, y;
            weigh(first + t * E, rows_of_tile, values + t * E * R::kPitch, x, y);
#pragma unroll
            for (int i = 0; i < kRegisters<T>; ++i) {
                x[i] *= y[i] - delta;
            }
#pragma unroll
            for (int p = 0; p < kParts<T>; ++p) {
                const Vec16 weights = weights_of<T>(x, p);
#pragma unroll
                for (int d = 0; d < R::kTiles; ++d) {
                    Mma<T>::run(acc[d], R::across(rows_of_tile, 16 * p, d, lane), weights);
                }
            }
        }
    }
    if (add_up<T, D, S::kShared>(reinterpret_cast<float*>(lds), wave, lane, acc) && there) {
        store_row<T, D>(gradients.grad_q + token * args.q.token + head * args.q.head, acc, args.scale, args.head_dim,
                        lane);
    }
}

template <typename T, int D, typename S>
__global__ __launch_bounds__(kThreads, kShareKeys<D>) void key_gradient_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                                const T* __restrict__ v, PackedGradients<T> gradients,
                                                                PackedArgs args, int slots) {
    using R = Rows<T, D>;
    using Acc = typename Mma<T>::Acc;
    constexpr int E = R::kE;
    constexpr int Q = S::kCount; // queries of a block
    constexpr int kTile = S::kTile;
    using Loads = typename S::Loads;
    extern __shared__ Vec16 lds_vectors[];
    unsigned char* const lds = reinterpret_cast<unsigned char*>(lds_vectors);
    // Behind the tiles: the block's log-sum-exps (times -log2 e) and deltas, two buffers.
    float* const numbers = reinterpret_cast<float*>(lds + 4 * Loads::kBytes);
    const Item item = item_of(blockIdx.x, slots, args.kv_heads, false);
    if (item.head < 0) {
        return; // the whole workgroup, before any barrier (so below)
    }
    const Spot spot = find(args.kv_starts, args.sequences, args.kv_tokens, 1, kTile, item.slot);
    if (spot.sequence < 0) {
        return;
    }
    const Span span = span_of(args, spot.sequence);
    const int first_key = spot.tile * kTile;
    if (first_key >= span.keys) {
        return;
    }
    const int lane = lane_id();
    const int thread = static_cast<int>(threadIdx.x);
    const int wave = __builtin_amdgcn_readfirstlane(thread / kWave);
    const unsigned int lds_base = __builtin_amdgcn_readfirstlane(lds_address(lds));
    const int share = wave % S::kShared; // which queries of a block are this wavefront's
    const int wave_key = first_key + wave / S::kShared * E;
    const int key = wave_key + lane % E;
    const bool there = key < span.keys;
    // Query i sees key j from i = j - (keys - queries) on.
    const int behind = span.keys - span.queries;
    const int from = args.causal ? max(key - behind, 0) : 0; // the first query that sees the lane's key
    const int wave_most = __builtin_amdgcn_readfirstlane(args.causal ? max(wave_key + E - 1 - behind, 0) : 0);
    const int wave_least = __builtin_amdgcn_readfirstlane(args.causal ? max(wave_key - behind, 0) : 0);
    const int start = __builtin_amdgcn_readfirstlane(args.causal ? max(first_key - behind, 0) / Q * Q : 0);

    const std::int64_t token = static_cast<std::int64_t>(span.first_key) + key;
    Vec16 kf[R::kBlocks], vf[R::kBlocks];
    load_rows<T, D>(there ? k + token * args.k.token + item.head * args.k.head : nullptr, args.head_dim, lane, kf);
    load_rows<T, D>(there ? v + token * args.v.token + item.head * args.v.head : nullptr, args.head_dim, lane, vf);
    const float c = args.scale * kLog2e;
    Acc grad_k[R::kTiles], grad_v[R::kTiles];
#pragma unroll
    for (int t = 0; t < R::kTiles; ++t) {
        grad_k[t] = Acc{};
        grad_v[t] = Acc{};
    }
    const std::int64_t first_query = span.first_query;
    for (int g = 0; g < args.group; ++g) {
        const int head = item.head * args.group + g;
        const Loads q_loads(q + first_query * args.q.token + head * args.q.head, args.q.token, args.head_dim, wave, lane);
        const Loads d_loads(gradients.grad_out + first_query * args.out.token + head * args.out.head, args.out.token,
                            args.head_dim, wave, lane);
        auto issue = [&](int first, int buffer) {
            const unsigned int to = lds_base + static_cast<unsigned int>(buffer * 2 * Loads::kBytes);
            q_loads.issue(first, span.queries - first, to, wave);
            d_loads.issue(first, span.queries - first, to + Loads::kBytes, wave);
        };
        // A row's two numbers by one thread each, kept until the tile's turn.
        const int which = thread / Q;
        const int number = thread % Q;
        auto fetch = [&](int first) -> float {
            if (which > 1 || first + number >= span.queries) {
                return which == 0 ? -INFINITY : 0.F; // (a row that is not there has weights of 0)
            }
            const std::int64_t at = (first_query + first + number) * args.heads + head;
            return which == 0 ? -gradients.lse[at] * kLog2e : static_cast<const float*>(gradients.workspace)[at];
        };
        if (start >= span.queries) {
            break; // no query sees these keys
        }
        __syncthreads(); // the last head's blocks are done with
        issue(start, 0);
        float held = fetch(start);
        int buffer = 0;
        for (int first = start; first < span.queries; first += Q) {
            if (which < 2) {
                numbers[(buffer * 2 + which) * Q + number] = held;
            }
            landed();
            if (first + Q < span.queries) {
                issue(first + Q, buffer ^ 1);
                held = fetch(first + Q);
            }
            const int mine = share * S::kTiles * E; // the block's queries from here on
            const unsigned char* const queries = lds + buffer * 2 * Loads::kBytes + mine * R::kPitch;
            const unsigned char* const grads = queries + Loads::kBytes;
            const float* const shifts = numbers + buffer * 2 * Q + mine;
            const float* const deltas = shifts + Q;
            buffer ^= 1;
            if (first + mine + S::kTiles * E <= wave_least) {
                continue;
            }
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
                Acc x{}, y{};
#pragma unroll
                for (int b = 0; b < R::kBlocks; ++b) {
                    Mma<T>::run(x, R::along(queries, t * E + lane % E, b, lane), kf[b]);
                    Mma<T>::run(y, R::along(grads, t * E + lane % E, b, lane), vf[b]);
                }
#pragma unroll
                for (int run = 0; run < Mma<T>::kRuns; ++run) {
                    const int at = t * E + Mma<T>::column(lane, run);
                    const Vec16 s = load16(shifts + at);
                    const Vec16 d = load16(deltas + at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 4 * run + e;
                        x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c, __uint_as_float(s.w[e])));
                        y[i] -= __uint_as_float(d.w[e]);
                    }
                }
                if (first + mine < wave_most) {
                    const int until = from - first - mine - row_of<T>(lane, 0); // compared with constants
#pragma unroll
                    for (int i = 0; i < kRegisters<T>; ++i) {
                        x[i] = t * E + row_of<T>(0, i) >= until ? x[i] : 0.F;
                    }
                }
#pragma unroll
                for (int i = 0; i < kRegisters<T>; ++i) {
                    y[i] *= x[i];
                }
#pragma unroll
                for (int p = 0; p < kParts<T>; ++p) {
                    const Vec16 weights = weights_of<T>(x, p);
                    const Vec16 slopes = weights_of<T>(y, p);
#pragma unroll
                    for (int d = 0; d < R::kTiles; ++d) {
                        Mma<T>::run(grad_v[d], R::across(grads, t * E + 16 * p, d, lane), weights);
                        Mma<T>::run(grad_k[d], R::across(queries, t * E + 16 * p, d, lane), slopes);
                    }
                }
            }
        }
    }
    float* const sums = reinterpret_cast<float*>(lds);
    add_up<T, D, S::kShared>(sums, wave, lane, grad_k);
    if (add_up<T, D, S::kShared>(sums, wave, lane, grad_v) && there) {
        store_row<T, D>(gradients.grad_k + token * args.k.token + item.head * args.k.head, grad_k, args.scale,
                        args.head_dim, lane);
        store_row<T, D>(gradients.grad_v + token * args.v.token + item.head * args.v.head, grad_v, 1.0F, args.head_dim,
                        lane);
    }
}

template <typename T>
hipError_t launch(const T* q, const T* k, const T* v, const PackedGradients<T>& gradients, const PackedArgs& args,
                  hipStream_t stream) {
    return with_width(args.head_dim, [&](auto width) -> hipError_t {
        constexpr int D = decltype(width)::value;
        const std::int64_t units = compute_units();
        /// @p run with @p sharing wavefronts to a tile (packed_choice.hpp).
        auto divided = [&](int sharing, auto&& run) -> hipError_t {
            static_assert(kMostShared<T, D> == most_sharing(D), "as the rules count them");
            if constexpr (sizeof(T) == 2) {
                if (sharing == 1) {
                    return run(Division<T, D, 1>{});
                }
            }
            if constexpr (kMostShared<T, D> > 2) {
                if (sharing > 2) {
                    return run(Division<T, D, kMostShared<T, D>>{});
                }
            }
            return run(Division<T, D, 2>{});
        };
        // Each launch's kernel, tiles and LDS for @p each.
        auto queries = [&](auto&& each) -> hipError_t {
            return divided(choose_query_sharing(args, sizeof(T) == 4, units), [&](auto division) -> hipError_t {
                using S = decltype(division);
                return each(KernelConstant<query_gradient_kernel<T, D, S>>{},
                            slots(args.tokens, args.group, S::kTile, args.sequences), S::kBlocks);
            });
        };
        auto keys = [&](auto&& each) -> hipError_t {
            return divided(choose_key_sharing(args, sizeof(T) == 4, units), [&](auto division) -> hipError_t {
                using S = decltype(division);
                return each(KernelConstant<key_gradient_kernel<T, D, S>>{},
                            slots(args.kv_tokens, 1, S::kTile, args.sequences),
                            S::kBlocks + 4 * S::kCount * sizeof(float));
            });
        };
        // What is refused is so before the first launch, which overwrites grad_q.
        auto check = [&](auto kernel_constant, std::int64_t tiles, std::size_t lds) -> hipError_t {
            return launchable(items(tiles, args.kv_heads), kThreads) ? allow_lds<decltype(kernel_constant)::kValue>(lds)
                                                                     : hipErrorInvalidConfiguration;
        };
        auto start = [&](auto kernel_constant, std::int64_t tiles, std::size_t lds) -> hipError_t {
            constexpr auto kernel = decltype(kernel_constant)::kValue;
            kernel<<<static_cast<unsigned int>(items(tiles, args.kv_heads)), kThreads, lds, stream>>>(
                q, k, v, gradients, args, static_cast<int>(tiles));
            return hipGetLastError();
        };
        hipError_t result = queries(check);
        result = result == hipSuccess ? keys(check) : result;
        result = result == hipSuccess ? queries(start) : result;
        return result == hipSuccess ? keys(start) : result;
    });
}

} // namespace
} // namespace packed

hipError_t packed_attention_backward(const float* q, const float* k, const float* v,
                                     const PackedGradients<float>& gradients, const PackedArgs& args,
                                     hipStream_t stream) {
    return packed::launch(q, k, v, gradients, args, stream);
}

hipError_t packed_attention_backward(const std::uint16_t* q, const std::uint16_t* k, const std::uint16_t* v,
                                     const PackedGradients<std::uint16_t>& gradients, const PackedArgs& args,
                                     hipStream_t stream) {
    return packed::launch(q, k, v, gradients, args, stream);
}

std::int64_t packed_attention_backward_workspace(const PackedArgs& args) {
    return static_cast<std::int64_t>(args.tokens) * args.heads * static_cast<std::int64_t>(sizeof(float));
}

} // namespace cuvit::detail
