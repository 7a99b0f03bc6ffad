// Attention over packed sequences: out = softmax(scale q.k^T).v for every row of every
// sequence, over its own sequence's keys, causal or all of them, and the rows'
// log-sum-exp; one pass over the keys with a running maximum and sum.
//
// A workgroup takes one key head and a tile of a sequence's rows (packed.hpp), 32 a
// wavefront in bf16, 16 in fp32; the keys and values of a block are brought to LDS for
// all four while the block before is worked on. Logits are computed keys by rows, so
// that a lane holds one row's logits: its maximum and sum are registers, its weights are
// the next product's operand where they lie, and causal masks compare with one number.
//
// Softmax. With m the running maximum and c = scale log2 e, a weight is exp2(x c - m c);
// m is raised only where a logit would exceed it by more than 2^kHeadroom in the
// exponential, so that the accumulators are seldom rescaled. Logits, sums, results and
// the log-sum-exp are fp32; bf16 weights are rounded once, for the matrix units, after
// they are summed. A row whose sums overflowed (values beyond 2^128 / (keys
// 2^kHeadroom)), or that met an infinity or NaN, which may lie in a key it does not see
// (0 times infinity), is taken again by itself over its own keys. A row without keys is
// zeros, its log-sum-exp -infinity; a row whose every logit is -infinity is NaN.
#include "packed.hpp"

namespace cuvit::detail {
namespace packed {
namespace {

constexpr float kHeadroom = 8.0F;

/// The running maximum and sum of a lane's row; shift is -(maximum c).
struct Running {
    float c;
    float maximum = -INFINITY;
    float shift = 0.F;
    float sum = 0.F;

    /// Raises the maximum to cover @p block, alike in all of a row's lanes, when any
    /// row of the wavefront needs it; true when what was accumulated takes @p factor.
    __device__ __forceinline__ bool raise(float block, float& factor) {
        if (!__any(fmaf(block, c, shift) > kHeadroom || maximum == -INFINITY)) {
            return false;
        }
        const float raised = fmaxf(maximum, block);
        // (While every logit so far is -infinity the shift stays 0: exp2(-infinity) is 0.)
        const float next = raised == -INFINITY ? 0.F : -(raised * c);
        factor = maximum == -INFINITY ? 0.F : __builtin_amdgcn_exp2f(next - shift);
        maximum = raised;
        shift = next;
        sum *= factor;
        return true;
    }

    __device__ __forceinline__ float weight(float logit) const {
        return __builtin_amdgcn_exp2f(fmaf(logit, c, shift));
    }
};

/// One row by a whole wavefront, over the keys it sees and no others: the exponent is a
/// difference of logits and what is accumulated stays normalised. Slow and seldom run.
template <typename T>
__device__ __forceinline__ void attend_alone(const T* q, const T* k, const T* v, T* out, float* lse, int keys,
                                             std::int64_t k_token, std::int64_t v_token, int head_dim, float c) {
    constexpr int kV = Elem<T>::kPerVec;
    const int lane = lane_id();
    float maximum = -INFINITY;
    float sum = 0.F;
    float value[4] = {0.F, 0.F, 0.F, 0.F}; // of dims lane + 64 i
#pragma clang loop unroll(disable)
    for (int first = 0; first < keys; first += kWave) {
        float logit = -INFINITY; // of key first + lane
        if (first + lane < keys) {
            const T* const row = k + (first + lane) * k_token;
            logit = 0.F;
#pragma clang loop unroll(disable)
            for (int d = 0; d < head_dim; d += kV) {
                const Vec16 a = load16(q + d);
                const Vec16 b = load16(row + d);
#pragma unroll
                for (int e = 0; e < kV; ++e) {
                    logit = fmaf(Elem<T>::get(a, e), Elem<T>::get(b, e), logit);
                }
            }
        }
        const bool bad = __any(logit != logit);
        const float raised = fmaxf(maximum, wave_allreduce(logit, Max{}));
        if (raised == -INFINITY && !bad) {
            continue;
        }
        const float weight = __builtin_amdgcn_exp2f((logit - raised) * c);
        const float kept = maximum == -INFINITY ? 0.F : sum * __builtin_amdgcn_exp2f((maximum - raised) * c);
        maximum = raised;
        sum = kept + wave_allreduce(weight, Sum{});
        if (sum != sum) {
            break; // NaN, whatever follows
        }
        const float share = weight / sum;
        const int there = min(keys - first, kWave);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            value[i] *= kept / sum;
        }
#pragma clang loop unroll(disable)
        for (int key = 0; key < there; ++key) {
            const float s = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(share), key));
            const T* const row = v + (first + key) * v_token;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (lane + kWave * i < head_dim) {
                    value[i] = fmaf(s, Elem<T>::load(row + lane + kWave * i), value[i]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (lane + kWave * i < head_dim) {
            Elem<T>::store(out + lane + kWave * i, sum > 0.F ? value[i] : __builtin_nanf(""));
        }
    }
    if (lse != nullptr && lane == 0) {
        *lse = (maximum * c + __builtin_amdgcn_logf(sum)) * kLn2; // (no logit above -infinity: -infinity)
    }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void packed_attention_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                                    const T* __restrict__ v, T* __restrict__ out,
                                                                    float* __restrict__ lse, PackedArgs args,
                                                                    int slots) {
    using R = Rows<T, D>;
    using Acc = typename Mma<T>::Acc;
    constexpr int E = R::kE;
    constexpr int K = kBlockRows<T, D>;
    constexpr int kTile = E * kWaves; // rows of a workgroup
    using Loads = Stage<T, D, K>;
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

    // The lane's row, and the keys that it, its wavefront and the workgroup see.
    const int row = first_row + wave * E + lane % E;
    const bool there = row < rows;
    const int query = row / args.group;
    const int head = item.head * args.group + row % args.group;
    const int behind = span.keys - span.queries;
    const auto sees = [&](int r) {
        return args.causal ? min(max(min(r, rows - 1) / args.group + 1 + behind, 0), span.keys) : span.keys;
    };
    const int seen = there ? sees(row) : 0;
    const int wave_least = __builtin_amdgcn_readfirstlane(sees(first_row + wave * E));
    const int wave_most = first_row + wave * E < rows ? __builtin_amdgcn_readfirstlane(sees(first_row + wave * E + E - 1)) : 0;
    const int most = __builtin_amdgcn_readfirstlane(sees(first_row + kTile - 1));

    const T* const k_head = k + span.first_key * args.k.token + item.head * args.k.head;
    const T* const v_head = v + span.first_key * args.v.token + item.head * args.v.head;
    const T* const q_row = there ? q + (static_cast<std::int64_t>(span.first_query) + query) * args.q.token + head * args.q.head
                                 : nullptr;
    const Loads k_loads(k_head, args.k.token, args.head_dim, wave, lane);
    const Loads v_loads(v_head, args.v.token, args.head_dim, wave, lane);
    auto issue = [&](int first, int buffer) {
        const unsigned int to = lds_base + static_cast<unsigned int>(buffer * 2 * Loads::kBytes);
        k_loads.issue(first, span.keys - first, to, wave);
        v_loads.issue(first, span.keys - first, to + Loads::kBytes, wave);
    };
    if (most > 0) {
        issue(0, 0);
    }
    Vec16 qf[R::kBlocks];
    load_rows<T, D>(q_row, args.head_dim, lane, qf);

    Running running{args.scale * kLog2e};
    Acc acc[R::kTiles];
#pragma unroll
    for (int t = 0; t < R::kTiles; ++t) {
        acc[t] = Acc{};
    }
    int buffer = 0;
    for (int first = 0; first < most; first += K) {
        landed(); // and every wavefront is done with the other buffer
        if (first + K < most) {
            issue(first + K, buffer ^ 1);
        }
        const unsigned char* const keys = lds + buffer * 2 * Loads::kBytes;
        const unsigned char* const values = keys + Loads::kBytes;
        buffer ^= 1;
        if (first >= wave_most) {
            continue;
        }
        Acc x[K / E];
#pragma unroll
        for (int t = 0; t < K / E; ++t) {
            x[t] = Acc{};
#pragma unroll
            for (int b = 0; b < R::kBlocks; ++b) {
                Mma<T>::run(x[t], R::along(keys, t * E + lane % E, b, lane), qf[b]);
            }
        }
        if (first + K > wave_least) {
#pragma unroll
            for (int t = 0; t < K / E; ++t) {
#pragma unroll
                for (int i = 0; i < kRegisters<T>; ++i) {
                    x[t][i] = first + t * E + row_of<T>(lane, i) < seen ? x[t][i] : -INFINITY;
                }
            }
        }
        float block = -INFINITY;
#pragma unroll
        for (int t = 0; t < K / E; ++t) {
#pragma unroll
            for (int i = 0; i < kRegisters<T>; ++i) {
                block = fmaxf(block, x[t][i]);
            }
        }
        block = combine_column<T>(block, Max{});
        float factor = 1.0F;
        if (running.raise(block, factor)) {
#pragma unroll
            for (int t = 0; t < R::kTiles; ++t) {
#pragma unroll
                for (int i = 0; i < kRegisters<T>; ++i) {
                    acc[t][i] *= factor;
                }
            }
        }
#pragma unroll
        for (int t = 0; t < K / E; ++t) {
#pragma unroll
            for (int i = 0; i < kRegisters<T>; ++i) {
                x[t][i] = running.weight(x[t][i]);
                running.sum += x[t][i];
            }
        }
#pragma unroll
        for (int t = 0; t < K / E; ++t) {
#pragma unroll
            for (int p = 0; p < kParts<T>; ++p) {
                const Vec16 weights = weights_of<T>(x[t], p);
#pragma unroll
                for (int d = 0; d < R::kTiles; ++d) {
                    Mma<T>::run(acc[d], R::across(values, t * E + 16 * p, d, lane), weights);
                }
            }
        }
    }

    const float total = combine_column<T>(running.sum, Sum{});
    float largest = 0.F;
#pragma unroll
    for (int t = 0; t < R::kTiles; ++t) {
#pragma unroll
        for (int i = 0; i < kRegisters<T>; ++i) { // (a NaN stays)
            largest = __builtin_elementwise_maximum(largest, fabsf(acc[t][i]));
        }
    }
    const bool usable = seen == 0 || (largest < INFINITY && total > 0.F && total < INFINITY);
    std::uint64_t bad = __ballot(there && !usable);
    T* const to = out + (static_cast<std::int64_t>(span.first_query) + query) * args.out.token + head * args.out.head;
    float* const lse_to =
        lse != nullptr ? lse + (static_cast<std::int64_t>(span.first_query) + query) * args.heads + head : nullptr;
    for (int half = 32; half >= E; half /= 2) { // any of a row's lanes
        bad |= bad >> half;
    }
    if (there && (bad >> (lane % E) & 1U) == 0) {
        store_row<T, D>(to, acc, seen > 0 ? 1.0F / total : 0.F, args.head_dim, lane);
        if (lse_to != nullptr && lane < E) {
            *lse_to = seen > 0 ? (__builtin_amdgcn_logf(total) - running.shift) * kLn2 : -INFINITY;
        }
    }
    bad &= E == 32 ? 0xFFFFFFFFU : 0xFFFFU;
    for (; __builtin_expect(bad != 0, 0); bad &= bad - 1) {
        const int r = first_row + wave * E + __builtin_ctzll(bad);
        const int h = item.head * args.group + r % args.group;
        const std::int64_t token = static_cast<std::int64_t>(span.first_query) + r / args.group;
        attend_alone<T>(q + token * args.q.token + h * args.q.head, k_head, v_head,
                        out + token * args.out.token + h * args.out.head,
                        lse != nullptr ? lse + token * args.heads + h : nullptr, sees(r), args.k.token, args.v.token,
                        args.head_dim, running.c);
    }
}

template <typename T>
hipError_t launch(const T* q, const T* k, const T* v, T* out, float* lse, const PackedArgs& args, hipStream_t stream) {
    return with_width(args.head_dim, [&](auto width) -> hipError_t {
        constexpr int D = decltype(width)::value;
        constexpr int kTile = Mma<T>::kEdge * kWaves;
        constexpr std::size_t kLds = 4 * Stage<T, D, kBlockRows<T, D>>::kBytes;
        constexpr auto kernel = packed_attention_kernel<T, D>;
        const std::int64_t tiles = slots(args.tokens, args.group, kTile, args.sequences);
        const std::int64_t blocks = items(tiles, args.kv_heads);
        if (!launchable(blocks, kThreads)) {
            return hipErrorInvalidConfiguration;
        }
        if (const hipError_t opted = allow_lds<kernel>(kLds); opted != hipSuccess) {
            return opted;
        }
        kernel<<<static_cast<unsigned int>(blocks), kThreads, kLds, stream>>>(q, k, v, out, lse, args,
                                                                             static_cast<int>(tiles));
        return hipGetLastError();
    });
}

} // namespace
} // namespace packed

hipError_t packed_attention(const float* q, const float* k, const float* v, float* out, float* lse, void*,
                            const PackedArgs& args, hipStream_t stream) {
    return packed::launch(q, k, v, out, lse, args, stream);
}

hipError_t packed_attention(const std::uint16_t* q, const std::uint16_t* k, const std::uint16_t* v, std::uint16_t* out,
                            float* lse, void*, const PackedArgs& args, hipStream_t stream) {
    return packed::launch(q, k, v, out, lse, args, stream);
}

std::int64_t packed_attention_workspace(const PackedArgs&) { return 0; }

} // namespace cuvit::detail
