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
// the log-sum-exp are fp32; bf16 weights are rounded once, for the matrix units, whose fp32
// rate is an eighth, after they are summed (2^-8 of a weight, 2.0e-3 to 2.3e-3 off in all,
// 1.7e-3 with fp32 weights). A row whose sums overflowed (values beyond 2^128 / (keys
// 2^kHeadroom)), or that met an infinity or NaN, which may lie in a key it does not see
// (0 times infinity), is taken again by itself over its own keys. A row without keys is
// zeros, its log-sum-exp -infinity, whatever its tile's other rows see; a row whose every
// logit is -infinity is NaN.
#include "packed.hpp"
#include "packed_choice.hpp"

namespace cuvit::detail {
namespace packed {
namespace {

constexpr float kHeadroom = 8.0F;

/// The running maximum and sum of a lane's row; shift is -(maximum c).
struct Running {
    float c = 0.F;
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
        bool open = false; // whether any value is one yet
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            open = open || (lane + kWave * i < head_dim && value[i] == value[i]);
        }
        if (!__any(open)) {
            break; // NaN, whatever follows
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (lane + kWave * i < head_dim) {
            Elem<T>::store(out + lane + kWave * i, sum > 0.F || keys == 0 ? value[i] : __builtin_nanf(""));
        }
    }
    if (lse != nullptr && lane == 0) {
        *lse = (maximum * c + __builtin_amdgcn_logf(sum)) * kLn2; // (no logit above -infinity: -infinity)
    }
}

/// How a workgroup's four wavefronts divide its work (packed_choice.hpp): kShared of them
/// take the same rows, each its own keys of every block, and add up at the end, which
/// shortens a tile's walk where tiles are few. In bf16 none share where there are rows enough
/// (kLarge, 128 of them), pairs do for fewer (kMiddle), all four for the fewest (kFew;
/// pairs of the widest heads, whose blocks would not fit otherwise); in fp32, whose
/// MFMAs leave nothing to overlap with in one wavefront, pairs do however many rows there are.
/// us, kFew / kMiddle / kLarge: bf16 64 x 577 tokens, 12 heads of 64 250 / 135 / 123,
/// 1 x 3136 72 / 65 / 84, 4 x 577 with 6 heads 10.1 / 10.9 / 15, 8192 tokens, 16 heads of
/// 128 1555 / 652 / 537; fp32 (kFew, pairs, none) 4 x 577 with 6 heads 34.6 / 29.2 / 33.9,
/// 4096 tokens, 16 heads 713 / 588 / 611. (Two tiles of rows a wavefront, whose MFMAs
/// share fragments, halve what LDS is read for, but leave two wavefronts a SIMD: 146 for
/// 123 at 64 x 577, 335 for 357 at 8192 tokens and 16 heads of 64.)
template <typename T, int D, Kind Way> struct Division {
    using R = Rows<T, D>;
    static constexpr bool kInParts = Way == Kind::kParts;
    static constexpr int kWaves = kInParts ? 1 : packed::kWaves;
    static constexpr int kThreads = kWaves * kWave;
    static constexpr int kPairs = kInParts || Way == Kind::kLarge ? 1 : 2;
    static constexpr int kShared =
        Way == Kind::kFew && R::kPitch <= 256 * static_cast<int>(sizeof(T)) / 2 ? 4 : kPairs;
    static constexpr int kRows = R::kE * kWaves / kShared; // of a workgroup
    static constexpr int kLeast = kInParts ? 32 : R::kE * kShared;
    static constexpr int kKeys = (Way == Kind::kMiddle || Way == Kind::kLarge) && kBlockRows<T, D> > kLeast
                                     ? kBlockRows<T, D>
                                     : kLeast; // of a block
    static constexpr int kTiles = kKeys / R::kE / kShared; // of keys, a wavefront's
    /// Wavefronts that share a SIMD. From two on the compiler keeps every accumulator in
    /// the registers that the VALU reads, instead of moving logits and weights over.
    static constexpr int kShare = D > 128 ? 1 : D > 64 ? 2 : Way == Kind::kLarge ? 4 : 3;
    using Loads = Stage<T, D, kKeys, kWaves>;
    // The sums of the wavefronts that add up: accumulators, shift and sum of each lane.
    static constexpr int kSums = R::kTiles * kRegisters<T> + 2;
    static constexpr int kExchange = kWaves / kShared * (kShared - 1) * kSums * kWave * 4;
    static constexpr int kLds = 4 * Loads::kBytes > kExchange ? 4 * Loads::kBytes : kExchange;
    static_assert(Way != Kind::kLarge || sizeof(T) == 2, "in fp32 it would be kMiddle");
    static_assert(kLds <= 128 * 1024, "two blocks of keys and values, or the sums");
    static_assert(Way == Kind::kFew || kRows == tile_rows(Way, sizeof(T) == 4), "as the rules count them");
    static_assert(!kInParts || kKeys == kPartKeys, "as the rules count them");
};

/// A row's partial sums in the workspace: head_dim floats and the shift and the sum.
__device__ __forceinline__ std::int64_t partial_at(const PackedArgs& args, std::int64_t row, int parts, int part) {
    return (row * parts + part) * (args.head_dim + 2);
}

/// The result and log-sum-exp of a row from its sums, or false where they are of no use
/// (see the top). @p largest is the largest size among the accumulators.
__device__ __forceinline__ bool usable(int seen, float largest, float total) {
    return largest < INFINITY && (seen == 0 || (total > 0.F && total < INFINITY));
}
__device__ __forceinline__ float log_sum_exp(int seen, float total, float shift) {
    return seen > 0 ? (__builtin_amdgcn_logf(total) - shift) * kLn2 : -INFINITY;
}

/// In parts (Kind::kParts) several workgroups take a tile, each its part of the keys, and leave
/// partial sums for join_kernel.
template <typename T, int D, typename S>
__global__ __launch_bounds__(S::kThreads, S::kShare) void packed_attention_kernel(const T* __restrict__ q,
                                                                                  const T* __restrict__ k,
                                                                                  const T* __restrict__ v,
                                                                                  T* __restrict__ out,
                                                                                  float* __restrict__ lse,
                                                                                  float* __restrict__ partial,
                                                                                  PackedArgs args, int slots,
                                                                                  int parts) {
    using R = Rows<T, D>;
    using Acc = typename Mma<T>::Acc;
    using Loads = typename S::Loads;
    constexpr int E = R::kE;
    constexpr int K = S::kKeys;
    constexpr bool Parts = S::kInParts;
    extern __shared__ Vec16 lds_vectors[];
    unsigned char* const lds = reinterpret_cast<unsigned char*>(lds_vectors);
    const int part = Parts ? static_cast<int>(blockIdx.x % static_cast<unsigned int>(parts)) : 0;
    const Item item = item_of(Parts ? blockIdx.x / static_cast<unsigned int>(parts) : blockIdx.x, slots, args.kv_heads,
                              args.causal);
    if (item.head < 0) {
        return; // the whole workgroup, before any barrier (so below)
    }
    const Spot spot = find(args.starts, args.sequences, args.tokens, args.group, S::kRows, item.slot);
    if (spot.sequence < 0) {
        return;
    }
    const Span span = span_of(args, spot.sequence);
    const int rows = span.queries * args.group;
    const int tile_row = spot.tile * S::kRows;
    if (tile_row >= rows) {
        return;
    }
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int share = wave % S::kShared; // which keys of a block are this wavefront's
    const int first_row = tile_row + wave / S::kShared * E;
    const unsigned int lds_base = __builtin_amdgcn_readfirstlane(lds_address(lds));

    // The keys that the lane's row, the wavefront and the workgroup see.
    const int behind = span.keys - span.queries;
    const auto sees = [&](int r) {
        return args.causal ? min(max(min(r, rows - 1) / args.group + 1 + behind, 0), span.keys) : span.keys;
    };
    const int row = first_row + lane % E;
    const bool there = row < rows;
    const int seen = there ? sees(row) : 0;
    const int wave_least = __builtin_amdgcn_readfirstlane(sees(first_row));
    const int wave_most = first_row < rows ? __builtin_amdgcn_readfirstlane(sees(first_row + E - 1)) : 0;
    int most = __builtin_amdgcn_readfirstlane(sees(tile_row + S::kRows - 1));
    int start = 0;
    if constexpr (Parts) {
        const Part mine = part_of(most, part, parts, K);
        start = __builtin_amdgcn_readfirstlane(mine.first);
        most = __builtin_amdgcn_readfirstlane(mine.last);
    }

    const T* const k_head = k + span.first_key * args.k.token + item.head * args.k.head;
    const T* const v_head = v + span.first_key * args.v.token + item.head * args.v.head;
    const Loads k_loads(k_head, args.k.token, args.head_dim, wave, lane);
    const Loads v_loads(v_head, args.v.token, args.head_dim, wave, lane);
    auto issue = [&](int first, int buffer) {
        const unsigned int to = lds_base + static_cast<unsigned int>(buffer * 2 * Loads::kBytes);
        k_loads.issue(first, span.keys - first, to, wave);
        v_loads.issue(first, span.keys - first, to + Loads::kBytes, wave);
    };
    if (start < most) {
        issue(start, 0);
    }
    /// A row's token and query head.
    struct Place {
        std::int64_t token;
        int head;
    };
    const auto place_of = [&](int row) {
        const int query = row / args.group;
        return Place{static_cast<std::int64_t>(span.first_query) + query,
                     item.head * args.group + row - query * args.group};
    };
    const Place at = place_of(row);
    Vec16 qf[R::kBlocks];
    load_rows<T, D>(there ? q + at.token * args.q.token + at.head * args.q.head : nullptr, args.head_dim, lane, qf);

    const float c = args.scale * kLog2e;
    Running running{c};
    Acc acc[R::kTiles];
#pragma unroll
    for (int t = 0; t < R::kTiles; ++t) {
        acc[t] = Acc{};
    }
    int buffer = 0;
    for (int block = start; block < most; block += K) {
        landed(); // and every wavefront is done with the other buffer
        if (block + K < most) {
            issue(block + K, buffer ^ 1);
        }
        const unsigned char* const keys = lds + buffer * 2 * Loads::kBytes + share * S::kTiles * E * R::kPitch;
        const unsigned char* const values = keys + Loads::kBytes;
        buffer ^= 1;
        const int first = block + share * S::kTiles * E; // this wavefront's first key
        if (first >= wave_most) {
            continue;
        }
        // Fragments are read a tile ahead of their MFMAs, the first values' behind the
        // last keys', so that their latency lies under the softmax; where the registers
        // do not hold them, as they are needed. (Whole tiles of heads of 128 spill ten.)
        constexpr bool kAhead = (D <= 96 && S::kShare < 4) || (D == 128 && sizeof(T) == 2 && !Parts);
        constexpr int kSets = S::kTiles > 1 ? 2 : 1;
        Vec16 kf[kSets][R::kBlocks], vf[kSets][kParts<T>][R::kTiles];
        auto read_keys = [&](int t) {
#pragma unroll
            for (int b = 0; b < R::kBlocks; ++b) {
                kf[t % kSets][b] = R::along(keys, t * E + lane % E, b, lane);
            }
        };
        auto read_values = [&](int t) {
#pragma unroll
            for (int p = 0; p < kParts<T>; ++p) {
#pragma unroll
                for (int d = 0; d < R::kTiles; ++d) {
                    vf[t % kSets][p][d] = R::across(values, t * E + 16 * p, d, lane);
                }
            }
        };
        Acc x[S::kTiles];
        if constexpr (kAhead) {
            read_keys(0);
        }
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
            x[t] = Acc{};
            if constexpr (kAhead) {
                if (t + 1 < S::kTiles) {
                    read_keys(t + 1);
                } else {
                    read_values(0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int b = 0; b < R::kBlocks; ++b) {
                Mma<T>::run(x[t], kAhead ? kf[t % kSets][b] : R::along(keys, t * E + lane % E, b, lane), qf[b]);
            }
            if constexpr (kAhead) {
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (first + S::kTiles * E > wave_least) {
            const int left = seen - first - row_of<T>(lane, 0); // compared with constants
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
#pragma unroll
                for (int i = 0; i < kRegisters<T>; ++i) {
                    x[t][i] = t * E + row_of<T>(0, i) < left ? x[t][i] : -INFINITY;
                }
            }
        }
        float largest = -INFINITY;
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
#pragma unroll
            for (int i = 0; i < kRegisters<T>; ++i) {
                largest = fmaxf(largest, x[t][i]);
            }
        }
        largest = combine_column<T>(largest, Max{});
        float factor = 1.0F;
        if (running.raise(largest, factor)) {
#pragma unroll
            for (int t = 0; t < R::kTiles; ++t) {
#pragma unroll
                for (int i = 0; i < kRegisters<T>; ++i) {
                    acc[t][i] *= factor;
                }
            }
        }
        float sums[4] = {0.F, 0.F, 0.F, 0.F};
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
#pragma unroll
            for (int i = 0; i < kRegisters<T>; ++i) {
                x[t][i] = running.weight(x[t][i]);
                sums[i % 4] += x[t][i];
            }
        }
        running.sum += (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
            if constexpr (kAhead) {
                if (t + 1 < S::kTiles) {
                    read_values(t + 1);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int p = 0; p < kParts<T>; ++p) {
                const Vec16 weights = weights_of<T>(x[t], p);
#pragma unroll
                for (int d = 0; d < R::kTiles; ++d) {
                    Mma<T>::run(acc[d], kAhead ? vf[t % kSets][p][d] : R::across(values, t * E + 16 * p, d, lane), weights);
                }
            }
            if constexpr (kAhead) {
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    float total = combine_column<T>(running.sum, Sum{});
    if constexpr (S::kShared > 1) {
        // The others' sums through LDS, each scaled to the larger maximum, in turn.
        __syncthreads();
        float* const sums = reinterpret_cast<float*>(lds) + wave / S::kShared * (S::kShared - 1) * S::kSums * kWave + lane;
        if (share > 0) {
            float* const to = sums + (share - 1) * S::kSums * kWave;
#pragma unroll
            for (int t = 0; t < R::kTiles; ++t) {
#pragma unroll
                for (int i = 0; i < kRegisters<T>; ++i) {
                    to[(t * kRegisters<T> + i) * kWave] = acc[t][i];
                }
            }
            to[(S::kSums - 2) * kWave] = running.maximum == -INFINITY ? INFINITY : running.shift;
            to[(S::kSums - 1) * kWave] = total;
        }
        __syncthreads();
        if (share > 0) {
            return;
        }
        float shift = running.maximum == -INFINITY ? INFINITY : running.shift;
#pragma unroll
        for (int o = 0; o < S::kShared - 1; ++o) {
            const float* const from = sums + o * S::kSums * kWave;
            const float other = from[(S::kSums - 2) * kWave];
            const float common = fminf(shift, other);
            // (No logit above -infinity yet: the shift is infinity, its sums 0.)
            const float mine = shift == INFINITY ? 0.F : __builtin_amdgcn_exp2f(common - shift);
            const float theirs = other == INFINITY ? 0.F : __builtin_amdgcn_exp2f(common - other);
            total = total * mine + from[(S::kSums - 1) * kWave] * theirs;
#pragma unroll
            for (int t = 0; t < R::kTiles; ++t) {
#pragma unroll
                for (int i = 0; i < kRegisters<T>; ++i) {
                    acc[t][i] = acc[t][i] * mine + from[(t * kRegisters<T> + i) * kWave] * theirs;
                }
            }
            shift = common;
        }
        running.shift = shift;
        running.maximum = shift == INFINITY ? -INFINITY : 0.F;
    }
    if constexpr (Parts) {
        if (there) {
            float* const to = partial + partial_at(args, at.token * args.heads + at.head, parts, part);
#pragma unroll
            for (int t = 0; t < R::kTiles; ++t) {
#pragma unroll
                for (int i = 0; i < kRegisters<T>; ++i) {
                    const int dim = t * E + row_of<T>(lane, i);
                    if (dim < args.head_dim) {
                        to[dim] = acc[t][i];
                    }
                }
            }
            if (lane < E) {
                to[args.head_dim] = running.maximum == -INFINITY ? INFINITY : running.shift;
                to[args.head_dim + 1] = total;
            }
        }
        return;
    }
    float largest = 0.F;
#pragma unroll
    for (int t = 0; t < R::kTiles; ++t) {
#pragma unroll
        for (int i = 0; i < kRegisters<T>; ++i) { // (a NaN stays)
            largest = __builtin_elementwise_maximum(largest, fabsf(acc[t][i]));
        }
    }
    std::uint64_t bad = __ballot(there && !usable(seen, largest, total));
    for (int half = 32; half >= E; half /= 2) { // any of a row's lanes
        bad |= bad >> half;
    }
    if (there && (bad >> (lane % E) & 1U) == 0) {
        store_row<T, D>(out + at.token * args.out.token + at.head * args.out.head, acc, seen > 0 ? 1.0F / total : 0.F,
                        args.head_dim, lane);
        if (lse != nullptr && lane < E) {
            lse[at.token * args.heads + at.head] = log_sum_exp(seen, total, running.shift);
        }
    }
    bad &= E == 32 ? 0xFFFFFFFFU : 0xFFFFU;
    for (; __builtin_expect(bad != 0, 0); bad &= bad - 1) {
        const int r = first_row + __builtin_ctzll(bad);
        const Place again = place_of(r);
        attend_alone<T>(q + again.token * args.q.token + again.head * args.q.head, k_head, v_head,
                        out + again.token * args.out.token + again.head * args.out.head,
                        lse != nullptr ? lse + again.token * args.heads + again.head : nullptr, sees(r), args.k.token,
                        args.v.token, args.head_dim, c);
    }
}

/// Workgroups to a tile's rows in the join.
constexpr int kJoiners = 8;

/// Adds up the parts of a row, wavefront w those of number w, w + 4, ..., then the four
/// wavefronts' sums in turn. Bound by the latency of its loads: all of a wavefront's are
/// in flight at once (32 parts of heads of 128: 22 us with a wavefront a row and a part after
/// the other).
template <typename T, int Tile>
__global__ __launch_bounds__(kThreads) void join_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                        const T* __restrict__ v, T* __restrict__ out,
                                                        float* __restrict__ lse, const float* __restrict__ partial,
                                                        PackedArgs args, int slots, int parts) {
    __shared__ float sums[kWaves][4 * kWave];
    __shared__ float totals[kWaves];
    __shared__ float shifts[kWaves];
    const Item item = item_of(blockIdx.x, slots, args.kv_heads, args.causal);
    if (item.head < 0) {
        return; // the whole workgroup, before any barrier (so below)
    }
    const Spot spot = find(args.starts, args.sequences, args.tokens, args.group, Tile, item.slot);
    if (spot.sequence < 0) {
        return;
    }
    const Span span = span_of(args, spot.sequence);
    const int rows = span.queries * args.group;
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int last = min(rows, spot.tile * Tile + Tile);
    const float c = args.scale * kLog2e;
    for (int row = spot.tile * Tile + static_cast<int>(blockIdx.y); row < last; row += kJoiners) {
        const int query = row / args.group;
        const int head = item.head * args.group + row % args.group;
        const std::int64_t token = static_cast<std::int64_t>(span.first_query) + query;
        const int seen = seen_by(query, span.keys - span.queries, span.keys, args.causal);
        const float* const from = partial + partial_at(args, token * args.heads + head, parts, 0);
        const int step = args.head_dim + 2;
        float shift = INFINITY; // no logit above -infinity yet
        float total = 0.F;
        float value[4] = {0.F, 0.F, 0.F, 0.F};
        int dim[4]; // (behind the last one the last one again, without a branch)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            dim[i] = min(lane + kWave * i, args.head_dim - 1);
        }
        for (int p0 = wave; p0 < parts; p0 += 8 * kWaves) {
            float there[8][4], others[8], totals_there[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int p = p0 + u * kWaves;
                const float* const at = from + min(p, parts - 1) * step;
                others[u] = p < parts ? at[args.head_dim] : INFINITY;
                totals_there[u] = at[args.head_dim + 1];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    there[u][i] = at[dim[i]];
                }
            }
            float common = shift;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                common = fminf(common, others[u]);
            }
            const float mine = shift == INFINITY ? 0.F : __builtin_amdgcn_exp2f(common - shift);
            total *= mine;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                value[i] *= mine;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float theirs = others[u] == INFINITY ? 0.F : __builtin_amdgcn_exp2f(common - others[u]);
                total += totals_there[u] * theirs;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    value[i] += there[u][i] * theirs;
                }
            }
            shift = common;
        }
        __syncthreads(); // the last row's sums are read
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sums[wave][lane + kWave * i] = value[i];
        }
        if (lane == 0) {
            totals[wave] = total;
            shifts[wave] = shift;
        }
        __syncthreads();
        if (wave != 0) {
            continue;
        }
        shift = fminf(fminf(shifts[0], shifts[1]), fminf(shifts[2], shifts[3]));
        float largest = 0.F;
        float factor[kWaves];
        total = 0.F;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            factor[w] = shifts[w] == INFINITY ? 0.F : __builtin_amdgcn_exp2f(shift - shifts[w]);
            total += totals[w] * factor[w];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            value[i] = 0.F;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                value[i] += sums[w][lane + kWave * i] * factor[w];
            }
            largest = __builtin_elementwise_maximum(largest, fabsf(value[i]));
        }
        T* const to = out + token * args.out.token + head * args.out.head;
        float* const lse_to = lse != nullptr ? lse + token * args.heads + head : nullptr;
        if (__builtin_expect(__any(!usable(seen, largest, total)), 0)) {
            attend_alone<T>(q + token * args.q.token + head * args.q.head,
                            k + span.first_key * args.k.token + item.head * args.k.head,
                            v + span.first_key * args.v.token + item.head * args.v.head, to, lse_to, seen, args.k.token,
                            args.v.token, args.head_dim, c);
            continue;
        }
        const float inverse = seen > 0 ? 1.0F / total : 0.F;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (lane + kWave * i < args.head_dim) {
                Elem<T>::store(to + lane + kWave * i, value[i] * inverse);
            }
        }
        if (lse_to != nullptr && lane == 0) {
            *lse_to = log_sum_exp(seen, total, shift);
        }
    }
}

template <typename T>
hipError_t launch(const T* q, const T* k, const T* v, T* out, float* lse, float* workspace, const PackedArgs& args,
                  hipStream_t stream) {
    return with_width(args.head_dim, [&](auto width) -> hipError_t {
        constexpr int D = decltype(width)::value;
        const Plan chosen = choose_forward(args, sizeof(T) == 4, compute_units());
        auto run = [&](auto division) -> hipError_t {
            using S = decltype(division);
            constexpr auto kernel = packed_attention_kernel<T, D, S>;
            const std::int64_t tiles = slots(args.tokens, args.group, S::kRows, args.sequences);
            const std::int64_t blocks = items(tiles, args.kv_heads) * chosen.parts;
            if (!launchable(blocks, S::kThreads)) {
                return hipErrorInvalidConfiguration;
            }
            if (const hipError_t opted = allow_lds<kernel>(S::kLds); opted != hipSuccess) {
                return opted;
            }
            kernel<<<static_cast<unsigned int>(blocks), S::kThreads, S::kLds, stream>>>(
                q, k, v, out, lse, workspace, args, static_cast<int>(tiles), chosen.parts);
            return hipGetLastError();
        };
        switch (chosen.kind) {
        case Kind::kLarge:
            if constexpr (sizeof(T) == 2) {
                return run(Division<T, D, Kind::kLarge>{});
            }
            [[fallthrough]];
        case Kind::kMiddle: return run(Division<T, D, Kind::kMiddle>{});
        case Kind::kFew: return run(Division<T, D, Kind::kFew>{});
        default: break;
        }
        using Parts = Division<T, D, Kind::kParts>;
        if (const hipError_t result = run(Parts{}); result != hipSuccess) {
            return result;
        }
        const std::int64_t tiles = slots(args.tokens, args.group, Parts::kRows, args.sequences);
        const dim3 grid(static_cast<unsigned int>(items(tiles, args.kv_heads)), kJoiners);
        join_kernel<T, Parts::kRows><<<grid, kThreads, 0, stream>>>(
            q, k, v, out, lse, workspace, args, static_cast<int>(tiles), chosen.parts);
        return hipGetLastError();
    });
}

std::int64_t workspace_of(const PackedArgs& args, bool single) {
    const Plan chosen = choose_forward(args, single, compute_units());
    return chosen.parts > 1 ? static_cast<std::int64_t>(args.tokens) * args.heads * chosen.parts * (args.head_dim + 2) *
                                  static_cast<std::int64_t>(sizeof(float))
                            : 0;
}

} // namespace
} // namespace packed

hipError_t packed_attention(const float* q, const float* k, const float* v, float* out, float* lse, void* workspace,
                            const PackedArgs& args, hipStream_t stream) {
    return packed::launch(q, k, v, out, lse, static_cast<float*>(workspace), args, stream);
}

hipError_t packed_attention(const std::uint16_t* q, const std::uint16_t* k, const std::uint16_t* v, std::uint16_t* out,
                            float* lse, void* workspace, const PackedArgs& args, hipStream_t stream) {
    return packed::launch(q, k, v, out, lse, static_cast<float*>(workspace), args, stream);
}

std::int64_t packed_attention_workspace(const PackedArgs& args) {
    const std::int64_t single = packed::workspace_of(args, true);
    const std::int64_t half = packed::workspace_of(args, false);
    return single > half ? single : half;
}

} // namespace cuvit::detail
