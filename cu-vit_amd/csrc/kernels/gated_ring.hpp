// The gated product on the LDS ring of gemm_ring.hpp: operands whose rows are
// whole 16-byte chunks, brought by direct-to-LDS loads. See gated.hip for what a
// tile is; here B's stage rows alternate between the gate's and the value's, an
// MFMA tile (32 or 16 rows) of each, so that the MFMA tiles j and j + 1 of a
// wavefront are the two factors of the same outputs.
#pragma once

#include "checkpoint.hpp"
#include "gate.hpp"
#include "gemm_ring.hpp"
#include "runs.hpp"

namespace cuvit::detail::gemm {

/// RingLoads with B's rows taken from both halves of the weight.
template <typename T, typename S> struct GatedLoads {
    sgpr4 resource_a;
    sgpr4 resource_b[2];
    unsigned int offset_a;
    unsigned int offset_b;
    unsigned int step_a;
    unsigned int row_bytes_b;
    unsigned int lds_base;
    int wave;
    int load_k;
    int depth;

    /// Rows from @p row0, outputs from @p out0 on.
    __device__ __forceinline__ GatedLoads(const T* a, const T* b, const GatedArgs& args, int row0, int out0, int wave_,
                                          int lane, unsigned int lds) {
        constexpr int kSize = static_cast<int>(sizeof(T));
        const int rows_a = min(args.m - row0, S::kBM);
        const int rows_b = min(args.n - out0, S::kBN / 2);
        resource_a = scalar_resource(a + static_cast<std::int64_t>(row0) * args.lda,
                                     static_cast<unsigned int>(rows_a * args.lda * kSize));
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            resource_b[half] =
                scalar_resource(b + (static_cast<std::int64_t>(half) * args.n + out0) * args.ldb,
                                static_cast<unsigned int>(rows_b * args.ldb * kSize));
        }
        wave = wave_;
        const int load_row = wave * S::kLoadRows + lane / S::kChunks;
        load_k = 16 / kSize * S::place(load_row, lane % S::kChunks);
        offset_a = static_cast<unsigned int>((load_row * args.lda + load_k) * kSize);
        offset_b = static_cast<unsigned int>((lane / S::kChunks * args.ldb + load_k) * kSize);
        step_a = static_cast<unsigned int>(__builtin_amdgcn_readfirstlane(S::kWaves * S::kLoadRows * args.lda * kSize));
        row_bytes_b = static_cast<unsigned int>(__builtin_amdgcn_readfirstlane(args.ldb * kSize));
        lds_base = lds + static_cast<unsigned int>(wave * 1024);
        depth = args.k;
    }

    /// Stage @p g into ring slot @p slot.
    __device__ __forceinline__ void issue(int g, int slot) const {
        const int k0 = g * S::kBK;
        const bool inside = load_k + k0 < depth;
        const unsigned int at = static_cast<unsigned int>(k0) * static_cast<unsigned int>(sizeof(T));
        const unsigned int from_a = inside ? offset_a + at : kOutside;
        const unsigned int from_b = inside ? offset_b + at : kOutside;
        const unsigned int m0 = lds_base + static_cast<unsigned int>(slot * S::kStageBytes);
#pragma unroll
        for (int p = 0; p < S::kLoadsA; ++p) {
            load_to_lds(m0 + static_cast<unsigned int>(p * S::kWaves * 1024),
                        from_a + static_cast<unsigned int>(p) * step_a, resource_a);
        }
#pragma unroll
        for (int p = 0; p < S::kLoadsB; ++p) {
            const int row = (p * S::kWaves + wave) * S::kLoadRows; // of the stage's B rows
            const int tile = row / S::kEdge;
            const unsigned int source = static_cast<unsigned int>(tile / 2 * S::kEdge + row % S::kEdge) * row_bytes_b;
            load_to_lds(m0 + static_cast<unsigned int>(S::kBM * S::kRowBytes + p * S::kWaves * 1024), from_b + source,
                        (tile & 1) != 0 ? resource_b[1] : resource_b[0]);
        }
    }
};

/// Four consecutive values to any value's address, or the first @p count of them.
template <typename T> __device__ __forceinline__ void store_quad(T* to, const float (&v)[4], int count) {
    const Run<T, 4> run = round_run<T, 4>(v);
    if (count >= 4) {
        store_run_unaligned<T, 4>(to, run);
    } else {
        store_some<T, 4>(to, run, count);
    }
}

/// A lane's four consecutive columns of one row, finished and stored.
template <typename T, Gate G>
__device__ __forceinline__ void finish_quad(const float (&gate)[4], const float (&value)[4], int row, int col, T* c,
                                            T* pre, const GatedArgs& args) {
    if (row >= args.m || col >= args.n) {
        return;
    }
    const int count = args.n - col;
    float out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        out[e] = gate_value<G>(gate[e]) * value[e];
    }
    store_quad(c + static_cast<std::int64_t>(row) * args.ldc + col, out, count);
    if (pre != nullptr) {
        T* const to = pre + static_cast<std::int64_t>(row) * args.ld_pre + col;
        store_quad(to, gate, count);
        store_quad(to + args.n, value, count);
    }
}

/// Where a tile's sums start: the bias, loaded into LDS ahead of the first stage
/// ([gate, value] of the tile's outputs), so that the epilogue neither adds nor
/// waits for it. Without a bias the loads read as zero.
template <typename T, typename S> struct StartAtBias {
    static constexpr bool kAfterFirst = true;
    const float* bias; // in LDS, of the lane's first output
    __device__ __forceinline__ void operator()(typename Mma<T>::Acc (&acc)[S::kTM][S::kTN]) const {
#pragma unroll
        for (int j = 0; j < S::kTN; ++j)
#pragma unroll
            for (int q = 0; q < Mma<T>::kRuns; ++q) {
                const Vec16 v = load16(bias + (j & 1) * (S::kBN / 2) + j / 2 * S::kEdge + 8 * q);
#pragma unroll
                for (int i = 0; i < S::kTM; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[i][j][4 * q + e] = __uint_as_float(v.w[e]);
            }
    }
};

/// LDS of a workgroup: the ring, and the 16 bytes a lane that the bias' load writes.
template <typename S> constexpr int kGatedLds = S::kBiasOffset + 16 * kWave;

/// Sends the bias of a tile's outputs on its way to LDS at @p m0 (a wavefront's 16
/// bytes a lane, zeros behind the last output).
template <int Outputs>
__device__ __forceinline__ void load_bias(const float* bias, int out0, int n, int lane, unsigned int m0) {
    static_assert(Outputs % 4 == 0 && Outputs <= 128, "one load of a wavefront");
    const int part = lane / (Outputs / 4); // the gate's, the value's, none
    const int at = part * n + out0 + 4 * (lane - part * (Outputs / 4));
    load_to_lds(m0, part < 2 ? static_cast<unsigned int>(at) * 4U : kOutside,
                scalar_resource(bias, bias != nullptr ? static_cast<unsigned int>(2 * n) * 4U : 0U));
}

/// Finishes a wavefront's tiles: outputs of TM x TN / 2 MFMA tiles from row
/// @p row and output column @p col on (the lane's own).
template <typename T, Gate G, int TM, int TN>
__device__ __forceinline__ void finish_tiles(const typename Mma<T>::Acc (&acc)[TM][TN], int lane, int row0, int col0,
                                             T* c, T* pre, const GatedArgs& args) {
    constexpr int E = Mma<T>::kEdge;
#pragma unroll
    for (int o = 0; o < TN / 2; ++o)
#pragma unroll
        for (int q = 0; q < Mma<T>::kRuns; ++q) {
            const int col = col0 + o * E + Mma<T>::column(lane, q);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                float gate[4], value[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    gate[e] = acc[i][2 * o][4 * q + e];
                    value[e] = acc[i][2 * o + 1][4 * q + e];
                }
                finish_quad<T, G>(gate, value, row0 + i * E + lane % E, col, c, pre, args);
            }
        }
}

/// A lane's part of a group's largest value: @p v's where @p col, the first one's, and
/// what follows lie before column @p n.
template <int Count> __device__ __forceinline__ void cut_columns(float (&v)[Count], int col, int n) {
#pragma unroll
    for (int e = 0; e < Count; ++e) {
        v[e] = col + e < n ? v[e] : 0.0F;
    }
}

/// The codes of a wavefront's tiles, from registers to memory: 4 bytes of a row a lane.
/// In bf16 an MFMA tile's 32 outputs are a group, a lane and the one across from it
/// holding a row of it; in fp32 two tiles of 16 are, of this wavefront or, where it has
/// only one, of this and the next one of the row, which trade their halves' largest
/// values through LDS (@p exchange: two for each of @p Rows rows of a half).
template <typename T, int TM, int TN, int Rows>
__device__ __forceinline__ void finish_codes(const typename Mma<T>::Acc (&acc)[TM][TN], int lane, int wave_n,
                                             int tile_row, int row0, int col0, float* exchange,
                                             const GatedArgs& args) {
    constexpr int E = Mma<T>::kEdge;
    constexpr int kTiles = kCodeGroup / E < TN / 2 ? kCodeGroup / E : TN / 2; // of this wavefront's in a group
    constexpr bool kTraded = kTiles * E < kCodeGroup;
    constexpr int kValues = E * E / kWave; // a lane's of a tile
    auto values = [&](int i, int o, int half, float (&v)[kValues]) {
#pragma unroll
        for (int q = 0; q < Mma<T>::kRuns; ++q) {
            float four[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                four[e] = acc[i][2 * o + half][4 * q + e];
            }
            cut_columns(four, col0 + o * E + Mma<T>::column(lane, q), args.n);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[4 * q + e] = four[e];
            }
        }
    };
    auto largest_of = [&](int i, int o0, int half) {
        float largest = 0.0F;
#pragma unroll
        for (int o = o0; o < o0 + kTiles; ++o) {
            float v[kValues];
            values(i, o, half, v);
            largest = fmaxf(largest, largest_finite(v));
        }
        if constexpr (sizeof(T) == 4) {
            largest = attention::combine_rows<16>(largest, Max{});
        }
        return attention::combine_rows<32>(largest, Max{});
    };
    if constexpr (kTraded) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < TM; ++i)
                exchange[(half * Rows + tile_row + i * E + lane % E) * 2 + (wave_n & 1)] = largest_of(i, 0, half);
        __syncthreads();
    }
    const int groups = (args.n + kCodeGroup - 1) / kCodeGroup;
#pragma unroll
    for (int o0 = 0; o0 < TN / 2; o0 += kTiles)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                float largest;
                if constexpr (kTraded) {
                    const float* const both = exchange + (half * Rows + tile_row + i * E + lane % E) * 2;
                    largest = fmaxf(both[0], both[1]);
                } else {
                    largest = largest_of(i, o0, half);
                }
                const int row = row0 + tile_row + i * E + lane % E;
                const std::uint32_t scale = code_scale(largest);
                const float inverse = code_inverse(scale);
                const int group = (col0 + o0 * E) / kCodeGroup;
                if (row >= args.m) {
                    continue;
                }
                if (lane < E && group < groups && (!kTraded || (wave_n & 1) == 0)) {
                    args.scales[static_cast<std::int64_t>(row) * 2 * groups + half * groups + group] =
                        static_cast<std::uint8_t>(scale);
                }
                std::uint8_t* const to = args.codes + static_cast<std::int64_t>(row) * args.ld_pre + half * args.n;
#pragma unroll
                for (int o = o0; o < o0 + kTiles; ++o) {
                    float v[kValues];
                    values(i, o, half, v);
#pragma unroll
                    for (int q = 0; q < Mma<T>::kRuns; ++q) {
                        const int col = col0 + o * E + Mma<T>::column(lane, q);
                        store_bytes<1>(to + col, {{four_codes(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3], inverse)}},
                                       args.n - col);
                    }
                }
            }
}

/// Where the codes of a bf16 tile lie in LDS: rows of the gate's, then the value's
/// codes, 16-byte pieces turned by the row so that the rows that a wavefront writes at
/// once spread over the banks; behind them a row's scales.
template <int BO> struct CodeRows {
    static constexpr int kPitch = 2 * BO;
    static constexpr int kPieces = kPitch / 16;
    static constexpr int kGroups = BO / kCodeGroup; // of a half
    __device__ __forceinline__ static int piece(int row, int at) {
        return row * kPitch + ((at ^ (row / (128 / BO) & (kPieces - 1))) << 4);
    }
    __device__ __forceinline__ static int scale(int rows, int row, int half, int group) {
        return rows * kPitch + (row * 2 + half) * kGroups + group;
    }
};

template <typename S>
__device__ __forceinline__ void stage_codes(const floatx16 (&acc)[S::kTM][S::kTN], unsigned char* lds, int wave_m,
                                            int wave_n, int lane, int col0, int n) {
    constexpr int E = S::kEdge;
    constexpr int kBO = S::kBN / 2;
    using Place = CodeRows<kBO>;
    static_assert(S::kBM * (Place::kPitch + 2 * Place::kGroups) <= S::kSlots * S::kStageBytes, "the ring holds the codes");
    static_assert(E == kCodeGroup, "a tile's row is a group");
    const bool whole = col0 + kBO <= n;
#pragma unroll
    for (int o = 0; o < S::kTN / 2; ++o)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < S::kTM; ++i) {
                const int tile = wave_n * (S::kTN / 2) + o;
                const int row = (wave_m * S::kTM + i) * E + lane % E;
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    v[e] = acc[i][2 * o + half][e];
                }
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        v[e] = col0 + tile * E + Mma<std::uint16_t>::column(lane, e / 4) + e % 4 < n ? v[e] : 0.0F;
                    }
                }
                const std::uint32_t scale = code_scale(attention::combine_rows<32>(largest_finite(v), Max{}));
                const float inverse = code_inverse(scale);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int at = half * kBO + tile * E + Mma<std::uint16_t>::column(lane, q);
                    *reinterpret_cast<std::uint32_t*>(lds + Place::piece(row, at / 16) + at % 16) =
                        four_codes(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3], inverse);
                }
                if (lane < E) {
                    lds[Place::scale(S::kBM, row, half, tile)] = static_cast<std::uint8_t>(scale);
                }
            }
}

template <int BM, int BO, int Threads, bool Streaming>
__device__ __forceinline__ void store_codes(const unsigned char* lds, int row0, int col0, const GatedArgs& args) {
    using Place = CodeRows<BO>;
    constexpr int kOfHalf = Place::kPieces / 2;
    for (int i = static_cast<int>(threadIdx.x); i < BM * Place::kPieces; i += Threads) {
        const int row = i / Place::kPieces;
        const int at = i % Place::kPieces;
        const int half = at / kOfHalf;
        const int col = col0 + at % kOfHalf * 16;
        if (row0 + row < args.m && col < args.n) {
            const Vec16 v = load16(lds + Place::piece(row, at));
            store_bytes<4, Streaming>(args.codes + static_cast<std::int64_t>(row0 + row) * args.ld_pre + half * args.n + col,
                           {{v.w[0], v.w[1], v.w[2], v.w[3]}}, args.n - col);
        }
    }
    const int groups = (args.n + kCodeGroup - 1) / kCodeGroup;
    for (int i = static_cast<int>(threadIdx.x); i < BM * 2; i += Threads) {
        const int row = i / 2;
        const int half = i % 2;
        if (row0 + row < args.m) {
            std::uint8_t* const to =
                args.scales + static_cast<std::int64_t>(row0 + row) * 2 * groups + half * groups + col0 / kCodeGroup;
#pragma unroll
            for (int g = 0; g < Place::kGroups; ++g) {
                if (col0 / kCodeGroup + g < groups) {
                    to[g] = lds[Place::scale(BM, row, half, g)];
                }
            }
        }
    }
}

/// finish_tiles for bf16, through the drained ring: the MFMA layout gives a lane 8
/// bytes of a row, 32 rows a store; from LDS the workgroup's rows go out as 16-byte
/// pieces, side by side (12608 x 2048 x 768: 105 -> 99 us when it came). @p Streaming:
/// C past the caches. @p Codes: the preactivations' codes, too.
template <typename S, Gate G, bool Streaming, bool Codes>
__device__ __forceinline__ void finish_staged(const floatx16 (&acc)[S::kTM][S::kTN], unsigned char* lds, bool loading,
                                              int wave_m, int wave_n, int lane, int row0, int col0, std::uint16_t* c,
                                              std::uint16_t* pre, const GatedArgs& args) {
    using T = std::uint16_t;
    constexpr int E = S::kEdge;
    constexpr int kBO = S::kBN / 2;
    constexpr int kV = Elem<T>::kPerVec;
    constexpr int kRowChunks = kBO / kV; // 16-byte pieces of a row
    static_assert(S::kBM * kRowChunks * 16 <= S::kSlots * S::kStageBytes, "the ring holds the outputs");
    static_assert((kRowChunks & (kRowChunks - 1)) == 0, "placed by exclusive or");
    auto staged = [&](int row, int chunk) {
        return lds + (row * kRowChunks + (chunk ^ ((row >> 1) & (kRowChunks - 1)))) * 16;
    };
    // One of C, the gate's and the value's preactivations (0, 1, 2).
    auto pass = [&](auto which, T* to, int ld) {
        constexpr int kWhich = decltype(which)::value;
        if (!loading) {
#pragma unroll
            for (int o = 0; o < S::kTN / 2; ++o)
#pragma unroll
                for (int q = 0; q < Mma<T>::kRuns; ++q) {
                    const int col = (wave_n * (S::kTN / 2) + o) * E + Mma<T>::column(lane, q);
#pragma unroll
                    for (int i = 0; i < S::kTM; ++i) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float gate = acc[i][2 * o][4 * q + e];
                            const float value = acc[i][2 * o + 1][4 * q + e];
                            v[e] = kWhich == 0 ? gate_value<G>(gate) * value : kWhich == 1 ? gate : value;
                        }
                        const int row = (wave_m * S::kTM + i) * E + lane % E;
                        store_run<T, 4, false>(reinterpret_cast<T*>(staged(row, col / kV)) + col % kV, round_run<T, 4>(v));
                    }
                }
        }
        __syncthreads();
        for (int i = static_cast<int>(threadIdx.x); i < S::kBM * kRowChunks; i += S::kThreads) {
            const int row = i / kRowChunks;
            const int chunk = i % kRowChunks;
            const int count = args.n - col0 - kV * chunk;
            if (row0 + row < args.m && count > 0) {
                const Run<T, kV> run = load_run<T, kV>(reinterpret_cast<const T*>(staged(row, chunk)));
                T* const at = to + static_cast<std::int64_t>(row0 + row) * ld + col0 + kV * chunk;
                if (count >= kV) {
                    store_run_unaligned<T, kV, Streaming && kWhich == 0>(at, run);
                } else {
                    store_some<T, kV>(at, run, count);
                }
            }
        }
    };
    pass(std::integral_constant<int, 0>{}, c, args.ldc);
    if constexpr (Codes) {
        stage_barrier(false); // (C is in registers on its way, not in LDS any more)
        if (!loading) {
            stage_codes<S>(acc, lds, wave_m, wave_n, lane, col0, args.n);
        }
        stage_barrier(false);
        store_codes<S::kBM, kBO, S::kThreads, Streaming>(lds, row0, col0, args);
    } else if (pre != nullptr) {
        __syncthreads();
        pass(std::integral_constant<int, 1>{}, pre, args.ld_pre);
        __syncthreads();
        pass(std::integral_constant<int, 2>{}, pre + args.n, args.ld_pre);
    }
}

/// ring_multiply with the next k-block's fragments read under a block's MFMAs. A
/// tile alone on its CU sends the next stage's loads off behind the first block's
/// MFMAs, which cover what issuing them costs (320 x 128 outputs: 12288 x 2048 x
/// 768 in 79 us before, 75 so); where workgroups share a CU, first of all (128 x 64:
/// 88 and 92).
template <typename S, typename Loads, typename Start>
__device__ __forceinline__ void gated_multiply(const Loads& loads, const unsigned char* lds, int wave_m, int wave_n,
                                               int lane, int stages, floatx16 (&acc)[S::kTM][S::kTN],
                                               const Start& start) {
    constexpr int E = S::kEdge;
    constexpr int kBlocks = S::kBK / kKBlock<std::uint16_t>;
    constexpr bool kAlone = S::kBN > 128;
    const unsigned int a_fragment = static_cast<unsigned int>((wave_m * E * S::kTM + lane % E) * S::kRowBytes);
    const unsigned int b_fragment = static_cast<unsigned int>((S::kBM + wave_n * E * S::kTN + lane % E) * S::kRowBytes);
    unsigned int column[kBlocks];
#pragma unroll
    for (int kb = 0; kb < kBlocks; ++kb) {
        column[kb] = static_cast<unsigned int>(S::place(lane % E, kWave / E * kb + lane / E) * 16);
    }
#pragma unroll
    for (int g = 0; g < S::kSlots - 1; ++g) {
        loads.issue(g, g);
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"((S::kSlots - 2) * S::kLoads) : "memory");
    start(acc);
    int slot = 0;
    int free_slot = S::kSlots - 1;
    for (int g = 0; g < stages; ++g) {
        // Stage g landed (each wavefront waits for its own pieces) and every
        // wavefront is done reading stage g - 1, whose slot is refilled.
        wait_fragments();
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((S::kSlots - 2) * S::kLoads) : "memory");
        const unsigned char* const base = lds + slot * S::kStageBytes;
        Vec16 fa[2][S::kTM];
        Vec16 fb[2][S::kTN];
        auto read = [&](int kb, int set) {
#pragma unroll
            for (int i = 0; i < S::kTM; ++i)
                fa[set][i] = load16(base + a_fragment + i * E * S::kRowBytes + column[kb]);
#pragma unroll
            for (int j = 0; j < S::kTN; ++j)
                fb[set][j] = load16(base + b_fragment + j * E * S::kRowBytes + column[kb]);
        };
        read(0, 0);
        if constexpr (!kAlone) {
            loads.issue(g + S::kSlots - 1, free_slot);
        }
        static_for<kBlocks>([&](auto block) {
            constexpr int kb = decltype(block)::value;
            if constexpr (kb + 1 < kBlocks) {
                read(kb + 1, (kb + 1) & 1);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < S::kTM; ++i)
#pragma unroll
                for (int j = 0; j < S::kTN; ++j)
                    Mma<std::uint16_t>::run(acc[i][j], fb[kb & 1][j], fa[kb & 1][i]);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kAlone && kb == 0) {
                loads.issue(g + S::kSlots - 1, free_slot);
                __builtin_amdgcn_sched_barrier(0);
            }
        });
        free_slot = slot;
        slot = slot + 1 == S::kSlots ? 0 : slot + 1;
    }
    stage_barrier(true);
}

template <typename T, typename S, Gate G, bool Streaming, bool Codes>
__global__ __launch_bounds__(S::kThreads) void gated_ring_kernel(const T* __restrict__ a, const T* __restrict__ b,
                                                                 const float* __restrict__ bias, T* c, T* pre,
                                                                 GatedArgs args, TileMap map) {
    static_assert(kGatedLds<S> <= 160 * 1024, "LDS");
    static_assert(S::kTN % 2 == 0, "a wavefront holds both factors of its outputs");
    static_assert(S::kWaves * S::kLoadRows % 16 == 0 && S::kEdge % S::kLoadRows == 0, "a piece is of one half");
    extern __shared__ Vec16 lds_vectors[];
    unsigned char* const lds = reinterpret_cast<unsigned char*>(lds_vectors);
    const unsigned int lds_base = __builtin_amdgcn_readfirstlane(lds_address(lds));
    const int lane = lane_id();
    const int wavefront = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const bool loading = S::kLoaders && wavefront >= S::kWaves;
    const int wave = loading ? wavefront - S::kWaves : wavefront;
    const int wave_m = wave / S::kWN;
    const int wave_n = wave % S::kWN;
    // The tile grid is that of a product with 2 n columns.
    GemmArgs grid{};
    grid.m = args.m;
    grid.n = 2 * args.n;
    grid.count = 1;
    int row0, col0;
    if (!ring_tile<S>(grid, map, RingSpot{0, static_cast<int>(blockIdx.x)}, row0, col0)) {
        return; // the whole workgroup, before any barrier
    }
    col0 /= 2;
    const GatedLoads<T, S> loads(a, b, args, row0, col0, wave, lane, lds_base);
    if (wavefront == (S::kLoaders ? S::kWaves : 0)) { // one that loads the stages too: they come in order
        load_bias<S::kBN / 2>(bias, col0, args.n, lane, lds_base + static_cast<unsigned int>(S::kBiasOffset));
    }
    const StartAtBias<T, S> start{reinterpret_cast<const float*>(lds + S::kBiasOffset) +
                                  wave_n * (S::kTN / 2) * S::kEdge + Mma<T>::column(lane, 0)};
    typename Mma<T>::Acc acc[S::kTM][S::kTN];
    const int stages = (args.k + 127) / 128 * (128 / S::kBK);
    if constexpr (S::kAhead) {
        ring_multiply<T, S>(loads, lds, wave_m, wave_n, lane, loading, stages, acc, start);
    } else {
        gated_multiply<S>(loads, lds, wave_m, wave_n, lane, stages, acc, start);
    }
    if constexpr (sizeof(T) == 2) {
        finish_staged<S, G, Streaming, Codes>(acc, lds, loading, wave_m, wave_n, lane, row0, col0, c, pre, args);
    } else if (!loading) { // 16 bytes a lane, 64 a row: no slower than through LDS
        finish_tiles<T, G, S::kTM, S::kTN>(acc, lane, row0 + wave_m * S::kEdge * S::kTM,
                                           col0 + wave_n * S::kEdge * S::kTN / 2, c, pre, args);
        if constexpr (Codes) {
            static_assert(!S::kLoaders, "every wavefront passes the barrier");
            finish_codes<T, S::kTM, S::kTN, S::kBM>(acc, lane, wave_n, wave_m * S::kEdge * S::kTM, row0,
                                                    col0 + wave_n * S::kEdge * S::kTN / 2,
                                                    reinterpret_cast<float*>(lds), args);
        }
    }
}

} // namespace cuvit::detail::gemm
