// The gated product: C = activation(gate) * value, [gate, value] = A.B^T + bias,
// B [2 n, k] with the gate's n rows before the value's.
//
// A workgroup's tile takes the same columns of both halves, and a wavefront the
// gate's and the value's MFMA tiles of the same outputs, so that both factors of
// an output are the same register of two accumulators: the epilogue multiplies
// them where they lie, and the [m, 2 n] preactivations never leave the chip
// unless they are asked for.
//
// Three kernels: gated_rows_kernel for single tokens and a few rows; gated_ring_kernel
// (gated_ring.hpp) for operands whose rows are whole 16-byte chunks; and
// gated_loose_kernel for any sizes, strides and alignment, where operands go through
// registers into LDS, a stage of 128 bytes of k ahead (two ahead: 788 x 2048 x 767 in
// bf16 18.4 -> 20.6 us), at any value's address (3152 x 2048 x 767: 45 us, x 768 on the
// ring 24.7). MFMAs, fragments and the placement in LDS are the GEMMs'
// (gemm_kernel.hpp, gemm_ring.hpp).
//
// Bound: the MFMAs and what feeds them. 12608 x 2048 x 768 in bf16 takes 77 to 84 us
// by card (1.03 to 0.94 PFLOP/s), the plain product of the same operands as one
// library call 82; fp32 runs at the 137 TFLOP/s that the clock under its MFMAs
// allows (6304 x 2048 x 768: 289 us).
#include "gated_choice.hpp"
#include "gated_ring.hpp"

#include <type_traits>

namespace cuvit::detail {
namespace gemm {
namespace {

/// WM x 2 wavefronts of TM x TO MFMA tiles of outputs.
template <typename T, int WM, int TM, int TO> struct LooseTile {
    static constexpr int kE = Mma<T>::kEdge;
    static constexpr int kThreads = 2 * kWave * WM;
    static constexpr int kBM = kE * TM * WM;
    static constexpr int kBO = 2 * kE * TO;  // outputs
    static constexpr int kTM = TM;           // a wavefront's MFMA tiles of rows
    static constexpr int kTO = TO;           // and of outputs
    static constexpr int kV = Elem<T>::kPerVec;
    static constexpr int kBK = 8 * kV;
    static constexpr int kRows = kBM + 2 * kBO; // of a stage: A's, then the gate's and the value's tiles in turn
    static constexpr int kStep = kThreads / 8;           // stage rows between a thread's chunks
    static constexpr int kChunks = kRows / kStep;        // 16-byte chunks a thread loads
    static_assert(kRows % kStep == 0 && kBM % kStep == 0, "whole chunks of either operand");
};

template <typename T, typename S, Gate G>
__global__ __launch_bounds__(S::kThreads) void gated_loose_kernel(const T* __restrict__ a, const T* __restrict__ b,
                                                                  const float* __restrict__ bias, T* c, T* pre,
                                                                  GatedArgs args) {
    constexpr int E = S::kE;
    __shared__ Vec16 stage[S::kRows * 8];
    const int tiles_n = (args.n + S::kBO - 1) / S::kBO;
    const int row0 = static_cast<int>(blockIdx.x / static_cast<unsigned int>(tiles_n)) * S::kBM;
    const int col0 = static_cast<int>(blockIdx.x % static_cast<unsigned int>(tiles_n)) * S::kBO;
    const int thread = static_cast<int>(threadIdx.x);
    const int lane = lane_id();
    const int wave_m = thread / kWave / 2;
    const int wave_n = thread / kWave % 2;

    // The rows this thread loads: chunk thread % 8 of stage rows
    // thread / 8 + kStep p.
    // Rows past the operands' ends repeat the last one: their sums are not stored.
    const int chunk = thread % 8;
    const T* from[S::kChunks];
    int left[S::kChunks]; // values from there to the operand's end, as far as it counts
#pragma unroll
    for (int p = 0; p < S::kChunks; ++p) {
        const int row = thread / 8 + S::kStep * p;
        std::int64_t behind;
        if (S::kStep * p < S::kBM) {
            const int at = min(row0 + row, args.m - 1);
            from[p] = a + static_cast<std::int64_t>(at) * args.lda;
            behind = static_cast<std::int64_t>(args.m - 1 - at) * args.lda;
        } else {
            const int tile = (row - S::kBM) / E; // even: the gate's, odd: the value's
            const int at = min(col0 + tile / 2 * E + (row - S::kBM) % E, args.n - 1) + ((tile & 1) != 0 ? args.n : 0);
            from[p] = b + static_cast<std::int64_t>(at) * args.ldb;
            behind = static_cast<std::int64_t>(2 * args.n - 1 - at) * args.ldb;
        }
        from[p] += chunk * S::kV;
        left[p] = args.k - chunk * S::kV + static_cast<int>(behind < S::kV ? behind : S::kV);
    }
    Run<T, S::kV> held[S::kChunks];
    auto load = [&](int k0) {
        if (k0 + S::kBK <= args.k) {
#pragma unroll
            for (int p = 0; p < S::kChunks; ++p)
                held[p] = load_run_unaligned<T, S::kV>(from[p] + k0);
        } else {
            // The last, cut stage: whole runs into the next row where there is one,
            // and zeros for what is not this row's.
            const int count = min(max(args.k - k0 - chunk * S::kV, 0), S::kV);
#pragma unroll
            for (int p = 0; p < S::kChunks; ++p) {
                if (left[p] - k0 >= S::kV) {
                    held[p] = keep_some<T, S::kV>(load_run_unaligned<T, S::kV>(from[p] + k0), count);
                } else {
                    held[p] = load_some<T, S::kV>(from[p] + k0, count);
                }
            }
        }
    };

    typename Mma<T>::Acc acc[S::kTM][2 * S::kTO];
    StartAtZero{}(acc);
    auto place = [](int row, int slot) { return row * 8 + (slot ^ ((row >> 1) & 7)); };
    if (args.k > 0) {
        load(0);
    }
    for (int k0 = 0; k0 < args.k; k0 += S::kBK) {
        __syncthreads(); // the last stage is read
#pragma unroll
        for (int p = 0; p < S::kChunks; ++p)
            stage[place(thread / 8 + S::kStep * p, chunk)] = __builtin_bit_cast(Vec16, held[p]);
        __syncthreads();
        if (k0 + S::kBK < args.k) {
            load(k0 + S::kBK);
        }
        constexpr int kPerBlock = kWave / E;
#pragma unroll
        for (int kb = 0; kb < 8 / kPerBlock; ++kb) {
            const int slot = kPerBlock * kb + lane / E;
            Vec16 fa[S::kTM];
            Vec16 fb[2 * S::kTO];
#pragma unroll
            for (int i = 0; i < S::kTM; ++i)
                fa[i] = stage[place((wave_m * S::kTM + i) * E + lane % E, slot)];
#pragma unroll
            for (int j = 0; j < 2 * S::kTO; ++j)
                fb[j] = stage[place(S::kBM + (wave_n * 2 * S::kTO + j) * E + lane % E, slot)];
#pragma unroll
            for (int i = 0; i < S::kTM; ++i)
#pragma unroll
                for (int j = 0; j < 2 * S::kTO; ++j)
                    Mma<T>::run(acc[i][j], fb[j], fa[i]);
        }
    }
    const int first_col = col0 + wave_n * S::kTO * E;
#pragma unroll
    for (int j = 0; j < 2 * S::kTO; ++j)
#pragma unroll
        for (int q = 0; q < Mma<T>::kRuns; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = first_col + j / 2 * E + Mma<T>::column(lane, q) + e;
                const float term = bias != nullptr && col < args.n ? bias[(j & 1) * args.n + col] : 0.0F;
#pragma unroll
                for (int i = 0; i < S::kTM; ++i)
                    acc[i][j][4 * q + e] += term;
            }
    finish_tiles<T, G, S::kTM, 2 * S::kTO>(acc, lane, row0 + wave_m * S::kTM * E, first_col, c, pre, args);
}

/// Sixteen MFMA rows against sixteen: bf16 by k-blocks of 32, fp32 of 16.
template <typename T> struct RowMma;
template <> struct RowMma<float> {
    static constexpr int kBlock = 16;
    __device__ __forceinline__ static void run(floatx4& acc, const Vec16& b, const Vec16& a) {
        Mma<float>::run(acc, b, a);
    }
};
template <> struct RowMma<std::uint16_t> {
    static constexpr int kBlock = 32;
    __device__ __forceinline__ static void run(floatx4& acc, const Vec16& b, const Vec16& a) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a),
                                                      acc, 0, 0, 0);
    }
};

/// Up to 16 TM rows (single tokens): bound by reading B once. A workgroup takes
/// eight outputs, their eight gate and eight value rows as one MFMA tile, so that
/// 2048 outputs fill the chip; its wavefronts split K, two k-blocks (a cache line of
/// each row) at a time, straight from memory into fragments, and add their parts in
/// LDS in a fixed order. Any alignment. In bf16, us (the 64-row tiles below): 1 x
/// 2048 x 768 3.5 (5.1), 32 rows of it 4.3 (5.1); 64 rows 6.0 (5.2), so those come
/// here only where the tiles would be the loose kernel's, 64 x 1958 x 741 12.7 (13.0),
/// in fp32 11.0 (65 rows in tiles 15.9).
template <typename T, int TM, Gate G>
__global__ __launch_bounds__(512) void gated_rows_kernel(const T* __restrict__ a, const T* __restrict__ b,
                                                         const float* __restrict__ bias, T* c, T* pre,
                                                         GatedArgs args) {
    constexpr int kWaves = 8;
    constexpr int kV = Elem<T>::kPerVec;
    constexpr int kBlock = RowMma<T>::kBlock;
    constexpr int kPair = 2 * kBlock;
    __shared__ float parts[kWaves][16 * TM][17];
    const int lane = lane_id();
    const int wave = static_cast<int>(threadIdx.x) / kWave;
    const int out0 = static_cast<int>(blockIdx.x) * 8;
    const int row = lane % 16;
    // (Rows and outputs past the last repeat it: their sums are not stored.)
    const int out = min(out0 + row % 8, args.n - 1);
    const int chunk = lane / 16 * kV;
    const T* from_a[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i)
        from_a[i] = a + static_cast<std::int64_t>(min(16 * i + row, args.m - 1)) * args.lda + chunk;
    const T* const from_b = b + (static_cast<std::int64_t>(row < 8 ? 0 : args.n) + out) * args.ldb + chunk;
    floatx4 acc[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i)
        acc[i] = floatx4{0.0F, 0.0F, 0.0F, 0.0F};
    constexpr int kTogether = TM == 1 ? 2 : 1;
    for (int k0 = wave * kPair; k0 < args.k; k0 += kTogether * kWaves * kPair) {
        Run<T, kV> fa[TM][2 * kTogether], fb[2 * kTogether];
#pragma unroll
        for (int p = 0; p < kTogether; ++p) {
            const int at = k0 + p * kWaves * kPair;
            const bool whole = at + kPair <= args.k;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = at + h * kBlock;
                const int count = min(max(args.k - k - chunk, 0), kV);
                auto load = [&](const T* from) {
                    return whole ? load_run_unaligned<T, kV>(from + k) : load_some<T, kV>(from + k, count);
                };
                fb[2 * p + h] = load(from_b);
#pragma unroll
                for (int i = 0; i < TM; ++i)
                    fa[i][2 * p + h] = load(from_a[i]);
            }
        }
#pragma unroll
        for (int p = 0; p < 2 * kTogether; ++p)
#pragma unroll
            for (int i = 0; i < TM; ++i)
                RowMma<T>::run(acc[i], __builtin_bit_cast(Vec16, fb[p]), __builtin_bit_cast(Vec16, fa[i][p]));
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            parts[wave][16 * i + row][4 * (lane / 16) + e] = acc[i][e];
    __syncthreads();
    const int thread = static_cast<int>(threadIdx.x);
    const int token = thread / 8; // up to 64 of them
    const int column = thread % 8;
    if (token >= args.m || out0 + column >= args.n) {
        return;
    }
    float gate = bias != nullptr ? bias[out0 + column] : 0.0F;
    float value = bias != nullptr ? bias[args.n + out0 + column] : 0.0F;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        gate += parts[w][token][column];
        value += parts[w][token][8 + column];
    }
    Elem<T>::store(c + static_cast<std::int64_t>(token) * args.ldc + out0 + column, gate_value<G>(gate) * value);
    if (pre != nullptr) {
        T* const to = pre + static_cast<std::int64_t>(token) * args.ld_pre + out0 + column;
        Elem<T>::store(to, gate);
        Elem<T>::store(to + args.n, value);
    }
}

/// @p run with the activation as a constant.
template <typename Run> hipError_t with_gate(Gate gate, Run&& run) {
    switch (gate) {
    case Gate::kSilu: return run(std::integral_constant<Gate, Gate::kSilu>{});
    case Gate::kGelu: return run(std::integral_constant<Gate, Gate::kGelu>{});
    default: return run(std::integral_constant<Gate, Gate::kGeluTanh>{});
    }
}

/// Whether C goes past the caches: where it is more than the L2s hold (32 MB) and
/// its rows are whole 16-byte pieces. With the down projection behind it, in us: 51.6
/// MB of C 141 -> 129; 12.9 MB 44 and 49, so there it stays in them.
template <typename T> bool past_caches(const T* c, const GatedArgs& args) {
    return static_cast<std::int64_t>(args.m) * args.n * static_cast<std::int64_t>(sizeof(T)) > (std::int64_t{32} << 20) &&
           aligned16(c) && args.ldc % Elem<T>::kPerVec == 0;
}

template <typename S, typename T>
hipError_t launch_ring(const T* a, const T* b, const float* bias, T* c, T* pre, const GatedArgs& args,
                       const TileMap& map, hipStream_t stream) {
    const std::int64_t tiles_m = (static_cast<std::int64_t>(args.m) + S::kBM - 1) / S::kBM;
    const std::int64_t tiles_n = (2 * static_cast<std::int64_t>(args.n) + S::kBN - 1) / S::kBN;
    const std::int64_t tiles =
        map.px > 0 ? 8 * ((tiles_m + map.px - 1) / map.px) * ((tiles_n + map.py - 1) / map.py) : tiles_m * tiles_n;
    if (!launchable(tiles, S::kThreads)) {
        return hipErrorInvalidConfiguration;
    }
    auto run = [&](auto chosen) -> hipError_t {
        constexpr auto kernel = decltype(chosen)::kValue;
        if (const hipError_t opted = allow_lds<kernel>(kGatedLds<S>); opted != hipSuccess) {
            return opted;
        }
        kernel<<<static_cast<unsigned int>(tiles), S::kThreads, kGatedLds<S>, stream>>>(a, b, bias, c, pre, args, map);
        return hipGetLastError();
    };
    return with_gate(args.gate, [&](auto gate) -> hipError_t {
        constexpr Gate kGate = decltype(gate)::value;
        // (Tiles alone on their CUs are those of the largest products.)
        if constexpr (S::kBN > 128) {
            if (past_caches(c, args)) {
                return run(KernelConstant<gated_ring_kernel<T, S, kGate, true>>{});
            }
        }
        return run(KernelConstant<gated_ring_kernel<T, S, kGate, false>>{});
    });
}

hipError_t launch_tile(const float* a, const float* b, const float* bias, float* c, float* pre, const GatedArgs& args,
                       hipStream_t stream) {
    auto launch = [&](auto shape) {
        using S = decltype(shape);
        return launch_ring<S>(a, b, bias, c, pre, args, gated_map_f32(args, S::kBM, S::kBN, compute_units()), stream);
    };
    switch (choose_gated_f32(args, compute_units())) {
    case GatedTileF32::k32x16Alone: return launch(RingShape<float, 2, 1, 1, 2, 3, true, true>{});
    case GatedTileF32::k32x32: return launch(RingShape<float, 2, 2, 1, 2, 2, true>{});
    case GatedTileF32::k32x32Alone: return launch(RingShape<float, 2, 2, 1, 2, 3, true>{});
    default: return launch(RingShape<float, 2, 2, 2, 2, 2, true>{});
    }
}

hipError_t launch_tile(const std::uint16_t* a, const std::uint16_t* b, const float* bias, std::uint16_t* c,
                       std::uint16_t* pre, const GatedArgs& args, hipStream_t stream) {
    using T = std::uint16_t;
    const GatedChoice choice = choose_gated(args, compute_units());
    auto launch = [&](auto shape) {
        return launch_ring<decltype(shape)>(a, b, bias, c, pre, args, choice.map, stream);
    };
    switch (choice.tile) {
    case GatedTile::k64x32Alone: return launch(RingShape<T, 2, 1, 1, 2, 4, true, true>{});
    case GatedTile::k64x64: return launch(RingShape<T, 2, 2, 1, 2, 2>{});
    case GatedTile::k64x64Alone: return launch(RingShape<T, 2, 2, 1, 2, 3>{});
    case GatedTile::k128x64: return launch(RingShape<T, 4, 2, 1, 2, 2>{});
    case GatedTile::k192x128: return launch(RingShape<T, 2, 4, 3, 2, 2>{});
    case GatedTile::k256x128: return launch(RingShape<T, 2, 4, 4, 2, 2>{});
    default: return launch(RingShape<T, 2, 4, 5, 2, 2>{});
    }
}

/// Whether an operand's rows are whole 16-byte chunks that the ring's loads reach
/// from a tile's first row.
template <typename T> bool ring_operand(const T* base, int ld, int depth) {
    return aligned16(base) && ld % Elem<T>::kPerVec == 0 && depth % Elem<T>::kPerVec == 0 &&
           static_cast<std::int64_t>(320) * ld * static_cast<std::int64_t>(sizeof(T)) < kMaxSpan;
}

template <typename T>
hipError_t launch_gated(const T* a, const T* b, const float* bias, T* c, T* pre, const GatedArgs& args,
                        hipStream_t stream) {
    auto rows = [&](auto tiles) -> hipError_t {
        const std::int64_t groups = (static_cast<std::int64_t>(args.n) + 7) / 8;
        if (!launchable(groups, 512)) {
            return hipErrorInvalidConfiguration;
        }
        return with_gate(args.gate, [&](auto gate) -> hipError_t {
            gated_rows_kernel<T, decltype(tiles)::value, decltype(gate)::value>
                <<<static_cast<unsigned int>(groups), 512, 0, stream>>>(a, b, bias, c, pre, args);
            return hipGetLastError();
        });
    };
    const bool whole_chunks = ring_operand(a, args.lda, args.k) && ring_operand(b, args.ldb, args.k);
    if (args.m <= kGatedRows / 4) {
        return rows(std::integral_constant<int, 1>{});
    }
    if (args.m <= kGatedRows / 2) {
        return rows(std::integral_constant<int, 2>{});
    }
    if (args.m <= kGatedRows && !whole_chunks) {
        return rows(std::integral_constant<int, 4>{});
    }
    // (The bias is loaded from one descriptor, 32-bit offsets.)
    if (whole_chunks && args.n < (1 << 27)) {
        return launch_tile(a, b, bias, c, pre, args, stream);
    }
    auto loose = [&](auto tile) -> hipError_t {
        using S = decltype(tile);
        const std::int64_t tiles = (static_cast<std::int64_t>(args.m) + S::kBM - 1) / S::kBM *
                                   ((static_cast<std::int64_t>(args.n) + S::kBO - 1) / S::kBO);
        if (!launchable(tiles, S::kThreads)) {
            return hipErrorInvalidConfiguration;
        }
        return with_gate(args.gate, [&](auto gate) -> hipError_t {
            gated_loose_kernel<T, S, decltype(gate)::value>
                <<<static_cast<unsigned int>(tiles), S::kThreads, 0, stream>>>(a, b, bias, c, pre, args);
            return hipGetLastError();
        });
    };
    auto tiles = [&](int rows) {
        return (static_cast<std::int64_t>(args.m) + rows - 1) / rows * ((static_cast<std::int64_t>(args.n) + 63) / 64);
    };
    const std::int64_t units = compute_units();
    if constexpr (sizeof(T) == 2) {
        // 64 x 64 outputs; 128 x 64 where such tiles fill the CUs twice, since what a
        // stage loads, at addresses that cross cache lines, is what bounds it (3152 x
        // 2048 x 767: 52 -> 45 us), and for the same reason no smaller ones (of 32 x 64:
        // 788 x 2048 x 767 18.2 and 24.7).
        return tiles(128) >= 2 * units ? loose(LooseTile<T, 4, 1, 1>{}) : loose(LooseTile<T, 2, 1, 1>{});
    } else {
        // fp32 is bound by the MFMAs of the CUs that have a tile: 32 x 32 outputs, 64 x 64
        // from four of these a CU on (64 x 64 against 32 x 32, in us: 100 x 2048 x 767 34.6
        // and 14.9; 788 x 1365 x 513 45.7 and 32.9; 3152 x 1365 x 513 104 and 108).
        return tiles(64) >= 4 * units ? loose(LooseTile<T, 2, 2, 2>{}) : loose(LooseTile<T, 2, 1, 1>{});
    }
}

} // namespace
} // namespace gemm

hipError_t gated_gemm(const float* a, const float* b, const float* bias, float* c, float* preactivations,
                      const GatedArgs& args, hipStream_t stream) {
    return gemm::launch_gated(a, b, bias, c, preactivations, args, stream);
}

hipError_t gated_gemm(const std::uint16_t* a, const std::uint16_t* b, const float* bias, std::uint16_t* c,
                      std::uint16_t* preactivations, const GatedArgs& args, hipStream_t stream) {
    return gemm::launch_gated(a, b, bias, c, preactivations, args, stream);
}

} // namespace cuvit::detail
