// The gated product's kernel for operands of any alignment, and the launches of both
// kernels with tiles, with or without codes of the preactivations (checkpoint.hpp).
// See gated.hip.
#pragma once

#include "gated_choice.hpp"
#include "gated_ring.hpp"

#include <type_traits>

namespace cuvit::detail::gemm {

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

template <typename T, typename S, Gate G, bool Codes>
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
    if constexpr (Codes) {
        __syncthreads(); // the last stage is read
        finish_codes<T, S::kTM, 2 * S::kTO, S::kBM>(acc, lane, wave_n, wave_m * S::kTM * E, row0, first_col,
                                                    reinterpret_cast<float*>(stage), args);
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

template <bool Codes, typename S, typename T>
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
                return run(KernelConstant<gated_ring_kernel<T, S, kGate, true, Codes>>{});
            }
        }
        return run(KernelConstant<gated_ring_kernel<T, S, kGate, false, Codes>>{});
    });
}

template <bool Codes>
hipError_t launch_tile(const float* a, const float* b, const float* bias, float* c, float* pre, const GatedArgs& args,
                       hipStream_t stream) {
    auto launch = [&](auto shape) {
        using S = decltype(shape);
        return launch_ring<Codes, S>(a, b, bias, c, pre, args, gated_map_f32(args, S::kBM, S::kBN, compute_units()), stream);
    };
    switch (choose_gated_f32(args, compute_units())) {
    case GatedTileF32::k32x16Alone:
        // (A group of codes takes 32 outputs.)
        if constexpr (!Codes) {
            return launch(RingShape<float, 2, 1, 1, 2, 3, true, true>{});
        }
        [[fallthrough]];
    case GatedTileF32::k32x32Alone: return launch(RingShape<float, 2, 2, 1, 2, 3, true>{});
    case GatedTileF32::k32x32: return launch(RingShape<float, 2, 2, 1, 2, 2, true>{});
    default: return launch(RingShape<float, 2, 2, 2, 2, 2, true>{});
    }
}

template <bool Codes>
hipError_t launch_tile(const std::uint16_t* a, const std::uint16_t* b, const float* bias, std::uint16_t* c,
                       std::uint16_t* pre, const GatedArgs& args, hipStream_t stream) {
    using T = std::uint16_t;
    const GatedChoice choice = choose_gated(args, compute_units());
    auto launch = [&](auto shape) {
        return launch_ring<Codes, decltype(shape)>(a, b, bias, c, pre, args, choice.map, stream);
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

/// Columns from which the ring, which loads the bias by one descriptor and 32-bit
/// offsets, does not take a product.
constexpr int kRingColumns = 1 << 27;

/// Whether an operand's rows are whole 16-byte chunks that the ring's loads reach
/// from a tile's first row.
template <typename T> bool ring_operand(const T* base, int ld, int depth) {
    return aligned16(base) && ld % Elem<T>::kPerVec == 0 && depth % Elem<T>::kPerVec == 0 &&
           static_cast<std::int64_t>(320) * ld * static_cast<std::int64_t>(sizeof(T)) < kMaxSpan;
}

/// The product on the loose kernel's tiles.
template <bool Codes, typename T>
hipError_t launch_loose(const T* a, const T* b, const float* bias, T* c, T* pre, const GatedArgs& args,
                        hipStream_t stream) {
    auto loose = [&](auto tile) -> hipError_t {
        using S = decltype(tile);
        const std::int64_t tiles = (static_cast<std::int64_t>(args.m) + S::kBM - 1) / S::kBM *
                                   ((static_cast<std::int64_t>(args.n) + S::kBO - 1) / S::kBO);
        if (!launchable(tiles, S::kThreads)) {
            return hipErrorInvalidConfiguration;
        }
        return with_gate(args.gate, [&](auto gate) -> hipError_t {
            gated_loose_kernel<T, S, decltype(gate)::value, Codes>
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

} // namespace cuvit::detail::gemm
