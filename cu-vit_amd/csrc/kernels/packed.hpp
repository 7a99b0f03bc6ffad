// What the packed attention kernels share: where a workgroup's rows lie, operand
// tiles in LDS and the fragments read from them, fp32 and bf16 alike.
//
// Rows. The query heads of a group see the same keys, so a sequence's rows are its
// queries times the group's heads, row r being query r / group of head r % group:
// keys and values are read once for all of them, and single queries fill a tile.
//
// Tiles in LDS are rows of kPitch bytes, a power of two, brought by direct-to-LDS
// loads (16 bytes a lane). They are read in two ways: 16-byte pieces of a row, a row a
// lane (a product over head_dim), and across rows (a product over rows), in bf16 by
// the transposing LDS load, four rows of 16 values to 16 lanes, in fp32 value by
// value. Pieces are placed so that neither way meets a bank twice in a cycle: piece c
// of row r in slot c ^ turned(r). In bf16 the four rows of a transposing load take the
// upper bits of the placement, since it reads two pieces of each row for 16 lanes and
// the two next for the other 16; in fp32 rows 4 g + e, one e at a time, do.
#pragma once

#include "attention_common.hpp"
#include "gemm_dma.hpp"
#include "packed_places.hpp"

namespace cuvit::detail::packed {

using namespace cuvit::device;
using attention::combine_rows;
using attention::Lds4x16;
using gemm::bf16x8;
using gemm::kOutside;
using gemm::load_to_lds;
using gemm::lds_address;
using gemm::Mma;
using gemm::scalar_resource;
using gemm::sgpr4;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr float kLog2e = 1.44269504088896341F;
constexpr float kLn2 = 0.69314718055994531F;

__device__ __forceinline__ Spot find(const std::int32_t* starts, int sequences, int limit, int times, int rows,
                                     int slot) {
    int low = 0;
    int count = sequences;
    while (count > 1) {
        const int step = (count + kWave - 1) / kWave;
        const int probe = low + lane_id() * step;
        const bool before = probe < low + count && first_slot(starts, probe, limit, times, rows) <= slot;
        const std::uint64_t those = __ballot(before);
        if (those == 0) {
            return {-1, 0};
        }
        const int last = 63 - __builtin_clzll(those);
        const int at = low + last * step;
        count = step == 1 ? 1 : min(step, low + count - at);
        low = at;
    }
    low = __builtin_amdgcn_readfirstlane(low);
    const int tile = __builtin_amdgcn_readfirstlane(slot - first_slot(starts, low, limit, times, rows));
    return tile >= 0 ? Spot{low, tile} : Spot{-1, 0};
}

/// Tiles of rows of up to D values of type T in LDS.
template <typename T, int D> struct Rows {
    static constexpr int kE = Mma<T>::kEdge;
    static constexpr int kV = Elem<T>::kPerVec;
    static constexpr int kGroups = kWave / kE;      // lanes that share a row of a fragment
    static constexpr int kBlocks = D / 16;          // 16 values of k in a fragment of either type
    static constexpr int kTiles = (D + kE - 1) / kE;
    static_assert(D % 16 == 0 && D <= 256 && kBlocks * 16 == D, "whole fragments");
    static constexpr int kBytes = D * static_cast<int>(sizeof(T));
    static constexpr int kLeast = sizeof(T) == 2 ? 128 : 256;
    static constexpr int kPitch = kBytes <= kLeast ? kLeast : kBytes <= 256 ? 256 : kBytes <= 512 ? 512 : 1024;
    static constexpr int kSlots = kPitch / 16;

    /// Its piece's slot is a piece's number ^ turned(row).
    __device__ __forceinline__ static int turned(int row) {
        if constexpr (sizeof(T) == 4) {
            return row & 15;
        } else if constexpr (kSlots == 8) { // two rows to a turn of the banks
            return ((row >> 1 & 1) << 2) | (row >> 2 & 3);
        } else {
            return ((row & 3) << 2) | (row >> 2 & 3);
        }
    }

    /// The 16 bytes of k-block @p block of the lane's row @p row (of the tile).
    __device__ __forceinline__ static Vec16 along(const unsigned char* tile, int row, int block, int lane) {
        const int piece = block * kGroups + lane / kE;
        return load16(tile + row * kPitch + ((piece ^ turned(row)) << 4));
    }

    /// The fragment across rows: values of dim d0 + lane % E, d0 = E * @p dims, of the
    /// rows from @p row0 on (a multiple of 16; 16 of them) in the order in which an
    /// accumulator's rows lie in a lane (fp32: 4 g + 0..3; bf16: 4 h + 0..3 and 8 + 4 h
    /// + 0..3), so that weights go from one product to the next in their registers.
    __device__ __forceinline__ static Vec16 across(const unsigned char* tile, int row0, int dims, int lane) {
        Vec16 fragment;
        if constexpr (sizeof(T) == 4) {
            const int dim = dims * kE + lane % kE;
            const int piece = dim / kV;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = row0 + 4 * (lane / kE) + e;
                fragment.w[e] = *reinterpret_cast<const std::uint32_t*>(tile + row * kPitch +
                                                                        ((piece ^ turned(row)) << 4) + dim % kV * 4);
            }
        } else {
            const int j = lane & 15;
            const int piece = dims * 4 + 2 * (lane >> 4 & 1) + (j >> 1 & 1);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int row = row0 + 8 * s + 4 * (lane >> 5) + (j >> 2);
                const unsigned char* const at =
                    tile + row * kPitch + ((piece ^ turned(row)) << 4) + (j & 1) * 8;
                const auto part = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4x16*)(at));
                const uint2 words = __builtin_bit_cast(uint2, part);
                fragment.w[2 * s] = words.x;
                fragment.w[2 * s + 1] = words.y;
            }
        }
        return fragment;
    }
};

/// Rows of a block, so that two operands of it, two buffers each, take 32 or 64 KB.
template <typename T, int D> constexpr int kBlockRows = Rows<T, D>::kPitch <= 256 ? 64 : 16384 / Rows<T, D>::kPitch;

/// Rows of E of an accumulator that across() takes at a time, as an operand: fp32
/// all 16, bf16 rows 16 @p part of 32.
template <typename T>
__device__ __forceinline__ Vec16 weights_of(const typename Mma<T>::Acc& acc, int part) {
    Vec16 v;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if constexpr (sizeof(T) == 4) {
            v.w[w] = __float_as_uint(acc[w]);
        } else {
            v.w[w] = pack_bf16x2(acc[8 * part + 2 * w], acc[8 * part + 2 * w + 1]);
        }
    }
    return v;
}
template <typename T> constexpr int kParts = Mma<T>::kEdge / 16;
template <typename T> constexpr int kRegisters = Mma<T>::kEdge * Mma<T>::kEdge / kWave;

/// The row (of E) that register @p i of an accumulator holds in a lane.
template <typename T> __device__ __forceinline__ int row_of(int lane, int i) {
    return Mma<T>::column(lane, i / 4) + i % 4;
}

/// Reduces over the lanes that share a column of an accumulator.
template <typename T, typename Op> __device__ __forceinline__ float combine_column(float value, Op op) {
    if constexpr (sizeof(T) == 4) {
        value = combine_rows<16>(value, op);
    }
    return combine_rows<32>(value, op);
}

/// Loads of @p Count consecutive rows (a token's stride apart) of one head into a
/// tile, by all @p Waves wavefronts of the workgroup, 1024 bytes a load. Rows past the
/// last and values past head_dim read as zeros.
template <typename T, int D, int Count, int Waves = kWaves> struct Stage {
    using R = Rows<T, D>;
    static constexpr int kBytes = Count * R::kPitch;
    static constexpr int kRowsOfPiece = 1024 / R::kPitch;
    static constexpr int kLoads = kBytes / 1024 / Waves;
    static_assert(kBytes % (1024 * Waves) == 0, "whole pieces for every wavefront");

    const T* base; // of the head, at the sequence's first row
    std::int64_t token;
    int head_dim;
    unsigned int offset[kLoads]; // of the lane's piece in each load, kOutside where it is behind head_dim

    __device__ __forceinline__ Stage(const T* base_, std::int64_t token_, int head_dim_, int wave, int lane)
        : base(base_), token(token_), head_dim(head_dim_) {
#pragma unroll
        for (int p = 0; p < kLoads; ++p) {
            const int row = (p * Waves + wave) * kRowsOfPiece + lane / R::kSlots;
            const int piece = lane % R::kSlots ^ R::turned(row);
            offset[p] = piece * R::kV < head_dim
                            ? static_cast<unsigned int>(row * static_cast<int>(token) * static_cast<int>(sizeof(T)) + piece * 16)
                            : kOutside;
        }
    }

    /// Rows @p first .. + Count, of which @p left are there, into LDS at @p lds.
    __device__ __forceinline__ void issue(int first, int left, unsigned int lds, int wave) const {
        const int rows = min(left, Count);
        const sgpr4 resource =
            scalar_resource(base + first * token, static_cast<unsigned int>(((rows - 1) * static_cast<int>(token) + head_dim) *
                                                                          static_cast<int>(sizeof(T))));
#pragma unroll
        for (int p = 0; p < kLoads; ++p) {
            load_to_lds(lds + static_cast<unsigned int>((p * Waves + wave) * 1024), offset[p], resource);
        }
    }
};

/// This wavefront's loads have landed, then the workgroup's.
__device__ __forceinline__ void landed() {
    __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0), as an instruction that the compiler knows
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

/// A wavefront's own rows as fragments along head_dim, straight from memory; zeros
/// where @p from is null and past head_dim.
template <typename T, int D>
__device__ __forceinline__ void load_rows(const T* from, int head_dim, int lane,
                                          Vec16 (&fragments)[Rows<T, D>::kBlocks]) {
    using R = Rows<T, D>;
#pragma unroll
    for (int b = 0; b < R::kBlocks; ++b) {
        const int dim = (b * R::kGroups + lane / R::kE) * R::kV;
        fragments[b] = from != nullptr && dim < head_dim ? load16(from + dim) : Vec16{{0, 0, 0, 0}};
    }
}

/// Four consecutive values of a row, rounded.
template <typename T> __device__ __forceinline__ void store_four(T* to, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(to) = make_float4(a, b, c, d);
    } else {
        *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
    }
}

/// A lane's row of accumulators (dims in registers), times @p factor.
template <typename T, int D>
__device__ __forceinline__ void store_row(T* to, const typename Mma<T>::Acc (&acc)[Rows<T, D>::kTiles], float factor,
                                          int head_dim, int lane) {
    using R = Rows<T, D>;
#pragma unroll
    for (int t = 0; t < R::kTiles; ++t) {
#pragma unroll
        for (int run = 0; run < Mma<T>::kRuns; ++run) {
            const int dim = t * R::kE + Mma<T>::column(lane, run);
            if (dim < head_dim) {
                store_four<T>(to + dim, acc[t][4 * run] * factor, acc[t][4 * run + 1] * factor,
                              acc[t][4 * run + 2] * factor, acc[t][4 * run + 3] * factor);
            }
        }
    }
}

/// @p run with the smallest D that holds @p head_dim.
template <typename Run> hipError_t with_width(int head_dim, Run&& run) {
    if (head_dim <= 32) {
        return run(std::integral_constant<int, 32>{});
    }
    if (head_dim <= 64) {
        return run(std::integral_constant<int, 64>{});
    }
    if (head_dim <= 96) {
        return run(std::integral_constant<int, 96>{});
    }
    if (head_dim <= 128) {
        return run(std::integral_constant<int, 128>{});
    }
    return run(std::integral_constant<int, 256>{});
}

} // namespace cuvit::detail::packed
