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
#include "gated_launch.hpp"

#include <type_traits>

namespace cuvit::detail {
namespace gemm {
namespace {

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
    if (whole_chunks && args.n < kRingColumns) {
        return launch_tile<false>(a, b, bias, c, pre, args, stream);
    }
    return launch_loose<false>(a, b, bias, c, pre, args, stream);
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
