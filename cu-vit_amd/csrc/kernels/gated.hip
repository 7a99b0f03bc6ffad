// The gated product: C = activation(gate) * value, [gate, value] = A.B^T + bias,
// B [2 n, k] with the gate's n rows before the value's.
//
// A workgroup's tile takes the same columns of both halves, and a wavefront the
// gate's and the value's MFMA tiles of the same outputs, so that both factors of
// an output are the same register of two accumulators: the epilogue multiplies
// them where they lie, and the [m, 2 n] preactivations never leave the chip
// unless they are asked for.
//
// gated_tile_kernel: any sizes, strides and alignment. Four wavefronts own 64 rows
// x 64 outputs; operands go through registers into LDS, a stage of 128 bytes of k
// ahead, at any value's address. MFMAs, fragments and the placement in LDS are the
// GEMMs' (gemm_kernel.hpp, gemm_ring.hpp).
#include "gate.hpp"
#include "gemm_choice.hpp"
#include "gemm_ring.hpp"
#include "runs.hpp"

#include <type_traits>

namespace cuvit::detail {
namespace gemm {
namespace {

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
__device__ __forceinline__ void finish_quad(const float (&gate_sum)[4], const float (&value_sum)[4],
                                            const float (&gate_bias)[4], const float (&value_bias)[4], int row, int col,
                                            T* c, T* pre, const GatedArgs& args) {
    if (row >= args.m || col >= args.n) {
        return;
    }
    const int count = args.n - col;
    float gate[4], value[4], out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        gate[e] = gate_sum[e] + gate_bias[e];
        value[e] = value_sum[e] + value_bias[e];
        out[e] = gate_value<G>(gate[e]) * value[e];
    }
    store_quad(c + static_cast<std::int64_t>(row) * args.ldc + col, out, count);
    if (pre != nullptr) {
        T* const to = pre + static_cast<std::int64_t>(row) * args.ld_pre + col;
        store_quad(to, gate, count);
        store_quad(to + args.n, value, count);
    }
}

/// The bias of four columns of each half, 0 without one and past the last.
__device__ __forceinline__ void read_bias(const float* bias, int col, int n, float (&gate)[4], float (&value)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool given = bias != nullptr && col + e < n;
        gate[e] = given ? bias[col + e] : 0.0F;
        value[e] = given ? bias[n + col + e] : 0.0F;
    }
}

template <typename T> struct GatedTile {
    static constexpr int kE = Mma<T>::kEdge;
    static constexpr int kThreads = 256;
    static constexpr int kBM = 64;
    static constexpr int kBO = 64;           // outputs
    static constexpr int kTM = kBM / 2 / kE; // a wavefront's MFMA tiles of rows
    static constexpr int kTO = kBO / 2 / kE; // and of outputs
    static constexpr int kV = Elem<T>::kPerVec;
    static constexpr int kBK = 8 * kV;
    static constexpr int kRows = kBM + 2 * kBO; // of a stage: A's, then the gate's and the value's tiles in turn
    static constexpr int kChunks = kRows * 8 / kThreads; // 16-byte chunks a thread loads
};

template <typename T, Gate G>
__global__ __launch_bounds__(256) void gated_tile_kernel(const T* __restrict__ a, const T* __restrict__ b,
                                                         const float* __restrict__ bias, T* c, T* pre,
                                                         GatedArgs args) {
    using S = GatedTile<T>;
    constexpr int E = S::kE;
    __shared__ Vec16 stage[S::kRows * 8];
    const int tiles_n = (args.n + S::kBO - 1) / S::kBO;
    const int row0 = static_cast<int>(blockIdx.x / static_cast<unsigned int>(tiles_n)) * S::kBM;
    const int col0 = static_cast<int>(blockIdx.x % static_cast<unsigned int>(tiles_n)) * S::kBO;
    const int thread = static_cast<int>(threadIdx.x);
    const int lane = lane_id();
    const int wave_m = thread / kWave / 2;
    const int wave_n = thread / kWave % 2;

    // The rows this thread loads: chunk thread % 8 of stage rows thread / 8 + 32 p.
    // Rows past the operands' ends repeat the last one: their sums are not stored.
    const int chunk = thread % 8;
    const T* from[S::kChunks];
#pragma unroll
    for (int p = 0; p < S::kChunks; ++p) {
        const int row = thread / 8 + 32 * p;
        if (32 * p < S::kBM) {
            from[p] = a + static_cast<std::int64_t>(min(row0 + row, args.m - 1)) * args.lda;
        } else {
            const int tile = (row - S::kBM) / E; // even: the gate's, odd: the value's
            const int col = min(col0 + tile / 2 * E + (row - S::kBM) % E, args.n - 1);
            from[p] = b + (static_cast<std::int64_t>((tile & 1) != 0 ? args.n : 0) + col) * args.ldb;
        }
        from[p] += chunk * S::kV;
    }
    Run<T, S::kV> held[S::kChunks];
    auto load = [&](int k0) {
        if (k0 + S::kBK <= args.k) {
#pragma unroll
            for (int p = 0; p < S::kChunks; ++p)
                held[p] = load_run_unaligned<T, S::kV>(from[p] + k0);
        } else {
            const int count = min(max(args.k - k0 - chunk * S::kV, 0), S::kV);
#pragma unroll
            for (int p = 0; p < S::kChunks; ++p)
                held[p] = load_some<T, S::kV>(from[p] + k0, count);
        }
    };

    typename Mma<T>::Acc acc[S::kTM][2 * S::kTO];
#pragma unroll
    for (int i = 0; i < S::kTM; ++i)
#pragma unroll
        for (int j = 0; j < 2 * S::kTO; ++j)
#pragma unroll
            for (int r = 0; r < 4 * Mma<T>::kRuns; ++r)
                acc[i][j][r] = 0.0F;
    auto place = [](int row, int slot) { return row * 8 + (slot ^ ((row >> 1) & 7)); };
    if (args.k > 0) {
        load(0);
    }
    for (int k0 = 0; k0 < args.k; k0 += S::kBK) {
        __syncthreads(); // the last stage is read
#pragma unroll
        for (int p = 0; p < S::kChunks; ++p)
            stage[place(thread / 8 + 32 * p, chunk)] = __builtin_bit_cast(Vec16, held[p]);
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
#pragma unroll
    for (int o = 0; o < S::kTO; ++o)
#pragma unroll
        for (int q = 0; q < Mma<T>::kRuns; ++q) {
            const int col = col0 + (wave_n * S::kTO + o) * E + Mma<T>::column(lane, q);
            float gate_bias[4], value_bias[4];
            read_bias(bias, col, args.n, gate_bias, value_bias);
#pragma unroll
            for (int i = 0; i < S::kTM; ++i) {
                float gate[4], value[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    gate[e] = acc[i][2 * o][4 * q + e];
                    value[e] = acc[i][2 * o + 1][4 * q + e];
                }
                finish_quad<T, G>(gate, value, gate_bias, value_bias, row0 + (wave_m * S::kTM + i) * E + lane % E, col,
                                  c, pre, args);
            }
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

template <typename T>
hipError_t launch_gated(const T* a, const T* b, const float* bias, T* c, T* pre, const GatedArgs& args,
                        hipStream_t stream) {
    using S = GatedTile<T>;
    const std::int64_t tiles = (static_cast<std::int64_t>(args.m) + S::kBM - 1) / S::kBM *
                               ((static_cast<std::int64_t>(args.n) + S::kBO - 1) / S::kBO);
    if (tiles > 0x7FFFFFFF) {
        return hipErrorInvalidConfiguration;
    }
    return with_gate(args.gate, [&](auto gate) -> hipError_t {
        gated_tile_kernel<T, decltype(gate)::value>
            <<<static_cast<unsigned int>(tiles), S::kThreads, 0, stream>>>(a, b, bias, c, pre, args);
        return hipGetLastError();
    });
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
