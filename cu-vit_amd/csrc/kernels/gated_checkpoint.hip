// The gated product that keeps its preactivations in 8 bits (checkpoint.hpp), and the
// gate's gradient from them.
//
// The product is gated.hip's, by the same kernels and tile rules; its epilogue turns the
// sums into codes in registers, where a lane and its neighbours hold a group, instead of
// storing them. The kernels for few rows do not keep codes: their workgroups take eight
// outputs, a quarter of a group.
//
// The gradient, from gate and value as the codes say them and the product's gradient dc:
//   dgate = dc value activation'(gate),  dvalue = dc activation(gate),
// and again the product itself, activation(gate) value, which the gradient of the down
// projection's weight needs, so that the forward need not keep that either.
// Bound: HBM. A thread takes one run of each operand, 16 bytes of the stored type.
#include "gated_launch.hpp"

#include <type_traits>

namespace cuvit::detail {
namespace gemm {
namespace {

template <typename T>
hipError_t launch_keeping(const T* a, const T* b, const float* bias, T* c, const GatedArgs& args, hipStream_t stream) {
    T* const none = nullptr;
    if (ring_operand(a, args.lda, args.k) && ring_operand(b, args.ldb, args.k) && args.n < kRingColumns) {
        return launch_tile<true>(a, b, bias, c, none, args, stream);
    }
    return launch_loose<true>(a, b, bias, c, none, args, stream);
}

} // namespace
} // namespace gemm

namespace {

using namespace cuvit::device;

constexpr int kThreads = 256;

template <typename T, Gate G, bool Streaming>
__global__ __launch_bounds__(kThreads) void gated_restore_kernel(const T* grad, T* grad_pre, T* hidden, GatedArgs args,
                                                                 std::int64_t total, int runs_of_row) {
    constexpr int U = Elem<T>::kPerVec;
    const int groups = (args.n + kCodeGroup - 1) / kCodeGroup;
    const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * kThreads;
    for (std::int64_t at = static_cast<std::int64_t>(blockIdx.x) * kThreads + threadIdx.x; at < total; at += step) {
        // (A 32-bit division where it does: the 64-bit one is the longer part of the kernel.)
        const std::int64_t row =
            total <= 0x7FFFFFFF ? static_cast<std::int64_t>(static_cast<std::uint32_t>(at) / static_cast<std::uint32_t>(runs_of_row))
                                : at / runs_of_row;
        const int column = static_cast<int>(at - row * runs_of_row) * U;
        const int count = min(args.n - column, U);
        const std::uint8_t* const codes = args.codes + row * args.ld_pre + column;
        const std::uint8_t* const scales = args.scales + row * 2 * groups + column / kCodeGroup;
        const T* const g = grad + row * args.ldc + column;
        const Bytes<U / 4> gate_codes = load_bytes<U / 4>(codes, count);
        const Bytes<U / 4> value_codes = load_bytes<U / 4>(codes + args.n, count);
        const float gate_scale = code_factor(scales[0]);
        const float value_scale = code_factor(scales[groups]);
        const Run<T, U> run = count == U ? load_run_unaligned<T, U>(g) : load_some<T, U>(g, count);
        float d[U], first[U], second[U], product[U];
        widen<T, U>(run, d);
#pragma unroll
        for (int w = 0; w < U / 4; ++w) {
            float gate[4], value[4];
            code_values(gate_codes.w[w], gate);
            code_values(value_codes.w[w], value);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * w + e;
                const float z = value[e] * value_scale;
                float slope;
                const float active = gate_value<G, sizeof(T) == 4>(gate[e] * gate_scale, slope);
                first[i] = d[i] * z * slope;
                second[i] = d[i] * active;
                product[i] = active * z;
            }
        }
        T* const to = grad_pre + row * args.ld_pre + column;
        T* const again = hidden + row * args.ldc + column;
        if (count == U) {
            store_run_unaligned<T, U, Streaming>(to, round_run<T, U>(first));
            store_run_unaligned<T, U, Streaming>(to + args.n, round_run<T, U>(second));
            if (hidden != nullptr) {
                store_run_unaligned<T, U, Streaming>(again, round_run<T, U>(product));
            }
        } else {
            store_some<T, U>(to, round_run<T, U>(first), count);
            store_some<T, U>(to + args.n, round_run<T, U>(second), count);
            if (hidden != nullptr) {
                store_some<T, U>(again, round_run<T, U>(product), count);
            }
        }
    }
}

template <typename T>
hipError_t launch(const T* grad, T* grad_pre, T* hidden, const GatedArgs& args, hipStream_t stream) {
    constexpr int U = Elem<T>::kPerVec;
    const int runs = static_cast<int>((static_cast<std::int64_t>(args.n) + U - 1) / U);
    const std::int64_t total = static_cast<std::int64_t>(args.m) * runs;
    const unsigned int grid = stride_grid(total, kThreads, 64);
    // More than half of what the L2s hold goes past them, as the gradient's of kept
    // preactivations does.
    const bool streaming = static_cast<std::int64_t>(args.m) * 2 * args.n * static_cast<std::int64_t>(sizeof(T)) >
                           (std::int64_t{16} << 20);
    return gemm::with_gate(args.gate, [&](auto gate) -> hipError_t {
        constexpr Gate kGate = decltype(gate)::value;
        if (streaming) {
            gated_restore_kernel<T, kGate, true><<<grid, kThreads, 0, stream>>>(grad, grad_pre, hidden, args, total, runs);
        } else {
            gated_restore_kernel<T, kGate, false><<<grid, kThreads, 0, stream>>>(grad, grad_pre, hidden, args, total, runs);
        }
        return hipGetLastError();
    });
}

} // namespace

hipError_t gated_checkpoint_gemm(const float* a, const float* b, const float* bias, float* c, const GatedArgs& args,
                                 hipStream_t stream) {
    return gemm::launch_keeping(a, b, bias, c, args, stream);
}

hipError_t gated_checkpoint_gemm(const std::uint16_t* a, const std::uint16_t* b, const float* bias, std::uint16_t* c,
                                 const GatedArgs& args, hipStream_t stream) {
    return gemm::launch_keeping(a, b, bias, c, args, stream);
}

hipError_t gated_checkpoint_backward(const float* grad, float* grad_preactivations, float* hidden,
                                     const GatedArgs& args, hipStream_t stream) {
    return launch(grad, grad_preactivations, hidden, args, stream);
}

hipError_t gated_checkpoint_backward(const std::uint16_t* grad, std::uint16_t* grad_preactivations,
                                     std::uint16_t* hidden, const GatedArgs& args, hipStream_t stream) {
    return launch(grad, grad_preactivations, hidden, args, stream);
}

} // namespace cuvit::detail
