// The gradient of activation(gate) * value with respect to both, from the kept
// preactivations z = [gate, value] and the product's gradient dc:
//   dgate = dc value activation'(gate),  dvalue = dc activation(gate).
//
// Bound: HBM, five values moved for each of C's. A thread takes one 16-byte run
// of each operand; rows need not start at a multiple of it, and the last run of a
// row may be short.
#include "gate.hpp"
#include "launch.hpp"
#include "runs.hpp"

#include <type_traits>

namespace cuvit::detail {
namespace {

using namespace cuvit::device;

constexpr int kThreads = 256;

template <typename T, Gate G, bool Streaming>
__global__ __launch_bounds__(kThreads) void gated_backward_kernel(const T* pre, const T* grad, T* grad_pre,
                                                                  GatedArgs args, std::int64_t total, int runs_of_row) {
    constexpr int U = Elem<T>::kPerVec;
    const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * kThreads;
    for (std::int64_t at = static_cast<std::int64_t>(blockIdx.x) * kThreads + threadIdx.x; at < total; at += step) {
        // (A 32-bit division where it does: the 64-bit one is the longer part of the kernel.)
        const std::int64_t row =
            total <= 0x7FFFFFFF ? static_cast<std::int64_t>(static_cast<std::uint32_t>(at) / static_cast<std::uint32_t>(runs_of_row))
                                : at / runs_of_row;
        const int column = static_cast<int>(at - row * runs_of_row) * U;
        const int count = min(args.n - column, U);
        const T* const z = pre + row * args.ld_pre + column;
        const T* const g = grad + row * args.ldc + column;
        T* const to = grad_pre + row * args.ld_pre + column;
        Run<T, U> gate_run, value_run, grad_run;
        if (count == U) {
            gate_run = load_run_unaligned<T, U>(z);
            value_run = load_run_unaligned<T, U>(z + args.n);
            grad_run = load_run_unaligned<T, U>(g);
        } else {
            gate_run = load_some<T, U>(z, count);
            value_run = load_some<T, U>(z + args.n, count);
            grad_run = load_some<T, U>(g, count);
        }
        float gate[U], value[U], d[U];
        widen<T, U>(gate_run, gate);
        widen<T, U>(value_run, value);
        widen<T, U>(grad_run, d);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            float slope;
            const float activation = gate_value<G, sizeof(T) == 4>(gate[i], slope);
            gate[i] = d[i] * value[i] * slope;
            value[i] = d[i] * activation;
        }
        if (count == U) {
            store_run_unaligned<T, U, Streaming>(to, round_run<T, U>(gate));
            store_run_unaligned<T, U, Streaming>(to + args.n, round_run<T, U>(value));
        } else {
            store_some<T, U>(to, round_run<T, U>(gate), count);
            store_some<T, U>(to + args.n, round_run<T, U>(value), count);
        }
    }
}

template <typename T>
hipError_t launch(const T* pre, const T* grad, T* grad_pre, const GatedArgs& args, hipStream_t stream) {
    constexpr int U = Elem<T>::kPerVec;
    const int runs = static_cast<int>((static_cast<std::int64_t>(args.n) + U - 1) / U);
    const std::int64_t total = static_cast<std::int64_t>(args.m) * runs;
    const unsigned int grid = stride_grid(total, kThreads, 64);
    // More than half of what the L2s hold goes past them (25.8 MB of gradients 11.2
    // -> 10.7 us; 1.1 MB 2.9 and 3.2).
    const bool streaming = static_cast<std::int64_t>(args.m) * 2 * args.n * static_cast<std::int64_t>(sizeof(T)) >
                           (std::int64_t{16} << 20);
    auto run = [&](auto gate) -> hipError_t {
        constexpr Gate kGate = decltype(gate)::value;
        if (streaming) {
            gated_backward_kernel<T, kGate, true><<<grid, kThreads, 0, stream>>>(pre, grad, grad_pre, args, total, runs);
        } else {
            gated_backward_kernel<T, kGate, false><<<grid, kThreads, 0, stream>>>(pre, grad, grad_pre, args, total, runs);
        }
        return hipGetLastError();
    };
    switch (args.gate) {
    case Gate::kSilu: return run(std::integral_constant<Gate, Gate::kSilu>{});
    case Gate::kGelu: return run(std::integral_constant<Gate, Gate::kGelu>{});
    default: return run(std::integral_constant<Gate, Gate::kGeluTanh>{});
    }
}

} // namespace

hipError_t gated_backward(const float* preactivations, const float* grad, float* grad_preactivations,
                          const GatedArgs& args, hipStream_t stream) {
    return launch(preactivations, grad, grad_preactivations, args, stream);
}

hipError_t gated_backward(const std::uint16_t* preactivations, const std::uint16_t* grad,
                          std::uint16_t* grad_preactivations, const GatedArgs& args, hipStream_t stream) {
    return launch(preactivations, grad, grad_preactivations, args, stream);
}

} // namespace cuvit::detail
