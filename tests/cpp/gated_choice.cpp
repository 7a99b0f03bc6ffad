// The gated product's tile rules (gated_choice.hpp) for test_gated_choice_cpu.py.
#include "kernels/gated_choice.hpp"

using namespace cuvit::detail;

namespace {

GatedArgs problem(int m, int n, int k) {
    GatedArgs args{};
    args.m = m;
    args.n = n;
    args.k = k;
    return args;
}

} // namespace

extern "C" {

/// A GatedTile's number; *px is its XCD split's.
int gated_bf16_choice(int m, int n, int k, int units, int* px) {
    const GatedChoice choice = choose_gated(problem(m, n, k), units);
    *px = choice.map.px;
    return static_cast<int>(choice.tile);
}

/// A GatedTileF32's number.
int gated_f32_choice(int m, int n, int k, int units) {
    return static_cast<int>(choose_gated_f32(problem(m, n, k), units));
}

} // extern "C"
