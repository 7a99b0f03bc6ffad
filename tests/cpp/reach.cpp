// The native binding's operand sizes (binding/reach.hpp) for test_reach_cpu.py.
#include "binding/reach.hpp"

extern "C" {

/// The elements that a rotary problem's input reaches, or -1 where it is refused.
std::int64_t rotary_input_reach(const cuvit_rotary_problem* problem) {
    std::int64_t reach = 0;
    return cuvit::binding::heads_reach(*problem, problem->input, &reach) ? reach : -1;
}

} // extern "C"
