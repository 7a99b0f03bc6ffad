// Which keys the parts and queries of packed attention take (kernels/packed_places.hpp)
// for test_packed_choice_cpu.py.
#include "kernels/packed_places.hpp"

using namespace cuvit::detail;
using namespace cuvit::detail::packed;

extern "C" {

/// {first, last} key of a part.
void packed_part(int keys, int part, int parts, int block, std::int32_t* out) {
    const Part found = part_of(keys, part, parts, block);
    out[0] = found.first;
    out[1] = found.last;
}

int packed_seen(int query, int queries, int keys, int causal) {
    return seen_by(query, keys - queries, keys, causal != 0);
}

} // extern "C"
