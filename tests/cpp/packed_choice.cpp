// How packed attention is divided (kernels/packed_choice.hpp), and which keys its parts
// and queries take (kernels/packed_places.hpp), for test_packed_choice_cpu.py.
#include "kernels/packed_choice.hpp"

using namespace cuvit::detail;
using namespace cuvit::detail::packed;

namespace {

PackedArgs problem(const std::int32_t* sizes) {
    PackedArgs args{};
    args.sequences = sizes[0];
    args.tokens = sizes[1];
    args.kv_tokens = sizes[2];
    args.heads = sizes[3];
    args.kv_heads = sizes[4];
    args.group = sizes[3] / sizes[4];
    args.head_dim = sizes[5];
    return args;
}

} // namespace

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

/// A Kind's number, and the parts; sizes are {sequences, tokens, kv_tokens, heads, kv_heads,
/// head_dim}.
int packed_forward_choice(const std::int32_t* sizes, int single, int units, std::int32_t* parts) {
    const Plan plan = choose_forward(problem(sizes), single != 0, units);
    *parts = plan.parts;
    return static_cast<int>(plan.kind);
}

/// Wavefronts to a tile of rows, and of keys.
int packed_query_sharing(const std::int32_t* sizes, int single, int units) {
    return choose_query_sharing(problem(sizes), single != 0, units);
}
int packed_key_sharing(const std::int32_t* sizes, int single, int units) {
    return choose_key_sharing(problem(sizes), single != 0, units);
}

} // extern "C"
