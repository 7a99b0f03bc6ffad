// Where packed attention's tiles and workgroups lie (kernels/packed_places.hpp) for
// test_packed_places_cpu.py.
#include "kernels/packed_places.hpp"

#include "binding/reach.hpp"

using namespace cuvit::detail;
using namespace cuvit::detail::packed;

extern "C" {

/// A sequence's span as {first query, queries, first key, keys}.
void packed_span(const std::int32_t* starts, const std::int32_t* kv_starts, const std::int32_t* kv_lengths, int tokens,
                 int kv_tokens, int sequence, std::int32_t* out) {
    PackedArgs args{};
    args.tokens = tokens;
    args.kv_tokens = kv_tokens;
    args.starts = starts;
    args.kv_starts = kv_starts;
    args.kv_lengths = kv_lengths;
    const Span span = span_of(args, sequence);
    out[0] = span.first_query;
    out[1] = span.queries;
    out[2] = span.first_key;
    out[3] = span.keys;
}

int packed_first_slot(const std::int32_t* starts, int sequence, int limit, int times, int rows) {
    return first_slot(starts, sequence, limit, times, rows);
}

std::int64_t packed_slots(int tokens, int times, int rows, int sequences) { return slots(tokens, times, rows, sequences); }

std::int64_t packed_items(std::int64_t slots, int heads) { return items(slots, heads); }

/// {head, slot} of a workgroup.
void packed_item(std::uint32_t block, int slots, int heads, int last_first, std::int32_t* out) {
    const Item item = item_of(block, slots, heads, last_first != 0);
    out[0] = item.head;
    out[1] = item.slot;
}

/// The elements that the native binding lets a launch touch, or -1 where it refuses.
std::int64_t packed_reach(int tokens, int heads, int head_dim, std::int64_t token, std::int64_t head) {
    std::int64_t reach = 0;
    return cuvit::binding::rows_reach(tokens, heads, head_dim, {token, head}, &reach) ? reach : -1;
}

} // extern "C"
