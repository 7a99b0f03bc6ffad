// Where packed attention's sequences, tiles and workgroups lie: whole numbers alone, for
// the kernels and for the host.
#pragma once

#include "launch.hpp"

namespace cuvit::detail::packed {

__host__ __device__ inline int smaller(int a, int b) { return a < b ? a : b; }
__host__ __device__ inline int larger(int a, int b) { return a > b ? a : b; }

/// A sequence's tokens: queries, and keys (as many as are filled).
struct Span {
    int first_query;
    int queries;
    int first_key;
    int keys;
};

/// Starts that do not fit the operands are cut to them, so that no access leaves
/// them whatever the numbers say.
__host__ __device__ inline Span span_of(const PackedArgs& args, int sequence) {
    Span s;
    s.first_query = smaller(larger(args.starts[sequence], 0), args.tokens);
    s.queries = smaller(larger(args.starts[sequence + 1], s.first_query), args.tokens) - s.first_query;
    s.first_key = smaller(larger(args.kv_starts[sequence], 0), args.kv_tokens);
    s.keys = smaller(larger(args.kv_starts[sequence + 1], s.first_key), args.kv_tokens) - s.first_key;
    if (args.kv_lengths != nullptr) {
        s.keys = smaller(larger(args.kv_lengths[sequence], 0), s.keys);
    }
    return s;
}

/// How many of a sequence's @p keys its query @p query sees, @p behind being the keys less
/// the queries (added up otherwise, query + keys may pass 2^31).
__host__ __device__ inline int seen_by(int query, int behind, int keys, bool causal) {
    return causal ? smaller(larger(query + 1 + behind, 0), keys) : keys;
}

/// The keys that part @p part of @p parts takes of the first @p keys, whole blocks of
/// @p block but for the last one. In 64 bits: parts * of_part * block passes keys.
struct Part {
    int first;
    int last;
};

__host__ __device__ inline Part part_of(int keys, int part, int parts, int block) {
    const std::int64_t blocks = (static_cast<std::int64_t>(keys) + block - 1) / block;
    const std::int64_t of_part = (blocks + parts - 1) / parts * block;
    const std::int64_t first = part * of_part;
    const std::int64_t last = first + of_part;
    return {first < keys ? static_cast<int>(first) : keys, last < keys ? static_cast<int>(last) : keys};
}

/// The sequence and tile of slot @p slot, each sequence's rows being cut into tiles
/// of @p rows: sequence s owns the slots from starts[s] * times / rows + s on (which
/// steps past all its tiles before the next one's), so that the grid needs no
/// lengths, and a wavefront finds s by comparing 64 starts at a time. -1: none.
struct Spot {
    int sequence;
    int tile;
};

__host__ __device__ inline int first_slot(const std::int32_t* starts, int sequence, int limit, int times, int rows) {
    const std::int64_t row = static_cast<std::int64_t>(smaller(larger(starts[sequence], 0), limit)) * times;
    return static_cast<int>(static_cast<std::uint32_t>(row) / static_cast<std::uint32_t>(rows)) + sequence;
}

/// Slots that cover tokens * times rows of any sequences.
inline std::int64_t slots(int tokens, int times, int rows, int sequences) {
    return static_cast<std::int64_t>(tokens) * times / rows + sequences;
}

/// Which key head and slot a workgroup takes: all heads of a slot before the next one's.
/// With @p last_first (causal: late rows see more keys) the longest walks start first, so
/// that none is left to run alone (clips of 12545 and 3137 tokens in a head's order 653 us,
/// so 409 then, 433 now).
struct Item {
    int head;
    int slot;
};

__host__ __device__ inline Item item_of(std::uint32_t block, int slots, int heads, bool last_first) {
    const int slot = static_cast<int>(block / static_cast<std::uint32_t>(heads));
    const int head = static_cast<int>(block) - slot * heads;
    if (slot >= slots) {
        return {-1, 0};
    }
    return {head, last_first ? slots - 1 - slot : slot};
}

/// Workgroups that item_of() needs.
inline std::int64_t items(std::int64_t slots, int heads) { return slots * heads; }

} // namespace cuvit::detail::packed
