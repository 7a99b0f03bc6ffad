// How a call of packed attention is divided: the rules alone, on the host.
#pragma once

#include "packed_places.hpp"

namespace cuvit::detail::packed {

/// How a workgroup's four wavefronts divide their work in the forward: kFew, kMiddle and
/// kLarge (bf16 alone) have all four, pairs or none of them on the same rows; in kParts
/// they are single ones, each with a part of the keys, joined by a second launch
/// (packed_attention.hip).
enum class Kind { kParts, kFew, kMiddle, kLarge };

struct Plan {
    Kind kind;
    int parts;
};

/// Rows of a workgroup's tile, of fp32 (@p single) or bf16. (kFew's are those of kParts,
/// twice as many for heads above 128, and count in no rule.)
constexpr int tile_rows(Kind kind, bool single) {
    return kind == Kind::kLarge ? 128 : kind == Kind::kMiddle ? (single ? 32 : 64) : single ? 16 : 32;
}

/// Keys of a block of a part.
constexpr int kPartKeys = 32;

/// By the call's sizes alone, which know a cache's room but not what is filled of it: into
/// the largest tiles of rows that still give every CU work, and for few rows over long keys
/// into as many parts of them as give the chip eight single wavefronts a CU, of four blocks
/// or more on average. us for
/// kMiddle / kLarge / parts of single queries: 64 over 8192 keys, 12 heads on 4 of 128 240
/// / 280 / 200 (4 parts), 256 over 2048, 32 on 8 389 / 405 / 450, 1024 over 577, 12 of 64
/// 303 / 311 / 470.
///
/// kFew walks a key in about 7.5 ns (heads of 64; fp32 19) and a join takes 2 us and 0.7 ns
/// for each of a row's parts (more in fp32, whose parts wait for MFMAs too): so parts where
/// there are at most 10 of these (20) for each key above 800. us for kFew / parts, bf16: 4 x
/// 577 tokens, 6 heads of 64 10.8 / 49, 1 query over 577 keys 8.8 / 10.7, 64 over 2048
/// 16.9 / 14.9, 256 over 2048 16.9 / 20.8, 577 over 12545 103 / 49; fp32 4 x 64 over 2048 47
/// / 34, 1 x 577 over 2048 36 / 51.
inline Plan choose_forward(const PackedArgs& args, bool single, std::int64_t units) {
    const auto tiles = [&](Kind kind) {
        return slots(args.tokens, args.group, tile_rows(kind, single), args.sequences) * args.kv_heads;
    };
    const std::int64_t lengths = args.kv_tokens / args.sequences; // on average
    const std::int64_t most = lengths / (4 * kPartKeys);
    // Where a sequence's rows fit the smallest tile on average, larger ones are no fewer.
    const bool small = static_cast<std::int64_t>(args.tokens) * args.group <=
                       static_cast<std::int64_t>(args.sequences) * tile_rows(Kind::kParts, single);
    if (!single && !small && tiles(Kind::kLarge) >= 2 * units) {
        return {Kind::kLarge, 1};
    }
    if (tiles(Kind::kMiddle) >= (small && most >= 16 ? 2 : 1) * units) {
        return {Kind::kMiddle, 1};
    }
    const std::int64_t wanted = 8 * units / tiles(Kind::kParts);
    const std::int64_t parts = wanted < most ? wanted : most;
    const bool longer = static_cast<std::int64_t>(args.tokens) * args.heads * parts <= (single ? 20 : 10) * (lengths - 800);
    return parts >= 4 && longer ? Plan{Kind::kParts, static_cast<int>(parts)} : Plan{Kind::kFew, 1};
}

/// Wavefronts that share a tile of rows, or of keys, in the gradients: at most (what the
/// blocks' LDS holds), and at least.
constexpr int most_sharing(int head_dim) { return head_dim <= 128 ? 4 : 2; }
constexpr int least_sharing(bool single) { return single ? 2 : 1; }

/// How many wavefronts share a tile in a gradient's launch over @p tokens times @p times
/// rows: the fewest whose tiles give the CUs two workgroups
/// each (one in fp32), or the most. Where a tile's walk, @p walk rows of the other side
/// on average, is short, splitting it gains less than it costs, and in fp32 pairs
/// of wavefronts share whatever the size (packed_attention.hip). us for 1 / 2 / 4
/// wavefronts to the same keys: 32 x 197 tokens, 3 heads of 64 21.7 / 22.6 / 28.9;
/// 1 x 3136, causal, 12 heads on 4 of 80 385 / 240 / 186, 4 of them of 128 663 /
/// 655 / 686; fp32 4 x 577, 6 heads 104.7 / 95.5 / 103.6.
inline int choose_sharing(const PackedArgs& args, bool single, int tokens, int times, std::int64_t walk,
                          std::int64_t units) {
    const auto enough = [&](int sharing) {
        const int rows = (single ? 16 : 32) * 4 / sharing;
        return slots(tokens, times, rows, args.sequences) * args.kv_heads >= (single ? 1 : 2) * units;
    };
    if (walk < std::int64_t{512} * args.sequences || enough(least_sharing(single))) {
        return least_sharing(single);
    }
    return most_sharing(args.head_dim) > 2 && !enough(2) ? most_sharing(args.head_dim) : 2;
}

/// The same for the launch over rows, which walks the keys, and the one over keys.
inline int choose_query_sharing(const PackedArgs& args, bool single, std::int64_t units) {
    return choose_sharing(args, single, args.tokens, args.group, args.kv_tokens, units);
}
inline int choose_key_sharing(const PackedArgs& args, bool single, std::int64_t units) {
    return choose_sharing(args, single, args.kv_tokens, 1, static_cast<std::int64_t>(args.tokens) * args.group, units);
}

} // namespace cuvit::detail::packed
