// How many elements of an operand a launch touches: what the native binding holds
// a tensor's size against. Whole numbers that do not fit are refused, never wrapped.
#pragma once

#include "cuvit/capi.h"

#include <cstdint>
#include <initializer_list>

namespace cuvit::binding {

/// The product of positive numbers, or false past 2^62.
inline bool product(std::int64_t* out, std::initializer_list<std::int64_t> factors) {
    std::int64_t total = 1;
    for (const std::int64_t f : factors) {
        if (f > (std::int64_t{1} << 62) / total) {
            return false;
        }
        total *= f;
    }
    *out = total;
    return true;
}

/// The elements that heads placed by strides reach, or false for strides that no
/// tensor holds.
inline bool heads_reach(const cuvit_rotary_problem& p, const cuvit_head_strides& s, std::int64_t* out) {
    constexpr std::int64_t kLimit = std::int64_t{1} << 40;
    std::int64_t image, token;
    if (!product(&image, {p.tokens, p.heads, p.head_dim}) || !product(&token, {p.heads, p.head_dim})) {
        return false;
    }
    image = s.image != 0 ? s.image : image;
    token = s.token != 0 ? s.token : token;
    const std::int64_t head = s.head != 0 ? s.head : p.head_dim;
    const std::int64_t strides[3] = {image, token, head};
    const std::int64_t extents[3] = {p.images, p.tokens, p.heads};
    std::int64_t reach = p.head_dim;
    for (int i = 0; i < 3; ++i) {
        std::int64_t span;
        if (strides[i] < 0 || strides[i] > kLimit || !product(&span, {extents[i], strides[i] + 1}) || span > kLimit) {
            return false;
        }
        reach += (extents[i] - 1) * strides[i];
    }
    *out = reach;
    return true;
}

} // namespace cuvit::binding
