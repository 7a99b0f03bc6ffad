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

/// The elements that the rows of packed attention reach, @p heads heads of @p tokens
/// tokens, or false for strides that no tensor holds.
inline bool rows_reach(std::int64_t tokens, std::int64_t heads, std::int64_t head_dim, const cuvit_token_strides& s,
                       std::int64_t* out) {
    constexpr std::int64_t kLimit = std::int64_t{1} << 40;
    std::int64_t token;
    if (tokens <= 0 || heads <= 0 || head_dim <= 0 || !product(&token, {heads, head_dim})) {
        return false;
    }
    token = s.token != 0 ? s.token : token;
    const std::int64_t head = s.head != 0 ? s.head : head_dim;
    std::int64_t span;
    if (token < 0 || token > kLimit || head < 0 || head > kLimit || !product(&span, {tokens, token + 1}) ||
        span > kLimit || !product(&span, {heads, head + 1}) || span > kLimit) {
        return false;
    }
    *out = (tokens - 1) * token + (heads - 1) * head + head_dim;
    return true;
}

} // namespace cuvit::binding
