// Preactivations kept in 8 bits: e4m3 codes (four bits of exponent, three of mantissa,
// up to 448), and for every 32 consecutive columns of a row a power of two, kept as its
// exponent plus 127 (e8m0). The power is the least, from 2^-117 on, that keeps the
// group's largest finite value within 448: multiplying by it and by its inverse is
// exact, so a value meets one rounding, to nearest-even, of 2^-4 of it at most (2^-10 of
// the power below 2^-6 of it). Infinities and NaN are kept as NaN.
#pragma once

#include "attention_common.hpp"
#include "device_common.hpp"
#include "launch.hpp"

namespace cuvit::device {

constexpr int kCodeGroup = 32;
/// The least scale's exponent: with it the smallest code, 2^-9 of it, is still a normal
/// float.
constexpr int kLeastScale = 127 - 117;

/// The largest size of a lane's finite values, 0 without one. (The maximum passes over
/// NaN by itself; only where an infinity is about are values looked at one by one.)
template <int Count> __device__ __forceinline__ float largest_finite(const float (&v)[Count]) {
    float largest = 0.0F;
#pragma unroll
    for (int e = 0; e < Count; ++e) {
        largest = fmaxf(largest, fabsf(v[e]));
    }
    if (__builtin_expect(__any(largest == INFINITY), 0)) {
        largest = 0.0F;
#pragma unroll
        for (int e = 0; e < Count; ++e) {
            largest = fmaxf(largest, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.0F);
        }
    }
    return largest;
}

/// The scale (its exponent plus 127) of a group whose largest size is @p largest:
/// 448 = 1.75 * 2^8.
__device__ __forceinline__ std::uint32_t code_scale(float largest) {
    const std::uint32_t bits = __float_as_uint(largest);
    const int exponent = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFFU) > 0x600000U ? 1 : 0);
    return static_cast<std::uint32_t>(max(exponent, kLeastScale));
}

__device__ __forceinline__ float code_inverse(std::uint32_t scale) { return __uint_as_float((254U - scale) << 23); }
__device__ __forceinline__ float code_factor(std::uint32_t scale) { return __uint_as_float(scale << 23); }

/// Four values times @p inverse as codes, the first in the low byte.
__device__ __forceinline__ std::uint32_t four_codes(float a, float b, float c, float d, float inverse) {
    int word = __builtin_amdgcn_cvt_pk_fp8_f32(a * inverse, b * inverse, 0, false);
    word = __builtin_amdgcn_cvt_pk_fp8_f32(c * inverse, d * inverse, word, true);
    return static_cast<std::uint32_t>(word);
}

/// The four values of a word of codes, before their scale.
__device__ __forceinline__ void code_values(std::uint32_t word, float (&v)[4]) {
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), false);
    const auto high = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), true);
    v[0] = low[0];
    v[1] = low[1];
    v[2] = high[0];
    v[3] = high[1];
}

template <int Words> struct Bytes {
    std::uint32_t w[Words];
};

/// Four bytes a word to any address, or the first @p count of them; whole ones with
/// @p Streaming past the caches.
template <int Words, bool Streaming = false>
__device__ __forceinline__ void store_bytes(std::uint8_t* to, const Bytes<Words>& bytes, int count) {
    typedef std::uint32_t words __attribute__((ext_vector_type(Words)));
    typedef words loose __attribute__((aligned(1)));
    if (count >= 4 * Words) {
        if constexpr (Streaming) {
            __builtin_nontemporal_store(__builtin_bit_cast(words, bytes), reinterpret_cast<loose*>(to));
        } else {
            *reinterpret_cast<loose*>(to) = __builtin_bit_cast(words, bytes);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4 * Words; ++i) {
            if (i < count) {
                to[i] = static_cast<std::uint8_t>(bytes.w[i / 4] >> (8 * (i % 4)));
            }
        }
    }
}

/// The same the other way; bytes that are not there are 0.
template <int Words> __device__ __forceinline__ Bytes<Words> load_bytes(const std::uint8_t* from, int count) {
    typedef std::uint32_t words __attribute__((ext_vector_type(Words)));
    typedef words loose __attribute__((aligned(1)));
    Bytes<Words> bytes;
    if (count >= 4 * Words) {
        bytes = __builtin_bit_cast(Bytes<Words>, static_cast<words>(*reinterpret_cast<const loose*>(from)));
    } else {
#pragma unroll
        for (int w = 0; w < Words; ++w) {
            bytes.w[w] = 0;
        }
#pragma unroll
        for (int i = 0; i < 4 * Words; ++i) {
            if (i < count) {
                bytes.w[i / 4] |= static_cast<std::uint32_t>(from[i]) << (8 * (i % 4));
            }
        }
    }
    return bytes;
}

} // namespace cuvit::device
