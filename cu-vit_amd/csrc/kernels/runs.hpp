// Runs of consecutive values between memory and registers, fp32 or bf16: whole,
// at the alignment of the run or of a value, or cut short by the end of a row.
#pragma once

#include "device_common.hpp"

namespace cuvit::device {

/// One run of @p U values of a type as they lie in memory.
template <typename T, int U> struct Run {
    static constexpr int kWords = U * static_cast<int>(sizeof(T)) / 4;
    std::uint32_t w[kWords];
};

template <typename T, int U> __device__ __forceinline__ Run<T, U> load_run(const T* from) {
    Run<T, U> run;
    if constexpr (Run<T, U>::kWords == 4) {
        const Vec16 v = load16(from);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            run.w[i] = v.w[i];
    } else {
        static_assert(Run<T, U>::kWords == 2, "runs of 16 or 8 bytes");
        const uint2 v = *reinterpret_cast<const uint2*>(from);
        run.w[0] = v.x;
        run.w[1] = v.y;
    }
    return run;
}

/// With Streaming non-temporal (store16_streaming says what that gives). (A choice
/// at run time loses it: the compiler makes one plain store of both.)
template <typename T, int U, bool Streaming> __device__ __forceinline__ void store_run(T* to, const Run<T, U>& run) {
    typedef std::uint32_t words __attribute__((ext_vector_type(Run<T, U>::kWords)));
    const words v = __builtin_bit_cast(words, run);
    if constexpr (Streaming) {
        __builtin_nontemporal_store(v, reinterpret_cast<words*>(to));
    } else {
        *reinterpret_cast<words*>(to) = v;
    }
}

/// The same at any value's address: one access too, on gfx950, if a slower one
/// where it crosses a cache line.
template <typename T, int U> __device__ __forceinline__ Run<T, U> load_run_unaligned(const T* from) {
    typedef std::uint32_t words __attribute__((ext_vector_type(Run<T, U>::kWords)));
    typedef words loose __attribute__((aligned(sizeof(T))));
    using RunType = Run<T, U>;
    return __builtin_bit_cast(RunType, static_cast<words>(*reinterpret_cast<const loose*>(from)));
}

template <typename T, int U, bool Streaming = false>
__device__ __forceinline__ void store_run_unaligned(T* to, const Run<T, U>& run) {
    typedef std::uint32_t words __attribute__((ext_vector_type(Run<T, U>::kWords)));
    typedef words loose __attribute__((aligned(sizeof(T))));
    if constexpr (Streaming) {
        __builtin_nontemporal_store(__builtin_bit_cast(words, run), reinterpret_cast<loose*>(to));
    } else {
        *reinterpret_cast<loose*>(to) = __builtin_bit_cast(words, run);
    }
}

/// The first @p count values of a run, one by one; the others are 0.
template <typename T, int U> __device__ __forceinline__ Run<T, U> load_some(const T* from, int count) {
    Run<T, U> run;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < U; ++i)
            run.w[i] = i < count ? __float_as_uint(from[i]) : 0U;
    } else {
#pragma unroll
        for (int i = 0; i < U; i += 2) {
            const std::uint32_t low = i < count ? from[i] : 0U;
            const std::uint32_t high = i + 1 < count ? from[i + 1] : 0U;
            run.w[i / 2] = low | (high << 16);
        }
    }
    return run;
}

/// The first @p count values of a run, the others 0 whatever they hold.
template <typename T, int U> __device__ __forceinline__ Run<T, U> keep_some(Run<T, U> run, int count) {
    constexpr int kPerWord = 4 / static_cast<int>(sizeof(T));
#pragma unroll
    for (int i = 0; i < Run<T, U>::kWords; ++i) {
        const int kept = count - kPerWord * i; // of this word
        const std::uint32_t part = kPerWord == 2 && kept == 1 ? 0xFFFFU : 0U;
        run.w[i] &= kept >= kPerWord ? 0xFFFFFFFFU : part;
    }
    return run;
}

template <typename T, int U>
__device__ __forceinline__ void store_some(T* to, const Run<T, U>& run, int count) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
        if (i < count) {
            if constexpr (sizeof(T) == 4) {
                to[i] = __uint_as_float(run.w[i]);
            } else {
                to[i] = static_cast<std::uint16_t>(run.w[i / 2] >> (16 * (i & 1)));
            }
        }
    }
}

template <typename T, int U> __device__ __forceinline__ void widen(const Run<T, U>& run, float (&v)[U]) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(run.w[i]);
        } else {
            v[i] = __uint_as_float((i & 1) != 0 ? run.w[i / 2] & 0xFFFF0000U : run.w[i / 2] << 16);
        }
    }
}

template <typename T, int U> __device__ __forceinline__ Run<T, U> round_run(const float (&v)[U]) {
    Run<T, U> run;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < U; ++i)
            run.w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < U; i += 2)
            run.w[i / 2] = pack_bf16x2(v[i], v[i + 1]);
    }
    return run;
}

} // namespace cuvit::device
