// What the rotation's forward and backward kernels share: how a head's values
// fall on lanes, the table of a token's turns, and the sums over a head.
//
// A team of 2^log_team lanes owns a head of D values. A lane holds two runs of
// U values ("first" and "second"), placed so that both values of a pair are in
// the same lane and no value crosses lanes:
//   halves     pairs (i, i + P): the runs at i and P + i; behind the 2 P rotated
//              values the unrotated rest is split in halves the same way
//   adjacent   pairs (2 i, 2 i + 1): any runs of whole pairs; with whole runs
//              (Vector) the halves of the head, else 2 U values in a row
// With Vector every run is one 16- or 8-byte access at a multiple of its size;
// without, whole runs are one at any value's address and the values of a cut one
// are moved one by one (any sizes and alignment).
#pragma once

#include "launch.hpp"
#include "runs.hpp"

namespace cuvit::detail::rotary {

using namespace cuvit::device;

constexpr int kThreads = 256;
constexpr int kMaxHeadDim = 512;

/// Where a lane's runs lie in a head. Of each run `count` values exist (all of
/// them with Vector, or none: a lane past the head, placed at its start).
struct Place {
    int at[2];
    int count[2];
    int pair[2];   // the first pair of a run (halves: of both)
    bool turned;   // halves: the runs are rotated ones
};

template <int U, bool Vector, bool Adjacent>
__device__ __forceinline__ Place place_of(int lane, int head_dim, int pairs) {
    const int half = head_dim / 2;
    Place p;
    if constexpr (Adjacent) {
        p.at[0] = Vector ? lane * U : 2 * lane * U;
        p.at[1] = Vector ? half + lane * U : p.at[0] + U;
        if constexpr (Vector) {
            p.count[0] = p.count[1] = lane * U < half ? U : 0;
        } else {
            p.count[0] = min(max(head_dim - p.at[0], 0), U);
            p.count[1] = min(max(head_dim - p.at[1], 0), U);
        }
        p.pair[0] = p.at[0] / 2;
        p.pair[1] = p.at[1] / 2;
        p.turned = true;
    } else {
        const int rotated = (pairs + U - 1) / U; // lanes with rotated runs
        p.turned = lane < rotated;
        const int index = p.turned ? lane * U : (lane - rotated) * U;
        const int span = p.turned ? pairs : half - pairs;
        p.at[0] = p.turned ? index : 2 * pairs + index;
        p.at[1] = p.at[0] + span;
        p.count[0] = p.count[1] = min(max(span - index, 0), U);
        p.pair[0] = p.pair[1] = index;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        p.at[r] = p.count[r] > 0 ? p.at[r] : 0;
        p.pair[r] = p.count[r] > 0 ? p.pair[r] : 0;
    }
    return p;
}

/// Lanes that a head needs, before rounding up to a power of two.
inline int lanes_of_head(int unit, bool adjacent, int head_dim, int pairs) {
    const int half = head_dim / 2;
    if (adjacent) {
        return (half + unit - 1) / unit;
    }
    return (pairs + unit - 1) / unit + (half - pairs + unit - 1) / unit;
}

/// The sum of a value over a team, the same bits in each of its lanes.
__device__ __forceinline__ float team_sum(float value, int log_team) {
    if (log_team > 0) {
        value += dpp_move<kDppQuadSwap1>(value);
    }
    if (log_team > 1) {
        value += dpp_move<kDppQuadSwap2>(value);
    }
    if (log_team > 2) {
        value += dpp_move<kDppRowHalfMirror>(value);
    }
    if (log_team > 3) {
        value += dpp_move<kDppRowMirror>(value);
    }
    if (log_team > 4) {
        value += __shfl_xor(value, 16, kWave);
    }
    if (log_team > 5) {
        value += __shfl_xor(value, 32, kWave);
    }
    return value;
}

/// cos and sin of position * frequency. The product of two floats is exact in
/// 64 bits; counted in quarter turns its whole part goes there too, so that what
/// is left, at most half a quarter turn, is as good for a position of 10^6 as for
/// 1. Taylor series on [-pi/4, pi/4], cut where the next term is below 2e-9.
__device__ __forceinline__ void turn_of(float position, float frequency, float& c, float& s) {
    const double quarters = static_cast<double>(position) * static_cast<double>(frequency) * 0.63661977236758134308;
    const double whole = rint(quarters);
    const float x = static_cast<float>(quarters - whole) * 1.57079632679489661923F;
    const int quadrant = static_cast<int>(whole - 4.0 * floor(0.25 * whole)); // 0 to 3
    const float xx = x * x;
    float odd = fmaf(xx, 2.7557319e-6F, -1.9841270e-4F);
    odd = fmaf(xx, odd, 8.3333333e-3F);
    odd = fmaf(xx, odd, -1.6666667e-1F);
    const float sine = fmaf(x * xx, odd, x);
    float even = fmaf(xx, -2.7557319e-7F, 2.4801587e-5F);
    even = fmaf(xx, even, -1.3888889e-3F);
    even = fmaf(xx, even, 4.1666667e-2F);
    even = fmaf(xx, even, -0.5F);
    const float cosine = fmaf(xx, even, 1.0F);
    c = (quadrant & 1) != 0 ? sine : cosine;
    s = (quadrant & 1) != 0 ? cosine : sine;
    c = quadrant == 1 || quadrant == 2 ? -c : c;
    s = quadrant >= 2 ? -s : s;
}

/// Floats of a token's row of cosines (and of its row of sines).
__host__ __device__ constexpr int table_pitch(int pairs) { return (pairs + 3) / 4 * 4; }

/// The turns of @p tokens tokens from row @p row0 (of images * tokens) into LDS:
/// token t's cosines at 2 t pitch, its sines a pitch behind them. Computed by the
/// workgroup once for all heads: a turn costs about 45 instructions, several times
/// the rotation itself.
__device__ __forceinline__ void fill_table(float* table, const Rotation& rotation, int row0, int tokens,
                                           int tokens_per_image, float sign) {
    const int pitch = table_pitch(rotation.pairs);
    const int count = tokens * rotation.pairs;
    for (int i = static_cast<int>(threadIdx.x); i < count; i += kThreads) {
        const int t = i / rotation.pairs;
        const int pair = i - t * rotation.pairs;
        const int axis = (rotation.axes > 1 && pair >= rotation.first[0] ? 1 : 0) +
                         (rotation.axes > 2 && pair >= rotation.first[1] ? 1 : 0);
        const int row = row0 + t;
        const int image = row / tokens_per_image;
        const int token = row - image * tokens_per_image;
        const float position = rotation.positions[image * rotation.position_stride +
                                                  static_cast<std::int64_t>(token) * rotation.axes + axis];
        float c, s;
        turn_of(position, rotation.frequencies[pair], c, s);
        table[2 * t * pitch + pair] = c;
        table[(2 * t + 1) * pitch + pair] = sign * s;
    }
}

/// A token's first element: row @p row of images * tokens, images that follow one
/// another like tokens (@p flat) or not.
__device__ __forceinline__ std::int64_t token_offset(const HeadStrides& strides, bool flat, int row, int tokens) {
    if (flat) {
        return row * strides.token;
    }
    const int image = row / tokens;
    return image * strides.image + static_cast<std::int64_t>(row - image * tokens) * strides.token;
}

/// A lane's runs of the head at @p from.
template <typename T, int U, bool Vector>
__device__ __forceinline__ void read_runs(const T* from, const Place& place, Run<T, U> (&runs)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if constexpr (Vector) {
            runs[r] = Run<T, U>{};
            if (place.count[r] > 0) {
                runs[r] = load_run<T, U>(from + place.at[r]);
            }
        } else {
            if (place.count[r] == U) {
                runs[r] = load_run_unaligned<T, U>(from + place.at[r]);
            } else {
                runs[r] = load_some<T, U>(from + place.at[r], place.count[r]);
            }
        }
    }
}

template <typename T, int U, bool Vector, bool Streaming>
__device__ __forceinline__ void write_runs(T* to, const Place& place, const float (&first)[U],
                                           const float (&second)[U]) {
    const Run<T, U> runs[2] = {round_run<T, U>(first), round_run<T, U>(second)};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if constexpr (Vector) {
            if (place.count[r] > 0) {
                store_run<T, U, Streaming>(to + place.at[r], runs[r]);
            }
        } else {
            if (place.count[r] == U) {
                store_run_unaligned<T, U>(to + place.at[r], runs[r]);
            } else {
                store_some<T, U>(to + place.at[r], runs[r], place.count[r]);
            }
        }
    }
}

/// Takes a head's mean from its runs (HeadNorm::kLayer) and returns the factor
/// that makes their root mean square 1.
/// (With whole runs the lanes past the head are kept out of the sums; what they
/// hold is not stored.)
template <HeadNorm Norm, bool Vector, int U>
__device__ __forceinline__ float normalise(float (&first)[U], float (&second)[U], const Place& place, int log_team,
                                           float inverse_dim, float epsilon) {
    const bool past = Vector && place.count[0] == 0;
    if constexpr (Norm == HeadNorm::kLayer) {
        // The mean, and once more of what is left, so that rows far from zero
        // keep their deviations.
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
            float sum = 0.0F;
#pragma unroll
            for (int i = 0; i < U; ++i)
                sum += first[i] + second[i];
            const float mean = team_sum(past ? 0.0F : sum, log_team) * inverse_dim;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                first[i] = Vector || i < place.count[0] ? first[i] - mean : 0.0F;
                second[i] = Vector || i < place.count[1] ? second[i] - mean : 0.0F;
            }
        }
    }
    float squares = 0.0F;
#pragma unroll
    for (int i = 0; i < U; ++i)
        squares = fmaf(first[i], first[i], fmaf(second[i], second[i], squares));
    return __builtin_amdgcn_rsqf(fmaf(team_sum(past ? 0.0F : squares, log_team), inverse_dim, epsilon));
}

/// Copies @p width values of each of @p tokens tokens, from element @p skip of
/// each on; with @p whole in 16-byte pieces.
template <typename T>
__device__ __forceinline__ void copy_tokens(const T* in, T* out, std::int64_t pitch, std::int64_t skip, int width,
                                            int row0, int tokens, bool whole) {
    constexpr int kPerVec = Elem<T>::kPerVec;
    const int pieces = whole ? width / kPerVec : width;
    for (int i = static_cast<int>(threadIdx.x); i < tokens * pieces; i += kThreads) {
        const int t = i / pieces;
        const std::int64_t at = (row0 + t) * pitch + skip;
        if (whole) {
            store16_streaming(out + at + (i - t * pieces) * kPerVec, load16(in + at + (i - t * pieces) * kPerVec));
        } else {
            out[at + i - t * pieces] = in[at + i - t * pieces];
        }
    }
}

/// N floats of LDS from a multiple of N (up to four).
template <int N, bool Vector> __device__ __forceinline__ void read_floats(const float* from, float (&to)[N]) {
    if constexpr (Vector && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(from + i);
            to[i] = v.x;
            to[i + 1] = v.y;
            to[i + 2] = v.z;
            to[i + 3] = v.w;
        }
    } else if constexpr (Vector && N == 2) {
        const float2 v = *reinterpret_cast<const float2*>(from);
        to[0] = v.x;
        to[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            to[i] = from[i];
    }
}

/// The cosines and sines of a lane's pairs: with halves of the pairs of both runs
/// (U of them), with adjacent pairs of the first run's, then the second's.
template <int U> struct Turns {
    float c[U];
    float s[U];
};

/// From a token's row of the table. A cut run reads past the pairs, within the
/// table, which has a run to spare: what lies there is another row's or was never
/// written, and turn_runs keeps it out.
template <int U, bool Vector, bool Adjacent>
__device__ __forceinline__ void read_turns(const float* row, const Place& place, int pairs, Turns<U>& turns) {
    const int pitch = table_pitch(pairs);
    if constexpr (Adjacent) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (place.pair[r] < pairs) {
                float c[U / 2], s[U / 2];
                read_floats<U / 2, Vector>(row + place.pair[r], c);
                read_floats<U / 2, Vector>(row + pitch + place.pair[r], s);
#pragma unroll
                for (int i = 0; i < U / 2; ++i) {
                    turns.c[r * (U / 2) + i] = c[i];
                    turns.s[r * (U / 2) + i] = s[i];
                }
            }
        }
    } else if (place.turned) {
        read_floats<U, Vector>(row + place.pair[0], turns.c);
        read_floats<U, Vector>(row + pitch + place.pair[0], turns.s);
    }
}

/// Turns the pairs of a lane's runs; a value that is not rotated, whatever it
/// holds, stays as it is, and so do the zeros behind a cut run, whose turns are
/// whatever the table holds there (0 times infinity would be NaN in a head's sums).
template <int U, bool Vector, bool Adjacent>
__device__ __forceinline__ void turn_runs(float (&first)[U], float (&second)[U], const Turns<U>& turns,
                                          const Place& place, int pairs) {
    if constexpr (Adjacent) {
        auto turn = [&](float(&v)[U], int r) {
            const int left = pairs - place.pair[r];
            if (left <= 0) {
                return;
            }
#pragma unroll
            for (int i = 0; i < U / 2; ++i) {
                const float c = turns.c[r * (U / 2) + i];
                const float s = turns.s[r * (U / 2) + i];
                const float x = v[2 * i];
                const float y = v[2 * i + 1];
                v[2 * i] = i < left ? fmaf(x, c, -(y * s)) : x;
                v[2 * i + 1] = i < left ? fmaf(y, c, x * s) : y;
            }
        };
        turn(first, 0);
        turn(second, 1);
    } else if (place.turned) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float x = first[i];
            const float y = second[i];
            const bool there = Vector || i < place.count[0];
            first[i] = there ? fmaf(x, turns.c[i], -(y * turns.s[i])) : x;
            second[i] = there ? fmaf(y, turns.c[i], x * turns.s[i]) : y;
        }
    }
}

/// Floats of LDS behind a table of @p tokens tokens: runs at its end read up to
/// a run past a row.
inline std::size_t table_floats(int tokens, int pairs) {
    return pairs == 0 ? 0 : static_cast<std::size_t>(2 * tokens) * table_pitch(pairs) + 8;
}

/// Whether every head's runs of @p unit values start at a multiple of their
/// size, for operands at @p addresses (or'ed) with @p strides (or'ed, elements).
inline bool whole_runs(int unit, std::size_t element, std::uintptr_t addresses, std::int64_t strides, int head_dim,
                       int pairs, bool adjacent) {
    const bool runs = head_dim % (2 * unit) == 0 && (adjacent || pairs % unit == 0);
    return runs && addresses % (unit * element) == 0 && strides % unit == 0;
}

/// The runs of a kernel without Vector: of four, or of eight where those of four
/// would take more lanes than a wavefront has.
inline bool loose_runs_of_four(const HeadArgs& a) {
    return lanes_of_head(4, a.rotation.adjacent, a.head_dim, a.rotation.pairs) <= kWave;
}

/// The least l with 2^l >= @p lanes.
inline int log_team_of(int lanes) {
    int log = 0;
    while ((1 << log) < lanes) {
        ++log;
    }
    return log;
}

} // namespace cuvit::detail::rotary
