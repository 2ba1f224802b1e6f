// Packed sequences of rows, and what attention kernels share: sums and
// maxima over the lanes that hold one column of a 16x16 product.
#pragma once

#include "common.hpp"

namespace s3dx {

// ---------------------------------------------------------------------------
// Packed sequences
// ---------------------------------------------------------------------------
struct Span {
    int64_t begin;
    int32_t rows;
};
// Rows [begin, begin + rows) of sequence s, cut to [0, total].
__device__ __forceinline__ Span sequence_span(const int32_t *starts, int64_t s, int64_t total) {
    const int64_t lo = min(max(static_cast<int64_t>(starts[s]), INT64_C(0)), total);
    const int64_t hi = min(max(static_cast<int64_t>(starts[s + 1]), lo), total);
    return {lo, static_cast<int32_t>(hi - lo)};
}

// The last sequence that begins at or before `unit`, by the whole wave: 64 beginnings at a
// time, so one trip to memory for up to 64 sequences and two for 4,096.
template <class F>
__device__ __forceinline__ int64_t last_sequence(int64_t sequences, int64_t unit, F &&begin) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, hi = sequences;  // begin(lo) <= unit < begin(hi)
    while (hi - lo > 1) {
        const int64_t step = (hi - lo + 63) >> 6, at = lo + lane * step;
        const bool before = lane == 0 || (at < hi && begin(at) <= unit);
        lo += (__popcll(__builtin_amdgcn_ballot_w64(before)) - 1) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}
// The sequence of a tile, where sequence s begins at tile (starts[s] * mul >> shift) + s: every
// sequence has room for its last, partial tile, and the beginnings rise with s, empty
// sequences or not.
__device__ __forceinline__ int64_t sequence_of_unit(const int32_t *starts, int64_t sequences, int64_t total,
                                                    int64_t mul, int shift, int64_t unit) {
    return last_sequence(sequences, unit, [&](int64_t s) {
        return (min(max(static_cast<int64_t>(starts[s]), INT64_C(0)), total) * mul >> shift) + s;
    });
}
// The sequence that holds row `row`, or -1.
__device__ __forceinline__ int64_t sequence_of_row(const int32_t *starts, int64_t sequences, int64_t row) {
    const int64_t s = last_sequence(sequences, row, [&](int64_t at) { return static_cast<int64_t>(starts[at]); });
    return starts[s] <= row && row < starts[s + 1] ? s : -1;
}

// A unit's sequence, its rows, its entry of another list by sequence, and its first unit.
struct Sequence {
    int64_t s;
    Span rows;
    int32_t entry;
    int64_t first, unit;
};
// Of a launch that gives sequence s its units(rows, entry): the sequence of unit at(all), all being how many there are or may be
// (bound), by the whole wave.  Up to 64 sequences' units follow each other; a lane fetches one's numbers, all in one
// trip to memory.  More sequences begin where a bound says: s at unit (starts[s] * mul >> shift) + apart * s.
template <class Units, class At>
__device__ __forceinline__ Sequence sequence_at(const int32_t *starts, const int32_t *list, int64_t sequences, int64_t total,
                                                int64_t mul, int shift, int apart, int64_t bound, Units units, At at) {
    const auto cut = [&](int32_t at) { return min(max(static_cast<int64_t>(at), INT64_C(0)), total); };
    if (sequences > 64) {
        const auto first = [&](int64_t s) { return (cut(starts[s]) * mul >> shift) + apart * s; };
        const int64_t unit = at(bound), s = last_sequence(sequences, unit, first);
        return {s, sequence_span(starts, s, total), list[s], first(s), unit};
    }
    const int lane = threadIdx.x & 63, mine = min(lane, static_cast<int>(sequences) - 1);
    const int64_t lo = cut(starts[mine]), hi = max(lo, cut(starts[mine + 1]));
    const int32_t entry = list[mine], rows = static_cast<int32_t>(hi - lo);
    int32_t end = units(rows, entry);
    for (int o = 1; o < sequences; o <<= 1) {
        const int32_t before = __shfl_up(end, o, 64);
        end += lane >= o ? before : 0;
    }
    // (the last one takes the units behind all)
    const int64_t unit = at(static_cast<int64_t>(__builtin_amdgcn_readlane(end, static_cast<int>(sequences) - 1)));
    const int s = min(__popcll(__builtin_amdgcn_ballot_w64(lane < sequences && end <= unit)), static_cast<int>(sequences) - 1);
    const int32_t first = s == 0 ? 0 : __builtin_amdgcn_readlane(end, s - 1);
    return {s, {__builtin_amdgcn_readlane(static_cast<int32_t>(lo), s), __builtin_amdgcn_readlane(rows, s)},
            __builtin_amdgcn_readlane(entry, s), first, unit};
}

// ---------------------------------------------------------------------------
// Lanes of a 16x16 product
// ---------------------------------------------------------------------------
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// (A vector's element goes through a variable of its own: a bit cast of the element as it stands
// reads the first one.)
__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }

// Largest over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_over_groups(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float m = fmaxf(as_float(a[0]), as_float(a[1]));
    const uint32_t w = __builtin_bit_cast(uint32_t, m);
    const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(as_float(b[0]), as_float(b[1]));
}

// Sum over the same lanes.
__device__ __forceinline__ float sum_over_groups(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float m = as_float(a[0]) + as_float(a[1]);
    const uint32_t w = __builtin_bit_cast(uint32_t, m);
    const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return as_float(b[0]) + as_float(b[1]);
}

}  // namespace s3dx
