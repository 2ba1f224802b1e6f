// Attention of new rows over a cache in 8 bits: all keys of a sequence, those up to
// a row's own place, or a window of them and the first ones.
//
// o = sum_j p_j step_v c_vj / sum_j p_j, p_j = exp(scale step_k q.c_kj - m): codes are whole
// numbers of 8 bits, which half precision holds exactly, so the products of both
// kinds run on its matrix units with no rounding of a key or a value; a query is taken in units of a
// power of two that fits its row, as one half-precision number (bfloat16 rows: exact) or
// as two (float32 rows: 22 bits).  Steps are of a whole block and multiply results.
//
// What bounds it: the codes, read once, for few rows; for many the vector
// instructions beside the products: exponentials, and the codes' way to half precision.
#include <cmath>

#include "kv_cache.hpp"

namespace s3dx {
namespace {

struct AttendArgs {
    CacheView cache;
    const void *q;
    void *o;
    float *lse;
    const int32_t *q_starts;
    int64_t total_q, q_stride, o_stride, sequences;
    int32_t heads, group, causal, window, sinks, splits, tile_groups;
    float scale;
    float *part_o;    // [splits][total_q][heads][d], divided by their sums
    float4 *part_ml;  // [splits][total_q][heads]: see sum_of
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;  // keys of a step: half or all of a block

// Weights are 2^(score - base), score in binary orders.  A base stands 2^7 below the largest score when it is set
// and moves once a weight would pass 2^15: half precision keeps its 11 bits of weights down to 2^-21 of the
// largest and some down to 2^-31; a base that follows every maximum would scale the sums at every step.
// Beyond 2^20 a base's own rounding would show in its weights: such rows are computed again, key by key.
constexpr float kUnder = 7.0f, kReach = 15.0f, kFar = 0x1p20f;
// Values count in units of the largest step met, and a smaller one's ratio goes into its codes: down to 2^-24 they
// stay exact in half precision.  Rows that meet steps further apart are computed again, key by key.
constexpr float kLeastRatio = 0x1p-24f;

// A row's sum of weights l relative to base hi + lo.
__device__ __forceinline__ float4 sum_of(float hi, float lo, float l, float unit) { return make_float4(hi, lo, l, unit); }
// Whether base a lies above base b.
__device__ __forceinline__ bool above_of(const float4 &a, const float4 &b) { return a.x > b.x || (a.x == b.x && a.y > b.y); }
__device__ __forceinline__ float weight_of(const float4 &a, const float4 &most) {
    return a.z == 0.0f ? 0.0f : __builtin_amdgcn_exp2f((a.x - most.x) + (a.y - most.y));
}
__device__ __forceinline__ float log_of(float hi, float lo, float l) {
    return l == 0.0f ? neg_inf() : fmaf(hi, kLn2, (lo + __builtin_amdgcn_logf(l)) * kLn2);
}

__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}
__device__ __forceinline__ f32x2 unpack_f16x2(uint32_t u) {
    return __builtin_convertvector(__builtin_bit_cast(f16x2, u), f32x2);
}
// Eight biased codes as half-precision numbers: 1024 + u is a byte in a number's low bits; times `ratio` and less
// 1152 of it.
__device__ __forceinline__ u32x4 codes_f16(uint32_t lo, uint32_t hi) {
    const f16x2 bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    const auto two = [&](uint32_t w, uint32_t sel) __attribute__((always_inline)) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, sel)) + bias);
    };
    return u32x4{two(lo, 0x04010400u), two(lo, 0x04030402u), two(hi, 0x04010400u), two(hi, 0x04030402u)};
}
__device__ __forceinline__ u32x4 codes_f16(uint32_t lo, uint32_t hi, f16x2 ratio, f16x2 bias) {
    const auto two = [&](uint32_t w, uint32_t sel) __attribute__((always_inline)) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(
                                                __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, sel)), ratio, bias));
    };
    return u32x4{two(lo, 0x04010400u), two(lo, 0x04030402u), two(hi, 0x04010400u), two(hi, 0x04030402u)};
}
__device__ __forceinline__ f32x4 product(const u32x4 &a, const u32x4 &b, f32x4 d) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), d, 0, 0, 0);
}

// What a tile of a sequence's rows (query rows times the heads that share a key head) sees, and how its keys are cut into
// steps: those of the first keys that stay visible, then from the window's beginning on.
struct Tile {
    Span qs;
    int64_t s;
    int r0, nrows, keys, lag;            // its first row, the sequence's rows, keys, their difference
    int least, low_all, sinks;           // keys that all rows see: below `least`, and from `low_all` on or below `sinks`
    int steps, sink_steps, skip;
    __device__ __forceinline__ int key_of(int step) const { return (step < sink_steps ? step : step + skip) * kStep; }
    // Whether some row of the tile does not see all keys of the step at key `at`.
    __device__ __forceinline__ bool cut(int at) const { return at + kStep > least || (at < low_all && at + kStep > sinks); }
};
// Keys [from, lim) and those below the tile's sinks: what a row sees.
struct Sight {
    int lim, from;
};
__device__ __forceinline__ Sight sight_of(const AttendArgs &a, const Tile &t, int tok) {
    return {a.causal ? max(0, min(t.keys, tok + t.lag + 1)) : t.keys, a.window ? tok + t.lag - a.window + 1 : 0};
}
// Rows [r0, r0 + rows) of sequence s; rows == 0: none.
__device__ __forceinline__ Tile tile_of(const AttendArgs &a, int64_t tile, int rows, int rows_log2) {
    Tile t = {};
    t.s = sequence_of_unit(a.q_starts, a.sequences, a.total_q, a.group, rows_log2, tile);
    t.qs = sequence_span(a.q_starts, t.s, a.total_q);
    const int64_t first = (tile - ((t.qs.begin * a.group >> rows_log2) + t.s)) << rows_log2;
    t.nrows = t.qs.rows * a.group;  // total_q * heads < 2^31
    if (first < 0 || first >= t.nrows) {
        t.nrows = 0;
        return t;
    }
    t.r0 = static_cast<int>(first);
    t.keys = cached_rows(a.cache, t.s);
    t.lag = t.keys - t.qs.rows;
    const Sight head = sight_of(a, t, t.r0 / a.group), tail = sight_of(a, t, (min(t.r0 + rows, t.nrows) - 1) / a.group);
    t.least = head.lim;
    t.low_all = max(0, tail.from);
    t.sinks = a.sinks;
    const int end = (tail.lim + kStep - 1) / kStep;
    t.sink_steps = min(end, (a.sinks + kStep - 1) / kStep);
    t.skip = max(0, max(0, head.from) / kStep - t.sink_steps);
    t.steps = t.sink_steps + max(0, end - t.sink_steps - t.skip);
    return t;
}

// A lane's queries: of each set of 16 rows that of its column, in units of a power of two, in P half-precision terms.
template <class T, int D, int NS>
struct Queries {
    static constexpr int P = sizeof(T) == 2 ? 1 : 2, QV = D / 32;
    u32x4 f[NS][QV][P];
    float unit[NS];  // binary orders of a score for each unit of its product, before the keys' step
    Sight sight[NS];

    __device__ __forceinline__ void load(const AttendArgs &a, const Tile &t, int r0, int kvh) {
        constexpr bool BF = sizeof(T) == 2;
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const int r = min(r0 + 16 * n + c, t.nrows - 1), tok = r / a.group;
            sight[n] = sight_of(a, t, tok);
            const T *q = static_cast<const T *>(a.q) + (t.qs.begin + tok) * a.q_stride + static_cast<int64_t>(kvh * a.group + r % a.group) * D;
            float x[QV][8];
            uint32_t big = 0;
#pragma unroll
            for (int j = 0; j < QV; ++j) {
                // products 2h and 2h + 1: channels 64h + 16g.., 64h + 16g + 8..; a last one by itself: 8g.. of the last 32
                const T *qj = q + (j == QV - 1 && QV % 2 ? 32 * j + 8 * g : 64 * (j / 2) + 16 * g + 8 * (j & 1));
                constexpr int N = 8 * static_cast<int>(sizeof(T)) / 16;
                uint4 v[N];
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = reinterpret_cast<const uint4 *>(qj)[i];
                const uint32_t *w = reinterpret_cast<const uint32_t *>(v);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t u = BF ? (e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16) : w[e];
                    x[j][e] = as_float(u);
                    big = max(big, u & 0x7fffffffu);
                }
            }
            // the row's power: its largest magnitude to [2^14, 2^15).  Magnitudes' bits rise with them, infinities and NaN above
            // all; their rows keep them, and give NaN.
            big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), 16, 64)));
            big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), 32, 64)));
            const int e = min(max(static_cast<int>(big >> 23) - 127, -100), 127);
            unit[n] = ldexpf(a.scale * kLog2e, e - 14);
#pragma unroll
            for (int j = 0; j < QV; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = ldexpf(x[j][2 * i], 14 - e), v = ldexpf(x[j][2 * i + 1], 14 - e);
                    f[n][j][0][i] = pack_f16x2(u, v);
                    if constexpr (P == 2) {
                        const f32x2 h = unpack_f16x2(f[n][j][0][i]);
                        f[n][j][1][i] = pack_f16x2(u - h[0], v - h[1]);
                    }
                }
        }
    }
};

// A lane's running results of NS sets of 16 rows.
template <int D, int NS, int P>
struct Sums {
    static constexpr int KT = kStep / 16, C = D / 16;
    f32x4 acc[NS][C];  // in units of `unit`
    float sum[NS], base[NS], above[NS];  // above: the score from which on the base moves (-inf: nothing seen yet)
    float unit;
    bool again;  // the rows are to be computed key by key

    __device__ __forceinline__ void clear() {
        unit = 0.0f;
        again = false;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            sum[n] = base[n] = 0.0f;
            above[n] = neg_inf();
#pragma unroll
            for (int t = 0; t < C; ++t) acc[n][t] = f32x4{0, 0, 0, 0};
        }
    }

    // From a set's products w of a step's keys (the lane's are at + 16g..) to its weights, ready to meet the values.
    __device__ __forceinline__ void weigh(int n, f32x4 (&w)[KT], float f, int at, bool cut, Sight see, int sinks, u32x4 (&pw)[KT / 2][P]) {
        if (cut) {
            // (the first key's place is made here, so that nothing of this is done where no key is hidden)
            int key = at + 16 * ((threadIdx.x & 63) >> 4);
            asm volatile("" : "+v"(key));
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = key + 4 * t + i;
                    w[t][i] = (k >= see.lim) | ((k < see.from) & (k >= sinks)) ? neg_inf() : w[t][i];
                }
        }
        f = fmaxf(f, 0x1p-126f);  // products of 0 stay 0, hidden ones -inf
        float mx = neg_inf();
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, w[t][i]);
        if (__builtin_amdgcn_ballot_w64(mx * f > above[n]) != 0) {
            mx = max_over_groups(mx) * f;
            const bool over = mx > above[n];
            const float to = over ? mx - kUnder : base[n];
            const float alpha = above[n] == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(base[n] - to);
            sum[n] *= alpha;
#pragma unroll
            for (int t = 0; t < C; ++t) acc[n][t] *= alpha;
            base[n] = to;
            above[n] = over ? to + kReach : above[n];
            // (past float32's range a row is NaN either way)
            again = again || __builtin_amdgcn_ballot_w64(fabsf(to) >= kFar && fabsf(to) < __builtin_inff()) != 0;
        }
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[t][i] = __builtin_amdgcn_exp2f(fmaf(w[t][i], f, -base[n]));
        // their sum in 32 bits, before they are rounded
#pragma unroll
        for (int t = 0; t < KT; ++t) sum[n] += (w[t][0] + w[t][1]) + (w[t][2] + w[t][3]);
        // half precision keeps 11 bits of a weight (2^-11 off at most), two terms 22
#pragma unroll
        for (int u = 0; u < KT / 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = w[2 * u + (i >> 1)][2 * (i & 1)], y = w[2 * u + (i >> 1)][2 * (i & 1) + 1];
                pw[u][0][i] = pack_f16x2(x, y);
                if constexpr (P == 2) {
                    const f32x2 t = unpack_f16x2(pw[u][0][i]);
                    pw[u][1][i] = pack_f16x2(x - t[0], y - t[1]);
                }
            }
    }

    // Makes the unit at least a step of values; the step's ratio to it.
    __device__ __forceinline__ float reach(float step_v) {
        if (step_v > unit) {
            const float ratio = unit / step_v;  // powers of two, or 0
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int t = 0; t < C; ++t) acc[n][t] *= ratio;
            again = again || (ratio < kLeastRatio && unit > 0.0f);
            unit = step_v;
        }
        const float ratio = unit > 0.0f ? step_v / unit : 0.0f;
        again = again || (ratio < kLeastRatio && step_v > 0.0f);
        return ratio;
    }
};

// Where a row's results go: the output, or its piece's place in the workspace.
template <class T, int D>
struct Place {
    int64_t cell, part;
    T *to;
    __device__ __forceinline__ Place(const AttendArgs &a, const Tile &t, int split, int r, int kvh) {
        const int64_t token = t.qs.begin + r / a.group;
        const int head = kvh * a.group + r % a.group;
        cell = token * a.heads + head;
        part = split * a.total_q * a.heads + cell;
        to = static_cast<T *>(a.o) + token * a.o_stride + static_cast<int64_t>(head) * D;
    }
    // (base + lo: what weights are relative to)
    __device__ __forceinline__ void sums(const AttendArgs &a, float base, float lo, float total) const {
        if (a.splits > 1) a.part_ml[part] = sum_of(base, lo, total, 1.0f);
        else if (a.lse) a.lse[cell] = log_of(base, lo, total);
    }
};

// A row's channels 16t + 4g.. out: divided by the sum before the unit, so that means of finite values are finite.
template <class T, int D>
__device__ __forceinline__ void put(const AttendArgs &a, const Tile &t, int split, int r, int kvh, const float (&y)[D / 4], float base,
                                    float total, float unit) {
    const int g = (threadIdx.x & 63) >> 4;
    if (r >= t.nrows) return;
    const Place<T, D> place(a, t, split, r, kvh);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) {
        const f32x4 z = {y[4 * e] * inv * unit, y[4 * e + 1] * inv * unit, y[4 * e + 2] * inv * unit, y[4 * e + 3] * inv * unit};
        if (a.splits > 1) *reinterpret_cast<f32x4 *>(a.part_o + place.part * D + 16 * e + 4 * g) = z;
        else if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2 *>(place.to + 16 * e + 4 * g) = u32x2{pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3])};
        else *reinterpret_cast<f32x4 *>(place.to + 16 * e + 4 * g) = z;
    }
    if (g == 0) place.sums(a, base, 0.0f, total);
}

// One row by the whole wave, key by key: of every `splits`-th run of `run` steps, scores with a key per lane, values with a
// channel per lane, in 32 bits.  A base is kept in two parts, its rounding apart, and weights are of differences: for rows
// whose scores or values' steps pass what the tiles hold.
template <class T, int D>
__device__ void row_by_keys(const AttendArgs &a, const Tile &t, int split, int run, int r, int kvh) {
    const int lane = threadIdx.x & 63, tok = r / a.group, block = 1 << a.cache.block_log2;
    const T *q = static_cast<const T *>(a.q) + (t.qs.begin + tok) * a.q_stride + static_cast<int64_t>(kvh * a.group + r % a.group) * D;
    const Sight see = sight_of(a, t, tok);
    float x[2], o[2] = {0.0f, 0.0f}, hi = neg_inf(), lo = 0.0f, total = 0.0f;
    uint32_t big = 0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        x[w] = lane + 64 * w < D ? load_as_f32<T>(q + lane + 64 * w) : 0.0f;
        big = max(big, __builtin_bit_cast(uint32_t, x[w]) & 0x7fffffffu);
    }
    for (int d = 1; d < 64; d <<= 1) big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), d, 64)));
    const int e = min(max(static_cast<int>(big >> 23) - 127, -100), 127);
#pragma unroll
    for (int w = 0; w < 2; ++w) x[w] = ldexpf(x[w], 14 - e);
    const int room = 32 - __builtin_clz(t.keys | 1);  // weights add up to 1 at most, so that sums of finite values stay finite
    for (int i = 0; i < t.steps; ++i) {
        if (i / run % a.splits != split) continue;
        const int k0 = t.key_of(i), page = page_of(a.cache, t.s, k0 >> a.cache.block_log2);
        if (page < 0) continue;
        const int64_t cell = static_cast<int64_t>(page) * a.cache.kv_heads + kvh;
        const float2 sizes = a.cache.steps[cell];
        const uint8_t *codes = a.cache.codes + cell * (2 * block * D);
        const uint8_t *kc = codes + ((k0 & (block - 1)) + lane) * D;
        float s = 0.0f;
        for (int c = 0; c < D; c += 4) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(kc + c);
#pragma unroll
            for (int b = 0; b < 4; ++b)
                s = fmaf(__shfl(c < 64 ? x[0] : x[1], (c + b) & 63, 64), static_cast<float>((w >> (8 * b)) & 0xffu) - 128.0f, s);
        }
        const float f = fmaxf(ldexpf(a.scale * kLog2e, e - 14) * sizes.x, 0x1p-126f);
        const int key = k0 + lane;
        const bool hidden = key >= see.lim || (key < see.from && key >= t.sinks);
        if (hidden) s = neg_inf();
        float mx = s;
        for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
        const float h = mx * f, l = fmaf(mx, f, -h);
        if (mx != neg_inf() && (h > hi || (h == hi && l > lo))) {
            const float alpha = hi == neg_inf() ? 0.0f : exp2f((hi - h) + (lo - l));
            total *= alpha;
            o[0] *= alpha;
            o[1] *= alpha;
            hi = h;
            lo = l;
        }
        const float p = hidden ? 0.0f : exp2f(hi == neg_inf() ? s : (fmaf(s, f, -hi) - lo) - static_cast<float>(room));
        float all = p;
        for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d, 64);
        total += all;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (64 * w >= D) continue;
            const uint8_t *vc = codes + ((D + min(lane + 64 * w, D - 1)) << a.cache.block_log2) + (k0 & (block - 1));
            for (int j = 0; j < kStep; j += 4) {
                const uint32_t v = *reinterpret_cast<const uint32_t *>(vc + j);
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    o[w] = fmaf(__shfl(p, j + b, 64), (static_cast<float>((v >> (8 * b)) & 0xffu) - 128.0f) * sizes.y, o[w]);
            }
        }
    }
    const Place<T, D> place(a, t, split, r, kvh);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if (lane + 64 * w >= D) continue;
        if (a.splits > 1) a.part_o[place.part * D + lane + 64 * w] = o[w] * inv;
        else store_from_f32<T>(place.to + lane + 64 * w, o[w] * inv);
    }
    if (lane == 0) place.sums(a, hi, lo + static_cast<float>(room), total);
}

// A wave's walk over its steps of a tile: pages and steps of 64 of them at a time, one a lane.
struct Walk {
    int it, pages, page, k0;
    float2 sizes;
    const uint8_t *codes;  // of the page's head

    // Goes to the next step of every `pieces`-th from `piece` on whose page is one; false: none is left.
    __device__ __forceinline__ bool next(const AttendArgs &a, const Tile &t, int kvh, int piece, int pieces, int head_bytes) {
        const int lane = threadIdx.x & 63;
        for (;;) {
            ++it;
            const int i = piece + it * pieces;
            if (i >= t.steps) return false;
            if ((it & 63) == 0) {
                const int mine = i + lane * pieces;
                pages = mine < t.steps ? page_of(a.cache, t.s, t.key_of(mine) >> a.cache.block_log2) : -1;
                sizes = pages >= 0 ? a.cache.steps[static_cast<int64_t>(pages) * a.cache.kv_heads + kvh] : make_float2(0.0f, 0.0f);
            }
            page = __builtin_amdgcn_readlane(pages, it & 63);
            if (page < 0) continue;  // no such page: its keys count for nothing
            k0 = t.key_of(i);
            codes = a.cache.codes + (static_cast<int64_t>(page) * a.cache.kv_heads + kvh) * head_bytes;
            return true;
        }
    }
    __device__ __forceinline__ float step_k() const { return as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, sizes.x), it & 63)); }
    __device__ __forceinline__ float step_v() const { return as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, sizes.y), it & 63)); }
};

// The operands of a step as they lie in a page.  S^T = K Q^T and O^T = V^T P^T, so that what one product leaves in a
// lane is what the next one wants there.  A 16x16 product leaves lane (c, g) = (lane & 15, lane >> 4) with rows 4g..4g+3 of
// column c; product t of a step takes key 16 (c >> 2) + 4t + (c & 3) as its row c, so that lane
// (c, g) gets keys 16g + 4t + i of query c: the lane's 16 weights are of keys 16g..16g+15, and the
// values' operand wants the same keys of a channel: one 16-byte piece of the cache.
// The keys' operand wants channels of a row, in any order that the queries share: 16 side by side for two products.
template <int D>
__device__ __forceinline__ void fetch_keys(const uint8_t *codes, int place, int t, uint32_t (&w)[D / 16]) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const uint8_t *p = codes + place * D + (16 * (c >> 2) + (c & 3)) * D + 4 * t * D;
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p + 64 * h + 16 * g);
        w[4 * h] = v.x, w[4 * h + 1] = v.y, w[4 * h + 2] = v.z, w[4 * h + 3] = v.w;
    }
    if constexpr (D % 64 != 0) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p + 64 * (D / 64) + 8 * g);
        w[D / 16 - 2] = v.x, w[D / 16 - 1] = v.y;
    }
}
template <int D>
__device__ __forceinline__ void fetch_values(const uint8_t *codes, int block_log2, int place, int t, uint32_t (&w)[4]) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const uint4 v = *reinterpret_cast<const uint4 *>(codes + ((D + 16 * t + c) << block_log2) + place + 16 * g);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
}

// Few rows: a tile of 16 of one sequence.  The workgroup's four waves take every fourth step each, and join through LDS.
// Codes go from memory to a product's registers through two instructions for every four, without LDS; the next step's
// keys are on their way from the first product on, its values from the last.
template <class T, int D>
__global__ void __launch_bounds__(256, 2) cache_rows_kernel(AttendArgs a) {
    using Q = Queries<T, D, 1>;
    constexpr int P = Q::P, QV = Q::QV, KT = kStep / 16, C = D / 16;
    __shared__ float part[4][4 * C][64];
    __shared__ float4 part_ml[4][16];
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = xcd_tile(blockIdx.x, gridDim.x);
    const int split = id / a.tile_groups % a.splits, kvh = id / a.tile_groups / a.splits;
    const Tile t = tile_of(a, id % a.tile_groups, 16, 4);
    if (t.nrows == 0) return;
    Q q;
    q.load(a, t, t.r0, kvh);
    Sums<D, 1, P> r;
    r.clear();
    const int piece = split * 4 + wave, pieces = a.splits * 4, block = 1 << a.cache.block_log2, head_bytes = 2 * block * D;
    Walk walk = {-1, 0, 0, 0, make_float2(0.0f, 0.0f), nullptr};
    uint32_t kr[KT][D / 16], vr[C][4];
    const auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KT; ++i) fetch_keys<D>(walk.codes, walk.k0 & (block - 1), i, kr[i]);
    };
    const auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < C; ++i) fetch_values<D>(walk.codes, a.cache.block_log2, walk.k0 & (block - 1), i, vr[i]);
    };
    bool more = walk.next(a, t, kvh, piece, pieces, head_bytes);
    if (more) {
        load_k();
        load_v();
    }
    while (more) {
        const float step_k = walk.step_k(), step_v = walk.step_v();
        const int at = walk.k0;
        f32x4 w[KT];
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            w[i] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < QV; ++j) {
                const u32x4 x = codes_f16(kr[i][2 * j], kr[i][2 * j + 1]);
#pragma unroll
                for (int p = P - 1; p >= 0; --p) w[i] = product(x, q.f[0][j][p], w[i]);
            }
        }
        more = walk.next(a, t, kvh, piece, pieces, head_bytes);
        if (more) load_k();
        u32x4 pw[KT / 2][P];
        r.weigh(0, w, q.unit[0] * step_k, at, t.cut(at), q.sight[0], t.sinks, pw);
        const float ratio = r.reach(step_v);
        const _Float16 h = static_cast<_Float16>(ratio), b = static_cast<_Float16>(-1152.0f * ratio);
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int u = 0; u < KT / 2; ++u) {
                const u32x4 x = codes_f16(vr[i][2 * u], vr[i][2 * u + 1], f16x2{h, h}, f16x2{b, b});
#pragma unroll
                for (int p = P - 1; p >= 0; --p) r.acc[0][i] = product(x, pw[u][p], r.acc[0][i]);
            }
        if (more) load_v();
    }

    // ---- the waves' results, joined by the first
    const float l = sum_over_groups(r.sum[0]);
    if (g == 0) part_ml[wave][c] = sum_of(r.base[0], r.again ? 1.0f : 0.0f, l, r.unit);
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[wave][4 * i + e][lane] = r.acc[0][i][e];
    __syncthreads();
    float least = __builtin_inff(), unit = 0.0f, base = neg_inf(), total = 0.0f, y[4 * C];
    bool again = false;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float4 m = part_ml[p][c];
        again = again || m.y != 0.0f;
        if (m.z != 0.0f) base = fmaxf(base, m.x);
        if (m.w > 0.0f) least = fminf(least, m.w);
        unit = fmaxf(unit, m.w);
    }
    if (again || least < unit * kLeastRatio) {  // the same for the workgroup
        for (int i = wave; i < min(16, t.nrows - t.r0); i += 4) row_by_keys<T, D>(a, t, split, 4, t.r0 + i, kvh);
        return;
    }
    if (wave != 0) return;
#pragma unroll
    for (int e = 0; e < 4 * C; ++e) y[e] = 0.0f;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float4 m = part_ml[p][c];
        // (a sum that is a NaN is not 0 and stays)
        const float wgt = m.z == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m.x - base), scaled = m.w > 0.0f ? wgt * (m.w / unit) : 0.0f;
        total += wgt * m.z;
#pragma unroll
        for (int e = 0; e < 4 * C; ++e) y[e] += scaled * part[p][e][lane];
    }
    put<T, D>(a, t, split, t.r0 + c, kvh, y, base, total, unit);
}

// Many rows: a tile of 64 NS of one sequence, 16 NS of them for each of the workgroup's four waves.  A step's codes
// become half precision once, a quarter of them by each wave, and lie in LDS (two buffers, one barrier a step) as the
// products' operands, lane by lane: reads and writes are whole rows of 1 KiB.
template <class T, int D, int NS>
__global__ void __launch_bounds__(256, 2) cache_chunk_kernel(AttendArgs a) {
    using Q = Queries<T, D, NS>;
    constexpr int P = Q::P, QV = Q::QV, KT = kStep / 16, C = D / 16, VT = (C + 3) / 4;
    constexpr int KEYS = KT * QV, VALUES = C * (KT / 2);  // operands of a step, 1 KiB each
    __shared__ u32x4 operands[2][KEYS + VALUES][64];
    const int lane = threadIdx.x & 63, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // consecutive workgroups of one XCD run neighbouring tiles of a head: its L2 holds their keys
    const int id = xcd_tile(blockIdx.x, gridDim.x);
    const int split = id / a.tile_groups % a.splits, kvh = id / a.tile_groups / a.splits;
    const Tile t = tile_of(a, id % a.tile_groups, 64 * NS, NS == 1 ? 6 : NS == 2 ? 7 : 8);
    if (t.nrows == 0) return;
    const int r0 = t.r0 + 16 * NS * wave;
    Q q;
    q.load(a, t, r0, kvh);
    Sums<D, NS, P> r;
    r.clear();
    const int block = 1 << a.cache.block_log2, head_bytes = 2 * block * D;
    Walk walk = {-1, 0, 0, 0, make_float2(0.0f, 0.0f), nullptr};
    uint32_t kr[D / 16], vr[VT][4];
    float unit = 0.0f, step_k = 0.0f, step_v = 0.0f;  // of the step whose codes are fetched
    const auto fetch = [&]() __attribute__((always_inline)) {
        fetch_keys<D>(walk.codes, walk.k0 & (block - 1), wave, kr);
#pragma unroll
        for (int i = 0; i < VT; ++i)
            if (wave + 4 * i < C) fetch_values<D>(walk.codes, a.cache.block_log2, walk.k0 & (block - 1), wave + 4 * i, vr[i]);
        step_k = walk.step_k();
        step_v = walk.step_v();
    };
    // fetched codes to a buffer
    const auto lay_out = [&](int buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < QV; ++j) operands[buffer][wave * QV + j][lane] = codes_f16(kr[2 * j], kr[2 * j + 1]);
        unit = fmaxf(unit, step_v);
        const float ratio = unit > 0.0f ? step_v / unit : 0.0f;  // as `reach` has it
        const _Float16 h = static_cast<_Float16>(ratio), b = static_cast<_Float16>(-1152.0f * ratio);
#pragma unroll
        for (int i = 0; i < VT; ++i)
            if (wave + 4 * i < C) {
#pragma unroll
                for (int u = 0; u < KT / 2; ++u)
                    operands[buffer][KEYS + (wave + 4 * i) * (KT / 2) + u][lane] = codes_f16(vr[i][2 * u], vr[i][2 * u + 1], f16x2{h, h}, f16x2{b, b});
            }
    };
    bool more = walk.next(a, t, kvh, split, a.splits, head_bytes);  // the same for all waves
    if (more) {
        fetch();
        lay_out(0);
    }
    for (int buffer = 0; more; buffer ^= 1) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int at = walk.k0;
        const float now_k = step_k, now_v = step_v;
        more = walk.next(a, t, kvh, split, a.splits, head_bytes);
        if (more) fetch();
        if (r0 < t.nrows) {
            // operands of the next few products are on their way while these run (the barriers to the compiler's order keep them there)
            const u32x4 (*from)[64] = operands[buffer];
            u32x4 x[2][QV], y[2][4];
            f32x4 w[NS][KT];
#pragma unroll
            for (int j = 0; j < QV; ++j) x[0][j] = from[j][lane];
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                if (i + 1 < KT) {
#pragma unroll
                    for (int j = 0; j < QV; ++j) x[(i + 1) & 1][j] = from[(i + 1) * QV + j][lane];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[0][j] = from[KEYS + j][lane];
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < NS; ++n) w[n][i] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < QV; ++j)
#pragma unroll
                    for (int n = 0; n < NS; ++n)
#pragma unroll
                        for (int p = P - 1; p >= 0; --p) w[n][i] = product(x[i & 1][j], q.f[n][j][p], w[n][i]);
            }
            const bool cut = t.cut(at);
            u32x4 pw[NS][KT / 2][P];
#pragma unroll
            for (int n = 0; n < NS; ++n) r.weigh(n, w[n], q.unit[n] * now_k, at, cut, q.sight[n], t.sinks, pw[n]);
            r.reach(now_v);
#pragma unroll
            for (int i = 0; i < C; i += 2) {  // two runs of 16 channels
                if (i + 2 < C) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[(i / 2 + 1) & 1][j] = from[KEYS + (i + 2) * 2 + j][lane];
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int n = 0; n < NS; ++n)
#pragma unroll
                        for (int p = P - 1; p >= 0; --p)
                            r.acc[n][i + j / 2] = product(y[(i / 2) & 1][j], pw[n][j & 1][p], r.acc[n][i + j / 2]);
            }
        }
        if (more) lay_out(buffer ^ 1);
    }
    if (r0 >= t.nrows) return;
    if (r.again) {
        for (int i = r0; i < min(r0 + 16 * NS, t.nrows); ++i) row_by_keys<T, D>(a, t, split, 1, i, kvh);
        return;
    }
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        float y[4 * C];
#pragma unroll
        for (int e = 0; e < 4 * C; ++e) y[e] = r.acc[n][e / 4][e % 4];
        put<T, D>(a, t, split, r0 + 16 * n + c, kvh, y, r.base[n], sum_over_groups(r.sum[n]), r.unit);
    }
}

// Joins the pieces of each (row, head), in their order; a wave each.
template <class T, int D>
__global__ void __launch_bounds__(256) cache_join_kernel(AttendArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t cell = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t cells = a.total_q * a.heads;
    if (cell >= cells) return;
    const int64_t row = cell / a.heads;
    const int head = static_cast<int>(cell - row * a.heads);
    if (sequence_of_row(a.q_starts, a.sequences, row) < 0) return;
    // a lane for each piece (there are at most 64): its weight, 0 for one without keys (a sum that is a NaN is not 0 and stays)
    const float4 none = sum_of(neg_inf(), 0.0f, 0.0f, 0.0f);
    const float4 mine = lane < a.splits ? a.part_ml[lane * cells + cell] : none;
    float4 top = mine.z != 0.0f ? mine : none;
    for (int d = 1; d < 64; d <<= 1) {
        const float4 other = sum_of(__shfl_xor(top.x, d, 64), __shfl_xor(top.y, d, 64), 0.0f, 0.0f);
        if (above_of(other, top)) top = other;
    }
    const float w = mine.z != 0.0f ? weight_of(mine, top) * mine.z : 0.0f;
    float total = w, o[2] = {0.0f, 0.0f};
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d, 64);
    // parts are divided by their sums: theirs are the weights, as shares of the whole, so that means stay finite
    const float share = total == 0.0f ? 0.0f : w / total;
    for (uint64_t left = __ballot(mine.z != 0.0f); left;) {
        float wp[4], x[4][2];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int p = left ? __builtin_ctzll(left) : -1;
            left &= left - 1;
            wp[u] = x[u][0] = x[u][1] = 0.0f;
            if (p < 0) continue;
            wp[u] = __shfl(share, p, 64);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (lane + 64 * e < D) x[u][e] = a.part_o[(p * cells + cell) * D + lane + 64 * e];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) o[e] += wp[u] * x[u][e];
    }
    T *to = static_cast<T *>(a.o) + row * a.o_stride + static_cast<int64_t>(head) * D;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < D) store_from_f32<T>(to + lane + 64 * e, o[e]);
    if (a.lse && lane == 0) a.lse[cell] = log_of(top.x, top.y, total);
}

// How a call is cut: by sequences' mean rows into tiles of 16 (four waves share a tile's keys) or of 64 and 128 (four waves share
// its rows), an upper bound of each, as the lengths are on the device; and, where there would be fewer than two waves for each
// SIMD, every tile's keys over several workgroups, with at least four steps a wave.
struct Cut {
    int64_t tile_groups;
    int32_t splits, sets;  // 0: tiles of 16 rows
};
Cut cut_of(int64_t total_q, int32_t heads, int32_t kv_heads, int32_t d, int64_t sequences, int64_t max_k, int32_t window, int32_t sinks) {
    constexpr int64_t kGroups = 256 * 2;
    const int64_t rows = total_q * (heads / kv_heads), per = rows / std::max<int64_t>(sequences, 1);
    const int32_t sets = per <= 16 ? 0 : per <= 64 ? 1 : 2;
    const int64_t tiles = rows / (sets == 0 ? 16 : 64 * sets) + sequences, groups = std::max<int64_t>(tiles * kv_heads, 1);
    const int64_t keys = window ? std::min<int64_t>(max_k, static_cast<int64_t>(window) + sinks + per + 2 * kStep) : max_k;
    int32_t splits = 1;
    while (splits < 64 && groups * splits * 2 <= kGroups && keys >= (sets == 0 ? 16 : 4) * kStep * splits) splits *= 2;
    return {tiles, splits, sets};
}

using AttendFn = void (*)(AttendArgs);
template <class T, int D>
AttendFn pick_tile(const Cut &cut) {
    return cut.sets == 0 ? cache_rows_kernel<T, D> : cut.sets == 1 ? cache_chunk_kernel<T, D, 1> : cache_chunk_kernel<T, D, 2>;
}
template <class T>
AttendFn pick_attend(int32_t d, const Cut &cut) {
    return d == 32 ? pick_tile<T, 32>(cut) : d == 64 ? pick_tile<T, 64>(cut) : d == 96 ? pick_tile<T, 96>(cut) : pick_tile<T, 128>(cut);
}
template <class T>
AttendFn pick_join(int32_t d) {
    return d == 32 ? cache_join_kernel<T, 32> : d == 64 ? cache_join_kernel<T, 64> : d == 96 ? cache_join_kernel<T, 96> : cache_join_kernel<T, 128>;
}

void check_call(const s3dx_cache *c, int64_t total_q, int32_t heads, int64_t sequences, int64_t max_k, int32_t window, int32_t sinks) {
    require(c, "cache is NULL");
    require(total_q >= 0 && total_q <= kMaxPlaces, "a row count is out of range (0 to 2^29)");
    require(max_k >= 0 && max_k <= kMaxPlaces, "max_k is out of range (0 to 2^29)");
    require(heads >= c->kv_heads && heads <= 65536 && heads % c->kv_heads == 0, "heads must be a multiple of kv_heads, at most 65536");
    require(total_q * heads <= std::numeric_limits<int32_t>::max(), "total_q * heads is out of range");
    require(sequences >= 0 && sequences <= (INT64_C(1) << 24), "sequences is out of range");
    require(window >= 0 && window <= kMaxPlaces, "window is out of range (0 to 2^29)");
    require(sinks >= 0 && sinks <= kMaxPlaces && (sinks == 0 || window > 0), "sinks is out of range, or without a window");
}

}  // namespace
}  // namespace s3dx

using namespace s3dx;

extern "C" {

S3DX_API s3dx_status s3dx_cache_attention_workspace_size(const s3dx_cache *cache, int64_t total_q, int32_t heads, int64_t sequences,
                                                         int64_t max_k, int32_t window, int32_t sinks, uint64_t *bytes,
                                                         char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        require(bytes, "bytes is NULL");
        check_call(cache, total_q, heads, sequences, max_k, window, sinks);
        const Cut cut = cut_of(total_q, heads, cache->kv_heads, cache->head_dim, sequences, max_k, window, sinks);
        *bytes = 0;
        if (cut.splits == 1) return;
        Sizer z;
        z.take<float>(static_cast<uint64_t>(cut.splits) * total_q * heads * cache->head_dim);
        z.take<float4>(static_cast<uint64_t>(cut.splits) * total_q * heads);
        *bytes = z.used;
    });
}

S3DX_API s3dx_status s3dx_cache_attention(const s3dx_cache *cache, const void *q, int32_t dtype, int64_t total_q, int32_t heads,
                                          int64_t q_stride, const int32_t *q_starts, const int32_t *table, int32_t table_stride,
                                          const int32_t *lengths, int64_t sequences, int64_t max_k, int32_t window,
                                          int32_t sinks, float softmax_scale, int32_t flags, void *o, int64_t o_stride,
                                          float *lse, void *workspace, uint64_t workspace_bytes, s3dx_stream stream, char *error,
                                          uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        check_call(cache, total_q, heads, sequences, max_k, window, sinks);
        check_table(cache, table, table_stride, lengths, sequences);
        require_dtype(dtype);
        require((flags & ~S3DX_BLOCK_CAUSAL) == 0, "unknown flags");
        require(window == 0 || (flags & S3DX_BLOCK_CAUSAL), "a window needs S3DX_BLOCK_CAUSAL");
        require(softmax_scale > 0.0f && softmax_scale < 1e6f, "softmax_scale must be above 0 and below 1e6");
        if (total_q == 0 || sequences == 0) return;
        for (const auto &[p, stride] : {std::pair(q, q_stride), std::pair(static_cast<const void *>(o), o_stride)}) {
            require(p && aligned(p, 16), "a row pointer is NULL or not 16-byte aligned");
            require(stride >= static_cast<int64_t>(heads) * cache->head_dim, "a row stride is shorter than its heads");
            require(stride <= (INT64_C(1) << 40) && stride * dtype_size(dtype) % 16 == 0,
                    "a row stride must be whole 16-byte pieces, at most 2^40 elements");
        }
        require(q_starts && aligned(q_starts, 4), "starts is NULL or not aligned");
        require(!lse || aligned(lse, 4), "lse is not aligned");
        const Cut cut = cut_of(total_q, heads, cache->kv_heads, cache->head_dim, sequences, max_k, window, sinks);
        AttendArgs a = {view_of(cache, table, table_stride, lengths), q, o, lse, q_starts, total_q, q_stride, o_stride, sequences,
                        heads, heads / cache->kv_heads, flags & S3DX_BLOCK_CAUSAL, window, sinks, cut.splits,
                        static_cast<int32_t>(cut.tile_groups), softmax_scale, nullptr, nullptr};
        if (cut.splits > 1) {
            require(workspace && aligned(workspace, 16), "workspace is NULL or not 16-byte aligned");
            Carver w(workspace, workspace_bytes);
            a.part_o = w.take<float>(static_cast<uint64_t>(cut.splits) * total_q * heads * cache->head_dim);
            a.part_ml = w.take<float4>(static_cast<uint64_t>(cut.splits) * total_q * heads);
        }
        const int64_t grid = cut.tile_groups * cache->kv_heads * cut.splits;
        require(grid <= 0xffffffffll / 256, "too many rows and sequences");
        const bool bf = dtype == S3DX_BF16;
        (bf ? pick_attend<uint16_t>(cache->head_dim, cut) : pick_attend<float>(cache->head_dim, cut))<<<
            dim3(static_cast<unsigned>(grid)), dim3(256), 0, as_stream(stream)>>>(a);
        launch_check("cache attention");
        if (cut.splits > 1) {
            (bf ? pick_join<uint16_t>(cache->head_dim) : pick_join<float>(cache->head_dim))<<<
                dim3(static_cast<unsigned>((total_q * heads + 3) / 4)), dim3(256), 0, as_stream(stream)>>>(a);
            launch_check("cache attention join");
        }
    });
}

}  // extern "C"
