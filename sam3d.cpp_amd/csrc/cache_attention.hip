// Attention of new rows over a cache in 8 bits: all keys of a sequence, those up to
// a row's own place, or a window of them and the first ones.
//
// o = sum_j p_j step_v c_vj / sum_j p_j, p_j = exp(scale step_k q.c_kj - m): codes are whole
// numbers of 8 bits, which half precision holds exactly, so the products of both
// kinds run on its matrix units with no rounding of a key or a value; a query is taken in units of a
// power of two that fits its row, as one half-precision number (bfloat16 rows: exact) or
// as two (float32 rows: 22 bits).  Steps are of a whole block and multiply results.
//
// What bounds it: few rows, the codes, read once (8 rows over 65,536 keys each, 32 / 8 heads x 128: 193 us, 5.6 TB/s, nearly what a
// kernel that reads alone reaches); many, products and the vector work beside them (exponentials, maxima, the codes' way to half
// precision), which hardly overlap: 4 chunks of 1,024 rows behind 8,192 keys, 32 / 8 heads x 128, take 640 us, 0.9 PFLOP/s,
// matrix units busy 39% and vector issue 50% of a SIMD's cycles.
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
    int32_t heads, group, causal, window, sinks, splits, tile_groups, at_once, slots;
    float scale;
    float *part_o;    // [splits][total_q][heads][d], divided by their sums
    float4 *part_ml;  // [splits][total_q][heads]: see sum_of
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;  // keys of a step: half or all of a block
constexpr uint32_t kInfBits = 0x7f800000u;

// Weights are 2^(score - base), score in binary orders.  A base stands 2^7 below the largest score when it is set
// and moves once a weight would pass 2^15: half precision keeps its 11 bits of weights down to 2^-21 of the
// largest and some down to 2^-31; a base that follows every maximum would scale the sums at every step.
// Beyond 2^20 a base's own rounding would show in its weights: such rows are computed again, key by key.
constexpr float kUnder = 7.0f, kReach = 15.0f, kFar = 0x1p20f;
// Values count in units of the largest step met, and a smaller one's ratio goes into its codes: down to 2^-24 they
// stay exact in half precision.  Rows that meet steps further apart are computed again, key by key.
constexpr float kLeastRatio = 0x1p-24f;

// step / unit of steps up to the unit, which are powers of two or 0 (below 2^-126: 0).
__device__ __forceinline__ float ratio_of(float step, float unit) {
    const int32_t bits = __builtin_bit_cast(int32_t, step) - __builtin_bit_cast(int32_t, unit) + 0x3f800000;
    return step > 0.0f && bits > 0 ? __builtin_bit_cast(float, bits) : 0.0f;
}

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
__device__ __forceinline__ f32x16 product(const u32x4 &a, const u32x4 &b, f32x16 d) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), d, 0, 0, 0);
}

// What a tile of a sequence's rows (query rows times the heads that share a key head) sees, and how its keys are cut into
// steps: those of the first keys that stay visible, then from the window's beginning on.
struct Tile {
    Span qs;
    int64_t s;
    int r0, nrows, keys, lag;            // its first row, the sequence's rows, keys, their difference
    int least, low_all, sinks;           // keys that all rows see: below `least`, and from `low_all` on or below `sinks`
    int steps, sink_steps, skip;
    int pieces;                          // workgroups that share its keys
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
// What a workgroup computes: tile i of n tiles of rows (n: none) by a piece of a head's keys.  Of eight (head, piece) each XCD takes one,
// whose keys its L2 then holds; the tiles of those left over are dealt out to all XCDs in turn.
// Workgroups without work stand behind all others.  An XCD's dispatcher fills its shader engines in turn and in order: one without
// work before it holds a workgroup back until the engine whose turn it is has room (8 sequences of 64 rows x 4 over 20,000 keys: 320 us
// with one behind every two for 225).
struct Work {
    int64_t i;
    int split, kvh;
};
__device__ __forceinline__ Work work_of(const AttendArgs &a, int n, bool ordered) {
    constexpr int kUnits = 32;  // compute units of an XCD: an XCD's workgroups x, x + 32, x + 64 are one's
    const int xcd = blockIdx.x % 8, x = blockIdx.x / 8, heads = a.cache.kv_heads * a.splits, each = heads / 8, left = heads - 8 * each;
    const int own = each * n, shared = (left * n - xcd + 7) / 8, mine = own + shared;
    if (x >= mine) return {n, 0, 0};
    int head, i;
    if (ordered && a.at_once) {
        // Causal rows see more keys the later they stand.  Where all workgroups run at once, the shortest tiles share compute units, the
        // longest of those with the shortest: by the tile's rank, 0 the longest.  (2,048 rows of 8 x 4 x 128 from the first on: 71 us
        // in order, longest first, for 65.)
        const int round = x / kUnits, over = min(max(mine - kUnits, 0), kUnits);
        const int rank = round == 0 ? (x < over ? kUnits - over + x : x - over) : round == 1 ? kUnits + over - 1 - (x - kUnits) : x;
        const int l = rank * shared / mine, o = rank - l;
        if ((rank + 1) * shared / mine > l) {
            const int q = 8 * l + xcd;
            head = 8 * each + q % left, i = n - 1 - q / left;
        } else {
            head = xcd * each + o % each, i = n - 1 - o / each;
        }
    } else {
        const int q = 8 * (x - own) + xcd;
        head = x < own ? xcd * each + x / n : 8 * each + q / n;
        i = x < own ? x % n : q % n;
        if (ordered) i = n - 1 - i;  // the longest first
    }
    return {i, head % a.splits, head / a.splits};
}

// Few rows of several sequences: workgroups are shared out by the sequences' lengths, each gets about as many steps (a piece a
// workgroup, `slots` for each head, up to a.splits pieces a tile).  Every lane tries a length of pieces, from the least that could do on,
// and the first is taken with which all tiles find room; the last lane's is one piece for every tile.  (Reciprocals of hardware are
// the same in every wave.)
__device__ __forceinline__ int pieces_of(float steps, float per_length, int most) {
    return max(1, min(static_cast<int>(ceilf(steps * per_length)), most));
}
__device__ __forceinline__ int shared_pieces(const AttendArgs &a, int tiles, float steps) {
    const int lane = threadIdx.x & 63;
    float all = 0.0f, longest = 0.0f;
    const auto of = [](float v, int s) { return as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, v), s)); };
    for (int s = 0; s < static_cast<int>(a.sequences); ++s) {
        all += static_cast<float>(__builtin_amdgcn_readlane(tiles, s)) * of(steps, s);
        longest = fmaxf(longest, of(steps, s));
    }
    const float least = fmaxf(4.0f, fmaxf(all * __builtin_amdgcn_rcpf(static_cast<float>(a.slots)), longest * __builtin_amdgcn_rcpf(static_cast<float>(a.splits))));
    const float per = lane == 63 ? 0.0f : __builtin_amdgcn_rcpf(least * (1.0f + static_cast<float>(lane) * 0.0625f));
    int room = a.slots;
    for (int s = 0; s < static_cast<int>(a.sequences); ++s)
        room -= __builtin_amdgcn_readlane(tiles, s) * pieces_of(of(steps, s), per, a.splits);
    const int taken = __builtin_ctzll(__builtin_amdgcn_ballot_w64(room >= 0 || lane == 63));
    return pieces_of(steps, of(per, taken), a.splits);
}

// A workgroup's rows [r0, r0 + rows) of sequence s; nrows == 0: none.
__device__ __forceinline__ Tile tile_of(const AttendArgs &a, Work &w, int rows, int rows_log2) {
    Tile t = {};
    int pieces = a.splits;
    const bool shared = rows != 128 && a.slots > 0;
    const Sequence q = sequence_at(
        a.q_starts, a.cache.lengths, a.sequences, a.total_q, a.group, rows_log2, 1, a.tile_groups,
        [&](int32_t n, int32_t length) {
            const int tiles = (n * a.group >> rows_log2) + ((n * a.group & (rows - 1)) != 0);
            if (!shared) return tiles;
            int keys = cached_rows(a.cache, length);
            if (a.window) keys = static_cast<int>(min(static_cast<int64_t>(keys), static_cast<int64_t>(a.window) + a.sinks + n + 2 * kStep));
            pieces = shared_pieces(a, tiles, ceilf(static_cast<float>(keys) * (1.0f / kStep)));
            return tiles * pieces;
        },
        [&](int64_t all) {
            if (shared) w = {blockIdx.x / a.cache.kv_heads, 0, static_cast<int>(blockIdx.x % a.cache.kv_heads)};
            else w = work_of(a, static_cast<int>(min(all, static_cast<int64_t>(a.tile_groups))), a.causal && rows == 128);
            return w.i;
        });
    int64_t place = q.unit - q.first;  // (below 2^31 where workgroups are shared out)
    t.pieces = a.splits;
    if (shared) {
        t.pieces = __builtin_amdgcn_readlane(pieces, static_cast<int>(q.s));
        const int i = static_cast<int>(place) / t.pieces;
        w.split = static_cast<int>(place) - i * t.pieces;
        place = i;
    }
    t.s = q.s;
    t.qs = q.rows;
    const int64_t first = place << rows_log2;
    t.nrows = t.qs.rows * a.group;  // total_q * heads < 2^31
    if (first < 0 || first >= t.nrows) {
        t.nrows = 0;
        return t;
    }
    t.r0 = static_cast<int>(first);
    t.keys = cached_rows(a.cache, q.entry);
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

// A lane's query, that of its column in products of COLUMNS, in units of a power of two, in P half-precision terms.  Lane
// (c, g) has channels 64 / COLUMNS times 16 apart: 16 side by side from 16g on for two products, and where there is no
// second one 8 from 8g on.
template <class T, int D, int COLUMNS>
struct Query {
    static constexpr int P = sizeof(T) == 2 ? 1 : 2, G = 64 / COLUMNS, QV = D / (8 * G);
    u32x4 f[QV][P];
    float unit;  // binary orders of a score for each unit of its product, before the keys' step
    Sight sight;

    __device__ __forceinline__ void load(const AttendArgs &a, const Tile &t, int r0, int kvh) {
        constexpr bool BF = sizeof(T) == 2;
        const int lane = threadIdx.x & 63, c = lane % COLUMNS, g = lane / COLUMNS;
        const int r = min(r0 + c, t.nrows - 1), tok = r / a.group;
        sight = sight_of(a, t, tok);
        const T *q = static_cast<const T *>(a.q) + (t.qs.begin + tok) * a.q_stride + static_cast<int64_t>(kvh * a.group + r % a.group) * D;
        float x[QV][8];
        uint32_t big = 0;
#pragma unroll
        for (int j = 0; j < QV; ++j) {
            const T *qj = q + (j == QV - 1 && QV % 2 ? 8 * G * j + 8 * g : 16 * G * (j / 2) + 16 * g + 8 * (j & 1));
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
        // all; their rows give NaN: one term is NaN throughout (an infinity alone can make all scores -inf, which weigh nothing), of two the
        // second is where they stand.
        if constexpr (G == 4) big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), 16, 64)));
        big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), 32, 64)));
        const int e = min(max(static_cast<int>(big >> 23) - 127, -100), 127);
        unit = ldexpf(a.scale * kLog2e, e - 14);
#pragma unroll
        for (int j = 0; j < QV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = ldexpf(x[j][2 * i], 14 - e), v = ldexpf(x[j][2 * i + 1], 14 - e);
                f[j][0][i] = pack_f16x2(u, v);
                if constexpr (P == 2) {
                    const f32x2 h = unpack_f16x2(f[j][0][i]);
                    f[j][1][i] = pack_f16x2(u - h[0], v - h[1]);
                } else {
                    f[j][0][i] = big < kInfBits ? f[j][0][i] : 0x7e007e00u;
                }
            }
    }
};

// Binary orders of a score for each unit of a product.  Never 0: products of 0 stay 0, hidden ones -inf.
__device__ __forceinline__ float score_unit(float query, float step_k) { return fmaxf(query * step_k, 0x1p-126f); }

// Largest and sum over the lanes that hold a column.
template <int COLUMNS>
__device__ __forceinline__ float column_max(float v) {
    if constexpr (COLUMNS == 16) return max_over_groups(v);
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(as_float(a[0]), as_float(a[1]));
}
template <int COLUMNS>
__device__ __forceinline__ float column_sum(float v) {
    if constexpr (COLUMNS == 16) return sum_over_groups(v);
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return as_float(a[0]) + as_float(a[1]);
}

// A lane's running results of its column's row.  Of a step it holds W products, of keys 16 side by side.
template <int D, int COLUMNS, int P>
struct Sums {
    static constexpr int W = COLUMNS == 16 ? 16 : 32, G = 64 / COLUMNS, C = D / COLUMNS;
    typedef float Four __attribute__((ext_vector_type(COLUMNS == 16 ? 4 : 16)));
    Four acc[C];  // in units of `unit`
    float sum, base, above;  // above: the score from which on the base moves (-inf: nothing seen yet)
    float unit;
    bool again;  // the rows are to be computed key by key

    __device__ __forceinline__ void clear() {
        unit = sum = base = 0.0f;
        above = neg_inf();
        again = false;
#pragma unroll
        for (int t = 0; t < C; ++t) acc[t] = 0.0f;
    }

    // Hides of a step's products w what the row does not see: the lane's are of keys at + 16g.., and from 16 G on of the next such.
    __device__ __forceinline__ static void hide(float (&w)[W], int at, Sight see, int sinks) {
        // (the first key's place is made here, so that nothing of this is done where no key is hidden)
        int key = at + 16 * ((threadIdx.x & 63) / COLUMNS);
        asm volatile("" : "+v"(key));
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int k = key + (i / 16) * 16 * G + i % 16;
            w[i] = (k >= see.lim) | ((k < see.from) & (k >= sinks)) ? neg_inf() : w[i];
        }
    }
    // Moves the base where a weight would pass its reach; f: binary orders of a score for each unit of a product.
    __device__ __forceinline__ void settle(const float (&w)[W], float f) {
        float mx = neg_inf();
#pragma unroll
        for (int i = 0; i < W; ++i) mx = fmaxf(mx, w[i]);
        if (__builtin_amdgcn_ballot_w64(mx * f > above) == 0) return;
        mx = column_max<COLUMNS>(mx) * f;
        const bool over = mx > above;
        const float to = over ? mx - kUnder : base;
        const float alpha = above == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(base - to);
        sum *= alpha;
#pragma unroll
        for (int t = 0; t < C; ++t) acc[t] *= alpha;
        base = to;
        above = over ? to + kReach : above;
        // (past float32's range a row is NaN either way)
        again = again || __builtin_amdgcn_ballot_w64(fabsf(to) >= kFar && fabsf(to) < __builtin_inff()) != 0;
    }
    // The weights of products 4i..: their sum in 32 bits, before they are rounded; then half precision keeps 11 bits of a weight (2^-11
    // off at most), two terms 22.
    __device__ __forceinline__ void weigh(int i, const float (&w)[W], float f, u32x4 (&pw)[W / 8][P]) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(w[4 * i + e], f, -base));
        sum += (x[0] + x[1]) + (x[2] + x[3]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t high = pack_f16x2(x[2 * e], x[2 * e + 1]);
            pw[i / 2][0][2 * (i & 1) + e] = high;
            if constexpr (P == 2) {
                const f32x2 h = unpack_f16x2(high);
                pw[i / 2][1][2 * (i & 1) + e] = pack_f16x2(x[2 * e] - h[0], x[2 * e + 1] - h[1]);
            }
        }
    }
    // Makes the unit at least a step of values; the step's ratio to it.
    __device__ __forceinline__ float reach(float step_v) {
        if (step_v > unit) {
            const float ratio = ratio_of(unit, step_v);
#pragma unroll
            for (int t = 0; t < C; ++t) acc[t] *= ratio;
            again = again || (ratio < kLeastRatio && unit > 0.0f);
            unit = step_v;
        }
        const float ratio = ratio_of(step_v, unit);
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
    __device__ __forceinline__ void sums(const AttendArgs &a, const Tile &t, float base, float lo, float total) const {
        if (a.splits > 1) a.part_ml[part] = sum_of(base, lo, total, static_cast<float>(t.pieces));
        else if (a.lse) a.lse[cell] = log_of(base, lo, total);
    }
};

// A row's channels out, the lane's D / G of them, four side by side 4 G apart: divided by the sum before the unit, so that
// means of finite values are finite.
template <class T, int D, int COLUMNS>
__device__ __forceinline__ void put(const AttendArgs &a, const Tile &t, int split, int r, int kvh, const float (&y)[D * COLUMNS / 64],
                                    float base, float total, float unit) {
    const int g = (threadIdx.x & 63) / COLUMNS;
    if (r >= t.nrows) return;
    const Place<T, D> place(a, t, split, r, kvh);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int e = 0; e < D * COLUMNS / 256; ++e) {
        const f32x4 z = {y[4 * e] * inv * unit, y[4 * e + 1] * inv * unit, y[4 * e + 2] * inv * unit, y[4 * e + 3] * inv * unit};
        const int ch = 256 / COLUMNS * e + 4 * g;
        if (a.splits > 1) *reinterpret_cast<f32x4 *>(a.part_o + place.part * D + ch) = z;
        else if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2 *>(place.to + ch) = u32x2{pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3])};
        else *reinterpret_cast<f32x4 *>(place.to + ch) = z;
    }
    if (g == 0) place.sums(a, t, base, 0.0f, total);
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
    for (int w = 0; w < 2; ++w) x[w] = big < kInfBits ? ldexpf(x[w], 14 - e) : __builtin_nanf("");
    const int room = 32 - __builtin_clz(t.keys | 1);  // weights add up to 1 at most, so that sums of finite values stay finite
    for (int i = 0; i < t.steps; ++i) {
        if (i / run % t.pieces != split) continue;
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
        const float p = hidden ? 0.0f : exp2f(hi == neg_inf() ? s * f : (fmaf(s, f, -hi) - lo) - static_cast<float>(room));
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
    if (lane == 0) place.sums(a, t, hi, lo + static_cast<float>(room), total);
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
// lane is what the next one wants there.  A product of 16 (32) columns leaves lane (c, g) = (lane % 16, lane / 16) with
// four rows of column c, 4g.., (with four such, 8 apart).  Rows take keys so that over a step lane (c, g) gets keys
// 16g..16g+15 of query c (and 32 + 16g..): then the values' operand wants 16 keys side by side of a channel, one 16-byte
// piece of the cache.  The keys' operand wants channels of a row, in any order that the queries share: 16 side by
// side for two products.
//
// 16 columns, product t of a step: 16 rows.
template <int D>
__device__ __forceinline__ void fetch_keys16(const uint8_t *codes, int place, int t, uint32_t (&w)[D / 16]) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const uint8_t *p = codes + (place + 16 * (c >> 2) + 4 * t + (c & 3)) * D;
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
// ... 16 channels from 16t on, of 64 keys.
template <int D>
__device__ __forceinline__ uint4 fetch_values16(const uint8_t *codes, int block_log2, int place, int t) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    return *reinterpret_cast<const uint4 *>(codes + ((D + 16 * t + c) << block_log2) + place + 16 * g);
}
// 32 columns: 32 keys of the step's half t, 32 channels from 32h on.
template <int D>
__device__ __forceinline__ uint4 fetch_keys32(const uint8_t *codes, int place, int t, int h) {
    const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
    // row 8i + 4g' + j of a product is lane group g's product 4i + j: key 16g' + 4i + j of the half
    const int key = 32 * t + 16 * ((c >> 2) & 1) + 4 * (c >> 3) + (c & 3);
    return *reinterpret_cast<const uint4 *>(codes + (place + key) * D + 32 * h + 16 * g);
}
// ... the same channels of the same keys.
template <int D>
__device__ __forceinline__ uint4 fetch_values32(const uint8_t *codes, int block_log2, int place, int t, int h) {
    const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
    return *reinterpret_cast<const uint4 *>(codes + ((D + 32 * h + c) << block_log2) + place + 32 * t + 16 * g);
}

// Few rows: a tile of 16 or 32 of one sequence.  The workgroup's four waves take every fourth step each, and join through LDS.
// Memory bounds it, so codes go from there to a product's registers through two instructions for every four, without LDS; the
// next step's keys are on their way from the first product on, its values from the last.  16 or 32 columns, by the rows there are: 40
// rows x 4 over 8 x 20,000 keys take 73 us (4.5 TB/s) in tiles of 32 and took 165 in the chunks' of 128.  (At 128 channels tiles of 32 fill the
// registers and spill 10 of them, 39 of float32 rows, which take 101 us.)
template <class T, int D, int COLUMNS>
__global__ void __launch_bounds__(256, 2) cache_rows_kernel(AttendArgs a) {
    using Q = Query<T, D, COLUMNS>;
    using S = Sums<D, COLUMNS, Q::P>;
    constexpr int P = Q::P, QV = Q::QV, W = S::W, KT = kStep / COLUMNS, C = S::C, Y = D * COLUMNS / 64;
    constexpr int E = COLUMNS * COLUMNS / 64;  // values of a product that a lane holds
    __shared__ float part[4][Y][64];
    __shared__ float4 part_ml[4][COLUMNS];
    const int lane = threadIdx.x & 63, c = lane % COLUMNS, g = lane / COLUMNS;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work work;
    const Tile t = tile_of(a, work, COLUMNS, COLUMNS == 16 ? 4 : 5);
    const int split = work.split, kvh = work.kvh;
    if (t.nrows == 0) return;
    Q q;
    q.load(a, t, t.r0, kvh);
    S r;
    r.clear();
    const int piece = split * 4 + wave, pieces = t.pieces * 4, block = 1 << a.cache.block_log2, head_bytes = 2 * block * D;
    Walk walk = {-1, 0, 0, 0, make_float2(0.0f, 0.0f), nullptr};
    uint32_t kr[KT][2 * QV];  // two dwords a product
    uint32_t vr[C][W / 4];    // a dword for four keys
    const auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            if constexpr (COLUMNS == 16) {
                fetch_keys16<D>(walk.codes, walk.k0 & (block - 1), i, kr[i]);
            } else {
#pragma unroll
                for (int h = 0; h < C; ++h) {
                    const uint4 w = fetch_keys32<D>(walk.codes, walk.k0 & (block - 1), i, h);
                    kr[i][4 * h] = w.x, kr[i][4 * h + 1] = w.y, kr[i][4 * h + 2] = w.z, kr[i][4 * h + 3] = w.w;
                }
            }
        }
    };
    const auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int h = 0; h < W / 16; ++h) {
                uint4 w;
                if constexpr (COLUMNS == 16) w = fetch_values16<D>(walk.codes, a.cache.block_log2, walk.k0 & (block - 1), i);
                else w = fetch_values32<D>(walk.codes, a.cache.block_log2, walk.k0 & (block - 1), h, i);
                vr[i][4 * h] = w.x, vr[i][4 * h + 1] = w.y, vr[i][4 * h + 2] = w.z, vr[i][4 * h + 3] = w.w;
            }
    };
    bool more = walk.next(a, t, kvh, piece, pieces, head_bytes);
    if (more) {
        load_k();
        load_v();
    }
    while (more) {
        const float step_k = walk.step_k(), step_v = walk.step_v();
        const int at = walk.k0;
        float w[W];
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            typename S::Four d = {};
#pragma unroll
            for (int j = 0; j < QV; ++j) {
                const u32x4 x = codes_f16(kr[i][2 * j], kr[i][2 * j + 1]);
#pragma unroll
                for (int p = P - 1; p >= 0; --p) d = product(x, q.f[j][p], d);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) w[E * i + e] = d[e];
        }
        more = walk.next(a, t, kvh, piece, pieces, head_bytes);
        if (more) load_k();
        u32x4 pw[W / 8][P];
        if (t.cut(at)) r.hide(w, at, q.sight, t.sinks);
        const float f = score_unit(q.unit, step_k);
        r.settle(w, f);
#pragma unroll
        for (int i = 0; i < W / 4; ++i) r.weigh(i, w, f, pw);
        const float ratio = r.reach(step_v);
        const _Float16 h = static_cast<_Float16>(ratio), b = static_cast<_Float16>(-1152.0f * ratio);
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int u = 0; u < W / 8; ++u) {
                const u32x4 x = codes_f16(vr[i][2 * u], vr[i][2 * u + 1], f16x2{h, h}, f16x2{b, b});
#pragma unroll
                for (int p = P - 1; p >= 0; --p) r.acc[i] = product(x, pw[u][p], r.acc[i]);
            }
        if (more) load_v();
    }

    // ---- the waves' results, joined by the first
    const float l = column_sum<COLUMNS>(r.sum);
    if (g == 0) part_ml[wave][c] = sum_of(r.base, r.again ? 1.0f : 0.0f, l, r.unit);
#pragma unroll
    for (int e = 0; e < Y; ++e) part[wave][e][lane] = r.acc[e / E][e % E];
    __syncthreads();
    float least = __builtin_inff(), unit = 0.0f, base = neg_inf(), total = 0.0f;
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
        for (int i = wave; i < min(COLUMNS, t.nrows - t.r0); i += 4) row_by_keys<T, D>(a, t, split, 4, t.r0 + i, kvh);
        return;
    }
    if (wave != 0) return;
    float y[Y];
#pragma unroll
    for (int e = 0; e < Y; ++e) y[e] = 0.0f;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float4 m = part_ml[p][c];
        // (a sum that is a NaN is not 0 and stays)
        const float wgt = m.z == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m.x - base), scaled = wgt * ratio_of(m.w, unit);
        total += wgt * m.z;
#pragma unroll
        for (int e = 0; e < Y; ++e) y[e] += scaled * part[p][e][lane];
    }
    put<T, D, COLUMNS>(a, t, split, t.r0 + c, kvh, y, base, total, unit);
}

// Many rows: a tile of 128 of one sequence, 32 of them for each of the workgroup's four waves.  A step's codes
// become half precision once, a quarter of them by each wave, and lie in LDS (two buffers, one barrier a step) as the
// products' operands, lane by lane: reads and writes are whole rows of 1 KiB.  (Straight from memory, as above, every wave turns all
// codes itself: 4 chunks of 1,024 rows 4,172 us for 640.)  Products of 32x32x16: one holds its SIMD from vector work for about 8
// cycles whatever its size (of 16x16x32: 686 for 654 us at the time).  Rare cases stand behind the loop, so that nothing in it spills.
template <class T, int D>
__global__ void __launch_bounds__(256, 2) cache_chunk_kernel(AttendArgs a) {
    using Q = Query<T, D, 32>;
    constexpr int P = Q::P, QV = Q::QV, C = D / 32;
    constexpr int PIECES = 2 * C, MINE = (PIECES + 3) / 4;  // of 32 keys and 32 channels: a 16-byte piece a lane, two operands
    __shared__ u32x4 key_rows[2][2 * PIECES][64], value_rows[2][2 * PIECES][64];
    const int lane = threadIdx.x & 63, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work work;
    const Tile t = tile_of(a, work, 128, 7);
    const int split = work.split, kvh = work.kvh;
    if (t.nrows == 0) return;
    const int r0 = t.r0 + 32 * wave;
    Q q;
    q.load(a, t, r0, kvh);
    Sums<D, 32, P> r;
    r.clear();
    const int block = 1 << a.cache.block_log2, head_bytes = 2 * block * D;
    Walk walk = {-1, 0, 0, 0, make_float2(0.0f, 0.0f), nullptr};
    uint4 kr[MINE], vr[MINE];
    float unit = 0.0f;  // of the last values laid out
    // A step on its way: whether it is one, its codes' page, first key and steps.
    struct Step {
        bool is;
        const uint8_t *codes;
        int at;
        float step_k, step_v;
    };
    const auto next = [&]() __attribute__((always_inline)) {  // the same for all waves
        Step x = {walk.next(a, t, kvh, split, t.pieces, head_bytes), walk.codes, walk.k0, 0.0f, 0.0f};
        if (x.is) x.step_k = walk.step_k(), x.step_v = walk.step_v();
        return x;
    };
    const auto fetch_k = [&](const Step &x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MINE; ++i)
            if (wave + 4 * i < PIECES) kr[i] = fetch_keys32<D>(x.codes, x.at & (block - 1), (wave + 4 * i) / C, (wave + 4 * i) % C);
    };
    const auto fetch_v = [&](const Step &x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MINE; ++i)
            if (wave + 4 * i < PIECES)
                vr[i] = fetch_values32<D>(x.codes, a.cache.block_log2, x.at & (block - 1), (wave + 4 * i) / C, (wave + 4 * i) % C);
    };
    // keys: operand 2h + b of half t; values: operand b of half t and channels 32h..
    const auto put_k = [&](int buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MINE; ++i)
            if (wave + 4 * i < PIECES) {
                key_rows[buffer][2 * (wave + 4 * i)][lane] = codes_f16(kr[i].x, kr[i].y);
                key_rows[buffer][2 * (wave + 4 * i) + 1][lane] = codes_f16(kr[i].z, kr[i].w);
            }
    };
    const auto put_v = [&](int buffer, const Step &x) __attribute__((always_inline)) {
        unit = fmaxf(unit, x.step_v);
        const float ratio = ratio_of(x.step_v, unit);  // as `reach` has it
        const _Float16 h = static_cast<_Float16>(ratio), b = static_cast<_Float16>(-1152.0f * ratio);
#pragma unroll
        for (int i = 0; i < MINE; ++i)
            if (wave + 4 * i < PIECES) {
                value_rows[buffer][2 * (wave + 4 * i)][lane] = codes_f16(vr[i].x, vr[i].y, f16x2{h, h}, f16x2{b, b});
                value_rows[buffer][2 * (wave + 4 * i) + 1][lane] = codes_f16(vr[i].z, vr[i].w, f16x2{h, h}, f16x2{b, b});
            }
    };
    const auto together = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    float w[32], f = 0.0f;
    u32x4 pw[4][P];
    // S^T; operands of the next products are on their way while some run (the barriers to the compiler's order keep them there)
    const auto scores = [&](const u32x4 (*keys)[64]) __attribute__((always_inline)) {
        f32x16 d[2];
        const f32x16 zeros = {};
        u32x4 x[3][2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) x[j][i] = keys[i * QV + j][lane];
#pragma unroll
        for (int j = 0; j < QV; ++j) {
            if (j + 2 < QV) {
#pragma unroll
                for (int i = 0; i < 2; ++i) x[(j + 2) % 3][i] = keys[i * QV + j + 2][lane];
            }
#pragma unroll
            for (int p = P - 1; p >= 0; --p)
#pragma unroll
                for (int i = 0; i < 2; ++i) d[i] = product(x[j % 3][i], q.f[j][p], j == 0 && p == P - 1 ? zeros : d[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = d[i / 16][i % 16];
    };
    // O^T
    const auto meet = [&](const u32x4 (*values)[64], float step_v) __attribute__((always_inline)) {
        r.reach(step_v);
        // operand b of half t and channels 32h.. stands at 2 (C t + h) + b
        u32x4 y[2][C];
#pragma unroll
        for (int h = 0; h < C; ++h) y[0][h] = values[2 * h][lane];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (u < 3) {
#pragma unroll
                for (int h = 0; h < C; ++h) y[(u + 1) & 1][h] = values[2 * (C * ((u + 1) / 2) + h) + ((u + 1) & 1)][lane];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = P - 1; p >= 0; --p)
#pragma unroll
                for (int h = 0; h < C; ++h) r.acc[h] = product(y[u & 1][h], pw[u][p], r.acc[h]);
        }
    };
    // ---- the first step's operands; the second's codes on their way
    Step now = next(), then = {false, nullptr, 0, 0.0f, 0.0f};
    if (now.is) {
        fetch_k(now);
        fetch_v(now);
        put_k(0);
        put_v(0, now);
        then = next();
        if (then.is) {
            fetch_k(then);
            fetch_v(then);
        }
    }
    Step after;
    int buffer = 0;
    // the workgroup's part of a step: the next one's operands to the other buffers, the codes behind them on their way
    const auto share = [&]() __attribute__((always_inline)) {
        together();
        after = {false, nullptr, 0, 0.0f, 0.0f};
        if (!then.is) return;
        put_k(buffer ^ 1);
        put_v(buffer ^ 1, then);
        after = next();
        if (after.is) {
            fetch_k(after);
            fetch_v(after);
        }
    };
    const auto advance = [&]() __attribute__((always_inline)) {
        now = then;
        then = after;
        buffer ^= 1;
    };
    if (r0 >= t.nrows) {  // no rows for this wave
        for (; now.is; advance()) share();
        return;
    }
    for (; now.is; advance()) {
        share();
        scores(key_rows[buffer]);
        f = score_unit(q.unit, now.step_k);
        if (t.cut(now.at)) r.hide(w, now.at, q.sight, t.sinks);
        r.settle(w, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.weigh(i, w, f, pw);
        meet(value_rows[buffer], now.step_v);
    }
    if (r.again) {
        for (int i = r0; i < min(r0 + 32, t.nrows); ++i) row_by_keys<T, D>(a, t, split, 1, i, kvh);
        return;
    }
    float y[D / 2];
#pragma unroll
    for (int e = 0; e < D / 2; ++e) y[e] = r.acc[e / 16][e % 16];
    put<T, D, 32>(a, t, split, r0 + c, kvh, y, r.base, column_sum<32>(r.sum), r.unit);
}

// The pieces' weights: shares of the whole, so that means of finite values stay finite.  Parts are divided by their sums,
// zeros where there were no keys; a sum that is a NaN is not 0 and stays.
constexpr int kFewPieces = 16;

// Joins up to N pieces (8 or kFewPieces) of each (row, head), in their order: D / 4 lanes of four channels each, and each for itself the
// pieces' weights (2,048 rows x 16 heads x 64 in two pieces: 19 us with a wave for each).  Places of all pieces that there may be are
// fetched at once; those that a row has not, as its first one says, are left out.
template <class T, int D, int N>
__global__ void __launch_bounds__(256) cache_join_few_kernel(AttendArgs a) {
    constexpr int LANES = D == 32 ? 8 : D == 64 ? 16 : 32;
    const int lane = threadIdx.x & (LANES - 1);
    const int64_t cell = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    const int64_t cells = a.total_q * a.heads;
    if (cell >= cells || 4 * lane >= D) return;
    const int64_t row = cell / a.heads;
    const int head = static_cast<int>(cell - row * a.heads);
    if (row < a.q_starts[0] || row >= a.q_starts[a.sequences]) return;  // no sequence's (its pieces hold anything)
    float4 ml[N];
    f32x4 x[N];
#pragma unroll
    for (int p = 0; p < N; ++p) {
        const int64_t at = min(p, a.splits - 1) * cells + cell;
        ml[p] = a.part_ml[at];
        x[p] = *reinterpret_cast<const f32x4 *>(a.part_o + at * D + 4 * lane);
    }
    const int pieces = static_cast<int>(ml[0].w);
    float4 top = sum_of(neg_inf(), 0.0f, 0.0f, 0.0f);
    float w[N], total = 0.0f;
#pragma unroll
    for (int p = 0; p < N; ++p)
        if (p < pieces && ml[p].z != 0.0f && above_of(ml[p], top)) top = ml[p];
#pragma unroll
    for (int p = 0; p < N; ++p) {
        w[p] = p < pieces && ml[p].z != 0.0f ? weight_of(ml[p], top) * ml[p].z : 0.0f;
        total += w[p];
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    f32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int p = 0; p < N; ++p)
        if (p < pieces) o += x[p] * (w[p] * inv);
    T *to = static_cast<T *>(a.o) + row * a.o_stride + static_cast<int64_t>(head) * D + 4 * lane;
    if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2 *>(to) = u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
    else *reinterpret_cast<f32x4 *>(to) = o;
    if (a.lse && lane == 0) a.lse[cell] = log_of(top.x, top.y, total);
}

// Joins up to 64 pieces of each (row, head): a workgroup each, whose waves take a quarter of the pieces, all on their way at once.
template <class T, int D>
__global__ void __launch_bounds__(256) cache_join_kernel(AttendArgs a) {
    constexpr int N = 16;
    __shared__ float part[4][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t cell = blockIdx.x, cells = a.total_q * a.heads, row = cell / a.heads;
    const int head = static_cast<int>(cell - row * a.heads);
    // a lane for each piece: its weight
    const float4 none = sum_of(neg_inf(), 0.0f, 0.0f, 0.0f);
    float4 mine = lane < a.splits ? a.part_ml[lane * cells + cell] : none;
    float x[N][2];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e)
            x[u][e] = N * wave + u < a.splits && lane + 64 * e < D ? a.part_o[((N * wave + u) * cells + cell) * D + lane + 64 * e] : 0.0f;
    if (row < a.q_starts[0] || row >= a.q_starts[a.sequences]) return;  // no sequence's (its pieces hold anything)
    const int pieces = static_cast<int>(as_float(__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, mine.w))));
    if (lane >= pieces) mine = none;
    float4 top = mine.z != 0.0f ? mine : none;
    for (int d = 1; d < 64; d <<= 1) {
        const float4 other = sum_of(__shfl_xor(top.x, d, 64), __shfl_xor(top.y, d, 64), 0.0f, 0.0f);
        if (above_of(other, top)) top = other;
    }
    const float w = mine.z != 0.0f ? weight_of(mine, top) * mine.z : 0.0f;
    float total = w, o[2] = {0.0f, 0.0f};
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d, 64);
    const float share = total == 0.0f ? 0.0f : w / total;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const float wp = __shfl(share, N * wave + u, 64);
#pragma unroll
        for (int e = 0; e < 2; ++e) o[e] += N * wave + u < pieces ? wp * x[u][e] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) part[wave][e][lane] = o[e];
    __syncthreads();
    if (wave != 0) return;
    T *to = static_cast<T *>(a.o) + row * a.o_stride + static_cast<int64_t>(head) * D;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < D)
            store_from_f32<T>(to + lane + 64 * e, (part[0][e][lane] + part[1][e][lane]) + (part[2][e][lane] + part[3][e][lane]));
    if (a.lse && lane == 0) a.lse[cell] = log_of(top.x, top.y, total);
}

// How a call is cut: by sequences' mean rows into tiles of 16 or 32 (four waves share a tile's keys) or of 128 (four waves share
// its rows), an upper bound of each, as the lengths are on the device; and every tile's keys over as many workgroups as run at once:
// two a compute unit, three for tiles of 128 up to 64 channels (1,300 rows of 12 x 64 over 3,000 keys: 44 us with two for 32), with at
// least four steps of keys each, two in tiles of 128, whose waves each take all of them.  (Powers of two alone: 500 rows of 8 x 4 x 128
// over 6,000 keys 116 us for 87, 3 rows of 12 x 128 over 30,000 each 74 for 59.)
struct Cut {
    int64_t tile_groups;
    int32_t splits, rows;  // of a tile
    int32_t slots;         // workgroups for each key head, shared out by lengths among up to `splits` pieces a tile (0: no such cut)
    bool at_once;          // all workgroups run at once (of sequences of one length; three a unit up to 64 channels, two beyond)
};
Cut cut_of(int64_t total_q, int32_t heads, int32_t kv_heads, int64_t sequences, int64_t max_k, int32_t window, int32_t sinks, int32_t head_dim) {
    const int64_t rows = total_q * (heads / kv_heads), each = std::max<int64_t>(sequences, 1), per = (rows + each - 1) / each;
    const int64_t keys = window ? std::min<int64_t>(max_k, static_cast<int64_t>(window) + sinks + per + 2 * kStep) : max_k;
    // workgroups (of sequences of one length, which take fewer tiles than the bound)
    const auto groups_of = [&](int32_t tile) { return std::max<int64_t>(each * ((per + tile - 1) / tile) * kv_heads, 1); };
    // 32 rows, too, where tiles of 128 with four steps a piece would leave compute units without one
    const int32_t tile = per <= 16 ? 16 : per <= 64 || groups_of(128) * std::max<int64_t>(keys / (4 * kStep), 1) < 256 ? 32 : 128;
    const int64_t groups = groups_of(tile), most = 256 * (tile == 128 && head_dim <= 64 ? 3 : 2);
    int32_t splits = static_cast<int32_t>(std::clamp<int64_t>(std::min(most / groups, keys / ((tile == 128 ? 2 : 4) * kStep)), 1, 64));
    // single rows of several sequences share workgroups out by length, the long ones up to twice as many as if all were alike, as long
    // as few are joined, and from 160 MB of codes on (about 30 us).  8 rows over 65,536 keys at most, 32 / 8 heads x 128: lengths
    // apart 139 us without for 121, alike 190 for 193; 16 x 12 heads x 64 over 8,192 at most 34 for 29; below, 24 x 3,000 x 8 x 32
    // 17.5 without for 19.6.
    int64_t slots = 0;
    if (tile == 16 && splits > 1 && splits <= kFewPieces / 2 && sequences > 1 && sequences <= 64 && groups * keys * 2 * head_dim >= (INT64_C(160) << 20)) {
        slots = std::max(most / kv_heads, rows / tile + sequences);
        splits = static_cast<int32_t>(std::min<int64_t>(2 * splits, keys / (4 * kStep)));
    }
    // few pieces join faster, a wave's lanes for several rows
    if (tile > 16 && splits > kFewPieces && splits < 2 * kFewPieces) splits = kFewPieces;
    return {rows / tile + sequences, splits, tile, static_cast<int32_t>(slots), groups * splits <= most};
}

using AttendFn = void (*)(AttendArgs);
template <class T, int D>
AttendFn pick_tile(const Cut &cut) {
    return cut.rows == 16 ? cache_rows_kernel<T, D, 16> : cut.rows == 32 ? cache_rows_kernel<T, D, 32> : cache_chunk_kernel<T, D>;
}
template <class T>
AttendFn pick_attend(int32_t d, const Cut &cut) {
    return d == 32 ? pick_tile<T, 32>(cut) : d == 64 ? pick_tile<T, 64>(cut) : d == 96 ? pick_tile<T, 96>(cut) : pick_tile<T, 128>(cut);
}
template <class T, int D>
AttendFn pick_join_of(int32_t pieces) {
    return pieces <= 8 ? cache_join_few_kernel<T, D, 8> : pieces <= kFewPieces ? cache_join_few_kernel<T, D, kFewPieces> : cache_join_kernel<T, D>;
}
template <class T>
AttendFn pick_join(int32_t d, int32_t pieces) {
    return d == 32 ? pick_join_of<T, 32>(pieces) : d == 64 ? pick_join_of<T, 64>(pieces) : d == 96 ? pick_join_of<T, 96>(pieces) : pick_join_of<T, 128>(pieces);
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
        const Cut cut = cut_of(total_q, heads, cache->kv_heads, sequences, max_k, window, sinks, cache->head_dim);
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
        // (a query's unit stays within float32's range)
        require(softmax_scale > 0.0f && softmax_scale < 8192.0f, "softmax_scale must be above 0 and below 2^13");
        if (total_q == 0 || sequences == 0) return;
        for (const auto &[p, stride] : {std::pair(q, q_stride), std::pair(static_cast<const void *>(o), o_stride)}) {
            require(p && aligned(p, 16), "a row pointer is NULL or not 16-byte aligned");
            require(stride >= static_cast<int64_t>(heads) * cache->head_dim, "a row stride is shorter than its heads");
            require(stride <= (INT64_C(1) << 40) && stride * dtype_size(dtype) % 16 == 0,
                    "a row stride must be whole 16-byte pieces, at most 2^40 elements");
        }
        require(q_starts && aligned(q_starts, 4), "starts is NULL or not aligned");
        require(!lse || aligned(lse, 4), "lse is not aligned");
        const Cut cut = cut_of(total_q, heads, cache->kv_heads, sequences, max_k, window, sinks, cache->head_dim);
        AttendArgs a = {view_of(cache, table, table_stride, lengths), q, o, lse, q_starts, total_q, q_stride, o_stride, sequences,
                        heads, heads / cache->kv_heads, flags & S3DX_BLOCK_CAUSAL, window, sinks, cut.splits,
                        static_cast<int32_t>(cut.tile_groups), cut.at_once, cut.slots, softmax_scale, nullptr, nullptr};
        if (cut.splits > 1) {
            require(workspace && aligned(workspace, 16), "workspace is NULL or not 16-byte aligned");
            Carver w(workspace, workspace_bytes);
            a.part_o = w.take<float>(static_cast<uint64_t>(cut.splits) * total_q * heads * cache->head_dim);
            a.part_ml = w.take<float4>(static_cast<uint64_t>(cut.splits) * total_q * heads);
        }
        const int64_t grid = cut.slots ? static_cast<int64_t>(cut.slots) * cache->kv_heads : cut.tile_groups * cache->kv_heads * cut.splits;
        require(grid <= 0xffffffffll / 256, "too many rows and sequences");
        const bool bf = dtype == S3DX_BF16;
        (bf ? pick_attend<uint16_t>(cache->head_dim, cut) : pick_attend<float>(cache->head_dim, cut))<<<
            dim3(static_cast<unsigned>(grid)), dim3(256), 0, as_stream(stream)>>>(a);
        launch_check("cache attention");
        if (cut.splits > 1) {
            const bool few = cut.splits <= kFewPieces;
            const int64_t cells = total_q * heads, each = !few ? 1 : cache->head_dim == 32 ? 32 : cache->head_dim == 64 ? 16 : 8;
            require((cells + each - 1) / each <= 0xffffffffll / 256, "too many rows and heads");
            (bf ? pick_join<uint16_t>(cache->head_dim, cut.splits) : pick_join<float>(cache->head_dim, cut.splits))<<<
                dim3(static_cast<unsigned>((cells + each - 1) / each)), dim3(256), 0, as_stream(stream)>>>(a);
            launch_check("cache attention join");
        }
    });
}

}  // extern "C"
