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
    float4 *part_ml;  // [splits][total_q][heads]: see Sum
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
// From 2^20 on a base is kept in two parts (lo: what hi is rounded by, and the 7), so that scores of any size have weights
// as exact as their difference.
constexpr float kUnder = 7.0f, kReach = 15.0f, kFar = 0x1p20f;

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

// Attention of a tile of 16 NS rows (query rows times the heads that share a key head).  A
// wave computes S^T = K Q^T and O^T = V^T P^T, so that what one product leaves in a
// lane is what the next one wants there.  A 16x16 product leaves lane (c, g) = (lane & 15, lane >> 4) with rows 4g..4g+3 of
// column c; product t of a step takes key 16 (c >> 2) + 4t + (c & 3) as its row c, so that lane
// (c, g) gets keys 16g + 4t + i of query c: the lane's 16 weights are of keys 16g..16g+15, and the
// values' operand wants the same keys of a channel: one 16-byte piece of the cache, as it lies.
// The keys' operand wants channels of a row, in any order that the queries share: 16 side by side for two products.
// So codes go from memory to a product's registers through two instructions for every four, without LDS.
//
// SHARES 4: the workgroup's waves take every fourth step of a tile each, and join through LDS; 1: a tile each.
template <class T, int D, int NS, int SHARES>
__global__ void __launch_bounds__(256, 2) cache_attend_kernel(AttendArgs a) {
    constexpr bool BF = sizeof(T) == 2;
    constexpr int P = BF ? 1 : 2;      // half-precision terms of a query's channel and of a weight
    constexpr int ROWS = 16 * NS, KT = kStep / 16;
    constexpr int QV = D / 32, C = D / 16;
    constexpr int KD = D / 16;         // dwords of a key row that a lane reads
    __shared__ float part[SHARES == 4 ? 4 : 1][SHARES == 4 ? NS * 4 * C : 1][64];
    __shared__ float4 part_ml[SHARES == 4 ? 4 : 1][NS][16];
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // consecutive workgroups of one XCD run neighbouring tiles of a head: its L2 holds their keys
    const int id = xcd_tile(blockIdx.x, gridDim.x);
    const int split = id / a.tile_groups % a.splits, kvh = id / a.tile_groups / a.splits;
    const int64_t tg = id % a.tile_groups, tile = SHARES == 4 ? tg : tg * 4 + wave;
    const int64_t s = sequence_of_unit(a.q_starts, a.sequences, a.total_q, a.group, ROWS == 64 ? 6 : ROWS == 32 ? 5 : 4, tile);
    const Span qs = sequence_span(a.q_starts, s, a.total_q);
    const int64_t first_row = (tile - (qs.begin * a.group / ROWS + s)) * ROWS;
    const int nrows = qs.rows * a.group;  // total_q * heads < 2^31
    if (first_row < 0 || first_row >= nrows) return;  // SHARES 4: the whole workgroup
    const int r0 = static_cast<int>(first_row);
    const int tok0 = r0 / a.group, last = (min(r0 + ROWS, nrows) - 1) / a.group;
    const int keys = cached_rows(a.cache, s), lag = keys - qs.rows;
    const int piece = split * SHARES + (SHARES == 4 ? wave : 0), pieces = a.splits * SHARES;

    // keys below `most` are seen by some row, below `least` by all as far as the causal end goes; from `low` on by some, from
    // `low_all` on by all as far as the window's beginning goes
    const int most = a.causal ? max(0, min(keys, last + lag + 1)) : keys;
    const int least = a.causal ? max(0, min(keys, tok0 + lag + 1)) : keys;
    const int low = a.window ? max(0, tok0 + lag - a.window + 1) : 0, low_all = a.window ? max(0, last + lag - a.window + 1) : 0;
    // steps: those of the first keys that stay visible, then from the window's beginning on
    const int end = (most + kStep - 1) / kStep, sink_steps = min(end, (a.sinks + kStep - 1) / kStep);
    const int skip = max(0, low / kStep - sink_steps), steps = sink_steps + max(0, end - sink_steps - skip);

    // ---- this lane's query of each set of 16
    int lim[NS], from[NS];  // it sees keys [from, lim) and those before a.sinks
    u32x4 qf[NS][QV][P];
    float fq[NS];           // binary orders of a score for each unit of its product, before the keys' step
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const int r = min(r0 + 16 * n + c, nrows - 1), tok = r / a.group;
        lim[n] = a.causal ? max(0, min(keys, tok + lag + 1)) : keys;
        from[n] = a.window ? tok + lag - a.window + 1 : 0;
        const T *q = static_cast<const T *>(a.q) + (qs.begin + tok) * a.q_stride + static_cast<int64_t>(kvh * a.group + r % a.group) * D;
        float x[QV][8];
        uint32_t big = 0;
#pragma unroll
        for (int j = 0; j < QV; ++j) {
            // products 2h and 2h + 1: channels 64h + 16g.., 64h + 16g + 8..; a last one by itself: 8g.. of the last 32
            const T *qj = q + (j == QV - 1 && QV % 2 ? 32 * j + 8 * g : 64 * (j / 2) + 16 * g + 8 * (j & 1));
            constexpr int N = 8 * static_cast<int>(sizeof(T)) / 16;
            uint4 t[N];
#pragma unroll
            for (int i = 0; i < N; ++i) t[i] = reinterpret_cast<const uint4 *>(qj)[i];
            const uint32_t *w = reinterpret_cast<const uint32_t *>(t);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t u = BF ? (e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16) : w[e];
                x[j][e] = as_float(u);
                big = max(big, u & 0x7fffffffu);
            }
        }
        // the row's power: its largest magnitude to [2^14, 2^15).  Magnitudes' bits rise with them, infinities and NaN above all;
        // their rows keep them, and give NaN.
        big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), 16, 64)));
        big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), 32, 64)));
        const int e = min(max(static_cast<int>(big >> 23) - 127, -100), 127);
        fq[n] = ldexpf(a.scale * kLog2e, e - 14);
#pragma unroll
        for (int j = 0; j < QV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = ldexpf(x[j][2 * i], 14 - e), v = ldexpf(x[j][2 * i + 1], 14 - e);
                qf[n][j][0][i] = pack_f16x2(u, v);
                if constexpr (P == 2) {
                    const f32x2 t = unpack_f16x2(qf[n][j][0][i]);
                    qf[n][j][1][i] = pack_f16x2(u - t[0], v - t[1]);
                }
            }
    }

    // ---- this wave's steps: pages and steps of 64 of them at a time, one a lane
    int it = -1, pages = 0, page = 0, k0 = 0, at = 0;
    float2 sizes = make_float2(0.0f, 0.0f);
    float step_k = 0.0f, step_v = 0.0f;
    const auto key_of = [&](int i) { return (i < sink_steps ? i : i + skip) * kStep; };
    const auto next = [&]() __attribute__((always_inline)) {  // false: none left
        for (;;) {
            ++it;
            const int i = piece + it * pieces;
            if (i >= steps) return false;
            if ((it & 63) == 0) {
                const int mine = i + lane * pieces;
                pages = mine < steps ? page_of(a.cache, s, key_of(mine) >> a.cache.block_log2) : -1;
                sizes = pages >= 0 ? a.cache.steps[static_cast<int64_t>(pages) * a.cache.kv_heads + kvh] : make_float2(0.0f, 0.0f);
            }
            page = __builtin_amdgcn_readlane(pages, it & 63);
            if (page < 0) continue;  // no such page: its keys count for nothing
            k0 = key_of(i);
            return true;
        }
    };
    const int block = 1 << a.cache.block_log2;
    uint32_t kr[KT][KD], vr[C][4];
    const int kat = (16 * (c >> 2) + (c & 3)) * D, vat = (c << a.cache.block_log2) + 16 * g;
    const uint8_t *codes = nullptr;
    const auto place = [&]() __attribute__((always_inline)) {
        codes = a.cache.codes + ((static_cast<int64_t>(page) * a.cache.kv_heads + kvh) << (a.cache.block_log2 + 1)) * D;
    };
    const auto load_k = [&]() __attribute__((always_inline)) {
        const uint8_t *p = codes + (k0 & (block - 1)) * D;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
#pragma unroll
            for (int h = 0; h < KD / 4; ++h) {
                const uint4 w = *reinterpret_cast<const uint4 *>(p + kat + 4 * t * D + 64 * h + 16 * g);
                kr[t][4 * h] = w.x, kr[t][4 * h + 1] = w.y, kr[t][4 * h + 2] = w.z, kr[t][4 * h + 3] = w.w;
            }
            if constexpr (KD % 4 != 0) {
                const uint2 w = *reinterpret_cast<const uint2 *>(p + kat + 4 * t * D + 64 * (KD / 4) + 8 * g);
                kr[t][KD - 2] = w.x, kr[t][KD - 1] = w.y;
            }
        }
    };
    const auto load_v = [&]() __attribute__((always_inline)) {
        const uint8_t *p = codes + block * D + (k0 & (block - 1));
#pragma unroll
        for (int t = 0; t < C; ++t) {
            const uint4 w = *reinterpret_cast<const uint4 *>(p + vat + (t << (a.cache.block_log2 + 4)));
            vr[t][0] = w.x, vr[t][1] = w.y, vr[t][2] = w.z, vr[t][3] = w.w;
        }
    };

    // ---- state
    f32x4 acc[NS][C];  // in units of `unit`, the largest step of values met
    float sum[NS], hi[NS], lo[NS], above[NS];  // above: the score from which on the base moves (-inf: nothing seen yet)
    float unit = 0.0f;
    bool far = false;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        sum[n] = hi[n] = lo[n] = 0.0f;
        above[n] = neg_inf();
#pragma unroll
        for (int t = 0; t < C; ++t) acc[n][t] = f32x4{0, 0, 0, 0};
    }

    bool more = next();
    if (more) {
        place();
        load_k();
        load_v();
    }
    while (more) {
        step_k = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, sizes.x), it & 63));
        step_v = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, sizes.y), it & 63));
        at = k0;
        // ---- S^T
        f32x4 w[NS][KT];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int t = 0; t < KT; ++t) w[n][t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int j = 0; j < QV; ++j) {
                const u32x4 x = codes_f16(kr[t][2 * j], kr[t][2 * j + 1]);
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int p = P - 1; p >= 0; --p) w[n][t] = product(x, qf[n][j][p], w[n][t]);
            }
        more = next();
        if (more) {
            place();
            load_k();
        }
        // ---- weights
        const bool cut = at + kStep > least || (at < low_all && at + kStep > a.sinks);
        u32x4 pw[NS][KT / 2][P];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            if (cut) {
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = at + 16 * g + 4 * t + i;
                        if (key >= lim[n] || (key < from[n] && key >= a.sinks)) w[n][t][i] = neg_inf();
                    }
            }
            const float f = fq[n] * step_k;
            float mx = neg_inf();
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, w[n][t][i]);
            if (__builtin_amdgcn_ballot_w64(mx != neg_inf() && mx * f > above[n]) != 0) {
                mx = max_over_groups(mx);
                const bool over = mx != neg_inf() && mx * f > above[n];
                float h = mx * f, l = fmaf(mx, f, -h) - kUnder;
                if (fabsf(h) < kFar) {
                    h += l;
                    l = 0.0f;
                }
                const float alpha = !over ? 1.0f : above[n] == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f((hi[n] - h) + (lo[n] - l));
                sum[n] *= alpha;
#pragma unroll
                for (int t = 0; t < C; ++t) acc[n][t] *= alpha;
                if (over) {
                    hi[n] = h;
                    lo[n] = l;
                    above[n] = h + (l + kReach);
                }
                far = far || __builtin_amdgcn_ballot_w64(lo[n] != 0.0f) != 0;
            }
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = fmaf(w[n][t][i], f, -hi[n]);
                    if (far) x -= lo[n];
                    if (cut && w[n][t][i] == neg_inf()) x = neg_inf();
                    w[n][t][i] = __builtin_amdgcn_exp2f(x);
                }
            // their sum in 32 bits, before they are rounded
#pragma unroll
            for (int t = 0; t < KT; ++t) sum[n] += (w[n][t][0] + w[n][t][1]) + (w[n][t][2] + w[n][t][3]);
            // half precision keeps 11 bits of a weight (2^-11 off at most), two terms 22
#pragma unroll
            for (int u = 0; u < KT / 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = w[n][2 * u + (i >> 1)][2 * (i & 1)], y = w[n][2 * u + (i >> 1)][2 * (i & 1) + 1];
                    pw[n][u][0][i] = pack_f16x2(x, y);
                    if constexpr (P == 2) {
                        const f32x2 t = unpack_f16x2(pw[n][u][0][i]);
                        pw[n][u][1][i] = pack_f16x2(x - t[0], y - t[1]);
                    }
                }
        }
        // ---- O^T.  Values count in units of the largest step met; a smaller one's ratio goes into its codes (down to 2^-24 they
        // stay exact), or, smaller still, into their products.
        if (step_v > unit) {
            const float ratio = unit / step_v;  // powers of two, or 0
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int t = 0; t < C; ++t) acc[n][t] *= ratio;
            unit = step_v;
        }
        const float ratio = unit > 0.0f ? step_v / unit : 0.0f;
        if (ratio >= 0x1p-24f) {
            const _Float16 r = static_cast<_Float16>(ratio), b = static_cast<_Float16>(-1152.0f * ratio);
#pragma unroll
            for (int t = 0; t < C; ++t)
#pragma unroll
                for (int u = 0; u < KT / 2; ++u) {
                    const u32x4 x = codes_f16(vr[t][2 * u], vr[t][2 * u + 1], f16x2{r, r}, f16x2{b, b});
#pragma unroll
                    for (int n = 0; n < NS; ++n)
#pragma unroll
                        for (int p = P - 1; p >= 0; --p) acc[n][t] = product(x, pw[n][u][p], acc[n][t]);
                }
        } else if (ratio > 0.0f) {
#pragma unroll
            for (int t = 0; t < C; ++t)
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    f32x4 d = {0, 0, 0, 0};
#pragma unroll
                    for (int u = 0; u < KT / 2; ++u)
#pragma unroll
                        for (int p = P - 1; p >= 0; --p) d = product(codes_f16(vr[t][2 * u], vr[t][2 * u + 1]), pw[n][u][p], d);
                    acc[n][t] += d * ratio;
                }
        }
        if (more) load_v();
    }

    // ---- out
    const bool parts = a.splits > 1;
    const auto finish = [&](int n, const float (&y)[4 * C], float h, float l, float total, float u) __attribute__((always_inline)) {
        const int r = r0 + 16 * n + c;
        if (r >= nrows) return;
        const int64_t token = qs.begin + r / a.group;
        const int head = kvh * a.group + r % a.group;
        // divided by the sum before the unit, so that means of finite values are finite
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        const int64_t cell = token * a.heads + head;
        if (parts) {
            float *to = a.part_o + (split * a.total_q * a.heads + cell) * D;
#pragma unroll
            for (int t = 0; t < C; ++t)
                *reinterpret_cast<f32x4 *>(to + 16 * t + 4 * g) =
                    f32x4{y[4 * t] * inv * u, y[4 * t + 1] * inv * u, y[4 * t + 2] * inv * u, y[4 * t + 3] * inv * u};
            if (g == 0) a.part_ml[split * a.total_q * a.heads + cell] = sum_of(h, l, total, 1.0f);
            return;
        }
        T *to = static_cast<T *>(a.o) + token * a.o_stride + static_cast<int64_t>(head) * D;
#pragma unroll
        for (int t = 0; t < C; ++t) {
            const f32x4 z = {y[4 * t] * inv * u, y[4 * t + 1] * inv * u, y[4 * t + 2] * inv * u, y[4 * t + 3] * inv * u};
            if constexpr (BF) *reinterpret_cast<u32x2 *>(to + 16 * t + 4 * g) = u32x2{pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3])};
            else *reinterpret_cast<f32x4 *>(to + 16 * t + 4 * g) = z;
        }
        if (a.lse && g == 0) a.lse[cell] = log_of(h, l, total);
    };
    if constexpr (SHARES == 1) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            float y[4 * C];
#pragma unroll
            for (int e = 0; e < 4 * C; ++e) y[e] = acc[n][e / 4][e % 4];
            finish(n, y, hi[n], lo[n], sum_over_groups(sum[n]), unit);
        }
    } else {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int t = 0; t < C; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave][(n * C + t) * 4 + i][lane] = acc[n][t][i];
            const float l = sum_over_groups(sum[n]);
            if (g == 0) part_ml[wave][n][c] = sum_of(hi[n], lo[n], l, unit);
        }
        __syncthreads();
        for (int n = wave; n < NS; n += 4) {
            float4 top = sum_of(neg_inf(), 0.0f, 0.0f, 0.0f);
            float u = 0.0f, total = 0.0f, y[4 * C];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float4 m = part_ml[p][n][c];
                if (m.z != 0.0f && above_of(m, top)) top = m;
                u = fmaxf(u, m.w);
            }
#pragma unroll
            for (int e = 0; e < 4 * C; ++e) y[e] = 0.0f;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float4 m = part_ml[p][n][c];
                const float wgt = m.z == 0.0f ? 0.0f : weight_of(m, top), scaled = m.w > 0.0f ? wgt * (m.w / u) : wgt * 0.0f;
                total += wgt * m.z;
#pragma unroll
                for (int e = 0; e < 4 * C; ++e) y[e] += scaled * part[p][n * 4 * C + e][lane];
            }
            finish(n, y, top.x, top.y, total, u);
        }
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

// How a call is cut: tiles of 16, 32 or 64 rows as sequences fill them (an upper bound, as the lengths are on the device); four
// waves to a tile, and several workgroups, where there would be fewer than two waves for each SIMD, with at least
// four steps a wave.
struct Cut {
    int64_t tile_groups;
    int32_t splits, sets, shares;
};
Cut cut_of(int64_t total_q, int32_t heads, int32_t kv_heads, int32_t d, int64_t sequences, int64_t max_k, int32_t window, int32_t sinks) {
    constexpr int64_t kWaves = 256 * 4 * 2;
    const int64_t rows = total_q * (heads / kv_heads), per = rows / std::max<int64_t>(sequences, 1);
    const int32_t sets = per <= 16 ? 1 : per <= 32 || d > 64 ? 2 : 4;
    const int64_t tiles = rows / (16 * sets) + sequences, waves = std::max<int64_t>(tiles * kv_heads, 1);
    const int64_t keys = window ? std::min<int64_t>(max_k, static_cast<int64_t>(window) + sinks + per + 2 * kStep) : max_k;
    const int32_t shares = waves >= kWaves || keys <= kStep ? 1 : 4;
    int32_t splits = 1;
    if (shares == 4)
        while (splits < 64 && waves * 4 * splits * 2 <= kWaves && keys >= 4 * kStep * 4 * splits) splits *= 2;
    return {shares == 4 ? tiles : (tiles + 3) / 4, splits, sets, shares};
}

using AttendFn = void (*)(AttendArgs);
template <class T, int D>
AttendFn pick_tile(const Cut &cut) {
    // float32's wide heads: two terms of 32 rows do not fit a lane's registers
    constexpr int MOST = sizeof(T) == 4 ? (D > 64 ? 1 : 2) : D > 64 ? 2 : 4;
    const bool all = cut.shares == 4;
    if constexpr (MOST >= 4)
        if (cut.sets == 4) return all ? cache_attend_kernel<T, D, 4, 4> : cache_attend_kernel<T, D, 4, 1>;
    if constexpr (MOST >= 2)
        if (cut.sets == 2) return all ? cache_attend_kernel<T, D, 2, 4> : cache_attend_kernel<T, D, 2, 1>;
    return all ? cache_attend_kernel<T, D, 1, 4> : cache_attend_kernel<T, D, 1, 1>;
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
        Cut cut = cut_of(total_q, heads, cache->kv_heads, cache->head_dim, sequences, max_k, window, sinks);
        // fewer rows of float32 a tile than of bfloat16: more tiles
        const int32_t most = dtype == S3DX_BF16 ? 4 : cache->head_dim > 64 ? 1 : 2;
        if (cut.sets > most) {
            const int64_t tiles = total_q * (heads / cache->kv_heads) / (16 * most) + sequences;
            cut.sets = most;
            cut.tile_groups = cut.shares == 4 ? tiles : (tiles + 3) / 4;
        }
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
