// Attention over key blocks that a cheap score selects for each query: the
// 8-bit index of the blocks' mean keys, the selection, and the attention over
// the selected blocks or all of them (the transformer blocks of the SLat flow,
// slat_flow_graph.cpp:304-434, and the decoders' windows,
// gs_decoder_graph.cpp:93-121, which the reference runs as dense attention).
#include <cmath>
#include <type_traits>

#include "common.hpp"

namespace s3dx {
namespace {

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

// ---------------------------------------------------------------------------
// 8-bit codes.  2^e <= most < 2^(e+1): x * 2^(6-e) is exact, the rounding to a
// whole number is the only one, and 127.5 and more is cut to 127.
// ---------------------------------------------------------------------------
__device__ __forceinline__ bool codes_fine(double most) {
    return most >= 0x1p-100 && most < __builtin_inf();
}
__device__ __forceinline__ int exponent_of(double most) {
    return static_cast<int>((__builtin_bit_cast(uint64_t, most) >> 52) & 0x7ffu) - 1023;
}
__device__ __forceinline__ double two_to(int e) {
    return __builtin_bit_cast(double, static_cast<uint64_t>(e + 1023) << 52);
}
__device__ __forceinline__ int code_of(double x, double up) {
    return max(-127, min(127, static_cast<int>(rint(x * up))));
}

struct IndexArgs {
    const void *k;
    const int32_t *k_starts;
    int64_t total_k, k_stride, sequences, rows;
    int32_t kv_heads, d, block, block_log2;
    int8_t *codes;
    float *scale;
};

// One workgroup per index row and up to 256 channels (whole heads): 32 lanes read a
// row's channels, 8 each, eight rows at a time; sums in 64 bits, so that their order does
// not show in a code.  The work is reading the keys once.
template <class T>
__global__ void __launch_bounds__(256) index_kernel(IndexArgs a) {
    __shared__ double sums[8][256];
    __shared__ uint64_t most[8];
    const int tid = threadIdx.x, lane = tid & 31, part = tid >> 5;
    const int per = 256 / a.d;  // heads of a workgroup
    const int64_t row = blockIdx.x;
    const int head0 = static_cast<int>(blockIdx.y) * per, channels = min(per, a.kv_heads - head0) * a.d;
    const int64_t s = sequence_of_unit(a.k_starts, a.sequences, a.total_k, 1, a.block_log2, row);
    const Span k = sequence_span(a.k_starts, s, a.total_k);
    const int64_t first = (row - ((k.begin >> a.block_log2) + s)) << a.block_log2;
    const int count = static_cast<int>(min(static_cast<int64_t>(a.block), k.rows - first));
    if (first < 0 || count <= 0) return;  // the whole workgroup
    if (tid < 8) most[tid] = 0;
    double m[8] = {};
    if (8 * lane < channels) {
        const T *x = static_cast<const T *>(a.k) + (k.begin + first) * a.k_stride + static_cast<int64_t>(head0) * a.d + 8 * lane;
#pragma unroll 4
        for (int r = part; r < count; r += 8) {
            constexpr int N = 8 * static_cast<int>(sizeof(T)) / 16;
            uint4 t[N];
#pragma unroll
            for (int i = 0; i < N; ++i) t[i] = reinterpret_cast<const uint4 *>(x + r * a.k_stride)[i];
            const uint32_t *w = reinterpret_cast<const uint32_t *>(t);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                m[e] += static_cast<double>(__builtin_bit_cast(
                    float, sizeof(T) == 4 ? w[e] : e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16));
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[part][8 * lane + e] = m[e];
    __syncthreads();
    double mean = 0.0;
    if (tid < channels) {
        for (int p = 0; p < 8; ++p) mean += sums[p][tid];
        mean /= count;
        // bits of magnitudes rise with them; infinities and NaN stand above all
        atomicMax(reinterpret_cast<unsigned long long *>(&most[tid / a.d]),
                  __builtin_bit_cast(unsigned long long, fabs(mean)));
    }
    __syncthreads();
    if (tid >= channels) return;
    const int head = head0 + tid / a.d, c = tid % a.d;
    const double big = __builtin_bit_cast(double, most[tid / a.d]);
    const bool fine = codes_fine(big);
    const int e = exponent_of(big);
    a.codes[(static_cast<int64_t>(head) * a.rows + row) * a.d + c] =
        static_cast<int8_t>(fine ? code_of(mean, two_to(6 - e)) : 0);
    if (c == 0) a.scale[static_cast<int64_t>(head) * a.rows + row] = fine ? static_cast<float>(two_to(e - 6)) : 0.0f;
}

// ---------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------
struct SelectArgs {
    const void *q;
    const int32_t *q_starts, *k_starts;
    const int8_t *codes;
    const float *scale;
    int32_t *selected;
    int64_t total_q, total_k, q_stride, sequences, rows;
    int32_t kv_heads, group, d, block, block_log2, top, most_blocks, flags, run;
};

// A float's order as an unsigned whole number: 0x007fffff (-inf) to 0xff800000 (inf).  -0 does not
// occur: scores are whole numbers times powers of two.
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Threads of a workgroup, and of the team that searches a query's keys.  Sixteen waves fetch the scores of a query by
// itself, and one of them searches: sums over more took longer than what they saved (30 us instead of 20 for 1,024 blocks).
constexpr int select_threads(int qt) { return qt == 1 ? 1024 : 256; }
constexpr int select_team(int qt) { return qt == 16 ? 16 : 64; }

// Sum over a team of 16 or 64 threads, in each of them.
template <int TEAM>
__device__ __forceinline__ int team_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false);  // row_ror:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x124, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x122, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x121, 0xf, 0xf, false);
    if constexpr (TEAM >= 64) {
        const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = static_cast<int>(a[0] + a[1]);
        const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = static_cast<int>(b[0] + b[1]);
    }
    return v;
}
// Sum over the team's threads before this one.
template <int TEAM>
__device__ __forceinline__ int team_before(int v) {
    const int at = threadIdx.x & (TEAM - 1);
    int x = v;
#pragma unroll
    for (int o = 1; o < TEAM; o <<= 1) {
        const int y = __shfl_up(x, o, TEAM);
        if (at >= o) x += y;
    }
    return x - v;
}

// A tile of QT queries of one key head.  Scores by integer products (16x16x64: blocks by
// queries), their order keys in LDS; then a team of 16 or 64 threads for each query, each with a run
// of blocks side by side, finds the `top`-th largest key by cutting the range of keys (it stops
// as soon as the count of the keys from the cut on is right) and writes its run's chosen
// blocks behind those of the threads before it, equal keys first come, first served.  RUN: a
// thread's blocks, whose keys stay in registers; 0: any number, from LDS each time.
// QT 16 fills the products; 4 and 1 are for few rows, and for more blocks than LDS
// holds of 16 queries.
template <class T, int QT, int RUN>
__global__ void __launch_bounds__(select_threads(QT)) select_kernel(SelectArgs a) {
    constexpr int TEAM = select_team(QT), WAVES = select_threads(QT) / 64;
    extern __shared__ uint32_t keys[];  // [QT][TEAM * run]
    __shared__ alignas(16) int8_t qc[16][128];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const int64_t tile = blockIdx.x / a.kv_heads;
    const int head = static_cast<int>(blockIdx.x - tile * a.kv_heads);
    const int64_t s = sequence_of_unit(a.q_starts, a.sequences, a.total_q, 1, QT == 16 ? 4 : QT == 4 ? 2 : 0, tile);
    const Span qs = sequence_span(a.q_starts, s, a.total_q), ks = sequence_span(a.k_starts, s, a.total_k);
    const int64_t first = (tile - (qs.begin / QT + s)) * QT;
    if (first < 0 || first >= qs.rows) return;  // the whole workgroup
    const int row0 = static_cast<int>(first), queries = min(QT, qs.rows - row0);

    // ---- the queries' codes, 16 threads each
    {
        const int q = (tid >> 4) & 15, l = tid & 15, per = a.d / 16;
        // this thread's channels of all heads, pairs (per is even), on their way before the first is used
        const T *x = static_cast<const T *>(a.q) + (qs.begin + row0 + min(q, queries - 1)) * a.q_stride +
                     static_cast<int64_t>(head) * a.group * a.d + l * per;
        const auto channels = [&](float (&v)[8]) __attribute__((always_inline)) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[2 * e] = w[2 * e + 1] = 0;
                if (2 * e >= per) continue;
                if constexpr (sizeof(T) == 4) {
                    const uint2 t = reinterpret_cast<const uint2 *>(x)[e];
                    w[2 * e] = t.x, w[2 * e + 1] = t.y;
                } else {
                    w[2 * e] = reinterpret_cast<const uint32_t *>(x)[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = __builtin_bit_cast(float, sizeof(T) == 4 ? w[2 * e] : w[2 * e] << 16);
                v[2 * e + 1] = __builtin_bit_cast(float, sizeof(T) == 4 ? w[2 * e + 1] : w[2 * e] & 0xffff0000u);
            }
        };
        float v[8];
        channels(v);
        if (a.group == 1) {
            // nothing is added up: the same codes in 32 bits (magnitudes' bits rise with them, NaN's above all)
            uint32_t most = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = max(most, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1)
                most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), o, 16)));
            const bool fine = most >= (127u - 100u) << 23 && most < 0x7f800000u;
            const int up = fine ? 6 - (static_cast<int>(most >> 23) - 127) : 0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < per)
                    qc[q][l * per + e] =
                        static_cast<int8_t>(fine ? min(127, max(-127, static_cast<int>(rintf(ldexpf(v[e], up))))) : 0);
        } else {
            double m[8], most = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) m[e] = static_cast<double>(v[e]);
            int h = 1;
            for (; h + 3 <= a.group; h += 3) {
                float w[3][8];
#pragma unroll
                for (int u = 0; u < 3; ++u) {
                    x += a.d;
                    channels(w[u]);
                }
#pragma unroll
                for (int u = 0; u < 3; ++u)
#pragma unroll
                    for (int e = 0; e < 8; ++e) m[e] += static_cast<double>(w[u][e]);
            }
            for (; h < a.group; ++h) {
                x += a.d;
                channels(v);
#pragma unroll
                for (int e = 0; e < 8; ++e) m[e] += static_cast<double>(v[e]);
            }
            bool fine = true;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                fine = fine && fabs(m[e]) < __builtin_inf();
                most = fmax(most, fabs(m[e]));
            }
            int all = fine ? 1 : 0;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                most = fmax(most, __shfl_xor(most, o, 16));
                all &= __shfl_xor(all, o, 16);
            }
            fine = all && codes_fine(most);
            const double up = two_to(6 - exponent_of(most));
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < per) qc[q][l * per + e] = static_cast<int8_t>(fine ? code_of(m[e], up) : 0);
        }
    }
    __syncthreads();

    // ---- scores
    const int nb = min((ks.rows + a.block - 1) >> a.block_log2, a.most_blocks), lag = ks.rows - qs.rows;
    const int run = RUN ? RUN : a.run;  // blocks of a thread, a multiple of 4
    const int64_t base = static_cast<int64_t>(head) * a.rows + (ks.begin >> a.block_log2) + s;
    const auto candidates = [&](int q) __attribute__((always_inline)) {  // blocks that query q may choose
        const int place = row0 + q + lag;
        return !(a.flags & S3DX_BLOCK_CAUSAL) ? nb : place < 0 ? 0 : min(nb, (place >> a.block_log2) + 1);
    };
    i32x4 qf[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
        qf[t] = 64 * t + 16 * g < a.d ? *reinterpret_cast<const i32x4 *>(&qc[c][64 * t + 16 * g]) : i32x4{0, 0, 0, 0};
    const auto near_of = [&](int q) __attribute__((always_inline)) {  // its own block, or -1
        const int place = row0 + q + lag, b = place >> a.block_log2;
        return a.flags & S3DX_BLOCK_NEAR && place >= 0 && b < nb ? b : -1;
    };
    const int seen = candidates(c), own = near_of(c);
    // Chunks of 16 blocks, U at a time, all their codes and scales on the way before the first is used; what is behind
    // the last block, or behind a code's end (there the query's codes are 0), is read where something is.
    const int chunks = TEAM * run / 16;
    constexpr int U = QT == 16 ? (RUN == 4 ? 1 : RUN == 8 ? 2 : 4) : 4;
    const int8_t *code0 = a.codes + base * a.d;
    const float *scale0 = a.scale + base;
    for (int j0 = wave; nb > 0 && j0 < chunks; j0 += WAVES * U) {
        i32x4 x[U][2];
        float scale[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + WAVES * u;
            const uint32_t code = static_cast<uint32_t>(__mul24(min(16 * j + c, nb - 1), a.d));
            x[u][0] = *reinterpret_cast<const i32x4 *>(code0 + (code + (16 * g < a.d ? 16 * g : 0)));
            if (a.d > 64) x[u][1] = *reinterpret_cast<const i32x4 *>(code0 + (code + (64 + 16 * g < a.d ? 64 + 16 * g : 0)));
#pragma unroll
            for (int i = 0; i < 4; ++i) scale[u][i] = scale0[static_cast<uint32_t>(min(16 * j + 4 * g + i, nb - 1))];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + WAVES * u;
            if (j >= chunks) break;
            i32x4 dot = {0, 0, 0, 0};
            dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[u][0], qf[0], dot, 0, 0, 0);
            if (a.d > 64) dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[u][1], qf[1], dot, 0, 0, 0);
            uint32_t key[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 16 * j + 4 * g + i;
                // |dot| < 2^21: the product with a power of two is exact.  The own block is chosen without a key.
                key[i] = at < seen && at != own ? order_key(static_cast<float>(dot[i]) * scale[u][i]) : 0u;
            }
            if (c < QT)
                *reinterpret_cast<uint4 *>(&keys[c * (TEAM * run) + 16 * j + 4 * g]) = make_uint4(key[0], key[1], key[2], key[3]);
        }
    }
    __syncthreads();

    // ---- the `top` largest, a team for each query
    if (tid >= QT * TEAM) return;
    const int q = tid / TEAM, t = tid & (TEAM - 1);
    const uint32_t *mine = keys + q * (TEAM * run) + t * run;
    uint32_t held[RUN ? RUN : 1];
    if constexpr (RUN > 0) {
#pragma unroll
        for (int i = 0; i < RUN; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(mine + i);
            held[i] = x.x, held[i + 1] = x.y, held[i + 2] = x.z, held[i + 3] = x.w;
        }
    }
    const auto each = [&](auto &&f) __attribute__((always_inline)) {  // f(key, index in the run)
        if constexpr (RUN > 0) {
#pragma unroll
            for (int i = 0; i < RUN; ++i) f(held[i], i);
        } else {
            for (int i = 0; i < run; i += 4) {
                const uint4 x = *reinterpret_cast<const uint4 *>(mine + i);
                f(x.x, i), f(x.y, i + 1), f(x.z, i + 2), f(x.w, i + 3);
            }
        }
    };
    const int near = q < queries ? near_of(q) : -1, all = q < queries ? candidates(q) : 0;
    // the own block apart (its place is in reach: it is a candidate): `take` of `may` others
    const int may = all - (near >= 0 ? 1 : 0), take = min(all, a.top) - (near >= 0 ? 1 : 0);
    uint32_t low = 0xffffffffu, high = 0;
    each([&](uint32_t k, int) {
        if (k) low = min(low, k);
        high = max(high, k);
    });
    {
#pragma unroll
        for (int o = 1; o < TEAM; o <<= 1) {
            low = min(low, static_cast<uint32_t>(__shfl_xor(static_cast<int>(low), o, TEAM)));
            high = max(high, static_cast<uint32_t>(__shfl_xor(static_cast<int>(high), o, TEAM)));
        }
    }
    // at least `take` keys are >= low (count of them: n_low), fewer than that are >= high
    high += 1;
    int n_low = may;
    if (take == 0) low = high = 1, n_low = 0;
    float f_low = of_key(low), f_high = of_key(high);
    for (int cut = 0;; ++cut) {
        const bool going = n_low != take && high - low > 1;
        if (__builtin_amdgcn_ballot_w64(going) == 0) break;
        // Cut halfway between the values (about eight cuts for 80 blocks; where it is made decides only how soon
        // it ends); from the 16th on, and where the values leave nothing between, halfway between the keys (at most 32 more).
        uint32_t mid = order_key(0.5f * f_low + 0.5f * f_high);
        if (__builtin_amdgcn_ballot_w64(going && (mid <= low || mid >= high || cut >= 16)) != 0 &&
            (mid <= low || mid >= high || cut >= 16))
            mid = low + (high - low) / 2;
        int n = 0;
        each([&](uint32_t k, int) { n += k >= mid ? 1 : 0; });
        n = team_sum<TEAM>(n);
        if (going) {
            if (n >= take) low = mid, f_low = of_key(mid), n_low = n;
            else high = mid, f_high = of_key(mid);
        }
    }
    // Chosen: keys above low, and of those that equal it the first ones (all, where the count came out right).
    int above = 0, equal = 0;
    if (take > 0)
        each([&](uint32_t k, int) {
            above += k > low ? 1 : 0;
            equal += k == low ? 1 : 0;
        });
    const int spare = take - team_sum<TEAM>(above);  // equal keys to choose
    const int equal_before = team_before<TEAM>(equal);
    int left = max(0, min(equal, spare - equal_before));  // ... of this thread's
    const int own_i = near >= t * run && near < t * run + run ? near - t * run : -1;
    int at = team_before<TEAM>(above + left + (own_i >= 0 ? 1 : 0));
    if (q >= queries) return;
    int32_t *out = a.selected + ((qs.begin + row0 + q) * a.kv_heads + head) * a.top;
    each([&](uint32_t k, int i) {
        const bool same = take > 0 && k == low && left > 0;
        if ((take > 0 && k > low) || same || i == own_i) out[at++] = t * run + i;
        if (same) --left;
    });
    for (int i = min(all, a.top) + t; i < a.top; i += TEAM) out[i] = -1;
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
struct AttendArgs {
    const void *q, *k, *v;
    void *o;
    float *lse;
    const int32_t *q_starts, *k_starts, *selected;
    int64_t total_q, total_k, q_stride, k_stride, v_stride, o_stride, sequences;
    int32_t heads, group, kv_heads, block, block_log2, top, causal, splits, tile_groups;
    float scale;
    float *part_o;   // [splits][total_q][heads][d]: not yet divided by the sum
    float2 *part_ml; // [splits][total_q][heads]: the power of two that weights are relative to, their sum
};

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kMostBase = 0x1p24f;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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

// Binary orders by which weights over `keys` keys are kept down, so that sums of finite values stay finite whatever the
// values: weights pass 1 by 8 orders and a base's rounding before that moves, and there are as many as keys.  Where
// again_of looks at the weights alone; elsewhere 0, as a sum that is not finite is made again, and small values keep their
// lowest bits.
template <class T>
__device__ __forceinline__ int room_of(const AttendArgs &a, int keys) {
    return sizeof(T) == 2 && !a.selected && !a.causal ? 9 + 32 - __builtin_clz(keys | 1) : 0;
}

// The logarithm of a sum of weights l relative to 2^m, `room` of whose orders kept them down; of nothing seen -inf.
__device__ __forceinline__ float log_of(float m, float l, int room) {
    return l == 0.0f ? neg_inf()
                     : fmaf(m - static_cast<float>(room), kLn2, __builtin_amdgcn_logf(ldexpf(l, room)) * kLn2);
}

// Whether a row's sums (l: the weights', y: anything made of its values') have to be made again: 0 times what is not
// finite is a NaN, also for a key that the row does not see.  Where every row sees every key the NaN or infinity is the
// result's own, unless the weights are not finite themselves (in three terms an infinity is not one) or nothing is seen.
template <class T>
__device__ __forceinline__ bool again_of(const AttendArgs &a, float l, float y) {
    const bool own = sizeof(T) == 2 && !a.selected && !a.causal && l != 0.0f;
    return (own ? l : l + y) * 0.0f != 0.0f;
}

// One row by the whole wave, key by key: scores with a key per lane, the running maximum
// and sum, values with a channel pair per lane.  Only keys that the row sees are
// multiplied, so nothing else reaches it: for rows whose tile gave no finite result, or none
// that its bases hold.
template <class T, int D>
__device__ void attend_row(const AttendArgs &a, int64_t row, int head, Span qs, Span ks) {
    const int lane = threadIdx.x & 63, kvh = head / a.group;
    const T *q = static_cast<const T *>(a.q) + row * a.q_stride + static_cast<int64_t>(head) * D;
    const T *k = static_cast<const T *>(a.k) + ks.begin * a.k_stride + static_cast<int64_t>(kvh) * D;
    const T *v = static_cast<const T *>(a.v) + ks.begin * a.v_stride + static_cast<int64_t>(kvh) * D;
    const int seen = a.causal ? max(0, min(ks.rows, static_cast<int>(row - qs.begin) + ks.rows - qs.rows + 1)) : ks.rows;
    const int blocks = (seen + a.block - 1) >> a.block_log2;
    const int32_t *list = a.selected ? a.selected + (row * a.kv_heads + kvh) * a.top : nullptr;
    float qv[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) qv[w] = lane + 64 * w < D ? load_as_f32<T>(q + lane + 64 * w) * a.scale : 0.0f;
    float m = neg_inf(), l = 0.0f, o[2] = {0.0f, 0.0f};
    const int room = 32 - __builtin_clz(seen | 1);  // weights add up to 1 at most, so that sums of finite values stay finite
    // A weight that is a NaN makes the whole row one: the rest need not be read (5,086 rows x 16 heads x 64
    // bf16 with a NaN among the keys: 0.9 ms; 30 ms key by key to the end).
    bool lost = false;
    for (int t = 0; t < (list ? a.top : blocks) && !lost; ++t) {
        const int b = list ? list[t] : t;
        if (b < 0 || b >= blocks) continue;
        if (list) {  // a block counts once
            bool before = false;
            for (int e = lane; e < t; e += 64) before = before || list[e] == b;
            if (__any(before)) continue;
        }
        for (int k0 = b << a.block_log2; k0 < min((b + 1) << a.block_log2, seen) && !lost; k0 += 64) {
            const int count = min(64, min((b + 1) << a.block_log2, seen) - k0);
            const T *kr = k + static_cast<int64_t>(k0 + min(lane, count - 1)) * a.k_stride;
            const T *vr = v + static_cast<int64_t>(k0) * a.v_stride;
            float sc = 0.0f;
            for (int c = 0; c < D; ++c) sc += __shfl(c < 64 ? qv[0] : qv[1], c & 63, 64) * load_as_f32<T>(kr + c);
            if (lane >= count) sc = neg_inf();
            float mx = sc;
            for (int w = 1; w < 64; w <<= 1) mx = fmaxf(mx, __shfl_xor(mx, w, 64));
            const float mn = fmaxf(m, mx), base = mn == neg_inf() ? 0.0f : mn;
            // the difference first: scores of the type's lowest value stay finite
            const float alpha = exp2f((m - base) * kLog2e), p = exp2f(fmaf(sc - base, kLog2e, -static_cast<float>(room)));
            l = l * alpha + (lane < count ? p : 0.0f);
            o[0] *= alpha;
            o[1] *= alpha;
            m = mn;
            lost = __any(lane < count && p != p);
            for (int j = 0; j < count; ++j) {
                const float pj = __shfl(p, j, 64);
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    if (lane + 64 * w < D) o[w] += pj * load_as_f32<T>(vr + j * a.v_stride + lane + 64 * w);
            }
        }
    }
    for (int w = 1; w < 64; w <<= 1) l += __shfl_xor(l, w, 64);
    const float r = l == 0.0f ? 0.0f : 1.0f / l;  // 0: nothing seen (a NaN is not 0 and stays)
    T *y = static_cast<T *>(a.o) + row * a.o_stride + static_cast<int64_t>(head) * D;
#pragma unroll
    for (int w = 0; w < 2; ++w)
        if (lane + 64 * w < D) store_from_f32<T>(y + lane + 64 * w, l == 0.0f ? 0.0f : o[w] * r);
    if (a.lse && lane == 0) a.lse[row * a.heads + head] = l == 0.0f ? neg_inf() : m + __builtin_amdgcn_logf(ldexpf(l, room)) * kLn2;
}

// N dwords at byte offset `at` of a buffer; zeros from its end on.
template <int N>
__device__ __forceinline__ void buffer_dwords(__amdgpu_buffer_rsrc_t r, int at, uint32_t *out) {
    static_assert(N >= 1 && N <= 4 || N == 6 || N == 8);
    if constexpr (N == 1) {
        out[0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
    } else if constexpr (N == 2) {
        const u32x2 t = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0);
        out[0] = t[0], out[1] = t[1];
    } else if constexpr (N == 3) {
        const u32x3 t = __builtin_amdgcn_raw_buffer_load_b96(r, at, 0, 0);
        out[0] = t[0], out[1] = t[1], out[2] = t[2];
    } else if constexpr (N == 4) {
        const u32x4 t = __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0);
        out[0] = t[0], out[1] = t[1], out[2] = t[2], out[3] = t[3];
    } else {
        buffer_dwords<N / 2>(r, at, out);
        buffer_dwords<N / 2>(r, at + 2 * N, out + N / 2);
    }
}

// Rows [first, first + rows) of a head as a buffer; reads behind the last row's
// channels give zeros.
template <class T, int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const void *x, int64_t row, int64_t stride, int head,
                                                              int rows) {
    const T *p = static_cast<const T *>(x) + row * stride + static_cast<int64_t>(head) * D;
    const int bytes = static_cast<int>(((rows - 1) * stride + D) * static_cast<int64_t>(sizeof(T)));
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(p), static_cast<short>(0), bytes, 0x00020000);
}

// x as the sum of three bfloat16 terms, each cut off from what the ones before left: 8 significant bits a
// term, 24 together, so nothing is lost (of magnitudes from 2^-102 on, whose last terms are normal
// numbers).  Pairs of values give pairs of terms.
__device__ __forceinline__ void three_terms(float x, float y, uint32_t (&out)[3]) {
    constexpr uint32_t kHigh = 0x07060302u;  // the high halves of both
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x), v = __builtin_bit_cast(uint32_t, y);
        out[p] = __builtin_amdgcn_perm(v, u, kHigh);
        if (p == 2) break;
        x -= __builtin_bit_cast(float, u & 0xffff0000u);
        y -= __builtin_bit_cast(float, v & 0xffff0000u);
    }
}

// Of 16 lanes, lane 4i + a gives the address of four 16-bit values (row i, columns 4a..) and
// gets column 4i + a of the four rows.
__device__ __forceinline__ u32x2 transposed(const char *p) {
    typedef short i16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) i16x4 *)(const_cast<char *>(p))));
}

// d += A B over 32 values: one product of bfloat16 operands, or, of operands in three terms, the six
// largest, the smallest of them first.  Terms are cut off, not rounded, so the second reaches 2^-7 of the first and the
// third 2^-15: what is left out is up to 2^-21 of a product, 2^-24.5 in the mean, and of the product's sign.
template <int P>
__device__ __forceinline__ f32x4 product(const u32x4 (&x)[P], const u32x4 (&y)[P], f32x4 d) {
    const auto one = [&](int i, int j) __attribute__((always_inline)) {
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[i]), __builtin_bit_cast(bf16x8, y[j]), d, 0, 0, 0);
    };
    if constexpr (P == 3) {
        one(2, 0), one(1, 1), one(0, 2);
        one(1, 0), one(0, 1);
    }
    one(0, 0);
    return d;
}

// Attention of a tile of 16 NS rows (query rows times the heads that share a key head)
// on matrix units.  A wave computes S^T = K Q^T and O^T = V^T P^T, so that what one
// product leaves in a lane is what the next one wants there: the weights stay in
// registers.  A 16x16 product leaves lane (c, g) = (lane & 15, lane >> 4) with rows
// 4g..4g+3 of column c: of S^T four keys of query c, and two such (keys 4g.. of one
// 16-key group and of the next) are the eight k-values that lane (c, g) holds of the
// operand P^T.  V^T's operand wants the same eight keys of one channel: the lane
// reads D/16 channels of eight rows and pairs them up by byte permutes; channel
// c*(D/16) + t goes with product t, so O^T leaves each lane D/4 channels that lie
// side by side.  K's rows are read whole, 16 bytes a lane one after the other, and turned in LDS, as
// K's operand read from memory takes 16 bytes from each of 16 rows (5,086 rows x 16 heads x 64 bf16,
// all keys: 157 us so, 138 us turned; 144 us with V through LDS as well).  Statistics, scales and
// masks are per query, hence per lane.
//
// What bounds it, at 130-136 us (780-815 TFLOP/s) for that call: a step of 64 rows and 32 keys is 32 products of 16 cycles
// and 166 vector instructions of about 800 cycles, 32 exponentials among them, and the two waves of a SIMD hardly cover
// one's products with the other's weights: by the counters both together are 84% of all cycles.  A tile's start, join
// and end cost about 11 us beside (16,384 rows: 865 TFLOP/s).
//
// The keys of a tile are those of any of its rows' blocks: a table in LDS gets, for each
// block, a bit for each row that chose it; rows that did not take weights 0.
// Neighbouring rows choose alike, which is what makes tiles of them pay.
//
// FP32 heads up to 64 wide: the same products on three bfloat16 terms of every value, six for one, each 16 times as
// fast as FP32's own (5,086 rows x 16 heads x 64, all keys: 615 us, 880 with FP32's).  Wider
// heads' terms do not fit a lane's registers: they take FP32's products.
//
// WAVES 4: the workgroup's waves take a tile together, every fourth step (of lists,
// block) each, and join them through LDS: a quarter of the tiles' length, so that the last
// ones to run leave fewer units idle.  WAVES 1: a tile each, for rows of few keys.
// HALVES 2: a tile of 32 NS rows, half of them for each pair of the waves, a pair's waves every second step.
// For heads whose 64 rows one wave's registers do not hold: the two waves of a step
// fetch half of its K and V rows each, into LDS that they share (two buffers, one barrier a step);
// V^T is read from there by the transposing reads of 16-bit data (12,001 ragged rows x 16 / 4 heads
// x 128, top 32: 596 us with a wave's 32 rows by itself, 546 us so).
template <class T, int D, int KC, int NS, bool LISTED, int WAVES, int HALVES>
__global__ void __launch_bounds__(256, 2) attend_kernel(AttendArgs a) {
    constexpr bool BF = sizeof(T) == 2;
    constexpr int ROWS = 16 * NS * HALVES, SETS = NS * HALVES;
    constexpr bool SHARED = HALVES == 2;
    constexpr bool FLAT = BF && !LISTED && WAVES == 4;
    constexpr int KT = KC / 16;              // 16-key groups of a step
    constexpr int P = BF ? 1 : D <= 64 ? 3 : 0; // bfloat16 terms of a value; 0: FP32's products
    constexpr int QV = P ? D / 32 : D / 16;  // products over a row's channels
    constexpr int C = D / 16;                // channels of a lane's V row
    constexpr int VW = C * static_cast<int>(sizeof(T)) / 4;
    constexpr int E = static_cast<int>(sizeof(T));
    static_assert(WAVES == 4 || (WAVES == 1 && HALVES == 1));
    static_assert(HALVES == 1 || (HALVES == 2 && BF));
    static_assert(ROWS == 32 || ROWS == 64);
    // LDS: each wave's K rows of a step (or the shared buffers); the table of blocks, TABLE of them at a time for each tile of the
    // workgroup; after the last step over both, the waves' results: element (set n, i, t) of every lane.
    constexpr int TABLE = 1024, TILES = 4 / WAVES;
    constexpr int CH = D * E / 16;                 // 16-byte pieces of a K row
    constexpr int NP = KC * CH / 64 / (SHARED ? 2 : 1);  // ... of a step, for each lane
    static_assert(KC * CH % (SHARED ? 128 : 64) == 0);
    constexpr int PLANE = KC * D * 2;              // a step's rows in bfloat16
    constexpr int KEYS = SHARED ? 2 * PLANE : P * PLANE, TABLES = LISTED ? TABLE * TILES * 8 : 0;
    constexpr int PART = WAVES == 4 ? 4 * NS * 4 * C * 64 * 4 : 0;
    constexpr int LDS = 4 * KEYS + TABLES > PART ? 4 * KEYS + TABLES : PART;
    __shared__ alignas(16) char lds[LDS > 0 ? LDS : 16];
    __shared__ float2 part_ml[WAVES == 4 ? 4 : 1][NS][16];
    auto part = reinterpret_cast<float (*)[NS * 4 * C][64]>(lds);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Consecutive workgroups of one XCD run neighbouring tiles of a head: its L2 holds
    // their keys.
    const int id = xcd_tile(blockIdx.x, gridDim.x);
    const int split = id / a.tile_groups % a.splits, kvh = id / a.tile_groups / a.splits;
    int tg = id % a.tile_groups;
    // Causal rows see more keys the later they stand: every eighth group in a row, so that the XCDs' runs cost alike,
    // and the longest first.
    if (a.causal) tg = a.tile_groups - 1 - (tg % (a.tile_groups >> 3) * 8 + tg / (a.tile_groups >> 3));
    const int64_t tile = WAVES == 4 ? tg : static_cast<int64_t>(tg) * 4 + wave;
    const int64_t s = sequence_of_unit(a.q_starts, a.sequences, a.total_q, a.group, ROWS == 64 ? 6 : 5, tile);
    const Span qs = sequence_span(a.q_starts, s, a.total_q), ks = sequence_span(a.k_starts, s, a.total_k);
    const int64_t first_row = (tile - (qs.begin * a.group / ROWS + s)) * ROWS;
    const int nrows = qs.rows * a.group;  // total_q * heads < 2^31
    if (first_row < 0 || first_row >= nrows) return;
    const int r0 = static_cast<int>(first_row);
    const int tok0 = r0 / a.group, ntok = (min(r0 + ROWS, nrows) - 1) / a.group - tok0 + 1;
    const int lag = ks.rows - qs.rows;
    // this wave's share of the tile: every `pieces`-th step or chosen block, a power of two
    constexpr int SHARES = WAVES / HALVES;
    const int half = HALVES == 2 ? wave >> 1 : 0;
    const int piece = split * SHARES + (SHARES > 1 ? wave & (SHARES - 1) : 0), pieces = a.splits * SHARES;
    const int r0w = r0 + half * 16 * NS;  // this wave's first row

    // this lane's query of each set of 16, and the keys that it sees: [0, lim)
    int lim[NS];
    u32x4 qf[NS][QV][P ? P : 1];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const int r = min(r0w + 16 * n + c, nrows - 1), tok = r / a.group;
        lim[n] = a.causal ? max(0, min(ks.rows, tok + lag + 1)) : ks.rows;
        const T *q = static_cast<const T *>(a.q) + (qs.begin + tok) * a.q_stride +
                     static_cast<int64_t>(kvh * a.group + r % a.group) * D;
#pragma unroll
        for (int j = 0; j < QV; ++j) {
            if constexpr (P == 3) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 t = *reinterpret_cast<const float2 *>(q + 32 * j + 8 * g + 2 * i);
                    uint32_t terms[3];
                    three_terms(t.x, t.y, terms);
#pragma unroll
                    for (int p = 0; p < 3; ++p) qf[n][j][p][i] = terms[p];
                }
            } else {
                qf[n][j][0] = *reinterpret_cast<const u32x4 *>(q + (BF ? 32 * j + 8 * g : 16 * j + 4 * g));
            }
        }
    }
    const int most = a.causal ? max(0, min(ks.rows, tok0 + ntok + lag)) : ks.rows;  // keys that some row sees
    const int least = a.causal ? max(0, min(ks.rows, tok0 + lag + 1)) : ks.rows;          // ... that all rows see

    // ---- the tile's steps of KC keys
    uint64_t *table = reinterpret_cast<uint64_t *>(lds + 4 * KEYS) + (WAVES == 4 ? 0 : wave * TABLE);
    const int blocks = (most + a.block - 1) >> a.block_log2;  // in reach of the tile
    int w0 = 0, chunk = 0, rank = 0;  // the table's first block, the next 64 of it, chosen blocks before them
    uint64_t todo = 0, mine = 0;      // this wave's blocks among the last 64; this lane's table entry of them
    uint64_t members = ~UINT64_C(0);
    int first, end;                   // the step's first key, the end of its block
    int whole = 0;                    // ... were it a whole one
    const auto next = [&]() __attribute__((always_inline)) {  // false: no step left in the table
        if constexpr (LISTED) {
            first += KC;
            // SHARED: every block takes all of its steps, also those behind the last key, so that the waves stay together
            if (SHARED ? first < whole : first < end) return !SHARED || first < end;
            while (todo == 0) {
                const int count = min(TABLE, blocks - w0);
                if (chunk >= count) {
                    first = 1 << 30;
                    return false;
                }
                mine = chunk + lane < count ? table[chunk + lane] : 0;
                const uint64_t chosen = __ballot(mine != 0);
                const int r = rank + __popcll(chosen & ((UINT64_C(1) << lane) - 1));
                todo = __ballot(mine != 0 && (r & (pieces - 1)) == piece);
                rank += __popcll(chosen);
                chunk += 64;
            }
            const int bit = __builtin_ctzll(todo);
            todo &= todo - 1;
            members = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine >> 32), bit))) << 32 |
                      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), bit));
            first = (w0 + chunk - 64 + bit) << a.block_log2;
            whole = first + a.block;
            end = min(whole, most);
            return true;
        } else {
            first += pieces * KC;
            return first < end;
        }
    };
    // The table's waves agree on it: the workgroup's, or this one alone.
    const auto together = [&]() __attribute__((always_inline)) {
        if constexpr (WAVES == 4) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    const auto fill_table = [&]() __attribute__((always_inline)) {
        const int id0 = WAVES == 4 ? static_cast<int>(threadIdx.x) : lane, step = 64 * WAVES;
        const int count = min(TABLE, blocks - w0);
        for (int e = id0; e < count; e += step) table[e] = 0;
        together();
        const int32_t *list = a.selected + ((qs.begin + tok0) * a.kv_heads + kvh) * a.top;
        const int64_t by = static_cast<int64_t>(a.kv_heads) * a.top;
        for (uint32_t e = id0; e < static_cast<uint32_t>(ntok * a.top); e += step) {
            const uint32_t t = e / static_cast<uint32_t>(a.top);
            const int b = list[t * by + (e - t * a.top)];
            if (b < w0 || b >= w0 + count) continue;
            // the tile's rows of query t: [t * group, t * group + group), less what is outside
            const int lo = max(static_cast<int>(t + tok0) * a.group - r0, 0);
            const int hi = min(static_cast<int>(t + tok0 + 1) * a.group - r0, min(ROWS, nrows - r0));
            __hip_atomic_fetch_or(&table[b - w0], (~UINT64_C(0) >> (64 - (hi - lo))) << lo, __ATOMIC_RELAXED,
                                  __HIP_MEMORY_SCOPE_WORKGROUP);
        }
        together();
    };

    // ---- state
    f32x4 acc[NS][C], sum[NS];
    // what weights are relative to, a power of two; the raw product from which on it moves (-inf: nothing seen yet, when
    // any finite base leaves weights of 0)
    float base[NS], above[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        above[n] = neg_inf();
        base[n] = 0.0f;
        sum[n] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < C; ++t) acc[n][t] = f32x4{0, 0, 0, 0};
    }
    const float cs = a.scale * kLog2e;
    const int room = room_of<T>(a, ks.rows);
    // Byte offsets of this lane's rows of V in a step: held where registers allow, else the first and the steps between.
    constexpr bool HELD = D < 128 && !SHARED;
    const int kstep = static_cast<int>(a.k_stride) * E, vstep = static_cast<int>(a.v_stride) * E;
    const int vat = 4 * g * vstep + c * (C * E);
    int voff[HELD ? KT : 1][4];
    if constexpr (HELD) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) voff[t][i] = vat + (16 * t + i) * vstep;
    }
    // K: lane l fetches pieces l, l + 64, ... of the step's rows, which lie in LDS row by row (a plane for each term), a
    // row's pieces xor-ed by its number so that eight neighbouring rows' pieces of one number lie in different banks.
    constexpr int ROW = D / 8;  // 16-byte pieces of a row in LDS
    const auto turned = [](int row, int piece) __attribute__((always_inline)) {
        return piece ^ (ROW % 16 == 0 ? row & 15 : ROW % 8 == 0 ? row & 7 : (row >> 1) & 3);
    };
    char *kt = SHARED ? lds + (wave & 1) * (4 * PLANE) : lds + wave * KEYS;
    int koff[P ? NP : KT], kput[P ? NP : 1], kget[P ? QV : 1], vsrc[SHARED ? NP : 1], vget[SHARED ? C : 1];
    if constexpr (P > 0) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int at = ((SHARED ? half * NP : 0) + p) * 64 + lane, row = at / CH, piece = at % CH;
            koff[p] = row * kstep + piece * 16;
            if constexpr (SHARED) vsrc[p] = row * vstep + piece * 16;
            kput[p] = BF ? (row * ROW + turned(row, piece)) * 16 : (row * ROW + turned(row, piece >> 1)) * 16 + (piece & 1) * 8;
        }
#pragma unroll
        for (int j = 0; j < QV; ++j) kget[j] = (c * ROW + turned(c, 4 * j + g)) * 16;
    } else {
#pragma unroll
        for (int t = 0; t < KT; ++t) koff[t] = (16 * t + c) * kstep + 16 * g;
    }
    if constexpr (SHARED) {
        // of each 16 lanes, lane 4i + a gives channels 16t + 4a.. of key 4g + i and gets channel 16t + 4i + a of the four keys
        const int row = 4 * g + (c >> 2);
#pragma unroll
        for (int t = 0; t < C; ++t) vget[t] = PLANE + (row * ROW + turned(row, 2 * t + ((c & 3) >> 1))) * 16 + (c & 1) * 8;
    }
    uint32_t kn[P ? NP : 1][4], vn[SHARED ? NP : 1][4];
    u32x4 kf[KT][QV][P ? P : 1];
    const auto load_k = [&]() __attribute__((always_inline)) {
        const auto r = rows_buffer<T, D>(a.k, ks.begin + first, a.k_stride, kvh, min(KC, ks.rows - first));
        if constexpr (P > 0) {
#pragma unroll
            for (int p = 0; p < NP; ++p) buffer_dwords<4>(r, koff[p], kn[p]);
            if constexpr (SHARED) {
                const auto rv = rows_buffer<T, D>(a.v, ks.begin + first, a.v_stride, kvh, min(KC, ks.rows - first));
#pragma unroll
                for (int p = 0; p < NP; ++p) buffer_dwords<4>(rv, vsrc[p], vn[p]);
            }
        } else {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int j = 0; j < QV; ++j) {
                    uint32_t x[4];
                    buffer_dwords<4>(r, koff[t] + 64 * j, x);
                    kf[t][j][0] = u32x4{x[0], x[1], x[2], x[3]};
                }
        }
    };

    if constexpr (LISTED) first = end = 0;
    else first = (piece - pieces) * KC, end = most;
    bool more;
    int buffer = 0, rank0 = 0;  // SHARED: the step's buffer; chosen blocks before the table
    const auto begin = [&]() __attribute__((always_inline)) {
        if constexpr (LISTED) fill_table();
        more = next();
        if (more) load_k();
    };
    // what is left to see once this table is through; a workgroup's waves agree on it
    const auto again = [&]() __attribute__((always_inline)) {
        if constexpr (!LISTED) return false;
        if (w0 + TABLE >= blocks) return false;
        w0 += TABLE;
        chunk = 0;
        // SHARED waves take as many steps as the longest of them and may leave a table before its last chunk, where their
        // own count ends: whose turn a block is goes by the whole table's count
        if constexpr (SHARED) rank = rank0;
        together();
        return true;
    };
    // A step: the keys from `at` on for the rows of `mem`, of the operands in kf and (vf or LDS).
    uint32_t vf[SHARED ? 1 : KT][4][VW];  // rows 16t + 4g + i
    const auto step = [&](int at, uint64_t mem) __attribute__((always_inline)) {
        f32x4 w[NS][KT];
        u32x4 pw[NS][KT / 2 > 0 ? KT / 2 : 1][P ? P : 1];
        // ---- of a set of 16 rows: S^T
        const auto scores = [&](int n) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                f32x4 d = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < QV; ++j) {
                    if constexpr (P > 0) {
                        d = product<P ? P : 1>(kf[t][j], qf[n][j], d);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            d = __builtin_amdgcn_mfma_f32_16x16x4f32(as_float(kf[t][j][0][i]), as_float(qf[n][j][0][i]), d, 0, 0, 0);
                    }
                }
                w[n][t] = d;
            }
        };
        const auto mask = [&](int n) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + 16 * t + 4 * g + i >= lim[n]) w[n][t][i] = neg_inf();
        };
        const auto largest = [&](int n) __attribute__((always_inline)) {
            float mx = neg_inf();
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, w[n][t][i]);
            return mx;
        };
        // What weights are relative to moves only where a weight would pass 2^8: far less often than the
        // maximum, and floating point loses nothing by it.
        const auto move = [&](int n, float mx, bool in) __attribute__((always_inline)) {
            mx = max_over_groups(mx);
            const bool over = in && mx > above[n];
            // A base is rounded to 24 bits, and its weights keep what that is off by: up to 2^-0.5 .. 2^0.5 of them below
            // 2^24, all of them and more far above (scores from 1e9 on).  There it is a NaN, and so are the row's weights
            // from now on: it is computed key by key, differences first.
            float to = fmaf(mx, cs, static_cast<float>(room));
            to = !over ? base[n] : fabsf(to) < kMostBase ? to : __builtin_nanf("");
            // From base to base, as they are: the products they were rounded from differ by up to 2^-24 of them, and a row
            // would carry that on with every move.  (Before the first there is nothing to keep.)
            const float alpha = above[n] == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(base[n] - to);
            sum[n] *= alpha;
#pragma unroll
            for (int t = 0; t < C; ++t) acc[n][t] *= alpha;
            base[n] = to;
            above[n] = over ? mx + 8.0f / cs : above[n];
        };
        const auto weights = [&](int n, float off) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[n][t][i] = __builtin_amdgcn_exp2f(fmaf(w[n][t][i], cs, off));
            // The sum: in 32 bits, lane by lane; of weights in three terms, which are exact, by products with ones below.
            if constexpr (P != 3) {
                float add = 0.0f;
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    const float four = (w[n][t][0] + w[n][t][1]) + (w[n][t][2] + w[n][t][3]);
                    add = t ? add + four : four;
                }
                sum[n][0] += add;
            }
            if constexpr (P > 0) {
                // BF16: weights are rounded to bfloat16 for the product (2^-8 of each at most, of either sign); their sum is
                // of the weights before that.
#pragma unroll
                for (int u = 0; u < KT / 2; ++u) {
                    const f32x4 lo = w[n][2 * u], hi = w[n][2 * u + 1];
                    if constexpr (BF) {
                        pw[n][u][0] = u32x4{pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(hi[0], hi[1]),
                                            pack_bf16x2(hi[2], hi[3])};
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const f32x4 &h = i < 2 ? lo : hi;
                            uint32_t terms[3];
                            three_terms(h[2 * (i & 1)], h[2 * (i & 1) + 1], terms);
#pragma unroll
                            for (int p = 0; p < P; ++p) pw[n][u][p][i] = terms[p];
                        }
                    }
                }
            }
        };
        // V^T's operand of product t, 32 keys from 32u on
        const auto values = [&](int u, int t, u32x4 (&x)[P ? P : 1]) __attribute__((always_inline)) {
            if constexpr (SHARED) {
                const char *from = kt + buffer + vget[t] + u * (32 * ROW * 16);
                const u32x2 lo = transposed(from), hi = transposed(from + 16 * ROW * 16);
                x[0] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            } else if constexpr (P > 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // a pair of keys: rows 2i, 2i + 1 of the lane's eight
                    const uint32_t(&r0v)[VW] = vf[2 * u + (i >> 1)][2 * (i & 1)];
                    const uint32_t(&r1v)[VW] = vf[2 * u + (i >> 1)][2 * (i & 1) + 1];
                    if constexpr (BF) {
                        x[0][i] = __builtin_amdgcn_perm(r1v[t / 2], r0v[t / 2], t & 1 ? 0x07060302u : 0x05040100u);
                    } else {
                        uint32_t terms[3];
                        three_terms(__builtin_bit_cast(float, r0v[t]), __builtin_bit_cast(float, r1v[t]), terms);
#pragma unroll
                        for (int p = 0; p < P; ++p) x[p][i] = terms[p];
                    }
                }
            }
        };
        if constexpr (FLAT) {
            // All keys: the sets in one run without branches, so that one set's products go on under the next one's weights
            // (5,086 rows x 16 heads x 64 bf16: 142 us set by set, 137 us so, on one card in turns).
            float mx[NS];
            bool over = false;
#pragma unroll
            for (int n = 0; n < NS; ++n) scores(n);
            if (at + KC > least) {
#pragma unroll
                for (int n = 0; n < NS; ++n) mask(n);
            }
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                mx[n] = largest(n);
                over = over || mx[n] > above[n];
            }
            if (__builtin_amdgcn_ballot_w64(over) != 0) {
#pragma unroll
                for (int n = 0; n < NS; ++n) move(n, mx[n], true);
            }
            u32x4 x[KT / 2][C][P ? P : 1];
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                weights(n, -base[n]);
                if (n == 0) {
#pragma unroll
                    for (int u = 0; u < KT / 2; ++u)
#pragma unroll
                        for (int t = 0; t < C; ++t) values(u, t, x[u][t]);
                }
#pragma unroll
                for (int u = 0; u < KT / 2; ++u)
#pragma unroll
                    for (int t = 0; t < C; ++t) acc[n][t] = product<P ? P : 1>(x[u][t], pw[n][u], acc[n][t]);
            }
            return;
        }
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            // the set's rows, a bit each (all keys: all of them), and the same for the four lanes of each
            const uint32_t rows = LISTED ? static_cast<uint32_t>(mem >> (32 * half + 16 * n)) & 0xffffu
                                         : r0w + 16 * n < nrows ? 0xffffu : 0u;
            if (rows == 0) {  // none sees the block: weights 0
#pragma unroll
                for (int t = 0; t < KT; ++t) w[n][t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < KT / 2; ++u)
#pragma unroll
                    for (int p = 0; p < P; ++p) pw[n][u][p] = u32x4{0, 0, 0, 0};
                continue;
            }
            const uint32_t twice = rows | rows << 16;
            const uint64_t lanes = static_cast<uint64_t>(twice) << 32 | twice;
            scores(n);
            if (at + KC > least) mask(n);
            const float mx = largest(n);
            const auto in = [&]() __attribute__((always_inline)) { return !LISTED || __builtin_amdgcn_inverse_ballot_w64(lanes); };
            if ((__builtin_amdgcn_ballot_w64(mx > above[n]) & lanes) != 0) move(n, mx, in());
            // rows that do not see the block: weights 2^-inf
            weights(n, in() ? -base[n] : neg_inf());
        }
        if constexpr (P == 0) {
            more = next();
            if (more) load_k();
        }
        // ---- O^T
        if constexpr (P > 0) {
#pragma unroll
            for (int u = 0; u < KT / 2; ++u) {
                if constexpr (P == 3) {
                    const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
                    for (int n = 0; n < NS; ++n)
#pragma unroll
                        for (int p = P - 1; p >= 0; --p)
                            sum[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ones),
                                                                             __builtin_bit_cast(bf16x8, pw[n][u][p]), sum[n], 0, 0, 0);
                }
#pragma unroll
                for (int t = 0; t < C; ++t) {
                    u32x4 x[P ? P : 1];
                    values(u, t, x);
#pragma unroll
                    for (int n = 0; n < NS; ++n) acc[n][t] = product<P ? P : 1>(x, pw[n][u], acc[n][t]);
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < NS; ++n) {
#pragma unroll
                        for (int x = 0; x < C; ++x)
                            acc[n][x] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vf[t][i][x]), w[n][t][i],
                                                                             acc[n][x], 0, 0, 0);
                    }
        }
    };
    const auto read_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int j = 0; j < QV; ++j)
#pragma unroll
                for (int p = 0; p < P; ++p)
                    kf[t][j][p] = *reinterpret_cast<const u32x4 *>(kt + (SHARED ? buffer : 0) + p * PLANE + kget[j] + t * (16 * ROW * 16));
    };
    do {
        begin();
        if constexpr (SHARED) {
            // The workgroup's steps: those of its piece that has most.
            const int p0 = split * 2;
            int steps = 0;
            if constexpr (LISTED) {
                int chosen = 0;
                for (int e = 0; e < min(TABLE, blocks - w0); e += 64)
                    chosen += __popcll(__ballot(e + lane < min(TABLE, blocks - w0) && table[e + lane] != 0));
                const auto before = [&](int r, int p) { return r > p ? (r - p + pieces - 1) / pieces : 0; };
                for (int p = p0; p < p0 + 2; ++p)
                    steps = max(steps, (before(rank0 + chosen, p) - before(rank0, p)) * (a.block / KC));
                rank0 += chosen;
            } else {
                steps = max(0, ((most + KC - 1) / KC - p0 + pieces - 1) / pieces);
            }
            for (int it = 0; it < steps; ++it) {
                const int at = first;
                const uint64_t mem = members;
                const bool now = more;
                char *to = kt + (it & 1) * (2 * PLANE);
                if (now) {
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        *reinterpret_cast<u32x4 *>(to + kput[p]) = u32x4{kn[p][0], kn[p][1], kn[p][2], kn[p][3]};
                        *reinterpret_cast<u32x4 *>(to + PLANE + kput[p]) = u32x4{vn[p][0], vn[p][1], vn[p][2], vn[p][3]};
                    }
                }
                more = it + 1 < steps && next();
                if (more) load_k();
                // this step's rows are in LDS (the next ones' fetches go on), and all have read the step before the last
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (now && (!LISTED || ((mem >> (32 * half)) & 0xffffffffu) != 0)) {
                    buffer = (it & 1) * (2 * PLANE);
                    read_k();
                    step(at, mem);
                }
            }
        } else {
            while (more) {
                const int at = first;
                const uint64_t mem = members;
                // ---- V of this step
                {
                    const auto r = rows_buffer<T, D>(a.v, ks.begin + at, a.v_stride, kvh, min(KC, ks.rows - at));
#pragma unroll
                    for (int t = 0; t < KT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            buffer_dwords<VW>(r, HELD ? voff[HELD ? t : 0][i] : vat + (16 * t + i) * vstep, vf[t][i]);
                }
                // ---- K of this step to its operand's lanes, the next step's on its way
                if constexpr (P > 0) {
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        if constexpr (BF) {
                            *reinterpret_cast<u32x4 *>(kt + kput[p]) = u32x4{kn[p][0], kn[p][1], kn[p][2], kn[p][3]};
                        } else {
                            uint32_t lo[3], hi[3];
                            three_terms(__builtin_bit_cast(float, kn[p][0]), __builtin_bit_cast(float, kn[p][1]), lo);
                            three_terms(__builtin_bit_cast(float, kn[p][2]), __builtin_bit_cast(float, kn[p][3]), hi);
#pragma unroll
                            for (int i = 0; i < 3; ++i) *reinterpret_cast<u32x2 *>(kt + i * PLANE + kput[p]) = u32x2{lo[i], hi[i]};
                        }
                    }
                    more = next();
                    if (more) load_k();
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    read_k();
                }
                step(at, mem);
            }
        }
    } while (again());

    // ---- out
    const bool parts = a.splits > 1;
    // Channels [ch, ch + N) of a row.
    const auto put = [&]<int N>(int t, int h, int ch, const float (&y)[N], float m, float l) __attribute__((always_inline)) {
        static_assert(N % 4 == 0);
        const int64_t token = qs.begin + tok0 + t;
        if (parts) {
            const int64_t cell = (static_cast<int64_t>(split) * a.total_q + token) * a.heads + h;
            float *to = a.part_o + cell * D + ch;
#pragma unroll
            for (int w = 0; w < N; w += 4) *reinterpret_cast<f32x4 *>(to + w) = f32x4{y[w], y[w + 1], y[w + 2], y[w + 3]};
            if (ch == 0) a.part_ml[cell] = make_float2(m, l);
            return;
        }
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        T *to = static_cast<T *>(a.o) + token * a.o_stride + static_cast<int64_t>(h) * D + ch;
        if constexpr (BF) {
#pragma unroll
            for (int w = 0; w < N; w += 4)
                *reinterpret_cast<u32x2 *>(to + w) = u32x2{pack_bf16x2(y[w] * r, y[w + 1] * r), pack_bf16x2(y[w + 2] * r, y[w + 3] * r)};
        } else {
#pragma unroll
            for (int w = 0; w < N; w += 4)
                *reinterpret_cast<f32x4 *>(to + w) = f32x4{y[w] * r, y[w + 1] * r, y[w + 2] * r, y[w + 3] * r};
        }
        if (a.lse && ch == 0) a.lse[token * a.heads + h] = log_of(m, l, room);
    };
    // A set's rows whose sums are not finite are left out, and computed again from the keys that they see alone.  The test costs nothing in the loop.
    const auto finish = [&](int n, const float (&y)[4 * C], float m, float l) __attribute__((always_inline)) {
        const int r = r0 + 16 * n + c;
        float odd = 0.0f;
#pragma unroll
        for (int e = 0; e < 4 * C; ++e) odd += y[e] * 0.0f;
        uint64_t bad = parts ? 0 : __ballot(r < nrows && again_of<T>(a, l, odd));  // pieces: the join looks
        bad = (bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffffu;
        if (r < nrows && !((bad >> c) & 1u)) {
            const int t0 = r / a.group - tok0, h = kvh * a.group + r % a.group;
            if constexpr (SHARED) {  // element i*C + t is channel 16t + 4g + i
#pragma unroll
                for (int t = 0; t < C; ++t) {
                    const float four[4] = {y[t], y[C + t], y[2 * C + t], y[3 * C + t]};
                    put(t0, h, 16 * t + 4 * g, four, m, l);
                }
            } else {  // ... channel (4g + i)*C + t
                put(t0, h, 4 * g * C, y, m, l);
            }
        }
        while (bad) {
            const int w = r0 + 16 * n + __builtin_ctzll(bad);
            bad &= bad - 1;
            attend_row<T, D>(a, qs.begin + w / a.group, kvh * a.group + w % a.group, qs, ks);
        }
    };
    if constexpr (WAVES == 1) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            float y[4 * C];
#pragma unroll
            for (int e = 0; e < 4 * C; ++e) y[e] = acc[n][e % C][e / C];
            finish(n, y, base[n], P == 3 ? sum[n][0] : sum_over_groups(sum[n][0]));
        }
    } else {
        __syncthreads();  // the steps' LDS is through
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int t = 0; t < C; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave][(n * 4 + i) * C + t][lane] = acc[n][t][i];
            const float l = P == 3 ? sum[n][0] : sum_over_groups(sum[n][0]);
            if (g == 0) part_ml[wave][n][c] = make_float2(base[n], l);
        }
        __syncthreads();
        if (wave >= SETS) return;
        // a set for each wave, from the pieces of its half
        constexpr int J = 4 / HALVES;
        const int n = wave % NS, p0 = wave / NS * J;
        float m = neg_inf(), l = 0.0f, wgt[J], y[4 * C];
#pragma unroll
        for (int p = 0; p < J; ++p)
            if (part_ml[p0 + p][n][c].y != 0.0f) m = fmaxf(m, part_ml[p0 + p][n][c].x);
#pragma unroll
        for (int p = 0; p < J; ++p) {
            const float2 ml = part_ml[p0 + p][n][c];
            wgt[p] = ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - m);  // a piece without keys: 0
            l += wgt[p] * ml.y;
        }
#pragma unroll
        for (int e = 0; e < 4 * C; ++e) {
            y[e] = 0.0f;
#pragma unroll
            for (int p = 0; p < J; ++p) y[e] += wgt[p] * part[p0 + p][(n * 4 + e / C) * C + e % C][lane];
        }
        finish(wave, y, m, l);
    }
}

// Joins the pieces of each (row, head), in their order; a wave each.
template <class T, int D>
__global__ void __launch_bounds__(256) join_kernel(AttendArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t cell = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t cells = a.total_q * a.heads;
    if (cell >= cells) return;
    const int64_t row = cell / a.heads;
    const int head = static_cast<int>(cell - row * a.heads);
    const int64_t s = sequence_of_row(a.q_starts, a.sequences, row);
    if (s < 0) return;
    const Span ks = sequence_span(a.k_starts, s, a.total_k);
    // a lane for each piece (there are at most 64): its weight, 0 for one without keys (a sum that is a NaN is not 0 and stays)
    const float2 ml = lane < a.splits ? a.part_ml[lane * cells + cell] : make_float2(neg_inf(), 0.0f);
    float m = ml.y != 0.0f ? ml.x : neg_inf();
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    const float w = ml.y != 0.0f ? exp2f(ml.x - m) : 0.0f;
    float l = ml.y != 0.0f ? w * ml.y : 0.0f, o[2] = {0.0f, 0.0f};
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
    // four pieces' values on their way at a time
    for (uint64_t left = __ballot(ml.y != 0.0f); left;) {
        float wp[4], x[4][2];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int p = left ? __builtin_ctzll(left) : -1;
            left &= left - 1;
            wp[u] = 0.0f;
            x[u][0] = x[u][1] = 0.0f;
            if (p < 0) continue;
            wp[u] = __shfl(w, p, 64);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (lane + 64 * e < D) x[u][e] = a.part_o[(p * cells + cell) * D + lane + 64 * e];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) o[e] += wp[u] * x[u][e];
    }
    if (__any(again_of<T>(a, l, o[0] * 0.0f + o[1] * 0.0f))) {
        attend_row<T, D>(a, row, head, sequence_span(a.q_starts, s, a.total_q), ks);
        return;
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < D)
            store_from_f32<T>(static_cast<T *>(a.o) + row * a.o_stride + static_cast<int64_t>(head) * D + lane + 64 * e,
                              l == 0.0f ? 0.0f : o[e] * r);
    if (a.lse && lane == 0) a.lse[cell] = log_of(m, l, room_of<T>(a, ks.rows));
}

// ---------------------------------------------------------------------------
// Argument checks
// ---------------------------------------------------------------------------
constexpr int64_t kMaxStride = INT64_C(1) << 22;
constexpr int32_t kMaxTop = 4096;
constexpr int64_t kMaxBlocks = 32768;

void check_total(int64_t total) {
    // places of keys plus a tile's steps stay below 2^31, and 2^30 ends a list of blocks
    require(total >= 0 && total <= (INT64_C(1) << 29), "a row count is out of range (0 to 2^29)");
}
// Threads of a launch along x stay below 2^32.
void check_grid(int64_t groups, int threads) {
    require(groups <= 0xffffffffll / threads, "too many rows and sequences");
}
void check_shape(int32_t dtype, int32_t heads, int32_t kv_heads, int32_t head_dim, int64_t sequences, int32_t block) {
    require_dtype(dtype);
    require(kv_heads >= 1 && heads >= kv_heads && heads <= 65536 && heads % kv_heads == 0,
            "heads must be a multiple of kv_heads, at most 65536");
    require(head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128,
            "head_dim must be 32, 64, 96 or 128");
    require(sequences >= 0 && sequences <= (INT64_C(1) << 24), "sequences is out of range");
    require(block == 32 || block == 64 || block == 128, "block must be 32, 64 or 128");
}
void check_rows(const void *p, int64_t stride, int32_t heads, int32_t head_dim, int32_t dtype) {
    require(p && aligned(p, 16), "a row pointer is NULL or not 16-byte aligned");
    require(stride >= static_cast<int64_t>(heads) * head_dim, "a row stride is shorter than its heads");
    require(stride < kMaxStride && stride * dtype_size(dtype) % 16 == 0,
            "a row stride must be whole 16-byte pieces, below 2^22 elements");
}
void check_starts(const int32_t *p) { require(p && aligned(p, 4), "starts is NULL or not aligned"); }
int32_t log2_of(int32_t block) { return block == 32 ? 5 : block == 64 ? 6 : 7; }
int64_t index_rows(int64_t total_k, int64_t sequences, int32_t block) { return total_k / block + sequences; }

// How an attention call is cut: tiles of rows (an upper bound, as the lengths are on the device),
// and four waves to a tile where rows see 512 keys and more, or 128 where the tiles are few (one
// sequence of 300 rows, 12 heads: 13.3 us with one wave, 10.2 with four; 78 windows of 334 rows at
// most: 26 us with one, 44 with four, whose joins cost more than the short loops). Tiles whose
// waves are still fewer than two for each SIMD go to several workgroups, with at least 128 keys a wave.
struct AttendCut {
    int64_t tile_groups;
    int32_t splits, waves, sets;
};
AttendCut attend_cut(bool bf, int64_t total_q, int32_t heads, int32_t kv_heads, int32_t head_dim, int64_t sequences,
                     int32_t block, int32_t top, int64_t max_k) {
    constexpr int64_t kWaves = 256 * 4 * 2;
    const int64_t keys = top ? std::min<int64_t>(top * static_cast<int64_t>(block), max_k) : max_k;
    const int64_t rows = total_q * (heads / kv_heads);
    const int32_t per_tile = keys >= 512 || (keys >= 128 && (rows / 32 + sequences) * kv_heads < 1024) ? 4 : 1;
    // by tiles of 32 rows in any case, so that the workspace does not depend on the type
    const int64_t waves = std::max<int64_t>((rows / 32 + sequences) * kv_heads * per_tile, 1);
    int32_t splits = 1;
    while (splits < 64 && waves * splits * 2 <= kWaves && keys >= 256 * splits * per_tile) splits *= 2;
    // Tiles of 64 rows read each key half as often; shorter sequences would leave half of the tile empty, and FP32's
    // products take longer than its reads.
    const int32_t sets = bf && per_tile == 4 && rows >= 48 * sequences ? 4 : 2;
    const int64_t tiles = rows / (16 * sets) + sequences;
    return {per_tile == 4 ? tiles : (tiles + 3) / 4, splits, per_tile, sets};
}

using AttendFn = void (*)(AttendArgs);
// Steps of keys as registers allow: of 64 for narrow heads and two sets of rows, of 32,
// FP32's widest heads of 16.
template <class T, int D, int SETS, int WAVES>
AttendFn pick_step(bool listed, int32_t block) {
    constexpr bool BF = sizeof(T) == 2;
    constexpr int NS = SETS == 4 && D <= 64 ? 4 : 2, HALVES = SETS / NS;
    if constexpr (BF && D <= 64 && NS == 2 && WAVES == 4)
        if (block >= 64 || !listed)
            return listed ? attend_kernel<T, D, 64, NS, true, WAVES, HALVES> : attend_kernel<T, D, 64, NS, false, WAVES, HALVES>;
    constexpr int KC = !BF && D > 64 ? 16 : 32;
    return listed ? attend_kernel<T, D, KC, NS, true, WAVES, HALVES> : attend_kernel<T, D, KC, NS, false, WAVES, HALVES>;
}
template <class T, int SETS, int WAVES>
AttendFn pick_dim(int32_t d, bool listed, int32_t block) {
    switch (d) {
        case 32: return pick_step<T, 32, SETS, WAVES>(listed, block);
        case 64: return pick_step<T, 64, SETS, WAVES>(listed, block);
        case 96: return pick_step<T, 96, SETS, WAVES>(listed, block);
        default: return pick_step<T, 128, SETS, WAVES>(listed, block);
    }
}
template <class T>
AttendFn pick_attend(int32_t d, bool listed, int32_t block, const AttendCut &cut) {
    if constexpr (sizeof(T) == 2)
        if (cut.sets == 4) return pick_dim<T, 4, 4>(d, listed, block);
    return cut.waves == 4 ? pick_dim<T, 2, 4>(d, listed, block) : pick_dim<T, 2, 1>(d, listed, block);
}
template <class T>
AttendFn pick_join(int32_t d) {
    return d == 32 ? join_kernel<T, 32> : d == 64 ? join_kernel<T, 64> : d == 96 ? join_kernel<T, 96> : join_kernel<T, 128>;
}

}  // namespace
}  // namespace s3dx

using namespace s3dx;

extern "C" {

S3DX_API s3dx_status s3dx_block_index_rows(int64_t total_k, int64_t sequences, int32_t block, int64_t *rows,
                                           char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        require(rows, "rows is NULL");
        check_total(total_k);
        check_shape(S3DX_F32, 1, 1, 64, sequences, block);
        *rows = index_rows(total_k, sequences, block);
    });
}

S3DX_API s3dx_status s3dx_block_index(const void *k, int32_t dtype, int64_t total_k, int32_t kv_heads, int32_t head_dim,
                                      int64_t k_stride, const int32_t *k_starts, int64_t sequences, int32_t block,
                                      int8_t *codes, float *scale, s3dx_stream stream, char *error,
                                      uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        check_total(total_k);
        check_shape(dtype, kv_heads, kv_heads, head_dim, sequences, block);
        if (total_k == 0 || sequences == 0) return;
        check_rows(k, k_stride, kv_heads, head_dim, dtype);
        check_starts(k_starts);
        require(codes && aligned(codes, 16) && scale && aligned(scale, 4), "codes or scale is NULL or not aligned");
        const IndexArgs a = {k, k_starts, total_k, k_stride, sequences, index_rows(total_k, sequences, block),
                             kv_heads, head_dim, block, log2_of(block), codes, scale};
        const int per = 256 / head_dim;
        require((kv_heads + per - 1) / per <= 65535, "too many heads");
        check_grid(a.rows, 256);
        (dtype == S3DX_BF16 ? index_kernel<uint16_t> : index_kernel<float>)<<<
            dim3(static_cast<unsigned>(a.rows), static_cast<unsigned>((kv_heads + per - 1) / per)), dim3(256), 0,
            as_stream(stream)>>>(a);
        launch_check("block index");
    });
}

S3DX_API s3dx_status s3dx_block_select(const void *q, int32_t dtype, int64_t total_q, int64_t total_k, int32_t heads,
                                       int32_t kv_heads, int32_t head_dim, int64_t q_stride, const int32_t *q_starts,
                                       const int32_t *k_starts, int64_t sequences, int32_t block, int32_t top,
                                       int64_t max_k, const int8_t *codes, const float *scale, int32_t flags,
                                       int32_t *selected, s3dx_stream stream, char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        check_total(total_q);
        check_total(total_k);
        check_shape(dtype, heads, kv_heads, head_dim, sequences, block);
        require(top >= 1 && top <= kMaxTop, "top must be 1 to 4096");
        require((flags & ~(S3DX_BLOCK_CAUSAL | S3DX_BLOCK_NEAR)) == 0, "unknown flags");
        require(max_k >= 0 && max_k <= kMaxBlocks * block, "max_k must be 0 to 32768 * block");
        if (total_q == 0 || sequences == 0) return;
        check_rows(q, q_stride, heads, head_dim, dtype);
        check_starts(q_starts);
        check_starts(k_starts);
        require(selected && aligned(selected, 4), "selected is NULL or not aligned");
        require(total_k == 0 || (codes && aligned(codes, 16) && scale && aligned(scale, 4)),
                "codes or scale is NULL or not aligned");
        SelectArgs a = {q, q_starts, k_starts, codes, scale, selected, total_q, total_k, q_stride, sequences,
                        index_rows(total_k, sequences, block), kv_heads, heads / kv_heads, head_dim, block, log2_of(block), top,
                        static_cast<int32_t>((std::min(max_k, total_k) + block - 1) / block), flags, 0};
        // Queries of a workgroup: 16, unless those leave most compute units without one or their keys take more than
        // 64 KiB of LDS (1,024 blocks; 4,096 of four queries).
        const int64_t rows = total_q * kv_heads;
        require(rows <= std::numeric_limits<int32_t>::max(), "total_q * kv_heads is out of range");
        const int qt = rows >= 16 * 512 && a.most_blocks <= 1024 ? 16 : rows >= 4 * 256 && a.most_blocks <= 4096 ? 4 : 1;
        const int team = select_team(qt);
        a.run = std::max((a.most_blocks + team - 1) / team + 3, 4) / 4 * 4;
        const bool bf = dtype == S3DX_BF16;
        a.run = a.run <= 4 ? 4 : a.run <= 8 ? 8 : a.run <= 16 ? 16 : a.run;
        const auto pick = [&](auto run) {
            constexpr int R = decltype(run)::value;
            if (qt == 16) return bf ? select_kernel<uint16_t, 16, R> : select_kernel<float, 16, R>;
            if (qt == 4) return bf ? select_kernel<uint16_t, 4, R> : select_kernel<float, 4, R>;
            return bf ? select_kernel<uint16_t, 1, R> : select_kernel<float, 1, R>;
        };
        const auto kernel = a.run == 4    ? pick(std::integral_constant<int, 4>{})
                            : a.run == 8  ? pick(std::integral_constant<int, 8>{})
                            : a.run == 16 ? pick(std::integral_constant<int, 16>{})
                                          : pick(std::integral_constant<int, 0>{});
        const size_t lds = static_cast<size_t>(qt) * team * a.run * 4;
        if (lds > 65536 - 4096)
            hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                          hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)),
                      "hipFuncSetAttribute");
        const int64_t grid = (total_q / qt + sequences) * kv_heads;
        check_grid(grid, select_threads(qt));
        kernel<<<dim3(static_cast<unsigned>(grid)), dim3(select_threads(qt)), lds, as_stream(stream)>>>(a);
        launch_check("block select");
    });
}

S3DX_API s3dx_status s3dx_block_attention_workspace_size(int64_t total_q, int32_t heads, int32_t kv_heads,
                                                         int32_t head_dim, int64_t sequences, int32_t block,
                                                         int32_t top, int64_t max_k, uint64_t *bytes, char *error,
                                                         uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        require(bytes, "bytes is NULL");
        check_total(total_q);
        check_total(max_k);
        check_shape(S3DX_F32, heads, kv_heads, head_dim, sequences, block);
        require(top >= 0 && top <= kMaxTop, "top must be 0 to 4096");
        const AttendCut cut = attend_cut(true, total_q, heads, kv_heads, head_dim, sequences, block, top, max_k);
        *bytes = 0;
        if (cut.splits == 1) return;
        Sizer z;
        z.take<float>(static_cast<uint64_t>(cut.splits) * total_q * heads * head_dim);
        z.take<float2>(static_cast<uint64_t>(cut.splits) * total_q * heads);
        *bytes = z.used;
    });
}

S3DX_API s3dx_status s3dx_block_attention(const void *q, const void *k, const void *v, int32_t dtype, int64_t total_q,
                                          int64_t total_k, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                          int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                          const int32_t *q_starts, const int32_t *k_starts, int64_t sequences,
                                          int32_t block, int64_t max_k, const int32_t *selected, int32_t top,
                                          float softmax_scale, int32_t flags, void *o, int64_t o_stride, float *lse,
                                          void *workspace, uint64_t workspace_bytes, s3dx_stream stream, char *error,
                                          uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        check_total(total_q);
        check_total(total_k);
        check_total(max_k);
        check_shape(dtype, heads, kv_heads, head_dim, sequences, block);
        require(selected ? top >= 1 && top <= kMaxTop : top == 0, "top must be 1 to 4096, or 0 without selected");
        require((flags & ~S3DX_BLOCK_CAUSAL) == 0, "unknown flags");
        require(softmax_scale > 0.0f && softmax_scale < 1e6f, "softmax_scale must be above 0 and below 1e6");
        if (total_q == 0 || sequences == 0) return;
        check_rows(q, q_stride, heads, head_dim, dtype);
        check_rows(o, o_stride, heads, head_dim, dtype);
        if (total_k) {
            check_rows(k, k_stride, kv_heads, head_dim, dtype);
            check_rows(v, v_stride, kv_heads, head_dim, dtype);
        }
        check_starts(q_starts);
        check_starts(k_starts);
        require(!selected || aligned(selected, 4), "selected is not aligned");
        require(!lse || aligned(lse, 4), "lse is not aligned");
        require(total_q * heads <= std::numeric_limits<int32_t>::max(), "total_q * heads is out of range");
        AttendCut cut = attend_cut(dtype == S3DX_BF16, total_q, heads, kv_heads, head_dim, sequences, block, top, max_k);
        if (flags & S3DX_BLOCK_CAUSAL) cut.tile_groups = (cut.tile_groups + 7) / 8 * 8;  // see the kernel's order of tiles
        AttendArgs a = {q, k, v, o, lse, q_starts, k_starts, selected, total_q, total_k, q_stride, k_stride, v_stride, o_stride,
                        sequences, heads, heads / kv_heads, kv_heads, block, log2_of(block), top,
                        flags & S3DX_BLOCK_CAUSAL, cut.splits, static_cast<int32_t>(cut.tile_groups), softmax_scale, nullptr,
                        nullptr};
        if (cut.splits > 1) {
            require(workspace && aligned(workspace, 16), "workspace is NULL or not 16-byte aligned");
            Carver w(workspace, workspace_bytes);
            a.part_o = w.take<float>(static_cast<uint64_t>(cut.splits) * total_q * heads * head_dim);
            a.part_ml = w.take<float2>(static_cast<uint64_t>(cut.splits) * total_q * heads);
        }
        const int64_t grid = cut.tile_groups * kv_heads * cut.splits;
        check_grid(grid, 256);
        const bool bf = dtype == S3DX_BF16;
        (bf ? pick_attend<uint16_t>(head_dim, selected, block, cut) : pick_attend<float>(head_dim, selected, block, cut))<<<
            dim3(static_cast<unsigned>(grid)), dim3(256), 0, as_stream(stream)>>>(a);
        launch_check("block attention");
        if (cut.splits > 1) {
            (bf ? pick_join<uint16_t>(head_dim) : pick_join<float>(head_dim))<<<
                dim3(static_cast<unsigned>((total_q * heads + 3) / 4)), dim3(256), 0, as_stream(stream)>>>(a);
            launch_check("block attention join");
        }
    });
}

}  // extern "C"
