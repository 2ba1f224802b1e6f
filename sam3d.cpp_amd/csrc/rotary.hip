// Rotary positions with several axes, and the norms of queries and keys with
// the rotation in the same pass.
//
// Per head row x[0, d): y = x * rsqrt(mean(x^2) + eps) * gain, then each pair
// (a, b) of channels turns by the angle p * f, p the row's position on the
// pair's axis: (a cos - b sin, a sin + b cos).  For attention between the sparse
// blocks (the SLat flow's place for it is slat_flow_graph.cpp:304-434) in models
// whose heads carry their rows' places; the reference's own flow adds an absolute
// embedding to its coarse rows instead (sparse_ops.cpp:49-173).
#include <cmath>
#include <vector>

#include "common.hpp"

// Angles as parts of a turn: frequency f rad per step is f / 2 pi turns, kept
// modulo one turn as a 64-bit fraction.  position * fraction modulo 2^64 is
// then the angle modulo one turn, off by at most 2^31 * 2^-64 turns for any
// int32 position: far positions cost nothing.
constexpr int kMaxPairs = 128;
constexpr int kMaxAxes = 8;
struct s3dx_rotary {
    int32_t head_dim, axes, pairs, pairing;
    uint64_t turns[kMaxPairs];
    uint8_t axis[kMaxPairs];
};

namespace s3dx {
namespace {

// A launch's table, by value: no device copy, nothing for calls to share.
struct TurnTable {
    uint64_t turns[kMaxPairs];
    uint8_t axis[kMaxPairs];
};

struct HeadRows {
    const void *x;
    void *y;
    const float *gain;  // NULL: none
    int64_t x_stride, y_stride;
    int32_t heads;
};

struct TurnArgs {
    HeadRows part[2];  // queries, keys
    const int32_t *positions;
    int64_t position_stride, first, n;  // rows [first, n)
    int32_t d, pairs, halves, inverse, norm, gain_stride, rows, lanes_log2;
    float eps;
};
constexpr int kMaxRows = 32;    // of a workgroup
constexpr int kMaxTurns = 512;  // pairs of those rows
// Heads whose squares' sum passes 2^128 (|x| of 2^60 and more) are summed again smaller: 256 squares of at most 2^116,
// beside which eps is nothing.
constexpr float kLess = 0x1p-70f;

// cos and sin of a 0.64 fixed-point part of a turn.  The quarter turn is split
// off in integers, so that the float holds at most an eighth of a turn.
__device__ __forceinline__ void turn_cos_sin(uint64_t phase, float *c, float *s) {
    const uint32_t top = static_cast<uint32_t>(phase >> 32);
    const uint32_t quarter = (top + 0x20000000u) >> 30;
    const int32_t rest = static_cast<int32_t>(top - (quarter << 30));
    float sn, cs;
    sincospif(static_cast<float>(rest) * 0x1p-31f, &sn, &cs);
    const bool swap = quarter & 1u;
    const float a = swap ? sn : cs, b = swap ? cs : sn;
    *c = (quarter == 1u || quarter == 2u) ? -a : a;
    *s = (quarter & 2u) ? -b : b;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// 8 elements at p (16-byte aligned) as floats, and back, rounded to nearest even.
template <class T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    constexpr int N = 8 * static_cast<int>(sizeof(T)) / 16;
    uint4 t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = reinterpret_cast<const uint4 *>(p)[i];
    const uint32_t *w = reinterpret_cast<const uint32_t *>(t);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        v[e] = sizeof(T) == 4 ? __builtin_bit_cast(float, w[e])
                              : __builtin_bit_cast(float, e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
}
template <class T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                                   pack_bf16x2(v[6], v[7]));
    } else {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
}

// A workgroup takes `rows` rows: it makes their angles' cosines and sines once, in LDS, for all heads;
// then its waves take the rows' heads.  The work is the memory's: every head is read
// and written once (28,265 rows x 16 heads x 64 BF16, 116 MB: 25 us at a copy's rate).
//
// WHOLE: a lane owns 16 channels, two pieces of 8 (bf16: 16 bytes): neighbours where
// neighbours are paired, else the piece of the first channels and that of the second; lane groups of
// a power of two take a head, so a wave takes several side by side.  For head_dim a multiple of 16 and
// aligned rows.  MEET: the same for halves that are not whole pieces: a lane keeps neighbouring
// channels and reads their partners in LDS (a form of its own, as its LDS costs the others a
// quarter of their rate).  Else, SINGLE, one wave takes a head, a pair (or a channel that does
// not turn) at a time in each lane, at any width and alignment (39,729 rows of 9 heads of 32
// in halves of 6 pairs: 190 us that way).  In all of them a wave reads the heads that it
// writes before it writes any, so y may be x.
enum Form { SINGLE, WHOLE, MEET };
template <class TI, class TO, int FORM>
__global__ void __launch_bounds__(256) turn_kernel(TurnArgs a, TurnTable t) {
    __shared__ float2 turns[kMaxTurns];
    constexpr int STAGE = 17;  // floats of a lane, one more than its channels: neighbours in other banks
    __shared__ float stage[FORM == MEET ? 4 : 1][FORM == MEET ? 64 * STAGE : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row0 = a.first + static_cast<int64_t>(blockIdx.x) * a.rows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(a.rows), a.n - row0));
    for (int e = threadIdx.x; e < rows * a.pairs; e += 256) {
        const int r = e / a.pairs, j = e - r * a.pairs;
        const int64_t pos = a.positions[(row0 + r) * a.position_stride + t.axis[j]];
        float c, s;
        turn_cos_sin(static_cast<uint64_t>(pos) * t.turns[j], &c, &s);
        turns[e] = make_float2(c, a.inverse ? -s : s);
    }
    __syncthreads();
    const int heads = a.part[0].heads + a.part[1].heads;
    const int lanes = FORM != SINGLE ? 1 << a.lanes_log2 : 64, side = 64 / lanes;  // lanes of a head, heads of a wave
    const int sets = (heads + side - 1) / side;
    for (int item = wave; item < rows * sets; item += 4) {
        const int r = item / sets;
        int head = (item - r * sets) * side + lane / lanes;
        const bool k = head >= a.part[0].heads;
        const HeadRows &p = a.part[k ? 1 : 0];
        const bool here = head < heads;
        if (k) head -= a.part[0].heads;
        const TI *from = static_cast<const TI *>(p.x) + (row0 + r) * p.x_stride + static_cast<int64_t>(head) * a.d;
        TO *y = static_cast<TO *>(p.y) + (row0 + r) * p.y_stride + static_cast<int64_t>(head) * a.d;
        const float *gain = p.gain ? p.gain + static_cast<int64_t>(head) * a.gain_stride : nullptr;
        if constexpr (FORM != SINGLE) {
            const int l = lane & (lanes - 1), turning = a.pairs / 8;
            const bool active = here && l < a.d / 16;
            // this lane's two pieces of 8 channels
            const bool halves = a.halves && FORM == WHOLE;
            const int c0 = halves && l < turning ? 8 * l : 16 * l;
            const int c1 = halves && l < turning ? c0 + a.pairs : c0 + 8;
            float u[8], v[8], gu[8], gv[8];
            if (active) {
                load8(from + c0, u);
                load8(from + c1, v);
                if (gain) {
                    load8(gain + c0, gu);
                    load8(gain + c1, gv);
                }
            }
            float scale = 1.0f;
            if (a.norm) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += active ? u[e] * u[e] + v[e] * v[e] : 0.0f;
                for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor(sum, o, 64);
                scale = rsqrtf(sum / static_cast<float>(a.d) + a.eps);
                if (!(sum < __builtin_inff())) {  // the same for a head's lanes
                    sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum += active ? (u[e] * kLess) * (u[e] * kLess) + (v[e] * kLess) * (v[e] * kLess) : 0.0f;
                    for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor(sum, o, 64);
                    scale = rsqrtf(sum / static_cast<float>(a.d)) * kLess;
                }
            }
            if (FORM == WHOLE && !active) continue;
            if (a.norm) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    u[e] *= gain ? gu[e] * scale : scale;
                    v[e] *= gain ? gv[e] * scale : scale;
                }
            }
            // pairs 8l..8l+7, in the table's order
            const float2 *cs = &turns[r * a.pairs + 8 * l];
            if constexpr (FORM == MEET) {
                float *own = &stage[wave][lane * STAGE];
                if (active) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) own[e] = u[e], own[8 + e] = v[e];
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the head's lanes are this wave's
                if (active) {
                    const float *first = &stage[wave][(lane - l) * STAGE];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int c = 16 * l + e;
                        if (c >= 2 * a.pairs) continue;
                        const int j = c < a.pairs ? c : c - a.pairs, other = c < a.pairs ? c + a.pairs : j;
                        const float2 q = turns[r * a.pairs + j];
                        const float x1 = first[(other >> 4) * STAGE + (other & 15)];
                        float &x0 = e < 8 ? u[e & 7] : v[e & 7];
                        x0 = c < a.pairs ? x0 * q.x - x1 * q.y : x1 * q.y + x0 * q.x;
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // read before the next heads take the place
                if (!active) continue;
            } else if (halves) {
                if (l < turning) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 q = cs[e];
                        const float first = u[e] * q.x - v[e] * q.y;
                        v[e] = u[e] * q.y + v[e] * q.x;
                        u[e] = first;
                    }
                }
            } else {
                // channels behind the last pair stay as they are (an infinity among them too)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (8 * l + e < a.pairs) {
                        const float2 q = cs[e];
                        const float first = u[2 * e] * q.x - u[2 * e + 1] * q.y;
                        u[2 * e + 1] = u[2 * e] * q.y + u[2 * e + 1] * q.x;
                        u[2 * e] = first;
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (8 * l + 4 + e < a.pairs) {
                        const float2 q = cs[4 + e];
                        const float first = v[2 * e] * q.x - v[2 * e + 1] * q.y;
                        v[2 * e + 1] = v[2 * e] * q.y + v[2 * e + 1] * q.x;
                        v[2 * e] = first;
                    }
            }
            store8(y + c0, u);
            store8(y + c1, v);
        } else {
            const int step = a.halves ? 1 : 2, apart = a.halves ? a.pairs : 1;
            float x[8], g[8];  // the pairs' first and second channels, the rest
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int j = lane + 64 * (q >> 1);
                const int c = q < 4 ? j * step + (q & 1) * apart : 2 * a.pairs + lane + 64 * (q - 4);
                const bool any = q < 4 ? j < a.pairs : c < a.d;
                x[q] = any ? load_as_f32<TI>(from + c) : 0.0f;
                g[q] = gain && any ? gain[c] : 1.0f;
            }
            if (a.norm) {
                const auto squares = [&]() __attribute__((always_inline)) {
                    float sum = 0.0f;
#pragma unroll
                    for (int q = 0; q < 8; ++q) sum += x[q] * x[q];
                    return wave_sum(sum);
                };
                float sum = squares(), eps = a.eps;
                if (!(sum < __builtin_inff())) {  // the same for the wave
#pragma unroll
                    for (int q = 0; q < 8; ++q) x[q] *= kLess;
                    sum = squares(), eps = 0.0f;
                }
                const float scale = rsqrtf(sum / static_cast<float>(a.d) + eps);
#pragma unroll
                for (int q = 0; q < 8; ++q) x[q] *= g[q] * scale;
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int j = lane + 64 * q, c = j * step;
                if (j >= a.pairs) continue;
                const float2 cs = turns[r * a.pairs + j];
                store_from_f32<TO>(y + c, x[2 * q] * cs.x - x[2 * q + 1] * cs.y);
                store_from_f32<TO>(y + c + apart, x[2 * q] * cs.y + x[2 * q + 1] * cs.x);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = 2 * a.pairs + lane + 64 * q;
                if (c < a.d) store_from_f32<TO>(y + c, x[4 + q]);
            }
        }
    }
}

using TurnFn = void (*)(TurnArgs, TurnTable);
template <int FORM>
TurnFn pick_turn(int32_t in, int32_t out) {
    if (in == S3DX_BF16) return out == S3DX_BF16 ? turn_kernel<uint16_t, uint16_t, FORM> : turn_kernel<uint16_t, float, FORM>;
    return out == S3DX_BF16 ? turn_kernel<float, uint16_t, FORM> : turn_kernel<float, float, FORM>;
}

bool whole_pieces(const HeadRows &p, int32_t in, int32_t out) {
    return p.heads == 0 || (aligned(p.x, 16) && aligned(p.y, 16) && aligned(p.gain, 16) &&
                            p.x_stride * dtype_size(in) % 16 == 0 && p.y_stride * dtype_size(out) % 16 == 0);
}

void check_rows(const HeadRows &p, int32_t d, int64_t n, int32_t in, int32_t out) {
    require(p.heads >= 1 && p.heads <= 65536, "heads must be 1 to 65536");
    const int64_t least = static_cast<int64_t>(p.heads) * d;
    require(p.x_stride >= least && p.y_stride >= least, "a row stride is shorter than heads * head_dim");
    require(p.x_stride <= (INT64_C(1) << 40) && p.y_stride <= (INT64_C(1) << 40), "a row stride is above 2^40");
    if (n == 0) return;
    require(p.x && p.y, "x or y is NULL");
    require(aligned(p.x, dtype_size(in)) && aligned(p.y, dtype_size(out)), "x or y is not aligned to its elements");
    require(!p.gain || aligned(p.gain, 4), "gain is not aligned");
    require(p.x != p.y || (in == out && (n == 1 || p.x_stride == p.y_stride)),
            "in place needs the same dtype and stride for x and y");
}

void launch_turn(TurnArgs a, const s3dx_rotary *rotary, int32_t in, int32_t out, hipStream_t stream) {
    if (a.n == 0) return;
    TurnTable t = {};
    if (rotary) {
        std::memcpy(t.turns, rotary->turns, sizeof t.turns);
        std::memcpy(t.axis, rotary->axis, sizeof t.axis);
    }
    const bool vec = a.d % 16 == 0 && whole_pieces(a.part[0], in, out) && whole_pieces(a.part[1], in, out);
    while ((16 << a.lanes_log2) < a.d) ++a.lanes_log2;
    // Four rows to a workgroup, unless that leaves compute units without one; more of narrow rows, up to
    // 4,608 channels, as a workgroup's launch and first loads take longer than the rest of four of them
    // (39,729 rows of 288 channels: 33 us with 4 rows, 23 us with 16; 2,048 channels: no difference).
    const int64_t channels = static_cast<int64_t>(a.part[0].heads + a.part[1].heads) * a.d;
    a.rows = a.n >= 4 * 256 ? 4 : 1;
    while (a.rows > 1 && a.rows < kMaxRows && 2 * a.rows * channels <= 4608 && 2 * a.rows * a.pairs <= kMaxTurns &&
           a.n >= 2 * a.rows * 1024)
        a.rows *= 2;
    const TurnFn fn = !vec                            ? pick_turn<SINGLE>(in, out)
                      : a.halves && a.pairs % 8 != 0 ? pick_turn<MEET>(in, out)
                                                     : pick_turn<WHOLE>(in, out);
    // A launch's threads stay below 2^32: 2^20 workgroups at a time.
    const int64_t n = a.n, most = a.rows * (INT64_C(1) << 20);
    for (; a.first < n; a.first += most) {
        a.n = std::min(n, a.first + most);
        fn<<<dim3(static_cast<unsigned>((a.n - a.first + a.rows - 1) / a.rows)), dim3(256), 0, stream>>>(a, t);
    }
    launch_check("rotary");
}

void check_turn(const s3dx_rotary *rotary, const int32_t *positions, int64_t position_stride, int64_t n,
                int64_t heads) {
    require(n >= 0 && n <= std::numeric_limits<int32_t>::max(), "n is out of range");
    require(n * heads <= (INT64_C(1) << 33), "n * heads is above 2^33");
    if (!rotary) return;
    require(position_stride >= rotary->axes && position_stride <= (INT64_C(1) << 31),
            "position_stride must be at least the axes");
    require(n == 0 || (positions && aligned(positions, 4)), "positions is NULL or not aligned");
}

}  // namespace
}  // namespace s3dx

using namespace s3dx;

extern "C" {

S3DX_API s3dx_status s3dx_rotary_create(int32_t head_dim, int32_t axes, int32_t pairs, const int32_t *host_axis,
                                        const double *host_frequency, int32_t pairing, s3dx_rotary **out,
                                        char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        require(out, "out is NULL");
        *out = nullptr;
        require(head_dim >= 1 && head_dim <= 2 * kMaxPairs, "head_dim must be 1 to 256");
        require(axes >= 1 && axes <= kMaxAxes, "axes must be 1 to 8");
        require(pairs >= 1 && pairs <= head_dim / 2, "pairs must be 1 to head_dim / 2");
        require(host_axis && host_frequency, "axis or frequency is NULL");
        require(pairing == S3DX_ROTARY_ADJACENT || pairing == S3DX_ROTARY_HALVES, "unknown pairing");
        for (int32_t j = 0; j < pairs; ++j) {
            require(host_axis[j] >= 0 && host_axis[j] < axes, "a pair's axis is out of range");
            require(std::fabs(host_frequency[j]) <= 1e6, "a frequency is not finite or above 1e6");
        }
        s3dx_rotary *r = new s3dx_rotary();
        r->head_dim = head_dim;
        r->axes = axes;
        r->pairs = pairs;
        r->pairing = pairing;
        for (int32_t j = 0; j < pairs; ++j) {
            const long double t = static_cast<long double>(host_frequency[j]) / 6.283185307179586476925286766559L;
            const long double part = (t - std::floor(t)) * 18446744073709551616.0L;
            // a tiny negative frequency's part rounds to a whole turn, which is none
            r->turns[j] = part >= 18446744073709551615.0L ? 0 : static_cast<uint64_t>(part);
            r->axis[j] = static_cast<uint8_t>(host_axis[j]);
        }
        *out = r;
    });
}

S3DX_API void s3dx_rotary_free(s3dx_rotary *rotary) { delete rotary; }

S3DX_API s3dx_status s3dx_rotary_apply(const s3dx_rotary *rotary, int32_t inverse, const void *x, int32_t x_dtype,
                                       int64_t n, int32_t heads, int64_t x_stride, const int32_t *positions,
                                       int64_t position_stride, void *y, int32_t y_dtype, int64_t y_stride,
                                       s3dx_stream stream, char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        require(rotary, "rotary is NULL");
        require(inverse == 0 || inverse == 1, "inverse must be 0 or 1");
        require_dtype(x_dtype);
        require_dtype(y_dtype);
        check_turn(rotary, positions, position_stride, n, heads);
        TurnArgs a = {};
        a.part[0] = {x, y, nullptr, x_stride, y_stride, heads};
        check_rows(a.part[0], rotary->head_dim, n, x_dtype, y_dtype);
        a.positions = positions;
        a.position_stride = position_stride;
        a.n = n;
        a.d = rotary->head_dim;
        a.pairs = rotary->pairs;
        a.halves = rotary->pairing == S3DX_ROTARY_HALVES;
        a.inverse = inverse;
        launch_turn(a, rotary, x_dtype, y_dtype, as_stream(stream));
    });
}

S3DX_API s3dx_status s3dx_qk_norm_rotary(const s3dx_rotary *rotary, const int32_t *positions, int64_t position_stride,
                                         const void *q, int32_t q_heads, int64_t q_stride, const float *q_gain,
                                         const void *k, int32_t k_heads, int64_t k_stride, const float *k_gain,
                                         int32_t gain_per_head, int32_t dtype, int64_t n, int32_t head_dim, float eps,
                                         void *q_out, int64_t q_out_stride, void *k_out, int64_t k_out_stride,
                                         int32_t out_dtype, s3dx_stream stream, char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        require_dtype(dtype);
        require_dtype(out_dtype);
        require(head_dim >= 1 && head_dim <= 2 * kMaxPairs, "head_dim must be 1 to 256");
        require(!rotary || rotary->head_dim == head_dim, "rotary was made for another head_dim");
        require(eps > 0.0f && eps <= 1.0f, "eps must be above 0 and at most 1");
        require(gain_per_head == 0 || gain_per_head == 1, "gain_per_head must be 0 or 1");
        require(k_heads >= 0 && (k_heads > 0 || (!k && !k_out && !k_gain)), "k without k_heads");
        require(q_heads >= 1 && q_heads <= 65536 && k_heads <= 65536, "heads must be 1 to 65536");
        check_turn(rotary, positions, position_stride, n, static_cast<int64_t>(q_heads) + k_heads);
        TurnArgs a = {};
        a.part[0] = {q, q_out, q_gain, q_stride, q_out_stride, q_heads};
        check_rows(a.part[0], head_dim, n, dtype, out_dtype);
        a.part[1] = {k, k_out, k_gain, k_stride, k_out_stride, k_heads};
        if (k_heads) check_rows(a.part[1], head_dim, n, dtype, out_dtype);
        a.positions = positions;
        a.position_stride = position_stride;
        a.n = n;
        a.d = head_dim;
        if (rotary) {
            a.pairs = rotary->pairs;
            a.halves = rotary->pairing == S3DX_ROTARY_HALVES;
        }
        a.norm = 1;
        a.gain_stride = gain_per_head ? head_dim : 0;
        a.eps = eps;
        launch_turn(a, rotary, dtype, out_dtype, as_stream(stream));
    });
}

}  // extern "C"
