// Rotary positions with several axes, and the norms of queries and keys with
// the rotation in the same pass.
//
// Per head row x[0, d): y = x * rsqrt(mean(x^2) + eps) * gain, then each pair
// (a, b) of channels turns by the angle p * f, p the row's position on the
// pair's axis: (a cos - b sin, a sin + b cos).  The transformer blocks of the
// SLat flow norm and turn their heads this way between the sparse blocks
// (slat_flow_graph.cpp:304-434); the reference's graph has an op for each step.
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
    int64_t position_stride, n;
    int32_t d, pairs, halves, inverse, norm, gain_stride;
    float eps;
};

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

// One wave per head row, any head_dim up to 256, any stride and alignment: lane
// l holds pairs l and l + 64 and, of the channels that are not turned, every
// 64th.  A lane reads what it writes and nothing else, so y may be x.
template <class TI, class TO>
__global__ void __launch_bounds__(256) turn_kernel(TurnArgs a, TurnTable t) {
    const int lane = threadIdx.x & 63;
    const int64_t heads = a.part[0].heads + a.part[1].heads;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (item >= a.n * heads) return;
    const int64_t row = item / heads;
    int32_t head = static_cast<int32_t>(item - row * heads);
    const HeadRows &p = head < a.part[0].heads ? a.part[0] : a.part[1];
    if (head >= a.part[0].heads) head -= a.part[0].heads;
    const TI *x = static_cast<const TI *>(p.x) + row * p.x_stride + static_cast<int64_t>(head) * a.d;
    TO *y = static_cast<TO *>(p.y) + row * p.y_stride + static_cast<int64_t>(head) * a.d;
    const float *gain = p.gain ? p.gain + static_cast<int64_t>(head) * a.gain_stride : nullptr;
    const int step = a.halves ? 1 : 2, apart = a.halves ? a.pairs : 1;
    float first[2], second[2], rest[4];
    float sum = 0.0f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int j = lane + 64 * q, c = j * step;
        first[q] = second[q] = 0.0f;
        if (j >= a.pairs) continue;
        first[q] = load_as_f32<TI>(x + c);
        second[q] = load_as_f32<TI>(x + c + apart);
        sum += first[q] * first[q] + second[q] * second[q];
        if (gain) {
            first[q] *= gain[c];
            second[q] *= gain[c + apart];
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int c = 2 * a.pairs + lane + 64 * q;
        rest[q] = 0.0f;
        if (c >= a.d) continue;
        rest[q] = load_as_f32<TI>(x + c);
        sum += rest[q] * rest[q];
        if (gain) rest[q] *= gain[c];
    }
    const float r = a.norm ? rsqrtf(wave_sum(sum) / static_cast<float>(a.d) + a.eps) : 1.0f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int j = lane + 64 * q, c = j * step;
        if (j >= a.pairs) continue;
        const int64_t pos = a.positions[row * a.position_stride + t.axis[j]];
        float cs, sn;
        turn_cos_sin(static_cast<uint64_t>(pos) * t.turns[j], &cs, &sn);
        if (a.inverse) sn = -sn;
        store_from_f32<TO>(y + c, (first[q] * cs - second[q] * sn) * r);
        store_from_f32<TO>(y + c + apart, (first[q] * sn + second[q] * cs) * r);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int c = 2 * a.pairs + lane + 64 * q;
        if (c < a.d) store_from_f32<TO>(y + c, rest[q] * r);
    }
}

using TurnFn = void (*)(TurnArgs, TurnTable);
TurnFn pick_turn(int32_t in, int32_t out) {
    if (in == S3DX_BF16) return out == S3DX_BF16 ? turn_kernel<uint16_t, uint16_t> : turn_kernel<uint16_t, float>;
    return out == S3DX_BF16 ? turn_kernel<float, uint16_t> : turn_kernel<float, float>;
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

void launch_turn(const TurnArgs &a, const s3dx_rotary *rotary, int32_t in, int32_t out, hipStream_t stream) {
    if (a.n == 0) return;
    TurnTable t = {};
    if (rotary) {
        std::memcpy(t.turns, rotary->turns, sizeof t.turns);
        std::memcpy(t.axis, rotary->axis, sizeof t.axis);
    }
    const int64_t items = a.n * (a.part[0].heads + a.part[1].heads);
    pick_turn(in, out)<<<dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256), 0, stream>>>(a, t);
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
