// The step between two branches of a transformer block, in one pass: the
// branch's own norm, its gate and the sum with the stream, and the norm and
// modulation that the next branch begins with (slat_flow_graph.cpp:304-434 runs
// them one by one).
//
//   y = x + residual_scale gate . post(branch),   h = pre(y) . (1 + scale) + shift
//
// What bounds it: memory.  A row is held in registers between its parts, so that x and
// branch are read once and y and h written once: 42,000 rows of 768 channels, float32 and
// bfloat16, take 80 us, 4.8 TB/s of the 5.16 that a large copy reaches; 5,086 rows of 1,024 in bfloat16 11 us of 8,
// as a launch this short ends in one round of workgroups; a single row is the call.
#include "common.hpp"

namespace s3dx {
namespace {

struct NormArgs {
    const void *x, *branch;
    void *y, *h;  // h NULL: the sum alone
    const float *post_w, *post_b, *pre_w, *pre_b, *gate, *scale, *shift;
    const int32_t *sets;
    int64_t first, n, x_stride, branch_stride, y_stride, h_stride, mod_stride, set_stride;
    int32_t c, set_count, post, pre, x_bf, branch_bf, h_bf, lanes_log2;
    float eps, residual_scale;
};

// Rows whose sums pass 2^128 are summed again smaller.  They hold a channel, or a difference from the mean, of 2^57 at least (2^14 squares),
// beside which eps is nothing: 2^-23 then, up to 2^49, and the sums of squares stay from 2^-46 to 2^112.  (Where the difference was the mean's
// rounding alone, channels are 2^75 at least and differ, if they do, by 2^52: 2^-28 then.)
constexpr float kLess = 0x1p-80f;
// A mean is off by some 2^-24 of itself, which rows whose channels differ by less than this share of it take for a difference: of equal
// channels of 100.7 the norm came out as 0.015 and of 1e10 as 1, for 0.
constexpr float kAlike = 0x1p-12f;

// Sum over a row's threads: 2^lanes_log2 lanes of a wave, or all of a workgroup (`turn`: of sums so far, so that a place in
// LDS is written again only after a barrier behind its last reader).
template <bool WIDE>
__device__ __forceinline__ float row_sum(float v, int lanes_log2, float (*across)[16], int &turn) {
    for (int o = 1; o < (WIDE ? 64 : 1 << lanes_log2); o <<= 1) v += __shfl_xor(v, o, 64);
    if constexpr (WIDE) {
        float *mine = across[turn++ & 1];
        if ((threadIdx.x & 63) == 0) mine[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
        for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) v += mine[w];
    }
    return v;
}

// Four words side by side at any element's address.
struct __attribute__((packed, aligned(2))) Words {
    uint32_t w[4];
};
__device__ __forceinline__ void load8(const uint16_t *p, float (&v)[8]) {
    const Words t = *reinterpret_cast<const Words *>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(float, e & 1 ? t.w[e >> 1] & 0xffff0000u : t.w[e >> 1] << 16);
}
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const Words t = reinterpret_cast<const Words *>(p)[h];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * h + e] = __builtin_bit_cast(float, t.w[e]);
    }
}
__device__ __forceinline__ void store8(uint16_t *p, const float (&v)[8]) {
    Words t;
#pragma unroll
    for (int e = 0; e < 4; ++e) t.w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<Words *>(p) = t;
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        Words t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t.w[e] = __builtin_bit_cast(uint32_t, v[4 * h + e]);
        reinterpret_cast<Words *>(p)[h] = t;
    }
}

// A thread holds PPL pieces of 8 channels, `threads` pieces apart.  Rows need not begin at whole 16 bytes: memory takes
// 16-byte accesses at any element.  A last, shorter piece begins earlier instead, at the row's last 8 channels; it counts none
// of its neighbour's in sums, and both store the same (20,000 rows of 333 channels: 20 us, 31 element by element).  REST: rows that
// have one.  Rows of fewer than 8 channels go one by one.
// WIDE: a row for each workgroup, of as many waves as leave its threads one piece, two beyond 2,048 channels (20,000 rows of 2,048
// channels in bfloat16: 136 us in a wave, 86 with two pieces, 83 with one; of 2,600 121 with two, 136 with one).
template <int PPL, bool WIDE, bool REST>
__global__ void __launch_bounds__(WIDE ? 1024 : 256) gated_norm_kernel(NormArgs a) {
    __shared__ float across[2][16];
    const int threads = WIDE ? blockDim.x : 1 << a.lanes_log2;
    const int t = WIDE ? threadIdx.x : threadIdx.x & (threads - 1), rows = WIDE ? 1 : 256 / threads;
    const int64_t row = a.first + static_cast<int64_t>(blockIdx.x) * rows + (WIDE ? 0 : threadIdx.x >> a.lanes_log2);
    if (row >= a.n) return;  // WIDE: the whole workgroup
    const bool tiny = REST && a.c < 8;
    // a piece's first channel, and how many of them are another's (8: all, there is no such piece)
    const auto channel = [&](int p) {
        const int c = (p * threads + t) * 8;
        return REST && !tiny && c < a.c ? min(c, a.c - 8) : c;
    };
    const auto others = [&](int p) {
        const int c = (p * threads + t) * 8;
        return c >= a.c ? 8 : REST && !tiny ? c - min(c, a.c - 8) : 0;
    };
    const auto pieces = [&](auto &&whole, auto &&single) __attribute__((always_inline)) {
        if (tiny) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (t == 0 && e < a.c) single(0, e, e);
            return;
        }
#pragma unroll
        for (int p = 0; p < PPL; ++p)
            if ((p * threads + t) * 8 < a.c) whole(p, channel(p));
    };
    const auto load = [&](const void *base, int64_t at, bool bf, float (&v)[PPL][8]) __attribute__((always_inline)) {
        if (bf) {
            const uint16_t *x = static_cast<const uint16_t *>(base) + at;
            pieces([&](int p, int c) { load8(x + c, v[p]); }, [&](int p, int e, int c) { v[p][e] = bf16_to_f32(x[c]); });
        } else {
            const float *x = static_cast<const float *>(base) + at;
            pieces([&](int p, int c) { load8(x + c, v[p]); }, [&](int p, int e, int c) { v[p][e] = x[c]; });
        }
    };
    const auto store = [&](void *base, int64_t at, bool bf, const float (&v)[PPL][8]) __attribute__((always_inline)) {
        if (bf) {
            uint16_t *x = static_cast<uint16_t *>(base) + at;
            pieces([&](int p, int c) { store8(x + c, v[p]); }, [&](int p, int e, int c) { x[c] = f32_to_bf16(v[p][e]); });
        } else {
            float *x = static_cast<float *>(base) + at;
            pieces([&](int p, int c) { store8(x + c, v[p]); }, [&](int p, int e, int c) { x[c] = v[p][e]; });
        }
    };
    const auto each = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < PPL; ++p)
#pragma unroll
            for (int e = 0; e < 8; ++e) f(p, e);
    };
    // Sum of f over the row's channels, each once.
    int turn = 0;
    const auto sum = [&](auto &&f) __attribute__((always_inline)) {
        float all = 0.0f;
#pragma unroll
        for (int p = 0; p < PPL; ++p) {
            const int skip = others(p), end = tiny ? a.c : 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = f(p, e);
                all += (REST ? e >= skip && e < end : skip == 0) ? x : 0.0f;
            }
        }
        return row_sum<WIDE>(all, a.lanes_log2, across, turn);
    };
    const auto norm = [&](float (&v)[PPL][8], int kind, const float *w, const float *b) __attribute__((always_inline)) {
        if (kind == S3DX_NORM_NONE) return;
        const float count = static_cast<float>(a.c);
        const auto mean_of = [&](float times) { return kind == S3DX_NORM_LAYER ? sum([&](int p, int e) { return v[p][e] * times; }) / count : 0.0f; };
        float mean = mean_of(1.0f), eps = a.eps;
        const auto squares = [&] {
            return sum([&](int p, int e) {
                const float d = v[p][e] - mean;
                return d * d;
            });
        };
        float q = squares();
        // the same for the row's threads (a wave may hold several rows: those that are through wait)
        const bool over = !(q < __builtin_inff());
        const float beside = mean * kAlike;
        if (over || (kind == S3DX_NORM_LAYER && q / count <= beside * beside)) {
            // the mean in two parts, as the rounding of one may be all the difference that channels have
            const float less = over ? kLess : 1.0f, part = mean_of(less);
            each([&](int p, int e) { v[p][e] = v[p][e] * less - part; });
            mean = mean_of(1.0f);
            q = squares();
            if (over) eps = 0.0f;
        }
        const float var = q / count + eps, rstd = var == 0.0f ? 0.0f : rsqrtf(var);
        float g[PPL][8];
        each([&](int p, int e) { v[p][e] = (v[p][e] - mean) * rstd; });
        if (w) {
            load(w, 0, false, g);
            each([&](int p, int e) { v[p][e] *= g[p][e]; });
        }
        if (b) {
            load(b, 0, false, g);
            each([&](int p, int e) { v[p][e] += g[p][e]; });
        }
    };

    const int32_t set = a.sets ? a.sets[row * a.set_stride] : 0;
    const bool in = set >= 0 && set < a.set_count;  // rows of no set: gate, scale and shift 0
    const int64_t mods = in ? set * a.mod_stride : 0;
    float v[PPL][8], y[PPL][8], g[PPL][8];
    load(a.branch, row * a.branch_stride, a.branch_bf, v);
    load(a.x, row * a.x_stride, a.x_bf, y);
    if (WIDE && REST) __syncthreads();  // y or h may take the place of what a neighbour's shorter piece reads as well
    norm(v, a.post, a.post_w, a.post_b);
    if (a.gate) {
        if (in) load(a.gate, mods, false, g);  // (there may be no set at all)
        each([&](int p, int e) { v[p][e] *= in ? g[p][e] : 0.0f; });
    }
    each([&](int p, int e) { y[p][e] = fmaf(v[p][e], a.residual_scale, y[p][e]); });
    store(a.y, row * a.y_stride, a.x_bf, y);
    if (!a.h) return;
    norm(y, a.pre, a.pre_w, a.pre_b);
    if (in && a.scale) {
        load(a.scale, mods, false, g);
        each([&](int p, int e) { y[p][e] = fmaf(y[p][e], g[p][e], y[p][e]); });
    }
    if (in && a.shift) {
        load(a.shift, mods, false, g);
        each([&](int p, int e) { y[p][e] += g[p][e]; });
    }
    store(a.h, row * a.h_stride, a.h_bf, y);
}

constexpr int32_t kMostChannels = 16384;

using NormFn = void (*)(NormArgs);
template <bool WIDE, bool REST>
NormFn pick_pieces(int per) {
    return per <= 1 ? gated_norm_kernel<1, WIDE, REST> : gated_norm_kernel<2, WIDE, REST>;
}

void check_rows(const void *p, int64_t stride, int64_t n, int32_t c, int32_t dtype, const char *what) {
    const std::string name(what);
    require_dtype(dtype);
    require(stride >= c && stride <= (INT64_C(1) << 40), (name + ": the row stride is out of range (channels to 2^40)").c_str());
    require(n == 0 || (p && aligned(p, dtype_size(dtype))), (name + " is NULL or not aligned to its elements").c_str());
}

}  // namespace
}  // namespace s3dx

using namespace s3dx;

extern "C" {

S3DX_API s3dx_status s3dx_gated_norm_rows(const void *x, int32_t x_dtype, int64_t x_stride, const void *branch, int32_t branch_dtype,
                                          int64_t branch_stride, int64_t n, int32_t c, int32_t post, const float *post_w,
                                          const float *post_b, float residual_scale, const float *gate, int32_t pre,
                                          const float *pre_w, const float *pre_b, const float *mod_scale, const float *mod_shift,
                                          int64_t mod_stride, const int32_t *sets, int64_t set_stride, int32_t set_count, float eps,
                                          void *y, int64_t y_stride, void *h, int32_t h_dtype, int64_t h_stride, s3dx_stream stream,
                                          char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        require(n >= 0 && n <= std::numeric_limits<int32_t>::max(), "n is out of range");
        require(c >= 1 && c <= kMostChannels, "c must be 1 to 16384");
        for (int32_t kind : {post, pre})
            require(kind == S3DX_NORM_NONE || kind == S3DX_NORM_LAYER || kind == S3DX_NORM_RMS, "unknown norm");
        require(post != S3DX_NORM_NONE || (!post_w && !post_b), "post_w or post_b without a norm");
        require(pre != S3DX_NORM_NONE || (!pre_w && !pre_b), "pre_w or pre_b without a norm");
        require(h || (pre == S3DX_NORM_NONE && !mod_scale && !mod_shift), "h is NULL beside a norm or modulation of it");
        require(eps > 0.0f && eps <= 1.0f, "eps must be above 0 and at most 1");
        require(std::abs(residual_scale) < std::numeric_limits<float>::infinity(), "residual_scale is not finite");
        check_rows(x, x_stride, n, c, x_dtype, "x");
        check_rows(branch, branch_stride, n, c, branch_dtype, "branch");
        check_rows(y, y_stride, n, c, x_dtype, "y");
        if (h) check_rows(h, h_stride, n, c, h_dtype, "h");
        const bool mods = gate || mod_scale || mod_shift;
        if (sets) {
            require(aligned(sets, 4) && set_stride >= 1 && set_stride <= (INT64_C(1) << 31), "sets is not aligned, or set_stride out of range");
            require(set_count >= 0, "set_count is out of range");
        }
        require(!mods || !sets || set_count == 0 || (mod_stride >= c && mod_stride <= (INT64_C(1) << 40)), "mod_stride is shorter than c, or above 2^40");
        for (const float *p : {post_w, post_b, pre_w, pre_b, gate, mod_scale, mod_shift}) require(aligned(p, 4), "a vector is not aligned");
        if (n == 0) return;
        // y and h may lie where x or branch does, row by row
        const auto beside = [&](const void *out, int64_t out_stride, int32_t out_dtype, const void *in, int64_t in_stride, int32_t in_dtype) {
            require(out != in || (out_dtype == in_dtype && (n == 1 || out_stride == in_stride)), "in place needs the same dtype and stride");
        };
        beside(y, y_stride, x_dtype, x, x_stride, x_dtype);
        beside(y, y_stride, x_dtype, branch, branch_stride, branch_dtype);
        if (h) {
            beside(h, h_stride, h_dtype, x, x_stride, x_dtype);
            beside(h, h_stride, h_dtype, branch, branch_stride, branch_dtype);
            require(h != y, "h and y are the same");
        }
        NormArgs a = {x, branch, y, h, post_w, post_b, pre_w, pre_b, gate, mod_scale, mod_shift, sets, 0, n, x_stride, branch_stride,
                      y_stride, h_stride, sets ? mod_stride : 0, set_stride, c, sets ? set_count : 1, post, pre, x_dtype == S3DX_BF16,
                      branch_dtype == S3DX_BF16, h_dtype == S3DX_BF16, 0, eps, residual_scale};
        const bool wide = c > 64 * 8 * 2, rest = c % 8 != 0;
        while (!wide && a.lanes_log2 < 6 && (8 << a.lanes_log2) < c) ++a.lanes_log2;
        const int threads = !wide ? 1 << a.lanes_log2 : c <= 2048 ? (c + 511) / 512 * 64 : (c + 1023) / 1024 * 64;
        const int per = (c + 8 * threads - 1) / (8 * threads), rows = wide ? 1 : 256 / threads, group = wide ? threads : 256;
        const NormFn fn = wide ? (rest ? pick_pieces<true, true>(per) : pick_pieces<true, false>(per))
                               : (rest ? pick_pieces<false, true>(per) : pick_pieces<false, false>(per));
        // a launch's threads stay below 2^32
        const int64_t most = rows * (INT64_C(1) << 21);
        for (; a.first < n; a.first += most) {
            a.n = std::min(n, a.first + most);
            fn<<<dim3(static_cast<unsigned>((a.n - a.first + rows - 1) / rows)), dim3(group), 0, as_stream(stream)>>>(a);
        }
        launch_check("gated norm");
    });
}

}  // extern "C"
