// Attention over key blocks that a cheap score selects for each query: the
// 8-bit index of the blocks' mean keys, the selection, and the attention over
// the selected blocks or all of them (the transformer blocks of the SLat flow,
// slat_flow_graph.cpp:304-434, and the decoders' windows,
// gs_decoder_graph.cpp:93-121, which the reference runs as dense attention).
#include <cmath>

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

// The last sequence whose first unit is not behind `unit`, where sequence s
// begins at unit floor(starts[s] * mul / div) + s: every sequence has room for its
// last, partial unit, and the units rise with s, empty sequences or not.
__device__ __forceinline__ int64_t sequence_of_unit(const int32_t *starts, int64_t sequences, int64_t total,
                                                    int64_t mul, int64_t div, int64_t unit) {
    int64_t lo = 0, hi = sequences;  // begin(lo) <= unit < begin(hi)
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        const int64_t at = min(max(static_cast<int64_t>(starts[mid]), INT64_C(0)), total) * mul / div + mid;
        if (at <= unit) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The sequence that holds row `row`, or -1.
__device__ __forceinline__ int64_t sequence_of_row(const int32_t *starts, int64_t sequences, int64_t row) {
    int64_t lo = 0, hi = sequences;
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    return starts[lo] <= row && row < starts[lo + 1] ? lo : -1;
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
    int32_t kv_heads, d, block;
    int8_t *codes;
    float *scale;
};

// One wave per (index row, key head); lane l sums channels l and l + 64 in 64
// bits, so that the order of the rows does not show.
template <class T>
__global__ void __launch_bounds__(256) index_kernel(IndexArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (item >= a.rows * a.kv_heads) return;
    const int64_t row = item / a.kv_heads;
    const int head = static_cast<int>(item - row * a.kv_heads);
    const int64_t s = sequence_of_unit(a.k_starts, a.sequences, a.total_k, 1, a.block, row);
    const Span k = sequence_span(a.k_starts, s, a.total_k);
    const int64_t first = (row - (k.begin / a.block + s)) * a.block;
    const int count = static_cast<int>(min(static_cast<int64_t>(a.block), k.rows - first));
    if (first < 0 || count <= 0) return;
    const T *x = static_cast<const T *>(a.k) + (k.begin + first) * a.k_stride + static_cast<int64_t>(head) * a.d;
    double m[2] = {0.0, 0.0};
    for (int r = 0; r < count; ++r)
        for (int q = 0; q < 2; ++q)
            if (lane + 64 * q < a.d) m[q] += static_cast<double>(load_as_f32<T>(x + r * a.k_stride + lane + 64 * q));
    double most = 0.0;
    bool fine = true;
    for (int q = 0; q < 2; ++q) {
        m[q] /= count;
        fine = fine && fabs(m[q]) < __builtin_inf();
        most = fmax(most, fabs(m[q]));
    }
    for (int o = 1; o < 64; o <<= 1) most = fmax(most, __shfl_xor(most, o, 64));
    fine = __all(fine) && codes_fine(most);
    const int e = exponent_of(most);
    const double up = two_to(6 - e);
    int8_t *c = a.codes + (static_cast<int64_t>(head) * a.rows + row) * a.d;
    for (int q = 0; q < 2; ++q)
        if (lane + 64 * q < a.d) c[lane + 64 * q] = static_cast<int8_t>(fine ? code_of(m[q], up) : 0);
    if (lane == 0)
        a.scale[static_cast<int64_t>(head) * a.rows + row] = fine ? static_cast<float>(two_to(e - 6)) : 0.0f;
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
    int32_t kv_heads, group, d, block, top, most_blocks, flags;
};

// A float's order as an unsigned whole number (-0 does not occur: scores are
// whole numbers times powers of two).
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One wave per (query row, key head): scores into LDS, then `top` times the
// largest that is left.
template <class T>
__global__ void __launch_bounds__(64) select_kernel(SelectArgs a) {
    extern __shared__ uint32_t keys[];
    __shared__ int8_t qc[128];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x / a.kv_heads;
    const int head = static_cast<int>(blockIdx.x - row * a.kv_heads);
    const int64_t s = sequence_of_row(a.q_starts, a.sequences, row);
    if (s < 0) return;
    const Span qs = sequence_span(a.q_starts, s, a.total_q), ks = sequence_span(a.k_starts, s, a.total_k);
    int32_t *out = a.selected + (row * a.kv_heads + head) * a.top;
    const T *q = static_cast<const T *>(a.q) + row * a.q_stride + static_cast<int64_t>(head) * a.group * a.d;
    double m[2] = {0.0, 0.0}, most = 0.0;
    bool fine = true;
    for (int w = 0; w < 2; ++w) {
        if (lane + 64 * w < a.d)
            for (int g = 0; g < a.group; ++g)
                m[w] += static_cast<double>(load_as_f32<T>(q + static_cast<int64_t>(g) * a.d + lane + 64 * w));
        fine = fine && fabs(m[w]) < __builtin_inf();
        most = fmax(most, fabs(m[w]));
    }
    for (int o = 1; o < 64; o <<= 1) most = fmax(most, __shfl_xor(most, o, 64));
    fine = __all(fine) && codes_fine(most);
    const double up = two_to(6 - exponent_of(most));
    for (int w = 0; w < 2; ++w)
        if (lane + 64 * w < a.d) qc[lane + 64 * w] = static_cast<int8_t>(fine ? code_of(m[w], up) : 0);
    __syncthreads();
    const int32_t place = static_cast<int32_t>(row - qs.begin) + ks.rows - qs.rows;
    int32_t nb = min((ks.rows + a.block - 1) / a.block, a.most_blocks);
    if (a.flags & S3DX_BLOCK_CAUSAL) nb = place < 0 ? 0 : min(nb, place / a.block + 1);
    const int64_t base = static_cast<int64_t>(head) * a.rows + ks.begin / a.block + s;
    for (int b = lane; b < nb; b += 64) {
        const int8_t *c = a.codes + (base + b) * a.d;
        int dot = 0;
        for (int i = 0; i < a.d; ++i) dot += static_cast<int>(qc[i]) * static_cast<int>(c[i]);
        uint32_t key = order_key(static_cast<float>(dot) * a.scale[base + b]);
        if ((a.flags & S3DX_BLOCK_NEAR) && place >= 0 && b == place / a.block) key = 0xffffffffu;
        keys[b] = key;
    }
    // The wave's lanes read one another's keys only through shuffles; a chosen
    // block's key becomes 0, which no score has.
    const int take = min(nb, a.top);
    for (int t = 0; t < take; ++t) {
        uint32_t best = 0;
        int at = 0x7fffffff;
        for (int b = lane; b < nb; b += 64)
            if (keys[b] > best) {
                best = keys[b];
                at = b;
            }
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t k2 = __shfl_xor(best, o, 64);
            const int a2 = __shfl_xor(at, o, 64);
            if (k2 > best || (k2 == best && a2 < at)) {
                best = k2;
                at = a2;
            }
        }
        if ((at & 63) == lane) keys[at] = 0;
    }
    int done = 0;
    for (int b0 = 0; b0 < nb; b0 += 64) {
        const bool is = b0 + lane < nb && keys[b0 + lane] == 0;
        const uint64_t mask = __ballot(is);
        if (is) out[done + __popcll(mask & ((UINT64_C(1) << lane) - 1))] = b0 + lane;
        done += __popcll(mask);
    }
    for (int t = done + lane; t < a.top; t += 64) out[t] = -1;
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
    int32_t heads, group, kv_heads, d, block, top, flags;
    float scale;
};

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.44269504088896341f;

// One wave per (query row, head), key by key: scores with a key per lane, the
// running maximum and sum, values with a channel pair per lane.  Only keys that the
// row sees are multiplied.
template <class T>
__global__ void __launch_bounds__(64) attend_row_kernel(AttendArgs a) {
    __shared__ float qf[128];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x / a.heads;
    const int head = static_cast<int>(blockIdx.x - row * a.heads);
    const int64_t s = sequence_of_row(a.q_starts, a.sequences, row);
    if (s < 0) return;
    const Span qs = sequence_span(a.q_starts, s, a.total_q), ks = sequence_span(a.k_starts, s, a.total_k);
    const int kvh = head / a.group;
    const T *q = static_cast<const T *>(a.q) + row * a.q_stride + static_cast<int64_t>(head) * a.d;
    for (int c = lane; c < a.d; c += 64) qf[c] = load_as_f32<T>(q + c) * a.scale;
    __syncthreads();
    int32_t seen = ks.rows;
    if (a.flags & S3DX_BLOCK_CAUSAL)
        seen = max(0, min(seen, static_cast<int32_t>(row - qs.begin) + ks.rows - qs.rows + 1));
    const int32_t nb = (ks.rows + a.block - 1) / a.block;
    const int32_t *list = a.selected ? a.selected + (row * a.kv_heads + kvh) * a.top : nullptr;
    float m = -__builtin_inff(), l = 0.0f, o[2] = {0.0f, 0.0f};
    for (int t = 0; t < (list ? a.top : nb); ++t) {
        const int32_t b = list ? list[t] : t;
        if (b < 0 || b >= nb) continue;
        for (int k0 = b * a.block; k0 < min((b + 1) * a.block, seen); k0 += 64) {
            const int count = min(64, min((b + 1) * a.block, seen) - k0);
            const T *kr = static_cast<const T *>(a.k) + (ks.begin + k0) * a.k_stride + static_cast<int64_t>(kvh) * a.d;
            const T *vr = static_cast<const T *>(a.v) + (ks.begin + k0) * a.v_stride + static_cast<int64_t>(kvh) * a.d;
            float sc = -__builtin_inff();
            if (lane < count) {
                sc = 0.0f;
                for (int c = 0; c < a.d; ++c) sc += qf[c] * load_as_f32<T>(kr + lane * a.k_stride + c);
            }
            float mx = sc;
            for (int w = 1; w < 64; w <<= 1) mx = fmaxf(mx, __shfl_xor(mx, w, 64));
            const float mn = fmaxf(m, mx), base = mn == -__builtin_inff() ? 0.0f : mn;
            // the difference first: scores of the type's lowest value stay finite
            const float alpha = exp2f((m - base) * kLog2e), p = exp2f((sc - base) * kLog2e);
            l = l * alpha + (lane < count ? p : 0.0f);
            o[0] *= alpha;
            o[1] *= alpha;
            m = mn;
            for (int j = 0; j < count; ++j) {
                const float pj = __shfl(p, j, 64);
                for (int w = 0; w < 2; ++w)
                    if (lane + 64 * w < a.d) o[w] += pj * load_as_f32<T>(vr + j * a.v_stride + lane + 64 * w);
            }
        }
    }
    for (int w = 1; w < 64; w <<= 1) l += __shfl_xor(l, w, 64);
    // l == 0: nothing seen (a NaN is not 0 and stays)
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    T *y = static_cast<T *>(a.o) + row * a.o_stride + static_cast<int64_t>(head) * a.d;
    for (int w = 0; w < 2; ++w)
        if (lane + 64 * w < a.d) store_from_f32<T>(y + lane + 64 * w, l == 0.0f ? 0.0f : o[w] * r);
    if (a.lse && lane == 0) a.lse[row * a.heads + head] = l == 0.0f ? -__builtin_inff() : m + log2f(l) * kLn2;
}

// ---------------------------------------------------------------------------
// Argument checks
// ---------------------------------------------------------------------------
constexpr int64_t kMaxStride = INT64_C(1) << 22;
constexpr int32_t kMaxTop = 4096;
constexpr int64_t kMaxBlocks = 32768;

void check_total(int64_t total) {
    require(total >= 0 && total <= std::numeric_limits<int32_t>::max(), "a row count is out of range");
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
int64_t index_rows(int64_t total_k, int64_t sequences, int32_t block) { return total_k / block + sequences; }

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
                             kv_heads, head_dim, block, codes, scale};
        const int64_t items = a.rows * kv_heads;
        require(items <= (INT64_C(1) << 32), "too many blocks");
        (dtype == S3DX_BF16 ? index_kernel<uint16_t> : index_kernel<float>)<<<
            dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256), 0, as_stream(stream)>>>(a);
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
                        index_rows(total_k, sequences, block), kv_heads, heads / kv_heads, head_dim, block, top,
                        static_cast<int32_t>((std::min(max_k, total_k) + block - 1) / block), flags};
        require(total_q * kv_heads <= std::numeric_limits<int32_t>::max(), "total_q * kv_heads is out of range");
        const auto kernel = dtype == S3DX_BF16 ? select_kernel<uint16_t> : select_kernel<float>;
        const size_t lds = static_cast<size_t>(a.most_blocks) * 4;
        if (lds > 65536)
            hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                          hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)),
                      "hipFuncSetAttribute");
        kernel<<<dim3(static_cast<unsigned>(total_q * kv_heads)), dim3(64), lds, as_stream(stream)>>>(a);
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
        *bytes = 0;
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
        (void)workspace;
        (void)workspace_bytes;
        const AttendArgs a = {q, k, v, o, lse, q_starts, k_starts, selected, total_q, total_k, q_stride, k_stride,
                              v_stride, o_stride, sequences, heads, heads / kv_heads, kv_heads, head_dim, block, top,
                              flags, softmax_scale};
        require(total_q * heads <= std::numeric_limits<int32_t>::max(), "total_q * heads is out of range");
        (dtype == S3DX_BF16 ? attend_row_kernel<uint16_t> : attend_row_kernel<float>)<<<
            dim3(static_cast<unsigned>(total_q * heads)), dim3(64), 0, as_stream(stream)>>>(a);
        launch_check("block attention");
    });
}

}  // extern "C"
