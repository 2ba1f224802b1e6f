// A cache of keys and values in 8 bits, in pages: rows quantised as they are
// written, and read back.  It stands beside the attention over packed rows (the SLat
// flow's transformer blocks, slat_flow_graph.cpp:304-434) for models that keep
// what earlier rows left; the reference keeps none.
//
// Step and codes of a block of rows and a head: with 2^e <= most < 2^(e+1), most the
// largest finite magnitude of its rows, step 2^(e-6) and c = round(x / step), halves
// to even, cut to +-127.  Steps are powers of two, so that x / step is exact and
// the rounding to a whole number the only one.
//
// Both ways memory bounds: a value is read once and written once (3 bytes in
// bfloat16, 5 in float32).  28,265 rows of 16 heads x 64 in bfloat16 take 38 us to
// write and 38 to read, 4.55 TB/s of the 5.16 that a large copy reaches; 60,000 rows of 8 x 128 77 us each
// way, 4.8 TB/s; a few rows what a launch takes.
// A workgroup takes a block of one head, blocks of neighbouring heads to one XCD, as
// their rows share lines of memory (dealt out in turn the same rows took 42 us to read).
#include "kv_cache.hpp"

namespace s3dx {
namespace {

struct RowArgs {
    CacheView cache;
    const void *k, *v;   // rows written
    void *k_out, *v_out; // rows read
    int64_t k_stride, v_stride, total, sequences;
    const int32_t *starts;
};

// The part of a sequence's rows that lies in one block: rows [row, row + count) of the packed
// ones, at the block's places [slot, slot + count).
struct Part {
    int64_t s, row;
    int32_t j, slot, count;
};
// Blocks are dealt out by unit.  (Beyond 64 sequences: s begins at unit starts[s] / block + 2 s, which leaves
// room for the blocks that its rows can lie in, wherever they begin.)
__device__ __forceinline__ Part part_of(const RowArgs &a, int64_t unit) {
    const int log2 = a.cache.block_log2, block = 1 << log2;
    const Sequence q = sequence_at(a.starts, a.cache.lengths, a.sequences, a.total, 1, log2, 2, 0, [&](int32_t n, int32_t entry) {
        const int32_t end = cached_rows(a.cache, entry);
        return n == 0 ? 0 : ((end - 1) >> log2) - ((end - n) >> log2) + 1;
    }, [&](int64_t) { return unit; });
    const int32_t first = cached_rows(a.cache, q.entry) - q.rows.rows;  // the first row's place, below 0 where there is no room for it
    const int64_t j = (first >> log2) + unit - q.first;
    const int64_t lo = max(static_cast<int64_t>(first), j << log2), hi = min(static_cast<int64_t>(first) + q.rows.rows, (j + 1) << log2);
    if (unit < q.first || hi <= lo) return {q.s, 0, 0, 0, 0};
    return {q.s, q.rows.begin + (lo - first), static_cast<int32_t>(j), static_cast<int32_t>(lo & (block - 1)), static_cast<int32_t>(hi - lo)};
}

// Eight channels as they lie in memory, and one of them as 32 bits.
template <class T>
struct Piece {
    static constexpr int N = 8 * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[N];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 t = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
        }
    }
    __device__ __forceinline__ uint32_t at(int e) const { return sizeof(T) == 4 ? w[e % N] : e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16; }
    __device__ __forceinline__ void clear(int e) {
        if constexpr (sizeof(T) == 4) w[e] = 0;
        else w[e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
    }
};

constexpr uint32_t kInfBits = 0x7f800000u, kLeastBits = (127u - 100u) << 23;
// A step from the largest finite magnitude's bits: 0 below 2^-100.
__device__ __forceinline__ float step_of(uint32_t most) {
    return most < kLeastBits ? 0.0f : __builtin_bit_cast(float, (most & kInfBits) - (6u << 23));
}
// 1 / step, exactly (steps are 0 or 2^-106 to 2^121).
__device__ __forceinline__ float per_step(float step) {
    return step == 0.0f ? 0.0f : __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, step));
}
// Four biased codes, of x cut to 127 steps.  x / step added to 1.5 * 2^23 is rounded to a whole number, halves to even, in the sum's
// low bits, 128 more to the biased code.
template <class T>
__device__ __forceinline__ uint32_t codes_of(const Piece<T> &x, int from, float step, float per) {
    constexpr float kWhole = 12582912.0f + 128.0f;
    const float most = 127.0f * step;
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        u[i] = __builtin_bit_cast(uint32_t, fmaf(__builtin_amdgcn_fmed3f(__builtin_bit_cast(float, x.at(from + i)), -most, most), per, kWhole));
    const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
// The four bytes of w counted in steps 1/ratio times as large.
__device__ __forceinline__ uint32_t counted_again(uint32_t w, float ratio) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        out |= (static_cast<uint32_t>(static_cast<int>(rintf((static_cast<float>((w >> (8 * i)) & 0xffu) - 128.0f) * ratio))) + 128u) << (8 * i);
    return out;
}
// Four rows of four bytes as four columns.
__device__ __forceinline__ void turn4(uint32_t (&w)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// A workgroup writes a block's rows of one head: fetched once, held in registers as they lay in memory (as 32
// bits each they leave room for half the waves: 60,000 rows of 8 x 128 took 95 us) while their
// largest magnitude is found, then coded.  Keys' codes go out a row's 8 channels at a time.  Values' are
// turned: in a block that begins with these rows through LDS, 16 rows of a channel at a time; in one that held
// rows before byte by byte, as their neighbours have to stay (a single new row: D bytes).
// A block whose step grows has what it held counted again first.
template <class T, int D, int BLOCK>
__global__ void __launch_bounds__(256) write_kernel(RowArgs a) {
    constexpr int PER = D / 8;                   // pieces of 8 channels of a row
    constexpr int NP = BLOCK * PER / 256;        // ... of a thread
    constexpr int LROW = D + 4;                  // bytes of a row in LDS
    static_assert(BLOCK * PER % 256 == 0);
    __shared__ uint32_t most[2];
    __shared__ alignas(16) uint8_t turned[BLOCK * LROW];
    const int tid = threadIdx.x;
    const int64_t id = xcd_tile(blockIdx.x, gridDim.x), unit = id / a.cache.kv_heads;
    const int head = static_cast<int>(id - unit * a.cache.kv_heads);
    const Part p = part_of(a, unit);
    if (p.count == 0) return;
    const int32_t page = page_of(a.cache, p.s, p.j);
    if (page < 0) return;
    const int64_t cell = static_cast<int64_t>(page) * a.cache.kv_heads + head;
    uint8_t *kc = a.cache.codes + cell * (2 * BLOCK * D), *vc = kc + BLOCK * D;
    const float2 was = p.slot > 0 ? a.cache.steps[cell] : make_float2(0.0f, 0.0f);  // read before anyone writes it (barriers below)
    if (tid < 2) most[tid] = 0;
    __syncthreads();
    Piece<T> x[2][NP] = {};
    uint32_t big[2] = {0, 0};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const T *from = static_cast<const T *>(w ? a.v : a.k) + head * D;
        const int64_t stride = w ? a.v_stride : a.k_stride;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int e = tid + 256 * i, r = e / PER, c = (e - r * PER) * 8;
            if (r < p.count) x[w][i].load(from + (p.row + r) * stride + c);
        }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int t = 0; t < 8; ++t) big[w] = max(big[w], x[w][i].at(t) & 0x7fffffffu);
        // magnitudes' bits rise with them, infinities and NaN above all: a thread that has one looks at the finite values alone, and
        // takes a NaN as 0 (its infinities are cut as large values are)
        if (big[w] >= kInfBits) {
            big[w] = 0;
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    const uint32_t m = x[w][i].at(t) & 0x7fffffffu;
                    if (m > kInfBits) x[w][i].clear(t);
                    if (m < kInfBits) big[w] = max(big[w], m);
                }
        }
        for (int o = 1; o < 64; o <<= 1) big[w] = max(big[w], static_cast<uint32_t>(__shfl_xor(static_cast<int>(big[w]), o, 64)));
        if ((tid & 63) == 0) atomicMax(&most[w], big[w]);
    }
    __syncthreads();
    float step[2] = {step_of(most[0]), step_of(most[1])};
    if (p.slot > 0) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const float old = w ? was.y : was.x;
            if (step[w] > old) {
                uint32_t *codes = reinterpret_cast<uint32_t *>(w ? vc : kc);
                const float ratio = old > 0.0f ? old * per_step(step[w]) : 0.0f;
                for (int e = tid; e < BLOCK * D / 4; e += 256) codes[e] = counted_again(codes[e], ratio);
            } else {
                step[w] = old;
            }
        }
        __syncthreads();  // in place before the new rows' bytes
    }
    if (tid == 0) a.cache.steps[cell] = make_float2(step[0], step[1]);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const float per = per_step(step[w]);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int e = tid + 256 * i, r = e / PER, c = (e - r * PER) * 8;
            const uint32_t lo = codes_of(x[w][i], 0, step[w], per), hi = codes_of(x[w][i], 4, step[w], per);
            if (w == 0) {
                if (r < p.count) *reinterpret_cast<uint2 *>(kc + (p.slot + r) * D + c) = make_uint2(lo, hi);
            } else if (p.slot == 0) {
                *reinterpret_cast<uint32_t *>(turned + r * LROW + c) = lo;
                *reinterpret_cast<uint32_t *>(turned + r * LROW + c + 4) = hi;
            } else if (r < p.count) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    vc[(c + t) * BLOCK + p.slot + r] = static_cast<uint8_t>(lo >> (8 * t));
                    vc[(c + 4 + t) * BLOCK + p.slot + r] = static_cast<uint8_t>(hi >> (8 * t));
                }
            }
        }
    }
    if (p.slot > 0) return;
    __syncthreads();
    // 16 rows of 4 channels a thread; rows behind the last one hold zeros
    for (int e = tid; e < BLOCK / 16 * (D / 4); e += 256) {
        const int c = e % (D / 4) * 4, r = e / (D / 4) * 16;
        if (r >= p.count) continue;
        uint32_t out[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t w[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) w[t] = *reinterpret_cast<const uint32_t *>(turned + (r + 4 * q + t) * LROW + c);
            turn4(w);
#pragma unroll
            for (int t = 0; t < 4; ++t) out[t][q] = w[t];
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
            *reinterpret_cast<uint4 *>(vc + (c + t) * BLOCK + r) = make_uint4(out[t][0], out[t][1], out[t][2], out[t][3]);
    }
}

template <class T>
__device__ __forceinline__ void store8(T *p, uint32_t lo, uint32_t hi, float step) {
    float v[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = (static_cast<float>(((t < 4 ? lo : hi) >> (8 * (t & 3))) & 0xffu) - 128.0f) * step;
    if constexpr (sizeof(T) == 2) {
        // seven bits of a code and a power of two: exact in bfloat16
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
}

// The way back: a workgroup gives a block's rows of one head, the values' codes turned through LDS.
// Rows that the cache does not hold are zeros.
template <class T, int D, int BLOCK>
__global__ void __launch_bounds__(256) read_kernel(RowArgs a) {
    constexpr int PER = D / 8, NP = BLOCK * PER / 256, LROW = D + 4;
    __shared__ alignas(16) uint8_t turned[BLOCK * LROW];
    const int tid = threadIdx.x;
    const int64_t id = xcd_tile(blockIdx.x, gridDim.x), unit = id / a.cache.kv_heads;
    const int head = static_cast<int>(id - unit * a.cache.kv_heads);
    const Part p = part_of(a, unit);
    if (p.count == 0) return;
    const int32_t page = page_of(a.cache, p.s, p.j);
    const int64_t cell = static_cast<int64_t>(max(page, 0)) * a.cache.kv_heads + head;
    const uint8_t *kc = a.cache.codes + cell * (2 * BLOCK * D), *vc = kc + BLOCK * D;
    const float2 step = page >= 0 ? a.cache.steps[cell] : make_float2(0.0f, 0.0f);
    uint2 k[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int e = tid + 256 * i, r = e / PER, c = (e - r * PER) * 8;
        k[i] = make_uint2(0x80808080u, 0x80808080u);
        if (page >= 0 && r < p.count) k[i] = *reinterpret_cast<const uint2 *>(kc + (p.slot + r) * D + c);
    }
    for (int e = tid; e < BLOCK / 16 * (D / 4); e += 256) {
        const int c = e / (BLOCK / 16) * 4, r = e % (BLOCK / 16) * 16;
        uint4 from[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
            from[t] = page >= 0 ? *reinterpret_cast<const uint4 *>(vc + (c + t) * BLOCK + r) : make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t w[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) w[t] = q == 0 ? from[t].x : q == 1 ? from[t].y : q == 2 ? from[t].z : from[t].w;
            turn4(w);
#pragma unroll
            for (int t = 0; t < 4; ++t) *reinterpret_cast<uint32_t *>(turned + (r + 4 * q + t) * LROW + c) = w[t];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int e = tid + 256 * i, r = e / PER, c = (e - r * PER) * 8;
        if (r >= p.count) continue;
        store8(static_cast<T *>(a.k_out) + (p.row + r) * a.k_stride + head * D + c, k[i].x, k[i].y, step.x);
        const uint8_t *v = turned + (p.slot + r) * LROW + c;
        store8(static_cast<T *>(a.v_out) + (p.row + r) * a.v_stride + head * D + c, *reinterpret_cast<const uint32_t *>(v),
               *reinterpret_cast<const uint32_t *>(v + 4), step.y);
    }
}

using RowFn = void (*)(RowArgs);
template <class T, int BLOCK>
RowFn pick_write(int32_t d) {
    return d == 32 ? write_kernel<T, 32, BLOCK> : d == 64 ? write_kernel<T, 64, BLOCK> : d == 96 ? write_kernel<T, 96, BLOCK> : write_kernel<T, 128, BLOCK>;
}
template <class T, int BLOCK>
RowFn pick_read(int32_t d) {
    return d == 32 ? read_kernel<T, 32, BLOCK> : d == 64 ? read_kernel<T, 64, BLOCK> : d == 96 ? read_kernel<T, 96, BLOCK> : read_kernel<T, 128, BLOCK>;
}

void check_shape(int32_t pages, int32_t kv_heads, int32_t head_dim, int32_t block) {
    require(pages >= 0, "pages is out of range");
    require(kv_heads >= 1 && kv_heads <= 65536, "kv_heads must be 1 to 65536");
    require(head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128, "head_dim must be 32, 64, 96 or 128");
    require(block == 64 || block == 128, "block must be 64 or 128");
}

// Checks and launches either way.
void launch_rows(const s3dx_cache *c, RowArgs a, const void *k, const void *v, int32_t dtype, const int32_t *table,
                 int32_t table_stride, const int32_t *lengths, bool write, hipStream_t stream) {
    check_table(c, table, table_stride, lengths, a.sequences);
    require_dtype(dtype);
    require(a.total >= 0 && a.total <= kMaxPlaces, "a row count is out of range (0 to 2^29)");
    if (a.total == 0 || a.sequences == 0) return;
    require(a.starts && aligned(a.starts, 4), "starts is NULL or not aligned");
    for (const auto &[p, stride] : {std::pair(k, a.k_stride), std::pair(v, a.v_stride)}) {
        require(p && aligned(p, 16), "a row pointer is NULL or not 16-byte aligned");
        require(stride >= static_cast<int64_t>(c->kv_heads) * c->head_dim, "a row stride is shorter than its heads");
        require(stride <= (INT64_C(1) << 40) && stride * dtype_size(dtype) % 16 == 0,
                "a row stride must be whole 16-byte pieces, at most 2^40 elements");
    }
    a.cache = view_of(c, table, table_stride, lengths);
    const int64_t grid = ((a.total >> a.cache.block_log2) + 2 * a.sequences) * c->kv_heads;
    require(grid <= 0xffffffffll / 256, "too many rows and sequences");
    const bool bf = dtype == S3DX_BF16, small = c->block == 64;
    const int32_t d = c->head_dim;
    const RowFn fn = write ? (bf ? (small ? pick_write<uint16_t, 64>(d) : pick_write<uint16_t, 128>(d))
                                 : (small ? pick_write<float, 64>(d) : pick_write<float, 128>(d)))
                           : (bf ? (small ? pick_read<uint16_t, 64>(d) : pick_read<uint16_t, 128>(d))
                                 : (small ? pick_read<float, 64>(d) : pick_read<float, 128>(d)));
    fn<<<dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream>>>(a);
    launch_check(write ? "cache write" : "cache read");
}

}  // namespace
}  // namespace s3dx

using namespace s3dx;

extern "C" {

S3DX_API s3dx_status s3dx_cache_size(int32_t pages, int32_t kv_heads, int32_t head_dim, int32_t block, uint64_t *bytes,
                                     char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        require(bytes, "bytes is NULL");
        check_shape(pages, kv_heads, head_dim, block);
        *bytes = cache_code_bytes(pages, kv_heads, head_dim, block) + static_cast<uint64_t>(pages) * kv_heads * sizeof(float2);
    });
}

S3DX_API s3dx_status s3dx_cache_create(void *buffer, int32_t pages, int32_t kv_heads, int32_t head_dim, int32_t block,
                                       s3dx_cache **out, char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        require(out, "out is NULL");
        *out = nullptr;
        check_shape(pages, kv_heads, head_dim, block);
        require(pages == 0 || (buffer && aligned(buffer, 16)), "buffer is NULL or not 16-byte aligned");
        *out = new s3dx_cache{buffer, pages, kv_heads, head_dim, block};
    });
}

S3DX_API void s3dx_cache_free(s3dx_cache *cache) { delete cache; }

S3DX_API s3dx_status s3dx_cache_write(const s3dx_cache *cache, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                                      int32_t dtype, int64_t total, const int32_t *starts, const int32_t *table,
                                      int32_t table_stride, const int32_t *lengths, int64_t sequences, s3dx_stream stream,
                                      char *error, uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        const RowArgs a = {{}, k, v, nullptr, nullptr, k_stride, v_stride, total, sequences, starts};
        launch_rows(cache, a, k, v, dtype, table, table_stride, lengths, true, as_stream(stream));
    });
}

S3DX_API s3dx_status s3dx_cache_read(const s3dx_cache *cache, void *k, int64_t k_stride, void *v, int64_t v_stride, int32_t dtype,
                                     int64_t total, const int32_t *starts, const int32_t *table, int32_t table_stride,
                                     const int32_t *lengths, int64_t sequences, s3dx_stream stream, char *error,
                                     uint64_t error_capacity) {
    return boundary(error, error_capacity, [&] {
        const RowArgs a = {{}, nullptr, nullptr, k, v, k_stride, v_stride, total, sequences, starts};
        launch_rows(cache, a, k, v, dtype, table, table_stride, lengths, false, as_stream(stream));
    });
}

}  // extern "C"
