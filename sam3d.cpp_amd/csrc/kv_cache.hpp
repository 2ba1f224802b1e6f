// The layout of a cache of keys and values in 8 bits, shared by the kernels
// that write and read it and the attention over it.
//
// A page holds `block` rows of every key head.  Of each head first the keys'
// codes, a row after the other ([block][d]), then the values', a channel after
// the other ([d][block]): the order in which the attention's products take them, so
// that a wave reads whole 16-byte pieces of both and turns neither.  A code is
// 128 + c for c from -127 to 127: biased codes become half-precision numbers by one
// byte permute and one addition.  Behind the codes of all pages stand the steps that codes
// count in, float32 (keys', values') of each page and head.
#pragma once

#include "packed_rows.hpp"

struct s3dx_cache {
    void *buffer;
    int32_t pages, kv_heads, head_dim, block;
};

namespace s3dx {

constexpr int64_t kMaxPlaces = INT64_C(1) << 29;  // of a sequence: places and steps stay below 2^31

inline uint64_t cache_code_bytes(int32_t pages, int32_t kv_heads, int32_t head_dim, int32_t block) {
    return static_cast<uint64_t>(pages) * kv_heads * 2 * block * head_dim;
}

// What a kernel needs of a cache and its table.
struct CacheView {
    uint8_t *codes;
    float2 *steps;  // [pages][kv_heads]
    const int32_t *table, *lengths;
    int32_t pages, kv_heads, block_log2, table_stride;
};

inline int32_t block_log2_of(int32_t block) { return block == 64 ? 6 : 7; }

inline CacheView view_of(const s3dx_cache *c, const int32_t *table, int32_t table_stride, const int32_t *lengths) {
    uint8_t *codes = static_cast<uint8_t *>(c->buffer);
    return {codes, reinterpret_cast<float2 *>(codes + cache_code_bytes(c->pages, c->kv_heads, c->head_dim, c->block)),
            table, lengths, c->pages, c->kv_heads, block_log2_of(c->block), table_stride};
}

inline void check_table(const s3dx_cache *c, const int32_t *table, int32_t table_stride, const int32_t *lengths,
                        int64_t sequences) {
    require(c, "cache is NULL");
    require(sequences >= 0 && sequences <= (INT64_C(1) << 24), "sequences is out of range");
    require(table_stride >= 0 && static_cast<int64_t>(table_stride) * c->block <= kMaxPlaces,
            "table_stride is out of range (0 to 2^29 places of a sequence)");
    if (sequences == 0) return;
    require(table_stride == 0 || (table && aligned(table, 4)), "table is NULL or not aligned");
    require(lengths && aligned(lengths, 4), "lengths is NULL or not aligned");
}

// Rows that a sequence of length `length` keeps: cut to what its table has room for.
__device__ __forceinline__ int32_t cached_rows(const CacheView &a, int32_t length) {
    return min(max(length, 0), a.table_stride << a.block_log2);
}
// The page of block j of sequence s, or -1.
__device__ __forceinline__ int32_t page_of(const CacheView &a, int64_t s, int32_t j) {
    if (j < 0 || j >= a.table_stride) return -1;
    const int32_t p = a.table[s * a.table_stride + j];
    return p >= 0 && p < a.pages ? p : -1;
}

}  // namespace s3dx
