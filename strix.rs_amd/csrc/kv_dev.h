// The paged 8-bit key/value cache as the kernels see it (layout: smx_kv_cache in strix_mi355.h).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "smx_internal.h"

namespace smx {

// Cache and batch of a launch, by value.
struct KvArgs {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    const int32_t* len;
    const int32_t* row0;   // null: one row for each sequence
    const int32_t* table;
    int table_ld, pages, page_blocks, kv_heads, dim, dim64;
    int nseq, rows, max_rows, max_len;
};

// One sequence of the batch as far as it is within the call's sizes: its rows [row, row + n) and the tokens [0, len) it holds; row j is the
// token len - n + j.  What is beyond rows, max_rows or max_len are a sequence's last rows, and go with their tokens: the others keep
// their positions.
struct KvSeq {
    int row, n, len;
};
// Rows of a sequence from its first one on, without a look at its tokens: within rows and max_rows, and all of them.
struct KvRows {
    int row, n, all;
};
__device__ __forceinline__ KvRows kv_rows(const KvArgs& a, int s) {
    int r0 = s, r1 = s + 1;   // (without row0 rows is nseq and max_rows 1)
    if (a.row0) { r0 = a.row0[s]; r1 = a.row0[s + 1]; }
    const int row = min(max(r0, 0), a.rows), all = max(r1, row) - row;
    return {row, min(all, min(a.rows - row, a.max_rows)), all};
}
__device__ __forceinline__ KvSeq kv_seq(const KvArgs& a, int s) {
    const int len = a.len[s];
    const KvRows r = kv_rows(a, s);
    const int held = max(max(len, 0) - (r.all - r.n), 0), over = max(held - a.max_len, 0);
    return {r.row, max(r.n - over, 0), held - over};
}
// Where a head's block `blk` (of SMX_KV_BLOCK tokens) of sequence s is: the page that the table names for it (any number at all), and its index
// among all blocks of the cache, with page numbers outside the cache clamped into it.
struct KvPlace {
    int page;
    int64_t block;
};
__device__ __forceinline__ KvPlace kv_place(const KvArgs& a, int s, int head, int blk) {
    const int p = blk / a.page_blocks, page = a.table[(int64_t)s * a.table_ld + min(p, a.table_ld - 1)];
    return {page, ((int64_t)min(max(page, 0), a.pages - 1) * a.kv_heads + head) * a.page_blocks + (blk - p * a.page_blocks)};
}
__device__ __forceinline__ int64_t kv_block(const KvArgs& a, int s, int head, int blk) { return kv_place(a, s, head, blk).block; }
// Byte of (token, channel) inside a block's keys / values.
__device__ __forceinline__ int kv_k_byte(int dim64, int t, int d) {
    return ((t >> 4) * (dim64 >> 6) + (d >> 6)) * 1024 + ((d >> 4) & 3) * 256 + (t & 15) * 16 + (d & 15);
}
__device__ __forceinline__ int kv_v_byte(int t, int d) {
    return (d >> 5) * 1024 + ((t >> 2) & 3) * 256 + (d & 15) * 16 + ((d >> 4) & 1) * 8 + (t >> 4) * 4 + (t & 3);
}

__device__ __forceinline__ float bf16_to_f32(uint16_t h) { return __uint_as_float((unsigned)h << 16); }
// round to nearest, ties to even; NaN stays NaN
__device__ __forceinline__ uint16_t f32_to_bf16(float f) {
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
template <bool BF16>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
    return BF16 ? bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}
template <bool BF16>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float v) {
    if (BF16) ((uint16_t*)p)[i] = f32_to_bf16(v);
    else ((float*)p)[i] = v;
}

// Host side: the checks that every call over a cache makes, and the launch form of its arguments.
int kv_args(smx_ctx* c, const char* who, const smx_kv_cache* cache, const smx_kv_batch* batch, KvArgs* out);

}  // namespace smx
