// paged.cuh -- device view and host checks of a paged KV cache (rkv_paged_cache).
#pragma once

#include "rkv_common.cuh"

namespace rkv {

constexpr int kMaxLen = 1 << 30;  // tokens per sequence: token counters may step past the end by a tile

struct PagedView {
    uint8_t* K;
    uint8_t* V;
    const int* table;  // [batch][table_stride]
    const int* lens;   // [batch]
    long long page_stride, head_stride, token_stride;  // bytes
    int table_stride, num_pages, page_size;
};

inline PagedView paged_view(const rkv_paged_cache& c) {
    PagedView v{};
    v.K = static_cast<uint8_t*>(c.K);
    v.V = static_cast<uint8_t*>(c.V);
    v.table = c.block_table;
    v.lens = c.lens;
    v.page_stride = c.page_stride;
    v.head_stride = c.head_stride;
    v.token_stride = c.token_stride;
    v.table_stride = c.table_stride;
    v.num_pages = c.num_pages;
    v.page_size = c.page_size;
    return v;
}

// Tokens of sequence b, clamped to what the table and the caller's bound cover.
__device__ __forceinline__ int paged_len(const PagedView& c, int b, int max_len) {
    const long long cap = (long long)c.table_stride * c.page_size;
    const int n = min(c.lens[b], max_len);
    return max(0, cap < n ? (int)cap : n);
}

// Byte offset of token t of (sequence b, head h) in K and V, or -1 where its
// page index lies outside the pool.  t / page_size < table_stride.
__device__ __forceinline__ long long paged_offset(const PagedView& c, int b, int h, int t) {
    const unsigned pg = (unsigned)t / (unsigned)c.page_size;
    const int p = c.table[(size_t)b * c.table_stride + pg];
    if ((unsigned)p >= (unsigned)c.num_pages) return -1;
    return p * c.page_stride + h * c.head_stride + (long long)((unsigned)t - pg * c.page_size) * c.token_stride;
}

inline bool paged_dtype(int dt) { return dt == RKV_F32 || dt == RKV_BF16 || dt == RKV_F16; }
inline int elem_size(int dt) { return dt == RKV_F32 ? 4 : 2; }

// Sizes, alignment and strides of a cache; lens_too: whether lens is read.  A batch without a sequence reads
// neither lens nor the table.
inline int paged_check(const rkv_paged_cache* c, bool lens_too, int batch) {
    if (!c || !paged_dtype(c->dtype)) return RKV_ERR_INVALID_ARG;
    if (c->num_heads_kv <= 0 || c->dim_head <= 0 || c->page_size <= 0 || c->num_pages < 0 || c->table_stride < 0)
        return RKV_ERR_INVALID_ARG;
    if (c->dim_head % 8 != 0 || c->dim_head > 256) return RKV_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(c->K) | reinterpret_cast<uintptr_t>(c->V)) & 15) return RKV_ERR_INVALID_ARG;
    if ((c->page_stride | c->head_stride | c->token_stride) & 15) return RKV_ERR_INVALID_ARG;
    const long long rowb = (long long)c->dim_head * elem_size(c->dtype);
    if ((c->page_size > 1 && c->token_stride < rowb) || (c->num_heads_kv > 1 && c->head_stride < rowb) ||
        (c->num_pages > 1 && c->page_stride < rowb))
        return RKV_ERR_INVALID_ARG;
    if (c->num_pages > 0 && (!c->K || !c->V)) return RKV_ERR_INVALID_ARG;
    if (batch == 0) return RKV_OK;
    if (c->table_stride > 0 && !c->block_table) return RKV_ERR_INVALID_ARG;
    if (lens_too && !c->lens) return RKV_ERR_INVALID_ARG;
    return RKV_OK;
}

inline int launched() {
    if (cudaGetLastError() == cudaSuccess) return RKV_OK;
    return RKV_ERR_CUDA;
}

}  // namespace rkv
