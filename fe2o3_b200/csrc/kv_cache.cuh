// The paged key-value cache: where a row lies, and what its elements stand for.
#pragma once
#include "common.cuh"

#ifdef __CUDACC__

struct KvCache {
    uint8_t *k, *v;
    float *k_scales, *v_scales;
    const uint32_t *page_table, *lengths;
    uint32_t pages, page_size, table_width, kv_heads, dim, batch;
    uint32_t *status;
};

template <typename Args>
static inline KvCache kv_cache_of(const fe2o3_ctx *ctx, const Args *a) {
    const uint64_t page = (uint64_t)a->kv_heads * a->page_size * a->dim;
    return KvCache{reinterpret_cast<uint8_t *>(a->k_cache.ptr),
                   reinterpret_cast<uint8_t *>(a->v_cache.ptr),
                   reinterpret_cast<float *>(a->k_scales.ptr),
                   reinterpret_cast<float *>(a->v_scales.ptr),
                   reinterpret_cast<const uint32_t *>(a->page_table.ptr),
                   reinterpret_cast<const uint32_t *>(a->lengths.ptr),
                   (uint32_t)(a->k_cache.len / page),
                   a->page_size,
                   a->table_width,
                   a->kv_heads,
                   a->dim,
                   a->batch,
                   ctx->status_word};
}

// Whether a sequence of n positions fits its row of the page table (and 31 bits).
__device__ __forceinline__ bool kv_fits(const KvCache &c, uint32_t n) {
    return n <= 0x7fffffffu && n <= (uint64_t)c.table_width * c.page_size;
}

// Row number of (sequence, head, position); ~0 and a report where the table names a page outside the cache.
// `shift`: log2 of the page size, or negative.
__device__ __forceinline__ uint32_t kv_row(const KvCache &c, uint32_t b, uint32_t h, uint32_t position, int32_t shift = -1) {
    const uint32_t in_table = shift >= 0 ? position >> shift : position / c.page_size, slot = position - in_table * c.page_size;
    const uint32_t page = c.page_table[(uint64_t)b * c.table_width + in_table];
    if (page >= c.pages) {
        kstatus_set(c.status, FE2O3_KSTATUS_SLOT_RANGE);
        return ~0u;
    }
    return (page * c.kv_heads + h) * c.page_size + slot;
}

template <uint32_t FORMAT>
constexpr uint32_t kKvBytes = FORMAT == FE2O3_KV_BF16 ? 2 : 1;   // of an element
template <uint32_t FORMAT>
constexpr float kKvTop = FORMAT == FE2O3_KV_E4M3 ? 448.f : 127.f;   // the largest code

#endif  // __CUDACC__
