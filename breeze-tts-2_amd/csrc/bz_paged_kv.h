// Shared by the kernels over a paged key/value cache (include/bz_paged.h).
#pragma once

#include <algorithm>

#include "bz_device.h"
#include "bz_paged.h"

namespace bz {

constexpr int kPagedMaxG = 16;  // query heads of one key/value head
constexpr int kPagedMaxGrid = 1 << 24;  // workgroups of 256 threads: less than this

// What a kernel needs of the cache; strides in bytes.
struct PagedKv {
    int T, B, HQ, HKV, G;
    int shift;       // log2 of the page size
    int num_pages;
    int width, prefix_width, groups;
    char* k;
    char* v;
    int64_t k_page, k_head, v_page, v_head;
    int64_t k_pos, v_pos;
    const float* k_scale;
    const float* v_scale;
    const int32_t* table;
    int64_t ld_table;
    const int32_t* kv_lens;
    const int32_t* q_starts;
    const int32_t* prefix_table;
    int64_t ld_prefix;
    const int32_t* prefix_lens;
    const int32_t* prefix_seqs;
};

// Rows [first, end) of sequence b.
struct RowRange {
    int first, end;
    bool back;  // its starts decrease (it is then empty)
};
__device__ __forceinline__ RowRange seq_rows(const PagedKv& c, int b) {
    if (!c.q_starts) return {b, b + 1, false};
    const int from = c.q_starts[b], to = c.q_starts[b + 1], s = min(max(from, 0), c.T);
    return {s, min(max(to, s), c.T), to < from};
}

// The sequence of row t: the number of ends at or before it (B for a row of no
// sequence behind the last one).  q_starts[1..B] is read 64 entries at a time.
__device__ __forceinline__ int seq_of_row(const PagedKv& c, int t, int lane) {
    if (!c.q_starts) return t;
    int b = 0;
    for (int i = 0; i < c.B; i += 64) {
        const int end = i + lane < c.B ? c.q_starts[i + lane + 1] : 0x7FFFFFFF;
        const int n = __builtin_popcountll(__ballot(end <= t));
        b += n;
        if (n < 64) break;
    }
    return b;
}

inline bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Sizes alone: what bz_paged_attn_workspace can be asked.
inline int paged_check_sizes(const bz_paged_kv* d) {
    if (!d) return BZ_ERR_INVALID_ARG;
    if (d->abi_version != BZ_ABI_VERSION) return BZ_ERR_ABI;
    if (d->T < 1 || d->B < 1 || d->HQ < 1 || d->HKV < 1 || d->HQ % d->HKV || d->num_pages < 1 || d->table_width < 1 ||
        d->groups < 0 || (d->groups > 0 && d->prefix_width < 1))
        return BZ_ERR_INVALID_ARG;
    if (d->kv_dtype != BZ_DT_BF16 && d->kv_dtype != BZ_KV_E4M3) return BZ_ERR_INVALID_ARG;
    if (d->D != 64 && d->D != 128 && d->D != 256) return BZ_ERR_UNSUPPORTED;
    if (d->HQ / d->HKV > kPagedMaxG) return BZ_ERR_UNSUPPORTED;
    if (d->page_size < 16 || d->page_size > 4096 || (d->page_size & (d->page_size - 1))) return BZ_ERR_UNSUPPORTED;
    // positions, and rows times heads, are 32-bit numbers
    if ((int64_t)d->table_width * d->page_size > 0x40000000 || (int64_t)d->T * d->HQ > 0x40000000 ||
        (d->groups > 0 && (int64_t)d->prefix_width * d->page_size > 0x40000000) || d->HQ > 0x10000)
        return BZ_ERR_UNSUPPORTED;
    return BZ_OK;
}

inline int paged_setup(const bz_paged_kv* d, PagedKv& c) {
    const int rc = paged_check_sizes(d);
    if (rc != BZ_OK) return rc;
    if (!d->k_pages || !d->v_pages || !d->block_table || !d->kv_lens) return BZ_ERR_INVALID_ARG;
    if (!d->q_starts && d->T != d->B) return BZ_ERR_SHAPE;
    const int es = d->kv_dtype == BZ_DT_BF16 ? 2 : 1;
    if ((es == 1) != (d->k_scale != nullptr) || (es == 1) != (d->v_scale != nullptr)) return BZ_ERR_INVALID_ARG;
    if (d->ld_table < d->table_width) return BZ_ERR_SHAPE;
    if (!aligned_to(d->k_pages, 16) || !aligned_to(d->v_pages, 16)) return BZ_ERR_ALIGNMENT;
    for (const int64_t s : {d->k_page, d->k_head, d->k_pos, d->v_page, d->v_head, d->v_pos}) {
        if (s < d->D) return BZ_ERR_SHAPE;
        if (s * es % 16) return BZ_ERR_ALIGNMENT;
    }
    // 32-bit offsets within one page of one head
    if (d->k_pos * es > 0x40000000 / d->page_size || d->v_pos * es > 0x40000000 / d->page_size)
        return BZ_ERR_UNSUPPORTED;
    if (d->groups > 0) {
        if (!d->prefix_table || !d->prefix_lens || (d->groups > 1 && !d->prefix_seqs)) return BZ_ERR_INVALID_ARG;
        if (d->ld_prefix < d->prefix_width) return BZ_ERR_SHAPE;
    }
    c.T = d->T;
    c.B = d->B;
    c.HQ = d->HQ;
    c.HKV = d->HKV;
    c.G = d->HQ / d->HKV;
    c.shift = __builtin_ctz((unsigned)d->page_size);
    c.num_pages = d->num_pages;
    c.width = d->table_width;
    c.groups = d->groups;
    c.prefix_width = d->groups > 0 ? d->prefix_width : 0;
    c.k = static_cast<char*>(d->k_pages);
    c.v = static_cast<char*>(d->v_pages);
    c.k_page = d->k_page * es;
    c.k_head = d->k_head * es;
    c.k_pos = d->k_pos * es;
    c.v_page = d->v_page * es;
    c.v_head = d->v_head * es;
    c.v_pos = d->v_pos * es;
    c.k_scale = d->k_scale;
    c.v_scale = d->v_scale;
    c.table = d->block_table;
    c.ld_table = d->ld_table;
    c.kv_lens = d->kv_lens;
    c.q_starts = d->q_starts;
    c.prefix_table = d->prefix_table;
    c.ld_prefix = d->ld_prefix;
    c.prefix_lens = d->prefix_lens;
    c.prefix_seqs = d->prefix_seqs;
    return BZ_OK;
}

}  // namespace bz
