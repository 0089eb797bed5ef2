/*
 * bz_paged.h -- C ABI of the operators over a paged key/value cache in
 * libbzgemv.so (gfx950): writing new tokens into the pages, and attention of
 * each sequence's newest rows over them, also for batches whose sequences
 * begin with a shared prefix.
 *
 * Conventions are those of bz_gemv.h (device pointers owned by the caller,
 * stream = hipStream_t as void*, errors detected on the host before any
 * launch, no allocation or host synchronization, bf16 = raw uint16).  No
 * counterpart in the reference, whose caches are static [B][HKV][S][D] tensors
 * of one fill position (models/fused/kernels.py:376-536).
 *
 * The cache is a pool of pages of page_size positions.  Position j of
 * sequence b lies in page block_table[b][j / page_size] at place
 * j % page_size; the table's entries of positions that are not attended or
 * written are never read.  An entry outside [0, num_pages) is a page that is not
 * there: nothing is written to its positions and no row attends them.
 *
 * Rows: T rows of qkv, q and out.  Sequence b has the rows q_starts[b] ..
 * q_starts[b + 1] - 1 (non-decreasing, else the rows hold anything; the ends clamped to [0, T]), one row b
 * each when q_starts is NULL (then T = B).  They are its newest positions:
 * with n rows, row i of the sequence is position kv_lens[b] - n + i, so
 * kv_lens counts the new rows.  A row at a negative position is written nowhere
 * and attends none of the sequence's own positions.  Rows of no sequence are not
 * touched: their q_out and out stay as they were.
 *
 * Lengths, tables and starts are read on the device when a call runs, so a
 * captured graph follows them.
 */
#ifndef BZ_PAGED_H
#define BZ_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "bz_gemv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* kv_dtype: BZ_DT_BF16, or BZ_KV_E4M3 (OCP e4m3 codes of value / scale). */
#define BZ_KV_E4M3 3

typedef struct bz_paged_kv {
    int32_t abi_version; /* BZ_ABI_VERSION */
    int32_t T;           /* rows; append, and attention that takes two launches, refuse 2^24 or more */
    int32_t B;           /* sequences */
    int32_t HQ, HKV, D;  /* HQ % HKV == 0, HQ / HKV <= 16; D 64, 128 or 256 */
    int32_t kv_dtype;
    int32_t page_size;   /* a power of two, 16 .. 4096 */
    int32_t num_pages;   /* pages of the pool */
    int32_t table_width; /* pages a row of block_table holds */
    int32_t groups;      /* shared prefixes; 0: none, and the fields of prefixes are not read */
    int32_t prefix_width;
    void* k_pages; /* 16-byte aligned, also every stride in bytes; a position's D elements are contiguous */
    void* v_pages;
    int64_t k_page, k_head, k_pos; /* elements from a page / kv head / position to the next */
    int64_t v_page, v_head, v_pos;
    const float* k_scale; /* [HKV], BZ_KV_E4M3 only: a code stands for code * scale (of any sign, or 0) */
    const float* v_scale;
    const int32_t* block_table; /* [B][ld_table] */
    int64_t ld_table;
    const int32_t* kv_lens;  /* [B] */
    const int32_t* q_starts; /* [B + 1], or NULL */
    /* Prefix g, prefix_lens[g] positions in the pages prefix_table[g][..], comes
     * before the own positions of the sequences prefix_seqs[g] ..
     * prefix_seqs[g + 1] - 1 (non-decreasing; NULL with one group: all). */
    const int32_t* prefix_table; /* [groups][ld_prefix] */
    int64_t ld_prefix;
    const int32_t* prefix_lens; /* [groups] */
    const int32_t* prefix_seqs; /* [groups + 1], or NULL */
} bz_paged_kv;

/* New tokens into the cache: per-head q/k RMSNorm (q_norm / k_norm bf16 [D],
 * both or neither) and rotate-half RoPE in fp32, k and v of every row into its
 * position's page (bf16, or e4m3 of value / scale, saturated at 448, NaN for 0 / 0), the
 * rotated q to q_out (bf16 [T][ld_q], head h at columns h D ..; must not overlap
 * qkv).  qkv bf16 [T][ld_qkv], columns [q heads | k heads | v heads] x D.
 * cos / sin [cs_rows][ld_cs], bf16 or fp32: row t uses row positions[t] (int64
 * [T]), or without positions its own position.  A row whose rotary row lies outside
 * [0, cs_rows) is written to no page and its q is zero.  Two rows of one place
 * (sequences that share a page they write to) leave one of the two there.
 * The prefix fields are not used.  qkv, q_out 16-byte aligned, also their rows;
 * cos and sin aligned to 8 elements. */
int bz_paged_rope_cache(const bz_paged_kv* kv, const void* qkv, int64_t ld_qkv,
                        const void* q_norm, const void* k_norm, float eps,
                        const void* cos, const void* sin, int32_t cs_dtype,
                        int64_t ld_cs, int64_t cs_rows,
                        const int64_t* positions, void* q_out, int64_t ld_q,
                        void* stream);

/* out[t][h] = softmax(scale q k^T) v of query head h of row t over its group's
 * prefix positions and its sequence's own positions up to the row's, key/value
 * head h / (HQ / HKV).  q bf16 [T][ld_q], out bf16 [T][ld_out] (must not overlap
 * q), head h at columns h D ..  A row that attends nothing is zero.  Keys and
 * values that a row does not attend have no part in it, whatever they hold.
 * scale > 0.  workspace: bz_paged_attn_workspace bytes, 16-byte aligned, zeroed
 * once before its first use (the kernels leave the counters at its front at zero
 * again, whatever the sizes of the calls); calls that share one must not overlap.
 * A call can be two launches that hand over through the workspace: host threads that
 * share one, on the same stream too, make their calls one after the other. */
int bz_paged_attn(const bz_paged_kv* kv, const void* q, int64_t ld_q,
                  float scale, void* workspace, size_t workspace_bytes,
                  void* out, int64_t ld_out, void* stream);

/* Workspace bytes of bz_paged_attn for these sizes (pointers and strides are not
 * read); 0 also for sizes that it refuses. */
size_t bz_paged_attn_workspace(const bz_paged_kv* kv);

#ifdef __cplusplus
}
#endif

#endif /* BZ_PAGED_H */
