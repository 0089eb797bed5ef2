// How the work of one attention call over a paged cache is cut (device side).
//
// A segment is a set of rows and the keys they attend together: sequence b's rows
// and its own positions (segment b), or a shared prefix and the rows of all its
// sequences (segment B + g).  A segment's rows, one for each query head of a
// key/value head, go in tiles of M; its keys in chunks of C; a (tile, chunk) is a
// slot, and a workgroup takes a slot of one key/value head.  Lengths are known on
// the device alone, so every workgroup works out the slots by itself from the
// lengths (64 segments at a time, one wave scan each).  C is the same for all segments, so
// that workgroups have like amounts however ragged the batch is: about
// 1 / target of all keys, at least min_chunk.
#pragma once

#include "bz_paged_kv.h"

namespace bz {

struct PagedSeg {
    int first, rows;  // rows of q and out
    int keys;
    int seq;    // the sequence, or B + the prefix
};

__device__ __forceinline__ PagedSeg paged_seg(const PagedKv& c, int s) {
    PagedSeg g = {0, 0, 0, s};
    if (s < c.B) {
        const RowRange r = seq_rows(c, s);
        g.first = r.first;
        g.rows = r.end - r.first;
        g.keys = min(max(c.kv_lens[s], 0), c.width << c.shift);
    } else if (s < c.B + c.groups) {
        const int p = s - c.B;
        int lo = 0, hi = c.B;
        if (c.prefix_seqs) {
            lo = min(max(c.prefix_seqs[p], 0), c.B);
            hi = min(max(c.prefix_seqs[p + 1], lo), c.B);
        }
        if (hi > lo) {
            g.first = seq_rows(c, lo).first;
            g.rows = max(seq_rows(c, hi - 1).end - g.first, 0);
        }
        g.keys = min(max(c.prefix_lens[p], 0), c.prefix_width << c.shift);
    }
    return g;
}

// The prefix of sequence b, or -1.
__device__ __forceinline__ int prefix_of_seq(const PagedKv& c, int b, int lane) {
    if (!c.prefix_seqs) return c.groups > 0 ? 0 : -1;
    for (int i = 0; i < c.groups; i += 64) {
        const int p = min(i + lane, c.groups - 1);
        const uint64_t hit = __ballot(i + lane < c.groups && c.prefix_seqs[p] <= b && b < c.prefix_seqs[p + 1]);
        if (hit) return i + __builtin_ctzll(hit);
    }
    return -1;
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int v) {
#define BZ_SCAN(ctrl, rows) v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xF, false)
    BZ_SCAN(0x111, 0xF);  // row_shr:1
    BZ_SCAN(0x112, 0xF);
    BZ_SCAN(0x114, 0xF);
    BZ_SCAN(0x118, 0xF);
    BZ_SCAN(kDppRowBcast15, 0xA);
    BZ_SCAN(kDppRowBcast31, 0xC);
#undef BZ_SCAN
    return v;
}

struct PagedSlot {
    PagedSeg seg;
    int tile, split, splits;  // splits of its segment
    int chunk;                // keys of a chunk
    int first_slot;           // of its tile
    bool any;
};

__device__ __forceinline__ int tiles_of(const PagedKv& c, int rows, int M) { return (rows * c.G + M - 1) / M; }

__device__ __forceinline__ PagedSlot paged_slot(const PagedKv& c, int M, float target, int min_chunk, int slot,
                                                int lane) {
    const int n = c.B + c.groups;
    float work = 0.0f;
    PagedSeg g = {};
    for (int i = 0; i < n; i += 64) {
        g = paged_seg(c, i + lane);
        work += (float)tiles_of(c, g.rows, M) * (float)g.keys;
    }
    work = wave_sum(work);
    const int chunk = __builtin_amdgcn_readfirstlane(
        max(min_chunk, ((int)ceilf(fminf(work / target, 1073741824.0f)) + 31) & ~31));
    PagedSlot r = {};
    r.chunk = chunk;
    int base = 0;
    for (int i = 0; i < n; i += 64) {
        if (n > 64) g = paged_seg(c, i + lane);
        const int splits = max(1, (int)(((unsigned)g.keys + chunk - 1) / (unsigned)chunk));
        const int mine = tiles_of(c, g.rows, M) * splits;
        const int end = base + wave_scan(mine);
        const uint64_t behind = __ballot(end > slot);
        if (behind) {
            const int k = __builtin_ctzll(behind);
            r.seg.first = __builtin_amdgcn_readlane(g.first, k);
            r.seg.rows = __builtin_amdgcn_readlane(g.rows, k);
            r.seg.keys = __builtin_amdgcn_readlane(g.keys, k);
            r.seg.seq = __builtin_amdgcn_readlane(g.seq, k);
            r.splits = __builtin_amdgcn_readlane(splits, k);
            const int at = slot - __builtin_amdgcn_readlane(end - mine, k);
            r.tile = at / r.splits;
            r.split = at - r.tile * r.splits;
            r.first_slot = slot - r.split;
            r.any = true;
            return r;
        }
        base = __builtin_amdgcn_readlane(end, 63);
    }
    return r;
}

// Where a tile's slots are noted for the joining of its chunks: distinct for the
// tiles of a call, and to be had from a row without the other segments (a
// sequence's rows before it fill at most first G / M tiles and one more each).
__device__ __forceinline__ int tile_note(const PagedKv& c, const PagedSeg& g, int tile, int M) {
    if (g.seq < c.B) return g.first * c.G / M + g.seq + tile;
    return c.T * c.G / M + c.B + g.first * c.G / M + (g.seq - c.B) + tile;
}

// Slots, and notes, that a call can have.
struct PagedBounds {
    int64_t slots, notes;
};
inline PagedBounds paged_bounds(const bz_paged_kv* d, int M, int target) {
    const int64_t rows = (int64_t)d->T * (d->HQ / d->HKV) / M;
    const int64_t tiles = rows + d->B + (d->groups > 0 ? rows + d->groups : 0);
    return {tiles + target + 64, tiles};  // (the sum of the work is in fp32)
}

}  // namespace bz
