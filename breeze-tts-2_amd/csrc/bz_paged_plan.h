// How the work of one attention launch over a paged cache is cut (device side).
//
// A segment is a set of rows and the keys they attend together: sequence b's rows
// and its own positions (segment b), or a shared prefix and the rows of all its
// sequences (segment B + g).  A segment's rows, one for each query head of a
// key/value head, go in tiles of M; the keys that a tile attends in chunks of C; a
// (tile, chunk) is a slot, and a workgroup takes a slot of one key/value head.
// Lengths are known on the device alone, so every workgroup works out the slots by
// itself from the lengths (64 segments at a time, one wave scan each).  C is the
// same for all segments, so that workgroups have like amounts however ragged the batch
// is: about 1 / target of all keys, at least min_chunk.
#pragma once

#include "bz_paged_kv.h"

namespace bz {

struct PagedSeg {
    int first, rows;  // rows of q and out
    int keys;
    int seq;    // the sequence, or B + the prefix
    bool back;  // its starts decrease
};

// Segment B + p: prefix p.
__device__ __forceinline__ PagedSeg paged_seg(const PagedKv& c, int s) {
    PagedSeg g = {0, 0, 0, s, false};
    if (s < c.B) {
        const RowRange r = seq_rows(c, s);
        g.first = r.first;
        g.rows = r.end - r.first;
        g.back = r.back;
        g.keys = min(max(c.kv_lens[s], 0), c.width << c.shift);
    } else {
        const int p = s - c.B;
        int lo = 0, hi = c.B;
        if (c.prefix_seqs) {
            const int from = c.prefix_seqs[p], to = c.prefix_seqs[p + 1];
            lo = min(max(from, 0), c.B);
            hi = min(max(to, lo), c.B);
            g.back = to < from;
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
    int tile, split;
    int chunk;       // keys of a chunk
    int first_slot;  // of its tile
    bool any;
};

struct PagedCut {
    int M, log2_M;
    float target;  // slots of one key/value head that the keys are cut for
    int min_chunk;
};

// How a segment's tiles are cut: tile t has 1 + (number of i >= 1 with from(i) <= t) chunks.
struct SegCut {
    int tiles, whole, most;  // chunks that all tiles have, that any has
    int behind;              // keys before the first row's own position (all attend them)
    int chunk, G, log2_M;
    // the first tile with more than i chunks, i >= whole: that of row i chunk - behind
    __device__ __forceinline__ int from(int i) const {
        return (int)min(((int64_t)i * chunk - behind) * G >> log2_M, (int64_t)tiles);
    }
    __device__ __forceinline__ int slots() const {
        int n = tiles * whole;
        for (int i = whole; i < most; ++i) n += tiles - from(i);
        return n;
    }
};
__device__ __forceinline__ SegCut seg_cut(const PagedKv& c, const PagedSeg& g, int chunk, const PagedCut& cut) {
    SegCut k;
    k.tiles = (g.rows * c.G + cut.M - 1) >> cut.log2_M;
    k.chunk = chunk;
    k.G = c.G;
    k.log2_M = cut.log2_M;
    k.most = max(1, (int)(((unsigned)g.keys + chunk - 1) / (unsigned)chunk));
    // row i of a sequence attends behind + i + 1 keys
    k.behind = g.seq < c.B ? max(c.kv_lens[min(g.seq, c.B - 1)], 0) - g.rows : g.keys;
    k.whole = k.most;
    if (g.seq < c.B && g.rows > 1) k.whole = min(k.most, k.behind >= 0 ? (int)((unsigned)k.behind / (unsigned)chunk) + 1 : 1);
    return k;
}

// Slot `slot`: the prefixes' come first, and of a sequence its last tiles' (whose rows
// attend most), so that long pieces start early.  Starts that decrease would put a row
// into several segments, more slots than there is room for: of such a batch there are none.
__device__ __forceinline__ PagedSlot paged_slot(const PagedKv& c, const PagedCut& cut, int slot, int lane) {
    const int n = c.groups + c.B;
    auto seg = [&](int i) {
        PagedSeg g = {};
        if (i < n) g = paged_seg(c, i < c.groups ? c.B + i : i - c.groups);
        return g;
    };
    float work = 0.0f;
    bool back = false;
    PagedSeg g = {};
    for (int i = 0; i < n; i += 64) {
        g = seg(i + lane);
        back |= g.back;
        float keys = (float)g.keys;
        if (g.seq < c.B && g.rows > 1) {  // of a tile on average, or more (a row attends half of the new ones)
            const float kv = (float)max(c.kv_lens[g.seq], 0);
            keys = fminf(keys, fmaxf(kv - 0.5f * (float)g.rows, 0.5f * kv) + (float)cut.M / (float)c.G + 1.0f);
        }
        work += (float)((g.rows * c.G + cut.M - 1) >> cut.log2_M) * keys;
    }
    work = wave_sum(work);
    const int chunk = __builtin_amdgcn_readfirstlane(
        max(cut.min_chunk, ((int)ceilf(fminf(work / cut.target, 1073741824.0f)) + 31) & ~31));
    PagedSlot r = {};
    r.chunk = chunk;
    if (__ballot(back)) return r;
    int base = 0;
    for (int i = 0; i < n; i += 64) {
        if (n > 64) g = seg(i + lane);
        SegCut sc = seg_cut(c, g, chunk, cut);
        const int mine = sc.slots();
        const int end = base + wave_scan(mine);
        const uint64_t behind = __ballot(end > slot);
        if (behind) {
            const int k = __builtin_ctzll(behind);
            r.seg.first = __builtin_amdgcn_readlane(g.first, k);
            r.seg.rows = __builtin_amdgcn_readlane(g.rows, k);
            r.seg.keys = __builtin_amdgcn_readlane(g.keys, k);
            r.seg.seq = __builtin_amdgcn_readlane(g.seq, k);
            sc.tiles = __builtin_amdgcn_readlane(sc.tiles, k);
            sc.whole = __builtin_amdgcn_readlane(sc.whole, k);
            sc.most = __builtin_amdgcn_readlane(sc.most, k);
            sc.behind = __builtin_amdgcn_readlane(sc.behind, k);
            int at = slot - __builtin_amdgcn_readlane(end - mine, k);
            // from the last tile down, those with the most chunks first
            int parts = sc.most, top = sc.tiles;
            for (;; --parts) {
                const int low = parts > sc.whole ? sc.from(parts - 1) : 0;
                const int slots = (top - low) * parts;
                if (at < slots || low == 0) break;
                at -= slots;
                top = low;
            }
            const int back = at / parts;
            r.tile = top - 1 - back;
            r.split = at - back * parts;
            r.first_slot = slot - r.split;
            r.any = true;
            return r;
        }
        base = __builtin_amdgcn_readlane(end, 63);
    }
    return r;
}

// Where a tile's first slot is noted for the joining of its chunks: distinct for the tiles
// of one kind, and to be had from a row without the other segments (those before it fill at
// most first G / M tiles and one more each).
__device__ __forceinline__ int tile_note(const PagedKv& c, const PagedSeg& g, int tile, int M) {
    return g.first * c.G / M + (g.seq < c.B ? g.seq : g.seq - c.B) + tile;
}

// Slots that a launch over so many tiles can have.
inline int64_t paged_slots(int64_t tiles, int target) { return tiles + target + 8; }  // (the work is summed in fp32)

}  // namespace bz
