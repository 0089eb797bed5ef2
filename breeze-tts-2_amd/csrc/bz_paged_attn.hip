// Attention of each sequence's newest rows over a paged key/value cache
// (include/bz_paged.h), with shared prefixes: the launches.
#include "bz_paged_attn.h"
#include "bz_paged_stream.h"
#include "bz_paged_tile.h"

namespace bz {

// Workgroups that the keys are cut for: as many as run at once, so that none starts late.
static int paged_workgroups(int D, bool f8, int M) {
    if (M > 32) return 1024;
    if (D == 256) return (f8 ? 512 : 256);
    return (D == 64 ? (M == 16 ? 1024 : 768) : (M == 16 ? 768 : 512));
}

// The parts of a row joined in a launch of its own: its prefix's, then its own.
// Four columns of a head to P threads, which take its parts in turn.
template <int D, int P>
__global__ void __launch_bounds__(256) paged_attn_bf16_join(PagedKv c, PagedAttn a, int M, bool f8) {
    constexpr int kItems = 256 / P;
    __shared__ float st[P > 1 ? 256 : 1][8];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int b = seq_of_row(c, t, lane);
    if (b >= c.B) return;
    const PagedSeg own = paged_seg(c, b);
    const int row = t - own.first;
    if (row < 0 || row >= own.rows) return;
    const int pre = prefix_of_seq(c, b, lane);
    const int item = blockIdx.y * kItems + tid % kItems, p = tid / kItems;
    const int h = item / (D / 4), d = 4 * (item - h * (D / 4));
    const bool on = h < c.HQ;
    const int head = min(h, c.HQ - 1) / c.G;

    int64_t at[2] = {};
    int n[2] = {};
    bool whole = false;  // written by the only workgroup that has keys of the row's tile
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        if (!part && pre < 0) continue;
        const PagedSeg g = part ? own : paged_seg(c, c.B + pre);
        const int k = (t - g.first) * c.G + (min(h, c.HQ - 1) - head * c.G), tile = k / M;
        const int2 note = a.notes[tile_note(c, g, tile, M)];
        const int kv_len = part ? max(c.kv_lens[b], 0) : 0;
        at[part] = ((int64_t)note.x * c.HKV + head) * M + (k - tile * M);
        n[part] = parts_of(row_limit(g, kv_len, part, row), note.y);
        if (c.groups == 0) {
            const int last = min(g.rows * c.G, (tile + 1) * M) - 1;
            whole = parts_of(row_limit(g, kv_len, true, last / c.G), note.y) == 1;
        }
    }
    PagedSum sum;
    if (on && !whole)
        for (int part = 0; part < 2; ++part) sum.add_parts<false>(a, at[part], (int64_t)c.HKV * M, n[part], p, P, D, d);
    sum.across(st, tid, P, kItems, on && p == 0);
    if (on && !whole && p == 0)
        sum.store(a.out + (int64_t)t * a.ld_out + (int64_t)h * D + d, f8 ? c.v_scale[head] : 1.0f);
}

struct PagedPlan {
    int M;       // rows of a tile
    int target;  // slots of one key/value head
    int min_chunk;
    int64_t slots, notes;
    bool join;   // a tile may have several parts
    bool inside; // which the last of its workgroups joins
    size_t part_at, ml_at, notes_at, bytes;  // of the workspace, whose first bytes are the counters
};

// Arrival counters, at the front of every workspace whatever the sizes of a call: they stay
// zero between calls of different sizes.
constexpr int kPagedCounters = 16384;

// Rows of a tile by what a segment has on average.
static PagedPlan paged_plan(const bz_paged_kv* d) {
    PagedPlan p = {};
    const int G = d->HQ / d->HKV;
    const int64_t segs = d->groups > 0 ? std::min(d->B, d->groups) : d->B;
    const int64_t rows = ((int64_t)d->T + segs - 1) / segs * G;
    p.M = rows <= 16 ? 16 : (rows <= 32 && d->D < 256 ? 32 : (rows <= 64 ? 64 : 128));
    p.target = std::max(1, paged_workgroups(d->D, d->kv_dtype != BZ_DT_BF16, p.M) / d->HKV);
    // a step for each of four waves; two where a part has more rows to be joined (verification
    // of 5 tokens, 16 sequences of up to 2043 positions, 8 / 2 heads of 128: 20.4 us with 128 and 17.2
    // with 256; one token, 2 of 610, 16 / 8 heads: 9.4 and 9.9)
    p.min_chunk = p.M == 16 ? 128 : 256;
    const PagedBounds b = paged_bounds(d, p.M, p.target);
    p.notes = b.notes;
    p.join = d->groups > 0 || (int64_t)d->table_width * d->page_size > p.min_chunk;
    p.slots = p.join ? b.slots : b.notes;
    p.inside = p.join && p.M <= 32 && d->groups == 0 && b.notes * d->HKV <= kPagedCounters && d->HKV <= 256;
    const size_t rows_all = p.join ? (size_t)p.slots * d->HKV * p.M : 0;
    p.part_at = kPagedCounters * sizeof(unsigned);
    p.ml_at = p.part_at + rows_all * d->D * sizeof(float);
    p.notes_at = p.ml_at + rows_all * sizeof(float2);
    p.bytes = p.notes_at + (size_t)p.notes * sizeof(int2);
    return p;
}

template <int D, bool F8>
static void launch_stream(const PagedKv& c, const PagedAttn& a, int M, hipStream_t st) {
    const dim3 grid((unsigned)(a.slots * c.HKV)), block(64 * kStreamWaves);
    if (M == 16)
        hipLaunchKernelGGL((paged_attn_bf16_stream<D, F8, 1>), grid, block, 0, st, c, a);
    else if (M == 128)
        hipLaunchKernelGGL((paged_attn_bf16_tile<D, F8, 4>), grid, block, 0, st, c, a);
    else if (M == 64)
        hipLaunchKernelGGL((paged_attn_bf16_tile<D, F8, 2>), grid, block, 0, st, c, a);
    else if constexpr (D < 256)
        hipLaunchKernelGGL((paged_attn_bf16_stream<D, F8, 2>), grid, block, 0, st, c, a);
}

template <int D>
static void launch_attn(const PagedKv& c, const PagedAttn& a, const PagedPlan& p, bool f8, hipStream_t st) {
    if (f8)
        launch_stream<D, true>(c, a, p.M, st);
    else
        launch_stream<D, false>(c, a, p.M, st);
    if (p.join && !p.inside) {
        const int items = c.HQ * (D / 4);
        constexpr int P = 1024 / D > 8 ? 8 : 1024 / D;
        if ((int64_t)c.T * items <= 65536)
            hipLaunchKernelGGL((paged_attn_bf16_join<D, P>), dim3(c.T, (items * P + 255) / 256), dim3(256), 0, st, c, a, p.M, f8);
        else
            hipLaunchKernelGGL((paged_attn_bf16_join<D, 1>), dim3(c.T, (items + 255) / 256), dim3(256), 0, st, c, a, p.M, f8);
    }
}

}  // namespace bz

using namespace bz;

extern "C" size_t bz_paged_attn_workspace(const bz_paged_kv* kv) {
    return paged_check_sizes(kv) == BZ_OK ? paged_plan(kv).bytes : 0;
}

extern "C" int bz_paged_attn(const bz_paged_kv* kv, const void* q, int64_t ld_q, float scale, void* workspace,
                             size_t workspace_bytes, void* out, int64_t ld_out, void* stream) {
    PagedKv c = {};
    const int rc = paged_setup(kv, c);
    if (rc != BZ_OK) return rc;
    if (!q || !out || !(scale > 0.0f) || scale > 3.0e38f) return BZ_ERR_INVALID_ARG;
    const int D = kv->D;
    if (ld_q < (int64_t)c.HQ * D || ld_out < (int64_t)c.HQ * D) return BZ_ERR_SHAPE;
    if (!aligned_to(q, 16) || !aligned_to(out, 16) || ld_q % 8 || ld_out % 8 || !aligned_to(workspace, 16))
        return BZ_ERR_ALIGNMENT;
    const PagedPlan p = paged_plan(kv);
    if (p.slots * c.HKV > 0x7FFFFFFF) return BZ_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < p.bytes) return BZ_ERR_INVALID_ARG;
    char* ws = static_cast<char*>(workspace);
    const PagedAttn a = {static_cast<const uint16_t*>(q),
                         ld_q,
                         scale,
                         static_cast<uint16_t*>(out),
                         ld_out,
                         (float)p.target,
                         p.min_chunk,
                         p.slots,
                         reinterpret_cast<float*>(ws + p.part_at),
                         reinterpret_cast<float2*>(ws + p.ml_at),
                         reinterpret_cast<int2*>(ws + p.notes_at),
                         p.inside ? reinterpret_cast<unsigned*>(ws) : nullptr};
    const bool f8 = kv->kv_dtype == BZ_KV_E4M3;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: launch_attn<64>(c, a, p, f8, st); break;
        case 128: launch_attn<128>(c, a, p, f8, st); break;
        default: launch_attn<256>(c, a, p, f8, st); break;
    }
    return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}
