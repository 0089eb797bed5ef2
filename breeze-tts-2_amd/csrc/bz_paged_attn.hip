// Attention of each sequence's newest rows over a paged key/value cache
// (include/bz_paged.h), with shared prefixes: the launches.
#include "bz_paged_attn.h"
#include "bz_paged_stream.h"
#include "bz_paged_tile.h"

namespace bz {

// Workgroups that the keys are cut for: for few rows about as many as run at once, so that none
// starts late.  us with the number here, and fewer and more, calls in a graph: 48 sequences of up to 4095 positions, 16 / 8
// heads of 128, 768 82 (512 87, 1024 85), of 64 1024 41 (768 44, 1280 39.5); four of 30 .. 65 thousand, 16 / 8 of 64 1024 88
// (768 85, 1280 91), of 128 768 165 (512 189, 1024 172), 16 / 4 of 256, e4m3, 512 101 (256 123, 768 106), bf16 256 225 (384
// 171, 512 183); five tokens for 16 of up to 2043, 8 / 2 of 128, 512 16.6 (256 .. 1024 the same), of up to 16000 45 (384 42, 768 53).
// For many rows two to a CU, less those that a tile's last, shorter chunk adds.
// us with 384 / 416 / 448 / 512, calls in a graph: a prompt of 2011 tokens, bf16, 16 / 8 heads of 128
// 39 / 38 / 38 / 51, of 64 27 / 27 / 27 / 38, 16 / 4 of 256 75 / 74 / 81 / 90; chunks of three prompts, 16 / 4
// of 256 298 / 281 / 282 / 311 (e4m3 302 / 288 / 283 / 321), 16 / 8 of 128 144 / 177 / 148 / 157 (e4m3 160 / 197 /
// 155 / 162), 6 / 2 of 64 49 / 46 / 46 / 58; 24 sequences in three groups, e4m3, 16 / 4 of 256 42 / 44 / 43 / 54.
// Not the best for every batch: how a batch's chunks fall into whole rounds of workgroups differs.
static int paged_workgroups(int D, bool f8, int M) {
    if (M > 32) return 416;
    if (D == 256) return f8 ? 512 : 256;
    return D == 64 ? (M == 16 ? 1024 : 768) : (M == 16 ? 768 : 512);
}

// The parts of a row joined in a launch of its own: its prefix's, then its own.
// Four columns of a head to P threads, which take its parts in turn.
template <int D, int P>
__global__ void __launch_bounds__(256) paged_attn_bf16_join(PagedKv c, PagedAttn a, bool f8) {
    constexpr int kItems = 256 / P;
    __shared__ float st[P > 1 ? 256 : 1][8];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, M = a.cut.M;
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
        const int k = max(t - g.first, 0) * c.G + (min(h, c.HQ - 1) - head * c.G), tile = k >> a.cut.log2_M;
        const uint64_t note = (part ? a.to.notes : a.to.prefix_notes)[(int64_t)tile_note(c, g, tile, M) * c.HKV + head];
        const int kv_len = part ? max(c.kv_lens[b], 0) : 0, chunk = (int)(note >> 32);
        const int slot = (int)min((uint32_t)note, (uint32_t)a.slots - 1u);  // (anything, if starts decrease)
        at[part] = ((int64_t)slot * c.HKV + head) * M + (k - tile * M);
        n[part] = min(parts_of(row_limit(g, kv_len, part, row), chunk), a.slots - slot);
        if (c.groups == 0) {
            const int last = min(g.rows * c.G, (tile + 1) * M) - 1;
            whole = parts_of(row_limit(g, kv_len, true, last / c.G), chunk) == 1;
        }
    }
    PagedSum sum;
    if (on && !whole)
        for (int part = 0; part < 2; ++part) sum.add_parts<false>(a.to, at[part], (int64_t)c.HKV * M, n[part], p, P, D, d);
    sum.across(st, tid, P, kItems, on && p == 0);
    if (on && !whole && p == 0)
        sum.store(a.out + (int64_t)t * a.ld_out + (int64_t)h * D + d, f8 ? c.v_scale[head] : 1.0f);
}

struct PagedPlan {
    PagedCut cut;
    int64_t slots;
    bool join;    // a tile may have several parts
    bool inside;  // which the last of its workgroups joins
    int notes;    // tiles of sequences
    size_t part_at, ml_at, notes_at, prefix_notes_at;  // in the workspace, whose first bytes are the counters
    size_t bytes;
};

// Arrival counters, at the front of every workspace whatever the sizes of a call: they stay
// zero between calls of different sizes.
constexpr int kPagedCounters = 16384;

// Rows of a tile for segments of `rows` query rows: the fewest of the sizes that hold a segment, so that
// its keys are read once; 128 for longer ones.  Both sides of the borders, us of a call in a graph, 16
// sequences of 97 .. 2043 positions before their rows, bf16:
//   8 / 2 heads of 128   20 rows in tiles of 16 / 32 19.9 / 16.6, 40 in 32 / 64 26.4 / 22.2, 80 in 64 / 128 27.3 / 27.8
//   16 / 8 of 128        18 in 16 / 32 29.7 / 31.9, 40 in 32 / 64 42.1 / 29.4, 80 in 64 / 128 29.2 / 32.4
//   16 / 1 of 64         32 in 16 / 32 11.8 / 13.1, 64 in 32 / 64 13.4 / 15.9, 128 in 64 / 128 17.3 / 20.4
//   16 / 4 of 256        20 in 16 / 64 43.4 / 42.0, 80 in 64 / 128 57.8 / 48.6 (e4m3 34.7 / 27.1 and 39.7 / 48.0)
// and in tiles of 64 / 128: a prompt of 2011 tokens, 16 / 8 of 128, 50.3 / 38.8; chunks of three prompts, 16 / 4 of 256, 536 /
// 281.  One rule for all heads and types: beside its borders another size can be up to a third faster (tiles
// of 64 for 18 .. 32 rows of 16 / 8 heads of 128, 26.4, and for 80 .. 128 rows in e4m3 of 256; of 32 for 64 .. 128 of 16 / 1 of 64).
static int paged_tile_rows(int64_t rows, int D) {
    if (rows <= 16) return 16;
    if (D == 256) return rows <= 64 ? 64 : 128;
    return rows <= 32 ? 32 : (rows <= 64 ? 64 : 128);
}

static PagedPlan paged_plan(const bz_paged_kv* d) {
    PagedPlan p = {};
    const int G = d->HQ / d->HKV;
    const bool f8 = d->kv_dtype != BZ_DT_BF16;
    // by what a segment has on average, a prefix's or a sequence's
    const int64_t segs = d->groups > 0 ? std::min(d->B, d->groups) : d->B;
    const int M = paged_tile_rows(((int64_t)d->T + segs - 1) / segs * G, d->D);
    const int target = std::max(1, paged_workgroups(d->D, f8, M) / d->HKV);
    p.cut.M = M;
    p.cut.log2_M = __builtin_ctz(M);
    p.cut.target = (float)target;
    // a step for each of four waves; two where a part has more rows to be joined (verification
    // of 5 tokens, 16 sequences of up to 2043 positions, 8 / 2 heads of 128: 20.4 us with 128 and 17.2
    // with 256; one token, 2 of 610, 16 / 8 heads: 9.4 and 9.9)
    p.cut.min_chunk = M == 16 ? 128 : 256;
    // tiles that there can be, and with them notes
    const int64_t notes = (int64_t)d->T * G / M + d->B, prefix_notes = d->groups > 0 ? (int64_t)d->T * G / M + d->groups : 0;
    p.join = d->groups > 0 || (int64_t)d->table_width * d->page_size > p.cut.min_chunk;
    p.inside = p.join && (notes + prefix_notes) * d->HKV <= kPagedCounters &&
               (d->groups == 0 || (M <= 32 && !d->q_starts && M % G == 0));
    p.notes = (int)notes;
    // (and no tile has more chunks than its table has room for; workgroups without a slot cost no time that
    // could be measured, 848 for 80 with one, but their room in the workspace)
    auto chunks = [&](int64_t positions) { return (positions + p.cut.min_chunk - 1) / p.cut.min_chunk; };
    const int64_t room = notes * chunks((int64_t)d->table_width * d->page_size) +
                         prefix_notes * chunks((int64_t)d->prefix_width * d->page_size);
    p.slots = p.join ? std::min(paged_slots(notes + prefix_notes, target), room) : notes;
    p.bytes = kPagedCounters * sizeof(unsigned);
    auto take = [&](size_t n) {
        const size_t at = p.bytes;
        p.bytes += (n + 15) & ~(size_t)15;
        return at;
    };
    const size_t rows = p.join ? (size_t)p.slots * d->HKV * M : 0;
    p.part_at = take(rows * d->D * sizeof(float));
    p.ml_at = take(rows * sizeof(float2));
    p.notes_at = take((size_t)notes * d->HKV * sizeof(uint64_t));
    p.prefix_notes_at = take((size_t)prefix_notes * d->HKV * sizeof(uint64_t));
    return p;
}

// Whether the launches' grids can be: one of less than 2^32 threads in each dimension, 256 or 512
// to a workgroup.
static bool paged_plan_fits(const bz_paged_kv* d, const PagedPlan& p) {
    return p.slots * d->HKV <= 0x7FFFFF && (!p.join || p.inside || d->T < kPagedMaxGrid);
}

template <int D, bool F8>
static void launch_tiles(const PagedKv& c, const PagedAttn& a, int64_t slots, hipStream_t st) {
    const dim3 grid((unsigned)(slots * c.HKV));
    switch (a.cut.M) {
        case 16:
            hipLaunchKernelGGL((paged_attn_bf16_stream<D, F8, 1>), grid, dim3(256), 0, st, c, a);
            break;
        case 32:
            if constexpr (D < 256) hipLaunchKernelGGL((paged_attn_bf16_stream<D, F8, 2>), grid, dim3(256), 0, st, c, a);
            break;
        case 64:
            hipLaunchKernelGGL((paged_attn_bf16_tile<D, F8, 4, true>), grid, dim3(256), 0, st, c, a);
            break;
        default:
            if constexpr (D == 256)
                hipLaunchKernelGGL((paged_attn_bf16_tile<D, F8, 8, true>), grid, dim3(512), 0, st, c, a);
            else
                hipLaunchKernelGGL((paged_attn_bf16_tile<D, F8, 4, false>), grid, dim3(256), 0, st, c, a);
    }
}

template <int D>
static void launch_attn(const PagedKv& c, PagedAttn a, const PagedPlan& p, char* ws, bool f8, hipStream_t st) {
    a.cut = p.cut;
    a.own_notes = p.notes;
    a.slots = (int)p.slots;
    a.to = {reinterpret_cast<float*>(ws + p.part_at), reinterpret_cast<float2*>(ws + p.ml_at),
            reinterpret_cast<uint64_t*>(ws + p.notes_at), reinterpret_cast<uint64_t*>(ws + p.prefix_notes_at)};
    if (f8)
        launch_tiles<D, true>(c, a, p.slots, st);
    else
        launch_tiles<D, false>(c, a, p.slots, st);
    if (!p.join || p.inside) return;
    const int items = c.HQ * (D / 4);
    // few items leave CUs idle, so several threads share one's parts.  us of a call in a graph with P and 1 threads:
    // rows behind one prefix of 6007, 16 / 8 heads of 128, 32768 items 40.3 and 40.4, 65536 61.0 and 57.5, 131072 117 and 109;
    // 16 / 4 of 256, 49152 39.7 and 41.0, 131072 76.2 and 73.2; 8 / 2 of 64, 16384 22.8 and 24.6, 65536 52.3 and 48.7
    constexpr int P = 1024 / D > 8 ? 8 : 1024 / D;
    if ((int64_t)c.T * items <= 65536)
        hipLaunchKernelGGL((paged_attn_bf16_join<D, P>), dim3(c.T, (items * P + 255) / 256), dim3(256), 0, st, c, a, f8);
    else
        hipLaunchKernelGGL((paged_attn_bf16_join<D, 1>), dim3(c.T, (items + 255) / 256), dim3(256), 0, st, c, a, f8);
}

}  // namespace bz

using namespace bz;

extern "C" size_t bz_paged_attn_workspace(const bz_paged_kv* kv) {
    if (paged_check_sizes(kv) != BZ_OK) return 0;
    const PagedPlan p = paged_plan(kv);
    return paged_plan_fits(kv, p) ? p.bytes : 0;
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
    if (!paged_plan_fits(kv, p)) return BZ_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < p.bytes) return BZ_ERR_INVALID_ARG;
    PagedAttn a = {};
    a.q = static_cast<const uint16_t*>(q);
    a.ld_q = ld_q;
    a.scale = scale;
    a.out = static_cast<uint16_t*>(out);
    a.ld_out = ld_out;
    a.arrived = p.inside ? static_cast<unsigned*>(workspace) : nullptr;
    const bool f8 = kv->kv_dtype == BZ_KV_E4M3;
    char* ws = static_cast<char*>(workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: launch_attn<64>(c, a, p, ws, f8, st); break;
        case 128: launch_attn<128>(c, a, p, ws, f8, st); break;
        default: launch_attn<256>(c, a, p, ws, f8, st); break;
    }
    return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}
