// Attention of each sequence's newest rows over a paged key/value cache
// (include/bz_paged.h), with shared prefixes: the launches.
#include "bz_paged_attn.h"
#include "bz_paged_stream.h"
#include "bz_paged_tile.h"

namespace bz {

constexpr int kPagedWorkgroups = 1024;  // that the keys are cut for

// The chunks' parts of a row, merged in the keys' order: its prefix's, then its
// own.  Four columns of a head to a thread.
template <int D>
__global__ void __launch_bounds__(256) paged_attn_bf16_join(PagedKv c, PagedAttn a, int M, bool f8) {
    const int t = blockIdx.x, lane = threadIdx.x & 63;
    const int b = seq_of_row(c, t, lane);
    if (b >= c.B) return;
    const PagedSeg own = paged_seg(c, b);
    const int row = t - own.first;
    if (row < 0 || row >= own.rows) return;
    const int pre = prefix_of_seq(c, b, lane);
    const int item = blockIdx.y * 256 + threadIdx.x;
    const int h = item / (D / 4), d = 4 * (item - h * (D / 4));
    if (h >= c.HQ) return;
    const int head = h / c.G;

    float m = -INFINITY, l = 0.0f, o[4] = {};
    for (int part = pre >= 0 ? 0 : 1; part < 2; ++part) {
        const PagedSeg g = part ? own : paged_seg(c, c.B + pre);
        const int k = (t - g.first) * c.G + (h - head * c.G), tile = k / M;
        const int2 note = a.notes[tile_note(c, g, tile, M)];
        if (c.groups == 0 && g.keys <= note.y) return;  // written by its only slot
        const int limit = row_limit(g, part ? max(c.kv_lens[b], 0) : 0, part, row);
        const int n = max(1, (int)(((unsigned)limit + note.y - 1) / (unsigned)note.y));
        const int64_t at = ((int64_t)note.x * c.HKV + head) * M + (k - tile * M), step = (int64_t)c.HKV * M;
        constexpr int U = 4;
        for (int s0 = 0; s0 < n; s0 += U) {
            float2 x[U];
            float4 v[U];
#pragma unroll
            for (int e = 0; e < U; ++e) {
                const int64_t i = at + min(s0 + e, n - 1) * step;
                x[e] = a.ml[i];
                v[e] = *reinterpret_cast<const float4*>(a.part + i * D + d);
            }
            float mn = m;
#pragma unroll
            for (int e = 0; e < U; ++e) mn = fmaxf(mn, x[e].x);
            const float ms = mn == -INFINITY ? 0.0f : mn;
            const float f = mn == -INFINITY ? 1.0f : pg_exp2(m - ms);
            l *= f;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] *= f;
            m = mn;
#pragma unroll
            for (int e = 0; e < U; ++e) {
                if (s0 + e >= n) break;
                const float w = mn == -INFINITY ? 1.0f : pg_exp2(x[e].x - ms);
                l += x[e].y * w;
                o[0] += v[e].x * w;
                o[1] += v[e].y * w;
                o[2] += v[e].z * w;
                o[3] += v[e].w * w;
            }
        }
    }
    const float f = m == -INFINITY ? (l > 0.0f ? __builtin_nanf("") : 0.0f) : 1.0f / l * (f8 ? c.v_scale[head] : 1.0f);
    *reinterpret_cast<uint2*>(a.out + (int64_t)t * a.ld_out + (int64_t)h * D + d) =
        make_uint2(pack_bf16x2(o[0] * f, o[1] * f), pack_bf16x2(o[2] * f, o[3] * f));
}

struct PagedPlan {
    int M;       // rows of a tile
    int target;  // slots of one key/value head
    int64_t slots, notes;
    bool join;
    size_t ml_at, notes_at, bytes;  // of the workspace
};

// Rows of a tile by what a segment has on average.
static PagedPlan paged_plan(const bz_paged_kv* d) {
    PagedPlan p = {};
    const int G = d->HQ / d->HKV;
    const int64_t segs = d->groups > 0 ? std::min(d->B, d->groups) : d->B;
    const int64_t rows = ((int64_t)d->T + segs - 1) / segs * G;
    p.M = rows <= 16 ? 16 : (rows <= 32 && d->D < 256 ? 32 : (rows <= 64 ? 64 : 128));
    p.target = std::max(1, kPagedWorkgroups / d->HKV);
    const PagedBounds b = paged_bounds(d, p.M, p.target);
    p.notes = b.notes;
    p.join = d->groups > 0 || (int64_t)d->table_width * d->page_size > kMinChunk;
    p.slots = p.join ? b.slots : b.notes;
    const size_t rows_all = (size_t)p.slots * d->HKV * p.M;
    p.ml_at = p.join ? rows_all * d->D * sizeof(float) : 0;
    p.notes_at = p.ml_at + (p.join ? rows_all * sizeof(float2) : 0);
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
    if (p.join) {
        const int per = c.HQ * (D / 4);
        hipLaunchKernelGGL((paged_attn_bf16_join<D>), dim3(c.T, (per + 255) / 256), dim3(256), 0, st, c, a, p.M, f8);
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
                         p.slots,
                         reinterpret_cast<float*>(ws),
                         reinterpret_cast<float2*>(ws + p.ml_at),
                         reinterpret_cast<int2*>(ws + p.notes_at)};
    const bool f8 = kv->kv_dtype == BZ_KV_E4M3;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: launch_attn<64>(c, a, p, f8, st); break;
        case 128: launch_attn<128>(c, a, p, f8, st); break;
        default: launch_attn<256>(c, a, p, f8, st); break;
    }
    return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}
