// Attention over a paged key/value cache: parameters and the kernels' common parts.
//
//   s_j = scale q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max_j s_j
//
// over the keys a row attends, in one pass: with m the maximum so far, the sum l
// and the accumulator are rescaled by e^(m_old - m) as m grows, in exponents of
// 2 of scale log2(e) s and in fp32.  A row of which a slot holds no key has m = -inf
// there; l is then 1 if it attends keys of it, all with a score of -inf (if that
// holds for all its keys the softmax is 0 / 0: NaN), and 0 if it attends none.
#pragma once

#include "bz_paged_plan.h"

namespace bz {

typedef __bf16 pg_bf16x8 __attribute__((ext_vector_type(8)));
typedef float pg_f32x4 __attribute__((ext_vector_type(4)));

constexpr float kPagedLog2e = 1.4426950408889634f;

// D = A B + C, 16x16x32: A[i][k] in lane i + 16 (k/8) element k%8, B[k][j] in
// lane j + 16 (k/8) element k%8, D[i][j] in lane j + 16 (i/4) element i%4.
__device__ __forceinline__ pg_f32x4 pg_mfma16(u32x4 a, u32x4 b, pg_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf16x8, a), __builtin_bit_cast(pg_bf16x8, b), c,
                                                  0, 0, 0);
}

typedef float pg_f32x16 __attribute__((ext_vector_type(16)));

// D = A B + C, 32x32x16: A[i][k] in lane i + 32 (k/8) element k%8, B[k][j] in
// lane j + 32 (k/8) element k%8, D[i][j] in lane j + 32 ((i/4)%2) element
// 4 (i/8) + i%4.
__device__ __forceinline__ pg_f32x16 pg_mfma32(u32x4 a, u32x4 b, pg_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pg_bf16x8, a), __builtin_bit_cast(pg_bf16x8, b), c,
                                                  0, 0, 0);
}

// 2^x with the hardware instruction alone (below 2^-126 it gives zero).
__device__ __forceinline__ float pg_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// The parts of one launch's slots, to be joined.
struct PagedPartsAt {
    float* part;          // [slots][HKV][M][D] accumulators
    float2* ml;           // [slots][HKV][M] (m, l)
    uint64_t* notes;      // [..][HKV] first slot | keys of a chunk << 32, of a sequence's tile
    uint64_t* prefix_notes;  // and of a prefix's
};

struct PagedAttn {
    const uint16_t* q;
    int64_t ld_q;
    float scale;
    uint16_t* out;
    int64_t ld_out;
    PagedCut cut;
    PagedPartsAt to;
    // [notes][HKV], then [prefix notes][HKV]: arrivals of the parts that are joined together, zero
    // between calls; the last to arrive joins them.  NULL: a launch of its own does.
    unsigned* arrived;
    int own_notes;
    int slots;
};

// The position behind the last key that a row attends in its segment: row i of n of a
// sequence is position kv_len - n + i; of a shared prefix every row attends all.
__device__ __forceinline__ int row_limit(const PagedSeg& g, int kv_len, bool own, int row) {
    return own ? min(max(kv_len - g.rows + row + 1, 0), g.keys) : g.keys;
}

__device__ __forceinline__ int parts_of(int keys, int chunk) {
    return max(1, (int)(((unsigned)keys + chunk - 1) / (unsigned)chunk));
}

// A workgroup's part of the work: a slot with the keys of its chunk that its rows attend.
struct PagedWork {
    PagedSlot u;
    bool own;     // a sequence's own positions, not a shared prefix
    int kv_len;
    int rows;     // query rows of the tile, head by head
    int begin, end;  // keys of the chunk that a row of the tile attends
    int all;      // the keys before it are attended by all rows
    int parts;    // chunks that have keys of the tile (or one that has none)
};
__device__ __forceinline__ bool paged_work(const PagedKv& c, const PagedAttn& a, int M, int slot, int lane, PagedWork& w) {
    w.u = paged_slot(c, a.cut, slot, lane);
    if (!w.u.any) return false;
    const PagedSeg& g = w.u.seg;
    w.own = g.seq < c.B;
    w.kv_len = w.own ? max(c.kv_lens[g.seq], 0) : 0;
    const int first = w.u.tile * M;
    w.rows = min(g.rows * c.G - first, M);
    const int tile_end = row_limit(g, w.kv_len, w.own, (first + w.rows - 1) / c.G);
    w.parts = parts_of(tile_end, w.u.chunk);
    w.begin = w.u.split * w.u.chunk;
    w.end = min(w.begin + w.u.chunk, tile_end);
    w.all = row_limit(g, w.kv_len, w.own, first / c.G);
    return w.u.split < w.parts;
}
// The tile's first slot, noted by the workgroup that has it.
__device__ __forceinline__ void note_tile(const PagedKv& c, const PagedAttn& a, const PagedWork& w, int M, int slot, int head) {
    uint64_t* to = (w.own ? a.to.notes : a.to.prefix_notes) + (int64_t)tile_note(c, w.u.seg, w.u.tile, M) * c.HKV + head;
    __hip_atomic_store(to, (uint64_t)(unsigned)w.u.chunk << 32 | (unsigned)slot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The factor of a head's scores, in exponents of 2, where they come from matrix products.  A masked
// score is -inf before it is multiplied and the maximum is taken of the products, so the factor is positive:
// an e4m3 head's scale gives its sign to the queries (exact), and a scale of 0, or a product that
// underflows, becomes the smallest number there is (2^-149: scores below 2^128 stay below 2^-21, and
// e^0 within that).  A scale that is NaN makes the queries NaN, so that masked scores stay -inf.
struct ScoreFactor {
    float f;
    uint32_t keep, flip;  // of two queries' bits
    __device__ __forceinline__ bool plain() const { return keep == ~0u && flip == 0u; }
    __device__ __forceinline__ u32x4 query(u32x4 q) const { return (q & keep) ^ flip; }
};
template <bool F8>
__device__ __forceinline__ ScoreFactor score_factor(const PagedKv& c, const PagedAttn& a, int head) {
    ScoreFactor s = {a.scale * kPagedLog2e, ~0u, 0u};
    if constexpr (F8) {
        const float ks = c.k_scale[head], f = s.f * fabsf(ks);
        s.f = f > 0.0f ? f : 0x1p-149f;
        if (ks < 0.0f) s.flip = 0x80008000u;
        if (ks != ks) s.keep = 0u, s.flip = 0x7FC07FC0u;
    }
    return s;
}

// One 16-position piece of a segment's keys, none of whose rows is read beyond `n`.
struct PagedPiece {
    __amdgpu_buffer_rsrc_t k, v;
    int n;  // positions that are there, from the first
};
// `page` is wave-uniform; `at` the piece's first position, `end` the segment's.
template <int ROW>  // bytes of a position
__device__ __forceinline__ PagedPiece paged_piece(const PagedKv& c, const char* kh, const char* vh, int page, int at,
                                                  int end) {
    PagedPiece p;
    p.n = (unsigned)page < (unsigned)c.num_pages ? min(max(end - at, 0), 16) : 0;
    const int64_t in_page = at & ((1 << c.shift) - 1);
    const int64_t pg = p.n > 0 ? page : 0;
    const uint32_t kb = p.n > 0 ? (uint32_t)((p.n - 1) * (int)c.k_pos + ROW) : 0u;
    const uint32_t vb = p.n > 0 ? (uint32_t)((p.n - 1) * (int)c.v_pos + ROW) : 0u;
    p.k = buffer_rsrc(kh + pg * c.k_page + in_page * c.k_pos, kb);
    p.v = buffer_rsrc(vh + pg * c.v_page + in_page * c.v_pos, vb);
    return p;
}

// Eight e4m3 codes as bf16 (exact).
__device__ __forceinline__ u32x4 f8_widen(uint32_t lo, uint32_t hi) {
    return u32x4{fp8x2_bf16<false>(lo), fp8x2_bf16<true>(lo), fp8x2_bf16<false>(hi), fp8x2_bf16<true>(hi)};
}

// Whether one of two bf16 is infinite or NaN.
__device__ __forceinline__ bool not_finite2(uint32_t w) {
    return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}
// Whether one of four e4m3 codes is NaN (they have no infinities).
__device__ __forceinline__ bool nan_f8x4(uint32_t w) { return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0; }

// The parts that one workgroup leaves: [M][D] accumulators and [M] (m, l).  Where the
// last workgroup of a tile joins them they are stored to the point at which all XCDs meet
// (as agent-scope atomics are); for a launch of its own the end of this one does that.
struct PagedParts {
    __amdgpu_buffer_rsrc_t acc, ml;
    bool agent;
    __device__ __forceinline__ PagedParts(const PagedAttn& a, const PagedKv& c, int slot, int head, int M, int D) {
        const int64_t at = ((int64_t)slot * c.HKV + head) * M;
        acc = buffer_rsrc(a.to.part + at * D, (uint32_t)(M * D) * 4u);
        ml = buffer_rsrc(a.to.ml + at, (uint32_t)M * 8u);
        agent = a.arrived != nullptr;
    }
    __device__ __forceinline__ void put(int i, float v) const {
        if (agent)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), acc, i * 4, 0, kCpolAgent);
        else
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), acc, i * 4, 0, 0);
    }
    __device__ __forceinline__ void put4(int i, float x, float y, float z, float w) const {
        const u32x4 v = {__float_as_uint(x), __float_as_uint(y), __float_as_uint(z), __float_as_uint(w)};
        if (agent)
            __builtin_amdgcn_raw_buffer_store_b128(v, acc, i * 4, 0, kCpolAgent);
        else
            __builtin_amdgcn_raw_buffer_store_b128(v, acc, i * 4, 0, 0);
    }
    // (of another workgroup)
    __device__ __forceinline__ u32x4 get4(int i) const {
        return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(acc, i * 4, 0, kCpolAgent));
    }
    __device__ __forceinline__ float get_m(int r) const {
        return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ml, r * 8, 0, kCpolAgent));
    }
    __device__ __forceinline__ float get_l(int r) const {
        return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ml, r * 8 + 4, 0, kCpolAgent));
    }
    __device__ __forceinline__ void put_ml(int r, float m, float l) const {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 v = {__float_as_uint(m), __float_as_uint(l)};
        if (agent)
            __builtin_amdgcn_raw_buffer_store_b64(v, ml, r * 8, 0, kCpolAgent);
        else
            __builtin_amdgcn_raw_buffer_store_b64(v, ml, r * 8, 0, 0);
    }
};

// A row's sums of four columns, joined from parts.
struct PagedSum {
    float m = -INFINITY, l = 0.0f, o[4] = {};
    // factors that bring a part with maximum x, and this sum, to the larger maximum
    __device__ __forceinline__ void add(float mx, float lx, float4 v) {
        const float mn = fmaxf(m, mx);
        const float f = mn == -INFINITY ? 1.0f : pg_exp2(m - mn), g = mn == -INFINITY ? 1.0f : pg_exp2(mx - mn);
        m = mn;
        l = l * f + lx * g;
        o[0] = o[0] * f + v.x * g;
        o[1] = o[1] * f + v.y * g;
        o[2] = o[2] * f + v.z * g;
        o[3] = o[3] * f + v.w * g;
    }
    // U parts: s, s + stride, .. (behind n the last again, not added)
    template <bool AGENT, int U>
    __device__ __forceinline__ void add_batch(const PagedPartsAt& a, int64_t at, int64_t step, int n, int s, int stride, int D,
                                              int d) {
        float2 x[U];
        float4 v[U];
#pragma unroll
        for (int e = 0; e < U; ++e) {
            const int64_t i = at + min(s + e * stride, n - 1) * step;
            if constexpr (AGENT) {
                const uint64_t w = __hip_atomic_load(reinterpret_cast<const uint64_t*>(a.ml + i), __ATOMIC_RELAXED,
                                                     __HIP_MEMORY_SCOPE_AGENT);
                x[e] = make_float2(__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32)));
                const uint64_t* p = reinterpret_cast<const uint64_t*>(a.part + i * D + d);
                const uint64_t w0 = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const uint64_t w1 = __hip_atomic_load(p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                v[e] = make_float4(__uint_as_float((uint32_t)w0), __uint_as_float((uint32_t)(w0 >> 32)),
                                   __uint_as_float((uint32_t)w1), __uint_as_float((uint32_t)(w1 >> 32)));
            } else {
                x[e] = a.ml[i];
                v[e] = *reinterpret_cast<const float4*>(a.part + i * D + d);
            }
        }
#pragma unroll
        for (int e = 0; e < U; ++e)
            if (s + e * stride < n) add(x[e].x, x[e].y, v[e]);
    }
    // parts first, first + stride, .. of n; part i is the row at + i step of [M] rows.  As many
    // under way at a time as are left, up to 16: a round trip to the parts takes about 2 us.
    template <bool AGENT>
    __device__ __forceinline__ void add_parts(const PagedPartsAt& a, int64_t at, int64_t step, int n, int first, int stride,
                                              int D, int d) {
        for (int s = first; s < n;) {
            if (n - s > 8 * stride) {
                add_batch<AGENT, 16>(a, at, step, n, s, stride, D, d);
                s += 16 * stride;
            } else if (n - s > 2 * stride) {
                add_batch<AGENT, 8>(a, at, step, n, s, stride, D, d);
                s += 8 * stride;
            } else {
                add_batch<AGENT, 2>(a, at, step, n, s, stride, D, d);
                s += 2 * stride;
            }
        }
    }
    // sums of P threads, `apart` threads from each other, into the first's, through LDS [256][8]
    __device__ __forceinline__ void across(float (*st)[8], int tid, int P, int apart, bool lead) {
        if (P == 1) return;
        float* s = st[tid];
        s[0] = o[0], s[1] = o[1], s[2] = o[2], s[3] = o[3], s[4] = m, s[5] = l;
        __syncthreads();
        if (lead)
            for (int p = 1; p < P; ++p) {
                const float* x = st[tid + p * apart];
                add(x[4], x[5], make_float4(x[0], x[1], x[2], x[3]));
            }
    }
    __device__ __forceinline__ void store(uint16_t* p, float vs) const {
        const float f = m == -INFINITY ? (l > 0.0f ? __builtin_nanf("") : 0.0f) : 1.0f / l * vs;
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(o[0] * f, o[1] * f), pack_bf16x2(o[2] * f, o[3] * f));
    }
};

// The last of the workgroups (256 threads) whose parts belong together joins them; all have
// been stored.  These are a tile's parts, or, with prefixes (one row each, M a multiple of G),
// those of a prefix's tile and of all the sequences whose rows are in it (eight sequences behind
// two prefixes, 16 / 8 heads of 128: 16.0 us a call with a launch for it, 12.3 so).
// st: LDS of 256 rows of 8.
template <int D, bool F8>
__device__ __forceinline__ void paged_join_last(const PagedKv& c, const PagedAttn& a, const PagedWork& w, int head, int M,
                                                int tid, int lane, float (*st)[8], int* last) {
    const PagedSeg& g = w.u.seg;
    const int chunk = w.u.chunk;
    int pre = -1, first = g.first, rows = w.rows, tile = w.u.tile, parts = w.parts, at = tile_note(c, g, tile, M);
    if (c.groups > 0) {
        pre = w.own ? prefix_of_seq(c, g.seq, lane) : g.seq - c.B;
        if (pre >= 0) {
            const PagedSeg p = paged_seg(c, c.B + pre);
            const int per = M / c.G;
            if (w.own) tile = (g.first - p.first) / per;
            first = p.first + tile * per;
            const int n = min(p.rows - tile * per, per);
            const int own = lane < n ? parts_of(paged_seg(c, first + lane).keys, chunk) : 0;
            rows = n * c.G;
            parts = parts_of(p.keys, chunk);
            at = a.own_notes + tile_note(c, p, tile, M);
            const int all = parts + __builtin_amdgcn_readlane(wave_scan(own), 63);
            if (tid == 0) *last = all;
        }
    }
    if (pre < 0 && tid == 0) *last = parts;
    // every thread's stores have arrived before the workgroup counts itself in
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    unsigned* count = a.arrived + (int64_t)at * c.HKV + head;
    if (tid == 0)
        *last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)*last - 1u;
    __syncthreads();
    if (!*last) return;
    if (tid == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const float vs = F8 ? c.v_scale[head] : 1.0f;
    auto noted = [&](const uint64_t* notes, int i) {
        const uint64_t n = __hip_atomic_load(notes + (int64_t)i * c.HKV + head, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return ((int64_t)(uint32_t)n * c.HKV + head) * M;
    };
    const int64_t step = (int64_t)c.HKV * M;
    const int64_t at0 = pre < 0 ? ((int64_t)w.u.first_slot * c.HKV + head) * M
                                : noted(a.to.prefix_notes, at - a.own_notes);
    const int items = rows * (D / 4);
    // few items: several threads to each, taking parts in turn
    int P = 1;
    while (2 * P * items <= 256 && P < parts) P *= 2;
    for (int i0 = 0; i0 < items; i0 += 256) {
        const int p = P > 1 ? tid / items : 0, i = i0 + tid - p * items;
        PagedSum sum;
        const bool on = P > 1 ? p < P : i < items;
        const int r = on ? i / (D / 4) : 0, d = 4 * (i % (D / 4));
        const int k = pre < 0 ? tile * M + r : r, row = k / c.G, h = head * c.G + (k - row * c.G);
        if (on) {
            if (pre >= 0) {
                PagedSeg own = paged_seg(c, first + row);
                sum.add_parts<true>(a.to, noted(a.to.notes, tile_note(c, own, 0, M)) + (k - row * c.G), step,
                                    parts_of(own.keys, chunk), p, P, D, d);
            }
            sum.add_parts<true>(a.to, at0 + r, step, parts, p, P, D, d);
        }
        sum.across(st, tid, P, items, on && p == 0);
        if (on && p == 0) sum.store(a.out + (int64_t)(first + row) * a.ld_out + (int64_t)h * D + d, vs);
    }
}

// The rows of a workgroup's tile one by one, a wave to a row and a key to a lane: for a
// tile in which a value that is not finite belongs to a key that only some of the rows
// attend (0 times it is NaN, so a matrix product would carry it into the others).
// Not fast; such a batch has a broken sequence in it.
// part_at(row, column): where a part has it.
template <int D, bool F8, typename X>
__device__ __forceinline__ void paged_rows_apart(const PagedKv& c, const PagedAttn& a, const PagedWork& w, int slot,
                                                 int head, int M, int wave, int waves, int lane, X part_at) {
    constexpr int DL = D / 64;
    const PagedSeg& g = w.u.seg;
    const int32_t* table = w.own ? c.table + (int64_t)g.seq * c.ld_table
                                 : c.prefix_table + (int64_t)(g.seq - c.B) * c.ld_prefix;
    const float sc = a.scale * kPagedLog2e * (F8 ? c.k_scale[head] : 1.0f), vs = F8 ? c.v_scale[head] : 1.0f;
    const bool whole = w.parts == 1 && c.groups == 0;
    const PagedParts parts(a, c, slot, head, M, D);
    for (int rr = wave; rr < w.rows; rr += waves) {
        const int k = w.u.tile * M + rr, row = k / c.G, h = head * c.G + (k - row * c.G);
        const uint16_t* q = a.q + (int64_t)(g.first + row) * a.ld_q + (int64_t)h * D;
        const int end = min(w.end, row_limit(g, w.kv_len, w.own, row));
        float m = -INFINITY, l = 0.0f, acc[DL] = {};
        bool seen = false;
        for (int j0 = w.begin; j0 < end; j0 += 64) {
            const int j = j0 + lane;
            const int page = j < end ? table[j >> c.shift] : -1;
            const bool there = (unsigned)page < (unsigned)c.num_pages;
            const int at = j & ((1 << c.shift) - 1);
            float s = -INFINITY;
            if (there) {
                const char* kr = c.k + page * c.k_page + head * c.k_head + at * c.k_pos;
                s = 0.0f;
#pragma unroll 4
                for (int d = 0; d < D; ++d)
                    s += bf16_to_f32(q[d]) * (F8 ? __builtin_amdgcn_cvt_f32_fp8((int)reinterpret_cast<const uint8_t*>(kr)[d], 0)
                                                 : bf16_to_f32(reinterpret_cast<const uint16_t*>(kr)[d]));
                s *= sc;
            }
            const float mn = fmaxf(m, wave_max(s)), ms = mn == -INFINITY ? 0.0f : mn;
            const float f = pg_exp2(m - ms), p = there ? pg_exp2(s - ms) : 0.0f;
            m = mn;
            l = l * f + wave_sum(p);
            for (int e = 0; e < DL; ++e) acc[e] *= f;
            uint64_t live = __ballot(there);
            seen |= live != 0;
            for (; live; live &= live - 1) {
                const int i = __builtin_ctzll(live);
                const float pi = __shfl(p, i, 64);
                const int pg = __shfl(page, i, 64), ai = (j0 + i) & ((1 << c.shift) - 1);
                const char* vr = c.v + pg * c.v_page + head * c.v_head + ai * c.v_pos;
                for (int e = 0; e < DL; ++e)
                    acc[e] += pi * (F8 ? __builtin_amdgcn_cvt_f32_fp8((int)reinterpret_cast<const uint8_t*>(vr)[DL * lane + e], 0)
                                       : bf16_to_f32(reinterpret_cast<const uint16_t*>(vr)[DL * lane + e]));
            }
        }
        if (whole) {
            uint16_t* o = a.out + (int64_t)(g.first + row) * a.ld_out + (int64_t)h * D + DL * lane;
            for (int e = 0; e < DL; ++e) o[e] = f32_to_bf16(seen ? acc[e] / l * vs : 0.0f);
        } else {
            for (int e = 0; e < DL; ++e) parts.put(part_at(rr, DL * lane + e), acc[e]);
            if (lane == 0) parts.put_ml(rr, m, m == -INFINITY ? (seen ? 1.0f : 0.0f) : l);
        }
    }
}

}  // namespace bz
