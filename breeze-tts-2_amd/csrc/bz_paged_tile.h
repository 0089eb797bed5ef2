// Attention over a paged cache for many rows (prompts, a shared prefix's rows): one
// workgroup per slot and key/value head, 64 keys at a time staged in LDS for all waves.
//
// Bound by the matrix cores, and by the softmax beside them.  A wave has 32 rows.  With
// D <= 128 it has them for itself; with D = 256 two waves share them (PAIR): each takes the
// scores of 32 of the 64 keys, then each the products with half of the columns over
// all 64, so that its accumulators leave room for two waves on a SIMD.
//   scores  transposed, A = 32 keys from LDS, B = 32 rows in registers
//           (v_mfma_f32_32x32x16_bf16): lane (row, half) gets keys 8 (r / 4) + 4 half + r % 4,
//           so a row's maximum is over its own numbers, one swap of the wave's halves and
//           (PAIR) what the other wave found
//   p v     A = the values transposed, by transposing LDS reads
//           (ds_read_b64_tr_b16: 4 keys of one column to a lane, of e4m3 8 with
//           ds_read_b64_tr_b8), in the order of keys in which the lanes have their
//           probabilities: these are the B operand as they are (PAIR: also the other wave's,
//           through LDS).  p is rounded to bf16 (at most 2^-8 of it, as much as the output's
//           own rounding; a second part would double these products); the sum l is over p
//           before it is rounded.  Whole outputs are then 1.3 to 1.4 times as far from the exact ones
//           as with p in 32 bits (0.0021 .. 0.0023 of their norm, 0.0016 .. 0.0017)
//   rescale only when a maximum grows by more than 2^8: until then p stays below
//           2^8, which costs fp32 sums nothing
//   order   in one round: the softmax of a tile beside the scores of the next one, then
//           its products; keys are fetched three tiles ahead, values one, and one
//           barrier (PAIR: two, the probabilities have one buffer) ends a round's first half
//   e4m3    stays as it is in LDS, which leaves room for a second workgroup on a CU, and is widened
//           by the wave that reads it (one instruction for two values)
//   LDS     16-byte pieces of a row are exchanged so that neither the row-wise reads of
//           keys nor the transposing ones of values meet on a bank.  Every buffer is a
//           variable of its own and the rounds take them in turn by name: that tells the
//           compiler that reads of one do not wait for loads under way into another
//   parts   joined by the tile's last workgroup, or with prefixes by a launch
// Measured: a prompt of 2011 tokens, 16 / 8 heads of 128, 39.5 us, of which 15 are start, first bytes and
// parts and 10 rounds take 2.4 each; chunks of three prompts over up to 8000 positions, 16 / 4
// heads of 256, 305 a call in a series (769 TFLOP/s; 337 traced one by one; without fetches 20% less, without the
// products 23%); 64 rows of one prefix of 6007, 16 / 8 heads of 128, 35.3 with the sequences' own keys; 24 sequences
// of three prefixes of up to 16383, e4m3, 16 / 4 heads of 256, 41.7.
#pragma once

#include "bz_paged_attn.h"

namespace bz {

constexpr int kTileKeys = 64;

typedef short pg_s16x4 __attribute__((ext_vector_type(4)));

// Four keys of one column: lane i of 16 points at key i / 4, columns 4 (i % 4) ..,
// and gets column i of the four keys.
__device__ __forceinline__ uint2 lds_column4(const char* p) {
    const auto v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) pg_s16x4*)(__attribute__((address_space(3))) void*)const_cast<char*>(p));
    return __builtin_bit_cast(uint2, v);
}

// What the other half of the wave has for the same row.
__device__ __forceinline__ float other_half_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Eight keys of one column, e4m3: lane i of 16 points at key i / 2, columns 8 (i % 2) ..,
// and gets column i of the eight keys.
__device__ __forceinline__ u32x4 lds_column8(const char* p) {
    typedef int s32x2 __attribute__((ext_vector_type(2)));
    const auto v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (__attribute__((address_space(3))) s32x2*)(__attribute__((address_space(3))) void*)const_cast<char*>(p));
    return f8_widen((uint32_t)v[0], (uint32_t)v[1]);
}

// A wave's RW rows of a tile's keys or values, straight into LDS.
template <int D, bool F8, int RW>
struct TileStage {
    static constexpr int ROW = D * (F8 ? 1 : 2);  // bytes of a position
    static constexpr int LR = ROW / 16;           // lanes of a row
    static constexpr int ROWS = 64 / LR;          // rows of a load
    static constexpr int N = RW * ROW / 1024;     // loads of a wave
    static_assert(N > 0 && N * 1024 == RW * ROW, "whole loads of a wave");

    // 16 bytes a lane one after the other: lane l writes piece l % LR of its row, so it reads
    // the piece that belongs there, piece p of row key at p ^ swap(key).  A load's rows are in
    // its scalar offset; a lane's offsets differ between loads only by the exchange of
    // pieces, which repeats.
    template <typename X>
    __device__ __forceinline__ static void load(__amdgpu_buffer_rsrc_t r, uint32_t pos, char* tile, int first, int lane,
                                                X swap) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                r, (__attribute__((address_space(3))) void*)(tile + (first + i * ROWS) * ROW), 16,
                (uint32_t)(lane / LR) * pos + 16 * ((lane % LR) ^ swap(first + i * ROWS + lane / LR)), i * ROWS * pos, 0, 0);
    }
};

// Order for the scheduler: N steps of P matrix products, each behind its R LDS reads, with the
// reads of A steps under way.
template <int N, int P, int R, int A>
__device__ __forceinline__ void read_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, R * A, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, P, 0);
        if (i + A < N) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    }
}

template <int D, bool F8, int WAVES, bool PAIR>
__global__ void __launch_bounds__(64 * WAVES, 2) paged_attn_bf16_tile(PagedKv c, PagedAttn a) {
    constexpr int W = PAIR ? 2 : 1;  // waves of a row
    constexpr int M = 32 * WAVES / W, RW = kTileKeys / WAVES, T = D / 16, ND = D / 32 / W, KB = 2 / W;
    constexpr int kAhead = 4;  // LDS reads under way, in steps
    using Stage = TileStage<D, F8, RW>;
    constexpr int ROW = Stage::ROW, kTileBytes = kTileKeys * ROW, kProbs = PAIR ? WAVES * 2048 : 16;
    __shared__ __attribute__((aligned(16))) char k0[kTileBytes], k1[kTileBytes], v0[kTileBytes], v1[kTileBytes];
    __shared__ __attribute__((aligned(16))) char probs[kProbs];
    __shared__ float top0[PAIR ? WAVES : 1][32], top1[PAIR ? WAVES : 1][32];  // a tile's maxima
    __shared__ int odd[2][WAVES];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave / W, kp = wave % W;
    const int slot = blockIdx.x / c.HKV, head = blockIdx.x - slot * c.HKV;

    PagedWork w;
    if (!paged_work(c, a, M, slot, lane, w)) return;
    const PagedSlot& u = w.u;
    const PagedSeg& g = u.seg;

    const bool idle = 32 * rg >= w.rows;
    // the lane's row (behind the tile's rows, its last one again)
    const int mine = u.tile * M + min(32 * rg + col, w.rows - 1);
    const int row = mine / c.G, qh = head * c.G + (mine - row * c.G);
    const int limit = row_limit(g, w.kv_len, w.own, row);
    u32x4 q[T];
    {
        const uint16_t* p = a.q + (int64_t)(g.first + row) * a.ld_q + (int64_t)qh * D;
        // (a lane's 16 bytes of e4m3 keys are those of two products)
#pragma unroll
        for (int t = 0; t < T; ++t) q[t] = ldg16(p + (F8 ? 32 * (t / 2) + 16 * half + 8 * (t % 2) : 16 * t + 8 * half));
    }
    const int32_t* table = w.own ? c.table + (int64_t)g.seq * c.ld_table
                                 : c.prefix_table + (int64_t)(g.seq - c.B) * c.ld_prefix;
    const char* kh = c.k + head * c.k_head;
    const char* vh = c.v + head * c.v_head;
    const ScoreFactor factor = score_factor<F8>(c, a, head);
    const float sc = factor.f;
    if (F8 && !factor.plain())
#pragma unroll
        for (int t = 0; t < T; ++t) q[t] = factor.query(q[t]);

    pg_f32x16 acc[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t) acc[t] = pg_f32x16{};
    float m = -INFINITY, l = 0.0f;
    bool seen = false, apart = false;

    // The next 16 tiles' pieces, one to a lane: where this wave's rows of its keys and values begin,
    // and how many positions are there (of a tile's four, a byte each).  Worked out for 16 tiles at a time: with
    // scalar instructions for each tile they were as many as all vector instructions.
    uint64_t k_from = 0, v_from = 0;
    uint32_t n_of = 0;
    int from_tile = -16;
    const int tiles = (max(w.end - w.begin, 0) + kTileKeys - 1) / kTileKeys;
    // (64 banks: the rows of ROW bytes begin on 256 / ROW places of them.  No conflicts; with 7 and 2 for all D
    // 40% of the LDS cycles were conflicts)
    auto k_swap = [](int key) {
        if (!F8) return key & (D == 64 ? 7 : 15);
        return ROW == 256 ? key & 15 : ROW == 128 ? key >> 1 & 7 : key >> 2 & 3;
    };
    auto v_swap = [](int key) {
        if (!F8) return (D == 64 ? 2 : 4) * (key & 3);
        const int bit3 = key >> 3 & 1;
        return 2 * (ROW == 256 ? (key & 3) + 4 * bit3 : ROW == 128 ? (key >> 1 & 1) + 2 * bit3 : bit3);
    };

    // where this lane reads: its key's pieces 2 t + half (t of 0..7, then 16 pieces on), and its columns of keys
    // 4 half + 0..3 (e4m3: and 8 on) of a block of 32 columns
    constexpr int TK = F8 ? T / 2 : T;  // reads of a key
    uint32_t k_at[TK < 8 ? TK : 8], v_at[ND];
    {
#pragma unroll
        for (int t = 0; t < 8 && t < TK; ++t) k_at[t] = (32 * KB * kp + col) * ROW + 16 * ((2 * t + half) ^ k_swap(col));
        const int i16 = lane & 15, r = F8 ? i16 >> 1 : i16 >> 2;
        const int key = 4 * half + (r & 3) + 8 * (r >> 2);
#pragma unroll
        for (int t = 0; t < ND; ++t) {
            const int block = kp * ND + t, hi = lane >> 4 & 1;
            v_at[t] = F8 ? key * ROW + 8 * (i16 & 1) + 16 * ((2 * block + hi) ^ v_swap(key))
                         : key * ROW + 8 * (i16 & 1) + 16 * ((4 * block + 2 * hi + (i16 >> 1 & 1)) ^ v_swap(key));
        }
    }

    struct Tile {
        uint32_t n;            // positions there
        uint32_t v_lo, v_hi;   // where this wave's rows of the values begin
    };
    auto rows_at = [&](uint32_t lo, uint32_t hi, uint32_t n, uint32_t pos) {
        const int there = (int)(n >> (8 * (RW * wave / 16)) & 0xFF) - RW * wave % 16;
        return buffer_rsrc(reinterpret_cast<const char*>((uint64_t)hi << 32 | lo),
                           there > 0 ? (uint32_t)(min(there, RW) - 1) * pos + Stage::ROW : 0u);
    };
    auto lane_of = [&](uint64_t x, int i, uint32_t& lo, uint32_t& hi) {
        lo = __builtin_amdgcn_readlane((int)(uint32_t)x, i);
        hi = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), i);
    };
    auto fetch_k = [&](int tile, char* to) {
        if (tile >= from_tile + 16) {
            from_tile = tile;
            const int at = w.begin + kTileKeys * tile + 16 * lane;
            const int page = at < w.end ? table[at >> c.shift] : -1;
            const bool there = (unsigned)page < (unsigned)c.num_pages;
            const int in_page = (at & ((1 << c.shift) - 1)) + RW * wave % 16;
            k_from = (uint64_t)kh + (there ? page : 0) * c.k_page + in_page * c.k_pos;
            v_from = (uint64_t)vh + (there ? page : 0) * c.v_page + in_page * c.v_pos;
            uint32_t n = (there ? (uint32_t)min(w.end - at, 16) : 0u) << (8 * (lane & 3));
            n |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)n, kDppXor1, 0xF, 0xF, false);
            n_of = n | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)n, kDppXor2, 0xF, 0xF, false);
        }
        const int first = 4 * (tile - from_tile), own = first + RW * wave / 16;
        Tile x;
        x.n = __builtin_amdgcn_readlane((int)n_of, first);
        lane_of(v_from, own, x.v_lo, x.v_hi);
        uint32_t lo, hi;
        lane_of(k_from, own, lo, hi);
        const __amdgpu_buffer_rsrc_t r = rows_at(lo, hi, x.n, (uint32_t)c.k_pos);
        Stage::load(r, (uint32_t)c.k_pos, to, RW * wave, lane, k_swap);
        return x;
    };
    auto fetch_v = [&](const Tile& x, char* to) {
        const __amdgpu_buffer_rsrc_t r = rows_at(x.v_lo, x.v_hi, x.n, (uint32_t)c.v_pos);
        Stage::load(r, (uint32_t)c.v_pos, to, RW * wave, lane, v_swap);
    };
    // scores of the wave's keys of a tile, masked, and their maximum (PAIR: to the other wave too)
    pg_f32x16 s[KB];
    auto scores = [&](int tile, const Tile& x, const char* kb, float (*top)[32]) {
#pragma unroll
        for (int b = 0; b < KB; ++b) s[b] = pg_f32x16{};
#pragma unroll
        for (int t = 0; t < TK; ++t)
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(kb + k_at[t & 7] + 256 * (t >> 3) + 32 * b * ROW);
                if constexpr (F8) {
                    s[b] = pg_mfma32(f8_widen(x[0], x[1]), q[2 * t], s[b]);
                    s[b] = pg_mfma32(f8_widen(x[2], x[3]), q[2 * t + 1], s[b]);
                } else {
                    s[b] = pg_mfma32(x, q[t], s[b]);
                }
            }
        read_ahead<KB * TK, F8 ? 2 : 1, 1, kAhead>();
        const int at = w.begin + kTileKeys * tile;
        if (at + kTileKeys > w.all || x.n != 0x10101010u) {
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    // key 8 (r / 4) + 4 half + r % 4 of the 32 is attended and there
                    const int there = x.n >> (16 * (KB * kp + b) + 8 * p) & 0xFF;
                    const int bound = min(limit - at - 32 * (KB * kp + b), 16 * p + there) - 4 * half;
                    seen |= 16 * p < bound;
#pragma unroll
                    for (int r = 8 * p; r < 8 * p + 8; ++r) s[b][r] = 8 * (r / 4) + r % 4 < bound ? s[b][r] : -INFINITY;
                }
        } else {
            seen = true;
        }
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
        mx = other_half_max(mx);
        if constexpr (PAIR)
            if (half == 0) top[wave][col] = mx;
        return mx;
    };
    float mx = 0.0f;
    Tile x0 = {}, x1 = {}, x2 = {};

    const bool whole = w.parts == 1 && c.groups == 0;  // no other slot has keys of these rows
    const bool inside = !whole && a.arrived;
    // Where a part has column d of row r.  If this kernel joins it, as the lanes hold it: four columns of 64 lanes
    // one after the other, whole lines past the L2 (row by row, as the joining launch reads them, 32 bytes at
    // a time: a prompt of 2011 tokens, 16 / 8 heads of 128, 49.7 us, and 40.1 so).
    auto part_at = [&](int r, int d) {
        if (!inside) return r * D + d;
        const int wv = r / 32 * W + d / (32 * ND), e = d % 32;
        return (((wv * ND + d / 32 % ND) * 4 + e / 8) * 64 + e / 4 % 2 * 32 + r % 32) * 4 + e % 4;
    };
    // Whether this workgroup is the last of its tile's to come; if not, or not sure of it beforehand, its part is stored.
    auto last_to_arrive = [&](auto store) {
        int* last = &odd[0][0];
        unsigned* count = a.arrived + (int64_t)tile_note(c, g, u.tile, M) * c.HKV + head;
        const unsigned others = (unsigned)w.parts - 1u;
        __syncthreads();
        if (tid == 0)
            *last = !apart && __hip_atomic_load(count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == others;
        __syncthreads();
        if (!__builtin_amdgcn_readfirstlane(*last)) {
            store();
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) *last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == others;
            __syncthreads();
            if (!__builtin_amdgcn_readfirstlane(*last)) return false;
        }
        if (tid == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return true;
    };

    // Up to where all waves' values of the tile (and keys of the one two on) are in LDS.
    auto arrive = [&](int tile, char* vb) __attribute__((always_inline)) {
        const int at = w.begin + kTileKeys * tile;
        const bool mask = at + kTileKeys > w.all || x0.n != 0x10101010u;
        const bool differ = mask && w.all < w.end;  // (behind all rows' limits there are zeros)
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        if (mask) {
            // places that are not there, as zeros; the other values looked at
            const int there = (int)(x0.n >> (8 * (RW * wave / 16)) & 0xFF) - RW * wave % 16;
            bool o = false;
            for (int i = lane; i < RW * Stage::LR; i += 64) {
                u32x4* y = reinterpret_cast<u32x4*>(vb + RW * wave * ROW) + i;
                if (i / Stage::LR >= there) {
                    *y = u32x4{0u, 0u, 0u, 0u};
                } else if (differ) {
                    const u32x4 z = *y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o |= F8 ? nan_f8x4(z[e]) : not_finite2(z[e]);
                }
            }
            o = __ballot(o) != 0;
            if (lane == 0) odd[tile & 1][wave] = o;
        }
        __syncthreads();
        if (differ) {
            int o = 0;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) o |= odd[tile & 1][i];
            apart |= __builtin_amdgcn_readfirstlane(o) != 0;  // (what is summed from here on is not used)
        }
    };
    auto fetch_next = [&](int tile, char* ko, char* vn) __attribute__((always_inline)) {
        // (behind the last tile no page is there: nothing is read)
        fetch_v(x1, vn);
        const Tile x3 = fetch_k(tile + 3, ko);
        return x3;
    };

    // Tile `tile`: its softmax, the next one's scores, its products.  ko: the next one's keys, and later those of
    // three tiles on.
    auto round = [&](int tile, char* ko, char* vb, char* vn, float (*top)[32],
                     float (*top_next)[32]) __attribute__((always_inline)) {
        if constexpr (PAIR) mx = fmaxf(mx, top[wave ^ 1][col]);
        mx *= sc;
        const bool grow = mx > m + 8.0f;
        if (__ballot(grow)) {
            const float mn = grow ? mx : m;
            const float f = mn == -INFINITY ? 1.0f : pg_exp2(m - mn);
            l *= f;
#pragma unroll
            for (int t = 0; t < ND; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[t][r] *= f;
            m = mn;
        }
#pragma unroll
        for (int t = 0; t < ND; ++t) asm("" : "+v"(acc[t]));  // (in place: without it both sides of the branch were kept)
        const float ms = m == -INFINITY ? 0.0f : m;
        u32x4 p[KB][2];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float e0 = pg_exp2(fmaf(s[b][r], sc, -ms)), e1 = pg_exp2(fmaf(s[b][r + 1], sc, -ms));
                l += e0 + e1;
                p[b][r / 8][r / 2 % 4] = pack_bf16x2(e0, e1);
            }
        if constexpr (PAIR) {
            char* to = probs + 2048 * wave + 16 * lane;
            *reinterpret_cast<u32x4*>(to) = p[0][0];
            *reinterpret_cast<u32x4*>(to + 1024) = p[0][1];
        }
        mx = scores(tile + 1, x1, ko, top_next);  // (behind the last tile: -inf)

        arrive(tile, vb);
        u32x4 o[2] = {};
        if constexpr (PAIR) {
            const char* from = probs + 2048 * (wave ^ 1) + 16 * lane;
            o[0] = *reinterpret_cast<const u32x4*>(from);
            o[1] = *reinterpret_cast<const u32x4*>(from + 1024);
            __syncthreads();
        }
        const Tile x3 = fetch_next(tile, ko, vn);
#pragma unroll
        for (int b = 0; b < 2; ++b) {  // (PAIR: the wave's own 32 keys, the other's)
            const char* vr = vb + 32 * (PAIR && b ? kp ^ 1 : PAIR ? kp : b) * ROW;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const u32x4 pj = PAIR && b ? o[j] : p[PAIR ? 0 : b][j];
#pragma unroll
                for (int t = 0; t < ND; ++t) {
                    const char* y = vr + 16 * j * ROW + v_at[t];
                    if constexpr (F8) {
                        acc[t] = pg_mfma32(lds_column8(y), pj, acc[t]);
                    } else {
                        const uint2 lo = lds_column4(y), hi = lds_column4(y + 8 * ROW);
                        acc[t] = pg_mfma32(u32x4{lo.x, lo.y, hi.x, hi.y}, pj, acc[t]);
                    }
                }
            }
        }
        read_ahead<4 * ND, 1, F8 ? 1 : 2, kAhead>();
        x0 = x1;
        x1 = x2;
        x2 = x3;
    };
    if (tiles > 0) {
        x0 = fetch_k(0, k0);
        x1 = fetch_k(1, k1);
        fetch_v(x0, v0);
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __syncthreads();
        if (!idle) mx = scores(0, x0, k0, top0);
        __syncthreads();
        x2 = fetch_k(2, k0);
    }
    // A wave without rows (a sequence's few beside a prefix's many) fetches alone, the same as the others.
    if (idle) {
        auto pass = [&](int tile, char* ko, char* vb, char* vn) {
            arrive(tile, vb);
            if constexpr (PAIR) __syncthreads();
            const Tile x3 = fetch_next(tile, ko, vn);
            x0 = x1;
            x1 = x2;
            x2 = x3;
        };
        int tile = 0;
        for (; tile + 1 < tiles; tile += 2) {
            pass(tile, k1, v0, v1);
            pass(tile + 1, k0, v1, v0);
        }
        if (tile < tiles) pass(tile, k1, v0, v1);
        __builtin_amdgcn_s_waitcnt(0x0F70);
        if constexpr (PAIR) {
            __syncthreads();
            __syncthreads();
        }
        if (apart) paged_rows_apart<D, F8>(c, a, w, slot, head, M, wave, WAVES, lane, part_at);
        if (inside) last_to_arrive([] {});
        return;
    }
    // (no way out between two rounds: it made the accumulators live twice)
    int tile = 0;
    for (; tile + 1 < tiles; tile += 2) {
        round(tile, k1, v0, v1, top0, top1);
        round(tile + 1, k0, v1, v0, top1, top0);
    }
    if (tile < tiles) round(tile, k1, v0, v1, top0, top1);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // (no load into LDS, empty as the last ones are, outlives the workgroup)
    if (u.split == 0 && tid == 0) note_tile(c, a, w, M, slot, head);

    l = other_half_sum(l);
    const bool any = __builtin_amdgcn_ballot_w64(seen) >> col & 0x100000001ull;
    if (m == -INFINITY) l = any ? 1.0f : 0.0f;
    if constexpr (PAIR) {
        __syncthreads();  // (the maxima have been read)
        if (half == 0) top0[wave][col] = l;
        __syncthreads();
        l += top0[wave ^ 1][col];
    }
    if (apart) paged_rows_apart<D, F8>(c, a, w, slot, head, M, wave, WAVES, lane, part_at);

    const int rr = 32 * rg + col, first = 32 * ND * kp + 4 * half;
    const PagedParts parts(a, c, slot, head, M, D);
    auto store_part = [&] {
        if (apart || rr >= w.rows) return;
        if (half == 0 && kp == 0) parts.put_ml(rr, m, l);
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                parts.put4(inside ? ((wave * ND + t) * 4 + r / 4) * 256 + 4 * lane : rr * D + first + 32 * t + 2 * r,
                           acc[t][r], acc[t][r + 1], acc[t][r + 2], acc[t][r + 3]);
    };
    if (!whole && !inside) {
        store_part();
        return;
    }
    if (inside) {
        if (!last_to_arrive(store_part)) return;
        // all parts in their order, this workgroup's own from its registers: whichever is last, the sums are the same
        float top = apart ? -INFINITY : m;
        for (int i = 0; i < w.parts; i += 4) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = PagedParts(a, c, u.first_slot + min(i + e, w.parts - 1), head, M, D).get_m(rr);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (apart || min(i + e, w.parts - 1) != u.split) top = fmaxf(top, x[e]);
        }
        pg_f32x16 sum[ND];
#pragma unroll
        for (int t = 0; t < ND; ++t) sum[t] = pg_f32x16{};
        float ls = 0.0f;
        for (int i = 0; i < w.parts; ++i) {
            if (!apart && i == u.split) {
                const float f = top == -INFINITY ? 1.0f : pg_exp2(m - top);
                ls = fmaf(l, f, ls);
#pragma unroll
                for (int t = 0; t < ND; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum[t][r] = fmaf(acc[t][r], f, sum[t][r]);
            } else {
                const PagedParts other(a, c, u.first_slot + i, head, M, D);
                u32x4 x[ND][4];
#pragma unroll
                for (int t = 0; t < ND; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[t][r] = other.get4(((wave * ND + t) * 4 + r) * 256 + 4 * lane);
                const float f = top == -INFINITY ? 1.0f : pg_exp2(other.get_m(rr) - top);
                ls = fmaf(other.get_l(rr), f, ls);
#pragma unroll
                for (int t = 0; t < ND; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum[t][r] = fmaf(__uint_as_float(x[t][r / 4][r % 4]), f, sum[t][r]);
            }
        }
        m = top;
        l = ls;
#pragma unroll
        for (int t = 0; t < ND; ++t) acc[t] = sum[t];
    } else if (apart) {
        return;  // (written there)
    }
    if (rr >= w.rows) return;
    const float f = m == -INFINITY ? (l > 0.0f ? __builtin_nanf("") : 0.0f) : 1.0f / l * (F8 ? c.v_scale[head] : 1.0f);
    uint16_t* o = a.out + (int64_t)(g.first + row) * a.ld_out + (int64_t)qh * D + first;
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<uint2*>(o + 32 * t + 2 * r) =
                make_uint2(pack_bf16x2(acc[t][r] * f, acc[t][r + 1] * f), pack_bf16x2(acc[t][r + 2] * f, acc[t][r + 3] * f));
}

}  // namespace bz
