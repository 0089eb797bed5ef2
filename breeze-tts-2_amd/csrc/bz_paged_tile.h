// Attention over a paged cache for many rows (prompts, a shared prefix's rows): one
// workgroup of four waves per slot and key/value head, 64 keys at a time staged in
// LDS for all waves.
//
// Bound by the matrix cores, and by the softmax beside them.  WR waves have 32 rows each
// (WR = 4: 128 rows, every wave takes all 64 keys; WR = 2: 64 rows, a wave takes
// 32 of them, and the two parts of a row are merged at the end).
//   scores  transposed, A = 32 keys from LDS, B = 32 rows in registers
//           (v_mfma_f32_32x32x16_bf16): lane (row, half) gets keys 8 (r / 4) + 4 half + r % 4,
//           so a row's maximum and sum are its own 16 or 32 numbers and one swap of the
//           wave's halves
//   p v     A = the values transposed, by transposing LDS reads
//           (ds_read_b64_tr_b16: 4 keys of one column to a lane), in the order of keys in
//           which the lane has its probabilities: these are the B operand as they
//           are.  p is rounded to bf16 (2^-9 of it on average, as much as the output's own
//           rounding; a second part would double these products); the sum l is over p
//           before it is rounded
//   rescale only when a maximum grows by more than 2^8: until then p stays below
//           2^8, which costs fp32 sums nothing
//   LDS     two buffers, one barrier a tile; 16-byte pieces of a row are exchanged
//           so that neither the row-wise reads of keys nor the transposing ones of values
//           meet on a bank
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

// One 16-key piece of keys or values on its way to LDS.
template <int D, bool F8>
struct TileStage {
    static constexpr int ROW = D * (F8 ? 1 : 2);   // bytes of a position
    static constexpr int LR = ROW / 16;            // lanes of a row
    static constexpr int N = 16 * ROW / 1024;      // loads of a wave
    u32x4 w[N];

    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t pos, int lane) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            w[i] = buffer_ld16(r, (uint32_t)(i * (64 / LR) + lane / LR) * pos + 16 * (lane % LR));
    }
    // rows key0 .. key0 + 15 of a tile of bf16 rows, piece p of row key at p ^ swap(key)
    template <typename X>
    __device__ __forceinline__ void store(char* tile, int key0, int lane, X swap) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int key = key0 + i * (64 / LR) + lane / LR, p = lane % LR;
            char* row = tile + key * (2 * D);
            if constexpr (F8) {
                *reinterpret_cast<u32x4*>(row + 16 * ((2 * p) ^ swap(key))) = f8_widen(w[i][0], w[i][1]);
                *reinterpret_cast<u32x4*>(row + 16 * ((2 * p + 1) ^ swap(key))) = f8_widen(w[i][2], w[i][3]);
            } else {
                *reinterpret_cast<u32x4*>(row + 16 * (p ^ swap(key))) = w[i];
            }
        }
    }
    // bf16 straight into LDS, 16 bytes a lane one after the other: lane l writes piece
    // l % LR of its row, so it reads the piece that belongs there.  A load's rows are in
    // its scalar offset; a lane's offsets differ between loads only by the exchange of
    // pieces, which repeats.
    template <typename X>
    __device__ __forceinline__ static void load_lds(__amdgpu_buffer_rsrc_t r, uint32_t pos, char* tile, int key0, int lane,
                                                    X swap) {
        constexpr int rows = 64 / LR;
#pragma unroll
        for (int i = 0; i < N; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                r, (__attribute__((address_space(3))) void*)(tile + (key0 + i * rows) * (2 * D)), 16,
                (uint32_t)(lane / LR) * pos + 16 * ((lane % LR) ^ swap(i * rows + lane / LR)), i * rows * pos, 0, 0);
    }
    __device__ __forceinline__ bool odd() const {
        bool o = false;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o |= F8 ? nan_f8x4(w[i][e]) : not_finite2(w[i][e]);
        return o;
    }
};

template <int D, bool F8, int WR>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) paged_attn_bf16_tile(PagedKv c, PagedAttn a) {
    constexpr int WK = 4 / WR, M = 32 * WR, T = D / 16, ND = D / 32;
    constexpr int KB = 2 / WK, GB = D == 256 ? 1 : KB;  // 32-key blocks of a wave, and at a time
    constexpr int kTileBytes = kTileKeys * D * 2;
    constexpr int kMerge = WK > 1 ? WR * 32 * (D + 4) * 4 : 0;
    __shared__ __attribute__((aligned(16))) char lds[4 * kTileBytes > kMerge ? 4 * kTileBytes : kMerge];
    __shared__ int odd[2][4];
    __shared__ float st_m[WK][M], st_l[WK][M];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wk = wave / WR;
    const int slot = blockIdx.x / c.HKV, head = blockIdx.x - slot * c.HKV;

    PagedWork w;
    if (!paged_work(c, a, M, slot, lane, w)) return;
    const PagedSlot& u = w.u;
    const PagedSeg& g = u.seg;

    // the lane's row (behind the tile's rows, its last one again)
    const int mine = u.tile * M + min(32 * wr + col, w.rows - 1);
    const int row = mine / c.G, qh = head * c.G + (mine - row * c.G);
    const int limit = row_limit(g, w.kv_len, w.own, row);
    u32x4 q[T];
    {
        const uint16_t* p = a.q + (int64_t)(g.first + row) * a.ld_q + (int64_t)qh * D + 8 * half;
#pragma unroll
        for (int t = 0; t < T; ++t) q[t] = ldg16(p + 16 * t);
    }
    const int32_t* table = w.own ? c.table + (int64_t)g.seq * c.ld_table
                                 : c.prefix_table + (int64_t)(g.seq - c.B) * c.ld_prefix;
    const char* kh = c.k + head * c.k_head;
    const char* vh = c.v + head * c.v_head;
    const float sc = a.scale * kPagedLog2e * (F8 ? c.k_scale[head] : 1.0f);

    pg_f32x16 acc[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t) acc[t] = pg_f32x16{};
    float m = -INFINITY, l = 0.0f;
    bool seen = false, apart = false;

    // pages of the next 16 tiles' pieces, one to a lane
    int pages = -1, page_tile = -16;
    auto refresh = [&](int tile) {
        if (tile < page_tile + 16) return;
        page_tile = tile;
        const int at = w.begin + kTileKeys * tile + 16 * lane;
        pages = at < w.end ? table[at >> c.shift] : -1;
    };
    auto page_of = [&](int tile, int piece) { return __builtin_amdgcn_readlane(pages, 4 * (tile - page_tile) + piece); };
    const int tiles = (max(w.end - w.begin, 0) + kTileKeys - 1) / kTileKeys;
    auto k_swap = [](int key) { return key & 7; };
    auto v_swap = [](int key) { return 2 * (key & 3); };

    TileStage<D, F8> sk, sv;  // (e4m3: on its way through registers, where it is widened)
    uint32_t n_next = 0;      // positions there of a tile's four pieces, a byte each
    auto fetch = [&](int tile, char* kt) {
        refresh(tile);
        const int at = w.begin + kTileKeys * tile;
        n_next = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p)
            n_next |= (unsigned)page_of(tile, p) < (unsigned)c.num_pages
                          ? (uint32_t)min(max(w.end - at - 16 * p, 0), 16) << (8 * p)
                          : 0u;
        const PagedPiece pc = paged_piece<TileStage<D, F8>::ROW>(c, kh, vh, page_of(tile, wave), at + 16 * wave, w.end);
        if constexpr (F8) {
            sk.load(pc.k, (uint32_t)c.k_pos, lane);
            sv.load(pc.v, (uint32_t)c.v_pos, lane);
        } else {
            sk.load_lds(pc.k, (uint32_t)c.k_pos, kt, 16 * wave, lane, k_swap);
            sv.load_lds(pc.v, (uint32_t)c.v_pos, kt + kTileBytes, 16 * wave, lane, v_swap);
        }
    };
    if (tiles > 0) fetch(0, lds);

    // where this lane reads: its key's pieces 2 t + half (t of 0..3, then 8 pieces on), and its columns of keys
    // 4 half + 0..3 (of an even and an odd block of 32 columns, then 8 pieces on)
    uint32_t k_at[4], v_at[2];
    {
#pragma unroll
        for (int t = 0; t < 4; ++t) k_at[t] = col * (2 * D) + 16 * ((2 * t + half) ^ k_swap(col));
        const int i16 = lane & 15, key = 4 * half + (i16 >> 2), piece = 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1);
#pragma unroll
        for (int t = 0; t < 2; ++t) v_at[t] = key * (2 * D) + 8 * (i16 & 1) + 16 * ((4 * t + piece) ^ v_swap(key));
    }

    for (int tile = 0; tile < tiles; ++tile) {
        const int at = w.begin + kTileKeys * tile;
        char* kt = lds + (tile & 1) * (2 * kTileBytes);
        char* vt = kt + kTileBytes;
        const uint32_t n_now = n_next;
        const bool mask = at + kTileKeys > w.all || n_now != 0x10101010u;
        const bool differ = mask && w.all < w.end;  // (behind all rows' limits there are zeros)
        const int own_n = n_now >> (8 * wave) & 0xFF;
        if constexpr (F8) {
            sk.store(kt, 16 * wave, lane, k_swap);
            sv.store(vt, 16 * wave, lane, v_swap);
            if (differ) {
                const bool o = __ballot(sv.odd()) != 0;
                if (lane == 0) odd[tile & 1][wave] = o;
            }
        } else {
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's pieces are in LDS
            if (mask) {
                // places that are not there, as zeros; the other values looked at
                bool o = false;
                for (int i = lane; i < 16 * D / 8; i += 64) {
                    u32x4* x = reinterpret_cast<u32x4*>(vt + 16 * wave * (2 * D)) + i;
                    if (i / (D / 8) >= own_n) {
                        *x = u32x4{0u, 0u, 0u, 0u};
                    } else if (differ) {
                        const u32x4 y = *x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o |= not_finite2(y[e]);
                    }
                }
                o = __ballot(o) != 0;
                if (lane == 0) odd[tile & 1][wave] = o;
            }
        }
        if constexpr (F8)
            if (tile + 1 < tiles) fetch(tile + 1, nullptr);
        __syncthreads();
        if (differ) {
            apart = __builtin_amdgcn_readfirstlane(odd[tile & 1][0] | odd[tile & 1][1] | odd[tile & 1][2] | odd[tile & 1][3]);
            if (apart) break;
        }
        // (the other buffer: every wave is done with its last tile)
        if constexpr (!F8)
            if (tile + 1 < tiles) fetch(tile + 1, lds + (~tile & 1) * (2 * kTileBytes));

#pragma unroll 1
        for (int b0 = KB * wk; b0 < KB * (wk + 1); b0 += GB) {  // 32-key blocks
            pg_f32x16 s[GB];
#pragma unroll
            for (int b = 0; b < GB; ++b) {
                s[b] = pg_f32x16{};
                const char* kr = kt + 32 * (b0 + b) * (2 * D);
#pragma unroll
                for (int t = 0; t < T; ++t)
                    s[b] = pg_mfma32(*reinterpret_cast<const u32x4*>(kr + k_at[t & 3] + 128 * (t >> 2)), q[t], s[b]);
            }
            if (mask) {
#pragma unroll
                for (int b = 0; b < GB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int in = 8 * (r / 4) + 4 * half + r % 4, p = 2 * (b0 + b) + r / 8;
                        const bool ok = at + 32 * (b0 + b) + in < limit && (in & 15) < (int)(n_now >> (8 * p) & 0xFF);
                        s[b][r] = ok ? s[b][r] : -INFINITY;
                        seen |= ok;
                    }
            } else {
                seen = true;
            }
            float mx = s[0][0];
#pragma unroll
            for (int b = 0; b < GB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
            mx = other_half_max(mx) * sc;
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
            const float ms = m == -INFINITY ? 0.0f : m;
            uint32_t pb[GB][8];
#pragma unroll
            for (int b = 0; b < GB; ++b)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float p0 = pg_exp2(fmaf(s[b][r], sc, -ms)), p1 = pg_exp2(fmaf(s[b][r + 1], sc, -ms));
                    l += p0 + p1;
                    pb[b][r / 2] = pack_bf16x2(p0, p1);
                }

#pragma unroll
            for (int b = 0; b < GB; ++b)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const u32x4 pj = {pb[b][4 * j], pb[b][4 * j + 1], pb[b][4 * j + 2], pb[b][4 * j + 3]};
                    const char* vr = vt + (32 * (b0 + b) + 16 * j) * (2 * D);
#pragma unroll
                    for (int t = 0; t < ND; ++t) {
                        const char* x = vr + v_at[t & 1] + 128 * (t >> 1);
                        const uint2 lo = lds_column4(x), hi = lds_column4(x + 8 * (2 * D));
                        acc[t] = pg_mfma32(u32x4{lo.x, lo.y, hi.x, hi.y}, pj, acc[t]);
                    }
                }
        }
    }
    if (u.split == 0 && head == 0 && tid == 0) a.notes[tile_note(c, g, u.tile, M)] = make_int2(slot, u.chunk);
    if (apart) {
        paged_rows_apart<D, F8>(c, a, w, slot, head, M, wave, 4, lane);
        return;
    }

    l = other_half_sum(l);
    const bool any = __builtin_amdgcn_ballot_w64(seen) >> col & 0x100000001ull;
    if (m == -INFINITY) l = any ? 1.0f : 0.0f;
    if constexpr (WK > 1) {
        // the second wave's part of each row to the first
        __syncthreads();
        float* st = reinterpret_cast<float*>(lds) + (wr * 32 + col) * (D + 4) + 4 * half;
        if (wk > 0) {
            if (half == 0) {
                st_m[0][32 * wr + col] = m;
                st_l[0][32 * wr + col] = l;
            }
#pragma unroll
            for (int t = 0; t < ND; ++t)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<float4*>(st + 32 * t + 2 * r) =
                        make_float4(acc[t][r], acc[t][r + 1], acc[t][r + 2], acc[t][r + 3]);
        }
        __syncthreads();
        if (wk > 0) return;
        const float m1 = st_m[0][32 * wr + col], l1 = st_l[0][32 * wr + col], mn = fmaxf(m, m1);
        const float f0 = mn == -INFINITY ? 1.0f : pg_exp2(m - mn), f1 = mn == -INFINITY ? 1.0f : pg_exp2(m1 - mn);
        m = mn;
        l = l * f0 + l1 * f1;
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const float4 x = *reinterpret_cast<const float4*>(st + 32 * t + 2 * r);
                acc[t][r] = acc[t][r] * f0 + x.x * f1;
                acc[t][r + 1] = acc[t][r + 1] * f0 + x.y * f1;
                acc[t][r + 2] = acc[t][r + 2] * f0 + x.z * f1;
                acc[t][r + 3] = acc[t][r + 3] * f0 + x.w * f1;
            }
    }

    const bool whole = w.parts == 1 && c.groups == 0;  // no other slot has keys of these rows
    if (32 * wr + col >= w.rows) return;
    const PagedParts parts(a, c, slot, head, M, D);
    const int rr = 32 * wr + col;
    const float f = m == -INFINITY ? (l > 0.0f ? __builtin_nanf("") : 0.0f) : 1.0f / l * (F8 ? c.v_scale[head] : 1.0f);
    uint16_t* o = a.out + (int64_t)(g.first + row) * a.ld_out + (int64_t)qh * D + 4 * half;
    if (!whole && half == 0) parts.put_ml(rr, m, l);
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            if (whole)
                *reinterpret_cast<uint2*>(o + 32 * t + 2 * r) =
                    make_uint2(pack_bf16x2(acc[t][r] * f, acc[t][r + 1] * f), pack_bf16x2(acc[t][r + 2] * f, acc[t][r + 3] * f));
            else
                parts.put4(rr * D + 4 * half + 32 * t + 2 * r, acc[t][r], acc[t][r + 1], acc[t][r + 2], acc[t][r + 3]);
        }
}

}  // namespace bz
