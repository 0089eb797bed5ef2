// Attention over a paged cache for few rows: one workgroup of four waves per
// slot and key/value head, the waves taking 32-key steps of the chunk in turn.
//
// Bound by HBM (decode): a step's keys and values are read once, straight into the
// operands of the matrix cores, the next step's while this one computes.
//   scores  transposed, A = 16 keys, B = 16 rows (v_mfma_f32_16x16x32_bf16, D / 32 of
//           them): lane (row, grp) gets the keys 4 grp .. 4 grp + 3 of each half step
//   p v     A = the values transposed, B = p: the eight probabilities that a lane has
//           are its operand as they are (the contraction runs over the keys in the
//           scores' order), and a value row's 16 bytes are loaded by the lane that needs
//           their columns, so nothing goes through LDS.  p goes in as two bf16 parts,
//           ~16 significant bits; the first is cut, not rounded, so that both are positive
//           and an infinite value gives its infinity
//   waves   merged through LDS at the end, in wave order
//   parts   joined by the last workgroup of those that have them
// Measured, heads of 128 unless said: one token for each of 48 sequences of 40 .. 4095 positions,
// 16 / 8 heads, 85.0 us (4.8 TB/s, 93% of a large copy's rate); four of 30 .. 65 thousand, e4m3, 16 / 4
// heads of 256, 100.7 (4.4 TB/s); five tokens for 16 of 97 .. 2043, 8 / 2 heads, 17.5; one for
// two of 610, 16 / 8 heads, 9.9: the chain of launch, lengths, table, keys, values, store, count
// and join.
#pragma once

#include "bz_paged_attn.h"

namespace bz {

constexpr int kStreamWaves = 4;
constexpr int kStep = 32;  // keys of a step

// Result of an operation over the four 16-lane rows of a wave, in every lane of a column.
template <typename F>
__device__ __forceinline__ float pg_across(float v, F f) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float t = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(t), __float_as_uint(t), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <int D, bool F8>
struct StreamStep {
    static constexpr int ES = F8 ? 1 : 2;
    static constexpr int KL = D * ES / 64;  // 16-byte loads of a key row and lane
    static constexpr int VB = D * ES / 16;  // bytes of a value row and lane
    static constexpr int VW = VB / 4;
    u32x4 k[2][KL];
    uint32_t v[2][4][VW];

    __device__ __forceinline__ void load_k(int h, const PagedPiece& p, uint32_t k_pos, int col, int grp) {
        const uint32_t o = col * k_pos + 16 * grp;
#pragma unroll
        for (int t = 0; t < KL; ++t) k[h][t] = buffer_ld16(p.k, o + 64 * t);
    }
    __device__ __forceinline__ void load_v(int h, const PagedPiece& p, uint32_t v_pos, int col, int grp) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t o = (4 * grp + r) * v_pos;
            if constexpr (VB >= 16) {
#pragma unroll
                for (int i = 0; i < VB / 16; ++i) {
                    const u32x4 w = buffer_ld16(p.v, o + 256 * i + 16 * col);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[h][r][4 * i + e] = w[e];
                }
            } else if constexpr (VB == 8) {
                const auto w = __builtin_amdgcn_raw_buffer_load_b64(p.v, o + 8 * col, 0, 0);
                v[h][r][0] = w[0];
                v[h][r][1] = w[1];
            } else {
                v[h][r][0] = buffer_ld4(p.v, o + 4 * col);
            }
        }
    }
};

// Column of row i of p v's tile t: what lane i's loads hold.
template <int D, bool F8>
__device__ __forceinline__ int stream_col(int t, int i) {
    constexpr int per = F8 ? (D == 256 ? 16 : D / 16) : (D == 64 ? 4 : 8);  // columns of one load
    return 16 * per * (t / per) + per * i + t % per;
}

// RT row tiles of 16.
template <int D, bool F8, int RT>
__global__ void __launch_bounds__(64 * kStreamWaves, D * RT < 256 || F8 || D == 128 ? 2 : 1)
    paged_attn_bf16_stream(PagedKv c, PagedAttn a) {
    using S = StreamStep<D, F8>;
    constexpr int M = 16 * RT, T = D / 32, NT = D / 16;
    constexpr int kRow = D + 4;
    __shared__ int st_apart[kStreamWaves];
    __shared__ float st_m[kStreamWaves][M], st_l[kStreamWaves][M];
    __shared__ __attribute__((aligned(16))) float st_acc[kStreamWaves][16][kRow];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slot = blockIdx.x / c.HKV, head = blockIdx.x - slot * c.HKV;

    PagedWork w;
    if (!paged_work(c, a, M, slot, lane, w)) return;
    const PagedSlot& u = w.u;
    const PagedSeg& g = u.seg;
    const bool own = w.own;
    const int nrow = w.rows, begin = w.begin, end = w.end;

    // queries: B operands, and each row's limit (behind the tile's rows, its last one again)
    u32x4 q[RT][T];
    int limit[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int i = u.tile * M + min(16 * rt + col, nrow - 1);
        const int row = i / c.G, h = head * c.G + (i - row * c.G);
        limit[rt] = row_limit(g, w.kv_len, own, row);
        const uint16_t* p = a.q + (int64_t)(g.first + row) * a.ld_q + (int64_t)h * D;
#pragma unroll
        for (int t = 0; t < T; ++t)
            q[rt][t] = ldg16(p + (F8 ? 64 * (t >> 1) + 16 * grp + 8 * (t & 1) : 32 * t + 8 * grp));
    }

    const int32_t* table = own ? c.table + (int64_t)g.seq * c.ld_table : c.prefix_table + (int64_t)(g.seq - c.B) * c.ld_prefix;
    const char* kh = c.k + head * c.k_head;
    const char* vh = c.v + head * c.v_head;
    const ScoreFactor factor = score_factor<F8>(c, a, head);
    const float sc = factor.f;
    if (F8 && !factor.plain())
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < T; ++t) q[rt][t] = factor.query(q[rt][t]);

    pg_f32x4 acc[RT][NT];
    float m[RT], l[RT];
    bool seen[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
        seen[rt] = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[rt][t] = pg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // the pages of this wave's next 32 steps, one 16-key half to a lane
    constexpr int kStride = kStreamWaves * kStep;
    int pages = -1, page_step = -32;
    auto page_of = [&](int step, int (&pg)[2]) {  // step: of this wave, uniform
        if (step >= page_step + 32) {
            page_step = step;
            const int at = begin + kStep * wave + kStride * (step + (lane >> 1)) + 16 * (lane & 1);
            pages = at < end ? table[at >> c.shift] : -1;
        }
        pg[0] = __builtin_amdgcn_readlane(pages, 2 * (step - page_step));
        pg[1] = __builtin_amdgcn_readlane(pages, 2 * (step - page_step) + 1);
    };
    const int steps = max(0, (end - begin - kStep * wave + kStride - 1) / kStride);

    S s;
    int pg[2];
    page_of(0, pg);
    int at = begin + kStep * wave;
    PagedPiece piece[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        piece[h] = paged_piece<D * S::ES>(c, kh, vh, pg[h], at + 16 * h, end);
        s.load_k(h, piece[h], c.k_pos, col, grp);
        s.load_v(h, piece[h], c.v_pos, col, grp);
    }
    bool apart = false;
    for (int step = 0; step < steps; ++step, at += kStride) {
        const int there[2] = {piece[0].n, piece[1].n};
        const bool mask = at + kStep > w.all || there[0] < 16 || there[1] < 16;
        if (mask && w.all < end) {  // (behind all rows' limits zeros were loaded)
            bool odd = false;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < S::VW; ++i) odd |= F8 ? nan_f8x4(s.v[h][e][i]) : not_finite2(s.v[h][e][i]);
            apart = __ballot(odd) != 0;
            if (apart) break;
        }
        pg_f32x4 score[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) score[rt][0] = score[rt][1] = pg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 kk;
                if constexpr (F8) {
                    kk = f8_widen(s.k[h][t >> 1][2 * (t & 1)], s.k[h][t >> 1][2 * (t & 1) + 1]);
                } else {
                    kk = s.k[h][t];
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) score[rt][h] = pg_mfma16(kk, q[rt][t], score[rt][h]);
            }
        // the next step's keys take the registers of this one's (past the last step nothing is loaded)
        page_of(step + 1, pg);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            piece[h] = paged_piece<D * S::ES>(c, kh, vh, pg[h], at + kStride + 16 * h, end);
            s.load_k(h, piece[h], c.k_pos, col, grp);
        }

        uint32_t pb[RT][2][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            pg_f32x4(&sv)[2] = score[rt];
            if (mask) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // key 4 grp + r of the half step is attended and there
                    const int bound = min(limit[rt] - at - 16 * h, there[h]) - 4 * grp;
                    seen[rt] |= bound > 0;
#pragma unroll
                    for (int r = 0; r < 4; ++r) sv[h][r] = r < bound ? sv[h][r] : -INFINITY;
                }
            } else {
                seen[rt] = true;
            }
            float mx = fmaxf(fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[0][2], sv[0][3])),
                             fmaxf(fmaxf(sv[1][0], sv[1][1]), fmaxf(sv[1][2], sv[1][3])));
            mx = pg_across(mx, [](float x, float y) { return fmaxf(x, y); });
            const float mn = fmaxf(m[rt], mx * sc);
            const float ms = mn == -INFINITY ? 0.0f : mn;
            if (__ballot(mn != m[rt])) {
                const float f = pg_exp2(m[rt] - ms);
                l[rt] *= f;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[rt][t][r] *= f;
                m[rt] = mn;
            }
            float p[8];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // (a masked score is -inf, and so is its product with the positive sc)
                    p[4 * h + r] = pg_exp2(fmaf(sv[h][r], sc, -ms));
                    l[rt] += p[4 * h + r];
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t x = __float_as_uint(p[2 * i]), y = __float_as_uint(p[2 * i + 1]);
                pb[rt][0][i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                // (a trace of p keeps the second part positive where p is a bf16)
                pb[rt][1][i] = pack_bf16x2(fmaf(p[2 * i], 0x1p-60f, p[2 * i] - __uint_as_float(x & 0xFFFF0000u)),
                                           fmaf(p[2 * i + 1], 0x1p-60f, p[2 * i + 1] - __uint_as_float(y & 0xFFFF0000u)));
            }
        }

        // values of column tile t as the A operand: elements 0..3 of the first half step, 4..7 of the second
        auto column = [&](int t) {
            u32x4 r;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (F8)
                        w[e] = (t & 2) ? fp8x2_bf16<true>(s.v[h][e][t >> 2]) : fp8x2_bf16<false>(s.v[h][e][t >> 2]);
                    else
                        w[e] = s.v[h][e][t >> 1];
                }
                const uint32_t sel = (t & 1) ? 0x07060302u : 0x05040100u;
                r[2 * h] = __builtin_amdgcn_perm(w[1], w[0], sel);
                r[2 * h + 1] = __builtin_amdgcn_perm(w[3], w[2], sel);
            }
            return r;
        };
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const u32x4 w = column(t);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const u32x4 b0 = {pb[rt][0][0], pb[rt][0][1], pb[rt][0][2], pb[rt][0][3]};
                const u32x4 b1 = {pb[rt][1][0], pb[rt][1][1], pb[rt][1][2], pb[rt][1][3]};
                acc[rt][t] = pg_mfma16(w, b0, acc[rt][t]);
                acc[rt][t] = pg_mfma16(w, b1, acc[rt][t]);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) s.load_v(h, piece[h], c.v_pos, col, grp);
    }

    // the waves' parts
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float ls = pg_across(l[rt], [](float x, float y) { return x + y; });
        const float any = pg_across(seen[rt] ? 1.0f : 0.0f, [](float x, float y) { return fmaxf(x, y); });
        if (m[rt] == -INFINITY) ls = any;
        if (grp == 0) {
            st_m[wave][16 * rt + col] = m[rt];
            st_l[wave][16 * rt + col] = ls;
        }
    }
    if (lane == 0) st_apart[wave] = apart;
    const bool whole = w.parts == 1 && c.groups == 0;  // no other slot has keys of these rows
    const PagedParts parts(a, c, slot, head, M, D);
    const float vs = F8 ? c.v_scale[head] : 1.0f;
    if ((!a.arrived || c.groups > 0) && u.split == 0 && tid == 0) note_tile(c, a, w, M, slot, head);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (16 * rt >= nrow) break;
        if (rt > 0) __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) st_acc[wave][col][stream_col<D, F8>(t, 4 * grp + r)] = acc[rt][t][r];
        __syncthreads();
        if (rt == 0 && __builtin_amdgcn_readfirstlane(st_apart[0] | st_apart[1] | st_apart[2] | st_apart[3])) {
            paged_rows_apart<D, F8>(c, a, w, slot, head, M, wave, kStreamWaves, lane, [](int r, int d) { return r * D + d; });
            break;
        }
        for (int i = tid; i < 4 * D; i += 64 * kStreamWaves) {  // 16 rows of D / 4 pieces
            const int r = i / (D / 4), d = 4 * (i % (D / 4)), rr = 16 * rt + r;
            if (rr >= nrow) continue;
            PagedSum sum;
#pragma unroll
            for (int k = 0; k < kStreamWaves; ++k) {
                const float4 x = *reinterpret_cast<const float4*>(&st_acc[k][r][d]);
                sum.add(st_m[k][rr], st_l[k][rr], x);
            }
            if (whole) {
                const int k = u.tile * M + rr, row = k / c.G, h = head * c.G + (k - row * c.G);
                sum.store(a.out + (int64_t)(g.first + row) * a.ld_out + (int64_t)h * D + d, vs);
            } else {
                parts.put4(rr * D + d, sum.o[0], sum.o[1], sum.o[2], sum.o[3]);
                if (d == 0) parts.put_ml(rr, sum.m, sum.l);
            }
        }
    }
    if (!whole && a.arrived) {
        __syncthreads();  // (st_acc is used again)
        paged_join_last<D, F8>(c, a, w, head, M, tid, lane, reinterpret_cast<float(*)[8]>(&st_acc[0][0][0]), &st_apart[0]);
    }
}

}  // namespace bz
