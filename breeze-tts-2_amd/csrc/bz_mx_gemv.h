// Few rows times a microscaled 4-bit weight, the rows quantised on the way:
// out[M, N] = q(x) @ w_eff^T (+ residual) for up to 32 rows of bf16 x, in one
// launch that reads every weight byte once.
//
// Bound by the weight's bytes and by the latency of a launch.  Measured on
// MI355X (graph replays, weights not in a cache): e2m1 N20480 K2560 M = 1 7.5 us
// (3.7 TB/s of weight), M = 16 9.1; N2560 K10240 M = 5 7.8 us, e4m3 7.8; N1024
// K2048 M = 1 3.4 us.  Quantising in a launch of its own, bz_mx_gemm behind it,
// took 15.0 us for the third of these.
//
// Work decomposition (that of the several-block streaming kernel,
// bz_gemv_wide.h, with the panel kernel's K slices, bz_gemv_panel.h)
//   * A workgroup owns T consecutive row blocks of the weight over the whole
//     K or one of nsl K slices; each of its waves UPW consecutive units of
//     every block.  All x loads go out first, then the first block's tiles;
//     x is quantised while they arrive and stays in registers for the T
//     blocks, whose tiles follow one another in two register sets.
//   * x is quantised in the lane that multiplies it: lane 16 g + j reads block
//     g of row j, 64 contiguous bytes, finds its largest magnitude and packs
//     the elements with the scaled conversion.  No lane needs another's
//     values, and quantising costs no launch (a launch of its own over a few
//     rows takes 2.9 us on MI355X).
//   * Up to 8 (4) rows leave half (three quarters) of an operand's rows free:
//     these hold the same rows' next unit(s), so that all lanes quantise and 2
//     (4) units share one operand.  Each unit's product is whole, into sums of
//     its own, of which only its own rows count; they meet after the last
//     unit.  Every workgroup quantises all the x it reads, so this is what
//     took longest (N2560 K4096 M = 1 4.78 -> 4.20 us, N1024 K8192 M = 1 6.25 ->
//     4.85 with the longer slices it allows, N20480 K2560 M = 5 7.97 -> 7.74).
//   * The waves' sums are added through LDS in wave order; over K slices the
//     last workgroup of a group to arrive adds the slices in their order.
//
// Arithmetic: v_mfma_scale_f32_16x16x128_f8f6f4 as in bz_mx_gemm.h.  For 8-bit
// elements the instruction wants k = 16 g .. + 15 and 64 + 16 g .. + 15 in lane
// row g: exchanging the second half of a lane's block with the first half of
// its odd neighbour row's (v_permlane16_swap) gives it blocks 0, 2, 1, 3 in
// this order, so the weight's lane rows 1 and 2 read each other's blocks and
// the scales follow.
#pragma once

#include "bz_mx_gemm.h"

namespace bz {

struct MxGemvParams {
    const uint16_t* x;
    int64_t ldx;
    const uint8_t* w;
    const void* res;
    int64_t ldr;
    void* out;
    int64_t ldo;
    uint32_t* cnt;   // nsl > 1: arrivals of each group (zero between calls)
    float* part;     // nsl > 1: fp32 sums [nsl][M][nblk * 16]
    int M, K, NU, nblk;
    int T;           // row blocks per workgroup
    int nsl, ups;    // K slices and units per slice
    int res_f32, out_f32;
};

constexpr int kMxGemvRows = 32;
constexpr int kMxGemvBlocks = 8;                        // most row blocks of a workgroup
constexpr int kMxGemvUpw[] = {1, 2, 3, 4, 5, 6, 8};  // units per wave
__host__ __device__ constexpr int mx_gemv_lds(int NW, int T, int MT) { return NW * T * MT * 1024 + 16; }
constexpr int kMxGemvMostLds = 160 * 1024;
// Units of a wave that share one operand of x: rows 16 / G and more of it belong
// to the next unit.
constexpr int mx_gemv_share(int M, int upw) { return M <= 4 && upw >= 3 ? 4 : M <= 8 && upw >= 2 ? 2 : 1; }
// Most waves of a workgroup: 16 while two sets of tiles and the quantised x of
// a wave's units leave room in 128 registers, else 8.
__host__ __device__ constexpr int mx_gemv_waves(int elem, int mt, int upw, int G) {
    return upw * 10 + (upw + G - 1) / G * mt * (elem == BZ_MX_E2M1 ? 5 : 9) <= 80 ? 16 : 8;
}
constexpr bool mx_gemv_built(int mt, int upw, int G) {
    return mt == 1 ? G == 1 || (G == 2 && upw >= 2) || (G == 4 && upw >= 3) : G == 1 && upw <= 5;
}

// Lane j of 16 gets that of lane (j - N) % 16.
template <int N>
__device__ __forceinline__ mx_acc_t ror16(mx_acc_t v) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        v[e] = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v[e]), 0x120 + N, 0xF, 0xF, false));
    return v;
}

// A block of 32 bf16 values: its scale code and elements (e2m1: the first
// four dwords; e4m3: eight).
template <int ELEM>
__device__ __forceinline__ uint32_t mx_quantize_block(const u32x4 (&v)[4], u32x4& lo, u32x4& hi) {
    us2_t m = {0, 0};  // magnitudes of bf16 compare as integers, NaN on top
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2_t, v[i][e] & 0x7FFF7FFFu));
    const uint32_t a = max((uint32_t)m[0], (uint32_t)m[1]);
    const uint32_t code = mx_code<ELEM == BZ_MX_E2M1 ? 2 : 8>(a >> 7);
    const float s = __uint_as_float(code << 23);
    if (ELEM == BZ_MX_E2M1) {
        lo = u32x4{mx4_pack_bf16(v[0], s), mx4_pack_bf16(v[1], s), mx4_pack_bf16(v[2], s), mx4_pack_bf16(v[3], s)};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t a, b;
            mx8_pack_bf16(v[i], code, s, a, b);
            if (i < 2)
                lo[2 * i] = a, lo[2 * i + 1] = b;
            else
                hi[2 * i - 4] = a, hi[2 * i - 3] = b;
        }
    }
    return code;
}

template <int ELEM, int MT, int UPW, int G>
__global__ void __launch_bounds__(64 * mx_gemv_waves(ELEM, MT, UPW, G)) mx_gemv(MxGemvParams p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr bool F8 = ELEM == BZ_MX_E4M3;
    const int nthr = blockDim.x, NW = nthr >> 6;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 15, g = lane >> 4;
    const int M = p.M, NU = p.NU, T = p.T;
    const int grp = (int)blockIdx.x / p.nsl, sl = (int)blockIdx.x - grp * p.nsl;
    const int blk0 = grp * T, nb = min(T, p.nblk - blk0);
    const int ue = min(NU, (sl + 1) * p.ups), u0 = sl * p.ups + wave * UPW;

    // x: rows past M and units past the slice read as zeros, without
    // requests; up to four units' rows are under way
    const __amdgpu_buffer_rsrc_t xrs = buffer_rsrc(p.x, (uint32_t)(((int64_t)(M - 1) * p.ldx + p.K) * 2));
    constexpr int R = 16 / G, NS = (UPW + G - 1) / G;  // rows of a unit in an operand, and operands
    constexpr int NX = NS * MT, XD = NX < 4 ? NX : 4;
    u32x4 xv[XD][4];
    auto x_load = [&](int i) __attribute__((always_inline)) {  // row group i % MT of operand i / MT
        const int m = 16 * (i % MT) + j % R, u = u0 + i / MT * G + j / R;
        const uint32_t o = ((m < M ? (uint32_t)((m * (int)p.ldx + 32 * g) * 2) : 0x80000000u) + (uint32_t)u * 256u) |
                           (u < ue ? 0u : 0x80000000u);
#pragma unroll
        for (int k = 0; k < 4; ++k) xv[i % XD][k] = buffer_ld16(xrs, o + k * 16u);
    };
#pragma unroll
    for (int i = 0; i < XD; ++i) x_load(i);

    // tiles of the workgroup's blocks; the sets are of even and odd blocks (a
    // tile carried around the loop made the compiler wait for every load)
    const int wl = F8 ? (g == 1 ? lane + 16 : g == 2 ? lane - 16 : lane) : lane;  // whose block of a tile this lane takes
    const uint32_t chunk = (uint32_t)mx4_chunk_bytes(NU);
    const __amdgpu_buffer_rsrc_t wrs = buffer_rsrc(p.w + (int64_t)blk0 * chunk, (uint32_t)nb * chunk);
    u32x4 wa[UPW], wb[UPW];
    uint32_t sa[UPW], sb[UPW];
    auto issue = [&](int jb, int q, u32x4* wv, uint32_t* sc) __attribute__((always_inline)) {
        const int u = u0 + q;
        const uint32_t past = jb < nb && u < ue ? 0u : 0x80000000u, base = (uint32_t)jb * chunk;
        wv[q] = buffer_ld16_nt(wrs, (base + (uint32_t)u * 1024u + wl * 16) | past);
        sc[q] = buffer_ld4(wrs, (base + (uint32_t)NU * 1024u + mx_scale_offset(u, wl)) | past);
    };
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();  // every wave's first x loads are issued before any weight load
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < UPW; ++q) issue(0, q, wa, sa);
    __builtin_amdgcn_sched_barrier(0);

    mx_op_t xq[NS][MT];
    uint32_t sx[NS][MT];
#pragma unroll
    for (int i = 0; i < NX; ++i) {
        u32x4 lo, hi = {0u, 0u, 0u, 0u};
        uint32_t c = mx_quantize_block<ELEM>(xv[i % XD], lo, hi);
        if (F8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const auto r = __builtin_amdgcn_permlane16_swap(lo[e], hi[e], false, false);
                lo[e] = r[0];
                hi[e] = r[1];
            }
            c = (uint32_t)__builtin_amdgcn_ds_bpermute(wl * 4, (int)c);
            xq[i / MT][i % MT] = mx_op(lo, hi);
        } else {
            xq[i / MT][i % MT] = mx_op(lo);
        }
        sx[i / MT][i % MT] = c;
        if (i + XD < NX) x_load(i + XD);
    }

    // the waves' sums, [wave][block][row group][row % 16][column]
    float* red = reinterpret_cast<float*>(smem);
    auto run_block = [&](int jb, const u32x4* cw, const uint32_t* cs, u32x4* nw2, uint32_t* ns2)
                         __attribute__((always_inline)) {
        mx_acc_t acc[MT][G];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int s = 0; s < G; ++s) acc[mt][s] = mx_acc_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < UPW; ++q) {
            const mx_op_t w = mx_op(cw[q]);
            const uint32_t sw = cs[q] >> (8 * ((u0 + q) & 3));
            issue(jb + 1, q, nw2, ns2);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                acc[mt][q % G] = mx_mfma<ELEM, 0>(w, xq[q / G][mt], acc[mt][q % G], sw, sx[q / G][mt]);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            mx_acc_t a = acc[mt][0];
#pragma unroll
            for (int s = 1; s < G; ++s) a = j / R == s ? acc[mt][s] : a;
            if (G >= 2) a += ror16<8>(a);
            if (G >= 4) a += ror16<4>(a);
            *reinterpret_cast<mx_acc_t*>(red + ((wave * T + jb) * MT + mt) * 256 + j * 16 + 4 * g) = a;
        }
    };
    int jb = 0;
    for (; jb + 1 < nb; jb += 2) {
        run_block(jb, wa, sa, wb, sb);
        run_block(jb + 1, wb, sb, wa, sa);
    }
    if (jb < nb) run_block(jb, wa, sa, wb, sb);
    __syncthreads();
    const int nitem = M * 4 * T, n_out = p.nblk * 16;
    auto finish = [&](mx_acc_t a, int m, int c) {  // columns c .. c + 3 of the workgroup's
        const int64_t ri = (int64_t)m * p.ldr + blk0 * 16 + c, oi = (int64_t)m * p.ldo + blk0 * 16 + c;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float v = a[q];
            if (p.res)
                v += p.res_f32 ? static_cast<const float*>(p.res)[ri + q]
                               : bf16_to_f32(static_cast<const uint16_t*>(p.res)[ri + q]);
            if (p.out_f32)
                static_cast<float*>(p.out)[oi + q] = v;
            else
                static_cast<uint16_t*>(p.out)[oi + q] = f32_to_bf16(v);
        }
    };
    const __amdgpu_buffer_rsrc_t prs = buffer_rsrc(p.part, p.nsl > 1 ? (uint32_t)((int64_t)p.nsl * M * n_out * 4) : 0u);
    for (int it = tid; it < nitem; it += nthr) {
        const int m = it / (4 * T), c = (it - m * 4 * T) * 4;
        if (blk0 + (c >> 4) >= p.nblk) continue;
        const float* rp = red + ((c >> 4) * MT + (m >> 4)) * 256 + (m & 15) * 16 + (c & 15);
        mx_acc_t a = {0.0f, 0.0f, 0.0f, 0.0f};
        // (all reads under way at once; slots of waves the workgroup does not have add zero)
        mx_acc_t v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = *reinterpret_cast<const mx_acc_t*>(rp + min(i, NW - 1) * T * MT * 256);
#pragma unroll
        for (int i = 0; i < 16; ++i) a += i < NW ? v[i] : mx_acc_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (p.nsl == 1)
            finish(a, m, c);
        else
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, a), prs,
                                                   (uint32_t)((((int64_t)sl * M + m) * n_out + blk0 * 16 + c) * 4), 0,
                                                   kCpolAgent);
    }
    if (p.nsl == 1) return;
    int& last = *reinterpret_cast<int*>(smem + mx_gemv_lds(NW, T, MT) - 16);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const unsigned prev = __hip_atomic_fetch_add(&p.cnt[grp], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = prev == (unsigned)p.nsl - 1u;
        if (last) __hip_atomic_store(&p.cnt[grp], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    for (int it = tid; it < nitem; it += nthr) {
        const int m = it / (4 * T), c = (it - m * 4 * T) * 4;
        if (blk0 + (c >> 4) >= p.nblk) continue;
        const uint32_t o = (uint32_t)(((int64_t)m * n_out + blk0 * 16 + c) * 4), step = (uint32_t)((int64_t)M * n_out * 4);
        mx_acc_t a = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s0 = 0; s0 < p.nsl; s0 += 4) {  // four loads under way
            u32x4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = __builtin_amdgcn_raw_buffer_load_b128(prs, o + (uint32_t)min(s0 + i, p.nsl - 1) * step, 0, kCpolAgent);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (s0 + i < p.nsl) a += __builtin_bit_cast(mx_acc_t, v[i]);
        }
        finish(a, m, c);
    }
}

struct MxGemvLaunch {
    int nw, mt, upw, share;
    unsigned grid;
    size_t lds;
};

}  // namespace bz
