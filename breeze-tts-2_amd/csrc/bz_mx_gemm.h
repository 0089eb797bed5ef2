// Products of microscaled rows with a microscaled 4-bit weight (bz_mx_device.h
// has layouts and formats): out[M, N] = q(x) @ w_eff^T (+ residual).
//
// Arithmetic: v_mfma_scale_f32_16x16x128_f8f6f4, A = 16 weight rows, B = 16
// rows of x, each lane with one block of 32 k and its scale code; D[n][m]
// lands in lane m + 16 (n / 4), element n % 4.  Sums stay in fp32 until the
// result's one rounding.
//
// Work decomposition
//   * A workgroup of eight waves owns a tile of 32 TM rows of x and 64 TN of
//     the weight, a unit (128 k) at a time.  Both operands are 1 KiB pieces
//     (2 KiB of 8-bit x) in the order of the instruction's lanes, so they go
//     from memory straight into LDS (16 bytes a lane) and from there to
//     registers without conversion, swizzle or bank conflict.
//   * Four stages of LDS: the loads of unit u + 3 go out in unit u, x operands
//     are read one unit ahead and weight operands one block ahead, so a unit
//     waits for nothing but its barrier.  Scale codes are a dword a lane for
//     four units, loaded a group ahead.
//   * A wave reads its own rows of x and of the weight from LDS, MT * XP + NT
//     KiB for MT * NT products, 128 bytes a cycle for the CU: that is what
//     bounds a unit of the narrower tiles.  Eight waves of half the
//     registers ran where four with 64 accumulator tiles each spilled their
//     operands to accumulator registers and back.
//   * Workgroups of one XCD go down `band` (at most 6) row tiles, then to the
//     next column tile: the XCD's L2 then holds x of 6 tiles and two or three
//     column tiles' weights (8192 x 20480 x 2560, e2m1: 226 us, whole
//     columns 257, single rows 244; e4m3 334, 376, 354).
//   * K slices where the tiles would leave CUs idle: fp32 sums to the
//     workspace, added in slice order by the last workgroup to arrive.
//
// Bound by the LDS reads in the narrower tiles, by power and LDS reads in large
// products: the card lowers its clock to 1.75 .. 1.9 GHz under the block-scaled
// instructions (over zeros the same kernel keeps 2.38 GHz: e2m1 8192 cubed 184
// us, 242 over random values).  The instruction alone, operands in registers,
// reaches 7400 TFLOP/s over random e2m1 (9800 over zeros) and 4700 over e4m3 x
// e2m1 (5000).  Two workgroups a CU of smaller tiles, wave priorities, waves
// half a unit apart and deeper stages changed nothing there.
// Measured on MI355X (graph replays; the ranges over cards and runs): e2m1 8192
// cubed 242 us (4550 TFLOP/s), 8192 x 20480 x 2560 226 .. 235 us (3800 .. 3650),
// 611 x 10240 x 2560 15.5 .. 15.8 us (2070); e4m3 8192 cubed 369 us (2980), 2011 x
// 2560 x 10240 45.1 .. 46.8 us (2340).  The card's large bf16 matmul reaches 1269.
#pragma once

#include <type_traits>

#include "bz_mx.h"
#include "bz_mx_device.h"

namespace bz {

typedef int mx_op_t __attribute__((ext_vector_type(8)));
typedef float mx_acc_t __attribute__((ext_vector_type(4)));

struct MxGemmParams {
    const uint8_t* x;
    const uint8_t* w;
    const void* res;
    int64_t ldr;
    void* out;
    int64_t ldo;
    uint32_t* cnt;   // nsl > 1: arrivals of each tile (zero between calls)
    float* part;     // nsl > 1: fp32 sums of the slices
    int M, N, NU, mblk, nblk;
    int mtiles, ntiles, nsl, gps;  // tiles, K slices, groups of four units per slice
    int band;                      // row tiles that neighbouring workgroups share columns over
    int res_f32, out_f32, vec;     // res NULL: none; vec: 16-byte accesses of out (and residual)
};

// Scale operands pick byte U of their dword.
template <int ELEM, int U>
__device__ __forceinline__ mx_acc_t mx_mfma(mx_op_t w, mx_op_t x, mx_acc_t c, uint32_t sw, uint32_t sx) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, ELEM == BZ_MX_E2M1 ? 4 : 0, U, (int)sw, U,
                                                            (int)sx);
}

__device__ __forceinline__ mx_op_t mx_op(u32x4 a) {
    return mx_op_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
}
__device__ __forceinline__ mx_op_t mx_op(u32x4 a, u32x4 b) {
    return mx_op_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// 16 bytes a lane straight into LDS, lane l's at p + 16 l.
__device__ __forceinline__ void mx_load_lds(__amdgpu_buffer_rsrc_t r, char* p, uint32_t lane_off, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)p, 16, lane_off, off, 0, 0);
}

constexpr int kMxWaves = 8;   // WM along the rows of x, the rest along the weight's
constexpr int kMxStages = 4;
constexpr int kMxCounters = 4096;
constexpr size_t kMxPartOffset = kMxCounters * 4;

template <int ELEM, int MT, int NT, int WM>
struct MxShape {
    static constexpr int XP = ELEM == BZ_MX_E2M1 ? 1 : 2;  // KiB of an x tile
    static constexpr int kWaves = kMxWaves, TM = MT * WM, TN = NT * (kWaves / WM);
    static constexpr int kPieces = TM * XP + TN;           // KiB of a stage
    // of each wave; few x tiles are loaded by several waves, to the same place
    static constexpr int kXLoads = (TM * XP + kWaves - 1) / kWaves, kLoads = kXLoads + TN / kWaves;
    static constexpr int kLds = kPieces * 1024 * kMxStages;
    static constexpr bool ok =
        TN % kWaves == 0 && kLds <= 160 * 1024 && MT * NT <= 32;
};

// s_waitcnt for all LDS operations and all but n vector memory ones (6 bits, split).
constexpr int mx_wait(int n) { return (n & 15) | (n >> 4) << 14 | 0x0070; }

template <int ELEM, int MT, int NT, int WM>
__global__ void __launch_bounds__(64 * kMxWaves, 2) mx_gemm(MxGemmParams p) {
    using S = MxShape<ELEM, MT, NT, WM>;
    constexpr int W = S::kWaves, XP = S::XP, TM = S::TM, TN = S::TN, L = S::kLoads, LX = S::kXLoads, SC = MT + NT;
    // one array a stage: the compiler then knows which loads into LDS a read waits for
    __shared__ __attribute__((aligned(16))) char s0[S::kPieces * 1024], s1[S::kPieces * 1024], s2[S::kPieces * 1024],
        s3[S::kPieces * 1024];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;

    // this workgroup's tile: XCD c = bid % 8 takes a run of consecutive ids,
    // which go down `band` row tiles, then to the next column tile
    const int nwg = (int)gridDim.x, bid = (int)blockIdx.x;
    const int per = nwg >> 3, rem = nwg & 7, xcd = bid & 7;
    const int id = xcd * per + min(xcd, rem) + (bid >> 3);
    const int sl = id % p.nsl, t = id / p.nsl;
    const int b0 = t / (p.band * p.ntiles), tb = t - b0 * p.band * p.ntiles;
    const int rows_b = min(p.band, p.mtiles - b0 * p.band);
    const int mt_i = b0 * p.band + tb % rows_b, nt_i = tb / rows_b;
    const int mb0 = mt_i * TM, nb0 = nt_i * TN;
    const int NU = p.NU;
    const int u_begin = sl * p.gps * 4, u_end = min(NU, u_begin + p.gps * 4);

    // x and w of the tile.  Blocks past the last repeat it (nothing of them is
    // stored); units past the slice lie out of range (zeros, no requests): an
    // offset with the top bit set, the host keeps a tile's rows below 2^31 bytes.
    const uint32_t xchunk = (uint32_t)(XP == 1 ? mx4_chunk_bytes(NU) : mx8_chunk_bytes(NU));
    const uint32_t wchunk = (uint32_t)mx4_chunk_bytes(NU);
    const int xlast = min(TM, p.mblk - mb0) - 1, wlast = min(TN, p.nblk - nb0) - 1;
    const __amdgpu_buffer_rsrc_t xr = buffer_rsrc(p.x + (int64_t)mb0 * xchunk, (uint32_t)(xlast + 1) * xchunk);
    const __amdgpu_buffer_rsrc_t wr = buffer_rsrc(p.w + (int64_t)nb0 * wchunk, (uint32_t)(wlast + 1) * wchunk);
    auto past = [&](int u) { return u < u_end ? 0u : 0x80000000u; };

    uint32_t piece_at[L];  // of each load, without the unit
    int piece_to[L];       // its place in a stage: x tiles, then w tiles
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const int piece = i < LX ? (W * i + wave) % (TM * XP) : W * (i - LX) + wave;
        piece_at[i] = i < LX ? (uint32_t)min(piece / XP, xlast) * xchunk + (uint32_t)(piece % XP) * 1024u
                             : (uint32_t)min(piece, wlast) * wchunk;
        piece_to[i] = (i < LX ? piece : TM * XP + piece) * 1024;
    }
    auto load = [&](int u, char* st) __attribute__((always_inline)) {
        const uint32_t v = (uint32_t)lane * 16u | past(u);
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const bool is_x = i < LX;
            mx_load_lds(is_x ? xr : wr, st + piece_to[i], v, piece_at[i] + (uint32_t)u * (is_x ? 1024u * XP : 1024u));
        }
    };
    uint32_t sx[MT], sw[NT], nx[MT], nw[NT];  // scale codes of this group and the next
    auto scales = [&](int u) __attribute__((always_inline)) {
        const uint32_t v = mx_scale_offset(u, lane) | past(u);
#pragma unroll
        for (int i = 0; i < MT; ++i)
            nx[i] = buffer_ld4(xr, v + ((uint32_t)min(wm * MT + i, xlast) * xchunk + (uint32_t)NU * (1024u * XP)));
#pragma unroll
        for (int i = 0; i < NT; ++i)
            nw[i] = buffer_ld4(wr, v + ((uint32_t)min(wn * NT + i, wlast) * wchunk + (uint32_t)NU * 1024u));
    };

    mx_acc_t acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mx_acc_t{0.0f, 0.0f, 0.0f, 0.0f};

    // the wave's rows of x, one unit ahead
    auto read_x = [&](mx_op_t (&o)[MT], int i, const char* st) __attribute__((always_inline)) {
        const char* a = st + (wm * MT + i) * (1024 * XP) + lane * 16;
        if (XP == 1)
            o[i] = mx_op(ldg16(a));
        else
            o[i] = mx_op(ldg16(a), ldg16(a + 1024));
    };
    auto unit = [&](auto q, int u, char* st, char* st1, char* next, mx_op_t (&xo)[MT], mx_op_t (&xn)[MT])
                    __attribute__((always_inline)) {
        constexpr int Q = decltype(q)::value;
        // the next unit's stage is in LDS (the loads of one more and, for Q =
        // 1, the next group's scales may be under way), and every wave has
        // read the stage that the next loads overwrite
        __builtin_amdgcn_s_waitcnt(mx_wait(L + (Q == 1 ? SC : 0)));
        __builtin_amdgcn_s_barrier();
        const char* wst = st + (TM * XP + wn * NT) * 1024 + lane * 16;
        u32x4 wv = ldg16(wst);
        // (fixed places: the wait counts above count on the loads' order, and
        // the scheduler would move them to the end of the unit)
        __builtin_amdgcn_sched_barrier(0);
        if (Q == 0) {
            scales(u + 4);
            __builtin_amdgcn_sched_barrier(0);
        }
        load(u + 3, next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const mx_op_t wo = mx_op(wv);
            if (j + 1 < NT) wv = ldg16(wst + (j + 1) * 1024);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                acc[i][j] = mx_mfma<ELEM, Q>(wo, xo[i], acc[i][j], sw[j], sx[i]);
                if ((j * MT + i + 1) % NT == 0) read_x(xn, (j * MT + i) / NT, st1);
            }
        }
        // LDS reads between the products, the last ones ahead of the unit's end
        constexpr int R = NT - 1 + MT * XP, P = MT * NT / (R + 3) > 0 ? MT * NT / (R + 3) : 1;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, P, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, MT * NT, 0);
    };
    scales(u_begin);
    __builtin_amdgcn_sched_barrier(0);
    load(u_begin, s0);
    load(u_begin + 1, s1);
    load(u_begin + 2, s2);
    mx_op_t xa[MT], xb[MT];
    __builtin_amdgcn_s_waitcnt(mx_wait(2 * L));
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int i = 0; i < MT; ++i) read_x(xa, i, s0);
    for (int u = u_begin; u < u_end; u += 4) {  // units past the slice multiply zeros
#pragma unroll
        for (int i = 0; i < MT; ++i) sx[i] = nx[i];
#pragma unroll
        for (int i = 0; i < NT; ++i) sw[i] = nw[i];
        unit(std::integral_constant<int, 0>{}, u, s0, s1, s3, xa, xb);
        unit(std::integral_constant<int, 1>{}, u + 1, s1, s2, s0, xb, xa);
        unit(std::integral_constant<int, 2>{}, u + 2, s2, s3, s1, xa, xb);
        unit(std::integral_constant<int, 3>{}, u + 3, s3, s0, s2, xb, xa);
    }
    __builtin_amdgcn_s_waitcnt(mx_wait(0));  // (no load into LDS outlives the workgroup)

    if (p.nsl > 1) {
        // the slice's sums to the workspace; the last workgroup of the tile
        // to arrive adds the slices in their order
        const int64_t wave_floats = MT * NT * 256, tile_floats = wave_floats * W;
        const int64_t tiles = (int64_t)p.mtiles * p.ntiles;
        const int64_t mine = (int64_t)(mt_i * p.ntiles + nt_i) * tile_floats + wave * wave_floats + lane * 4;
        auto slice = [&](int s) { return buffer_rsrc(p.part + s * tiles * tile_floats + mine - lane * 4, (uint32_t)(wave_floats * 4)); };
        const __amdgpu_buffer_rsrc_t own = slice(sl);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[i][j]), own,
                                                       (uint32_t)(((i * NT + j) * 64 + lane) * 16), 0, kCpolAgent);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        int* last = reinterpret_cast<int*>(s0);
        uint32_t* cnt = p.cnt + mt_i * p.ntiles + nt_i;
        if (threadIdx.x == 0) {
            const unsigned prev = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *last = prev == (unsigned)p.nsl - 1u;
            if (*last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!__builtin_amdgcn_readfirstlane(*last)) return;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mx_acc_t{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < p.nsl; ++s) {
            const __amdgpu_buffer_rsrc_t r = slice(s);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] += __builtin_bit_cast(mx_acc_t, __builtin_amdgcn_raw_buffer_load_b128(
                                                                  r, (uint32_t)(((i * NT + j) * 64 + lane) * 16), 0, kCpolAgent));
        }
    }

    // A lane's four columns 4 g .. 4 g + 3 (g = lane / 16) of two neighbouring
    // blocks become eight columns of one: after the swap of 16-lane rows g has
    // columns 8 (g / 2) .. + 7 of block g % 2, 64 bytes of bf16 a row and store.
    static_assert(NT % 2 == 0, "blocks in pairs");
    const int g = lane >> 4;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = (mb0 + wm * MT + i) * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i][j][e]),
                                                                __float_as_uint(acc[i][j + 1][e]), false, false);
                v[e] = __uint_as_float(r[0]);
                v[4 + e] = __uint_as_float(r[1]);
            }
            const int blk = nb0 + wn * NT + j + (g & 1), c = blk * 16 + 8 * (g >> 1);
            if (m >= p.M || blk >= p.nblk) continue;
            if (p.res) {
                const int64_t ri = (int64_t)m * p.ldr + c;
                if (p.vec && !p.res_f32) {
                    const u32x4 r = ldg16(static_cast<const uint16_t*>(p.res) + ri);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += (e & 1) ? bf16_hi(r[e >> 1]) : bf16_lo(r[e >> 1]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        v[e] += p.res_f32 ? static_cast<const float*>(p.res)[ri + e]
                                          : bf16_to_f32(static_cast<const uint16_t*>(p.res)[ri + e]);
                }
            }
            const int64_t o = (int64_t)m * p.ldo + c;
            if (p.out_f32) {
                float* q = static_cast<float*>(p.out) + o;
                if (p.vec) {
                    *reinterpret_cast<float4*>(q) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4*>(q + 4) = make_float4(v[4], v[5], v[6], v[7]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) q[e] = v[e];
                }
            } else {
                uint16_t* q = static_cast<uint16_t*>(p.out) + o;
                const u32x4 b = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                 pack_bf16x2(v[6], v[7])};
                if (p.vec) {
                    *reinterpret_cast<u32x4*>(q) = b;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) q[e] = (uint16_t)(b[e >> 1] >> (16 * (e & 1)));
                }
            }
        }
    }
}

struct MxGemmLaunch {
    int tm, tn;  // 32 rows of x and 64 of the weight in a tile
    unsigned grid;
};

// The tiles that are built, in 32 rows of x and 64 of the weight.
constexpr bool mx_shape_ok(int elem, int tm, int tn) {
    return tn == 2 ? tm == 1 || tm == 2 || tm == 4 || tm == 6
                   : tn == 4 && (tm == 4 || tm == (elem == BZ_MX_E2M1 ? 8 : 6));
}
// Waves along the rows of x: four over the narrow tiles, where two would read
// more of LDS for the same products (e4m3 6 x 2: 14 KiB a wave for 12, with four
// 10; 2011 x 2560 x 10240 48.9 -> 46.7 us) and, for e2m1 6 x 2, need 128
// registers and more, so that a CU held one workgroup (2011 x 20480 x 2560 81.5
// -> 66.9 us).  4 x 4: 94.3 us with two, 95.3 with four.
constexpr int mx_waves_m(int tm, int tn) { return tn == 2 && tm >= 4 ? 4 : 2; }

template <int ELEM, int TM, int TN>
int launch_mx_gemm_kernel(const MxGemmParams& p, const MxGemmLaunch& l, hipStream_t st) {
    if constexpr (mx_shape_ok(ELEM, TM, TN)) {
        constexpr int WM = mx_waves_m(TM, TN), MT = 2 * TM / WM, NT = TN * 4 * WM / kMxWaves;
        static_assert(MxShape<ELEM, MT, NT, WM>::ok && MT * WM == 2 * TM);
        hipLaunchKernelGGL((mx_gemm<ELEM, MT, NT, WM>), dim3(l.grid), dim3(64 * kMxWaves), 0, st, p);
        return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
    } else {
        return BZ_ERR_INVALID_ARG;
    }
}
template <int ELEM, int TN>
int launch_mx_gemm_tn(const MxGemmParams& p, const MxGemmLaunch& l, hipStream_t st) {
    switch (l.tm) {
        case 1: return launch_mx_gemm_kernel<ELEM, 1, TN>(p, l, st);
        case 2: return launch_mx_gemm_kernel<ELEM, 2, TN>(p, l, st);
        case 4: return launch_mx_gemm_kernel<ELEM, 4, TN>(p, l, st);
        case 6: return launch_mx_gemm_kernel<ELEM, 6, TN>(p, l, st);
        case 8: return launch_mx_gemm_kernel<ELEM, 8, TN>(p, l, st);
        default: return BZ_ERR_INVALID_ARG;
    }
}
template <int ELEM>
int launch_mx_gemm_elem(const MxGemmParams& p, const MxGemmLaunch& l, hipStream_t st) {
    switch (l.tn) {
        case 2: return launch_mx_gemm_tn<ELEM, 2>(p, l, st);
        case 4: return launch_mx_gemm_tn<ELEM, 4>(p, l, st);
        default: return BZ_ERR_INVALID_ARG;
    }
}

int launch_mx_gemm_e2m1(const MxGemmParams& p, const MxGemmLaunch& l, hipStream_t st);
int launch_mx_gemm_e4m3(const MxGemmParams& p, const MxGemmLaunch& l, hipStream_t st);

}  // namespace bz
