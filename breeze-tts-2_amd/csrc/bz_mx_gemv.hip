// Host side of the few-row products of rows quantised on the way (C ABI
// entries bz_mx_gemv and bz_mx_gemv_workspace).
#include <algorithm>

#include "bz_gemv_kernel.h"
#include "bz_mx_gemv.h"

namespace bz {

struct MxGemvPlan {
    MxGemvLaunch l;
    int T, nsl, ups;
    size_t ws;
};

// Built-in rule (sweeps of blocks, units per wave and slices on MI355X, M = 1
// .. 32, us): about one workgroup per CU.  One slice while the x that every
// workgroup then reads is short: up to 32 units, up to 48 for 8 rows, 64 for 5
// and 96 for 2 (e4m3 N4096 K6144 M = 8 one slice 7.03, two 7.82; N1024 K8192 M =
// 4 5.70, four 6.25, M = 8 7.0, three 6.65; N2560 K10240 M = 2 6.87, four 7.57; M
// = 4 7.9, 7.79).  Beyond, slices of about 25 units, at most four, for up to 8
// rows (N320 K16384 M = 5 four 6.20, seven 6.56), of 20, at least four, for up to
// 16 (e4m3 N4096 K6144 M = 16 four 8.64, three 9.74) and of 13 for more (N2560
// K10240 M = 32: 6 slices of 4 blocks
// 11.2, 4 of 3 12.2).  Units per wave: 2 (N20480 K2560 M = 5: 5 blocks x 2 units
// 7.97, x 4 8.22, 3 blocks x 2 8.41); 4, which share their operands of x, for up
// to 8 rows where 2 would need 16 waves or more (N16384 K4096 M = 1 8.65, 2 units
// 8.97) and for up to 4 over one or two blocks (N1024 K2048 M = 1 3.42, 3.54;
// N10240 K2560 M = 4, three blocks, 5.97, 5.92); 1 for more than 16 rows in slices
// (e4m3 N10240 K2560: 2 slices of 5 11.0, one of 3 11.6).
// More than 16 rows keep up to 16 KiB of sums a wave, which may not fit LDS:
// then fewer slices, so fewer blocks a workgroup (N4096 K10240 M = 17: 4 slices
// of 4 blocks 11.4, 6 of 6 with two units a wave 16.2, quantising in a launch of
// its own 15.4; N8192 K5120 M = 32 12.8, 18.6, 13.6), and over one slice more units
// a wave (N20480 K4096 M = 17 3 units 14.0, 2 units over 4 blocks 16.6).
static int mx_gemv_plan(int elem, int M, int N, int K, int cfg, MxGemvPlan& pl) {
    const int NU = K / 128, nblk = N / 16, mt = M > 16 ? 2 : 1;
    const int cT = cfg & 255, cu = (cfg >> 8) & 255, cs = cfg >> 16;
    if (cT > kMxGemvBlocks || cs > 64) return BZ_ERR_INVALID_ARG;
    auto blocks = [&](int slices) { return cT ? cT : (int)(((int64_t)nblk * slices + 255) / 256); };
    const bool whole = NU <= 32 || (NU <= 48 && M <= 8) || (NU <= 64 && M <= 5) || (NU <= 96 && M <= 2);
    int nsl = cs        ? cs
              : mt == 2 ? std::max(1, (NU + 6) / 13)
              : whole   ? 1
              : M <= 8  ? std::min(4, (NU + 24) / 25)
                        : std::max(4, (NU + 19) / 20);
    if (!cs && blocks(nsl) > kMxGemvBlocks) nsl = 1;
    nsl = std::min(nsl, NU);
    auto most = [&](int slices) { return std::min(kMxGemvBlocks, blocks(slices)); };
    bool over = false;  // the waves hold some shape that LDS or the workspace does not
    // The fewest units per wave with which the waves of workgroups of t blocks
    // hold a slice, or, where their sums do not fit LDS and `more`, the fewest
    // with which they do; 0: none.
    auto units = [&](int slices, int t, bool more) {
        const int ups = (NU + slices - 1) / slices;
        const bool four = M <= 8 && (ups >= 32 || (slices == 1 && M <= 4 && t <= 2 && NU >= 16));
        const int least = ups == 1 || (slices > 1 && mt == 2) ? 1 : four ? 4 : 2;
        const bool counted = slices == 1 || ((nblk + t - 1) / t <= kMxCounters && (int64_t)slices * M * N * 4 < (int64_t)1 << 31);
        for (int u : kMxGemvUpw) {
            const int share = mx_gemv_share(M, u);
            if (!mx_gemv_built(mt, u, share) || (cu ? u != cu : u < least) || mx_gemv_waves(elem, mt, u, share) * u < ups)
                continue;
            if (counted && mx_gemv_lds((ups + u - 1) / u, t, mt) <= kMxGemvMostLds) return u;
            over = true;
            if (!more) break;
        }
        return 0;
    };
    const int T0 = most(nsl);
    int s = nsl, T = T0, upw = units(s, T, s == 1 || cs);
    if (!cs)
        while (!upw && over && s > 1) {
            --s;
            T = most(s);
            upw = units(s, T, s == 1);
        }
    if (!upw) s = nsl;
    while (!upw) {  // more slices where the waves do not hold the row, fewer blocks where their sums never fit
        for (T = T0; !(upw = units(s, T, true)) && T > 1 && !cT;) --T;
        if (upw) break;
        if (cu || cs) return over ? BZ_ERR_UNSUPPORTED : BZ_ERR_INVALID_ARG;
        if (++s > 64) return BZ_ERR_UNSUPPORTED;
    }
    pl.ups = (NU + s - 1) / s;
    pl.nsl = (NU + pl.ups - 1) / pl.ups;
    pl.l.upw = upw;
    pl.l.share = mx_gemv_share(M, upw);
    pl.l.nw = (pl.ups + upw - 1) / upw;
    pl.T = T;
    pl.l.mt = mt;
    pl.l.grid = (unsigned)((nblk + T - 1) / T * pl.nsl);
    pl.l.lds = (size_t)mx_gemv_lds(pl.l.nw, T, mt);
    pl.ws = pl.nsl > 1 ? kMxPartOffset + (size_t)pl.nsl * M * N * 4 : 0;
    return BZ_OK;
}

template <int ELEM, int MT, int UPW, int G>
static int launch_share(const MxGemvParams& p, const MxGemvLaunch& l, hipStream_t st) {
    if constexpr (mx_gemv_built(MT, UPW, G)) {
        auto kern = mx_gemv<ELEM, MT, UPW, G>;
        if (l.lds > 65536 && raise_lds_limit(reinterpret_cast<const void*>(kern)) != BZ_OK) return BZ_ERR_LAUNCH;
        hipLaunchKernelGGL(kern, dim3(l.grid), dim3(64 * l.nw), l.lds, st, p);
        return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
    } else {
        return BZ_ERR_INVALID_ARG;
    }
}
template <int ELEM, int MT, int UPW>
static int launch_kernel(const MxGemvParams& p, const MxGemvLaunch& l, hipStream_t st) {
    switch (l.share) {
        case 1: return launch_share<ELEM, MT, UPW, 1>(p, l, st);
        case 2: return launch_share<ELEM, MT, UPW, 2>(p, l, st);
        default: return launch_share<ELEM, MT, UPW, 4>(p, l, st);
    }
}
template <int ELEM, int MT>
static int launch_t(const MxGemvParams& p, const MxGemvLaunch& l, hipStream_t st) {
    switch (l.upw) {
        case 1: return launch_kernel<ELEM, MT, 1>(p, l, st);
        case 2: return launch_kernel<ELEM, MT, 2>(p, l, st);
        case 3: return launch_kernel<ELEM, MT, 3>(p, l, st);
        case 4: return launch_kernel<ELEM, MT, 4>(p, l, st);
        case 5: return launch_kernel<ELEM, MT, 5>(p, l, st);
        case 6: return launch_kernel<ELEM, MT, 6>(p, l, st);
        default: return launch_kernel<ELEM, MT, 8>(p, l, st);
    }
}
template <int ELEM>
static int launch_mt(const MxGemvParams& p, const MxGemvLaunch& l, hipStream_t st) {
    return l.mt == 1 ? launch_t<ELEM, 1>(p, l, st) : launch_t<ELEM, 2>(p, l, st);
}

static int mx_gemv_check(int elem, int M, int N, int K) {
    if (M < 1 || N < 1 || K < 1 || (elem != BZ_MX_E2M1 && elem != BZ_MX_E4M3)) return BZ_ERR_INVALID_ARG;
    if (N % 16 || K % 128) return BZ_ERR_SHAPE;
    return M > kMxGemvRows || K > (1 << 22) ? BZ_ERR_UNSUPPORTED : BZ_OK;
}

}  // namespace bz

using namespace bz;

extern "C" size_t bz_mx_gemv_workspace(int32_t elem, int32_t M, int32_t N, int32_t K, int32_t cfg) {
    MxGemvPlan pl;
    if (cfg < 0 || mx_gemv_check(elem, M, N, K) != BZ_OK) return (size_t)-1;
    return mx_gemv_plan(elem, M, N, K, cfg, pl) == BZ_OK ? pl.ws : (size_t)-1;
}

extern "C" int bz_mx_gemv(int32_t elem, const void* x, int64_t ldx, int32_t M, const void* w, int32_t N, int32_t K,
                          const void* residual, int32_t residual_dtype, int64_t ldr, void* out, int32_t out_dtype,
                          int64_t ldo, void* workspace, size_t workspace_bytes, int32_t cfg, void* stream) {
    if (!x || !w || !out || cfg < 0) return BZ_ERR_INVALID_ARG;
    if (out_dtype != BZ_DT_BF16 && out_dtype != BZ_DT_F32) return BZ_ERR_INVALID_ARG;
    if (residual && residual_dtype != BZ_DT_BF16 && residual_dtype != BZ_DT_F32) return BZ_ERR_INVALID_ARG;
    const int rc = mx_gemv_check(elem, M, N, K);
    if (rc != BZ_OK) return rc;
    if (ldx < K || ldo < N || (residual && ldr < N)) return BZ_ERR_INVALID_ARG;
    auto off = [](const void* q, uintptr_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) != 0; };
    if (off(x, 16) || ldx % 8 || off(w, 16) || off(out, out_dtype == BZ_DT_F32 ? 4 : 2) ||
        (residual && off(residual, residual_dtype == BZ_DT_F32 ? 4 : 2)))
        return BZ_ERR_ALIGNMENT;
    if (((int64_t)(M - 1) * ldx + K) * 2 >= (int64_t)1 << 31) return BZ_ERR_UNSUPPORTED;  // 32-bit offsets
    MxGemvPlan pl;
    const int prc = mx_gemv_plan(elem, M, N, K, cfg, pl);
    if (prc != BZ_OK) return prc;
    if (pl.ws && (!workspace || off(workspace, 16) || workspace_bytes < pl.ws)) return BZ_ERR_INVALID_ARG;
    MxGemvParams p{};
    p.x = static_cast<const uint16_t*>(x);
    p.ldx = ldx;
    p.w = static_cast<const uint8_t*>(w);
    p.res = residual;
    p.ldr = ldr;
    p.out = out;
    p.ldo = ldo;
    p.cnt = static_cast<uint32_t*>(workspace);
    p.part = pl.ws ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kMxPartOffset) : nullptr;
    p.M = M;
    p.K = K;
    p.NU = K / 128;
    p.nblk = N / 16;
    p.T = pl.T;
    p.nsl = pl.nsl;
    p.ups = pl.ups;
    p.res_f32 = residual_dtype == BZ_DT_F32;
    p.out_f32 = out_dtype == BZ_DT_F32;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return elem == BZ_MX_E2M1 ? launch_mt<BZ_MX_E2M1>(p, pl.l, st) : launch_mt<BZ_MX_E4M3>(p, pl.l, st);
}
