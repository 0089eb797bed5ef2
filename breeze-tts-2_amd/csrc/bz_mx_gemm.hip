// Host side of the products of microscaled rows (C ABI entries bz_mx_gemm and
// bz_mx_gemm_workspace).
#include <algorithm>

#include "bz_mx_gemm.h"

namespace bz {

struct MxGemmPlan {
    MxGemmLaunch l;
    int mtiles, ntiles, nsl, gps;
    size_t ws;
};

static int mx_gemm_shape(int M, int N, int K, int mt, int nt, int nsl, MxGemmPlan& pl) {
    const int mblk = (M + 15) / 16, nblk = N / 16, groups = (K / 128 + 3) / 4;
    const int tm = mt * kMxWavesM, tn = nt * kMxWn;
    pl.l.mt = mt;
    pl.l.nt = nt;
    pl.mtiles = (mblk + tm - 1) / tm;
    pl.ntiles = (nblk + tn - 1) / tn;
    const int64_t tiles = (int64_t)pl.mtiles * pl.ntiles;
    nsl = std::max(1, std::min(nsl, groups));
    if (tiles > kMxCounters) nsl = 1;
    pl.gps = (groups + nsl - 1) / nsl;
    pl.nsl = (groups + pl.gps - 1) / pl.gps;
    if (tiles * pl.nsl * 512 >= (int64_t)1 << 32) return BZ_ERR_UNSUPPORTED;
    pl.l.grid = (unsigned)(tiles * pl.nsl);
    pl.ws = pl.nsl > 1 ? kMxPartOffset + (size_t)pl.nsl * tiles * tm * tn * 256 * 4 : 0;
    return BZ_OK;
}

// Microseconds a launch shape is expected to take, from which the rule picks
// the smallest: a workgroup's start and end (wg0) and its units; with room for
// several workgroups on a CU a unit takes the longer of one workgroup's time
// and of the CU's for all it holds (full); the workspace's traffic where K is
// sliced; and reading x and the weight for every tile.  Fitted to graph
// replays over 13 (N, K) (the model's layers, 1024 squared, 656 x 384 and 7408
// x 3968), M = 33 .. 2048 and 1 .. 8 slices on MI355X, 7211 timings.  Over
// those the shape it picks takes 2.2% (e2m1) / 1.8% (e4m3) longer than the
// best one of the sweep, which had 19 shapes, on average; at worst 19% (M =
// 100, N 20480, K 2560: 11.4 us for 9.6) / 39% (M = 400, N 2560, K 10240: 28.6
// for 20.6).
struct MxGemmCost {
    int mt, nt;
    float wg0, unit, full, sum0, sum_mb, traffic_mb;
};
constexpr MxGemmCost kMxCostE2m1[] = {
    {1, 2, 3.435f, 0.1493f, 0.1647f, 2.297f, 0.3003f, 0.01155f},
    {2, 2, 3.695f, 0.1696f, 0.1919f, 2.457f, 0.2701f, 0.01151f},
    {4, 2, 4.149f, 0.2301f, 0.2958f, 2.936f, 0.2929f, 0.01471f},
    {6, 2, 4.86f, 0.313f, 0.4354f, 4.551f, 0.2658f, 0.02368f},
    {4, 4, 5.208f, 0.3543f, 0.03681f, 6.453f, 0.1808f, 0.01889f},
    {8, 4, 8.477f, 0.5144f, 0.1102f, 10.3f, 0.1231f, 0.0387f},
};
constexpr MxGemmCost kMxCostE4m3[] = {
    {1, 2, 3.481f, 0.1694f, 0.1605f, 2.288f, 0.3089f, 0.01263f},
    {2, 2, 3.702f, 0.1891f, 0.2153f, 2.427f, 0.3021f, 0.01287f},
    {4, 2, 4.202f, 0.3289f, 0.3259f, 3.312f, 0.2267f, 0.01016f},
    {6, 2, 5.035f, 0.4422f, 0.1915f, 5.155f, 0.2229f, 0.01297f},
    {4, 4, 5.432f, 0.4727f, 0.253f, 7.898f, 0.1254f, 0.02434f},
    {6, 4, 6.983f, 0.706f, 0.2364f, 8.631f, 0.1302f, 0.03006f},
};

static float mx_gemm_cost(int elem, int M, int N, int K, const MxGemmCost& c, const MxGemmPlan& pl) {
    const int xp = elem == BZ_MX_E2M1 ? 1 : 2;
    const int lds = (kMxWavesM * c.mt * xp + kMxWn * c.nt) * kMxStages;  // KiB
    const float units = 4.0f * pl.gps, full = (float)pl.l.grid / 256.0f, room = (float)(160 / lds);
    float t;
    if (room < 2.0f)
        t = (c.wg0 + units * c.unit) * (float)((pl.l.grid + 255) / 256);
    else if (full <= room)
        t = c.wg0 + units * std::max(c.unit, c.full * full);
    else
        t = (c.wg0 + units * c.full * room) * full / room;
    const float tile_mb = (float)(kMxWavesM * c.mt * kMxWn * c.nt) * 1024e-6f;
    if (pl.nsl > 1) t += c.sum0 + c.sum_mb * (float)pl.l.grid * tile_mb;
    const float w_mb = (float)N * (float)K * 0.53e-6f, x_mb = (float)M * (float)K * 0.53e-6f * xp;
    return t + c.traffic_mb * ((float)pl.mtiles * w_mb + (float)pl.ntiles * x_mb);
}

constexpr int kMxSlices[] = {1, 2, 3, 4, 6, 8};
constexpr unsigned kMxSlicedGrid = 600;  // more workgroups than this never won with slices

static int mx_gemm_plan(int elem, int M, int N, int K, int cfg, MxGemmPlan& pl) {
    const int cmt = cfg & 255, cnt = (cfg >> 8) & 255, csl = cfg >> 16;
    if (csl > 64) return BZ_ERR_INVALID_ARG;
    float best = 0.0f;
    bool found = false;
    auto look = [&](const MxGemmCost& c) -> int {
        if ((cmt && cmt != c.mt) || (cnt && cnt != c.nt)) return BZ_OK;
        for (int nsl : kMxSlices) {
            MxGemmPlan q;
            const int rc = mx_gemm_shape(M, N, K, c.mt, c.nt, csl ? csl : nsl, q);
            if (rc != BZ_OK) return rc;
            if (!csl && nsl > 1 && (q.l.grid > kMxSlicedGrid || q.nsl != nsl)) continue;
            const float t = mx_gemm_cost(elem, M, N, K, c, q);
            if (!found || t < best) {
                best = t;
                pl = q;
                found = true;
            }
            if (csl) break;
        }
        return BZ_OK;
    };
    int rc = BZ_ERR_INVALID_ARG;
    if (elem == BZ_MX_E2M1) {
        for (const MxGemmCost& c : kMxCostE2m1)
            if ((rc = look(c)) != BZ_OK) return rc;
    } else {
        for (const MxGemmCost& c : kMxCostE4m3)
            if ((rc = look(c)) != BZ_OK) return rc;
    }
    return found ? BZ_OK : BZ_ERR_INVALID_ARG;
}

static int mx_gemm_check(int elem, int M, int N, int K) {
    if (M < 1 || N < 1 || K < 1 || (elem != BZ_MX_E2M1 && elem != BZ_MX_E4M3)) return BZ_ERR_INVALID_ARG;
    if (N % 16 || K % 128) return BZ_ERR_SHAPE;
    // 32-bit offsets within a tile's rows
    return K > (1 << 22) ? BZ_ERR_UNSUPPORTED : BZ_OK;
}

}  // namespace bz

using namespace bz;

extern "C" size_t bz_mx_gemm_workspace(int32_t elem, int32_t M, int32_t N, int32_t K, int32_t cfg) {
    MxGemmPlan pl;
    if (cfg < 0 || mx_gemm_check(elem, M, N, K) != BZ_OK) return 0;
    return mx_gemm_plan(elem, M, N, K, cfg, pl) == BZ_OK ? pl.ws : 0;
}

extern "C" int bz_mx_gemm(int32_t elem, const void* xq, int32_t M, const void* w, int32_t N, int32_t K,
                          const void* residual, int32_t residual_dtype, int64_t ldr, void* out, int32_t out_dtype,
                          int64_t ldo, void* workspace, size_t workspace_bytes, int32_t cfg, void* stream) {
    if (!xq || !w || !out || cfg < 0) return BZ_ERR_INVALID_ARG;
    if (out_dtype != BZ_DT_BF16 && out_dtype != BZ_DT_F32) return BZ_ERR_INVALID_ARG;
    if (residual && residual_dtype != BZ_DT_BF16 && residual_dtype != BZ_DT_F32) return BZ_ERR_INVALID_ARG;
    const int rc = mx_gemm_check(elem, M, N, K);
    if (rc != BZ_OK) return rc;
    if (ldo < N || (residual && ldr < N)) return BZ_ERR_INVALID_ARG;
    auto off = [](const void* q, uintptr_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) != 0; };
    const int osz = out_dtype == BZ_DT_F32 ? 4 : 2, rsz = residual_dtype == BZ_DT_F32 ? 4 : 2;
    if (off(xq, 16) || off(w, 16) || off(out, osz) || (residual && off(residual, rsz))) return BZ_ERR_ALIGNMENT;
    MxGemmPlan pl;
    const int prc = mx_gemm_plan(elem, M, N, K, cfg, pl);
    if (prc != BZ_OK) return prc;
    if (pl.ws && (!workspace || off(workspace, 16) || workspace_bytes < pl.ws)) return BZ_ERR_INVALID_ARG;
    MxGemmParams p{};
    p.x = static_cast<const uint8_t*>(xq);
    p.w = static_cast<const uint8_t*>(w);
    p.res = residual;
    p.ldr = ldr;
    p.out = out;
    p.ldo = ldo;
    p.cnt = static_cast<uint32_t*>(workspace);
    p.part = pl.ws ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kMxPartOffset) : nullptr;
    p.M = M;
    p.N = N;
    p.NU = K / 128;
    p.mblk = (M + 15) / 16;
    p.nblk = N / 16;
    p.mtiles = pl.mtiles;
    p.ntiles = pl.ntiles;
    p.nsl = pl.nsl;
    p.gps = pl.gps;
    // row tiles in bands of at most 6, as even as can be
    const int bands = (pl.mtiles + 5) / 6;
    p.band = (pl.mtiles + bands - 1) / bands;
    p.res_f32 = residual_dtype == BZ_DT_F32;
    p.out_f32 = out_dtype == BZ_DT_F32;
    p.vec = !off(out, 16) && ldo * osz % 16 == 0 && (!residual || (!off(residual, 16) && ldr * rsz % 16 == 0));
    hipStream_t st = static_cast<hipStream_t>(stream);
    return elem == BZ_MX_E2M1 ? launch_mx_gemm_e2m1(p, pl.l, st) : launch_mx_gemm_e4m3(p, pl.l, st);
}
