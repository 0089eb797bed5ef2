// Host side of the products of microscaled rows (C ABI entries bz_mx_gemm and
// bz_mx_gemm_workspace).
#include <algorithm>

#include "bz_mx_gemm.h"
#include "bz_plans.h"

namespace bz {

struct MxGemmPlan {
    MxGemmLaunch l;
    int mtiles, ntiles, nsl, gps;
    size_t ws;
};

static int mx_gemm_shape(int M, int N, int K, int tm32, int tn64, int nsl, MxGemmPlan& pl) {
    const int mblk = (M + 15) / 16, nblk = N / 16, groups = (K / 128 + 3) / 4;
    const int tm = 2 * tm32, tn = 4 * tn64;
    pl.l.tm = tm32;
    pl.l.tn = tn64;
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
// the smallest: a workgroup's start and end (wg0) and its units, which take the
// longer of one workgroup's time (unit) and, where several fit a CU, of the
// CU's for all it holds (full each); the workspace's traffic where K is sliced;
// and reading x and the weight for every tile.  Workgroups come in whole rounds
// over the 256 CUs; where one fills a CU, the last round's are spread a little
// (0.2 of it counts by its share).  Fitted to graph replays over 15 (N, K) (the
// model's layers, 1024 squared, 656 x 384, 4800 x 640 and 7408 x 3968), M = 33
// .. 2048 and 1 .. 8 slices on MI355X, 6169 timings.  Over those the shape it
// picks takes 1.0% (e2m1) / 0.3% (e4m3) longer than the best one on average, at
// worst 20% (M = 400, N 2560, K 10240: 22.3 us for 18.6) / 7%.
struct MxGemmCost {
    int tm, tn;
    float wg0, unit, full, sum0, sum_mb, traffic_mb;
};
constexpr MxGemmCost kMxCostE2m1[] = {
    {1, 2, 3.492f, 0.1442f, 0.1346f, 2.414f, 0.2298f, 0.01163f},
    {2, 2, 3.798f, 0.1564f, 0.1414f, 2.791f, 0.2351f, 0.01697f},
    {4, 2, 4.336f, 0.2222f, 0.2074f, 2.97f, 0.269f, 0.01945f},
    {6, 2, 5.324f, 0.2988f, 0.294f, 3.458f, 0.2343f, 0.02057f},
    {4, 4, 5.804f, 0.3463f, 0.0f, 5.006f, 0.2019f, 0.01741f},
    {8, 4, 8.683f, 0.5218f, 0.0f, 9.015f, 0.1578f, 0.03885f},
};
constexpr MxGemmCost kMxCostE4m3[] = {
    {1, 2, 3.503f, 0.1696f, 0.14f, 2.381f, 0.2329f, 0.01058f},
    {2, 2, 3.774f, 0.1825f, 0.1605f, 2.503f, 0.295f, 0.01348f},
    {4, 2, 4.103f, 0.3225f, 0.0f, 3.248f, 0.2535f, 0.009315f},
    {6, 2, 4.817f, 0.4247f, 0.0f, 3.577f, 0.236f, 0.01382f},
    {4, 4, 5.961f, 0.4698f, 0.0f, 5.354f, 0.1974f, 0.02202f},
    {6, 4, 7.125f, 0.7275f, 0.0f, 7.692f, 0.1409f, 0.02822f},
};

static float mx_gemm_cost(int elem, int M, int N, int K, const MxGemmCost& c, const MxGemmPlan& pl) {
    const int xp = elem == BZ_MX_E2M1 ? 1 : 2;
    const int lds = (2 * c.tm * xp + 4 * c.tn) * kMxStages;  // KiB
    const int room = 160 / lds;                              // workgroups on a CU
    const float units = 4.0f * pl.gps, rounds = (float)((pl.l.grid + 255) / 256);
    float t;
    if (room < 2)
        t = (c.wg0 + units * c.unit) * (0.8f * rounds + 0.2f * std::max(1.0f, (float)pl.l.grid / 256.0f));
    else if (rounds <= (float)room)
        t = c.wg0 + units * std::max(c.unit, c.full * rounds);
    else
        t = (c.wg0 + units * c.full * (float)room) * rounds / (float)room;
    const float tile_mb = (float)(8 * c.tm * c.tn) * 1024e-6f;
    if (pl.nsl > 1) t += c.sum0 + c.sum_mb * (float)pl.l.grid * tile_mb;
    const float w_mb = (float)N * (float)K * 0.53e-6f, x_mb = (float)M * (float)K * 0.53e-6f * xp;
    return t + c.traffic_mb * ((float)pl.mtiles * w_mb + (float)pl.ntiles * x_mb);
}

constexpr int kMxSlices[] = {1, 2, 3, 4, 6, 8};
constexpr unsigned kMxSlicedGrid = 600;  // more workgroups than this never won with slices

static int mx_gemm_choose(int elem, int M, int N, int K, int cfg, MxGemmPlan& pl) {
    const int ctm = cfg & 255, ctn = (cfg >> 8) & 255, csl = cfg >> 16;
    if (csl > 64) return BZ_ERR_INVALID_ARG;
    float best = 0.0f;
    bool found = false;
    int rc = BZ_ERR_INVALID_ARG;
    auto look = [&](const MxGemmCost& c) {
        if ((ctm && ctm != c.tm) || (ctn && ctn != c.tn)) return;
        for (int nsl : kMxSlices) {
            MxGemmPlan q;
            if (mx_gemm_shape(M, N, K, c.tm, c.tn, csl ? csl : nsl, q) != BZ_OK) {
                rc = BZ_ERR_UNSUPPORTED;  // (too many workgroups: a larger tile may do)
                continue;
            }
            if (!csl && nsl > 1 && (q.l.grid > kMxSlicedGrid || q.nsl != nsl)) continue;
            const float t = mx_gemm_cost(elem, M, N, K, c, q);
            if (!found || t < best) {
                best = t;
                pl = q;
                found = true;
            }
            if (csl) break;
        }
    };
    if (elem == BZ_MX_E2M1)
        for (const MxGemmCost& c : kMxCostE2m1) look(c);
    else
        for (const MxGemmCost& c : kMxCostE4m3) look(c);
    return found ? BZ_OK : rc;
}

static int mx_gemm_plan(int elem, int M, int N, int K, int cfg, MxGemmPlan& pl) {
    return planned(PlanKey{elem, M, N, K, cfg}, pl, [&](MxGemmPlan& q) { return mx_gemm_choose(elem, M, N, K, cfg, q); });
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
