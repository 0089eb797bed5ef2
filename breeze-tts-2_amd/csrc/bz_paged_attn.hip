// Attention of each sequence's newest rows over a paged key/value cache
// (include/bz_paged.h), with shared prefixes.
//
//   s_j = scale q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max_j s_j
//
// over the keys a row attends, in one pass: with m the maximum so far, the sum l
// and the accumulator are rescaled by e^(m_old - m) as m grows (kept as exponents
// of 2, scale log2(e) s).  The simple form: a wave per (row, query head), a key
// per lane for the scores, D / 64 columns per lane for the values.
#include "bz_paged_kv.h"

namespace bz {

constexpr float kLog2e = 1.4426950408889634f;

template <int D, bool F8>
__global__ void __launch_bounds__(256) paged_attn_bf16_row(PagedKv c, const uint16_t* q, int64_t ld_q, float scale,
                                                           uint16_t* out, int64_t ld_out) {
    constexpr int DL = D / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x, h = blockIdx.y * 4 + wave;
    const int b = seq_of_row(c, t, lane);
    if (b >= c.B) return;
    const RowRange r = seq_rows(c, b);
    if (t < r.first || t >= r.end || h >= c.HQ) return;
    const int head = h / c.G;
    const int pos = max(c.kv_lens[b], 0) - (r.end - t);
    int group = -1;
    if (c.groups > 0) {
        int g = 0;
        if (c.prefix_seqs)
            for (; g < c.groups; ++g)
                if (c.prefix_seqs[g] <= b && b < c.prefix_seqs[g + 1]) break;
        if (g < c.groups) group = g;
    }
    const float ks = F8 ? c.k_scale[head] : 1.0f;
    const uint16_t* qr = q + (int64_t)t * ld_q + (int64_t)h * D;
    float m = -INFINITY, l = 0.0f, acc[DL] = {};
    bool seen = false;
    for (int part = 0; part < 2; ++part) {
        const int32_t* table = part ? c.table + (int64_t)b * c.ld_table : c.prefix_table + (int64_t)group * c.ld_prefix;
        int n = 0;
        if (part)
            n = min(pos + 1, c.width << c.shift);
        else if (group >= 0)
            n = min(c.prefix_lens[group], c.prefix_width << c.shift);
        for (int j0 = 0; j0 < n; j0 += 64) {
            const int j = j0 + lane;
            const int page = j < n ? table[j >> c.shift] : -1;
            const bool there = (unsigned)page < (unsigned)c.num_pages;
            const int at = j & ((1 << c.shift) - 1);
            float s = -INFINITY;
            if (there) {
                const char* kr = c.k + page * c.k_page + head * c.k_head + at * c.k_pos;
                s = 0.0f;
                for (int d = 0; d < D; ++d) {
                    float kv;
                    if constexpr (F8)
                        kv = __builtin_amdgcn_cvt_f32_fp8((int)reinterpret_cast<const uint8_t*>(kr)[d], 0);
                    else
                        kv = bf16_to_f32(reinterpret_cast<const uint16_t*>(kr)[d]);
                    s += bf16_to_f32(qr[d]) * kv;
                }
                s = s * ks * scale * kLog2e;
            }
            const float mn = fmaxf(m, wave_max(s));
            const float ms = mn == -INFINITY ? 0.0f : mn;
            const float f = exp2f(m - ms), p = there ? exp2f(s - ms) : 0.0f;
            m = mn;
            l = l * f + wave_sum(p);
            for (int e = 0; e < DL; ++e) acc[e] *= f;
            uint64_t live = __ballot(there);
            seen |= live != 0;
            for (; live; live &= live - 1) {
                const int k = __builtin_ctzll(live);
                const float pk = __shfl(p, k, 64);
                const int pg = __shfl(page, k, 64), ak = (j0 + k) & ((1 << c.shift) - 1);
                const char* vr = c.v + pg * c.v_page + head * c.v_head + ak * c.v_pos;
                for (int e = 0; e < DL; ++e) {
                    float v;
                    if constexpr (F8)
                        v = __builtin_amdgcn_cvt_f32_fp8((int)reinterpret_cast<const uint8_t*>(vr)[DL * lane + e], 0);
                    else
                        v = bf16_to_f32(reinterpret_cast<const uint16_t*>(vr)[DL * lane + e]);
                    acc[e] += pk * v;
                }
            }
        }
    }
    const float vs = F8 ? c.v_scale[head] : 1.0f;
    for (int e = 0; e < DL; ++e)
        out[(int64_t)t * ld_out + (int64_t)h * D + DL * lane + e] = f32_to_bf16(seen ? acc[e] / l * vs : 0.0f);
}

template <bool F8>
static void launch_paged(int D, const PagedKv& c, const uint16_t* q, int64_t ld_q, float scale, uint16_t* out,
                         int64_t ld_out, hipStream_t st) {
    const dim3 grid(c.T, (c.HQ + 3) / 4), block(256);
    switch (D) {
        case 64:
            hipLaunchKernelGGL((paged_attn_bf16_row<64, F8>), grid, block, 0, st, c, q, ld_q, scale, out, ld_out);
            break;
        case 128:
            hipLaunchKernelGGL((paged_attn_bf16_row<128, F8>), grid, block, 0, st, c, q, ld_q, scale, out, ld_out);
            break;
        default:
            hipLaunchKernelGGL((paged_attn_bf16_row<256, F8>), grid, block, 0, st, c, q, ld_q, scale, out, ld_out);
    }
}

}  // namespace bz

using namespace bz;

extern "C" size_t bz_paged_attn_workspace(const bz_paged_kv* kv) {
    if (paged_check_sizes(kv) != BZ_OK) return 0;
    return 0;
}

extern "C" int bz_paged_attn(const bz_paged_kv* kv, const void* q, int64_t ld_q, float scale, void* workspace,
                             size_t workspace_bytes, void* out, int64_t ld_out, void* stream) {
    PagedKv c = {};
    const int rc = paged_setup(kv, c);
    if (rc != BZ_OK) return rc;
    if (!q || !out || !(scale > 0.0f) || scale > 3.0e38f) return BZ_ERR_INVALID_ARG;
    const int D = kv->D;
    if (ld_q < (int64_t)c.HQ * D || ld_out < (int64_t)c.HQ * D) return BZ_ERR_SHAPE;
    if (!aligned_to(q, 16) || !aligned_to(out, 16) || ld_q % 8 || ld_out % 8) return BZ_ERR_ALIGNMENT;
    const size_t need = bz_paged_attn_workspace(kv);
    if (need && (!workspace || workspace_bytes < need)) return BZ_ERR_INVALID_ARG;
    if (!aligned_to(workspace, 16)) return BZ_ERR_ALIGNMENT;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const uint16_t* qp = static_cast<const uint16_t*>(q);
    uint16_t* op = static_cast<uint16_t*>(out);
    if (kv->kv_dtype == BZ_KV_E4M3)
        launch_paged<true>(D, c, qp, ld_q, scale, op, ld_out, st);
    else
        launch_paged<false>(D, c, qp, ld_q, scale, op, ld_out, st);
    return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}
