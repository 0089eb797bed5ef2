// New tokens into a paged key/value cache (include/bz_paged.h): per-head q/k
// RMSNorm, rotate-half RoPE, keys and values into their pages, queries out.
//
// For head vector x of row t at rotary row r (all in fp32):
//   y = x / sqrt(mean(x^2) + eps) * w            (q and k heads, with norms)
//   z_d = y_d cos[r][d] - y_{d + D/2} sin[r][d]  for d < D/2
//   z_d = y_d cos[r][d] + y_{d - D/2} sin[r][d]  for d >= D/2
// q out and a bf16 cache round z (a value head: x itself) once; an e4m3 cache
// rounds z / scale, or x / scale, saturated at 448, once.
//
// Bound by HBM, ((HQ + 2 HKV) D 2 + HQ D 2 + 2 HKV D es) bytes a row, or for few
// rows by the chain starts -> length -> page -> store.  A thread holds 8 elements
// of each half of a head: the rotary partner is its own, every access is 16
// bytes (8 into an e4m3 cache), and a head's sum of squares is 2 to 4 DPP steps over
// the D / 16 threads of the head.  Measured: seven prompts of 33 .. 611 tokens, bf16, 16 / 4 heads
// of 256, 14.6 us (4.6 TB/s), a chunk of 8191 tokens into e4m3, 16 / 8 heads of 128, 27.1 (4.7 TB/s;
// 5.2 is what a large copy reaches), two rows 2.9.
#include "bz_paged_kv.h"

namespace bz {

constexpr int kPagedRopeThreads = 256;

struct PagedRope {
    const uint16_t* qkv;
    int64_t ld_qkv;
    const uint16_t* qn;
    const uint16_t* kn;
    float eps;
    const void* cos;
    const void* sin;
    int64_t ld_cs, cs_rows;
    const int64_t* positions;
    uint16_t* q_out;
    int64_t ld_q;
};

__device__ __forceinline__ void widen8(const uint16_t* p, float (&v)[8]) {
    const u32x4 w = ldg16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_lo(w[i]);
        v[2 * i + 1] = bf16_hi(w[i]);
    }
}
__device__ __forceinline__ void widen8(const float* p, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const u32x4 w = ldg16(p + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * i + e] = __uint_as_float(w[e]);
    }
}

__device__ __forceinline__ u32x4 narrow8(const float (&v)[8]) {
    return u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}

// value / scale as e4m3, round to nearest even, saturated at 448; NaN stays NaN.
__device__ __forceinline__ float f8_range(float v, float scale) {
    const float q = v / scale;
    return q != q ? q : fminf(fmaxf(q, -448.0f), 448.0f);
}
__device__ __forceinline__ uint2 narrow8_f8(const float (&v)[8], float scale) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int t = __builtin_amdgcn_cvt_pk_fp8_f32(f8_range(v[4 * i], scale), f8_range(v[4 * i + 1], scale), 0, false);
        t = __builtin_amdgcn_cvt_pk_fp8_f32(f8_range(v[4 * i + 2], scale), f8_range(v[4 * i + 3], scale), t, true);
        w[i] = (uint32_t)t;
    }
    return make_uint2(w[0], w[1]);
}

template <int D, bool F8, typename CS>
__global__ void __launch_bounds__(kPagedRopeThreads) paged_qkv_rope_cache_kernel(PagedKv c, PagedRope a) {
    constexpr int LPH = D / 16;  // threads of a head
    const int t = blockIdx.x, tid = threadIdx.x;
    const int h = blockIdx.y * (kPagedRopeThreads / LPH) + tid / LPH, i = tid % LPH;
    const int heads = c.HQ + 2 * c.HKV;
    const int lo = 8 * i, hi = D / 2 + 8 * i;  // the thread's elements

    const uint16_t* row = a.qkv + (int64_t)t * a.ld_qkv + (int64_t)min(h, heads - 1) * D;
    float x[8], y[8];
    widen8(row + lo, x);
    widen8(row + hi, y);

    const int b = seq_of_row(c, t, tid & 63);
    if (b >= c.B) return;
    const RowRange r = seq_rows(c, b);
    if (t < r.first || t >= r.end) return;
    const int pos = max(c.kv_lens[b], 0) - (r.end - t);
    const int64_t at = a.positions ? a.positions[t] : pos;
    const bool turned = at >= 0 && at < a.cs_rows;
    if (h >= heads) return;
    const bool is_q = h < c.HQ, is_v = h >= c.HQ + c.HKV;

    char* dst = nullptr;
    int head = 0;
    if (!is_q) {
        if (!turned || pos < 0 || (pos >> c.shift) >= c.width) return;
        const int page = c.table[(int64_t)b * c.ld_table + (pos >> c.shift)];
        if ((unsigned)page >= (unsigned)c.num_pages) return;
        const int in_page = pos & ((1 << c.shift) - 1);
        head = h - c.HQ - (is_v ? c.HKV : 0);
        dst = is_v ? c.v + page * c.v_page + head * c.v_head + in_page * c.v_pos
                   : c.k + page * c.k_page + head * c.k_head + in_page * c.k_pos;
    }
    if (!is_v) {
        if (a.qn) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[e] * x[e] + y[e] * y[e];
            ss = LPH == 4 ? sum4(ss) : (LPH == 8 ? sum8(ss) : sum16_dpp(ss));
            const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
            const uint16_t* w = is_q ? a.qn : a.kn;
            float wx[8], wy[8];
            widen8(w + lo, wx);
            widen8(w + hi, wy);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = x[e] * inv * wx[e];
                y[e] = y[e] * inv * wy[e];
            }
        }
        if (turned) {
            const CS* cp = static_cast<const CS*>(a.cos) + at * a.ld_cs;
            const CS* sp = static_cast<const CS*>(a.sin) + at * a.ld_cs;
            float cx[8], cy[8], sx[8], sy[8];
            widen8(cp + lo, cx);
            widen8(cp + hi, cy);
            widen8(sp + lo, sx);
            widen8(sp + hi, sy);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = x[e] * cx[e] - y[e] * sx[e];
                y[e] = y[e] * cy[e] + x[e] * sy[e];
                x[e] = p;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.0f;
        }
    }
    if (is_q) {
        uint16_t* q = a.q_out + (int64_t)t * a.ld_q + (int64_t)h * D;
        *reinterpret_cast<u32x4*>(q + lo) = narrow8(x);
        *reinterpret_cast<u32x4*>(q + hi) = narrow8(y);
    } else if constexpr (F8) {
        const float scale = (is_v ? c.v_scale : c.k_scale)[head];
        *reinterpret_cast<uint2*>(dst + lo) = narrow8_f8(x, scale);
        *reinterpret_cast<uint2*>(dst + hi) = narrow8_f8(y, scale);
    } else {
        *reinterpret_cast<u32x4*>(dst + 2 * lo) = narrow8(x);
        *reinterpret_cast<u32x4*>(dst + 2 * hi) = narrow8(y);
    }
}

template <int D, bool F8>
static void launch_rope(const PagedKv& c, const PagedRope& a, bool cs_f32, hipStream_t st) {
    const int per = kPagedRopeThreads / (D / 16);
    const dim3 grid(c.T, (c.HQ + 2 * c.HKV + per - 1) / per);
    if (cs_f32)
        hipLaunchKernelGGL((paged_qkv_rope_cache_kernel<D, F8, float>), grid, dim3(kPagedRopeThreads), 0, st, c, a);
    else
        hipLaunchKernelGGL((paged_qkv_rope_cache_kernel<D, F8, uint16_t>), grid, dim3(kPagedRopeThreads), 0, st, c, a);
}

}  // namespace bz

using namespace bz;

extern "C" int bz_paged_rope_cache(const bz_paged_kv* kv, const void* qkv, int64_t ld_qkv, const void* q_norm,
                                   const void* k_norm, float eps, const void* cos, const void* sin, int32_t cs_dtype,
                                   int64_t ld_cs, int64_t cs_rows, const int64_t* positions, void* q_out, int64_t ld_q,
                                   void* stream) {
    PagedKv c = {};
    const int rc = paged_setup(kv, c);
    if (rc != BZ_OK) return rc;
    if (kv->T >= kPagedMaxGrid) return BZ_ERR_UNSUPPORTED;
    if (!qkv || !cos || !sin || !q_out || (q_norm == nullptr) != (k_norm == nullptr)) return BZ_ERR_INVALID_ARG;
    if (cs_dtype != BZ_DT_BF16 && cs_dtype != BZ_DT_F32) return BZ_ERR_INVALID_ARG;
    const int D = kv->D;
    if (ld_qkv < (int64_t)(c.HQ + 2 * c.HKV) * D || ld_q < (int64_t)c.HQ * D || ld_cs < D || cs_rows < 1)
        return BZ_ERR_SHAPE;
    if (!aligned_to(qkv, 16) || !aligned_to(q_out, 16) || !aligned_to(cos, 16) || !aligned_to(sin, 16) ||
        !aligned_to(q_norm, 16) || !aligned_to(k_norm, 16) || !aligned_to(positions, 8) || ld_qkv % 8 || ld_q % 8 ||
        ld_cs % 8)
        return BZ_ERR_ALIGNMENT;
    const PagedRope a = {static_cast<const uint16_t*>(qkv),
                         ld_qkv,
                         static_cast<const uint16_t*>(q_norm),
                         static_cast<const uint16_t*>(k_norm),
                         eps,
                         cos,
                         sin,
                         ld_cs,
                         cs_rows,
                         positions,
                         static_cast<uint16_t*>(q_out),
                         ld_q};
    const bool f8 = kv->kv_dtype == BZ_KV_E4M3, cs_f32 = cs_dtype == BZ_DT_F32;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: f8 ? launch_rope<64, true>(c, a, cs_f32, st) : launch_rope<64, false>(c, a, cs_f32, st); break;
        case 128: f8 ? launch_rope<128, true>(c, a, cs_f32, st) : launch_rope<128, false>(c, a, cs_f32, st); break;
        default: f8 ? launch_rope<256, true>(c, a, cs_f32, st) : launch_rope<256, false>(c, a, cs_f32, st); break;
    }
    return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}
