// Products of microscaled rows with a microscaled 4-bit weight (bz_mx_device.h
// has layouts and formats): out[M, N] = q(x) @ w_eff^T (+ residual).
//
// Arithmetic: v_mfma_scale_f32_16x16x128_f8f6f4, A = 16 weight rows, B = 16
// rows of x, each lane with one block of 32 k and its scale code; D[n][m]
// lands in lane m + 16 (n / 4), element n % 4, so a lane finishes four
// consecutive columns of one output row.  The products of elements and the
// two powers of two are exact; sums are fp32.
#include "bz_mx.h"
#include "bz_mx_device.h"

namespace bz {

typedef int mx_op_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct MxGemmParams {
    const uint8_t* x;
    const uint8_t* w;
    const void* res;
    int64_t ldr;
    void* out;
    int64_t ldo;
    int M, NU, mblk, nblk;
    int res_f32, out_f32;  // res NULL: none
};

template <int ELEM, int U>
__device__ __forceinline__ f32x4_t mx_mfma(mx_op_t w, mx_op_t x, f32x4_t c, uint32_t sw, uint32_t sx) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, ELEM == BZ_MX_E2M1 ? 4 : 0, U, (int)sw, U,
                                                            (int)sx);
}

// One wave per 16 rows of x and 16 of the weight, operands from memory.
template <int ELEM>
__global__ void __launch_bounds__(256) mx_gemm(MxGemmParams p) {
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (int64_t)p.mblk * p.nblk) return;
    const int nb = (int)(id / p.mblk), mb = (int)(id - (int64_t)nb * p.mblk);
    constexpr int TB = ELEM == BZ_MX_E2M1 ? 1024 : 2048;
    const int64_t xchunk = ELEM == BZ_MX_E2M1 ? mx4_chunk_bytes(p.NU) : mx8_chunk_bytes(p.NU);
    const uint8_t* xb = p.x + mb * xchunk;
    const uint8_t* wb = p.w + nb * mx4_chunk_bytes(p.NU);
    const __amdgpu_buffer_rsrc_t xr = buffer_rsrc(xb, (uint32_t)p.NU * TB), wr = buffer_rsrc(wb, (uint32_t)p.NU * 1024u);
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int u = 0; u < p.NU; u += 4) {  // tiles past the row read as zeros
        const uint32_t sx = *reinterpret_cast<const uint32_t*>(xb + (int64_t)p.NU * TB + mx_scale_offset(u, lane));
        const uint32_t sw = *reinterpret_cast<const uint32_t*>(wb + (int64_t)p.NU * 1024 + mx_scale_offset(u, lane));
        mx_op_t xo[4], wo[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const u32x4 a = buffer_ld16(wr, (uint32_t)(u + q) * 1024u + lane * 16);
            const u32x4 b = buffer_ld16(xr, (uint32_t)(u + q) * TB + lane * 16);
            u32x4 c = {0u, 0u, 0u, 0u};
            if (ELEM == BZ_MX_E4M3) c = buffer_ld16(xr, (uint32_t)(u + q) * TB + 1024 + lane * 16);
            wo[q] = mx_op_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
            xo[q] = mx_op_t{(int)b[0], (int)b[1], (int)b[2], (int)b[3], (int)c[0], (int)c[1], (int)c[2], (int)c[3]};
        }
        acc = mx_mfma<ELEM, 0>(wo[0], xo[0], acc, sw, sx);
        acc = mx_mfma<ELEM, 1>(wo[1], xo[1], acc, sw, sx);
        acc = mx_mfma<ELEM, 2>(wo[2], xo[2], acc, sw, sx);
        acc = mx_mfma<ELEM, 3>(wo[3], xo[3], acc, sw, sx);
    }
    const int m = mb * 16 + (lane & 15), c = nb * 16 + 4 * (lane >> 4);
    if (m >= p.M) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float v = acc[q];
        if (p.res)
            v += p.res_f32 ? reinterpret_cast<const float*>(p.res)[(int64_t)m * p.ldr + c + q]
                           : bf16_to_f32(reinterpret_cast<const uint16_t*>(p.res)[(int64_t)m * p.ldr + c + q]);
        if (p.out_f32)
            reinterpret_cast<float*>(p.out)[(int64_t)m * p.ldo + c + q] = v;
        else
            reinterpret_cast<uint16_t*>(p.out)[(int64_t)m * p.ldo + c + q] = f32_to_bf16(v);
    }
}

}  // namespace bz

using namespace bz;

extern "C" int bz_mx_gemm(int32_t elem, const void* xq, int32_t M, const void* w, int32_t N, int32_t K,
                          const void* residual, int32_t residual_dtype, int64_t ldr, void* out, int32_t out_dtype,
                          int64_t ldo, void* stream) {
    if (!xq || !w || !out || M < 1 || N < 1 || K < 1 || ldo < N) return BZ_ERR_INVALID_ARG;
    if (elem != BZ_MX_E2M1 && elem != BZ_MX_E4M3) return BZ_ERR_INVALID_ARG;
    if (out_dtype != BZ_DT_BF16 && out_dtype != BZ_DT_F32) return BZ_ERR_INVALID_ARG;
    if (residual && ((residual_dtype != BZ_DT_BF16 && residual_dtype != BZ_DT_F32) || ldr < N)) return BZ_ERR_INVALID_ARG;
    if (N % 16 || K % 128) return BZ_ERR_SHAPE;
    auto off = [](const void* q, uintptr_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) != 0; };
    if (off(xq, 16) || off(w, 16) || off(out, out_dtype == BZ_DT_F32 ? 4 : 2) ||
        (residual && off(residual, residual_dtype == BZ_DT_F32 ? 4 : 2)))
        return BZ_ERR_ALIGNMENT;
    MxGemmParams p{};
    p.x = static_cast<const uint8_t*>(xq);
    p.w = static_cast<const uint8_t*>(w);
    p.res = residual;
    p.ldr = ldr;
    p.out = out;
    p.ldo = ldo;
    p.M = M;
    p.NU = K / 128;
    p.mblk = (M + 15) / 16;
    p.nblk = N / 16;
    p.res_f32 = residual_dtype == BZ_DT_F32;
    p.out_f32 = out_dtype == BZ_DT_F32;
    const int64_t waves = (int64_t)p.mblk * p.nblk, grid = (waves + 3) / 4;
    if (grid * 256 >= (int64_t)1 << 32) return BZ_ERR_UNSUPPORTED;
    auto kern = elem == BZ_MX_E2M1 ? mx_gemm<BZ_MX_E2M1> : mx_gemm<BZ_MX_E4M3>;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), 0, static_cast<hipStream_t>(stream), p);
    return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}
