// Microscaled blocks (bz_mx_device.h): quantising rows and reading them back.
//
// Both are one pass over memory and bound by it; a few rows by the launch.
// Measured on MI355X (kernel trace, three tensors in turn; a copy of 1 GiB
// reaches 5.2 TB/s): 10240 x 2560 fp32 to e2m1 21.3 us (5.6 TB/s), 2011 x 10240
// bf16 to e4m3 11.8 us (5.3) and back 11.2 us (5.6), tiled 12.3 us (5.1); 8192 x
// 2560 bf16 to e2m1, tiled, 10.8 us by itself (4.9), 20 behind a product whose
// 335 MB are still on their way to memory; 2 x 2560 1.5 us and back 1.6 us.
#include <algorithm>

#include "bz_mx.h"
#include "bz_mx_device.h"
#include "bz_row_runs.h"

namespace bz {

// x types: the loads of eight values and what their largest magnitude is
// found on.  bf16 keeps two values a register: magnitudes compare as 15-bit
// integers, NaN and infinity above every number.
struct MxBf16 {
    static constexpr int kBytes = 2;
    u32x4 v;
    __device__ __forceinline__ void load(const uint8_t* p) { v = ldg16(p); }
    __device__ __forceinline__ void load_any(const uint8_t* p) {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (uint32_t)h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
    }
    __device__ __forceinline__ void zero() { v = u32x4{0u, 0u, 0u, 0u}; }
    __device__ __forceinline__ float at(int i) const { return (i & 1) ? bf16_hi(v[i >> 1]) : bf16_lo(v[i >> 1]); }
    __device__ __forceinline__ uint32_t pack4(float s) const { return mx4_pack_bf16(v, s); }
    __device__ __forceinline__ void pack8(uint32_t code, float s, uint32_t& lo, uint32_t& hi) const {
        mx8_pack_bf16(v, code, s, lo, hi);
    }
};
struct MxF32 {
    static constexpr int kBytes = 4;
    float v[8];
    __device__ __forceinline__ void load(const uint8_t* p) {
        const u32x4 a = ldg16(p), b = ldg16(p + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __uint_as_float(a[i]);
            v[i + 4] = __uint_as_float(b[i]);
        }
    }
    __device__ __forceinline__ void load_any(const uint8_t* p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = reinterpret_cast<const float*>(p)[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
    __device__ __forceinline__ float at(int i) const { return v[i]; }
    __device__ __forceinline__ uint32_t pack4(float s) const { return mx4_pack_f32(v, s); }
    __device__ __forceinline__ void pack8(uint32_t, float s, uint32_t& lo, uint32_t& hi) const {
        lo = mx8_pack_f32(v[0], v[1], v[2], v[3], s);
        hi = mx8_pack_f32(v[4], v[5], v[6], v[7], s);
    }
};
struct MxF16 : MxF32 {  // (widened: exact)
    static constexpr int kBytes = 2;
    __device__ __forceinline__ void load(const uint8_t* p) {
        const u32x4 a = ldg16(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(a[i >> 1] >> (16 * (i & 1))));
    }
    __device__ __forceinline__ void load_any(const uint8_t* p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)reinterpret_cast<const _Float16*>(p)[i];
    }
};

// Largest magnitude of eight values as fp32 bits (integers in the order of
// the magnitudes, NaN on top: fmaxf would drop it).
template <class X>
__device__ __forceinline__ uint32_t mx_amax(const X& x) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x.at(i)) & 0x7FFFFFFFu);
    return m;
}

template <int ELEM>
constexpr int kMxEmax = ELEM == BZ_MX_E2M1 ? 2 : 8;

template <int ELEM, class X>
__device__ __forceinline__ void mx_store8(uint8_t* at, const X& x, uint32_t code) {
    const float s = __uint_as_float(code << 23);
    if (ELEM == BZ_MX_E2M1) {
        *reinterpret_cast<uint32_t*>(at) = x.pack4(s);
    } else {
        uint2 q;
        x.pack8(code, s, q.x, q.y);
        uint32_t* o = reinterpret_cast<uint32_t*>(at);
        o[0] = q.x;
        o[1] = q.y;
    }
}

// Row-major: eight values per lane, a block per quad of lanes, so loads and
// stores of a wave are contiguous and the largest magnitude of a block takes
// two exchanges within the quad.  One item a lane: there is nothing to keep
// from one to the next, and the grid's waves hide the loads.
template <int ELEM, class X>
__global__ void __launch_bounds__(256) mx_quantize_rows(const uint8_t* x, int64_t ldx, uint32_t items, int K8, bool vec,
                                                        uint8_t* codes, uint8_t* scales) {
    const uint32_t it = blockIdx.x * 256u + threadIdx.x;
    if (it >= items) return;  // (items % 4 == 0: a quad leaves as one)
    const uint32_t m = it / (uint32_t)K8, k8 = it - m * (uint32_t)K8;
    const uint8_t* p = x + ((int64_t)m * ldx + (int64_t)k8 * 8) * X::kBytes;
    X v;
    if (vec)  // uniform
        v.load(p);
    else
        v.load_any(p);
    uint32_t a = mx_amax(v);
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, kDppXor1, 0xF, 0xF, false));
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, kDppXor2, 0xF, 0xF, false));
    const uint32_t code = mx_code<kMxEmax<ELEM>>(a >> 23);
    mx_store8<ELEM>(codes + (int64_t)it * (ELEM == BZ_MX_E2M1 ? 4 : 8), v, code);
    if ((it & 3) == 0) scales[it >> 2] = (uint8_t)code;
}

// Tiled: a workgroup takes four units of a row block, a wave one of them, a
// lane a block (lane 16 g + r: block g of row r), so a tile is stored in one
// instruction and the four units' scale codes leave as one dword a lane, by way
// of LDS.  A lane's loads are 64 contiguous bytes, four of them a line of a
// row.  Rows past M are zeros.
template <int ELEM, class X>
__global__ void __launch_bounds__(256) mx_quantize_tiled(const uint8_t* x, int64_t ldx, int M, int NU, bool vec,
                                                         uint8_t* out, int64_t chunk, int groups) {
    __shared__ uint32_t sc[4][64];
    constexpr int TB = ELEM == BZ_MX_E2M1 ? 1024 : 2048;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int blk = blockIdx.x / groups, grp = blockIdx.x - blk * groups;
    const int u = grp * 4 + w, r = lane & 15, g = lane >> 4;
    const int m = blk * 16 + r;
    uint8_t* cb = out + blk * chunk;
    uint32_t code = 0;
    if (u < NU) {
        X v[4];
        const uint8_t* p = x + ((int64_t)m * ldx + u * 128 + g * 32) * X::kBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (m >= M)
                v[i].zero();
            else if (vec)
                v[i].load(p + i * 8 * X::kBytes);
            else
                v[i].load_any(p + i * 8 * X::kBytes);
        }
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) a = max(a, mx_amax(v[i]));
        code = mx_code<kMxEmax<ELEM>>(a >> 23);
        const float s = __uint_as_float(code << 23);
        uint8_t* t = cb + (int64_t)u * TB;
        if (ELEM == BZ_MX_E2M1) {
            *reinterpret_cast<u32x4*>(t + lane * 16) = u32x4{v[0].pack4(s), v[1].pack4(s), v[2].pack4(s), v[3].pack4(s)};
        } else {
            // the block's halves are pieces 2 g and 2 g + 1 of the row's eight
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = 2 * g + h;
                uint32_t q[4];
                v[2 * h].pack8(code, s, q[0], q[1]);
                v[2 * h + 1].pack8(code, s, q[2], q[3]);
                *reinterpret_cast<u32x4*>(t + (c >> 2) * 1024 + (16 * (c & 3) + r) * 16) = u32x4{q[0], q[1], q[2], q[3]};
            }
        }
    }
    sc[w][lane] = code;
    __syncthreads();
    if (w == 0)
        *reinterpret_cast<uint32_t*>(cb + (int64_t)NU * TB + grp * 256 + lane * 4) =
            sc[0][lane] | sc[1][lane] << 8 | sc[2][lane] << 16 | sc[3][lane] << 24;
}

// Eight elements per lane.
template <int ELEM>
__global__ void __launch_bounds__(256) mx_dequantize_rows(const uint8_t* codes, const uint8_t* scales, uint32_t items,
                                                          int K8, uint8_t* out, int64_t ldo, bool f32, bool vec) {
    const uint32_t it = blockIdx.x * 256u + threadIdx.x;
    if (it >= items) return;
    const uint32_t m = it / (uint32_t)K8, k8 = it - m * (uint32_t)K8;
    const float s = __uint_as_float((uint32_t)scales[it >> 2] << 23);
    float v[8];
    u32x4 b;
    if (ELEM == BZ_MX_E2M1) {
        const uint32_t q = reinterpret_cast<const uint32_t*>(codes)[it];
        if (f32) {
            typedef float f2 __attribute__((ext_vector_type(2)));
            const f2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 1);
            const f2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 3);
            v[0] = p0[0], v[1] = p0[1], v[2] = p1[0], v[3] = p1[1], v[4] = p2[0], v[5] = p2[1], v[6] = p3[0], v[7] = p3[1];
        } else {
            b = mx4_weights(q, s);
        }
    } else {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(codes) + 2 * (int64_t)it;
        if (f32) {
            typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[h], s, false);
                const f2 hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[h], s, true);
                v[4 * h] = lo[0], v[4 * h + 1] = lo[1], v[4 * h + 2] = hi[0], v[4 * h + 3] = hi[1];
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                b[2 * h] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[h], s, false));
                b[2 * h + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[h], s, true));
            }
        }
    }
    const int64_t o = (int64_t)m * ldo + (int64_t)k8 * 8;
    if (f32) {
        float* p = reinterpret_cast<float*>(out) + o;
        if (vec) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = v[i];
        }
    } else {
        uint16_t* p = reinterpret_cast<uint16_t*>(out) + o;
        if (vec) {
            *reinterpret_cast<u32x4*>(p) = b;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = (uint16_t)(b[i >> 1] >> (16 * (i & 1)));
        }
    }
}

static bool mx_elem_ok(int elem) { return elem == BZ_MX_E2M1 || elem == BZ_MX_E4M3; }
static bool off(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }
static int launched() { return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH; }

template <int ELEM, class X>
static int launch_quantize(const void* x, int64_t ldx, int M, int K, int layout, void* codes, void* scales,
                           hipStream_t st) {
    const uint8_t* xp = static_cast<const uint8_t*>(x);
    const bool vec = !off(x, 16) && (ldx * X::kBytes) % 16 == 0;
    if (layout == BZ_MX_TILED) {
        const int NU = K / 128, groups = (NU + 3) / 4;
        const int64_t grid = (int64_t)((M + 15) / 16) * groups;
        if (grid * 256 >= (int64_t)1 << 32) return BZ_ERR_UNSUPPORTED;
        const int64_t chunk = ELEM == BZ_MX_E2M1 ? mx4_chunk_bytes(NU) : mx8_chunk_bytes(NU);
        hipLaunchKernelGGL((mx_quantize_tiled<ELEM, X>), dim3((unsigned)grid), dim3(256), 0, st, xp, ldx, M, NU, vec,
                           static_cast<uint8_t*>(codes), chunk, groups);
        return launched();
    }
    const int64_t row_codes = ELEM == BZ_MX_E2M1 ? K / 2 : K;
    return for_row_runs(M, K, [&](int64_t m0, int rows) {
        const uint32_t items = (uint32_t)rows * (uint32_t)(K / 8);
        hipLaunchKernelGGL((mx_quantize_rows<ELEM, X>), dim3((items + 255) / 256), dim3(256), 0, st,
                           xp + m0 * ldx * X::kBytes, ldx, items, K / 8, vec,
                           static_cast<uint8_t*>(codes) + m0 * row_codes, static_cast<uint8_t*>(scales) + m0 * (K / 32));
        return launched();
    });
}

template <int ELEM>
static int quantize_elem(const void* x, int dt, int64_t ldx, int M, int K, int layout, void* codes, void* scales,
                         hipStream_t st) {
    if (dt == BZ_DT_F32) return launch_quantize<ELEM, MxF32>(x, ldx, M, K, layout, codes, scales, st);
    if (dt == BZ_MX_F16) return launch_quantize<ELEM, MxF16>(x, ldx, M, K, layout, codes, scales, st);
    return launch_quantize<ELEM, MxBf16>(x, ldx, M, K, layout, codes, scales, st);
}

}  // namespace bz

using namespace bz;

extern "C" size_t bz_mx_rows_bytes(int32_t elem, int32_t M, int32_t K) {
    if (!mx_elem_ok(elem) || M < 1 || K < 1 || K % 128) return 0;
    const int NU = K / 128;
    return (size_t)((M + 15) / 16) * (size_t)(elem == BZ_MX_E2M1 ? mx4_chunk_bytes(NU) : mx8_chunk_bytes(NU));
}

extern "C" int bz_mx_quantize(const void* x, int32_t x_dtype, int64_t ldx, int32_t M, int32_t K, int32_t elem,
                              int32_t layout, void* codes, void* scales, void* stream) {
    if (!x || !codes || M < 1 || K < 1 || ldx < K || !mx_elem_ok(elem)) return BZ_ERR_INVALID_ARG;
    if (x_dtype != BZ_DT_BF16 && x_dtype != BZ_DT_F32 && x_dtype != BZ_MX_F16) return BZ_ERR_INVALID_ARG;
    if (layout != BZ_MX_ROWS && layout != BZ_MX_TILED) return BZ_ERR_INVALID_ARG;
    if ((layout == BZ_MX_ROWS) != (scales != nullptr)) return BZ_ERR_INVALID_ARG;
    if (K % (layout == BZ_MX_TILED ? 128 : 32)) return BZ_ERR_SHAPE;
    if (off(x, x_dtype == BZ_DT_F32 ? 4 : 2) || off(codes, layout == BZ_MX_TILED ? 16 : 4)) return BZ_ERR_ALIGNMENT;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return elem == BZ_MX_E2M1 ? quantize_elem<BZ_MX_E2M1>(x, x_dtype, ldx, M, K, layout, codes, scales, st)
                              : quantize_elem<BZ_MX_E4M3>(x, x_dtype, ldx, M, K, layout, codes, scales, st);
}

extern "C" int bz_mx_dequantize(const void* codes, const void* scales, int32_t elem, int32_t M, int32_t K, void* out,
                                int32_t out_dtype, int64_t ldo, void* stream) {
    if (!codes || !scales || !out || M < 1 || K < 1 || ldo < K || !mx_elem_ok(elem)) return BZ_ERR_INVALID_ARG;
    if (out_dtype != BZ_DT_BF16 && out_dtype != BZ_DT_F32) return BZ_ERR_INVALID_ARG;
    if (K % 32) return BZ_ERR_SHAPE;
    const bool f32 = out_dtype == BZ_DT_F32;
    if (off(codes, 4) || off(out, f32 ? 4 : 2)) return BZ_ERR_ALIGNMENT;
    const bool vec = !off(out, 16) && (ldo * (f32 ? 4 : 2)) % 16 == 0;
    const int64_t row_codes = elem == BZ_MX_E2M1 ? K / 2 : K;
    return for_row_runs(M, K, [&](int64_t m0, int rows) {
        const uint32_t items = (uint32_t)rows * (uint32_t)(K / 8);
        auto kern = elem == BZ_MX_E2M1 ? mx_dequantize_rows<BZ_MX_E2M1> : mx_dequantize_rows<BZ_MX_E4M3>;
        hipLaunchKernelGGL(kern, dim3((items + 255) / 256), dim3(256), 0, static_cast<hipStream_t>(stream),
                           static_cast<const uint8_t*>(codes) + m0 * row_codes,
                           static_cast<const uint8_t*>(scales) + m0 * (K / 32), items, K / 8,
                           static_cast<uint8_t*>(out) + m0 * ldo * (f32 ? 4 : 2), ldo, f32, vec);
        return launched();
    });
}
