// Attention over a paged key/value cache: parameters and the kernels' common parts.
//
//   s_j = scale q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max_j s_j
//
// over the keys a row attends, in one pass: with m the maximum so far, the sum l
// and the accumulator are rescaled by e^(m_old - m) as m grows, in exponents of
// 2 of scale log2(e) s and in fp32.  A row of which a slot holds no key has m = -inf
// there; l is then 1 if it attends keys of it, all with a score of -inf (if that
// holds for all its keys the softmax is 0 / 0: NaN), and 0 if it attends none.
#pragma once

#include "bz_paged_plan.h"

namespace bz {

typedef __bf16 pg_bf16x8 __attribute__((ext_vector_type(8)));
typedef float pg_f32x4 __attribute__((ext_vector_type(4)));

constexpr float kPagedLog2e = 1.4426950408889634f;

// D = A B + C, 16x16x32: A[i][k] in lane i + 16 (k/8) element k%8, B[k][j] in
// lane j + 16 (k/8) element k%8, D[i][j] in lane j + 16 (i/4) element i%4.
__device__ __forceinline__ pg_f32x4 pg_mfma16(u32x4 a, u32x4 b, pg_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf16x8, a), __builtin_bit_cast(pg_bf16x8, b), c,
                                                  0, 0, 0);
}

// 2^x with the hardware instruction alone (below 2^-126 it gives zero).
__device__ __forceinline__ float pg_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

struct PagedAttn {
    const uint16_t* q;
    int64_t ld_q;
    float scale;
    uint16_t* out;
    int64_t ld_out;
    float target;  // slots of one key/value head that the keys are cut for
    int64_t slots;
    float* part;   // [slots][HKV][M][D] accumulators
    float2* ml;    // [slots][HKV][M] (m, l)
    int2* notes;   // [notes] (first slot, keys of a chunk) of a tile
};

// The position behind the last key that a row attends in its segment: row i of n of a
// sequence is position kv_len - n + i; of a shared prefix every row attends all.
__device__ __forceinline__ int row_limit(const PagedSeg& g, int kv_len, bool own, int row) {
    return own ? min(max(kv_len - g.rows + row + 1, 0), g.keys) : g.keys;
}

// One 16-position piece of a segment's keys, none of whose rows is read beyond `n`.
struct PagedPiece {
    __amdgpu_buffer_rsrc_t k, v;
    int n;  // positions that are there, from the first
};
// `page` is wave-uniform; `at` the piece's first position, `end` the segment's.
template <int ROW>  // bytes of a position
__device__ __forceinline__ PagedPiece paged_piece(const PagedKv& c, const char* kh, const char* vh, int page, int at,
                                                  int end) {
    PagedPiece p;
    p.n = (unsigned)page < (unsigned)c.num_pages ? min(max(end - at, 0), 16) : 0;
    const int64_t in_page = at & ((1 << c.shift) - 1);
    const int64_t pg = p.n > 0 ? page : 0;
    const uint32_t kb = p.n > 0 ? (uint32_t)((p.n - 1) * (int)c.k_pos + ROW) : 0u;
    const uint32_t vb = p.n > 0 ? (uint32_t)((p.n - 1) * (int)c.v_pos + ROW) : 0u;
    p.k = buffer_rsrc(kh + pg * c.k_page + in_page * c.k_pos, kb);
    p.v = buffer_rsrc(vh + pg * c.v_page + in_page * c.v_pos, vb);
    return p;
}

// Sixteen e4m3 codes as bf16 (exact).
__device__ __forceinline__ void f8_widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = fp8x2_bf16<false>(w);
    hi = fp8x2_bf16<true>(w);
}

// Whether one of two bf16 is infinite or NaN.
__device__ __forceinline__ bool not_finite2(uint32_t w) {
    return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}
// Whether one of four e4m3 codes is NaN (they have no infinities).
__device__ __forceinline__ bool nan_f8x4(uint32_t w) { return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0; }
// The halves of w that `f` holds for (a function of 16 bits), as ones; else zeros.
template <typename F>
__device__ __forceinline__ uint32_t ones2(uint32_t w, F f) {
    return (f(w & 0xFFFFu) ? 0x3F80u : 0u) | (f(w >> 16) ? 0x3F800000u : 0u);
}
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
    return ((w & 0x7F80u) == 0x7F80u ? 0u : w & 0xFFFFu) | ((w & 0x7F800000u) == 0x7F800000u ? 0u : w & 0xFFFF0000u);
}

// What infinities and NaN among the attended values of a column make of its sum,
// given how many there are of each.
__device__ __forceinline__ float taint(float nan, float pos, float neg) {
    if (nan > 0.0f || (pos > 0.0f && neg > 0.0f)) return __builtin_nanf("");
    return pos > 0.0f ? INFINITY : (neg > 0.0f ? -INFINITY : 0.0f);
}

}  // namespace bz
