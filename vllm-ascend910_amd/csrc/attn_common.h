// Device helpers shared by the attention kernels (attention.hip, attention_kv8.hip):
// the bf16 MFMA, the running softmax state of a query row and its combination, and
// the pieces of the rotary embedding that a decode step fuses in.
#pragma once

#include <math.h>

#include "common.h"

namespace w4a8 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma_bf16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Running state of one query row.  The row's four lanes (c, j = 0..3) each
// hold m and l and the slice
// O^T[16 dt + 4 j + e][c], e = 0..3, of its O.
template <int D>
struct RowState {
    float m, l;
    f32x4 o[D / 16];
};

template <int D>
__device__ __forceinline__ void state_clear(RowState<D>& s) {
    s.m = -INFINITY;
    s.l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) s.o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// The split combine (+): coefficients from the two maxima, then every value
// as x1 * a1 + x2 * a2 with one rounding of the product x2 * a2 and a fused
// multiply-add.  Shared by the prefill kernel and the combine kernel.
__device__ __forceinline__ void fold_coeffs(float m1, float m2, float& mn, float& a1, float& a2) {
#pragma clang fp contract(off)
    mn = fmaxf(m1, m2);
    a1 = exp2f(m1 - mn);
    a2 = exp2f(m2 - mn);
}

__device__ __forceinline__ float fold_value(float x1, float a1, float x2, float a2) {
#pragma clang fp contract(off)
    return fmaf(x1, a1, x2 * a2);
}

// The larger of two, NaN if either is (v_maximum3_f32: unlike fmaxf it needs no
// canonicalising move per MFMA result).
__device__ __forceinline__ float vmax(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// The four lanes of a row (lane ^ 16, lane ^ 32) reduced by the gfx950 lane
// swaps: x against itself gives one register holding the even and one holding
// the odd 16-lane (32-lane) halves, so no LDS permute and no wait.
template <class F>
__device__ __forceinline__ float row_reduce(float x, F f) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(f(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// s = s (+) t; an empty state (l == 0: no position of the row in that split) is
// the identity.
template <int D>
__device__ __forceinline__ void state_fold(RowState<D>& s, const RowState<D>& t) {
#pragma clang fp contract(off)
    if (t.l == 0.0f) return;
    if (s.l == 0.0f) {
        s = t;
        return;
    }
    float mn, a1, a2;
    fold_coeffs(s.m, t.m, mn, a1, a2);
    s.l = fold_value(s.l, a1, t.l, a2);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s.o[dt][e] = fold_value(s.o[dt][e], a1, t.o[dt][e], a2);
    s.m = mn;
}

// x (+ bias, rounded as a bf16 add), as w4a8_rope_kv reads an input element.
__device__ __forceinline__ float rope_in(uint32_t xbits, uint32_t bbits, bool has_bias) {
#pragma clang fp contract(off)
    const float v = bf16_bits_to_f32(xbits);
    return has_bias ? bf16_bits_to_f32(f32_to_bf16_bits(v + bf16_bits_to_f32(bbits))) : v;
}

}  // namespace w4a8
