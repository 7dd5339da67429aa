// Grouped-query attention over the 8-bit KV cache of kv8.h (gfx950, fp16 and bf16 MFMA).
//
// The query heads that share a KV head are the rows of one problem, as in
// attention.hip: row r = t * G + g of pair (b, h) is head h G + g of query token t, at
// position p = pos[b] + t.  It attends to the positions k <= p, with a window only to
// those with k > p - window or k < sinks.  The cache is walked in chunks of 64
// positions, which are its blocks:
//   scores  S^T = C . Q^T by v_mfma_f32_16x16x32_f16 on the block's codes C, which are
//           fp16 numbers (int8 and e4m3 alike), and the query scaled into fp16 by a power
//           of two 2^-e of its own, times ck = log2(e) * scale * k_scale * 2^e
//   chunk   running (m, l, O): m' = max(m, max s), a = 2^(m - m'), P = 2^(s - m'),
//           l' = l a + sum P,  O' = O a + f16(P * v_scale * f) . codes
//   output  bf16(O / (f l)); zeros for a row that attends to nothing
// so that neither operand is dequantised element by element: a block's scales enter with
// ck and with the exponent.  f is a power of two that keeps v_scale * f in [2^3, 2^11],
// with P (up to 2^4) in the upper half of fp16's range: P is then rounded to 11 bits, where
// bf16 would leave 8, below 2^-17 to steps of 2^-27 at most (relative error of a step's output
// over 1000 positions 1.568e-3, of which the output's own rounding is 1.562e-3).  The query
// loses bits only below 2^-31 of its largest element.  The open block's keys and values are
// the bf16 ones of the tails, its products bf16's, with P as a pair of them.
#include <algorithm>
#include <cmath>

#include "attn_common.h"
#include "kv8.h"
#include "launch.h"

namespace w4a8 {
namespace {

constexpr int kHead = 4;          // floats before O in a workspace state: m, l, 2 unused

// Operand order.  A lane's 16-byte load holds 16 consecutive codes.  K: key
// key_row(kt, c) of tile kt, dimensions 64 i + 16 j .. +16, the halves of which are the
// MFMAs 2 i and 2 i + 1 (any order of the summed dimensions will do as long as Q has
// the same).  V: dimension 16 dt + c at positions 16 j .. +16, its halves the key blocks
// 0 and 1; the score that lane group j holds at slot e of tile kt is then that of
// position slot_pos(kt, j, e), which makes a lane's P^T operand its own scores.
__device__ __forceinline__ int key_row(int kt, int c) { return 16 * (c >> 2) + 4 * kt + (c & 3); }
__device__ __forceinline__ int slot_pos(int kt, int j, int e) { return 16 * j + 4 * kt + e; }

template <int D>
struct Codes {
    uint4 k[4][D / 64];
    uint4 v[D / 16];
    float ks, vs;
};

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return mfma_bf16(a, b, c); }

// Sixteen codes -> the two MFMA operands.
template <bool FP8>
__device__ __forceinline__ void operands(const uint4& w, f16x8& lo, f16x8& hi) {
    const uint2 a = codes_to_f16<FP8>(w.x), b = codes_to_f16<FP8>(w.y);
    const uint2 c = codes_to_f16<FP8>(w.z), d = codes_to_f16<FP8>(w.w);
    lo = __builtin_bit_cast(f16x8, make_uint4(a.x, a.y, b.x, b.y));
    hi = __builtin_bit_cast(f16x8, make_uint4(c.x, c.y, d.x, d.y));
}

// Two fp32 -> two elements of an operand, rounded to nearest even.
__device__ __forceinline__ uint32_t pack2(float a, float b, f16x8) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, bf16x8) { return f32x2_to_bf16x2_bits(a, b); }

// A row's query (the lane's slice, bf16) as fp16 times 2^-e with its largest element in
// [2^14, 2^15); returns 2^e.  An infinity stays one.
template <int D>
__device__ __forceinline__ float query_f16(const uint4 (&q)[D / 32], f16x8 (&qh)[D / 32]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) m = max(m, abs_bits_max8(q[i]));
    m = __float_as_uint(row_reduce(__uint_as_float(m), [](float a, float b) {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    }));
    const int e = min(max(static_cast<int>(m >> 7) - 127 - 14, -100), 113);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            o[k] = pack2(__uint_as_float(w[k] << 16) * down, __uint_as_float(w[k] & 0xffff0000u) * down, f16x8{});
        qh[i] = __builtin_bit_cast(f16x8, make_uint4(o[0], o[1], o[2], o[3]));
    }
    return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// The units of a wave's O, which holds f times the sum (f a power of two, the same for
// all rows of the wave; 0 before the first chunk that sets it: O holds the sum itself).
// One chunk's V scale in them:
struct VScale {
    float g;       // v_scale * f
    float lg;      // log2(g)
    float inv;     // 1 / g
    bool plain;    // g is in [kLeastG, kMostG]
};

// A row's m is the reference of its exponents, not quite its maximum: it is raised to the
// maximum only where that has passed it by 2^kSlack, so that after the first chunks O is
// hardly ever rescaled (in tiles of sixteen rows some row's maximum moves in half of the
// first 64 chunks).  P is then at most 2^kSlack, and g at most 2^(15 - kSlack).
//
// fp16 has steps of 2^-24 below 2^-14: P is off by 2^-25 / g there.  The denominator is the
// sum of the same rounded P, at least 1 over all of a row's positions, so with g from 2^3 on
// a position takes at most 2^-28 from it, and as much of its own value from the product
// (2^-13 over 32768 positions; an output's rounding is 2^-9).  f is set to bring g into
// [2^9, 2^10): later blocks may be twice as large, or 64 times as small, before it is set
// again (with O rescaled).
constexpr float kSlack = 4.0f;
constexpr float kLeastG = 0x1p3f, kMostG = 0x1p11f;

// The exponent of a number (-1 for zero, infinities and NaN), by a vector instruction: from
// its bits the compiler takes scales to scalar registers, and waits for a chunk's loads as
// soon as they are requested (a windowed step of 32 sequences 34 us instead of 27).
__device__ __forceinline__ int exponent(float x) { return __builtin_amdgcn_frexp_expf(x) - 1; }

// `rescale(x)`: O takes the factor x, a power of two; `room()`: O has no element from 2^90 on
// (an open block's values, taken first, may be there before f is set).  f is set by the
// first block whose scale is a number from 2^-23 on (one of zeros, or of values that small,
// says nothing of the others) and set again where such a block is not plain.  It stays in
// [2^-32, 2^30], so that f times a sum stays inside fp32's range for rows that do not see
// the block, and rises only where O stays below 2^120: a sum of 2^25 positions with P up to
// 2^4 and codes up to 448 is below 2^38 `most`, the largest scale before.
template <class F, class G>
__device__ __forceinline__ VScale v_scale(float vs, float& f, float& most, F rescale, G room) {
    VScale v;
    v.g = vs * f;
    if (v.g < kLeastG || v.g > kMostG) {              // (f is 0, too; as a negation of plain it spills)
        const float was = f == 0.0f ? 1.0f : f, fn = ldexpf(1.0f, min(max(9 - exponent(vs), -32), 30));
        v.g = vs * was;
        if (vs >= 0x1p-23f && vs < INFINITY && fn != f && (f == 0.0f ? room() : most * fn < 0x1p82f)) {
            rescale(fn / was);
            f = fn;
            v.g = vs * fn;
        }
    }
    most = fmaxf(most, vs < INFINITY ? vs : 0.0f);
    v.plain = v.g >= kLeastG && v.g <= kMostG;        // false for NaN
    v.lg = __builtin_amdgcn_logf(v.g);
    v.inv = __builtin_amdgcn_rcpf(v.g);                // off by one unit in the last place at most
    return v;
}

// A chunk whose scale is not plain (values of quite another size than those of the blocks
// before, zeros, NaN).  A row that sees some of it takes its O times 2^k for that chunk's
// product and back after it: k brings v_scale * f * 2^k into [2^9, 2^10) where that leaves
// O below 2^120 (beyond, the chunk is below 2^-90 of what the row holds) and the units at
// most 2^100.
// P's factor, v_scale * f * 2^k, is returned.  largest: of the row's O; unit(k): O takes the
// factor 2^k.
template <class F>
__device__ __forceinline__ float own_unit(int& k, bool sees, float vs, float f, float largest, F unit) {
    const int fe = f == 0.0f ? 0 : exponent(f);
    k = sees && vs < INFINITY ? min(min(9 - exponent(vs), 100) - fe, 119 - exponent(largest)) : 0;
    unit(k);
    return sees ? ldexpf(vs, fe + k) : 0.0f;
}

// The chunks that any row of a tile attends to: the first nsink, then wlo .. wlo + n - nsink - 1.
struct Visible {
    int lo, hi;            // positions of the tile's first and last token inside [0, L); hi < lo: none
    int nsink, wlo, n;
    __device__ __forceinline__ int chunk(int i) const { return i < nsink ? i : wlo + (i - nsink); }
};

__device__ __forceinline__ Visible visible(const AttnKv8Args& a, int64_t pos, int tok0, int tok1) {
    Visible v;
    v.lo = static_cast<int>(max(pos + tok0, int64_t{0}));
    v.hi = static_cast<int>(min(pos + tok1, static_cast<int64_t>(a.L) - 1));
    v.nsink = v.wlo = v.n = 0;
    if (v.hi < v.lo) return v;
    if (a.window > 0) {
        v.wlo = max(v.lo - a.window + 1, 0) / kKvBlock;
        v.nsink = min((a.sinks + kKvBlock - 1) / kKvBlock, v.wlo);
    }
    v.n = v.nsink + v.hi / kKvBlock - v.wlo + 1;
    return v;
}

// Chunks per split: `ns` splits of the visible ones, at least one chunk per wave.
__device__ __forceinline__ int chunks_per_split(int n, int ns, const FastDiv& by_ns, int waves) {
    return max(by_ns(n + ns - 1), waves);
}

// The lane's sixteen positions of a chunk that its row sees, one bit each: those up to
// the row's own and, with a window, behind its lower end or among the sinks.
__device__ __forceinline__ uint32_t first_bits(int n) { return (1u << min(max(n, 0), 16)) - 1u; }

__device__ __forceinline__ uint32_t seen_bits(const AttnKv8Args& a, int p_row, int c0, int j) {
    const int o = c0 + 16 * j;
    uint32_t m = first_bits(p_row + 1 - o);
    if (a.window > 0) m &= ~first_bits(p_row - a.window + 1 - o) | first_bits(a.sinks - o);
    return m;
}

// All ones where bit i of m is set, else 0.
__device__ __forceinline__ uint32_t bit_mask(uint32_t m, int i) {
    return static_cast<uint32_t>(static_cast<int>(m << (31 - i)) >> 31);
}

// The bits of x where mask is set, those of y elsewhere (v_bfi_b32).
__device__ __forceinline__ uint32_t bit_select(uint32_t mask, uint32_t x, uint32_t y) { return (mask & x) | (~mask & y); }

template <int D>
__device__ __forceinline__ void scale_o(RowState<D>& st, float x) {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[dt][e] = st.o[dt][e] * x;
}

// O times 2^k; the largest element of a row's O.
template <int D>
__device__ __forceinline__ void shift_o(RowState<D>& st, int k) {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[dt][e] = ldexpf(st.o[dt][e], k);
}

template <int D>
__device__ __forceinline__ float largest_o(const RowState<D>& st) {
    float x = 0.0f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) x = fmaxf(x, fabsf(st.o[dt][e]));
    return row_reduce(x, [](float a, float b) { return fmaxf(a, b); });
}

// The scores that a row does not see taken as -inf.
__device__ __forceinline__ void hide(f32x4 (&sc)[4], uint32_t seen) {
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            sc[kt][e] = __uint_as_float(bit_select(bit_mask(seen, slot_pos(kt, 0, e)), __float_as_uint(sc[kt][e]), 0xff800000u));
}

// The softmax update of one chunk: its raw scores become P^T (times the chunk's V scale;
// where that is not plain, times what `factor(sees)` gives), m and l of the state follow, and
// where a row's reference is raised `rescale(alpha)`: O takes the factor alpha.  ck >= 0: what
// a raw score is multiplied by.
//
// Where every row's maximum is a number below 2^12 the exponent is one fused multiply-add
// of the raw score, s ck + (lg - m): lg - m is off by at most 2^-13, the relative error
// of all of the row's probabilities in the chunk, 2^-18 at maxima below 100.  Elsewhere
// (maxima beyond, no position seen yet, NaN, a V scale that is not plain) the
// exponent is the difference of two rounded products, exactly 0 for the largest.
//
// On the first way the sum of P, like the output, is the matrix unit's (sum_p: P^T times
// ones, of which the row's l takes linv): the sixteen additions and the lane reduction
// were a quarter of the vector instructions.  On the other l is complete, linv 0.
template <class F, class G>
__device__ __forceinline__ void softmax8(float& m, float& l, float& linv, f32x4 (&sc)[4], float ck, const VScale& v, F rescale,
                                         G factor) {
#pragma clang fp contract(off)
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = vmax(top, sc[kt][e]);
    top = row_reduce(top, [](float p, float q) { return vmax(p, q); }) * ck;
    const float mn = vmax(m, top);
    if (__builtin_expect(v.plain && __builtin_amdgcn_ballot_w64(!(fabsf(mn) < 4096.0f && ck > 0.0f)) == 0, 1)) {
        if (__builtin_amdgcn_ballot_w64(mn > m + kSlack) != 0) {
            const float alpha = __builtin_amdgcn_exp2f(m - mn);
            l = l * alpha;
            m = mn;
            rescale(alpha);
        }
        const float off = v.lg - m;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[kt][e] = __builtin_amdgcn_exp2f(fmaf(sc[kt][e], ck, off));
        linv = v.inv;
    } else {
        top = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (a hidden score stays hidden where ck is 0 or NaN)
                sc[kt][e] = sc[kt][e] == -INFINITY ? -INFINITY : sc[kt][e] * ck;
                top = vmax(top, sc[kt][e]);
            }
        top = row_reduce(top, [](float p, float q) { return vmax(p, q); });
        const float mx = vmax(m, top);
        const float mz = mx == -INFINITY ? 0.0f : mx;    // nothing seen yet: everything stays 0
        const float alpha = m != -INFINITY ? __builtin_amdgcn_exp2f(m - mz) : 1.0f;
        float ls = 0.0f;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sc[kt][e] = __builtin_amdgcn_exp2f(sc[kt][e] - mz);
                ls = ls + sc[kt][e];
            }
        l = fmaf(l, alpha, row_reduce(ls, [](float a, float b) { return a + b; }));
        linv = 0.0f;
        m = mx;
        rescale(alpha);
        // a row that sees nothing of the chunk takes nothing from it, whatever its scale
        const float g = v.plain ? v.g : factor(top != -INFINITY);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[kt][e] = sc[kt][e] * g;
    }
}

// P^T as the B operands of a chunk's two key blocks.
template <class E>
__device__ __forceinline__ void operands_p(const f32x4 (&sc)[4], E (&pop)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int kt = 2 * s + k / 2, e = 2 * (k & 1);
            w[k] = pack2(sc[kt][e], sc[kt][e + 1], E{});
        }
        pop[s] = __builtin_bit_cast(E, make_uint4(w[0], w[1], w[2], w[3]));
    }
}

// What the bf16 operands hi leave of P.  (An infinite or NaN P leaves nothing.)
__device__ __forceinline__ void rest_p(f32x4 (&sc)[4], const bf16x8 (&hi)[2]) {
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[kt][e] = sc[kt][e] - static_cast<float>(hi[kt / 2][4 * (kt & 1) + e]);
}

// The sums of P^T's columns, each in every lane and element of its row: ones times P^T.
template <class E>
__device__ __forceinline__ float sum_p(const E (&pop)[2]) {
    E ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = 1.0f;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    s = mfma(ones, pop[0], s);
    s = mfma(ones, pop[1], s);
    return s[0];
}

// A wave's state over chunks of codes: its O holds f times the sum.
template <int D>
struct CodeState : RowState<D> {
    float f, most;
};

// The state with O itself, as the tail's products, the folds and the output take it.
template <int D>
__device__ __forceinline__ void end_codes(CodeState<D>& st) {
    if (st.f != 0.0f) scale_o<D>(st, 1.0f / st.f);
}

// One chunk of codes into a row's state.  ck: log2(e) * scale * 2^e of the row's query.
// next_k(), next_v(): called where w.k (w.v) has been used, to request the next chunk's.
template <int D, bool FP8, class FK, class FV>
__device__ __forceinline__ void chunk_codes(CodeState<D>& st, const f16x8 (&qh)[D / 32], Codes<D>& w, float ck,
                                            uint32_t seen, FK next_k, FV next_v) {
    const float ks = w.ks, vs = w.vs;
    f32x4 sc[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        sc[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            f16x8 lo, hi;
            operands<FP8>(w.k[kt][i], lo, hi);
            sc[kt] = mfma(lo, qh[2 * i], sc[kt]);
            sc[kt] = mfma(hi, qh[2 * i + 1], sc[kt]);
        }
        if (kt & 1) __builtin_amdgcn_sched_barrier(0);   // two tiles' operands at a time: all at once, they spill
    }
    __builtin_amdgcn_sched_barrier(0);
    next_k();
    __builtin_amdgcn_sched_barrier(0);
    const VScale v = v_scale(vs, st.f, st.most, [&](float x) __attribute__((always_inline)) { scale_o<D>(st, x); },
                             [&]() __attribute__((always_inline)) { return __builtin_amdgcn_ballot_w64(largest_o<D>(st) >= 0x1p90f) == 0; });
    float linv;
    f16x8 pop[2];
    hide(sc, seen);
    int k = 0;
    softmax8(st.m, st.l, linv, sc, ck * ks, v, [&](float x) __attribute__((always_inline)) { scale_o<D>(st, x); },
             [&](bool sees) __attribute__((always_inline)) {
                 return own_unit(k, sees, vs, st.f, largest_o<D>(st), [&](int n) { shift_o<D>(st, n); });
             });
    operands_p(sc, pop);
    const float sum = sum_p(pop);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
        f16x8 lo, hi;
        operands<FP8>(w.v[dt], lo, hi);
        st.o[dt] = mfma(lo, pop[0], st.o[dt]);
        st.o[dt] = mfma(hi, pop[1], st.o[dt]);
        if (dt & 1) __builtin_amdgcn_sched_barrier(0);
    }
    st.l = fmaf(sum, linv, st.l);
    next_v();
    if (__builtin_expect(!v.plain, 0)) shift_o<D>(st, -k);
    __builtin_amdgcn_sched_barrier(0);
}

// Dword k of a lane's V operand of key block s (positions 16 j + 8 s + 2 k, + 1), the
// bits of the positions set in m.
__device__ __forceinline__ uint32_t pair_mask(uint32_t m, int s, int k) {
    return bit_select(0xffffu, bit_mask(m, 8 * s + 2 * k), bit_mask(m, 8 * s + 2 * k + 1));
}

__device__ __forceinline__ uint4 and4(const uint4& v, const uint32_t (&m)[4]) {
    return make_uint4(v.x & m[0], v.y & m[1], v.z & m[2], v.w & m[3]);
}

// The open block's operands, brought straight from memory into LDS, each lane's in
// slots of its own ([unit][lane], so every access is free of bank conflicts) in the order
// of Codes, two 16-byte units where that has one.  One wave loads and uses them: in
// registers they would be 128 of a lane's at D = 128 (the step kernel then spilled 250
// and a step of one sequence took 16 us instead of 8).
template <int D>
struct TailLds {
    uint4 k[4 * (D / 32)][64];
    uint4 v[D / 16 * 2][64];
};

// Requested are the first n slots (of V in units of eight); what stands in the others is
// hidden and masked by those who use them.
template <int D>
__device__ __forceinline__ void request_tail(TailLds<D>& t, const AttnKv8Args& a, int64_t pair, int n, int c, int j) {
    const __amdgpu_buffer_rsrc_t kr = make_rsrc(a.k_tail + pair * (kKvBlock * D), static_cast<uint32_t>(n * D * 2));
    const __amdgpu_buffer_rsrc_t vr = make_rsrc(a.vt_tail + pair * (kKvBlock * D), kKvBlock * D * 2);
    const uint32_t ko = static_cast<uint32_t>((key_row(0, c) * D + 16 * j) * 2), vo = static_cast<uint32_t>((c * kKvBlock + 16 * j) * 2);
    const uint32_t beyond[2] = {16 * j < n ? 0u : 0x40000000u, 16 * j + 8 < n ? 0u : 0x40000000u};   // past the buffer's end
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            buf_load16_lds(kr, t.k[kt * (D / 32) + i], ko + static_cast<uint32_t>((4 * kt * D + 64 * (i >> 1) + 8 * (i & 1)) * 2));
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int s = 0; s < 2; ++s)
            buf_load16_lds(vr, t.v[dt * 2 + s], (vo | beyond[s]) + static_cast<uint32_t>((16 * dt * kKvBlock + 8 * s) * 2));
}

__device__ __forceinline__ void await_tail() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The open block (positions c0 .. held - 1 hold values, the tail's other slots whatever
// was there) into a row's state.  Its values are not fp16 numbers; P is the sum of two bf16
// operands (2^-16), so that a short sequence is as precise as a long one: over 40 positions
// the output is off by 1.87e-3 with one, 1.61e-3 with two, all of it its own rounding (a
// step of one sequence 10.6 / 10.9 us).  hidden: some of those positions are hidden from a row;
// an infinity or NaN among their values must not reach it through 0 * value.
template <int D>
__device__ __forceinline__ void chunk_tail(RowState<D>& st, const TailLds<D>& t, const uint4 (&q)[D / 32],
                                           const AttnKv8Args& a, int p_row, int c0, int held, bool hidden, int lane) {
    const int c = lane & 15, j = lane >> 4;
    f32x4 sc[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        sc[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            sc[kt] = mfma_bf16(__builtin_bit_cast(bf16x8, t.k[kt * (D / 32) + i][lane]), __builtin_bit_cast(bf16x8, q[i]), sc[kt]);
        __builtin_amdgcn_sched_barrier(0);   // one tile's operands at a time: all at once, they spill
    }
    float linv;
    bf16x8 hi[2], lo[2];
    hide(sc, seen_bits(a, p_row, c0, j));
    softmax8(st.m, st.l, linv, sc, a.cs, VScale{1.0f, 0.0f, 1.0f, true}, [&](float x) __attribute__((always_inline)) { scale_o<D>(st, x); },
             [](bool) { return 1.0f; });
    operands_p(sc, hi);
    rest_p(sc, hi);
    operands_p(sc, lo);
    st.l = fmaf(sum_p(hi) + sum_p(lo), linv, st.l);
    // o + V . P; where the product with hi alone is no number it stays (lo may be 0, or negative)
    auto products = [&](f32x4& o, int dt, const uint32_t (&in)[2][4]) __attribute__((always_inline)) {
        f32x4 x;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const bf16x8 v = __builtin_bit_cast(bf16x8, and4(t.v[dt * 2 + s][lane], in[s]));
            o = mfma_bf16(v, hi[s], o);
            x = mfma_bf16(v, lo[s], s == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : x);
        }
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool number = fabsf(o[e]) < INFINITY;
            odd = odd | !number;
            o[e] = number ? o[e] + x[e] : o[e];
        }
        return odd;
    };
    uint32_t in[2][4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) in[s][k] = pair_mask(first_bits(held - c0 - 16 * j), s, k);
    f32x4 o[D / 16];
    bool odd = false;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
        o[dt] = st.o[dt];
        odd = odd | products(o[dt], dt, in);
        if (dt & 1) __builtin_amdgcn_sched_barrier(0);
    }
    if (__builtin_expect(hidden && __builtin_amdgcn_ballot_w64(odd) != 0, 0)) {
        // row by row, the values of the positions that the row does not see taken as 0
#pragma unroll 1
        for (int r = 0; r < 16; ++r) {
            const uint32_t m = seen_bits(a, __builtin_amdgcn_readlane(p_row, r), c0, j) & first_bits(held - c0 - 16 * j);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int k = 0; k < 4; ++k) in[s][k] = pair_mask(m, s, k);
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) {
                f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
                products(x, dt, in);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c == r) o[dt][e] = st.o[dt][e] + x[e];
            }
        }
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) st.o[dt] = o[dt];
}

// ---- a decode step's rotary embedding and append ----
// A lane's elements 64 i + 16 j + 8 h .. +8 of a head of the qkv projection's output, their
// partners in the other half (in the same lane at D = 128), and the bias of both; requested
// as early as the row is known.
template <int D>
struct Head {
    uint4 x[D / 32], b[D / 32];
    uint4 px[D == 128 ? 1 : D / 32], pb[D == 128 ? 1 : D / 32];
};

template <int D>
__device__ __forceinline__ void request_head(Head<D>& t, const uint16_t* row, const uint16_t* bias, int col, int j) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const int d = col + 64 * (i >> 1) + 16 * j + 8 * (i & 1);
        t.x[i] = *reinterpret_cast<const uint4*>(row + d);
        t.b[i] = bias ? *reinterpret_cast<const uint4*>(bias + d) : make_uint4(0, 0, 0, 0);
        if constexpr (D == 64) {
            const int d2 = j < 2 ? d + 32 : d - 32;
            t.px[i] = *reinterpret_cast<const uint4*>(row + d2);
            t.pb[i] = bias ? *reinterpret_cast<const uint4*>(bias + d2) : make_uint4(0, 0, 0, 0);
        }
    }
}

// The angles of the lane's elements (the same for i and i + 2 at D = 128).
struct Angles {
    float4 c[2][2], s[2][2];
};

template <int D>
__device__ __forceinline__ void request_angles(Angles& t, const float* cosr, const float* sinr, int j) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = (16 * j + 8 * i) & (D / 2 - 1);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            t.c[i][k] = *reinterpret_cast<const float4*>(cosr + d + 4 * k);
            t.s[i][k] = *reinterpret_cast<const float4*>(sinr + d + 4 * k);
        }
    }
}

// y[d] = bf16(fl(x[d] c) -/+ fl(x[d'] s)), d' the other half's element, as w4a8_rope_kv8.
template <int D>
__device__ __forceinline__ void rotate_head(const Head<D>& t, const Angles& an, bool has_bias, int j, uint4 (&y)[D / 32]) {
#pragma clang fp contract(off)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const bool upper = D == 128 ? i >= 2 : j >= 2;
        const uint4 &x1 = t.x[i], &b1 = t.b[i];
        const uint4 &x2 = D == 128 ? t.x[i ^ 2] : t.px[D == 128 ? 0 : i], &b2 = D == 128 ? t.b[i ^ 2] : t.pb[D == 128 ? 0 : i];
        const float4(&cs)[2] = an.c[i & 1], (&sn)[2] = an.s[i & 1];
        const uint32_t w1[4] = {x1.x, x1.y, x1.z, x1.w}, w2[4] = {x2.x, x2.y, x2.z, x2.w};
        const uint32_t e1[4] = {b1.x, b1.y, b1.z, b1.w}, e2[4] = {b2.x, b2.y, b2.z, b2.w};
        const float cv[8] = {cs[0].x, cs[0].y, cs[0].z, cs[0].w, cs[1].x, cs[1].y, cs[1].z, cs[1].w};
        const float sv[8] = {sn[0].x, sn[0].y, sn[0].z, sn[0].w, sn[1].x, sn[1].y, sn[1].z, sn[1].w};
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float r[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float u = rope_in(h ? w1[k] >> 16 : w1[k] & 0xffffu, h ? e1[k] >> 16 : e1[k] & 0xffffu, has_bias);
                const float v = rope_in(h ? w2[k] >> 16 : w2[k] & 0xffffu, h ? e2[k] >> 16 : e2[k] & 0xffffu, has_bias);
                const float s = sv[2 * k + h];
                r[h] = u * cv[2 * k + h] + v * (upper ? s : -s);
            }
            o[k] = f32x2_to_bf16x2_bits(r[0], r[1]);
        }
        y[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// The step's v elements 16 dt + c and their bias.
template <int D>
struct StepV {
    uint32_t x[D / 16], b[D / 16];
};

template <int D>
__device__ __forceinline__ void request_v(StepV<D>& t, const uint16_t* row, const uint16_t* bias, int col) {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
        t.x[dt] = row[col + 16 * dt];
        t.b[dt] = bias ? bias[col + 16 * dt] : 0u;
    }
}

// A decode step's rotated k (y) and v (vn), at slot pp of the last block, into their places
// among the operands in LDS (which have arrived) and, where the block stays open, in the
// tail.  writes: this wave's row tile writes.
template <int D>
__device__ __forceinline__ void append_step(TailLds<D>& t, const AttnKv8Args& a, const uint4 (&y)[D / 32], const StepV<D>& v,
                                            int64_t pair, int pp, bool writes, int lane) {
    const int c = lane & 15, j = lane >> 4;
    // slot pp: key 4 (pp / 16) + pp % 4 of key tile (pp % 16) / 4, element pp % 8 of lane
    // group pp / 16's key block (pp % 16) / 8
    const bool mine_k = c == 4 * (pp >> 4) + (pp & 3), mine_v = j == pp >> 4, open = pp < kKvBlock - 1;
    if (mine_k) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) t.k[((pp & 15) >> 2) * (D / 32) + i][lane] = y[i];
    }
    uint32_t vn[D / 16];
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) vn[dt] = a.bias ? f32_to_bf16_bits(rope_in(v.x[dt], v.b[dt], true)) : v.x[dt];
    if (mine_v) {
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
            reinterpret_cast<uint16_t*>(&t.v[dt * 2 + ((pp & 15) >> 3)][lane])[pp & 7] = static_cast<uint16_t>(vn[dt]);
    }
    if (writes && open && mine_k) {
        uint16_t* to = a.k_tail + (pair * kKvBlock + pp) * D + 16 * j;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) *reinterpret_cast<uint4*>(to + 64 * (i >> 1) + 8 * (i & 1)) = y[i];
    }
    if (writes && open && mine_v) {
        uint16_t* to = a.vt_tail + pair * (kKvBlock * D) + c * kKvBlock + pp;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) to[16 * dt * kKvBlock] = static_cast<uint16_t>(vn[dt]);
    }
}

// The block that a decode step completes, by all NW waves of the workgroup: the bf16
// operands in LDS quantised, the codes written, and put in the operands' place as fp16.
// Wave w takes key tiles and dimension tiles w, w + NW, ...  red: 2 NW words of LDS.
// Returns the scales.  (One wave alone: a step of 64 sequences 36 us where four took 31.)
template <int D, bool FP8, int NW>
__device__ __forceinline__ float2 complete_block(TailLds<D>& t, uint32_t* red, const AttnKv8Args& a, int64_t blk, bool writes,
                                                 int wave, int lane) {
    const int c = lane & 15, j = lane >> 4;
    uint32_t km = 0, vm = 0;
    for (int kt = wave; kt < 4; kt += NW)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) km = max(km, abs_bits_max8(t.k[kt * (D / 32) + i][lane]));
    for (int dt = wave; dt < D / 16; dt += NW)
#pragma unroll
        for (int s = 0; s < 2; ++s) vm = max(vm, abs_bits_max8(t.v[dt * 2 + s][lane]));
    km = wave_max(km);
    vm = wave_max(vm);
    if (lane == 0) {
        red[wave] = km;
        red[NW + wave] = vm;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        km = max(km, red[w]);
        vm = max(vm, red[NW + w]);
    }
    const KvQuant<FP8> zk(km), zv(vm);
    const uint32_t n = writes ? kKvBlock * D : 0;
    const __amdgpu_buffer_rsrc_t kw = make_rsrc(a.k_codes + blk * (kKvBlock * D), n);
    const __amdgpu_buffer_rsrc_t vw = make_rsrc(a.vt_codes + blk * (kKvBlock * D), n);
    auto code16 = [&](const KvQuant<FP8>& z, uint4& x0, uint4& x1, __amdgpu_buffer_rsrc_t to, int off) __attribute__((always_inline)) {
        const uint2 w0 = z.codes(x0), w1 = z.codes(x1);
        const uint4 w = make_uint4(w0.x, w0.y, w1.x, w1.y);
        buf_store16(to, static_cast<uint32_t>(off), w);
        f16x8 lo, hi;
        operands<FP8>(w, lo, hi);
        x0 = __builtin_bit_cast(uint4, lo);
        x1 = __builtin_bit_cast(uint4, hi);
    };
    for (int kt = wave; kt < 4; kt += NW)
#pragma unroll
        for (int x = 0; x < D / 64; ++x)
            code16(zk, t.k[kt * (D / 32) + 2 * x][lane], t.k[kt * (D / 32) + 2 * x + 1][lane], kw, key_row(kt, c) * D + 16 * j + 64 * x);
    for (int dt = wave; dt < D / 16; dt += NW) code16(zv, t.v[dt * 2][lane], t.v[dt * 2 + 1][lane], vw, (16 * dt + c) * kKvBlock + 16 * j);
    if (writes && wave == 0 && lane == 0) *reinterpret_cast<float2*>(a.kv_scale + blk * 2) = make_float2(zk.scale, zv.scale);
    __syncthreads();
    return make_float2(zk.scale, zv.scale);
}

// That block's fp16 operands into a state that is empty before.
template <int D>
__device__ __forceinline__ void chunk_completed(RowState<D>& st, const TailLds<D>& t, const f16x8 (&qh)[D / 32], float ck,
                                                float2 scale, uint32_t seen, int lane) {
    f32x4 sc[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        sc[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            sc[kt] = mfma(__builtin_bit_cast(f16x8, t.k[kt * (D / 32) + i][lane]), qh[i], sc[kt]);
    }
    float linv;
    f16x8 pop[2];
    hide(sc, seen);
    softmax8(st.m, st.l, linv, sc, ck * scale.x, VScale{0x1p6f, 6.0f, 0x1p-6f, true}, [](float) {}, [](bool) { return 1.0f; });
    operands_p(sc, pop);
    st.l = fmaf(sum_p(pop), linv, st.l);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int s = 0; s < 2; ++s) st.o[dt] = mfma(__builtin_bit_cast(f16x8, t.v[dt * 2 + s][lane]), pop[s], st.o[dt]);
    scale_o<D>(st, scale.y * 0x1p-6f);
}

__device__ __forceinline__ uint4 flip(const uint4& v, uint32_t m) {
    return make_uint4(v.x ^ m, v.y ^ m, v.z ^ m, v.w ^ m);
}

// bf16(O / l) of the lane's slice of a row; zeros where the row attends to nothing.
template <int D>
__device__ __forceinline__ void write_row(uint16_t* o, const RowState<D>& st, bool inside, int j) {
    const float inv = inside && st.l != 0.0f ? 1.0f / st.l : 0.0f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
        uint2 w = make_uint2(f32x2_to_bf16x2_bits(st.o[dt][0] * inv, st.o[dt][1] * inv),
                             f32x2_to_bf16x2_bits(st.o[dt][2] * inv, st.o[dt][3] * inv));
        if (!inside) w = make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(o + 16 * dt + 4 * j) = w;
    }
}

// Workgroup (split, row tile, pair): its NW waves (four, or two) take the split's chunks in turn, the
// next chunk's K requested once the scores are formed, its V once the output is (one set
// of registers, two waves a SIMD: 128 KB a CU under way; three waves, or more splits for
// more workgroups, read no faster), and fold their states through LDS (halves onto halves,
// a fixed order).  With one split that holds chunks the result goes to out, otherwise the
// state to the workspace for attn8_combine_kernel.
//
// Bound by the codes' way from memory: with the arithmetic left out (loads alone) the step
// of 8 sequences of 28000 positions on average, 40 heads over 8 of 128 in int8 (535 MB),
// took 91 us; it takes 90 to 100, 5.4 to 5.9 TB/s.  64 sequences of 1050 (140 MB): 30.0 us,
// 4.7 TB/s, of which some 5 us pass before the first products and in the uneven ends.
// K's loads keep the default cache policy (non-temporal ones fetched its 128-byte lines
// twice, a wave reading half a line at a time), V's are non-temporal where one row tile
// reads them.
//
// How many splits there are is fixed by the launch, which chunks each takes by the
// positions read on the device, so a captured step spreads whatever is visible.
//
// ROPE: the row tile's queries are rotated here from the qkv projection's output.  The
// wave that holds the step's own block puts the step's k and v into its operands (row
// tile 0 also into the tail), and quantises the block if the step completes it.
template <int D, bool FP8, bool ROPE, bool NT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn8_split_kernel(const AttnKv8Args a, int ns, FastDiv by_ns, int tiles,
                                                                             FastDiv by_tiles, int groups) {
    __shared__ TailLds<D> tail;                      // and in its place the waves' O, at the end
    __shared__ float2 lds_ml[NW / 2][64];
    __shared__ uint32_t lds_red[2 * NW];
    f32x4 (*lds_o)[D / 16][64] = reinterpret_cast<f32x4 (*)[D / 16][64]>(&tail);
    static_assert(NW / 2 * sizeof(*lds_o) <= sizeof(tail), "the waves' O take the tail's place");
    // ids run over eight (pair, split) groups, then the row tiles, so that the tiles of
    // one group, which read the same codes, lie on one XCD
    const int id = static_cast<int>(blockIdx.x);
    const int oct = by_tiles(id >> 3), rt = (id >> 3) - oct * tiles, g = oct * 8 + (id & 7);
    if (g >= groups) return;
    const int pair = by_ns(g), split = g - pair * ns;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int lane = static_cast<int>(threadIdx.x) & 63, c = lane & 15, j = lane >> 4;
    const int b = a.by_kvh(pair), h = pair - b * a.KVH;
    const int R = a.G * a.T;
    const int64_t pos = kv_pos(a.pos, a.pos_stride, b, a.T, a.L);
    const Visible vis = visible(a, pos, a.by_g(rt * 16), a.by_g(min(rt * 16 + 15, R - 1)));
    const int per = chunks_per_split(vis.n, ns, by_ns, NW);
    const int i0 = split * per, i1 = min(i0 + per, vis.n);
    if (i0 >= i1 && split > 0) return;
    // this lane's row
    const int r = rt * 16 + c;
    const bool real = r < R;
    const int tok = !ROPE && real ? a.by_g(r) : 0, gq = real ? r - tok * a.G : 0;   // a step: T = 1
    const int64_t p64 = pos + tok;
    const bool inside = real && p64 >= 0 && p64 < a.L;
    // rows past the problem or outside [0, L) go along with the tile's last position (so that
    // they see something in every chunk, as softmax8's first way asks); their output is zero
    const int p_row = inside ? static_cast<int>(p64) : vis.hi;
    const int64_t row_off = ((static_cast<int64_t>(b) * a.T + tok) * a.H + h * a.G + gq) * D;
    const int held = kv_span(pos, a.T, a.L).hi;
    // the last visible chunk is the open block's where that is what it is, and in a
    // decode step always the step's own
    const int last_chunk = vis.n > 0 ? vis.chunk(vis.n - 1) : -1;
    const bool own_last = vis.n > 0 && (ROPE || (held % kKvBlock != 0 && last_chunk == held / kKvBlock));
    const int code_end = min(i1, own_last ? vis.n - 1 : vis.n);
    // it goes to a wave with the fewest chunks of codes, which takes it first
    const bool tail_wave = own_last && i1 == vis.n && wave == (code_end - i0) % NW;

    const int64_t block = static_cast<int64_t>(pair) * a.NB;
    const uint32_t ko = static_cast<uint32_t>(key_row(0, c) * D + 16 * j), vo = static_cast<uint32_t>(c * kKvBlock + 16 * j);
    // chunk i of the wave's; behind its last one nothing is read (an empty buffer gives zeros)
    auto load_k = [&](Codes<D>& w, int i) __attribute__((always_inline)) {
        const bool more = i < code_end;
        const int64_t blk = block + (more ? vis.chunk(i) : 0);
        const __amdgpu_buffer_rsrc_t r = make_rsrc(a.k_codes + blk * (kKvBlock * D), more ? kKvBlock * D : 0);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int x = 0; x < D / 64; ++x) w.k[kt][x] = buf_load16(r, ko + static_cast<uint32_t>(4 * kt * D + 64 * x));
        w.ks = a.kv_scale[blk * 2];
        w.vs = a.kv_scale[blk * 2 + 1];
    };
    auto load_v = [&](Codes<D>& w, int i) __attribute__((always_inline)) {
        const bool more = i < code_end;
        const int64_t blk = block + (more ? vis.chunk(i) : 0);
        const __amdgpu_buffer_rsrc_t r = make_rsrc(a.vt_codes + blk * (kKvBlock * D), more ? kKvBlock * D : 0);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
            const uint32_t o = vo + static_cast<uint32_t>(16 * dt * kKvBlock);
            w.v[dt] = NT ? buf_load16_nt(r, o) : buf_load16(r, o);
        }
    };
    auto load = [&](Codes<D>& w, int i) __attribute__((always_inline)) {
        load_k(w, i);
        load_v(w, i);
    };
    const uint16_t* qkv = ROPE ? a.qkv + b * a.ldq : nullptr;
    const float* cosr = ROPE ? a.cos + (vis.n > 0 ? pos : 0) * a.ldc : nullptr;   // no position: any row of the table
    const float* sinr = ROPE ? a.sin + (vis.n > 0 ? pos : 0) * a.ldc : nullptr;
    // the queries' rows (in the wave of the last block also the step's k and v, and that
    // block) are requested before the first codes: loads return in order
    Codes<D> w;
    uint4 q[D / 32];
    CodeState<D> st;
    state_clear(st);
    st.f = st.most = 0.0f;
    f16x8 qh[D / 32];
    float ck;
    const int c0 = last_chunk * kKvBlock;
    if constexpr (ROPE) {
        Angles an;
        Head<D> hq;
        request_head<D>(hq, qkv, a.bias, (h * a.G + gq) * D, j);
        request_angles<D>(an, cosr, sinr, j);
        // the step completes its block: all waves of the workgroup that holds it join in
        const bool completes = own_last && i1 == vis.n && pos == c0 + kKvBlock - 1;
        float2 scale = make_float2(0.0f, 0.0f);
        if (tail_wave) {
            Head<D> hk;
            StepV<D> v;
            request_head<D>(hk, qkv, a.bias, (a.H + h) * D, j);
            request_v<D>(v, qkv, a.bias, (a.H + a.KVH + h) * D + c);
            request_tail<D>(tail, a, pair, static_cast<int>(pos) - c0, c, j);
            uint4 y[D / 32];
            rotate_head<D>(hk, an, a.bias != nullptr, j, y);
            await_tail();
            append_step<D>(tail, a, y, v, pair, static_cast<int>(pos) - c0, rt == 0, lane);
        } else {
            load(w, i0 + wave);
        }
        rotate_head<D>(hq, an, a.bias != nullptr, j, q);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) q[i] = inside ? flip(q[i], a.flip) : make_uint4(0, 0, 0, 0);
        if (completes) {
            __syncthreads();
            scale = complete_block<D, FP8, NW>(tail, lds_red, a, block + last_chunk, rt == 0, wave, lane);
        }
        ck = a.cs * query_f16<D>(q, qh);
        if (tail_wave) {
            if (completes) chunk_completed<D>(st, tail, qh, ck, scale, seen_bits(a, p_row, c0, j), lane);
            else chunk_tail<D>(st, tail, q, a, p_row, c0, held, a.window > 0 && c0 <= vis.hi - a.window, lane);
            load(w, i0 + wave);
        }
    } else {
        const uint16_t* qr = a.q + row_off + 16 * j;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            q[i] = inside ? flip(*reinterpret_cast<const uint4*>(qr + 64 * (i >> 1) + 8 * (i & 1)), a.flip) : make_uint4(0, 0, 0, 0);
        if (tail_wave) {
            request_tail<D>(tail, a, pair, held - c0, c, j);
            await_tail();
            chunk_tail<D>(st, tail, q, a, p_row, c0, held, vis.lo < held - 1 || (a.window > 0 && c0 <= vis.hi - a.window), lane);
        }
        load(w, i0 + wave);
        ck = a.cs * query_f16<D>(q, qh);
    }
    for (int i = i0 + wave; i < code_end; i += NW)
        chunk_codes<D, FP8>(st, qh, w, ck, seen_bits(a, p_row, vis.chunk(i) * kKvBlock, j),
                            [&]() __attribute__((always_inline)) { load_k(w, i + NW); },
                            [&]() __attribute__((always_inline)) { load_v(w, i + NW); });
    end_codes(st);
    __syncthreads();                                 // the tail has been read
#pragma unroll
    for (int s = NW / 2; s > 0; s /= 2) {
        if (wave >= s && wave < 2 * s) {
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) lds_o[wave - s][dt][lane] = st.o[dt];
            lds_ml[wave - s][lane] = make_float2(st.m, st.l);
        }
        __syncthreads();
        if (wave < s) {
            RowState<D> t;
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) t.o[dt] = lds_o[wave][dt][lane];
            t.m = lds_ml[wave][lane].x;
            t.l = lds_ml[wave][lane].y;
            state_fold<D>(st, t);
        }
        if (s > 1) __syncthreads();
    }
    if (wave > 0 || !real) return;
    if (per >= vis.n) {                              // the only split that holds chunks
        write_row<D>(a.out + row_off, st, inside, j);
        return;
    }
    float* to = a.ws + ((static_cast<int64_t>(pair) * R + r) * ns + split) * (D + kHead);
    if (j == 0) *reinterpret_cast<float2*>(to) = make_float2(st.m, st.l);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<f32x4*>(to + kHead + 16 * dt + 4 * j) = st.o[dt];
}

// Many query tokens: workgroup (split, row group, pair) of four waves, each with RT row
// tiles.  A chunk's codes are converted to operands once per workgroup: wave w loads key
// tile w of K and dimension tiles w D/64 .. of V a chunk ahead into registers, and writes
// the fp16 operands into one of two LDS buffers in operand order ([unit][lane]: no bank
// conflicts, no address arithmetic), from where every wave reads them, each read serving
// its RT tiles.
//
// Bound by the vector work beside the products: 4096 tokens of 40 heads of 128 in int8
// take 203 us (0.85 PFLOP/s), the matrix pipe busy for 35% of the cycles and the vector
// ALU for 55% (exponentials, maxima, the conversion), nearly one after the other in a
// wave, with two waves a SIMD to overlap.  Without softmax and conversion the same loop
// took 129 us where all of it took 200, without the softmax 168, without the conversion 182,
// without the exponentials 193.  With two row tiles a wave the operands' way from LDS takes as long as
// their products at the pipe's full rate; four would need 512 registers.  Tried and
// slower: eight waves in two halves that take turns at the matrix pipe, a barrier a phase
// (274 us); a chunk's exponentials between the products of the next (215 us).
constexpr int kLoopWaves = 4;

template <int D>
struct ChunkLds {
    uint4 k[4 * (D / 32)][64];
    uint4 v[D / 16 * 2][64];
};

// Workgroup -> (pair, row group, split), the row groups with the most positions first, as
// attention.hip's loop_tile: a multiple of eight pairs in contiguous runs per XCD, other
// counts row group by row group over all pairs.
__device__ __forceinline__ void loop_tile8(int pairs, int groups, int ns, int& pair, int& grp, int& split) {
    const int bid = static_cast<int>(blockIdx.x);
    int rank;
    if (pairs % 8 == 0) {
        const int per = groups * ns, lin = (bid & 7) * (pairs / 8 * per) + (bid >> 3);
        pair = lin / per;
        const int rest = lin - pair * per;
        rank = rest / ns;
        split = rest - rank * ns;
    } else {
        const int rest = bid / pairs;
        pair = bid - rest * pairs;
        rank = rest / ns;
        split = rest - rank * ns;
    }
    grp = groups - 1 - rank;
}

// A lane's row of a loop kernel (looked up where it is needed: registers are short there).
struct LoopRow {
    bool real, in;
    int p;              // its position; of rows that have none `hi`, as in attn8_split_kernel
    int64_t off;        // element offset in q and out
};

template <int D>
__device__ __forceinline__ LoopRow loop_row(const AttnKv8Args& a, int64_t pos, int b, int h, int R, int r, int hi) {
    LoopRow w;
    w.real = r < R;
    const int tok = w.real ? a.by_g(r) : 0, g = w.real ? r - tok * a.G : 0;
    const int64_t p = pos + tok;
    w.in = w.real && p >= 0 && p < a.L;
    w.p = w.in ? static_cast<int>(p) : hi;
    w.off = ((static_cast<int64_t>(b) * a.T + tok) * a.H + h * a.G + g) * D;
    return w;
}

template <int D>
__device__ __forceinline__ void loop_query(const AttnKv8Args& a, const LoopRow& w, int j, uint4 (&q)[D / 32]) {
    const uint16_t* qr = a.q + w.off + 16 * j;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        q[i] = w.in ? flip(*reinterpret_cast<const uint4*>(qr + 64 * (i >> 1) + 8 * (i & 1)), a.flip) : make_uint4(0, 0, 0, 0);
}

// The open block into LDS for all waves of the workgroup, once they are done with what
// was there.
template <int D>
__device__ __forceinline__ void loop_tail(TailLds<D>& tail, int wave, const AttnKv8Args& a, int pair, int n, int c, int j) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (wave == 0) {
        request_tail<D>(tail, a, pair, n, c, j);
        await_tail();
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A row's result, or where other splits hold chunks too (!whole) its state.
template <int D>
__device__ __forceinline__ void loop_write(const AttnKv8Args& a, const LoopRow& w, const RowState<D>& st, bool whole, int pair, int R,
                                           int r, int ns, int split, int j) {
    if (!w.real) return;
    if (whole) {
        write_row<D>(a.out + w.off, st, w.in, j);
        return;
    }
    float* to = a.ws + ((static_cast<int64_t>(pair) * R + r) * ns + split) * (D + kHead);
    if (j == 0) *reinterpret_cast<float2*>(to) = make_float2(st.m, st.l);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<f32x4*>(to + kHead + 16 * dt + 4 * j) = st.o[dt];
}

template <int D, bool FP8, int RT>
__global__ __launch_bounds__(64 * kLoopWaves, 2) void attn8_loop_kernel(const AttnKv8Args a, int ns, FastDiv by_ns, int groups) {
    constexpr int NW = kLoopWaves, X = D / 64;
    __shared__ ChunkLds<D> buf[2];
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int lane = static_cast<int>(threadIdx.x) & 63, c = lane & 15, j = lane >> 4;
    int pair, grp, split;
    loop_tile8(a.B * a.KVH, groups, ns, pair, grp, split);
    const int b = a.by_kvh(pair), h = pair - b * a.KVH;
    const int R = a.G * a.T;
    const int64_t pos = kv_pos(a.pos, a.pos_stride, b, a.T, a.L);
    const int r0 = grp * (16 * RT * NW), rw = r0 + wave * (16 * RT);      // the workgroup's, the wave's first row
    const Visible vis = visible(a, pos, a.by_g(r0), a.by_g(min(r0 + 16 * RT * NW - 1, R - 1)));
    const int per = chunks_per_split(vis.n, ns, by_ns, 1);
    const int i0 = split * per, i1 = min(i0 + per, vis.n);
    if (i0 >= i1 && split > 0) return;
    const int held = kv_span(pos, a.T, a.L).hi;
    const int last_chunk = vis.n > 0 ? vis.chunk(vis.n - 1) : -1;
    const bool own_last = vis.n > 0 && held % kKvBlock != 0 && last_chunk == held / kKvBlock;
    const int code_end = min(i1, own_last ? vis.n - 1 : vis.n);

    const int64_t block = static_cast<int64_t>(pair) * a.NB;
    const uint32_t ko = static_cast<uint32_t>(key_row(wave, c) * D + 16 * j);
    const uint32_t vo = static_cast<uint32_t>((16 * X * wave + c) * kKvBlock + 16 * j);
    uint4 rk[X], rv[X];
    auto load = [&](int i) __attribute__((always_inline)) {
        const bool more = i < code_end;
        const int64_t blk = block + (more ? vis.chunk(i) : 0);
        const uint32_t n = more ? kKvBlock * D : 0;
        const __amdgpu_buffer_rsrc_t kr = make_rsrc(a.k_codes + blk * (kKvBlock * D), n);
        const __amdgpu_buffer_rsrc_t vr = make_rsrc(a.vt_codes + blk * (kKvBlock * D), n);
#pragma unroll
        for (int x = 0; x < X; ++x) rk[x] = buf_load16(kr, ko + static_cast<uint32_t>(64 * x));
#pragma unroll
        for (int x = 0; x < X; ++x) rv[x] = buf_load16(vr, vo + static_cast<uint32_t>(16 * x * kKvBlock));
    };
    auto store = [&](ChunkLds<D>& to) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < X; ++x) {
            f16x8 lo, hi;
            operands<FP8>(rk[x], lo, hi);
            to.k[wave * (D / 32) + 2 * x][lane] = __builtin_bit_cast(uint4, lo);
            to.k[wave * (D / 32) + 2 * x + 1][lane] = __builtin_bit_cast(uint4, hi);
        }
#pragma unroll
        for (int x = 0; x < X; ++x) {
            f16x8 lo, hi;
            operands<FP8>(rv[x], lo, hi);
            to.v[(wave * X + x) * 2][lane] = __builtin_bit_cast(uint4, lo);
            to.v[(wave * X + x) * 2 + 1][lane] = __builtin_bit_cast(uint4, hi);
        }
    };
    load(i0);
    // the wave's positions inside [0, L)
    const int lo = static_cast<int>(max(pos + a.by_g(rw), int64_t{0}));
    const int hi = rw < R ? static_cast<int>(min(pos + a.by_g(min(rw + 16 * RT - 1, R - 1)), static_cast<int64_t>(a.L) - 1)) : -1;
    auto row = [&](int t) __attribute__((always_inline)) { return loop_row<D>(a, pos, b, h, R, rw + 16 * t + c, hi); };
    auto load_q = [&](int t, uint4 (&q)[D / 32]) __attribute__((always_inline)) { loop_query<D>(a, row(t), j, q); };
    f16x8 qh[RT][D / 32];
    float ck[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        uint4 q[D / 32];
        load_q(t, q);
        ck[t] = a.cs * query_f16<D>(q, qh[t]);
    }
    CodeState<D> st[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        state_clear(st[t]);
        st[t].f = st[t].most = 0.0f;
    }
    auto step = [&](const ChunkLds<D>& from, int i) __attribute__((always_inline)) {
        const int ch = vis.chunk(i), c0 = ch * kKvBlock;
        // a chunk that lies behind the wave's rows or before their windows
        if (c0 > hi || (a.window > 0 && c0 + kKvBlock - 1 <= lo - a.window && c0 >= a.sinks)) return;
        const bool masked = c0 + kKvBlock - 1 > lo || (a.window > 0 && c0 <= hi - a.window && c0 + kKvBlock > a.sinks);
        const float ks = a.kv_scale[(block + ch) * 2], vs = a.kv_scale[(block + ch) * 2 + 1];
        // operands a group of GU units ahead of their use, so that their way from LDS passes
        // behind the group before (K's units, then V's); the products at a raised priority,
        // so that the SIMD's other wave does not hold up the matrix pipe (two chunks of 500
        // tokens 203 / 196 us)
        f32x4 sc[RT][4];
        constexpr int GU = 2, KG = 4 * (D / 32) / GU, VG = D / 8 / GU;
        uint4 x[2][GU];
        auto read = [&](int g) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < GU; ++n)
                x[g & 1][n] = g < KG ? from.k[g * GU + n][lane] : from.v[(g - KG) * GU + n][lane];
        };
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) sc[t][kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        read(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            read(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < GU; ++n) {
                const int u = g * GU + n, kt = u / (D / 32);
#pragma unroll
                for (int t = 0; t < RT; ++t) sc[t][kt] = mfma(__builtin_bit_cast(f16x8, x[g & 1][n]), qh[t][u % (D / 32)], sc[t][kt]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        const VScale v = v_scale(vs, st[0].f, st[0].most, [&](float x) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < RT; ++t) scale_o<D>(st[t], x);
        }, []() { return true; });                       // the open block comes last here
        f16x8 pop[RT][2];
        float linv[RT];
        int k[RT] = {};
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            if (masked) hide(sc[t], seen_bits(a, row(t).p, c0, j));
            softmax8(st[t].m, st[t].l, linv[t], sc[t], ck[t] * ks, v,
                     [&](float x) __attribute__((always_inline)) { scale_o<D>(st[t], x); },
                     [&](bool sees) __attribute__((always_inline)) {
                         return own_unit(k[t], sees, vs, st[0].f, largest_o<D>(st[t]), [&](int n) { shift_o<D>(st[t], n); });
                     });
            operands_p(sc[t], pop[t]);
        }
        float sum[RT];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int t = 0; t < RT; ++t) sum[t] = sum_p(pop[t]);
#pragma unroll
        for (int g = KG; g < KG + VG; ++g) {
            if (g + 1 < KG + VG) read(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < GU; ++n) {
                const int u = (g - KG) * GU + n;
#pragma unroll
                for (int t = 0; t < RT; ++t) st[t].o[u / 2] = mfma(__builtin_bit_cast(f16x8, x[g & 1][n]), pop[t][u % 2], st[t].o[u / 2]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int t = 0; t < RT; ++t) st[t].l = fmaf(sum[t], linv[t], st[t].l);
        if (__builtin_expect(!v.plain, 0)) {
#pragma unroll
            for (int t = 0; t < RT; ++t) shift_o<D>(st[t], -k[t]);
        }
    };
    store(buf[0]);
    load(i0 + 1);
    for (int i = i0; i < code_end; ++i) {
        // chunk i is in LDS (every wave's part), and every wave is done with chunk i - 1
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        store(buf[(i - i0 + 1) & 1]);
        load(i + 2);
        step(buf[(i - i0) & 1], i);
    }
#pragma unroll
    for (int t = 1; t < RT; ++t) st[t].f = st[0].f;
#pragma unroll
    for (int t = 0; t < RT; ++t) end_codes(st[t]);
    if (own_last && i1 == vis.n) {
        const int c0 = last_chunk * kKvBlock;
        static_assert(sizeof(TailLds<D>) == sizeof(ChunkLds<D>), "the tail takes a chunk's place");
        TailLds<D>& tail = *reinterpret_cast<TailLds<D>*>(&buf[0]);
        loop_tail<D>(tail, wave, a, pair, held - c0, c, j);
        if (c0 <= hi) {
            const bool hidden = lo < held - 1 || (a.window > 0 && c0 <= hi - a.window);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                uint4 q[D / 32];
                load_q(t, q);
                chunk_tail<D>(st[t], tail, q, a, row(t).p, c0, held, hidden, lane);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) loop_write<D>(a, row(t), st[t], per >= vis.n, pair, R, rw + 16 * t + c, ns, split, j);
}

// The split states of a row, combined: NW waves take the splits w, w + NW, ... of the row
// (kBatch requested at a time, the first before the position is known: which splits hold
// something follows from it), then their sums in wave order.  Lane l owns O values
// l D/64 .. +D/64.  With NW = 1 a workgroup takes four rows.  Latency: 3 to 5 us for the
// rows of a step; for 40000 rows of prompts the states' bytes (20 us).
constexpr int kBatch = 8;

template <int D, int NW>
__global__ __launch_bounds__(256) void attn8_combine_kernel(const AttnKv8Args a, int ns, FastDiv by_ns, int waves, int rows,
                                                          FastDiv by_rows, int total) {
#pragma clang fp contract(off)
    constexpr int V = D / 64;
    __shared__ float lds[NW > 1 ? NW : 1][2 + V][64];
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int pr = NW > 1 ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x) * 4 + wave;
    const int first = NW > 1 ? wave : 0;
    if (pr >= total) return;
    const int R = a.G * a.T;
    const int pair = by_rows(pr), r = pr - pair * R;
    const int b = a.by_kvh(pair), h = pair - b * a.KVH;
    const float* w0 = a.ws + static_cast<int64_t>(pr) * ns * (D + kHead);
    float M = -INFINITY, Ls = 0.0f, O[V];
#pragma unroll
    for (int v = 0; v < V; ++v) O[v] = 0.0f;
    auto fold = [&](float m2, float l2, const float (&o2)[V]) __attribute__((always_inline)) {
        if (l2 == 0.0f) return;
        if (Ls == 0.0f) {
            M = m2;
            Ls = l2;
#pragma unroll
            for (int v = 0; v < V; ++v) O[v] = o2[v];
            return;
        }
        float mn, a1, a2;
        fold_coeffs(M, m2, mn, a1, a2);
        Ls = fold_value(Ls, a1, l2, a2);
#pragma unroll
        for (int v = 0; v < V; ++v) O[v] = fold_value(O[v], a1, o2[v], a2);
        M = mn;
    };
    int live = ns;
    int64_t pos = 0;
    for (int s0 = first; s0 < live; s0 += NW * kBatch) {
        float2 ml[kBatch];
        float o2[kBatch][V];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const float* w = w0 + static_cast<int64_t>(min(s0 + NW * u, live - 1)) * (D + kHead);
            ml[u] = *reinterpret_cast<const float2*>(w);
            if constexpr (V == 2) {
                const float2 x = *reinterpret_cast<const float2*>(w + kHead + 2 * lane);
                o2[u][0] = x.x;
                o2[u][1] = x.y;
            } else {
                o2[u][0] = w[kHead + lane];
            }
        }
        if (s0 == first) {
            pos = kv_pos(a.pos, a.pos_stride, b, a.T, a.L);
            const int r0 = r & -rows;              // the row's tile or group
            const Visible vis = visible(a, pos, a.by_g(r0), a.by_g(min(r0 + rows - 1, R - 1)));
            const int per = chunks_per_split(vis.n, ns, by_ns, waves);
            if (per >= vis.n) return;                    // one split held everything and has written the row
            live = (vis.n + per - 1) / per;
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (s0 + NW * u < live) fold(ml[u].x, ml[u].y, o2[u]);
    }
    if constexpr (NW > 1) {
        lds[wave][0][lane] = M;
        lds[wave][1][lane] = Ls;
#pragma unroll
        for (int v = 0; v < V; ++v) lds[wave][2 + v][lane] = O[v];
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            float o2[V];
#pragma unroll
            for (int v = 0; v < V; ++v) o2[v] = lds[w][2 + v][lane];
            fold(lds[w][0][lane], lds[w][1][lane], o2);
        }
    }
    const int tok = a.by_g(r), g = r - tok * a.G;
    const int64_t p = pos + tok;
    const bool inside = p >= 0 && p < a.L;
    const float inv = inside && Ls != 0.0f ? 1.0f / Ls : 0.0f;
    uint16_t* o = a.out + ((static_cast<int64_t>(b) * a.T + tok) * a.H + h * a.G + g) * D + lane * V;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = inside ? static_cast<uint16_t>(f32_to_bf16_bits(O[v] * inv)) : uint16_t{0};
}

// How a call runs: `loop` on attn8_loop_kernel with rt row tiles a wave, else on
// attn8_split_kernel with nw waves; groups row groups (row tiles) per pair, ns splits.
struct Plan {
    bool loop = false;
    int rt = 1, nw = 4;
    int64_t groups = 1, ns = 1;
};

// The plan with the least estimated time.  The estimates (us) are fits to measured times
// of 26 prompt and 16 decode shapes at 1 to 48 splits, one to 4096 query tokens over 64 to
// 32000 positions; what they weigh: a chunk of 64 positions costs a workgroup ca where it
// has a CU to itself and cp where two share one; more workgroups than two a CU take
// rounds; splits cost the combine launch and their states' way through memory.  In the
// split kernel a wave's chunk takes c; its codes come at 5.8 TB/s, less where the CUs hold
// uneven numbers of workgroups or half of them hold none, a second row tile's in part
// from the caches; and a round of workgroups begins with loads that wait for each other
// (position, projection and open block, first codes).  (Decode, heads of 64, 32 sequences
// of 4000: one split 25.0 us, two 27.3, three 30.0; heads of 128, 8 of 4000: 31.4, 23.7,
// 21.0, 21.3 with four.)
//
// Two waves a workgroup instead of four: more workgroups at a time, so fewer such rounds
// where there are many sequences, for chunks that follow each other in a wave (heads of
// 128, 200 sequences of 150 positions 43.7 / 32.0 us, 100 of 400 30.0 / 23.0, 64 of 1000
// 28.0 / 26.3; heads of 64, 64 of 3000 34.3 / 36.6, 32 of 1000 11.2 / 13.0, four / two).
// One wave is no better (31.1, 24.5, 28.3 at heads of 128).  In one round either way two
// waves win where the codes take less than about 35 us.  With splits two waves serve few
// sequences, a chunk for each wave (heads of 128, one sequence of 1000: nine splits 10.5 us,
// five of four waves 11.7, three 11.6).
//
// It is made for the cache's capacity, not for what its sequences hold: 64 sequences of
// 1000 positions take 30 us in a cache of 1024, 4096 or 16384, but 200 of 150 positions 31 us
// in one of 192 or 4096 and 76 in one of 16384, where it splits them.
//
// Split kernel or loop kernel: one row tile, or two, against 64 or more rows that share
// the conversion (40 rows over 8000 positions 24.2 / 19.5 us, 25 rows of each of 8
// sequences over 4096 26.0 / 29.0, split / loop).
Plan plan(int64_t B, int64_t T, int64_t G, int64_t KVH, int64_t D, int64_t NB, int64_t window, int64_t sinks) {
    const int64_t pairs = B * KVH, tiles = (G * T + 15) / 16, cus = device_cu_count(), slots = 2 * cus;
    // the most chunks a row tile can see, and the average over the row tiles
    const int64_t seen = window > 0 && window < 64 * NB ? (window + 62) / 64 + 1 + std::min<int64_t>((sinks + 63) / 64, NB) : NB;
    const int64_t n = std::min(NB, seen);
    const double avg = n < NB ? n : std::max(1.0, n - T / 128.0);
    auto combine = [&](int64_t ns) { return ns > 1 ? 4.0 + 3.0 * ((ns - 1) / 32) + B * T * G * KVH * ns * (D + kHead) * 8 / 3.0e6 : 0.0; };
    Plan best;
    double least = 1.0e30;
    auto consider = [&](bool loop, int rt, int64_t groups, int64_t ns, double t) {
        if (t >= least) return;
        least = t;
        best.loop = loop;
        best.rt = rt;
        best.groups = groups;
        best.ns = ns;
    };
    static constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    if (T == 1 || tiles < 3) {
        const double bytes = (1.3 + 0.7 * tiles) * pairs * n * 64 * D;
        // in units of four waves: what fits the card at once
        const int64_t places = D == 128 ? slots : 3 * cus;
        for (const int nw : {4, 2})
            for (const int64_t ns : kSplits) {
                if (ns > 1 && ns * nw / 2 > n) break;
                const int64_t x = pairs * tiles * ns, units = std::max<int64_t>(x * nw / 4, 1);
                const int64_t iterations = (n + nw * ns - 1) / (nw * ns);
                if (nw == 2 && ns > 1 && (iterations > 1 || 2 * units > cus)) continue;
                const bool alone = units <= cus;
                const double c = D == 128 ? (alone ? 1.45 : 1.9) : (alone ? 0.95 : 1.25);
                const double rounds = static_cast<double>((units + places - 1) / places);
                const double even = static_cast<double>((x + cus - 1) / cus * cus) / x;
                const double memory = bytes / 5.8e6 * (alone ? std::sqrt(static_cast<double>(cus) / units) : 0.5 + 0.5 * even);
                const double start = (D == 128 ? 8.0 : 6.0) * rounds + (nw == 4 ? 0.7 : 0.02 * memory);
                const double t = start + std::max(rounds * iterations * c, memory) + (ns > 1 ? combine(ns) - 1.3 : 0.0);
                if (t >= least) continue;
                consider(false, 1, tiles, ns, t);
                best.nw = nw;
            }
        return best;
    }
    for (const int rt : {1, 2}) {
        const double ca = D == 128 ? (rt == 1 ? 1.39 : 1.95) : (rt == 1 ? 1.0 : 1.4);
        const double cp = D == 128 ? (rt == 1 ? 1.9 : 2.6) : (rt == 1 ? 1.2 : 1.9);
        const int64_t groups = (tiles + kLoopWaves * rt - 1) / (kLoopWaves * rt);
        for (const int64_t ns : kSplits) {
            if (ns > n) break;
            const int64_t x = pairs * groups * ns, per = (n + ns - 1) / ns, rest = x % slots;
            double t = per * (x <= cus ? ca : cp);
            if (x > slots) {
                const double even = per * (x / slots * cp + (rest == 0 ? 0.0 : rest <= cus ? ca : cp));
                const double mixed = x * (avg / ns) * cp / slots + 0.3 * per * cp;   // long groups first
                t = std::max(t, std::min(even, mixed));
            }
            consider(true, rt, groups, ns, t + combine(ns));
        }
    }
    return best;
}

template <int D, bool FP8>
void launch(const AttnKv8Args& a, const Plan& p, hipStream_t stream) {
    const int pairs = a.B * a.KVH, ns = static_cast<int>(p.ns), groups = static_cast<int>(p.groups);
    const FastDiv by_ns(static_cast<uint32_t>(ns));
    if (p.loop) {
        const dim3 grid(static_cast<unsigned>(pairs * p.groups * p.ns)), block(64 * kLoopWaves);
        if (p.rt == 2) attn8_loop_kernel<D, FP8, 2><<<grid, block, 0, stream>>>(a, ns, by_ns, groups);
        else attn8_loop_kernel<D, FP8, 1><<<grid, block, 0, stream>>>(a, ns, by_ns, groups);
    } else {
        const dim3 grid(static_cast<unsigned>((pairs * p.ns + 7) / 8 * 8 * p.groups)), block(64 * p.nw);
        const FastDiv by_tiles(static_cast<uint32_t>(groups));
        auto go = [&](auto kernel) { kernel<<<grid, block, 0, stream>>>(a, ns, by_ns, groups, by_tiles, pairs * ns); };
        auto pick = [&](auto nw) {
            constexpr int NW = decltype(nw)::value;
            if (a.qkv) groups == 1 ? go(attn8_split_kernel<D, FP8, true, true, NW>) : go(attn8_split_kernel<D, FP8, true, false, NW>);
            else groups == 1 ? go(attn8_split_kernel<D, FP8, false, true, NW>) : go(attn8_split_kernel<D, FP8, false, false, NW>);
        };
        if (p.nw == 2) pick(std::integral_constant<int, 2>{});
        else pick(std::integral_constant<int, 4>{});
    }
    if (ns > 1) {
        // rows: those that share a list of visible chunks (a power of two)
        const int total = a.B * a.T * a.H, waves = p.loop ? 1 : p.nw, rows = p.loop ? 16 * kLoopWaves * p.rt : 16;
        const FastDiv by_rows(static_cast<uint32_t>(a.G * a.T));
        if (ns > kBatch)
            attn8_combine_kernel<D, 4><<<dim3(static_cast<unsigned>(total)), dim3(256), 0, stream>>>(a, ns, by_ns, waves, rows,
                                                                                                 by_rows, total);
        else
            attn8_combine_kernel<D, 1><<<dim3(static_cast<unsigned>((total + 3) / 4)), dim3(256), 0, stream>>>(
                a, ns, by_ns, waves, rows, by_rows, total);
    }
}

}  // namespace

int64_t attention_kv8_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t KVH, int64_t D, int64_t NB, int64_t window,
                                      int64_t sinks) {
    const int64_t ns = plan(B, T, H / KVH, KVH, D, NB, window, sinks).ns;
    return ns > 1 ? B * T * H * ns * (D + kHead) * 4 : 0;
}

bool attention_kv8_fits(int64_t B, int64_t T, int64_t H, int64_t KVH, int64_t D, int64_t NB, int64_t window, int64_t sinks) {
    const Plan p = plan(B, T, H / KVH, KVH, D, NB, window, sinks);
    // the attention's workgroups, and the combine's: one a row, or one for four
    return (B * KVH * p.ns + 7) / 8 * 8 <= kMaxWorkgroups / p.groups && B * T < (1ll << 31) / H &&
           (p.ns == 1 || B * T * H <= kMaxWorkgroups * (p.ns > kBatch ? 1 : 4));
}

hipError_t launch_attention_kv8(const AttnKv8Args& a, hipStream_t stream) {
    const Plan p = plan(a.B, a.T, a.G, a.KVH, a.D, a.NB, a.window, a.sinks);
    if (a.D == 128) {
        if (a.fp8) launch<128, true>(a, p, stream);
        else launch<128, false>(a, p, stream);
    } else {
        if (a.fp8) launch<64, true>(a, p, stream);
        else launch<64, false>(a, p, stream);
    }
    return hipGetLastError();
}

}  // namespace w4a8
