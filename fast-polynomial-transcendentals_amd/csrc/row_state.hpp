// row_state.hpp -- the softmax of attention rows over parts of their keys, for the serving
// attentions (shared_prefix.hip, paged_attn.hip): a lane keeps one row of 32, its O,
// maximum and sum, in the layout of v_mfma_f32_32x32x16 products S^T = K Q^T and
// O^T = V^T P^T.
#pragma once

#include <hip/hip_runtime.h>

#include "flash_attn.hpp"

namespace pt {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr float kEmptyMax = -__FLT_MAX__;  // log2 units: below any score, and no infinity
// From this maximum on (log2 units) scores lose the maximum in a step of its own: an FMA
// keeps the product's rounding, half a step of the maximum, which passes the exponents'
// range beyond 2^30, and is 2^-4 here.
constexpr float kFarMax = 0x1p20f;

// The rows that a lane's query has seen so far.
template <int HD>
struct RowState {
    f32x16_t o[HD / 32];  // O^T: o[dt][r] = element dt*32 + 8(r/4) + 4h + r%4 of row c32
    float m, l;           // log2 units; l of this lane's half of the keys

    __device__ __forceinline__ RowState() : m(kEmptyMax), l(0.0f) {
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt) o[dt] = (f32x16_t){};
    }
};

// One tile of NT 32-key accumulators of scores, to become probabilities 2^(s f - m)
// with the factor f that score_state returns.  O and l are rescaled if the tile raises
// the maximum by more than 8 (log2).  BF16 probabilities have FP32's range, and m is a
// maximum; FP16's end at 2^-24, so m lies 7 below one, which keeps what is 2^-31 of the
// largest, and the exponents at 15 and below.  MASKED: keys k0 + 32 kt + 8(r/4) + 4h + r%4
// past klast count nothing; diag = k0 + 4h - klast.
template <int MODE, int HD, bool BF, int NT, bool MASKED>
__device__ __forceinline__ float score_state(f32x16_t (&s)[NT], RowState<HD>& st, const ScoreConsts& k, int diag) {
    if constexpr (!attn_is_plain_softmax(MODE)) {
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
            float x[16];
            softmax_exponents<MODE>(s[kt], k, x);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kt][r] = x[r];
        }
    }
    float mx[4] = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (MASKED && diag + kt * 32 + 8 * (r >> 2) + (r & 3) > 0) s[kt][r] = -__builtin_inff();
            mx[r & 3] = __builtin_fmaxf(mx[r & 3], s[kt][r]);
        }
    const float mt = half_max(__builtin_fmaxf(__builtin_fmaxf(mx[0], mx[1]), __builtin_fmaxf(mx[2], mx[3]))) * k.sl;
    constexpr float kBelow = BF ? 0.0f : 7.0f;
    const bool move = mt - st.m > 8.0f + kBelow;  // both lanes of a row decide alike
    __builtin_amdgcn_sched_barrier(0);
    if (__any(move)) {
        const float m = move ? mt - kBelow : st.m;
        const float alpha = __builtin_amdgcn_exp2f(st.m - m);
        st.m = m;
        st.l *= alpha;
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt) st.o[dt] *= alpha;
    }
    float mul = k.sl;
    const bool far = __builtin_fabsf(st.m) >= kFarMax;
    if (__any(far)) {
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kt][r] = far ? s[kt][r] * mul : s[kt][r];
        mul = far ? 1.0f : mul;
    }
    __builtin_amdgcn_sched_barrier(0);
    return mul;
}
template <int HD, int NT>
__device__ __forceinline__ void score_exps(f32x16_t (&s)[NT], RowState<HD>& st, float mul) {
    float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], mul, -st.m));
            ls[r & 3] += s[kt][r];
        }
    st.l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
}

// Probabilities 8 cc .. 8 cc + 7 of an accumulator as the B operand of P V, in
// the operands' 16-bit type (l adds them unrounded).
template <bool BF>
__device__ __forceinline__ bf16x8_t prob_frag(const f32x16_t& s, int cc) {
    if constexpr (BF) {
        bf16x8_t f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (__bf16)s[8 * cc + e];
        return f;
    } else {
        f16x8_t f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (_Float16)s[8 * cc + e];
        return __builtin_bit_cast(bf16x8_t, f);
    }
}
// What that rounding left, as a second operand.
template <bool BF>
__device__ __forceinline__ bf16x8_t prob_rest(const f32x16_t& s, int cc, bf16x8_t hi) {
    f32x16_t r = s;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        r[8 * cc + e] -= BF ? (float)hi[e] : (float)__builtin_bit_cast(f16x8_t, hi)[e];
    return prob_frag<BF>(r, cc);
}

// FP32 rows of O in LDS, 16-byte chunks swizzled by the row.
template <int HD>
__device__ __forceinline__ uint32_t o_chunk(int row, int chunk) {
    return (uint32_t)(row * HD * 4 + ((chunk ^ row) & (HD / 4 - 1)) * 16);
}
template <int HD>
__device__ __forceinline__ void spill_rows(unsigned char* region, const RowState<HD>& st, int h, int c32) {
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4_t*>(region + o_chunk<HD>(c32, dt * 8 + 2 * g + h)) =
                (f32x4_t){st.o[dt][4 * g], st.o[dt][4 * g + 1], st.o[dt][4 * g + 2], st.o[dt][4 * g + 3]};
}

}  // namespace pt
