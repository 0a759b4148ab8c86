// k_attn_row.h — one query row of the masked and the 8-bit-cache attention, by one wave.
//
// s_j = scale q . k_j; capped: s <- cap tanh(s / cap); sloped: s <- s - slope |p - j|; over the keys
// that the row sees, o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), m the largest score of all keys that the
// row sees (fp32 throughout). A masked key's score is not computed, and a key whose weight is zero (below 2^-126
// of the largest) adds nothing whatever its value holds, so neither infinities nor NaN there reach the row. For
// that m is found first: against a running maximum a far key's value would have entered the sum before its weight
// went to zero, and a part's own maximum is not the row's. The tiled kernels, whose matrix products multiply a
// masked key's value by a zero weight, take this path for the rows that came out not finite.
#pragma once
#include "mgh_common.h"
#include "mgh_kernels.h"

namespace mgh {

// The score in log2 units from q . k. tanh(x) = 1 - 2 / (exp(2x) + 1): exp2 of an overflowing argument
// is inf (its reciprocal 0: +cap), of an underflowing one 0 (-cap). Argument, exp2, sum, reciprocal and fma, a step
// or half of one each, leave an absolute 6 2^-24 cap. Where that shows (score_mod) |x| < 3/4 takes x + x^3 Q(x^2), Q of
// degree 4 with the least largest error relative to tanh x (4e-8 with its roundings), in all off by 10 2^-24 of the
// score; beyond, the quotient is no farther off.
constexpr float kSmallArg = 0.75f;
__device__ __forceinline__ float cap_small(float s, const ScoreMod& m) {
    const float x = s * m.cap_x, z = x * x;
    const float q = fmaf(z, fmaf(z, fmaf(z, fmaf(z, -0.0047694925f, 0.019664917f), -0.05339026f), 0.13326521f), -0.3333307f);
    return m.cap2 * x * fmaf(z, q, 1.f);
}
__device__ __forceinline__ float cap_score(float s, const ScoreMod& m) {
    const float e = __builtin_amdgcn_exp2f(s * m.cap_in);
    const float y = fmaf(__builtin_amdgcn_rcpf(e + 1.f), -2.f * m.cap2, m.cap2);
    return m.cap_x != 0.f && fabsf(s * m.cap_x) < kSmallArg ? cap_small(s, m) : y;
}
// whether all of a wave's scores, the largest of a lane's |q . k| being `big`, are small ones (a NaN comes out as NaN)
__device__ __forceinline__ bool all_small(float big, const ScoreMod& m) {
    return m.cap_x != 0.f && __all(big * fabsf(m.cap_x) < kSmallArg);
}

// The reference of a row that has seen nothing: below every finite score in sight, and finite
constexpr float kNoScore = -3e38f;

// A row's partial result: weights relative to 2^m
struct RowState {
    float m, l;
    float o[2];        // features lane and lane + 64
};

// keys [lo, hi) of one row that sees keys of [0, end) and no others. qs: the row's q in LDS (fp32, D values), pl: 64
// floats of LDS; both this wave's own. src.seen(j), src.dot(j, qs), src.value(j, d).
template <class Src>
__device__ __forceinline__ RowState attn_row(const Src& src, const ScoreMod& mod, float slope2, int64_t p, int64_t end, int64_t lo,
                                             int64_t hi, int D, const float* qs, float* pl, int lane) {
    auto score = [&](int64_t j, int64_t to) {
        if (j >= to || !src.seen(j)) return -INFINITY;
        const float x = src.dot(j, qs);
        return (mod.cap2 != 0.f ? cap_score(x, mod) : x * mod.scale2) - slope2 * fabsf((float)(p - j));
    };
    float m = -INFINITY;
    for (int64_t j0 = 0; j0 < end; j0 += 64) {
        const float s = score(j0 + lane, end);
        // a NaN is the whole row's, and so is an infinite score: infinity minus itself
        if (__any(!(s < INFINITY))) {
            const float nan = __builtin_nanf("");
            return RowState{nan, nan, {nan, nan}};
        }
        m = fmaxf(m, s);
    }
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) m = fmaxf(m, __shfl_xor(m, i));
    RowState st{m, 0.f, {0.f, 0.f}};
    if (m == -INFINITY) return st;
    for (int64_t j0 = lo; j0 < hi; j0 += 64) {
        const float w = __builtin_amdgcn_exp2f(score(j0 + lane, hi) - m);
        if (__all(w == 0.f)) continue;
        st.l += w;
        pl[lane] = w;
        __builtin_amdgcn_wave_barrier();
        // 8 keys' values on their way at once; those of weight zero are read and left out
        for (int k = 0; k < 64 && j0 + k < hi; k += 8) {
            float x[2][8];
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (64 * i < D)
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const int64_t j = j0 + k + u < hi ? j0 + k + u : hi - 1;
                        x[i][u] = src.value(j, lane + 64 * i < D ? lane + 64 * i : D - 1);
                    }
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float pk = pl[k + u];
#pragma unroll
                for (int i = 0; i < 2; i++)
                    if (64 * i < D) st.o[i] = pk == 0.f ? st.o[i] : fmaf(pk, x[i][u], st.o[i]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) st.l += __shfl_xor(st.l, i);
    return st;
}

}  // namespace mgh
