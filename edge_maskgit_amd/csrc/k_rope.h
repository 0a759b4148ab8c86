// k_rope.h — the rotation of pairs of features by their token's positions (include/mgh.h has the orders).
//
// (a, b) -> (a cos t - b sin t, a sin t + b cos t), t = f p. Angles are kept in turns of 2^-64: the frequency as a whole
// number F = 2^64 f / 2 pi (mod 2^64), so that p F mod 2^64 is the angle with its whole turns gone and no rounding,
// however far the position; its highest 32 bits are used (off by less than 2^-32 turns and what F's rounding gives,
// |p| 2^-65). The remainder within an eighth of a turn of the nearest quarter goes through odd and even polynomials
// (least largest error, 2^-28 of the sine and 2^-33), fp32 throughout.
#pragma once
#include "mgh_common.h"
#include "mgh_kernels.h"

namespace mgh {

struct SinCos {
    float s, c;
};
__device__ __forceinline__ SinCos sincos_turns(uint32_t t) {
    const uint32_t q = (t + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(t - (q << 30)) * 1.4629180792671596e-9f;        // 2 pi 2^-32
    const float z = x * x;
    const float s = fmaf(x * z, fmaf(z, fmaf(z, -0.00019517235f, 0.008332178f), -0.16666655f), x);
    const float c = fmaf(z * z, fmaf(z, fmaf(z, 2.443838e-05f, -0.0013887367f), 0.041666646f), fmaf(z, -0.5f, 1.f));
    const uint32_t a = __builtin_bit_cast(uint32_t, q & 1 ? c : s), b = __builtin_bit_cast(uint32_t, q & 1 ? s : c);
    return {__builtin_bit_cast(float, a ^ ((q & 2) << 30)), __builtin_bit_cast(float, b ^ (((q + 1) & 2) << 30))};
}

// The same in 64 bits, for values whose rounding decides about a code: sine and cosine of t 2^-64 turns to 2^-45, by their series
// (t itself is off by F's rounding, as above: 2^-45 turns at positions of 2^20, 2^-34 at 2^31)
struct SinCos64 {
    double s, c;
};
__device__ __forceinline__ SinCos64 sincos_turns64(uint64_t t) {
    const uint32_t q = (uint32_t)((t + (1ull << 61)) >> 62);
    const int64_t r = (int64_t)(t - ((uint64_t)q << 62));
    const double x = fma((double)(int32_t)(r >> 32), 4294967296., (double)(uint32_t)r) * 3.406121580086554e-19;       // 2 pi 2^-64
    const double z = x * x, z2 = z * z;
    const double s1 = fma(z, 0.008333333333333333, -0.16666666666666666), s2 = fma(z, 2.7557319223985893e-06, -0.0001984126984126984);
    const double s3 = fma(z, 1.6059043836821613e-10, -2.505210838544172e-08);
    const double s = fma(x * z, fma(fma(s3, z2, s2), z2, s1), x);
    const double c1 = fma(z, 0.041666666666666664, -0.5), c2 = fma(z, 2.48015873015873e-05, -0.001388888888888889);
    const double c3 = fma(z, 2.08767569878681e-09, -2.755731922398589e-07);
    const double c = fma(z, fma(fma(fma(z2, -1.1470745597729725e-11, c3), z2, c2), z2, c1), 1.);
    const bool odd = q & 1;
    const double a = odd ? c : s, b = odd ? s : c;
    return {q & 2 ? -a : a, (q + 1) & 2 ? -b : b};
}

// to fp16 with one rounding: to fp32 by way of the neighbour whose last bit is 1 where v is not one of them (what fp32 rounds
// to 0 or infinity fp16 does too)
__device__ __forceinline__ _Float16 half_of(double v) {
    const float f = (float)v;
    const double e = v - (double)f;
    uint32_t u = __builtin_bit_cast(uint32_t, f);
    if (e != 0. && !(u & 1) && f != 0.f && f - f == 0.f) u += (e > 0.) == (f > 0.f) ? 1u : ~0u;
    return (_Float16)__builtin_bit_cast(float, u);
}

// p F mod 2^64: two 32-bit products, p's sign taken off the upper half
__device__ __forceinline__ uint64_t turns64_at(int32_t p, uint64_t F) {
    const uint32_t lo = (uint32_t)F, hi = (uint32_t)(F >> 32), less = p < 0 ? lo : 0u;
    return (uint64_t)(uint32_t)p * lo + ((uint64_t)((uint32_t)p * hi - less) << 32);
}
__device__ __forceinline__ uint32_t turns_at(int32_t p, uint64_t F) { return (uint32_t)(turns64_at(p, F) >> 32); }

// a token's positions along the axes (`i` its index in the call, `run` its position where none are given): loads that
// depend on nothing but the arguments, all four of them, so that none waits for another
struct TokenPos {
    int32_t p0, p1, p2, p3;
    // (by masks: a choice between members would keep them in memory)
    __device__ __forceinline__ int32_t of(const Rotation& r, int pair) const {
        auto pick = [](int32_t a, int32_t b, bool c) {
            const int32_t m = -(int32_t)c;
            return (b & m) | (a & ~m);
        };
        return pick(pick(pick(p0, p1, pair >= r.start[1]), p2, pair >= r.start[2]), p3, pair >= r.start[3]);
    }
};
__device__ __forceinline__ TokenPos token_pos(const Rotation& r, int64_t b, int64_t i, int32_t run) {
    if (!r.pos) return {run, run, run, run};
    const int32_t* p = r.pos + i * r.pst[0] + b * r.pst[1];
    const int64_t st = r.pst[2];
    return {p[0], p[r.axes > 1 ? st : 0], p[r.axes > 2 ? 2 * st : 0], p[r.axes > 3 ? 3 * st : 0]};
}

// V pairs' turns per unit of position
template <int V>
struct Turns {
    uint64_t f[V];
    __device__ __forceinline__ void load(const Rotation& r, int pair) {      // (the table is as long as a row may be)
#pragma unroll
        for (int i = 0; i < V; i++) f[i] = r.turn[pair + i];
    }
};

// The arguments that every thread needs, asked for at once where this stands: left to itself the compiler loads each
// where it is used, behind the branches before it, a round trip to memory at a time.
__device__ __forceinline__ void ask_rotation(const Rotation& r) {
    asm volatile("" ::"s"(r.axes), "s"(r.P), "s"(r.order), "s"(r.start[1]), "s"(r.start[2]), "s"(r.start[3]), "s"(r.start[4]), "s"(r.pos),
                 "s"(r.pst[0]), "s"(r.pst[1]), "s"(r.pst[2]));
}

// Where the features of V pairs in a row lie: V from fa on and V from fb on. Pairs past the rotated ones are the rest of the
// features, two and two in order.
struct Where {
    int fa, fb;
};
__device__ __forceinline__ Where pairs_at(const Rotation& r, int pair, int V) {
    if (pair >= r.P || r.order == kRopePairs) return {2 * pair, 2 * pair + V};
    if (r.order == kRopeHalves) return {pair, r.P + pair};
    int s = 0, n = r.start[1];
#pragma unroll
    for (int a = 1; a < 4; a++)
        if (pair >= r.start[a]) s = r.start[a], n = r.start[a + 1] - r.start[a];
    return {s + pair, s + pair + n};
}

// cos and sin of V pairs
template <int V>
__device__ __forceinline__ void angles(const Rotation& r, const TokenPos& t, const Turns<V>& f, int pair, SinCos* sc) {
#pragma unroll
    for (int i = 0; i < V; i++) sc[i] = sincos_turns(turns_at(t.of(r, pair + i), f.f[i]));
}

// x: V features from fa on, V from fb on
template <int V>
__device__ __forceinline__ void rotate(const Rotation& r, const SinCos* sc, float* x) {
    // (kept in registers as fp32: an fma that rounds to fp16 by itself would skip a rounding, in some kernels and not in others)
    auto turn = [](float& a, float& b, const SinCos& w) {
        float u = fmaf(a, w.c, -(b * w.s)), v = fmaf(a, w.s, b * w.c);
        asm("" : "+v"(u), "+v"(v));
        a = u, b = v;
    };
    if (r.order == kRopePairs) {
#pragma unroll
        for (int i = 0; i < V; i++) turn(x[2 * i], x[2 * i + 1], sc[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) turn(x[i], x[V + i], sc[i]);
    }
}

// x as rotate's, in 64 bits, to fp16
template <int V>
__device__ __forceinline__ void rotate64(const Rotation& r, const TokenPos& t, const Turns<V>& f, int pair, const float* x, _Float16* y) {
    auto turn = [&](int i, float a0, float b0, _Float16& u, _Float16& v) {
        const SinCos64 w = sincos_turns64(turns64_at(t.of(r, pair + i), f.f[i]));
        const double a = a0, b = b0;
        u = half_of(fma(a, w.c, -(b * w.s)));
        v = half_of(fma(a, w.s, b * w.c));
    };
    if (r.order == kRopePairs) {
#pragma unroll
        for (int i = 0; i < V; i++) turn(i, x[2 * i], x[2 * i + 1], y[2 * i], y[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) turn(i, x[i], x[V + i], y[i], y[V + i]);
    }
}

// V features from e on: one access of up to 16 bytes where VEC, else one by one, `st` apart
template <int V, bool H16, bool VEC>
__device__ __forceinline__ void load_features(const void* p, int64_t e, int64_t st, float* x) {
    if constexpr (VEC && V > 1) {
        constexpr int N = H16 || V < 4 ? V : 4;
        if constexpr (H16) {
            typedef _Float16 hn __attribute__((ext_vector_type(N)));
            const hn v = *(const hn*)((const _Float16*)p + e);
#pragma unroll
            for (int j = 0; j < N; j++) x[j] = (float)v[j];
        } else {
            typedef float fn __attribute__((ext_vector_type(N)));
#pragma unroll
            for (int i = 0; i < V; i += N) {
                const fn v = *(const fn*)((const float*)p + e + i);
#pragma unroll
                for (int j = 0; j < N; j++) x[i + j] = v[j];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = H16 ? (float)((const _Float16*)p)[e + i * st] : ((const float*)p)[e + i * st];
    }
}
template <int V, bool H16, bool VEC>
__device__ __forceinline__ void store_features(void* p, int64_t e, int64_t st, const float* x) {
    if constexpr (VEC && V > 1) {
        constexpr int N = H16 || V < 4 ? V : 4;
        if constexpr (H16) {
            typedef _Float16 hn __attribute__((ext_vector_type(N)));
            hn v;
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = (_Float16)x[j];
            *(hn*)((_Float16*)p + e) = v;
        } else {
            typedef float fn __attribute__((ext_vector_type(N)));
#pragma unroll
            for (int i = 0; i < V; i += N) {
                fn v;
#pragma unroll
                for (int j = 0; j < N; j++) v[j] = x[i + j];
                *(fn*)((float*)p + e + i) = v;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (H16) ((_Float16*)p)[e + i * st] = (_Float16)x[i];
            else ((float*)p)[e + i * st] = x[i];
        }
    }
}

// V pairs of `n` heads `step` apart, of one token: the angles once, then head by head. x and y: the token's first of these heads
template <int V, bool IN16, bool OUT16, bool VEC>
__device__ __forceinline__ void rope_heads(const Rotation& r, const TokenPos& t, const Turns<V>& f, int pair, const void* x, int64_t ex, int64_t hx,
                                           int64_t dx, void* y, int64_t ey, int64_t hy, int64_t dy, int n) {
    const Where w = pairs_at(r, pair, V);
    const bool turned = pair < r.P;
    SinCos sc[V];
    for (int h = 0; h < n; h++) {
        float v[2 * V];
        load_features<V, IN16, VEC>(x, ex + h * hx + w.fa * dx, dx, v);
        load_features<V, IN16, VEC>(x, ex + h * hx + w.fb * dx, dx, v + V);
        if (h == 0) angles<V>(r, t, f, pair, sc);         // while the first head's features are on their way
        if (turned) rotate<V>(r, sc, v);
        store_features<V, OUT16, VEC>(y, ey + h * hy + w.fa * dy, dy, v);
        store_features<V, OUT16, VEC>(y, ey + h * hy + w.fb * dy, dy, v + V);
    }
}

}  // namespace mgh
