// k_kv8.hip — the 8-bit key / value cache: writing it and reading it back (gfx950).
//
// A sequence's tokens lie in blocks of 32; block i of sequence b is page table[b][i] of the pool. Per
// block and head K and V have one scale each, d = fp32(max|x| / 127), and every value is the code
// round(x / d), halves away from zero. The quotient is rounded exactly: with y = |x| (127 / max) in
// fp32 only near the true quotient, the code is floor(y) or the next, and the sign of
// fma(-(floor(y) + 1/2), d, |x|), which a single rounding cannot change, tells which. A block gets its
// codes once its 32 tokens are there, from their fp16 values, which a ring of 64 tokens per sequence and
// head keeps until then; so the cache does not depend on how tokens were grouped into calls, no code
// is ever rescaled, and a sequence may be shortened by up to 32 tokens.
#include <algorithm>
#include <type_traits>

#include "k_kv8.h"
#include "k_rope.h"

namespace mgh {

namespace {

// code + 128, a whole number (a conversion to a byte takes it as it is)
__device__ __forceinline__ float code_of(_Float16 x, float d, float id) {
    const float a = fabsf((float)x), h = floorf(a * id) + 0.5f;
    return 128.f + copysignf(h + (fmaf(-h, d, a) >= 0.f ? 0.5f : -0.5f), (float)x);
}

// N consecutive features of a row: 16-byte loads where rows are aligned for them (VEC), else one by one
template <int N, bool IN16, bool VEC>
__device__ __forceinline__ void load_row(const void* p, int64_t e, int64_t st, _Float16* x) {
    if (VEC && IN16) {
        typedef _Float16 hn __attribute__((ext_vector_type(N > 8 ? 8 : N)));
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const hn v = *(const hn*)((const _Float16*)p + e + i);
#pragma unroll
            for (int j = 0; j < (N > 8 ? 8 : N); j++) x[i + j] = v[j];
        }
    } else if (VEC) {
        typedef float fn __attribute__((ext_vector_type(N > 4 ? 4 : N)));
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const fn v = *(const fn*)((const float*)p + e + i);
#pragma unroll
            for (int j = 0; j < (N > 4 ? 4 : N); j++) x[i + j] = (_Float16)v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = IN16 ? ((const _Float16*)p)[e + i * st] : (_Float16)((const float*)p)[e + i * st];
    }
}

// One workgroup per touched block, head and sequence. Threads take 16 features of a token of K and two
// features of 8 tokens of V: the 16 bytes of codes that they write. The largest |x| goes by its bits, which put
// NaN above infinity: a block that holds either has that scale, and all its values come out NaN.
// The ring: each workgroup stores the new ones of its tokens, unless the call touches more than two blocks and the
// first one's earlier tokens are still in the ring, where the third block's slots are theirs: then the first
// workgroup stores all, after its reads. Four prompts of 2050 tokens, 8 heads of 128, 50 MB: 15.2 us, 5 us more
// where the first workgroup stores all.
// ROT: keys are rotated on the way (k_rope.h), before they are rounded to fp16: the 16 features are 8 pairs, in
// granules of ROT pairs, whose features lie in two runs; 0: as they come, 16 in a row. In 64 bits: with fp32's 2^-23 one value
// in 2^12 rounds to the other fp16 number, and one in 2^16 to another code, an error of 1 / 127 of the block's largest, which
// made half of what all roundings to fp16 together make (2.4e-4 against 2.1e-4 of the values read back).
template <bool IN16, bool VEC, int ROT, int NT>
__device__ __forceinline__ void append_block(const Kv8AppendArgs& a, const Rotation* r) {
    __shared__ uint32_t mx[2][NT / 64];
    const Kv8& c = a.c;
    if constexpr (ROT != 0)
        asm volatile("" ::"s"(c.k), "s"(c.v), "s"(c.scales), "s"(c.k_tail), "s"(c.v_tail), "s"(c.table), "s"(c.table_stride), "s"(c.pages),
                     "s"(a.k), "s"(a.v), "s"(a.st[0]), "s"(a.st[1]), "s"(a.st[2]), "s"(a.st[3]));
    const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, D = c.D;
    int len, total;
    if (!spans(c, a.lens, a.fresh, a.S, b, len, total)) return;
    const int first = len & ~(kKvBlock - 1), t0 = first + kKvBlock * blockIdx.x;     // the block's first token
    if (total == len || t0 >= total) return;
    const int64_t src = b * a.st[3] + hk * a.st[2];
    _Float16* ring_k = c.k_tail + ((int64_t)b * c.Hkv + hk) * kKvRing * D;
    _Float16* ring_v = c.v_tail + ((int64_t)b * c.Hkv + hk) * D * kKvRing;
    auto at = [&](int t, int d) { return src + (int64_t)(t - len) * a.st[1] + d * a.st[0]; };
    const bool whole = t0 + kKvBlock <= total, each = len == first || total - first <= 2 * kKvBlock;
    const int r0 = total - kKvRing > len ? total - kKvRing : len;        // tokens from here on go to the ring
    auto halves = [](const _Float16* x) { return f16x8{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]}; };
    // two features' new ones of tokens t .. t + 7 to the ring
    auto ring_v8 = [&](int t, int d, const _Float16* x) {
        _Float16* to = ring_v + d * kKvRing + t % kKvRing;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (t >= r0 && t + 8 <= total) {
                *(f16x8*)(to + h * kKvRing) = halves(x + 8 * h);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (t + j >= r0 && t + j < total) to[h * kKvRing + j] = x[8 * h + j];
            }
        }
    };
    auto load_v8 = [&](int t, int d, int from, _Float16* x) {            // the input's from token `from` on
        const int64_t e = at(t, d);
        auto one = [&](int i) {
            _Float16 two[2];
            load_row<2, IN16, VEC>(a.v, e + i * a.st[1], a.st[0], two);
            x[i] = two[0], x[8 + i] = two[1];
        };
        if (t >= from && t + 8 <= total) {                               // no branch between the loads
#pragma unroll
            for (int i = 0; i < 8; i++) one(i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (t + i >= from && t + i < total) one(i);
        }
    };
    // 16 features of K that a thread takes, those of unit u of a token: runs of N
    constexpr int N = ROT ? ROT : 16, NU = 16 / N;
    auto runs = [&](int u, auto f) {                                     // f(index of 16, feature) per run
        if constexpr (ROT == 0) {
            f(std::integral_constant<int, 0>{}, 16 * u);
        } else {
#pragma unroll
            for (int g = 0; g < NU / 2; g++) {
                const Where w = pairs_at(*r, 8 * u + ROT * g, ROT);
                f(2 * ROT * g, w.fa);
                f(2 * ROT * g + ROT, w.fb);
            }
        }
    };
    auto load_new_k = [&](int t, int u, _Float16* x) {
        if constexpr (ROT == 0) {
            load_row<16, IN16, VEC>(a.k, at(t, 16 * u), a.st[0], x);
        } else {
            const TokenPos p = token_pos(*r, b, t - len, t);
            Turns<ROT> f[NU / 2];
#pragma unroll
            for (int g = 0; g < NU / 2; g++) f[g].load(*r, 8 * u + ROT * g);
            float v[16];
            runs(u, [&](int i, int d) { load_features<ROT, IN16, VEC>(a.k, at(t, d), a.st[0], v + i); });
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = (_Float16)v[i];
#pragma unroll
            for (int g = 0; g < NU / 2; g++) {
                const int pair = 8 * u + ROT * g;
                if (pair < r->P) rotate64<ROT>(*r, p, f[g], pair, v + 2 * ROT * g, x + 2 * ROT * g);
            }
        }
    };
    auto load_ring_k = [&](int t, int u, _Float16* x) {
        if constexpr (ROT == 0) {
            load_row<16, true, true>(ring_k, (t % kKvRing) * D + 16 * u, 1, x);
        } else {
            float v[16];
            runs(u, [&](int i, int d) { load_features<ROT, true, true>(ring_k, (t % kKvRing) * D + d, 1, v + i); });
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = (_Float16)v[i];
        }
    };
    auto put_ring_k = [&](int t, int u, const _Float16* x) {
        _Float16* to = ring_k + (t % kKvRing) * D;
        if constexpr (ROT == 0) {
            *(f16x8*)(to + 16 * u) = halves(x);
            *(f16x8*)(to + 16 * u + 8) = halves(x + 8);
        } else {
            typedef _Float16 hn __attribute__((ext_vector_type(N)));
            runs(u, [&](int i, int d) {
                hn v;
#pragma unroll
                for (int j = 0; j < N; j++) v[j] = x[i + j];
                *(hn*)(to + d) = v;
            });
        }
    };

    const bool has = tid < 2 * D;                                        // 32 D / 16 units of K, as many of V
    const int kt = t0 + tid / (D / 16), ku = tid % (D / 16);
    const int vt = t0 + 8 * (tid & 3), vd = 2 * (tid >> 2);
    _Float16 xk[16], xv[16];
    if (has && (whole || (each && kt >= r0 && kt < total))) {
        if (kt < len) load_ring_k(kt, ku, xk);
        else load_new_k(kt, ku, xk);
    }
    if (has && (whole || each)) {
        if (whole && vt < len) {                                         // 8 tokens of a feature side by side
            load_row<8, true, true>(ring_v, vd * kKvRing + vt % kKvRing, 1, xv);
            load_row<8, true, true>(ring_v, (vd + 1) * kKvRing + vt % kKvRing, 1, xv + 8);
        }
        load_v8(vt, vd, len, xv);
    }
    if (has && each) {
        if (kt >= r0 && kt < total) put_ring_k(kt, ku, xk);
        ring_v8(vt, vd, xv);
    }
    if (whole) {
        const int64_t page = page_of(c, b, t0 / kKvBlock);
        uint32_t m[2] = {0, 0};
        auto widen = [](uint32_t m, _Float16 x) {
            const uint32_t u = __builtin_bit_cast(uint16_t, x) & 0x7fffu;
            return m > u ? m : u;
        };
        if (has) {
#pragma unroll
            for (int i = 0; i < 16; i++) m[0] = widen(m[0], xk[i]), m[1] = widen(m[1], xv[i]);
        }
#pragma unroll
        for (int w = 0; w < 2; w++) {
#pragma unroll
            for (int i = 1; i < 64; i <<= 1) {
                const uint32_t o = __shfl_xor(m[w], i);
                m[w] = m[w] > o ? m[w] : o;
            }
            if ((tid & 63) == 0) mx[w][tid >> 6] = m[w];
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 2; w++) {
            uint32_t u = 0;
#pragma unroll
            for (int i = 0; i < NT / 64; i++) u = u > mx[w][i] ? u : mx[w][i];
            const float top = h2f(u), d = top / 127.f, id = u && u < 0x7c00u ? 127.f / top : 0.f;
            if (page < 0 || !has) continue;
            const _Float16* x = w ? xv : xk;
            u32x4 q = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
            if (id > 0.f)
#pragma unroll
                for (int i = 0; i < 16; i++) q[i >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(code_of(x[i], d, id), i & 3, q[i >> 2]);
            const int64_t block = (page * c.Hkv + hk) * kKvBlock * D;
            if (ROT == 0 || w) {
                *(u32x4*)((w ? c.v : c.k) + block + (int64_t)16 * tid) = q;
            } else {
                uint8_t* to = c.k + block + (kt - t0) * D;
                runs(ku, [&](int i, int f) {
                    if constexpr (N == 8) {
                        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
                        *(u32x2*)(to + f) = u32x2{q[i / 4], q[i / 4 + 1]};
                    } else if constexpr (N == 4) {
                        *(uint32_t*)(to + f) = q[i / 4];
                    } else {
                        to[f] = (uint8_t)(q[i / 4] >> (8 * (i % 4)));
                    }
                });
            }
            if (tid == 0) c.scales[(page * c.Hkv + hk) * 2 + w] = d;
        }
    }
    if (each || blockIdx.x) return;
    __syncthreads();                     // what the ring held has been read
    if constexpr (ROT == 0) {
        for (int i = tid; i < (total - r0) * (D / 8); i += NT) {
            const int t = r0 + i / (D / 8), d = 8 * (i % (D / 8));
            _Float16 x[8];
            load_row<8, IN16, VEC>(a.k, at(t, d), a.st[0], x);
            *(f16x8*)(ring_k + (t % kKvRing) * D + d) = halves(x);
        }
    } else {
        for (int i = tid; i < (total - r0) * (D / 16); i += NT) {
            _Float16 x[16];
            load_new_k(r0 + i / (D / 16), i % (D / 16), x);
            put_ring_k(r0 + i / (D / 16), i % (D / 16), x);
        }
    }
    const int g0 = r0 >> 3, groups = ((total + 7) >> 3) - g0;
    for (int i = tid; i < groups * (D / 2); i += NT) {
        const int t = 8 * (g0 + i / (D / 2)), d = 2 * (i % (D / 2));
        _Float16 x[16];
        load_v8(t, d, r0, x);
        ring_v8(t, d, x);
    }
}

template <bool IN16, bool VEC>
__global__ __launch_bounds__(256) void k_kv8_append(Kv8AppendArgs a) {
    append_block<IN16, VEC, 0, 256>(a, nullptr);
}

// The same with the keys rotated, and workgroups past the first `blocks` of a head and sequence rotating its query heads:
// V pairs of the heads g, g + HG, ... of one token per thread, so that their angles are computed once.
template <bool IN16, bool VEC, int ROT, int V, int NT>
__global__ __launch_bounds__(NT) void k_kv8_append_rope(Kv8RopeArgs a, int blocks, int HG) {
    ask_rotation(a.r);
    asm volatile("" ::"s"(a.a.c.max_blocks), "s"(a.a.c.D), "s"(a.a.c.Hkv), "s"(a.a.lens), "s"(a.a.fresh), "s"(a.a.S));
    if ((int)blockIdx.x < blocks) {
        append_block<IN16, VEC, ROT, NT>(a.a, &a.r);
        return;
    }
    const Kv8& c = a.a.c;
    asm volatile("" ::"s"(a.q), "s"(a.qo), "s"(a.qst[0]), "s"(a.qst[1]), "s"(a.qst[2]), "s"(a.qst[3]), "s"(a.qost[0]), "s"(a.qost[1]),
                 "s"(a.qost[2]), "s"(a.qost[3]), "s"(a.H), "s"(c.Hkv), "s"(c.D));
    const int hk = blockIdx.y, b = blockIdx.z, G = a.H / c.Hkv, units = c.D / (2 * V), per = units * HG;
    const uint32_t at = (blockIdx.x - blocks) * (uint32_t)NT, i0 = at / per;
    const int x = (int)(at - i0 * per) + threadIdx.x, di = x / per, item = x - di * per;
    const int i = (int)i0 + di, g = item / units, pair = (item - g * units) * V, h = hk * G + g;
    Turns<V> f;
    f.load(a.r, pair);
    int len, total;
    const bool fits = spans(c, a.a.lens, a.a.fresh, a.a.S, b, len, total);
    const TokenPos t = token_pos(a.r, b, min(i, a.a.S - 1), len + i);
    if (!fits || i >= total - len) return;
    rope_heads<V, IN16, true, (V > 1)>(a.r, t, f, pair, a.q, b * a.qst[3] + i * a.qst[1] + h * a.qst[2], HG * a.qst[2], a.qst[0], a.qo,
                                       b * a.qost[3] + i * a.qost[1] + h * a.qost[2], HG * a.qost[2], a.qost[0], (G - g + HG - 1) / HG);
}

// Values of tokens [first, first + n) that a sequence has: codes times their scale, or the ring's fp16. One
// workgroup per block that the call touches; V, whose features lie apart, goes through LDS. Four times 2050 tokens of 8
// heads of 128 to fp16, 50 MB: 10.7 us (4.7 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8ReadArgs a, T* out_k, T* out_v) {
    constexpr int LD = 128 + 8;
    __shared__ __attribute__((aligned(16))) _Float16 vs[kKvBlock * LD];
    const Kv8& c = a.c;
    const int hk = blockIdx.y, b = blockIdx.z, D = c.D, tid = threadIdx.x;
    const int total = a.lens[b], first = a.first ? a.first[b] : 0;
    const int64_t row = ((int64_t)b * c.Hkv + hk) * a.n;
    const float nan = __builtin_nanf("");
    if (total < 0 || first < 0 || total > (int64_t)c.max_blocks * kKvBlock) {     // numbers that the cache cannot hold
        for (int i = tid; i < kKvBlock * D; i += 256) {
            const int64_t t = (int64_t)blockIdx.x * kKvBlock + i / D;
            if (t < a.n) out_k[(row + t) * D + i % D] = out_v[(row + t) * D + i % D] = (T)nan;
        }
        return;
    }
    const int64_t t0 = (first & ~(kKvBlock - 1)) + (int64_t)kKvBlock * blockIdx.x;
    if (t0 >= total) return;
    const bool whole = t0 + kKvBlock <= total;
    int64_t page = whole ? page_of(c, b, (int)(t0 / kKvBlock)) : 0;
    const bool lost = page < 0;
    const int64_t at = (lost ? 0 : page) * c.Hkv + hk;
    const float dk = !whole ? 1.f : lost ? nan : c.scales[2 * at], dv = !whole ? 1.f : lost ? nan : c.scales[2 * at + 1];
    const int64_t ring = ((int64_t)b * c.Hkv + hk) * kKvRing * D;
    const bool has = tid < 2 * D;
    const int s = tid / (D / 16), d0 = 16 * (tid % (D / 16));            // this thread's token of the block and features
    float k[16];
    if (has) {
        const int vt = 8 * (tid & 3), vd = 2 * (tid >> 2);               // and the 2 x 8 values of V that it moves
        if (whole) {
            u32x4 qk = {0, 0, 0, 0}, qv = {0, 0, 0, 0};
            if (!lost) {
                qk = *(const u32x4*)(c.k + at * kKvBlock * D + 16 * tid);
                qv = *(const u32x4*)(c.v + at * kKvBlock * D + 16 * tid);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                k[i] = (float)((int)(qk[i >> 2] >> (8 * (i & 3)) & 255) - 128) * dk;
                vs[(vt + (i & 7)) * LD + vd + (i >> 3)] = (_Float16)((int)(qv[i >> 2] >> (8 * (i & 3)) & 255) - 128);
            }
        } else {
            const int slot = (int)(t0 % kKvRing);
            _Float16 x[16];
            load_row<16, true, true>(c.k_tail + ring, (slot + s) * D + d0, 1, x);
#pragma unroll
            for (int i = 0; i < 16; i++) k[i] = (float)x[i];
            load_row<8, true, true>(c.v_tail + ring, vd * kKvRing + slot + vt, 1, x);
            load_row<8, true, true>(c.v_tail + ring, (vd + 1) * kKvRing + slot + vt, 1, x + 8);
#pragma unroll
            for (int i = 0; i < 16; i++) vs[(vt + (i & 7)) * LD + vd + (i >> 3)] = x[i];
        }
    }
    __syncthreads();
    const int64_t t = t0 + s, o = t - first;
    if (!has || o < 0 || o >= a.n || t >= total) return;
    const int64_t e = (row + o) * D + d0;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = (float)vs[s * LD + d0 + i] * dv;
    if (a.vec) {
        typedef T tn __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 16; i += N) {
            tn pk, pv;
#pragma unroll
            for (int j = 0; j < N; j++) pk[j] = (T)k[i + j], pv[j] = (T)v[i + j];
            *(tn*)(out_k + e + i) = pk;
            *(tn*)(out_v + e + i) = pv;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) out_k[e + i] = (T)k[i], out_v[e + i] = (T)v[i];
    }
}

// Lengths after a step. Numbers that append and attention refuse (spans) leave the length as it is, so that the next
// step refuses it too instead of taking ring slots that were never written for tokens. Past the table, whose width is
// not at hand here, the length grows: no later call takes it either.
__global__ void k_kv8_advance(int32_t* lens, const int32_t* fresh, int B, int S) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= B) return;
    const int len = lens[b], n = fresh ? fresh[b] : S;
    if (len >= 0 && n >= 0 && n <= S && n <= INT32_MAX - len) lens[b] = len + n;
}

}  // namespace

hipError_t launch_kv8_append(const Kv8AppendArgs& a, hipStream_t s) {
    // blocks that S tokens can touch: the open one and what follows
    const dim3 grid((unsigned)(((int64_t)a.S + 2 * kKvBlock - 2) / kKvBlock), (unsigned)a.c.Hkv, (unsigned)a.c.B);
    if (a.in16 && a.vec) hipLaunchKernelGGL((k_kv8_append<true, true>), grid, dim3(256), 0, s, a);
    else if (a.in16) hipLaunchKernelGGL((k_kv8_append<true, false>), grid, dim3(256), 0, s, a);
    else if (a.vec) hipLaunchKernelGGL((k_kv8_append<false, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_kv8_append<false, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

namespace {

template <bool IN16, int ROT, int NT>
void launch_append_rope(const Kv8RopeArgs& a, bool vec_q, dim3 grid, int blocks, int hg, hipStream_t s) {
    auto go = [&](auto vec) {
        constexpr bool VEC = decltype(vec)::value;
        if (vec_q) hipLaunchKernelGGL((k_kv8_append_rope<IN16, VEC, ROT, ROT, NT>), grid, dim3(NT), 0, s, a, blocks, hg);
        else hipLaunchKernelGGL((k_kv8_append_rope<IN16, VEC, ROT, 1, NT>), grid, dim3(NT), 0, s, a, blocks, hg);
    };
    if (a.a.vec) go(std::true_type{});
    else go(std::false_type{});
}

}  // namespace

hipError_t launch_kv8_append_rope(const Kv8RopeArgs& a, hipStream_t s) {
    const int blocks = (int)(((int64_t)a.a.S + 2 * kKvBlock - 2) / kKvBlock), D = a.a.c.D, rot = rope_granule(a.r, D);
    const bool vec_q = a.vec_q >= rot;
    const int v = vec_q ? rot : 1;
    // up to 8 heads of a thread: with one head each 4 prompts of 2050 tokens (32 heads of 128 on 8, read back) take 73.4 us instead
    // of 58.1; with more only where 8 waves per SIMD are left, 3 x 812 (16 heads of 112 on 4) 21.0 instead of 17.3 and 54 x 11 17.6
    // instead of 14.5
    const int G = a.q ? a.H / a.a.c.Hkv : 1, hg = (G + 7) / 8;
    const int64_t per = (int64_t)hg * (D / (2 * v));
    // 2 D threads have codes of a block: 128 where that is enough (4 x 1025 tokens, 16 heads of 48 in fp32, read back: 27.9 us, with
    // 256 threads 31.2; calls of a few tokens the same)
    const int nt = 2 * D <= 128 ? 128 : 256;
    const int64_t wgs = a.q ? ((int64_t)a.a.S * per + nt - 1) / nt : 0;
    const dim3 grid((unsigned)(blocks + wgs), (unsigned)a.a.c.Hkv, (unsigned)a.a.c.B);
    auto go = [&](auto in16, auto threads) {
        constexpr bool IN16 = decltype(in16)::value;
        constexpr int NT = decltype(threads)::value;
        if (rot == 8) launch_append_rope<IN16, 8, NT>(a, vec_q, grid, blocks, hg, s);
        else if (rot == 4) launch_append_rope<IN16, 4, NT>(a, vec_q, grid, blocks, hg, s);
        else launch_append_rope<IN16, 1, NT>(a, vec_q, grid, blocks, hg, s);
    };
    auto of = [&](auto in16) {
        if (nt == 128) go(in16, std::integral_constant<int, 128>{});
        else go(in16, std::integral_constant<int, 256>{});
    };
    if (a.a.in16) of(std::true_type{});
    else of(std::false_type{});
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8ReadArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(((int64_t)a.n + 2 * kKvBlock - 2) / kKvBlock), (unsigned)a.c.Hkv, (unsigned)a.c.B);
    if (a.k16) hipLaunchKernelGGL(k_kv8_read<_Float16>, grid, dim3(256), 0, s, a, a.k16, a.v16);
    else hipLaunchKernelGGL(k_kv8_read<float>, grid, dim3(256), 0, s, a, a.k, a.v);
    return hipGetLastError();
}

hipError_t launch_kv8_advance(int32_t* lens, const int32_t* fresh, int B, int S, hipStream_t s) {
    hipLaunchKernelGGL(k_kv8_advance, dim3((unsigned)((B + 255) / 256)), dim3(256), 0, s, lens, fresh, B, S);
    return hipGetLastError();
}

}  // namespace mgh
