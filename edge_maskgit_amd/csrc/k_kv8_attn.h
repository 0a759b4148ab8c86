// k_kv8_attn.h — attention of rows over blocks of the 8-bit cache, by one workgroup (k_kv8_attn.hip has the method).
#pragma once
#include <type_traits>

#include "k_attn_row.h"
#include "k_kv8.h"

namespace mgh {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// values of a sequence's tokens in the cache
struct CacheSrc {
    const Kv8& c;
    int b, hk, cut;        // tokens before `cut` are in whole blocks
    int b1, same;          // the first `same` blocks' pages are those of sequence b1
    __device__ int64_t page(int64_t block) const { return page_of(c, block < same ? b1 : b, (int)block); }
    __device__ bool seen(int64_t) const { return true; }
    __device__ float dot(int64_t j, const float* qs) const {
        float s = 0.f;
        if (j < cut) {
            const int64_t at_page = page(j / kKvBlock);
            if (at_page < 0) return __builtin_nanf("");
            const uint8_t* k = c.k + ((at_page * c.Hkv + hk) * kKvBlock + j % kKvBlock) * c.D;
            for (int d = 0; d < c.D; d += 16) {
                const u32x4 x = *(const u32x4*)(k + d);
#pragma unroll
                for (int i = 0; i < 16; i++) s = fmaf(qs[d + i], (float)((int)(x[i >> 2] >> (8 * (i & 3)) & 255) - 128), s);
            }
            return s * c.scales[(at_page * c.Hkv + hk) * 2];
        }
        const _Float16* k = c.k_tail + (((int64_t)b * c.Hkv + hk) * kKvRing + j % kKvRing) * c.D;
        for (int d = 0; d < c.D; d += 8) {
            const f16x8 x = *(const f16x8*)(k + d);
#pragma unroll
            for (int i = 0; i < 8; i++) s = fmaf(qs[d + i], (float)x[i], s);
        }
        return s;
    }
    __device__ float value(int64_t j, int d) const {
        if (j < cut) {
            const int64_t at_page = page(j / kKvBlock);
            if (at_page < 0) return __builtin_nanf("");
            const int64_t at = at_page * c.Hkv + hk;
            return (float)((int)c.v[at * kKvBlock * c.D + v_at((int)(j % kKvBlock), d)] - 128) * c.scales[2 * at + 1];
        }
        return (float)c.v_tail[(((int64_t)b * c.Hkv + hk) * c.D + d) * kKvRing + j % kKvRing];
    }
};

// 8 codes + 128 as fp16 codes
__device__ __forceinline__ f16x8 widen(uint32_t a, uint32_t b) {
    const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
    auto two = [&](uint32_t x, uint32_t sel) {
        const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, sel)) - off;
        return __builtin_bit_cast(uint32_t, h);
    };
    const u32x4 v = {two(a, 0x04010400u), two(a, 0x04030402u), two(b, 0x04010400u), two(b, 0x04030402u)};
    return __builtin_bit_cast(f16x8, v);
}

// A wave's QT tiles of 16 rows on their way over the blocks: lane l16 + 16 lg holds row l16's scores of the keys 8 lg + 0 .. 7 of a
// block, and its output's features 32 g + 8 lg + 2 r + (c & 1), c = 2 g + ..., r
template <int DG, int QT, bool PS, bool MOD>
struct CacheRows {
    static constexpr int DK = (DG + 1) / 2;
    f16x8 qf[QT][2 * DK];                // rows of Q as the B operand: features 64 g + 16 lg + 8 j + e
    float slope2[QT];
    int lim[QT];                         // a row's position, the last key it sees; -1: none
    float mref[QT], S1[QT];
    f32x4 O[QT][2 * DG];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < QT; t++) {
            mref[t] = kNoScore;
            S1[t] = 0.f;
#pragma unroll
            for (int c = 0; c < 2 * DG; c++) O[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // tile t's row of this lane: sequence b, token i, head h. A branch for each piece: all pieces asked for at once, those that are
    // not there from clamped places, took more registers than it saved waits (64 sequences of up to 8000 tokens, capped, 95.4 us
    // instead of 94.8, of 500 14.9 / 14.6, one of 100000 45.3 / 44.6; 64 on 8000 shared ones 37.7 / 36.9)
    __device__ __forceinline__ void load(const Kv8AttnArgs& a, int t, int b, int i, int h, int last) {
        const int D = a.c.D, lg = (threadIdx.x >> 4) & 3;
        lim[t] = last;
        slope2[t] = MOD && a.slopes ? a.slopes[h] * kLog2e : 0.f;
        const int64_t e = b * a.qst[3] + (int64_t)h * a.qst[2] + i * a.qst[1];
#pragma unroll
        for (int c = 0; c < 2 * DK; c++) {
            const int d = 64 * (c >> 1) + 16 * lg + 8 * (c & 1);
            qf[t][c] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (d < D && last >= 0) {
                if (a.vec_q) {
                    qf[t][c] = *(const f16x8*)((const _Float16*)a.q + e + d);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int64_t x = e + (int64_t)(d + j) * a.qst[0];
                        qf[t][c][j] = a.in16 ? ((const _Float16*)a.q)[x] : (_Float16)((const float*)a.q)[x];
                    }
                }
            }
        }
    }
    // one block: kf(t, c) K's fragment of key tile t and features c, vf(c) V's of features 32 (c / 2) + 2 l16 + c % 2, between(): what
    // is asked for while the scores become weights. MASK: some row may not see some key
    template <bool MASK, class KF, class VF>
    __device__ __forceinline__ void block(const ScoreMod& mod, int blk, float ks, float vs, KF kf, VF vf) {
        block<MASK>(mod, blk, ks, vs, kf, vf, [] {});
    }
    template <bool MASK, class KF, class VF, class B>
    __device__ __forceinline__ void block(const ScoreMod& mod, int blk, float ks, float vs, KF kf, VF vf, B between) {
        const f16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
        f32x4 sc[QT][2];
#pragma unroll
        for (int n = 0; n < 2; n++) {
#pragma unroll
            for (int t = 0; t < QT; t++) sc[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2 * DK; c++) {
                const f16x8 k = kf(n, c);
#pragma unroll
                for (int t = 0; t < QT; t++) sc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[t][c], sc[t][n], 0, 0, 0);
            }
        }
        between();
        const int j0 = blk * kKvBlock + 8 * ((threadIdx.x >> 4) & 3);              // this lane's keys: j0 + 4 n + r
        const float scale = ks * (MOD && mod.cap2 != 0.f ? 1.f : mod.scale2);
        auto mapped = [&](auto map) {                        // scores of the map, then slopes (of the keys that a row sees)
#pragma unroll
            for (int t = 0; t < QT; t++) {
                const float d0 = (float)(lim[t] - j0);
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float s = map(sc[t][n][r] * scale);
                        sc[t][n][r] = MOD ? fmaf(-slope2[t], d0 - (float)(4 * n + r), s) : s;
                    }
            }
        };
        if (MOD && mod.cap2 != 0.f) {
            float big = 0.f;
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    big = fmaxf(fmaxf(big, fabsf(sc[t][n][0])), fabsf(sc[t][n][1]));
                    big = fmaxf(fmaxf(big, fabsf(sc[t][n][2])), fabsf(sc[t][n][3]));
                }
            if (all_small(big * scale, mod)) mapped([&](float x) { return cap_small(x, mod); });
            else mapped([&](float x) { return cap_score(x, mod); });
        } else {
            mapped([](float x) { return x; });
        }
        float mx[QT];
        bool any = false;
#pragma unroll
        for (int t = 0; t < QT; t++) {
            mx[t] = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float s = MASK && j0 + 4 * n + r > lim[t] ? -INFINITY : sc[t][n][r];
                    sc[t][n][r] = s;
                    mx[t] = fmaxf(mx[t], s);
                }
            any = any || __any(mx[t] > mref[t] + 15.f);
        }
        if (any) {
#pragma unroll
            for (int t = 0; t < QT; t++) {
                float v = fmaxf(mx[t] - 7.f, mref[t]);
                v = fmaxf(v, __shfl_xor(v, 16));
                v = fmaxf(v, __shfl_xor(v, 32));
                const float al = __builtin_amdgcn_exp2f(mref[t] - v);
                mref[t] = v;
                S1[t] *= al;
#pragma unroll
                for (int c = 0; c < 2 * DG; c++) O[t][c] *= al;
            }
        }
        f16x8 ph[QT], pl[QT];
#pragma unroll
        for (int t = 0; t < QT; t++) {
            u32x4 hi, lo;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f32x2 e = {__builtin_amdgcn_exp2f(sc[t][j >> 1][2 * (j & 1)] - mref[t]),
                                 __builtin_amdgcn_exp2f(sc[t][j >> 1][2 * (j & 1) + 1] - mref[t])};
                const f16x2 h = __builtin_convertvector(e, f16x2);
                hi[j] = __builtin_bit_cast(uint32_t, h);
                if (PS) {
                    const f32x2 d = {e[0] - (float)h[0], e[1] - (float)h[1]};
                    lo[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(d, f16x2));
                }
            }
            ph[t] = __builtin_bit_cast(f16x8, hi);
            if (PS) pl[t] = __builtin_bit_cast(f16x8, lo);
            f32x4 s1 = {0.f, 0.f, 0.f, 0.f};
            if (PS) s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[t], s1, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph[t], s1, 0, 0, 0);
            S1[t] += s1[0];
        }
#pragma unroll
        for (int c = 0; c < 2 * DG; c++) {
            const f16x8 v = vf(c);
#pragma unroll
            for (int t = 0; t < QT; t++) {
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
                if (PS) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[t], o, 0, 0, 0);
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[t], o, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) O[t][c][r] = fmaf(vs, o[r], O[t][c][r]);
            }
        }
    }
};

// What a workgroup's rows and blocks are. kAlone: one sequence's rows over its blocks. Sequences that share their first
// blocks: kOwn, one sequence's rows over the blocks behind the shared ones; kShared, the rows of all sequences of a
// group over the shared ones, which the group's first sequence's row of the table names and which all its rows see whole.
enum { kAlone, kOwn, kShared };

// tokens of sequence b and the blocks it shares; false: numbers that do not fit
template <int MODE>
__device__ __forceinline__ bool spans_of(const Kv8AttnArgs& a, int b, int& len, int& total, int& same) {
    bool ok = spans(a.c, a.lens, a.fresh, a.S, b, len, total);
    same = 0;
    if (MODE != kAlone) {
        same = a.shared[b / a.group];
        ok = ok && same >= 0 && same <= a.max_shared && (int64_t)same * kKvBlock <= len;
        if (!ok) same = 0;
    }
    return ok;
}

// DG 32-feature groups (D <= 32 DG), QT 16-row tiles, PS: weights as hi + lo, MOD: capped or sloped. The part sp of this
// launch's `splits` is part part0 + sp of all `parts` that the join sees.
template <int DG, int QT>
struct CacheLds {
    __attribute__((aligned(16))) float so[4][16 * QT][32 * DG + 4];
    float sm[4][16 * QT][2];
    int odd[16 * QT], gone[4];
};
template <int DG, int QT, bool PS, bool MOD, int MODE>
__device__ __forceinline__ void cache_attention(const Kv8AttnArgs& a, int wg, int tiles, int splits, int least, int parts, int part0,
                                                CacheLds<DG, QT>& lds) {
    constexpr int DK = (DG + 1) / 2, ROWS = 16 * QT;
    auto& so = lds.so;
    auto& sm = lds.sm;
    auto& odd = lds.odd;
    auto& gone = lds.gone;
    const Kv8& cache = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lg = lane >> 4, D = cache.D;
    // heads innermost, so that each XCD (blockIdx % 8) gets as many of the first parts, which every sequence has
    const int sets = MODE == kShared ? (cache.B + a.group - 1) / a.group : cache.B;
    const int heads = cache.Hkv * sets, hb = wg % heads, in_h = wg / heads;
    const int sp = in_h / tiles, tile = in_h - sp * tiles;
    const int hk = hb % cache.Hkv, G = a.H / cache.Hkv, b = hb / cache.Hkv * (MODE == kShared ? a.group : 1);
    const int RB = a.S * G;                                  // rows of a sequence
    const int64_t rows = (int64_t)cache.B * cache.Hkv * RB;
    float* ml = a.ws + parts * rows * D;
    int len, total, same;
    bool fits;
    if constexpr (MODE == kShared) {
        same = a.shared[b / a.group], len = total = 0, fits = same >= 0 && same <= a.max_shared;
    } else {
        fits = spans_of<MODE>(a, b, len, total, same);
    }
    const int RS = MODE == kShared ? min(a.group, cache.B - b) * RB : RB;
    const int R = MODE == kShared ? RS : (fits ? total - len : a.S) * G, r0 = tile * ROWS;
    // row r of this head: its sequence, index and head among the group's; whether it is one of the call's
    struct Row {
        int b, i, g, p;
        bool live;
    };
    auto row_of = [&](int r) {
        if constexpr (MODE == kShared) {
            const int s = r / RB, x = r - s * RB, i = x / G;
            int l, t, n;
            const bool ok = spans_of<MODE>(a, b + s, l, t, n);
            return Row{b + s, i, x - i * G, l + i, ok && i < t - l};
        } else {
            const int i = r / G;
            return Row{b, i, r - i * G, len + i, r < R};
        }
    };
    auto ws_row = [&](const Row& x) { return ((int64_t)x.b * cache.Hkv + hk) * RB + x.i * G + x.g; };

    // blocks of this part: whole ones, then the open one; none past what the tile's last row sees
    const int whole = MODE == kShared ? same : fits ? total / kKvBlock : 0, cut = whole * kKvBlock;
    const int last = r0 < R ? len + (min(r0 + ROWS, R) - 1) / G : -1;       // the last row's position
    const int lo = MODE == kOwn ? same : 0;
    const int nb = MODE == kShared ? (fits && r0 < R ? same : 0)
                                   : fits && r0 < R ? min((total + kKvBlock - 1) / kKvBlock, last / kKvBlock + 1) - lo : 0;
    const int per = max((nb + splits - 1) / splits, least), b0 = lo + min(sp * per, nb), b1 = lo + min(b0 - lo + per, nb);

    // rows past the sequence's own: marked for the joining kernel, which leaves them alone; a part without blocks: 0
    if constexpr (MODE == kShared) {
        if (tid < ROWS && r0 + tid < RS) {
            const Row x = row_of(r0 + tid);
            odd[tid] = x.live ? 0 : -1;                  // (read past the barriers below)
            if (!x.live || b0 >= b1) *(f32x2*)(ml + 2 * ((part0 + sp) * rows + ws_row(x))) = f32x2{kNoScore, 0.f};
        }
        if (b0 >= b1) return;
    } else {
        if (parts > 1 && tid < ROWS && r0 + tid < RS && (r0 + tid >= R || b0 >= b1))
            *(f32x2*)(ml + 2 * ((part0 + sp) * rows + (int64_t)hb * RS + r0 + tid)) = f32x2{kNoScore, r0 + tid >= R ? -1.f : 0.f};
        if (parts > 1 && b0 >= b1 && fits) return;
    }

    CacheRows<DG, QT, PS, MOD> st;
    st.clear();
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const Row row = row_of(min(r0 + 16 * t + l16, RS - 1));
        st.load(a, t, row.b, row.i, hk * G + row.g, r0 + 16 * t + l16 < R && row.live ? row.p : -1);
    }

    // where this lane reads in a block: K's key and features of tile t (+ 4 keys), V's feature pair and keys;
    // lanes past D read some code of the block, which is finite and meets a zero of Q or is not stored
    const int key = 8 * (l16 >> 2) + (l16 & 3);
    uint32_t ka[DK], va[DG];
#pragma unroll
    for (int g = 0; g < DK; g++) ka[g] = key * D + (64 * g + 16 * lg < D ? 64 * g + 16 * lg : 0);
#pragma unroll
    for (int g = 0; g < DG; g++) va[g] = 32 * g + 2 * l16 < D ? ((16 * g + l16) * 4 + lg) * 16 : 0;

    // this wave's whole blocks b0 + wave, + 4, ..., two sets of registers in turn. Every load is made, past the last
    // block that one's again and for a page outside the pool page 0's: behind a branch around them the compiler
    // could not count the loads and would wait for all. ids: the pages of 64 of the blocks
    struct Set {
        u32x4 k[2 * DK], v[DG];
        f32x2 s;
    };
    const int w1 = min(b1, whole), w0 = b0 + wave;
    bool lost = w0 < w1 && cache.pages == 0;         // a page outside the pool
    int ids = 0, id0 = 0;
    auto load = [&](int blk, Set& x) {
        blk = min(blk, w0 + (w1 - 1 - w0) / 4 * 4);
        if (blk == w0 || blk - id0 >= 256) {
            id0 = blk;
            ids = blk + 4 * lane < w1 ? cache.table[b * cache.table_stride + blk + 4 * lane] : 0;
        }
        const int id = __builtin_amdgcn_readlane(ids, (blk - id0) >> 2);
        const bool in = id >= 0 && id < cache.pages;
        lost = lost || !in;
        const int64_t at = (int64_t)(in ? id : 0) * cache.Hkv + hk;
        const uint8_t* K = cache.k + at * kKvBlock * D;
        const uint8_t* V = cache.v + at * kKvBlock * D;
#pragma unroll
        for (int g = 0; g < DK; g++) {
            x.k[2 * g] = *(const u32x4*)(K + ka[g]);
            x.k[2 * g + 1] = *(const u32x4*)(K + ka[g] + 4 * D);
        }
#pragma unroll
        for (int g = 0; g < DG; g++) x.v[g] = *(const u32x4*)(V + va[g]);
        x.s = *(const f32x2*)(cache.scales + 2 * at);
    };
    auto use = [&](int blk, const Set& x) {
        st.template block<true>(a.mod, blk, x.s[0], x.s[1],
              [&](int n, int c) { const u32x4 w = x.k[2 * (c >> 1) + n]; return c & 1 ? widen(w[2], w[3]) : widen(w[0], w[1]); },
              [&](int c) { const u32x4 w = x.v[c >> 1]; return c & 1 ? widen(w[2], w[3]) : widen(w[0], w[1]); });
    };
    if (w0 < w1 && cache.pages) {
        Set A, B;
        load(w0, A);
        for (int blk = w0; blk < w1; blk += 8) {
            load(blk + 4, B);
            use(blk, A);
            if (blk + 4 >= w1) break;
            load(blk + 8, A);
            use(blk + 4, B);
        }
    }
    // the open block
    if (MODE != kShared && b1 > whole && b0 <= whole && ((whole - b0) & 3) == wave) {
        const int64_t at = (int64_t)b * cache.Hkv + hk;
        const _Float16* K = cache.k_tail + at * kKvRing * D;
        const _Float16* V = cache.v_tail + at * D * kKvRing;
        const int slot = cut % kKvRing, left = total - cut - 8 * lg;         // values of this lane's 8 keys
        // (the compiler is not to know these features for those of Q's rows: it kept a place of them across the loop, whose registers
        // spilled for it. 64 sequences of up to 8000 tokens, capped, 97.0 us with that, 95.4 without)
        int kg = lg;
        asm volatile("" : "+v"(kg));
        st.template block<true>(a.mod, whole, 1.f, 1.f,
              [&](int n, int c) {
                  const int d = 64 * (c >> 1) + 16 * kg + 8 * (c & 1);
                  const f16x8 k = *(const f16x8*)(K + (slot + key + 4 * n) * D + (d < D ? d : 0));
                  // (past D zeros: the key's own values may be infinite, and Q's zeros would make NaN of them)
                  return d < D ? k : f16x8{0, 0, 0, 0, 0, 0, 0, 0};
              },
              [&](int c) {
                  const int d = 32 * (c >> 1) + 2 * l16 + (c & 1);
                  f16x8 v = *(const f16x8*)(V + (d < D ? d : 0) * kKvRing + slot + 8 * lg);
#pragma unroll
                  for (int j = 0; j < 8; j++) v[j] = j < left ? v[j] : (_Float16)0.f;
                  return v;
              });
    }

    // the waves' states, joined by the threads: row, 4 features
#pragma unroll
    for (int t = 0; t < QT; t++) {
#pragma unroll
        for (int g = 0; g < DG; g++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                // features 32 g + 8 lg + 2 r + (c & 1), r = 2 h, 2 h + 1
                const f32x4 v = {st.O[t][2 * g][2 * h], st.O[t][2 * g + 1][2 * h], st.O[t][2 * g][2 * h + 1], st.O[t][2 * g + 1][2 * h + 1]};
                *(f32x4*)&so[wave][16 * t + l16][32 * g + 8 * lg + 4 * h] = v;
            }
        if (lg == 0) sm[wave][16 * t + l16][0] = st.mref[t], sm[wave][16 * t + l16][1] = st.S1[t];
    }
    if (MODE != kShared && tid < ROWS) odd[tid] = 0;
    if (lane == 0) gone[wave] = lost;
    __syncthreads();
    const bool again = !fits || gone[0] || gone[1] || gone[2] || gone[3];
    auto put = [&](int r, int d, f32x4 o, float m, float l) {
        const Row row = row_of(r);
        if (parts > 1) {
            const int64_t at = (part0 + sp) * rows + ws_row(row);
            *(f32x4*)(a.ws + at * D + d) = o;
            if (d == 0) *(f32x2*)(ml + 2 * at) = f32x2{m, l};
            return;
        }
        const int64_t e = row.b * a.ost[3] + (int64_t)(hk * G + row.g) * a.ost[2] + row.i * a.ost[1];
        const f32x4 v = l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o / l;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            if (a.o16) a.o16[e + (d + x) * a.ost[0]] = (_Float16)v[x];
            else a.o[e + (d + x) * a.ost[0]] = v[x];
        }
    };
    const int nr = min(ROWS, R - r0);
    auto join = [&](int x, float& m, float& l) {
        const int r = x / (D / 4), d = 4 * (x - r * (D / 4));
        m = fmaxf(fmaxf(sm[0][r][0], sm[1][r][0]), fmaxf(sm[2][r][0], sm[3][r][0]));
        l = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float al = __builtin_amdgcn_exp2f(sm[w][r][0] - m);
            l = fmaf(al, sm[w][r][1], l);
            o += *(const f32x4*)&so[w][r][d] * al;
        }
        return o;
    };
    for (int x = tid; x < nr * (D / 4); x += 256) {
        float m, l;
        const f32x4 o = join(x, m, l);
        const float z = (o[0] + o[1] + o[2] + o[3]) * 0.f + l;
        if ((again || !(z - z == 0.f)) && (MODE != kShared || odd[x / (D / 4)] == 0)) odd[x / (D / 4)] = 1;
    }
    __syncthreads();
    for (int x = tid; x < nr * (D / 4); x += 256) {
        if (odd[x / (D / 4)]) continue;
        float m, l;
        const f32x4 o = join(x, m, l);
        put(r0 + x / (D / 4), 4 * (x % (D / 4)), o, m, l);
    }
    __syncthreads();
    // rows that are not finite: again, key by key
    float* qs = &so[wave][0][0];
    for (int r = wave; r < nr; r += 4) {
        if (MODE == kShared ? odd[r] != 1 : !odd[r]) continue;
        const Row row = row_of(r0 + r);
        RowState again_st{0.f, 1.f, {__builtin_nanf(""), __builtin_nanf("")}};
        if (fits) {
            const int64_t e = row.b * a.qst[3] + (int64_t)(hk * G + row.g) * a.qst[2] + row.i * a.qst[1];
            for (int d = lane; d < D; d += 64) {
                const int64_t x = e + d * a.qst[0];
                qs[d] = a.in16 ? (float)((const _Float16*)a.q)[x] : (float)(_Float16)((const float*)a.q)[x];
            }
            __builtin_amdgcn_wave_barrier();
            const int64_t p = row.p;
            int row_cut = cut, row_same = same;
            if (MODE == kShared) {
                int l, n;
                spans_of<MODE>(a, row.b, l, n, row_same);
                row_cut = n / kKvBlock * kKvBlock;
            }
            again_st = attn_row(CacheSrc{cache, row.b, hk, row_cut, MODE == kAlone ? b : row.b / a.group * a.group, row_same}, a.mod,
                          a.slopes ? a.slopes[hk * G + row.g] * kLog2e : 0.f, p, p + 1, (int64_t)b0 * kKvBlock,
                          min((int64_t)b1 * kKvBlock, p + 1), D, qs, qs + 128, lane);
            __builtin_amdgcn_wave_barrier();
        }
        qs[lane] = again_st.o[0], qs[lane + 64] = again_st.o[1];
        __builtin_amdgcn_wave_barrier();
        if (4 * lane < D) put(r0 + r, 4 * lane, *(const f32x4*)&qs[4 * lane], again_st.m == -INFINITY ? kNoScore : again_st.m, again_st.l);
        __builtin_amdgcn_wave_barrier();
    }
}

// f(groups of 32 features, 16-row tiles, hi + lo weights, capped or sloped) as constants
template <class F>
inline void with_cache_kernel(const Kv8AttnArgs& a, int qt, F f) {
    using std::integral_constant;
    auto mod = [&](auto dg, auto q, auto ps) {
        if (a.mod.cap2 != 0.f || a.slopes) f(dg, q, ps, std::true_type{});
        else f(dg, q, ps, std::false_type{});
    };
    auto weights = [&](auto dg, auto q) {
        if (a.o16) mod(dg, q, std::false_type{});
        else mod(dg, q, std::true_type{});
    };
    auto rows = [&](auto dg) {
        if (qt == 2) weights(dg, integral_constant<int, 2>{});
        else weights(dg, integral_constant<int, 1>{});
    };
    switch ((a.c.D + 31) / 32) {
        case 1: rows(integral_constant<int, 1>{}); break;
        case 2: rows(integral_constant<int, 2>{}); break;
        case 3: rows(integral_constant<int, 3>{}); break;
        default: rows(integral_constant<int, 4>{}); break;
    }
}

inline hipError_t join_parts(const Kv8AttnArgs& a, int parts, hipStream_t s) {
    JoinArgs j{};
    j.ws = a.ws; j.o = a.o; j.o16 = a.o16;
    for (int i = 0; i < 4; i++) j.ost[i] = a.ost[i];
    j.G = a.H / a.c.Hkv; j.Hkv = a.c.Hkv; j.D = a.c.D; j.splits = parts;
    j.vec_o = a.vec_o;
    j.R = a.S * j.G;
    j.rows = j.R * a.c.Hkv * a.c.B;
    return launch_attn_join(j, s);
}

}  // namespace mgh
