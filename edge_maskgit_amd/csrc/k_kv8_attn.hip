// k_kv8_attn.hip — attention of the newest tokens over the 8-bit cache (gfx950).
//
// Bound by the cache's bytes: 2 D bytes per token and key head against 4 D flop per query row. A workgroup
// takes one key head's rows (the G = H / Hkv query heads of each new token, 16 QT rows) over a part of the
// sequence's blocks; its 4 waves take every fourth block each, straight from memory to registers, the next
// block's 2 x 32 D bytes on their way while one is computed, with no barrier until their states are joined
// in LDS; parts of a sequence are joined by a second kernel. The parts are cut on the device from the lengths
// there, so a captured call serves a growing sequence.
//  * A lane's 16 bytes of K are 16 features of one key, its 16 bytes of V two features of 8 keys: both are
//    operands of v_mfma_f32_16x16x32_f16 once each byte is a fp16 (the byte under the exponent of 1024, minus
//    1152: exact, one permutation and one packed addition per two codes). Which key is which row of the
//    score operand is free, so scores come out as the 8 consecutive keys that V's operand needs.
//  * Codes stay whole numbers in the products; K's scale multiplies a block's scores, V's its share of the
//    output, both in fp32. Weights are fp16 (hi + lo for an fp32 output, PS).
//  * The tokens behind the last whole block are one more block, of fp16 rows.
// Rows that are not finite (a scale of V that is not, infinities among the open block's values, weights past fp16
// where scores lie farther apart than the reference's distance), and all rows of a part with a page outside the pool, are
// taken again by attn_row.
//
// Measured (32 heads on 8 of 128): one sequence of 100000 tokens, 205 MB, 39.5 us (5.2 TB/s) and the join 4.8; 64 of 2700
// tokens 69 us (5.2 TB/s), of up to 8000 with capped scores 90 (4.1 TB/s: long sequences' parts at the end). A block takes
// a wave 0.88 us, so short sequences are latency: 4 of 1030, 16 heads of 48, five rows: 7.3 us and the join 2.8.
#include <algorithm>

#include "k_attn_row.h"
#include "k_kv8.h"

namespace mgh {

namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct CacheSrc {
    const Kv8& c;
    int b, hk, cut;        // tokens before `cut` are in whole blocks
    __device__ bool seen(int64_t) const { return true; }
    __device__ float dot(int64_t j, const float* qs) const {
        float s = 0.f;
        if (j < cut) {
            const int64_t page = page_of(c, b, (int)(j / kKvBlock));
            if (page < 0) return __builtin_nanf("");
            const uint8_t* k = c.k + ((page * c.Hkv + hk) * kKvBlock + j % kKvBlock) * c.D;
            for (int d = 0; d < c.D; d += 16) {
                const u32x4 x = *(const u32x4*)(k + d);
#pragma unroll
                for (int i = 0; i < 16; i++) s = fmaf(qs[d + i], (float)((int)(x[i >> 2] >> (8 * (i & 3)) & 255) - 128), s);
            }
            return s * c.scales[(page * c.Hkv + hk) * 2];
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
            const int64_t page = page_of(c, b, (int)(j / kKvBlock));
            if (page < 0) return __builtin_nanf("");
            const int64_t at = page * c.Hkv + hk;
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

// DG 32-feature groups (D <= 32 DG), QT 16-row tiles, PS: weights as hi + lo, MOD: capped or sloped
template <int DG, int QT, bool PS, bool MOD>
__global__ __launch_bounds__(256, QT == 1 ? 3 : 2) void k_kv8_attn(Kv8AttnArgs a, int tiles, int splits, int least) {
    constexpr int DK = (DG + 1) / 2, ROWS = 16 * QT, OLD = 32 * DG + 4;
    __shared__ __attribute__((aligned(16))) float so[4][ROWS][OLD];
    __shared__ float sm[4][ROWS][2];
    __shared__ int odd[ROWS], gone[4];
    const Kv8& cache = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lg = lane >> 4, D = cache.D;
    // heads innermost, so that each XCD (blockIdx % 8) gets as many of the first parts, which every sequence has
    const int heads = cache.Hkv * cache.B, hb = blockIdx.x % heads, in_h = blockIdx.x / heads;
    const int sp = in_h / tiles, tile = in_h - sp * tiles;
    const int hk = hb % cache.Hkv, b = hb / cache.Hkv, G = a.H / cache.Hkv;
    int len, total;
    const bool fits = spans(cache, a.lens, a.fresh, a.S, b, len, total);
    const int R = (fits ? total - len : a.S) * G, RS = a.S * G, r0 = tile * ROWS;
    const int64_t rows = (int64_t)cache.B * cache.Hkv * RS, row0 = (int64_t)hb * RS;
    float* ml = a.ws + splits * rows * D;

    // blocks of this part: whole ones, then the open one; none past what the tile's last row sees
    const int whole = fits ? total / kKvBlock : 0, cut = whole * kKvBlock;
    const int last = r0 < R ? len + (min(r0 + ROWS, R) - 1) / G : -1;       // the last row's position
    const int nb = fits && r0 < R ? min((total + kKvBlock - 1) / kKvBlock, last / kKvBlock + 1) : 0;
    const int per = max((nb + splits - 1) / splits, least), b0 = min(sp * per, nb), b1 = min(b0 + per, nb);

    // rows past the sequence's own: marked for the joining kernel, which leaves them alone; a part without blocks: 0
    if (splits > 1 && tid < ROWS && r0 + tid < RS && (r0 + tid >= R || b0 >= b1))
        *(f32x2*)(ml + 2 * (sp * rows + row0 + r0 + tid)) = f32x2{kNoScore, r0 + tid >= R ? -1.f : 0.f};
    if (splits > 1 && b0 >= b1 && fits) return;

    // rows of Q as the B operand: features 64 g + 16 lg + 8 j + e
    f16x8 qf[QT][2 * DK];
    float slope2[QT];
    int lim[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int r = min(r0 + 16 * t + l16, RS - 1), i = r / G, g = r - i * G;
        lim[t] = r0 + 16 * t + l16 < R ? len + i : -1;
        slope2[t] = MOD && a.slopes ? a.slopes[hk * G + g] * kLog2e : 0.f;
        const int64_t e = b * a.qst[3] + (int64_t)(hk * G + g) * a.qst[2] + i * a.qst[1];
#pragma unroll
        for (int c = 0; c < 2 * DK; c++) {
            const int d = 64 * (c >> 1) + 16 * lg + 8 * (c & 1);
            qf[t][c] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (d < D && lim[t] >= 0) {
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

    // where this lane reads in a block: K's key and features of tile t (+ 4 keys), V's feature pair and keys;
    // lanes past D read some code of the block, which is finite and meets a zero of Q or is not stored
    const int key = 8 * (l16 >> 2) + (l16 & 3);
    uint32_t ka[DK], va[DG];
#pragma unroll
    for (int g = 0; g < DK; g++) ka[g] = key * D + (64 * g + 16 * lg < D ? 64 * g + 16 * lg : 0);
#pragma unroll
    for (int g = 0; g < DG; g++) va[g] = 32 * g + 2 * l16 < D ? ((16 * g + l16) * 4 + lg) * 16 : 0;

    float mref[QT], S1[QT];
    f32x4 O[QT][2 * DG];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        mref[t] = kNoScore;
        S1[t] = 0.f;
#pragma unroll
        for (int c = 0; c < 2 * DG; c++) O[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const f16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};

    // one block: kf(t, c) K's fragment of key tile t and features c, vf(c) V's of features 32 (c / 2) + 2 l16 + c % 2
    auto block = [&](int blk, float ks, float vs, auto kf, auto vf) {
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
        const int j0 = blk * kKvBlock + 8 * lg;              // this lane's keys: j0 + 4 n + r
        const float scale = ks * (MOD && a.mod.cap2 != 0.f ? 1.f : a.mod.scale2);
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
        if (MOD && a.mod.cap2 != 0.f) {
            float big = 0.f;
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    big = fmaxf(fmaxf(big, fabsf(sc[t][n][0])), fabsf(sc[t][n][1]));
                    big = fmaxf(fmaxf(big, fabsf(sc[t][n][2])), fabsf(sc[t][n][3]));
                }
            if (all_small(big * scale, a.mod)) mapped([&](float x) { return cap_small(x, a.mod); });
            else mapped([&](float x) { return cap_score(x, a.mod); });
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
                    const float s = j0 + 4 * n + r > lim[t] ? -INFINITY : sc[t][n][r];
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
    };

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
        block(blk, x.s[0], x.s[1],
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
    if (b1 > whole && b0 <= whole && ((whole - b0) & 3) == wave) {
        const int64_t at = (int64_t)b * cache.Hkv + hk;
        const _Float16* K = cache.k_tail + at * kKvRing * D;
        const _Float16* V = cache.v_tail + at * D * kKvRing;
        const int slot = cut % kKvRing, left = total - cut - 8 * lg;         // values of this lane's 8 keys
        block(whole, 1.f, 1.f,
              [&](int n, int c) {
                  const int d = 64 * (c >> 1) + 16 * lg + 8 * (c & 1);
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
                const f32x4 v = {O[t][2 * g][2 * h], O[t][2 * g + 1][2 * h], O[t][2 * g][2 * h + 1], O[t][2 * g + 1][2 * h + 1]};
                *(f32x4*)&so[wave][16 * t + l16][32 * g + 8 * lg + 4 * h] = v;
            }
        if (lg == 0) sm[wave][16 * t + l16][0] = mref[t], sm[wave][16 * t + l16][1] = S1[t];
    }
    if (tid < ROWS) odd[tid] = 0;
    if (lane == 0) gone[wave] = lost;
    __syncthreads();
    const bool again = !fits || gone[0] || gone[1] || gone[2] || gone[3];
    auto put = [&](int r, int d, f32x4 o, float m, float l) {
        if (splits > 1) {
            *(f32x4*)(a.ws + (sp * rows + row0 + r) * D + d) = o;
            if (d == 0) *(f32x2*)(ml + 2 * (sp * rows + row0 + r)) = f32x2{m, l};
            return;
        }
        const int i = r / G, g = r - i * G;
        const int64_t e = b * a.ost[3] + (int64_t)(hk * G + g) * a.ost[2] + i * a.ost[1];
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
        if (again || !(z - z == 0.f)) odd[x / (D / 4)] = 1;
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
        if (!odd[r]) continue;
        const int i = (r0 + r) / G, g = r0 + r - i * G;
        RowState st{0.f, 1.f, {__builtin_nanf(""), __builtin_nanf("")}};
        if (fits) {
            const int64_t e = b * a.qst[3] + (int64_t)(hk * G + g) * a.qst[2] + i * a.qst[1];
            for (int d = lane; d < D; d += 64) {
                const int64_t x = e + d * a.qst[0];
                qs[d] = a.in16 ? (float)((const _Float16*)a.q)[x] : (float)(_Float16)((const float*)a.q)[x];
            }
            __builtin_amdgcn_wave_barrier();
            const int64_t p = (int64_t)len + i;
            st = attn_row(CacheSrc{cache, b, hk, cut}, a.mod, a.slopes ? a.slopes[hk * G + g] * kLog2e : 0.f, p, p + 1,
                          (int64_t)b0 * kKvBlock, min((int64_t)b1 * kKvBlock, p + 1), D, qs, qs + 128, lane);
            __builtin_amdgcn_wave_barrier();
        }
        qs[lane] = st.o[0], qs[lane + 64] = st.o[1];
        __builtin_amdgcn_wave_barrier();
        if (4 * lane < D) put(r0 + r, 4 * lane, *(const f32x4*)&qs[4 * lane], st.m == -INFINITY ? kNoScore : st.m, st.l);
        __builtin_amdgcn_wave_barrier();
    }
}

template <int DG, int QT, bool PS>
void launch_cache_t(const Kv8AttnArgs& a, const Kv8Plan& p, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.tiles * p.splits * a.c.Hkv * a.c.B));
    if (a.mod.cap2 != 0.f || a.slopes) hipLaunchKernelGGL((k_kv8_attn<DG, QT, PS, true>), grid, dim3(256), 0, s, a, p.tiles, p.splits, p.least);
    else hipLaunchKernelGGL((k_kv8_attn<DG, QT, PS, false>), grid, dim3(256), 0, s, a, p.tiles, p.splits, p.least);
}

template <int DG>
void launch_cache_d(const Kv8AttnArgs& a, const Kv8Plan& p, hipStream_t s) {
    if (p.qt == 2) {
        if (a.o16) launch_cache_t<DG, 2, false>(a, p, s);
        else launch_cache_t<DG, 2, true>(a, p, s);
    } else {
        if (a.o16) launch_cache_t<DG, 1, false>(a, p, s);
        else launch_cache_t<DG, 1, true>(a, p, s);
    }
}

}  // namespace

Kv8Plan kv8_plan(const Kv8AttnArgs& a) {
    const int64_t R = (int64_t)a.S * (a.H / a.c.Hkv), heads = (int64_t)a.c.Hkv * a.c.B;
    Kv8Plan p{};
    // Past 16 rows two tiles share the codes' way to operands: 32 rows over 100000 tokens 51 against 59 us with one, 20 rows
    // 48 / 55, 32 rows over 16 sequences of up to 5000 35 / 38, 64 rows 46 / 58.
    p.qt = R > 16 ? 2 : 1;
    p.tiles = (int)((R + 16 * p.qt - 1) / (16 * p.qt));
    const int64_t wgs = heads * p.tiles;
    // Few workgroups: parts until every CU has one, of at least 8 blocks (2 per wave). Enough of them: parts only of
    // sequences past 96 blocks, for the balance of ragged batches (the table's width is all that the host knows of
    // their lengths): a second launch costs 3-6 us. (Of 48, 64 or 96 blocks: 64 of 2700 80 / 78 / 71 us, 64 of up
    // to 8000 92 / 90 / 95.) Measured (32 heads on 8 of 128 features, one token), parts
    // 1 / 2 / 3 / 4 / 8 / 32: one sequence of 100000 tokens 631 / 323 / 221 / 169 / 92 / 45 us, one of 9000 68 / 42 / 31 / 27 /
    // 19 / 14, 16 of 9000 78 / 61 / 68 / 62 / 65 / 74, 64 of 2700 69 / 77 / 74 / 79 / 86 / 105, 64 of up to 8000 98 / 104 / 93 / 93 /
    // 92 / 114, 64 of up to 500 14 / 22 / 19 / 25 / 20 / 40.
    const int fill = (int)std::max<int64_t>(1, (256 + wgs - 1) / wgs), least = fill > 1 ? 192 * fill : 96;
    p.least = fill > 1 ? 8 : 96;
    p.splits = (int)std::min<int64_t>(kMostSplits, (int64_t)fill * std::max(1, (a.c.max_blocks + least - 1) / least));
    // (a table far wider than its sequences: no more than 8 workgroups per CU, most of them without blocks)
    p.splits = (int)std::min<int64_t>(p.splits, std::max<int64_t>(1, 2048 / wgs));
    p.splits = std::max(1, std::min(p.splits, (a.c.max_blocks + p.least - 1) / p.least));
    if (p.splits > 1) p.ws_bytes = (size_t)p.splits * heads * R * (a.c.D + 2) * sizeof(float);
    return p;
}

hipError_t launch_kv8_attn(const Kv8AttnArgs& a, const Kv8Plan& p, hipStream_t s) {
    switch ((a.c.D + 31) / 32) {
        case 1: launch_cache_d<1>(a, p, s); break;
        case 2: launch_cache_d<2>(a, p, s); break;
        case 3: launch_cache_d<3>(a, p, s); break;
        default: launch_cache_d<4>(a, p, s); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    JoinArgs j{};
    j.ws = a.ws; j.o = a.o; j.o16 = a.o16;
    for (int i = 0; i < 4; i++) j.ost[i] = a.ost[i];
    j.G = a.H / a.c.Hkv; j.Hkv = a.c.Hkv; j.D = a.c.D; j.splits = p.splits;
    j.vec_o = a.vec_o;
    j.R = a.S * j.G;
    j.rows = j.R * a.c.Hkv * a.c.B;
    return launch_attn_join(j, s);
}

}  // namespace mgh
