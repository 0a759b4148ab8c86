// k_kv8_shared.hip — attention of the newest tokens over the 8-bit cache where sequences share their first blocks (gfx950).
//
// Softmax over all of a row's keys is the join of softmaxes over parts of them (k_attn_masked.hip has the join): the rows of
// all sequences of a group meet the shared blocks together, so these are read once per tile of rows and not once per
// sequence, each sequence's own blocks follow as in k_kv8_attn.hip, and the parts of both are joined. Shared tokens cost a
// row 4 D flop each and next to no bytes: bound by the VALU that stands beside the matrix products (per 32 rows and 32 keys
// 64 fma that scale a block's share of the output, 64 issue slots of exponentials, 16 to 32 of each other step).
//
// Measured (32 heads on 8 of 128, one launch and the join; in brackets k_kv8_attn on the same tables, which reads the shared
// blocks from the caches): 64 sequences on 8000 shared and up to 500 own tokens 37 us (108; 8.6 GFLOP, 40 MB), 8 groups of 8 on
// up to 4000 with capped scores 31 (58), 32 sequences on 32000 52 (191), 16 on 8000 21 (34), 8 on 8000 18 (22). With few sequences
// there is little to share: 4 on 8000 18 (16), 4 drafts of 5 tokens on 1024 10.4 (9.7). With fp32 outputs 38, 34, 57, 22, 20, 20 and 10.7.
// Loop of one 128-row tile: 1.16 us a block beside the own blocks' workgroups (some 400 instructions a wave); before it 4.8 us of
// dependent loads (arguments, lengths, pages, codes and queries), after it 2 of partial results (17 MB in all).
#include <algorithm>

#include "k_kv8_attn.h"

namespace mgh {

namespace {

// Many rows over the shared blocks: each of the 4 waves has 16 QT rows of its own and all take the same blocks, whose codes go
// through LDS as fp16, once for the workgroup: 16 bytes of codes of a thread become two pieces of 8 values, stored where the
// fragments that the waves read have them (places in a fragment exchanged so that neither side meets a bank twice). The
// next block's codes are on their way from memory while one is computed; one barrier a block.
template <int DG>
struct RowsLds {
    f16x8 buf[2][(4 * ((DG + 1) / 2) + 2 * DG) * 64];
    float again[4][192];
};
template <int DG, int QT, bool PS, bool MOD>
__device__ __forceinline__ void rows_attention(const Kv8AttnArgs& a, int wg, int tiles, int splits, int least, int parts, int part0,
                                               RowsLds<DG>& lds) {
    constexpr int DK = (DG + 1) / 2, KF = 4 * DK, FR = KF + 2 * DG, U = DG > 2 ? 2 : 1;       // fragments of K, of a block; units of a thread
    auto& buf = lds.buf;
    auto& again = lds.again;
    const Kv8& cache = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lg = lane >> 4, D = cache.D;
    const int sets = (cache.B + a.group - 1) / a.group, heads = cache.Hkv * sets, hb = wg % heads, in_h = wg / heads;
    const int sp = in_h / tiles, tile = in_h - sp * tiles, hk = hb % cache.Hkv, set = hb / cache.Hkv, bf = set * a.group;
    const int G = a.H / cache.Hkv, RB = a.S * G, RS = min(a.group, cache.B - bf) * RB, r0 = (tile * 4 + wave) * 16 * QT;
    const int64_t rows = (int64_t)cache.B * cache.Hkv * RB;
    float* ml = a.ws + parts * rows * D;
    const int said = a.shared[set], same = said >= 0 && said <= a.max_shared ? said : 0;
    const int per = max((same + splits - 1) / splits, least), b0 = min(sp * per, same), b1 = min(b0 + per, same);

    struct Row {
        int b, i, h, p;
        bool live;
    };
    auto row_of = [&](int r) {
        const int s = r / RB, x = r - s * RB, i = x / G;
        int len, total, n;
        const bool ok = spans_of<kShared>(a, bf + s, len, total, n);
        return Row{bf + s, i, hk * G + x - i * G, len + i, ok && i < total - len};
    };
    auto at_ws = [&](const Row& x) { return (part0 + sp) * rows + ((int64_t)x.b * cache.Hkv + hk) * RB + x.i * G + x.h - hk * G; };
    // this lane's rows
    Row row[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) row[t] = row_of(min(r0 + 16 * t + l16, RS - 1));
    int64_t at[QT];                                          // where the rows' results go, -1: nowhere
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const bool mine = r0 + 16 * t + l16 < RS;
        at[t] = mine && row[t].live ? at_ws(row[t]) : -1;
        if (mine && lg == 0 && (at[t] < 0 || b0 >= b1)) *(f32x2*)(ml + 2 * at_ws(row[t])) = f32x2{kNoScore, 0.f};
    }
    if (b0 >= b1) return;

    // units of 16 bytes: K's first, then V's; the places of their two pieces (none: the first unit's code again, not stored)
    int from[U], to[U][2];
    bool of_v[U];
#pragma unroll
    for (int x = 0; x < U; x++) {
        const int unit = tid + 256 * x < 4 * D ? tid + 256 * x : 0;
        of_v[x] = unit >= 2 * D;
        if (!of_v[x]) {
            const int key = unit / (D / 16), u = unit - key * (D / 16), g = u >> 2, kg = u & 3, row = 4 * (key >> 3) + (key & 3);
            const int slot = 64 * ((key >> 2 & 1) * 2 * DK + 2 * g) + 16 * kg + (row ^ (4 * kg) ^ (2 * g));
            from[x] = 16 * unit, to[x][0] = slot, to[x][1] = slot + 64;
        } else {
            const int y = unit - 2 * D, pair = y >> 2, kg = y & 3;
            const int slot = 64 * (KF + 2 * (pair >> 4)) + 16 * kg + ((pair & 15) ^ (4 * kg));
            from[x] = 16 * y, to[x][0] = slot, to[x][1] = slot + 64;
        }
    }
    const int read = 16 * lg + (l16 ^ (4 * lg));
    // features past D are zeros that no block overwrites
    if (D % 64)
        for (int i = tid; i < FR * 64; i += 256) buf[0][i] = buf[1][i] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};

    struct Set {
        u32x4 c[U];
        f32x2 s;
    };
    bool lost = false;
    int ids = 0, id0 = b0;
    // (every load is made, past the last block that one's again and for a page outside the pool page 0's: behind a branch the
    // compiler could not count them)
    auto load = [&](int blk, Set& x) {
        blk = min(blk, b1 - 1);
        if (blk == b0 || blk - id0 >= 64) {
            id0 = blk;
            ids = blk + lane < b1 ? cache.table[bf * cache.table_stride + blk + lane] : 0;
        }
        const int id = __builtin_amdgcn_readlane(ids, blk - id0);
        const bool in = id >= 0 && id < cache.pages;
        lost = lost || !in;
        const int64_t page = (int64_t)(in ? id : 0) * cache.Hkv + hk;
#pragma unroll
        for (int u = 0; u < U; u++) x.c[u] = *(const u32x4*)((of_v[u] ? cache.v : cache.k) + page * kKvBlock * D + from[u]);
        x.s = *(const f32x2*)(cache.scales + 2 * page);
    };
    auto store = [&](int which, const Set& x) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (tid + 256 * u < 4 * D) {
                buf[which][to[u][0]] = widen(x.c[u][0], x.c[u][1]);
                buf[which][to[u][1]] = widen(x.c[u][2], x.c[u][3]);
            }
        }
    };
    CacheRows<DG, QT, PS, MOD> st;
    st.clear();
    auto queries = [&] {
#pragma unroll
        for (int t = 0; t < QT; t++) st.load(a, t, row[t].b, row[t].i, row[t].h, at[t] >= 0 ? row[t].p : -1);
    };
    if (cache.pages) {
        Set x0, x1;
        load(b0, x0);
        load(b0 + 1, x1);
        queries();                                           // (behind the codes: their pages had to be asked for first)
        if (D % 64) __syncthreads();
        store(0, x0);
        f32x2 scale = x0.s;
        load(b0 + 2, x0);
        stage_sync<63>();
        // A block's fragments are asked for all at once, V's while the scores become weights: read where they are used, two
        // at a time, they took a third of the block's time in waits.
        auto step = [&](int blk, Set& x) {
            const f16x8* f = buf[(blk - b0) & 1];
            f16x8 k[KF], v[2 * DG];
#pragma unroll
            for (int i = 0; i < KF; i++) k[i] = f[64 * i + (read ^ (2 * ((i % (2 * DK)) >> 1)))];
            __builtin_amdgcn_sched_barrier(0);
            st.template block<false>(a.mod, blk, scale[0], scale[1], [&](int n, int c) { return k[2 * DK * n + c]; }, [&](int c) { return v[c]; },
                                     [&] {
#pragma unroll
                                         for (int i = 0; i < 2 * DG; i++) v[i] = f[64 * (KF + i) + read];
                                         __builtin_amdgcn_sched_barrier(0);
                                     });
            store((blk + 1 - b0) & 1, x);
            scale = x.s;
            load(blk + 3, x);
            stage_sync<63>();
            return blk + 1 < b1;
        };
        for (int blk = b0; step(blk, x1) && step(blk + 1, x0); blk += 2) {}
    } else {
        queries();
        lost = true;
    }

    // this wave's rows; those that are not finite again, key by key
#pragma unroll
    for (int t = 0; t < QT; t++) {
        float z = st.S1[t] * 0.f;
#pragma unroll
        for (int c = 0; c < 2 * DG; c++) z += (st.O[t][c][0] + st.O[t][c][1] + st.O[t][c][2] + st.O[t][c][3]) * 0.f;
        const uint64_t odd = __ballot(lost || !(z == 0.f)), live = __ballot(at[t] >= 0);
        uint32_t redo = (uint32_t)(odd | odd >> 16 | odd >> 32 | odd >> 48) & (uint32_t)live & 0xffffu;
        if (at[t] >= 0 && !(redo >> l16 & 1)) {
            float* o = a.ws + at[t] * D;
#pragma unroll
            for (int g = 0; g < DG; g++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int d = 32 * g + 8 * lg + 4 * h;
                    if (d < D) *(f32x4*)(o + d) = f32x4{st.O[t][2 * g][2 * h], st.O[t][2 * g + 1][2 * h], st.O[t][2 * g][2 * h + 1], st.O[t][2 * g + 1][2 * h + 1]};
                }
            if (lg == 0) *(f32x2*)(ml + 2 * at[t]) = f32x2{st.mref[t], st.S1[t]};
        }
        float* qs = again[wave];
        for (; redo; redo &= redo - 1) {
            const Row one = row_of(r0 + 16 * t + __builtin_ctz(redo));
            const int64_t e = one.b * a.qst[3] + (int64_t)one.h * a.qst[2] + one.i * a.qst[1];
            for (int d = lane; d < D; d += 64) {
                const int64_t y = e + d * a.qst[0];
                qs[d] = a.in16 ? (float)((const _Float16*)a.q)[y] : (float)(_Float16)((const float*)a.q)[y];
            }
            __builtin_amdgcn_wave_barrier();
            int len, total, n;
            spans_of<kShared>(a, one.b, len, total, n);
            const RowState s = attn_row(CacheSrc{cache, one.b, hk, total / kKvBlock * kKvBlock, bf, same}, a.mod,
                                        a.slopes ? a.slopes[one.h] * kLog2e : 0.f, one.p, one.p + 1, (int64_t)b0 * kKvBlock,
                                        (int64_t)b1 * kKvBlock, D, qs, qs + 128, lane);
            __builtin_amdgcn_wave_barrier();
            const int64_t w = at_ws(one);
            for (int i = 0; i < 2; i++)
                if (lane + 64 * i < D) a.ws[w * D + lane + 64 * i] = s.o[i];
            if (lane == 0) *(f32x2*)(ml + 2 * w) = f32x2{s.m == -INFINITY ? kNoScore : s.m, s.l};
        }
    }
}

// What a launch's first workgroups do with the shared blocks: rows of a group few (each wave every fourth block, as for a
// sequence alone), 64 or 128 of them to a workgroup
enum { kFew, kRows64, kRows128 };

// The shared blocks' workgroups first, then each sequence's own blocks': the former wait for the VALU, the latter for memory, and
// side by side on a CU they take little more than the former alone.
template <int DG, bool PS, bool MOD, int KIND>
__global__ __launch_bounds__(256, KIND == kRows128 ? 2 : 3) void k_kv8_attn_shared(Kv8AttnArgs a, Kv8SharedPlan p, int first, int parts) {
    union Lds {
        CacheLds<DG, 1> own;
        RowsLds<DG> rows;
    };
    __shared__ __attribute__((aligned(16))) char raw[KIND == kFew ? sizeof(CacheLds<DG, 1>) : sizeof(Lds)];
    const int wg = blockIdx.x;
    if (wg >= first) {
        cache_attention<DG, 1, PS, MOD, kOwn>(a, wg - first, p.own.tiles, p.own.splits, p.own.least, parts, 0, *(CacheLds<DG, 1>*)raw);
    } else if constexpr (KIND == kFew) {
        cache_attention<DG, 1, PS, MOD, kShared>(a, wg, p.shared.tiles, p.shared.splits, p.shared.least, parts, p.own.splits, *(CacheLds<DG, 1>*)raw);
    } else {
        rows_attention<DG, KIND == kRows128 ? 2 : 1, PS, MOD>(a, wg, p.shared.tiles, p.shared.splits, p.shared.least, parts, p.own.splits,
                                                              *(RowsLds<DG>*)raw);
    }
}

template <int DG, bool PS, bool MOD>
void launch_shared(const Kv8AttnArgs& a, const Kv8SharedPlan& p, hipStream_t s) {
    const int64_t sets = (a.c.B + a.group - 1) / a.group;
    const int first = (int)(p.shared.tiles * p.shared.splits * a.c.Hkv * sets), parts = p.own.splits + p.shared.splits;
    const dim3 grid((unsigned)(first + (int64_t)p.own.tiles * p.own.splits * a.c.Hkv * a.c.B));
    auto go = [&](auto kind) {
        hipLaunchKernelGGL((k_kv8_attn_shared<DG, PS, MOD, decltype(kind)::value>), grid, dim3(256), 0, s, a, p, first, parts);
    };
    if (!p.rows) go(std::integral_constant<int, kFew>{});
    else if (p.shared.qt == 1) go(std::integral_constant<int, kRows64>{});
    else go(std::integral_constant<int, kRows128>{});
}

}  // namespace

Kv8SharedPlan kv8_shared_plan(const Kv8AttnArgs& a) {
    Kv8SharedPlan p{};
    const int64_t G = a.H / a.c.Hkv, sets = (a.c.B + a.group - 1) / a.group;
    // each sequence's own blocks: as a cache of the blocks that are left, its parts cut as for kv8_plan's tiles, but in tiles of 16 rows
    Kv8AttnArgs own = a;
    own.c.max_blocks = a.c.max_blocks - std::min(a.max_shared, a.c.max_blocks);
    p.own = kv8_plan(own);
    p.own.qt = 1;
    p.own.tiles = (int)((a.S * G + 15) / 16);
    // the shared ones: the rows of a group
    Kv8Plan& sh = p.shared;
    const int64_t R = (int64_t)std::min(a.group, a.c.B) * a.S * G;
    // (64 sequences of one row of 4 heads in groups of 64 / 16 / 8 / 4 over 8000 or 4000 tokens: few 44.1 / 28.2 / 33.7 / 23.0 us, 64
    // rows 41.6 / 27.8 / 46.2 / 23.3, 128 rows 38.3 / 32.9 / 61.9 / 26.6)
    p.rows = R > 32;
    sh.qt = R > 64 ? 2 : 1;
    const int tile = p.rows ? 64 * sh.qt : 16;
    sh.tiles = (int)((R + tile - 1) / tile);
    const int64_t wgs = sets * a.c.Hkv * sh.tiles;
    sh.least = 8;
    // A workgroup of the shared blocks per CU, beside which the sequences' own ones run: 128 / 256 / 384 / 512 workgroups over 8000
    // tokens of 64 sequences 50.8 / 38.2 / 43.6 / 46.6 us, 4000 of 8 groups of 8 (capped) 47.5 / 33.6 / 37.7 / 41.4. (Over 32000
    // tokens 384 would be a little better, 51.2 against 53.6.)
    sh.splits = (int)std::max<int64_t>(1, std::min<int64_t>((256 + wgs - 1) / wgs, (a.max_shared + sh.least - 1) / sh.least));
    sh.splits = std::min(sh.splits, kMostSplits - std::min(p.own.splits, kMostSplits / 2));
    p.own.splits = std::min(p.own.splits, kMostSplits / 2);
    p.ws_bytes = (size_t)(p.own.splits + sh.splits) * a.c.Hkv * a.c.B * a.S * G * (a.c.D + 2) * sizeof(float);
    return p;
}

hipError_t launch_kv8_attn_shared(const Kv8AttnArgs& a, const Kv8SharedPlan& p, hipStream_t s) {
    auto mod = [&](auto dg, auto ps) {
        if (a.mod.cap2 != 0.f || a.slopes) launch_shared<decltype(dg)::value, decltype(ps)::value, true>(a, p, s);
        else launch_shared<decltype(dg)::value, decltype(ps)::value, false>(a, p, s);
    };
    auto weights = [&](auto dg) {
        if (a.o16) mod(dg, std::false_type{});
        else mod(dg, std::true_type{});
    };
    switch ((a.c.D + 31) / 32) {
        case 1: weights(std::integral_constant<int, 1>{}); break;
        case 2: weights(std::integral_constant<int, 2>{}); break;
        case 3: weights(std::integral_constant<int, 3>{}); break;
        default: weights(std::integral_constant<int, 4>{}); break;
    }
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : join_parts(a, p.own.splits + p.shared.splits, s);
}

}  // namespace mgh
