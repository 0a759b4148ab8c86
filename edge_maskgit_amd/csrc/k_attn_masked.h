// k_attn_masked.h — the tiled kernel of k_attn_masked*.hip: attention under masks (gfx950).
//
// Rows: the G = H / Hkv query heads of a key head are G rows of each query position, so a workgroup's 4
// waves hold 64 QT rows (row r = query r / G, head r % G) against one head's keys, taken 64 at a time.
//  * K and V chunks go from memory to LDS by 16-byte buffer loads, two buffers in turn, one barrier per
//    chunk; pieces are XOR-swizzled by their row (a property of the lane's source address) so that both
//    ways of reading are free of bank conflicts. Rows past the last key and features past D arrive as
//    zeros (outside the buffer's range). V needs no transposed copy: ds_read_b64_tr_b16 hands each lane
//    4 keys of its feature.
//  * S^T = K Q^T on v_mfma_f32_16x16x32_f16: a lane holds scores of one row (query l16), 4 keys per
//    register quadruple, which is the operand of O^T = V^T P^T as it stands. Row sums by the same
//    instruction on ones, so they add exactly the weights that meet V.
//  * The softmax reference of a row stays within [-7, 15] (log2 units) of its maximum: it moves, and O is
//    rescaled, only when a score passes it by 15, a wave-uniform branch. Weights lie in fp16's normal
//    range up to 2^15; with an fp32 output (PS) a weight is hi + lo in fp16, both to nearest, and a
//    chunk's products are summed apart from O. With an fp16 output a weight is fp16: over thousands of keys the
//    outputs are then 2.3-2.8e-4 off (relative, root mean square) where their own rounding alone makes 2.1e-4, and
//    lo would take 40-50% longer (two rows of 4097 tokens, 16 heads of 64, 283 us against 189; 4097 tokens, 32
//    heads on 8 of 128, 452 against 330).
//  * Which keys a row sees is one bound per row (causal and prefix together), known per wave, so that whole
//    chunks need no test; ids of documents are compared only in chunks where they can differ: a first
//    pass over the ids notes for each chunk whether any row of the workgroup can see it and whether all
//    see all of it.
// A masked key's weight is 0, but 0 times an infinity or NaN of V is not: rows that come out not finite are taken
// again by attn_row, which uses what a row sees and nothing else. Rows whose sum of weights is not finite too: they may
// have seen no NaN, but weights past fp16, which a moving reference then multiplied by 0: all that a row saw of a
// chunk were infinite products at the lower end of a cap, or scores past 1e8 lie farther apart than the
// reference's distance. Two rows of 4097 tokens in nine documents each, 197 places of NaN behind them: 3.5 ms against
// 0.075, the time of the last documents' rows, whose keys end in a chunk with NaN. Values that no row of the workgroup
// sees zeroed in LDS would make that 0.075 too, but cost every call 4-5%.
//
// Measured: 16 heads of 64, 2 x 4096 tokens 173 us (794 TFLOP/s), 2 x 4097 189: the last row's workgroups are a
// round of their own (32 heads of 128: 266, 333); 32 heads on 8 of 128, 512 rows of each of two
// prompts of 12345 in 207 us (980 TFLOP/s), 8191 tokens causal with a prefix of 1000 530, capped 660
// (840 TFLOP/s: two exponentials and a reciprocal per score); one row of 8000 keys, 8 sequences: 53 us, 4.9 TB/s.
// Tiles of 32 rows on v_mfma_f32_32x32x16_f16 (half the softmax state) ran 3-11% longer.
#pragma once
#include <type_traits>

#include "k_attn_row.h"

namespace mgh {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kMaskKeys = 64;              // keys per chunk
constexpr int kMaskScan = 16384;           // chunks whose documents are noted (1 M keys)

struct MaskedSrc {
    const MaskedAttnArgs& a;
    const _Float16* k;     // the head's rows
    const _Float16* v;
    int64_t stride;
    int lim;               // the last key that causal and prefix leave
    const int32_t* docs;   // the sequence's ids, or null
    int doc;
    __device__ bool seen(int64_t j) const { return j <= lim && (!docs || (docs[j] == doc && doc >= 0)); }
    __device__ float dot(int64_t j, const float* qs) const {
        const _Float16* p = k + j * stride;
        float s = 0.f;
#pragma unroll 2
        for (int d = 0; d < a.D; d += 8) {
            const f16x8 x = *(const f16x8*)(p + d);
#pragma unroll
            for (int i = 0; i < 8; i++) s = fmaf(qs[d + i], (float)x[i], s);
        }
        return s;
    }
    __device__ float value(int64_t j, int d) const { return (float)v[j * stride + d]; }
};

// XOR of a 16-byte piece's place in its LDS row. 256 bytes of LDS are read at a time: two pieces side by side of
// 8 rows (a transposing read), or a score operand's pieces of 16 lanes, which are not consecutive lanes: rows
// 0-3 and 12-15 of one piece with rows 4-11 of the next. With it they fall on different banks, whether 256
// bytes are one row, two or four. (SQ_LDS_BANK_CONFLICT: 0; by 8 rows of 128 bytes, half of the LDS cycles.)
template <int PPR>
__device__ __forceinline__ int piece_swz(int r) {
    const int h = (r >> 3) & 1;
    return 2 * (PPR == 16 ? (r & 7) ^ 4 * h : PPR == 8 ? ((r >> 1) & 3) ^ 2 * h : ((r >> 2) & 1) ^ h) + h;
}

// DC 16-feature chunks (D <= 16 DC), QT 16-row tiles per wave, PS: weights as hi + lo; MOD 0: scores times a
// positive scale, 1: any scale and slopes (0: none), 2: capped, weights in fp16, 3: capped with any scale and cap, then
// slopes; small scores by a form of their own (4097 tokens, 32 heads on 8 of 128, cap 50, fp32 output 594 us, 547 without it).
// The VALU is the busier unit below 128 features and with a cap (per score two exponentials and a reciprocal, at
// a quarter of its rate), so MOD 0 and 2 keep the raw scores: both maps rise with them, so the maximum is
// taken raw, and the reference goes into the map's last fma.
constexpr float kMasked = -3e38f;          // below every raw score (at most 128 65504^2), where -infinity is one
template <int DC, int QT, bool PS, int MOD>
__global__ __launch_bounds__(256, 2) void k_attn_masked(MaskedAttnArgs a, int tiles, int splits) {
    constexpr int PPR = DC <= 2 ? 4 : DC <= 4 ? 8 : 16;       // 16-byte pieces of an LDS row
    constexpr int KC = (DC + 1) / 2, NT = kMaskKeys / 16, NI = kMaskKeys * PPR / 256;
    constexpr int ROWB = PPR * 16, CH = kMaskKeys * ROWB;     // bytes of an LDS row, of a K or V chunk
    constexpr int WROWS = 16 * QT;
    // two objects, so that the compiler can tell a chunk's reads from the next one's loads (with one it waits for
    // those before the first read); K, V, the ids of documents
    __shared__ __attribute__((aligned(1024))) char lds0[2 * CH + kMaskKeys * 4], lds1[2 * CH + kMaskKeys * 4];
    __shared__ uint32_t bits[2][kMaskScan / 32];              // chunks that some row sees; that all rows see all of
    __shared__ int range[3][4];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lg = lane >> 4;
    // each XCD takes contiguous runs of (key head, sequence), sequences innermost, whose masks may leave unlike work; of
    // a head the last rows, which see most, first
    const int lid = xcd_remap(blockIdx.x, gridDim.x);
    const int at = lid / (tiles * splits), in_h = lid - at * (tiles * splits);
    const int tile = tiles - 1 - in_h / splits, sp = in_h % splits;
    const int hk = at / a.B, b = at - hk * a.B, hb = b * a.Hkv + hk, G = a.H / a.Hkv, R = a.Sq * G, off = a.Sk - a.Sq;
    const int prefix = a.prefix ? max(min(a.prefix[b], a.Sk), 0) : 0;
    auto bound_of = [&](int i) { return a.causal ? min(max(off + i, prefix - 1), a.Sk - 1) : a.Sk - 1; };
    const int r0 = tile * 4 * WROWS, rw = r0 + wave * WROWS;
    const int wg_hi = bound_of((min(r0 + 4 * WROWS, R) - 1) / G);
    const int w_lo = rw < R ? bound_of(rw / G) : -1, w_hi = rw < R ? bound_of((min(rw + WROWS, R) - 1) / G) : -1;

    // this lane's rows
    int lim[QT], doc[QT];
    float pos[QT], slope2[QT];
    const int32_t* docs = a.docs ? a.docs + (int64_t)b * a.doc_stride : nullptr;
    f16x8 qf[QT][KC];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int r = rw + 16 * t + l16, i = min(r, R - 1) / G, g = min(r, R - 1) - i * G;
        lim[t] = r < R ? bound_of(i) : -1;
        pos[t] = (float)(off + i);
        doc[t] = docs && off + i >= 0 && r < R ? docs[off + i] : -1;
        slope2[t] = MOD && a.slopes ? a.slopes[hk * G + g] * kLog2e : 0.f;
        const _Float16* q = (const _Float16*)a.q + b * a.qst[3] + (int64_t)(hk * G + g) * a.qst[2] + i * a.qst[1];
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const int d = 32 * c + 8 * lg;
            qf[t][c] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (d < a.D) qf[t][c] = *(const f16x8*)(q + d);
        }
    }

    // this split's chunks
    const int nch = wg_hi / kMaskKeys + 1, per = (nch + splits - 1) / splits;
    const int c0 = wg_hi < 0 ? 0 : sp * per, c1 = wg_hi < 0 ? 0 : min(nch, c0 + per);
    const bool scan = docs && c1 > c0 && c1 - c0 <= kMaskScan;
    if (scan) {
        // 8 chunks' ids at once, the first ones with the rows' own; each wave takes 8 of 32 chunks, a byte of the noted bits
        int x[8];
        auto load_ids = [&](int c) {
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = docs[min((c + k) * kMaskKeys + lane, a.Sk - 1)];
        };
        load_ids(c0 + 8 * wave);
        // the workgroup's ids: smallest, largest, and whether every row has one
        const int i0 = r0 / G, i1 = (min(r0 + 4 * WROWS, R) - 1) / G;
        int lo = INT32_MAX, hi = -1, all = 1;
        for (int i = i0 + tid; i <= i1; i += 256) {
            const int x = off + i >= 0 ? docs[off + i] : -1;
            if (x < 0) all = 0;
            else lo = min(lo, x), hi = max(hi, x);
        }
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) lo = min(lo, __shfl_xor(lo, s)), hi = max(hi, __shfl_xor(hi, s)), all &= __shfl_xor(all, s);
        if (lane == 0) range[0][wave] = lo, range[1][wave] = hi, range[2][wave] = all;
        for (int i = tid; i < (c1 - c0 + 31) / 32; i += 256) bits[0][i] = bits[1][i] = 0;
        __syncthreads();
        for (int w = 0; w < 4; w++) lo = min(lo, range[0][w]), hi = max(hi, range[1][w]), all &= range[2][w];
        all = all && lo == hi;
        for (int w0 = c0 + 8 * wave; w0 < c1; w0 += 32) {
            if (w0 != c0 + 8 * wave) load_ids(w0);
            uint32_t some = 0, whole = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if (w0 + k < c1 && __any(x[k] >= lo && x[k] <= hi)) {     // (past the last key: its id again)
                    some |= 1u << k;
                    if (all && __all(x[k] == hi)) whole |= 1u << k;
                }
            }
            if (lane == 0) {
                ((uint8_t*)bits[0])[(w0 - c0) >> 3] = (uint8_t)some;
                ((uint8_t*)bits[1])[(w0 - c0) >> 3] = (uint8_t)whole;
            }
        }
        __syncthreads();
    }
    // the next chunk from c on that some row sees, or c1; `same`: whether all rows see all of it, as far as documents
    // go. The bits of 32 chunks at a time stay in scalar registers.
    uint32_t seen = 0, full = 0;
    int word = -1;
    auto find = [&](int c, bool& same) {
        same = !docs;
        if (!scan) return c;
        for (; c < c1; c = c0 + 32 * (word + 1)) {
            const int at = (c - c0) >> 5, bit = (c - c0) & 31;
            if (at != word) {
                word = at;
                seen = __builtin_amdgcn_readfirstlane(bits[0][at]);
                full = __builtin_amdgcn_readfirstlane(bits[1][at]);
            }
            if (seen >> bit) {
                const int n = bit + __builtin_ctz(seen >> bit);
                same = full >> n & 1;
                return c0 + 32 * word + n;       // (no bits past c1)
            }
        }
        return c1;
    };

    // staging: thread n = 256 u + tid of a chunk fills slot n of the buffer; the piece that belongs there
    const int64_t kv0 = b * a.kvst[3] + hk * a.kvst[2];
    const uint32_t rowb = (uint32_t)a.kvst[1] * 2;
    uint32_t src[NI];
#pragma unroll
    for (int u = 0; u < NI; u++) {
        const int n = 256 * u + tid, r = n / PPR, p = (n % PPR) ^ piece_swz<PPR>(r);
        src[u] = 8 * p < a.D ? r * rowb + 16 * p : 0x80000000u;
    }
    auto stage = [&](int c, auto bufc) {
        constexpr int buf = decltype(bufc)::value;
        const int left = a.Sk - c * kMaskKeys;               // rows from this chunk on, >= 1
        const uint32_t ext = (uint32_t)(min(left, kMaskKeys) - 1) * rowb + 2 * a.D;
        const int64_t at = kv0 + (int64_t)c * kMaskKeys * a.kvst[1];
        auto rsrc = [&](const void* p) {
            return __builtin_amdgcn_make_buffer_rsrc((void*)((const _Float16*)p + at), (short)0, (int)ext, 0x00020000);
        };
        const __amdgpu_buffer_rsrc_t rk = rsrc(a.k), rv = rsrc(a.v);
        char* B = (buf ? lds1 : lds0) + wave * 1024;
#pragma unroll
        for (int u = 0; u < NI; u++) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(B + 4096 * u), 16, (int)src[u], 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(B + CH + 4096 * u), 16, (int)src[u], 0, 0, 0);
        }
        if (docs && wave == 0) {
            const __amdgpu_buffer_rsrc_t rd =
                __builtin_amdgcn_make_buffer_rsrc((void*)(docs + c * kMaskKeys), (short)0, 4 * min(left, kMaskKeys), 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rd, (lds_void*)((buf ? lds1 : lds0) + 2 * CH), 4, 4 * lane, 0, 0, 0);
        }
    };
    // where this lane reads: K row l16 of a tile, pieces 4 c + lg; V rows 4 lg + l16 / 4 (of 16), 4 features at
    // 16 c + 4 (l16 % 4)
    uint32_t ka[KC], va[DC];
#pragma unroll
    for (int c = 0; c < KC; c++) ka[c] = l16 * ROWB + ((4 * c + lg) ^ piece_swz<PPR>(l16)) * 16;
#pragma unroll
    for (int c = 0; c < DC; c++) {
        const int r = 4 * lg + (l16 >> 2), p = 2 * c + ((l16 & 3) >> 1);
        va[c] = r * ROWB + (p ^ piece_swz<PPR>(r)) * 16 + 8 * (l16 & 1);
    }

    float mref[QT], S1[QT];
    f32x4 O[QT][DC];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        mref[t] = kNoScore;
        S1[t] = 0.f;
#pragma unroll
        for (int c = 0; c < DC; c++) O[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const f16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
    const float scale2 = a.mod.scale2;

    // one chunk, in the buffer that is a constant of the call; returns the next one
    auto step = [&](auto bufc, int c, bool& same) {
        constexpr int buf = decltype(bufc)::value;
        bool next_same;
        const int cn = find(c + 1, next_same);
        stage_sync<0>();                     // this buffer is filled, the other one no longer read
        if (cn < c1) stage(cn, std::integral_constant<int, buf ^ 1>{});
        const int k0 = c * kMaskKeys;
        if (k0 <= w_hi) {
            const char* K = (buf ? lds1 : lds0);
            const char* V = K + CH;
            // scores, a tile of 16 keys after the other, K's next operands read into the registers just used; this wave's
            // products before another's softmax (3% at two waves per SIMD)
            f32x4 sc[QT][NT];
            f16x8 kf[KC];
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < KC; i++) kf[i] = *(const f16x8*)(K + ka[i]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int i = 0; i < KC; i++) {
#pragma unroll
                    for (int t = 0; t < QT; t++)
                        sc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], qf[t][i], i ? sc[t][n] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                    if (n + 1 < NT) kf[i] = *(const f16x8*)(K + ka[i] + 16 * (n + 1) * ROWB);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            auto mapped = [&](auto map, auto sloped) {           // scores of the map, then slopes
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    const float d0 = pos[t] - (float)(k0 + 4 * lg);      // (whole numbers below 2^24 throughout)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float d = fabsf(d0 - (float)(16 * n + r));
                            if (MOD == 1) sc[t][n][r] = fmaf(sc[t][n][r], scale2, -slope2[t] * d);
                            else sc[t][n][r] = decltype(sloped)::value ? fmaf(-slope2[t], d, map(sc[t][n][r])) : map(sc[t][n][r]);
                        }
                }
            };
            if (MOD == 3) {                          // their form alone where all of the tile's scores are small
                float big = 0.f;
#pragma unroll
                for (int t = 0; t < QT; t++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        big = fmaxf(fmaxf(big, fabsf(sc[t][n][0])), fabsf(sc[t][n][1]));
                        big = fmaxf(fmaxf(big, fabsf(sc[t][n][2])), fabsf(sc[t][n][3]));
                    }
                auto small = [&](float x) { return cap_small(x, a.mod); };
                if (!all_small(big, a.mod)) mapped([&](float x) { return cap_score(x, a.mod); }, std::true_type{});
                else if (a.slopes) mapped(small, std::true_type{});
                else mapped(small, std::false_type{});
            } else if (MOD == 1) {
                mapped([](float x) { return x; }, std::true_type{});
            }
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            constexpr float kHidden = MOD == 2 ? kMasked : -INFINITY;
            const bool edge = k0 + kMaskKeys - 1 > w_lo, part = edge || !same;
            if (edge) {
#pragma unroll
                for (int t = 0; t < QT; t++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (k0 + 16 * n + 4 * lg + r > lim[t]) sc[t][n][r] = kHidden;
            }
            if (!same) {
                const int32_t* ids = (const int32_t*)((buf ? lds1 : lds0) + 2 * CH);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const i32x4 id = *(const i32x4*)(ids + 16 * n + 4 * lg);
#pragma unroll
                    for (int t = 0; t < QT; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (id[r] != doc[t] || doc[t] < 0) sc[t][n][r] = kHidden;
                }
            }
            float mx[QT];
            bool up[QT], any = false;
#pragma unroll
            for (int t = 0; t < QT; t++) {
                float v = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    v = fmaxf(fmaxf(v, sc[t][n][0]), sc[t][n][1]);
                    v = fmaxf(fmaxf(v, sc[t][n][2]), sc[t][n][3]);
                }
                mx[t] = MOD == 2 ? (v == kMasked ? -INFINITY : cap_score(v, a.mod)) : MOD ? v : v * scale2;
                up[t] = __any(mx[t] > mref[t] + 15.f);
                any = any || up[t];
            }
            if (any) {
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    float v = up[t] ? fmaxf(mx[t] - 7.f, mref[t]) : mref[t];
                    v = fmaxf(v, __shfl_xor(v, 16));
                    v = fmaxf(v, __shfl_xor(v, 32));
                    const float al = __builtin_amdgcn_exp2f(mref[t] - v);
                    mref[t] = v;
                    S1[t] *= al;
#pragma unroll
                    for (int cc = 0; cc < DC; cc++) O[t][cc] *= al;
                }
            }
            // weights of keys 32 p .. 32 p + 31 of row tile t, as the operand of P V
            float top[QT];
            f16x8 ph[2][QT], pl[2][QT];
            auto weights = [&](int p, int t) {
                float e[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float x = sc[t][2 * p + j / 4][j % 4];
                    if (MOD == 2) {
                        const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * a.mod.cap_in) + 1.f);
                        e[j] = __builtin_amdgcn_exp2f(fmaf(r, -2.f * a.mod.cap2, top[t]));
                    } else {
                        e[j] = __builtin_amdgcn_exp2f(MOD ? x - mref[t] : fmaf(x, scale2, -mref[t]));
                    }
                }
                if (MOD == 2 && part) {
#pragma unroll
                    for (int j = 0; j < 8; j++) e[j] = sc[t][2 * p + j / 4][j % 4] == kMasked ? 0.f : e[j];
                }
                u32x4 hi, lo;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const f16x2 h = __builtin_convertvector((f32x2{e[2 * j], e[2 * j + 1]}), f16x2);
                    hi[j] = __builtin_bit_cast(uint32_t, h);
                    if (PS) {
                        const f32x2 d = {e[2 * j] - (float)h[0], e[2 * j + 1] - (float)h[1]};
                        lo[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(d, f16x2));
                    }
                }
                ph[p][t] = __builtin_bit_cast(f16x8, hi);
                if (PS) pl[p][t] = __builtin_bit_cast(f16x8, lo);
            };
            f32x4 s1[QT], oc[QT][DC];
#pragma unroll
            for (int t = 0; t < QT; t++) {
                top[t] = a.mod.cap2 - mref[t];
                s1[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int cc = 0; cc < DC; cc++) oc[t][cc] = PS ? f32x4{0.f, 0.f, 0.f, 0.f} : O[t][cc];
                weights(0, t);
            }
            // V's operands are read AHEAD of their products (else each pair of products waits for its read); the weights
            // of the second half are made among the products of the first
            constexpr int AHEAD = DC < 4 ? DC : 4, M = QT * (PS ? 2 : 1);
            f16x8 vf[AHEAD];
            auto load_v = [&](int x) {               // operand x: half x / DC, features 16 (x % DC)
                const char* at = V + va[x % DC] + 32 * (x / DC) * ROWB;
                const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
                const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 16 * ROWB));
                vf[x % AHEAD] = __builtin_bit_cast(f16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
            };
#pragma unroll
            for (int x = 0; x < AHEAD; x++) load_v(x);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < 2; p++) {
#pragma unroll
                for (int cc = 0; cc < DC; cc++) {
                    const int x = p * DC + cc;
#pragma unroll
                    for (int t = 0; t < QT; t++) {
                        if (PS) oc[t][cc] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[x % AHEAD], pl[p][t], oc[t][cc], 0, 0, 0);
                        oc[t][cc] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[x % AHEAD], ph[p][t], oc[t][cc], 0, 0, 0);
                    }
                    if (x + AHEAD < 2 * DC) load_v(x + AHEAD);
                    if (p == 0 && cc < QT) weights(1, cc);
                    if (p) __builtin_amdgcn_sched_barrier(0);
                }
                if (p == 0) {                        // a product, vector operations, ..., two reads
#pragma unroll
                    for (int i = 0; i < DC; i++) {
#pragma unroll
                        for (int m = 0; m < M; m++) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x002, QT * (MOD == 2 ? 56 : 22) / (DC * M) + 1, 0);
                        }
                        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    if (PS) s1[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[p][t], s1[t], 0, 0, 0);
                    s1[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph[p][t], s1[t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int t = 0; t < QT; t++) {
                S1[t] += s1[t][0];
#pragma unroll
                for (int cc = 0; cc < DC; cc++) O[t][cc] = PS ? O[t][cc] + oc[t][cc] : oc[t][cc];
            }
        }
        same = next_same;
        return cn;
    };
    bool same;
    int c = find(c0, same);
    if (c < c1) stage(c, std::integral_constant<int, 0>{});
    while (c < c1) {
        c = step(std::integral_constant<int, 0>{}, c, same);
        if (c >= c1) break;
        c = step(std::integral_constant<int, 1>{}, c, same);
    }

    // rows that are not finite: again, key by key
    __syncthreads();
    float* qs = (float*)lds0 + wave * 256;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        float z = S1[t];
#pragma unroll
        for (int cc = 0; cc < DC; cc++)
#pragma unroll
            for (int r = 0; r < 4; r++) z += O[t][cc][r] * 0.f;
        uint64_t m = __ballot(!(z - z == 0.f) && rw + 16 * t + l16 < R);
        m = (m | m >> 16 | m >> 32 | m >> 48) & 0xffff;
        while (m) {
            const int l = __builtin_ctzll(m), r = rw + 16 * t + l, i = r / G, g = r - i * G;
            m &= m - 1;
            const _Float16* q = (const _Float16*)a.q + b * a.qst[3] + (int64_t)(hk * G + g) * a.qst[2] + i * a.qst[1];
            for (int d = lane; d < 128; d += 64) qs[d] = d < a.D ? (float)q[d] : 0.f;
            __builtin_amdgcn_wave_barrier();
            const MaskedSrc s{a, (const _Float16*)a.k + kv0, (const _Float16*)a.v + kv0, a.kvst[1], bound_of(i), docs,
                              docs && off + i >= 0 ? docs[off + i] : -1};
            const float sl = a.slopes ? a.slopes[hk * G + g] * kLog2e : 0.f;
            const RowState st = attn_row(s, a.mod, sl, off + i, s.lim + 1, (int64_t)c0 * kMaskKeys,
                                         min((int64_t)c1 * kMaskKeys, (int64_t)s.lim + 1), a.D, qs, qs + 128, lane);
            __builtin_amdgcn_wave_barrier();
            qs[lane] = st.o[0], qs[lane + 64] = st.o[1];
            __builtin_amdgcn_wave_barrier();
            if (l16 == l) {
                mref[t] = st.m == -INFINITY ? kNoScore : st.m;
                S1[t] = st.l;
#pragma unroll
                for (int cc = 0; cc < DC; cc++)
#pragma unroll
                    for (int x = 0; x < 4; x++) O[t][cc][x] = qs[16 * cc + 4 * lg + x];
            }
            __builtin_amdgcn_wave_barrier();
        }
    }

#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int r = rw + 16 * t + l16;
        if (r >= R) continue;
        if (splits > 1) {
            const int64_t rows = (int64_t)a.B * a.Hkv * R, row = (int64_t)hb * R + r;
            float* w = a.ws + (sp * rows + row) * a.D;
#pragma unroll
            for (int cc = 0; cc < DC; cc++)
                if (16 * cc < a.D) *(f32x4*)(w + 16 * cc + 4 * lg) = O[t][cc];
            if (lg == 0) *(f32x2*)(a.ws + splits * rows * a.D + 2 * (sp * rows + row)) = f32x2{mref[t], S1[t]};
            continue;
        }
        const int i = r / G, g = r - i * G;
        const float inv = S1[t] == 0.f ? 0.f : 1.f / S1[t];
        const int64_t ro = (int64_t)b * a.ost[3] + (int64_t)(hk * G + g) * a.ost[2] + (int64_t)i * a.ost[1];
#pragma unroll
        for (int cc = 0; cc < DC; cc++) {
            const int d = 16 * cc + 4 * lg;
            if (d >= a.D) continue;
            const f32x4 v = S1[t] == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : O[t][cc] * inv;
            if (a.vec_o) {
                if (a.o16) *(f16x4*)(a.o16 + ro + d) = __builtin_convertvector(v, f16x4);
                else *(f32x4*)(a.o + ro + d) = v;
            } else {
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int64_t e = ro + (int64_t)(d + x) * a.ost[0];
                    if (a.o16) a.o16[e] = (_Float16)v[x];
                    else a.o[e] = v[x];
                }
            }
        }
    }
}

template <int DC, int QT, bool PS>
hipError_t launch_masked_t(const MaskedAttnArgs& a, int splits, hipStream_t s) {
    const int tiles = (int)(((int64_t)a.Sq * (a.H / a.Hkv) + 64 * QT - 1) / (64 * QT));
    const dim3 grid((unsigned)((int64_t)tiles * splits * a.Hkv * a.B));
    constexpr bool kCapped = QT == 1 || DC > 4;      // (masked_plan takes one tile for capped scores of up to 64 features)
    if (a.mod.cap2 != 0.f) {
        const bool fine = PS || a.slopes || !(a.mod.cap_in > 0.f) || a.mod.cap_x != 0.f;
        if constexpr (!kCapped) return hipErrorInvalidValue;
        else if (fine) hipLaunchKernelGGL((k_attn_masked<DC, QT, PS, 3>), grid, dim3(256), 0, s, a, tiles, splits);
        else if constexpr (!PS) hipLaunchKernelGGL((k_attn_masked<DC, QT, PS, 2>), grid, dim3(256), 0, s, a, tiles, splits);
    } else if (a.slopes || !(a.mod.scale2 > 0.f)) hipLaunchKernelGGL((k_attn_masked<DC, QT, PS, 1>), grid, dim3(256), 0, s, a, tiles, splits);
    else hipLaunchKernelGGL((k_attn_masked<DC, QT, PS, 0>), grid, dim3(256), 0, s, a, tiles, splits);
    return hipGetLastError();
}

template <int DC>
hipError_t launch_masked_d(const MaskedAttnArgs& a, const MaskedPlan& p, hipStream_t s) {
    if (p.qt == 2) return a.o16 ? launch_masked_t<DC, 2, false>(a, p.splits, s) : launch_masked_t<DC, 2, true>(a, p.splits, s);
    return a.o16 ? launch_masked_t<DC, 1, false>(a, p.splits, s) : launch_masked_t<DC, 1, true>(a, p.splits, s);
}

}  // namespace mgh
