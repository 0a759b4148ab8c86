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
// Measured (32 heads on 8 of 128, two sets of inputs in turn): one sequence of 100000 tokens, 205 MB, 39.4 us (5.2 TB/s) and the join
// 4.8; 64 of 2700 tokens 67 us (5.3 TB/s), of up to 8000 with capped scores 91 (4.0 TB/s: long sequences' parts at the end). A block takes
// a wave 0.88 us, so short sequences are latency: 4 of 1030, 16 heads of 48, five rows: 7.3 us and the join 2.8.
#include <algorithm>

#include "k_kv8_attn.h"

namespace mgh {

namespace {

template <int DG, int QT, bool PS, bool MOD>
__global__ __launch_bounds__(256, QT == 1 ? 3 : 2) void k_kv8_attn(Kv8AttnArgs a, int tiles, int splits, int least) {
    __shared__ CacheLds<DG, QT> lds;
    cache_attention<DG, QT, PS, MOD, kAlone>(a, blockIdx.x, tiles, splits, least, splits, 0, lds);
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
    const dim3 grid((unsigned)((int64_t)p.tiles * p.splits * a.c.Hkv * a.c.B));
    with_cache_kernel(a, p.qt, [&](auto dg, auto qt, auto ps, auto mod) {
        hipLaunchKernelGGL((k_kv8_attn<decltype(dg)::value, decltype(qt)::value, decltype(ps)::value, decltype(mod)::value>), grid, dim3(256),
                           0, s, a, p.tiles, p.splits, p.least);
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    return join_parts(a, p.splits, s);
}

}  // namespace mgh
