// k_kv8_shared.hip — attention of the newest tokens over the 8-bit cache where sequences share their first blocks (gfx950).
//
// The rows of all sequences of a group meet the shared blocks together, so these are read once per tile of rows and not once
// per sequence; each sequence's own blocks follow as in k_kv8_attn.hip, and the parts of both are joined.
#include <algorithm>

#include "k_kv8_attn.h"

namespace mgh {

namespace {

template <int DG, int QT, bool PS, bool MOD, int MODE>
__global__ __launch_bounds__(256, QT == 1 ? 3 : 2) void k_kv8_attn_part(Kv8AttnArgs a, int tiles, int splits, int least, int parts,
                                                                         int part0) {
    cache_attention<DG, QT, PS, MOD, MODE>(a, tiles, splits, least, parts, part0);
}

}  // namespace

Kv8SharedPlan kv8_shared_plan(const Kv8AttnArgs& a) {
    Kv8SharedPlan p{};
    const int64_t G = a.H / a.c.Hkv, groups = (a.c.B + a.group - 1) / a.group;
    // each sequence's own blocks: as a cache of the blocks that are left
    Kv8AttnArgs own = a;
    own.c.max_blocks = a.c.max_blocks - std::min(a.max_shared, a.c.max_blocks);
    p.own = kv8_plan(own);
    // the shared ones: the rows of a group
    Kv8Plan& sh = p.shared;
    const int64_t R = (int64_t)std::min(a.group, a.c.B) * a.S * G;
    sh.qt = R > 16 ? 2 : 1;
    sh.tiles = (int)((R + 16 * sh.qt - 1) / (16 * sh.qt));
    const int64_t wgs = groups * a.c.Hkv * sh.tiles;
    sh.least = 8;
    sh.splits = (int)std::max<int64_t>(1, std::min<int64_t>((512 + wgs - 1) / wgs, (a.max_shared + sh.least - 1) / sh.least));
    sh.splits = std::min(sh.splits, kMostSplits - std::min(p.own.splits, kMostSplits / 2));
    p.own.splits = std::min(p.own.splits, kMostSplits / 2);
    p.ws_bytes = (size_t)(p.own.splits + sh.splits) * a.c.Hkv * a.c.B * a.S * G * (a.c.D + 2) * sizeof(float);
    return p;
}

hipError_t launch_kv8_attn_shared(const Kv8AttnArgs& a, const Kv8SharedPlan& p, hipStream_t s) {
    const int parts = p.own.splits + p.shared.splits;
    auto go = [&](auto mode, const Kv8Plan& q, int64_t sets, int part0) {
        const dim3 grid((unsigned)(q.tiles * q.splits * a.c.Hkv * sets));
        with_cache_kernel(a, q.qt, [&](auto dg, auto qt, auto ps, auto mod) {
            hipLaunchKernelGGL((k_kv8_attn_part<decltype(dg)::value, decltype(qt)::value, decltype(ps)::value, decltype(mod)::value,
                                                decltype(mode)::value>), grid, dim3(256), 0, s, a, q.tiles, q.splits, q.least, parts, part0);
        });
        return hipGetLastError();
    };
    hipError_t e = go(std::integral_constant<int, kShared>{}, p.shared, (a.c.B + a.group - 1) / a.group, p.own.splits);
    if (e != hipSuccess) return e;
    e = go(std::integral_constant<int, kOwn>{}, p.own, a.c.B, 0);
    if (e != hipSuccess) return e;
    return join_parts(a, parts, s);
}

}  // namespace mgh
