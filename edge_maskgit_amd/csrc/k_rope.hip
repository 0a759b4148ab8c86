// k_rope.hip — rotary positions on the heads of queries and keys (gfx950).
//
// Bound by its bytes: every feature is read and written once. A thread takes V pairs (two accesses of up to 16 bytes in,
// two out) of up to 8 heads of one token, so their angles are computed once for those heads. Measured: 2 x 8191 tokens, 40 heads
// of 128 in fp16, 67.0 us (5.0 TB/s); 3 x 1021, 40 heads of 64 in fp32, 11.4; one image (257 tokens) 6, of which the launch is most. Rows, heads or
// pointers that are not at multiples of 4 elements go feature by feature, one pair per thread: the first of these 90.6 us.
#include <algorithm>

#include "k_rope.h"

namespace mgh {

namespace {

// items of a sequence: token, head of a step, V pairs; a thread takes heads hl, hl + HG, ...
template <int V, bool IN16, bool OUT16>
__global__ __launch_bounds__(256) void k_rope(RopeArgs a, int HG) {
    const Rotation& r = a.r;
    ask_rotation(r);
    asm volatile("" ::"s"(a.x), "s"(a.y), "s"(a.xst[0]), "s"(a.xst[1]), "s"(a.xst[2]), "s"(a.xst[3]), "s"(a.yst[0]), "s"(a.yst[1]), "s"(a.yst[2]),
                 "s"(a.yst[3]), "s"(a.D), "s"(a.S), "s"(a.H), "s"(a.first), "s"(a.fresh));
    const int units = a.D / (2 * V), per = units * HG, b = blockIdx.y;
    const uint32_t at = blockIdx.x * 256u, i0 = at / per;
    const int x = (int)(at - i0 * per) + threadIdx.x, di = x / per, item = x - di * per;
    const int i = (int)i0 + di, hl = item / units, pair = (item - hl * units) * V;
    Turns<V> f;
    f.load(r, pair);
    const TokenPos t = token_pos(r, b, min(i, a.S - 1), (int32_t)((a.first ? (uint32_t)a.first[b] : 0u) + (uint32_t)i));
    int n = a.S;
    asm volatile("" : "+s"(n));                          // (else loaded by a pointer chosen between the two)
    if (a.fresh) n = a.fresh[b];
    if (i >= n || n > a.S) return;
    rope_heads<V, IN16, OUT16, (V > 1)>(r, t, f, pair, a.x, b * a.xst[3] + i * a.xst[1] + hl * a.xst[2], HG * a.xst[2], a.xst[0], a.y,
                                        b * a.yst[3] + i * a.yst[1] + hl * a.yst[2], HG * a.yst[2], a.yst[0], (a.H - hl + HG - 1) / HG);
}

template <int V>
void launch_rope_v(const RopeArgs& a, const RopePlan& p, hipStream_t s) {
    const dim3 grid((unsigned)p.wgs, (unsigned)a.B);
    if (a.in16 && a.out16) hipLaunchKernelGGL((k_rope<V, true, true>), grid, dim3(256), 0, s, a, p.hg);
    else if (a.in16) hipLaunchKernelGGL((k_rope<V, true, false>), grid, dim3(256), 0, s, a, p.hg);
    else if (a.out16) hipLaunchKernelGGL((k_rope<V, false, true>), grid, dim3(256), 0, s, a, p.hg);
    else hipLaunchKernelGGL((k_rope<V, false, false>), grid, dim3(256), 0, s, a, p.hg);
}

}  // namespace

// pairs in a row whose features lie in two runs: 8, 4 or 1
int rope_granule(const Rotation& r, int D) {
    auto fits = [&](int n) {
        if (r.P % n || D % (2 * n)) return false;
        for (int i = 0; i < r.axes && r.order == kRopeAxisHalves; i++)
            if ((r.start[i + 1] - r.start[i]) % n) return false;
        return true;
    };
    return fits(8) ? 8 : fits(4) ? 4 : 1;
}

RopePlan rope_plan(const RopeArgs& a) {
    RopePlan p{};
    const int g = rope_granule(a.r, a.D);
    // (8 pairs where both sides are fp16: 2 x 8191 tokens, 40 heads of 128, 71.5 us instead of 67.0)
    p.v = std::min(g, a.vec) >= 4 ? 4 : 1;
    const int64_t units = a.D / (2 * p.v), all = (int64_t)a.B * a.S * units;
    // heads of a thread: more where threads enough for 2 waves per SIMD are left (for 8 waves 3 x 1021 tokens, 40 heads of 64, take
    // 11.9 us instead of 11.4; always 8 heads: one image's kernel 5.8 instead of 3.8)
    int n = 1;
    while (n < 8 && n < a.H && all * a.H / (2 * n) >= 256 * 512) n *= 2;
    p.hg = (a.H + n - 1) / n;
    p.wgs = (a.S * units * p.hg + 255) / 256;
    return p;
}

hipError_t launch_rope(const RopeArgs& a, const RopePlan& p, hipStream_t s) {
    if (p.v == 4) launch_rope_v<4>(a, p, s);
    else if (p.v == 1) launch_rope_v<1>(a, p, s);
    else return hipErrorInvalidValue;                    // (the plan's workgroups are those of v pairs per thread)
    return hipGetLastError();
}

}  // namespace mgh
