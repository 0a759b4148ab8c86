// k_sample.hip — drawing a token from logits (gfx950).
//
// Per row: m the largest logit, w = exp((l - m) / T); tokens in descending l, equal ones in the order of their ids; kept is
// the shortest prefix of that order which top-k (its length), top-p (its share of the first k's mass) and min-p (its
// last w) allow; drawn is the first kept token, in the order of the ids, whose running sum exceeds u times the kept mass.
//
// Which token a sum's border falls on must not depend on how sums are split, so masses are whole numbers of 2^-S of the
// largest weight, exp2 in 64 bits rounded once: they add up exactly in any order, atomics included. S leaves room for the
// row (63 bits for its sum) and is at most 51, where the rounding is an addition of 2^52.
#include "mgh_common.h"
#include "mgh_kernels.h"

namespace mgh {

namespace {

// order of the logits as whole numbers (-0 is 0)
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t u = __builtin_bit_cast(uint32_t, l + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 2^t, t <= 0, off by 2^-51 of it and 2^-53 |t|: the nearest whole number's power and the series of the rest, |f| <= 1/2
__device__ __forceinline__ double exp2_64(double t) {
    if (t < -1000.) return 0.;
    const double n = rint(t), f = t - n;
    double p = 2.5678435993488206e-11;
    p = fma(p, f, 4.44553827187081e-10);
    p = fma(p, f, 7.054911620801121e-09);
    p = fma(p, f, 1.0178086009239696e-07);
    p = fma(p, f, 1.3215486790144305e-06);
    p = fma(p, f, 1.5252733804059838e-05);
    p = fma(p, f, 0.00015403530393381606);
    p = fma(p, f, 0.0013333558146428441);
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.055504108664821576);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.);
    return ldexp(p, (int)n);
}

struct Weights {
    double m, c;           // largest logit, log2(e) / T
    double unit;           // 2^S
    // weight of a logit relative to the largest one's
    __device__ __forceinline__ double of(float l) const {
        if ((double)l == m) return 1.;                   // (infinities among themselves)
        if (l == -INFINITY || m == INFINITY) return 0.;  // (whatever T is)
        return exp2_64(((double)l - m) * c);
    }
    __device__ __forceinline__ uint64_t mass(double w) const {
        return __builtin_bit_cast(uint64_t, fma(w, unit, 4503599627370496.)) & 0xfffffffffffffull;
    }
};

constexpr int kThreads = 1024, kWaves = kThreads / 64;

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
    const uint32_t lo = __shfl_up((uint32_t)v, d), hi = __shfl_up((uint32_t)(v >> 32), d);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int l) {
    const uint32_t lo = __shfl((uint32_t)v, l), hi = __shfl((uint32_t)(v >> 32), l);
    return (uint64_t)hi << 32 | lo;
}
// sums of the lanes up to and with this one
__device__ __forceinline__ uint64_t scan64(uint64_t v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = shfl_up64(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// One workgroup per row, passes over the row in memory.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_sample(SampleArgs a) {
    __shared__ uint32_t cnt[256];
    __shared__ uint64_t mass[256], seg[kWaves];
    __shared__ uint32_t ties[kWaves];
    __shared__ float redf[kWaves];
    __shared__ int redi[kWaves];
    __shared__ uint64_t picked[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.V;
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.x_stride;
    float m = -INFINITY;
    bool nan = false;
    for (int i = tid; i < V; i += kThreads) {
        const float l = (float)x[i];
        nan = nan || l != l;
        m = fmaxf(m, l);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    const bool any = __any(nan);
    if (lane == 0) redf[wave] = m, redi[wave] = any;
    __syncthreads();
    nan = false;
    for (int w = 0; w < kWaves; w++) m = fmaxf(m, redf[w]), nan = nan || redi[w];
    __syncthreads();
    auto answer = [&](int id, float p) {
        a.ids[row] = id;
        if (a.prob) a.prob[row] = p;
    };
    if (nan || m == -INFINITY) {
        if (tid == 0) answer(-1, nan ? __builtin_nanf("") : 0.f);
        return;
    }
    const float temp = a.temp ? a.temp[row] : 1.f;
    if (!(temp > 0.f)) {
        int best = V;
        for (int i = tid; i < V && best == V; i += kThreads)
            if ((float)x[i] == m) best = i;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) best = min(best, __shfl_xor(best, d));
        if (lane == 0) redi[wave] = best;
        __syncthreads();
        for (int w = 0; w < kWaves; w++) best = min(best, redi[w]);
        if (tid == 0) answer(best, 1.f);
        return;
    }
    const Weights wt{(double)m, 1.4426950408889634 / (double)temp, a.unit};
    // kept: keys above t, and the first nt of the tokens at t
    uint32_t t = 0, nt = V;
    uint64_t total = 0;

    // the key and the number of its tokens where a running count reaches `k`, or a running mass `target`; `total` the mass up to there
    auto cut = [&](bool by_count, uint64_t k, double target) {
        uint32_t prefix = 0;
        uint64_t above_n = 0, above_m = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kThreads) cnt[i] = 0, mass[i] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += kThreads) {
                const float l = (float)x[i];
                const uint32_t key = key_of(l);
                if (shift < 24 && key >> (shift + 8) != prefix) continue;
                atomicAdd(&cnt[key >> shift & 255], 1u);
                atomicAdd((unsigned long long*)&mass[key >> shift & 255], (unsigned long long)wt.mass(wt.of(l)));
            }
            __syncthreads();
            if (wave == 0) {                             // four bins of a lane, highest first
                uint64_t n4 = 0, m4 = 0;
                for (int j = 0; j < 4; j++) n4 += cnt[255 - 4 * lane - j], m4 += mass[255 - 4 * lane - j];
                uint64_t n = above_n + scan64(n4, lane) - n4, s = above_m + scan64(m4, lane) - m4;
                const bool here = by_count ? n + n4 >= k : (double)(s + m4) >= target && n4;
                const uint64_t who = __ballot(here);
                // (a target that rounding puts past the whole mass: the last bin that holds something)
                const uint64_t held = __ballot(n4 != 0);
                const int l0 = who ? __builtin_ctzll(who) : 63 - __builtin_clzll(held);
                if (lane == l0) {
                    int bin = -1;
                    for (int j = 0; j < 4; j++) {
                        const int q = 255 - 4 * lane - j;
                        if (!cnt[q]) continue;
                        if (bin >= 0) n += cnt[bin], s += mass[bin];
                        bin = q;
                        if (by_count ? n + cnt[q] >= k : (double)(s + mass[q]) >= target) break;
                    }
                    picked[0] = n, picked[1] = s, picked[2] = (uint64_t)bin, picked[3] = (uint64_t)cnt[bin];
                }
            }
            __syncthreads();
            above_n = picked[0], above_m = picked[1];
            prefix = prefix << 8 | (uint32_t)picked[2];
        }
        const uint64_t held = picked[3], each = wt.mass(wt.of(logit_of(prefix)));
        uint64_t n = 0;
        if (by_count) {
            n = k - above_n;
        } else {                                         // tokens at the key whose running sum before them is below the target
            const double left = target - (double)above_m;
            n = left <= 0. ? 0 : each ? (uint64_t)(left / (double)each) : held;
            while (n > 0 && (double)(above_m + (n - 1) * each) >= target) n--;
            while (n < held && (double)(above_m + n * each) < target) n++;
        }
        t = prefix;
        nt = (uint32_t)(n < 1 ? 1 : n > held ? held : n);
        total = above_m + nt * each;
        __syncthreads();
    };
    const int k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
    bool have = false;
    if (k > 0 && k < V) cut(true, (uint64_t)k, 0.), have = true;
    if (top_p < 1.f) {
        if (!have) {
            uint64_t s = 0;
            for (int i = tid; i < V; i += kThreads) s += wt.mass(wt.of((float)x[i]));
            s = scan64(s, lane);
            if (lane == 63) seg[wave] = s;
            __syncthreads();
            for (int w = 0; w < kWaves; w++) total += seg[w];
            __syncthreads();
        }
        cut(false, 0, (double)top_p * (double)total);
    }
    // the draw: each wave a run of the row
    const int len = ((V + kWaves - 1) / kWaves + 63) & ~63, lo = min(wave * len, V), hi = min(lo + len, V);
    uint32_t n = 0;
    for (int i = lo; i < hi; i += 64) n += __popcll(__ballot(i + lane < hi && key_of((float)x[min(i + lane, V - 1)]) == t));
    if (lane == 0) ties[wave] = n;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; w++) before += ties[w];
    // mass of the token i + lane, 0 where it is not kept
    auto kept = [&](int i, uint32_t& rank) {
        const float l = i + lane < hi ? (float)x[i + lane] : -INFINITY;
        const uint32_t key = key_of(l);
        const uint64_t same = __ballot(i + lane < hi && key == t);
        const uint32_t r = rank + __popcll(same & ((1ull << lane) - 1));
        rank += __popcll(same);
        const double w = wt.of(l);
        return i + lane < hi && (key > t || (key == t && r < nt)) && (!(min_p > 0.f) || w >= fmin((double)min_p, 1.)) ? wt.mass(w) : 0;
    };
    uint32_t rank = before;
    uint64_t s = 0;
    for (int i = lo; i < hi; i += 64) s += kept(i, rank);
    s = scan64(s, lane);
    if (lane == 63) seg[wave] = s;
    __syncthreads();
    uint64_t all = 0, ahead = 0, mine = seg[wave];
    for (int w = 0; w < kWaves; w++) all += seg[w], ahead += w < wave ? seg[w] : 0;
    const float u = a.u[row];
    // (past every sum, where u is 1 or more: the last kept token)
    const double most = (double)all * (u > 0.f ? (double)u : 0.);
    uint64_t at = (uint64_t)fmin(most, (double)all);
    at = at < all ? at : all - 1;                        // a token's running sum must exceed it
    if (at < ahead || at >= ahead + mine) return;
    rank = before;
    for (int i = lo; i < hi; i += 64) {
        const uint64_t w = kept(i, rank), sum = ahead + scan64(w, lane);
        const uint64_t who = __ballot(sum > at);
        if (who) {
            if (lane == __builtin_ctzll(who)) answer(i + lane, (float)((double)w / (double)all));
            return;
        }
        ahead = shfl64(sum, 63);
    }
}

}  // namespace

double sample_unit(int V) {
    int bits = 0;
    while ((1ll << bits) < V) bits++;
    const int s = 62 - bits < 51 ? 62 - bits : 51;
    return (double)(1ull << s);
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)a.rows);
    if (a.f16) hipLaunchKernelGGL(k_sample<_Float16>, grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL(k_sample<float>, grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace mgh
