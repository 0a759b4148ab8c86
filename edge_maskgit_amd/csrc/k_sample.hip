// k_sample.hip — drawing a token from logits (gfx950).
//
// Per row: m the largest logit, w = exp((l - m) / T); tokens in descending l, equal ones in the order of their ids; kept is
// the shortest prefix of that order which top-k (its length), top-p (its share of the first k's mass) and min-p (its
// last w) allow; drawn is the first kept token, in the order of the ids, whose running sum exceeds u times the kept mass.
//
// A token's place in that order is a whole number of 64 bits (its key's complement, then its id), and what is kept is all up
// to one place. Where that lies, for top-k and then for top-p: tokens are counted and their masses summed by bins of
// log2 w, the bin that the border falls into is found by a scan, and its tokens (few) are ranked against one another;
// more than a list holds are first shared out again by their places, as often as it takes.
//
// Which token a sum's border falls on must not depend on how sums are split, so masses are whole numbers of 2^-S of the
// largest weight, exp2 in 64 bits rounded once: they add up exactly in any order, atomics included. S leaves room for the
// row (63 bits for its sum) and is at most 51, where the rounding is an addition of 2^52.
//
// Measured: one row of 2025 with top-k and top-p 13 us, 1028 rows with min-p 9.7 (0.9 TB/s; the exponentials); 64 rows of 128001
// 33 us without a cut or with min-p, 43 with top-k and top-p, 55 with top-p alone; one row of 128001 17, 27 and 32, of a million 17,
// 44 and 70.
#include <algorithm>

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

// 2^t, t = d c <= 0, off by 2^-51 of it and 2^-53 |t|: the nearest whole number's power and the series of the rest, |f| <= 1/2, by
// pairs of terms (Horner's rule is a chain of 13 dependent steps: a row of 2025 tokens 16.5 us with it). Every fused step
// is written out: kernels that must agree on a token's mass to the last bit do not leave it to the compiler
__device__ __forceinline__ double exp2_64(double d, double c) {
    const double t = d * c, n = rint(fmax(t, -1100.)), f = fma(d, c, -n), f2 = f * f, f4 = f2 * f2;
    const double p0 = fma(0.6931471805599453, f, 1.), p1 = fma(0.055504108664821576, f, 0.2402265069591007);
    const double p2 = fma(0.0013333558146428441, f, 0.009618129107628477), p3 = fma(1.5252733804059838e-05, f, 0.00015403530393381606);
    const double p4 = fma(1.0178086009239696e-07, f, 1.3215486790144305e-06), p5 = fma(4.44553827187081e-10, f, 7.054911620801121e-09);
    const double q0 = fma(p1, f2, p0), q1 = fma(p3, f2, p2), q2 = fma(fma(2.5678435993488206e-11, f2, p5), f2, p4);
    const double p = fma(fma(q2, f4, q1), f4, q0);
    return t < -1000. ? 0. : ldexp(p, (int)n);
}

struct Weights {
    double m, c;           // largest logit, log2(e) / T
    double unit;           // 2^S
    // weight of a logit relative to the largest one's
    __device__ __forceinline__ double of(float l) const {
        const double w = exp2_64((double)l - m, c);
        // (whatever T is; infinities among themselves)
        return (double)l == m ? 1. : l == -INFINITY || m == INFINITY ? 0. : w;
    }
    __device__ __forceinline__ uint64_t mass(double w) const {
        return __builtin_bit_cast(uint64_t, fma(w, unit, 4503599627370496.)) & 0xfffffffffffffull;
    }
};

// sums of the lanes up to and with this one
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t scan64(uint64_t v) {
    v += moved<0x111, 0xf>(v);           // one, two, four, eight lanes up within rows of 16
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);           // a row's last lane to the next row, then the first half's to the second
    v += moved<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int l) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
__device__ __forceinline__ uint64_t sum64(uint64_t v) { return lane64(scan64(v), 63); }

constexpr int kBins = 512, kMostWaves = 16;
typedef unsigned long long ull;

// LIST: tokens of a bin that it holds
template <int LIST, int THREADS>
struct Lds {
    static constexpr int kList = LIST, kThreads = THREADS;
    uint64_t mass[kBins], place[LIST + 64], w[LIST + 64];      // (the last 64: those that are ranked)
    uint64_t part[kMostWaves], lo[kMostWaves], hi[kMostWaves], found[4];
    uint32_t cnt[kBins];
    float redf[kMostWaves][2];
    int redi[kMostWaves];
    uint32_t n;
};

// what a row asks for
struct Ask {
    float temp, top_p, min_p, u;
    int k;
    bool greedy, by_k, by_p;
    // whether min-p leaves a token of this weight in
    __device__ __forceinline__ bool likely(double w) const { return !(min_p > 0.f) || w >= fmin((double)min_p, 1.); }
};
__device__ __forceinline__ Ask ask_of(const SampleArgs& a, int64_t row) {
    Ask q;
    q.temp = a.temp ? a.temp[row] : 1.f;
    q.k = a.top_k ? a.top_k[row] : 0;
    q.top_p = a.top_p ? a.top_p[row] : 1.f;
    q.min_p = a.min_p ? a.min_p[row] : 0.f;
    q.u = a.u[row];
    q.greedy = !(q.temp > 0.f);
    q.by_k = q.k > 0 && q.k < a.V;
    q.by_p = q.top_p < 1.f;
    return q;
}

// weights and bins of a row whose logits lie between lo (the least that is finite) and m: bins of equal parts of that span,
// or of the 64 octaves below m where it is wider. fp32: all that a bin needs is that a larger logit's is no later
struct Scale {
    Weights wt;
    float m, cs;           // largest logit, bins per unit of logit
    __device__ __forceinline__ Scale(float most, float lo, float temp, double unit) {
        wt = Weights{(double)most, 1.4426950408889634 / (double)temp, unit};
        m = most;
        const double span = (double)most - (double)lo, octaves = 64. / wt.c;
        cs = span > 0. ? (float)((kBins - 1) / (span < octaves ? span : octaves)) : 0.f;
    }
    __device__ __forceinline__ int bin(float l) const {
        const float x = (m - l) * cs;
        return l == m ? 0 : x < (float)(kBins - 1) ? (int)x : kBins - 1;
    }
    __device__ __forceinline__ uint64_t mass(float l) const { return wt.mass(wt.of(l)); }
};
__device__ __forceinline__ uint64_t place_of(float l, int i) { return (uint64_t)(~key_of(l)) << 32 | (uint32_t)i; }

// The least key of a logit that is no NaN for which ok holds, as it does from there up to `hi`: 64 candidates at a time, by every
// wave for itself
template <class F>
__device__ __forceinline__ uint32_t least_key(uint32_t hi, F ok) {
    const int lane = threadIdx.x & 63;
    uint32_t lo = 0;
    while (lo < hi) {                    // the key is in lo .. hi
        const uint32_t step = (hi - lo) / 64 + 1, off = step * lane;
        const uint32_t x = off < hi - lo ? lo + off : hi;
        const float l = logit_of(x);
        const uint64_t some = __ballot(l == l && ok(l));              // (keys below -infinity's are NaN)
        const int first = some ? __builtin_ctzll(some) : 64;
        if (first < 64) hi = (uint32_t)__builtin_amdgcn_readlane((int)x, first);
        if (first > 0) lo = (uint32_t)__builtin_amdgcn_readlane((int)x, first - 1) + 1;
    }
    return hi;
}
// Where a running count or mass, over the bins in order, reaches `k` or `target`: found = count and mass before the bin, its
// number, its count. By wave 0; the others wait.
template <class L>
__device__ __forceinline__ void find_bin(L& s, bool by_count, uint64_t k, double target, uint64_t n, uint64_t m) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid < 64) {
        constexpr int E = kBins / 64;
        uint32_t c[E];
        uint64_t w[E], cn = 0, wn = 0;
#pragma unroll
        for (int j = 0; j < E; j++) cn += c[j] = s.cnt[E * tid + j], wn += w[j] = s.mass[E * tid + j];
        n += scan64(cn) - cn;
        m += scan64(wn) - wn;
        auto there = [&](uint64_t nn, uint64_t mm) { return by_count ? nn >= k : (double)mm >= target; };
        const uint64_t who = __ballot(cn && there(n + cn, m + wn)), held = __ballot(cn != 0);
        // (a target that rounding puts past the whole mass: the last bin that holds something)
        if (tid == (who ? __builtin_ctzll(who) : 63 - __builtin_clzll(held))) {
            int at = -1;
            uint32_t have = 0;
            uint64_t weight = 0;
            bool done = false;
#pragma unroll
            for (int j = 0; j < E; j++) {
                if (done || !c[j]) continue;
                n += have, m += weight;
                at = E * tid + j, have = c[j], weight = w[j];
                done = there(n + have, m + weight);
            }
            s.found[0] = n, s.found[1] = m, s.found[2] = (uint64_t)at, s.found[3] = have;
        }
    }
    __syncthreads();
}

struct Cut {
    uint64_t place;        // of the last token kept
    uint64_t mass;         // of the tokens up to it
    int bin;               // whose tokens the list holds, -1: none
    bool intact;           // the bins are as they were
    uint32_t held;         // tokens of the bin
};

// The last place that a count of k or a mass of `target` keeps, at least the first: the row's bins are in s.cnt and s.mass;
// each(bin, f) calls f(logit, id) for the tokens of a bin (and maybe others). A list is filled where it holds the bin.
template <class L, class Each>
__device__ __forceinline__ Cut cut_at(L& s, const Scale& sc, bool by_count, uint64_t k, double target, Each each) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nt = L::kThreads;
    find_bin(s, by_count, k, target, 0, 0);
    uint64_t n = s.found[0], m = s.found[1];
    const int bin = (int)s.found[2];
    uint32_t held = (uint32_t)s.found[3];
    const uint32_t all = held;
    const bool listed = L::kList && held <= (uint32_t)L::kList;
    uint64_t lo = 0, hi = ~0ull;                         // places that are left
    auto gather = [&](auto from, int at) {               // tokens left, in any order
        if (tid == 0) s.n = 0;
        __syncthreads();
        from([&](uint64_t p, auto mass) {
            if (p < lo || p > hi) return;
            const uint32_t i = at + atomicAdd(&s.n, 1u);
            s.place[i] = p, s.w[i] = mass();
        });
        __syncthreads();
    };
    auto row = [&](auto f) {
        each(bin, [&](float l, int i) {
            if (sc.bin(l) == bin) f(place_of(l, i), [&] { return sc.mass(l); });
        });
    };
    auto list = [&](auto f) {
        for (uint32_t i = tid; i < all; i += nt) f(s.place[i], [&] { return s.w[i]; });
    };
    if (listed) gather(row, 0);
    auto narrow = [&](auto from) {                       // shared out again, by 9 bits of the span of the places left
        uint64_t a = ~0ull, b = 0;
        from([&](uint64_t p, auto) {
            if (p >= lo && p <= hi) a = p < a ? p : a, b = p > b ? p : b;
        });
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t x = (uint64_t)__shfl_xor((ull)a, d), y = (uint64_t)__shfl_xor((ull)b, d);
            a = x < a ? x : a, b = y > b ? y : b;
        }
        __syncthreads();
        if (lane == 0) s.lo[wave] = a, s.hi[wave] = b;
        for (int i = tid; i < kBins; i += nt) s.cnt[i] = 0, s.mass[i] = 0;
        __syncthreads();
        for (int w = 0; w < nt / 64; w++) a = s.lo[w] < a ? s.lo[w] : a, b = s.hi[w] > b ? s.hi[w] : b;
        const int bits = b > a ? 64 - __builtin_clzll(b - a) : 0, shift = bits > 9 ? bits - 9 : 0;
        from([&](uint64_t p, auto mass) {
            if (p < a || p > b) return;
            atomicAdd(&s.cnt[(p - a) >> shift], 1u);
            atomicAdd((ull*)&s.mass[(p - a) >> shift], (ull)mass());
        });
        find_bin(s, by_count, k, target, n, m);
        n = s.found[0], m = s.found[1], held = (uint32_t)s.found[3];
        lo = a + (s.found[2] << shift);
        hi = lo + ((1ull << shift) - 1);
    };
    bool intact = true;
    while (held > 64) {
        intact = false;
        if (listed) narrow(list);
        else narrow(row);
    }
    if (listed) gather(list, L::kList);
    else gather(row, L::kList);
    if (wave == 0) {                                     // ranked against one another
        const uint64_t p = lane < (int)held ? s.place[L::kList + lane] : ~0ull, w = lane < (int)held ? s.w[L::kList + lane] : 0;
        uint32_t rank = 0;
        uint64_t before = 0;
        for (uint32_t j = 0; j < held; j++) {
            const bool b = lane64(p, j) < p;
            rank += b;
            before += b ? lane64(w, j) : 0;
        }
        const bool keep = lane < (int)held && (by_count ? n + rank < k : n + rank == 0 || (double)(m + before) < target);
        const int last = __popcll(__ballot(keep));       // kept ones are the first of them
        if (lane < (int)held && (int)rank + 1 == last) s.found[0] = p, s.found[1] = m + before + w;
    }
    __syncthreads();
    const Cut c{s.found[0], s.found[1], listed ? bin : -1, intact, all};
    __syncthreads();
    return c;
}

// largest, least finite logit and whether there is a NaN, of a workgroup
template <class L>
__device__ __forceinline__ void reduce_range(L& s, float& m, float& lo, bool& nan) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d)), lo = fminf(lo, __shfl_xor(lo, d));
    const bool any = __any(nan);
    if (lane == 0) s.redf[wave][0] = m, s.redf[wave][1] = lo, s.redi[wave] = any;
    __syncthreads();
    nan = false;
    for (int w = 0; w < L::kThreads / 64; w++) m = fmaxf(m, s.redf[w][0]), lo = fminf(lo, s.redf[w][1]), nan = nan || s.redi[w];
}

struct Answer {
    int32_t* id;
    float* prob;
    __device__ __forceinline__ void put(int i, float p) const {
        *id = i;
        if (prob) *prob = p;
    }
};

// masses of a workgroup's tokens (NV of a thread), wave by wave in s.part, and their sum
template <int NV, class L>
__device__ __forceinline__ uint64_t wave_sums(L& s, const uint64_t* mass) {
    uint64_t v = 0;
#pragma unroll
    for (int j = 0; j < NV; j++) v += mass[j];
    v = sum64(v);
    if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t all = 0;
    for (int w = 0; w < L::kThreads / 64; w++) all += s.part[w];
    return all;
}
// what a running sum must exceed: u of the whole, short of all of it
__device__ __forceinline__ uint64_t draw_at(float u, uint64_t all) {
    const double most = (double)all * (u > 0.f ? fmin((double)u, 1.) : 0.);
    const uint64_t at = (uint64_t)most;
    return at < all ? at : all - 1;
}
// The draw among a workgroup's tokens, of which (wave NV + j) 64 + lane weighs mass[j] (sums in s.part): `all` the row's mass, `at`
// what the running sum must exceed, `ahead` the sum before the first token, id0 its id
template <int NV, class L>
__device__ __forceinline__ void draw(L& s, const uint64_t* mass, uint64_t ahead, uint64_t all, uint64_t at, int id0, const Answer& out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int w = 0; w < wave; w++) ahead += s.part[w];
    if (at < ahead || at >= ahead + s.part[wave]) return;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const uint64_t run = ahead + scan64(mass[j]);
        const uint64_t who = __ballot(run > at);
        if (who) {
            if (lane == __builtin_ctzll(who)) out.put(id0 + (wave * NV + j) * 64 + lane, (float)((double)mass[j] / (double)all));
            return;
        }
        ahead = lane64(run, 63);
    }
}

// Short rows: a workgroup holds a row in LDS, NV tokens of a thread: (wave NV + j) 64 + lane. Top-k counts only, so that with
// it the exponentials are those of the first k tokens.
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void k_sample(SampleArgs a) {
    __shared__ Lds<0, NT> s;
    __shared__ float val[NT * NV];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.V;
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.x_stride;
    const Answer out{a.ids + row, a.prob ? a.prob + row : nullptr};
    float m = -INFINITY, lo = INFINITY;
    bool nan = false;
    const int first = wave * NV * 64 + lane;
    {
        float l[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) l[j] = first + 64 * j < V ? (float)x[first + 64 * j] : -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            val[first + 64 * j] = l[j];
            nan = nan || l[j] != l[j];
            m = fmaxf(m, l[j]);
            lo = l[j] > -INFINITY ? fminf(lo, l[j]) : lo;
        }
    }
    const Ask q = ask_of(a, row);
    reduce_range(s, m, lo, nan);
    if (nan || m == -INFINITY) {
        if (tid == 0) out.put(-1, nan ? __builtin_nanf("") : 0.f);
        return;
    }
    if (q.greedy) {                      // the first of the largest
        int best = INT32_MAX;
        for (int j = NV - 1; j >= 0; j--) {
            const uint64_t who = __ballot(val[first + 64 * j] == m);
            best = who ? (wave * NV + j) * 64 + __builtin_ctzll(who) : best;
        }
        __syncthreads();
        if (lane == 0) s.redi[wave] = best;
        __syncthreads();
        for (int w = 0; w < NT / 64; w++) best = min(best, s.redi[w]);
        if (tid == 0) out.put(best, 1.f);
        return;
    }
    const Scale sc(m, lo, q.temp, a.unit);
    uint64_t last = ~0ull;               // the last place that is kept
    auto each = [&](int, auto f) {       // this thread's tokens that are left
#pragma unroll (NT == 256 ? NV : 2)
        for (int j = 0; j < NV; j++) {
            const int i = first + 64 * j;
            const float l = val[i];
            if (i < V && place_of(l, i) <= last) f(l, i);
        }
    };
    auto fill = [&](bool masses) {
        for (int i = tid; i < kBins; i += NT) s.cnt[i] = 0, s.mass[i] = 0;
        __syncthreads();
        each(0, [&](float l, int) {
            const int b = sc.bin(l);
            atomicAdd(&s.cnt[b], 1u);
            if (masses) atomicAdd((ull*)&s.mass[b], (ull)sc.mass(l));
        });
    };
    if (q.by_k) {
        fill(false);
        last = cut_at(s, sc, true, (uint64_t)q.k, 0., each).place;
    }
    if (q.by_p) {
        fill(true);
        __syncthreads();
        uint64_t v = 0;
        for (int i = tid; i < kBins; i += NT) v += s.mass[i];
        const uint64_t total = wave_sums<1>(s, &v);
        last = cut_at(s, sc, false, 0, (double)q.top_p * (double)total, each).place;
    }
    uint64_t mass[NV];
    constexpr int U = NT == 256 ? 4 : 2;                 // exponentials beside one another
#pragma unroll
    for (int j0 = 0; j0 < NV; j0 += U) {
        float l[U];
        bool keep[U], some = false;
#pragma unroll
        for (int j = 0; j < U; j++) {
            const int i = first + 64 * (j0 + j);
            l[j] = val[i];
            keep[j] = i < V && place_of(l[j], i) <= last;
            some = some || keep[j];
            mass[j0 + j] = 0;
        }
        if (!__any(some)) continue;
#pragma unroll
        for (int j = 0; j < U; j++) {
            const double w = sc.wt.of(l[j]);
            // (likely(w), written out: by a call of it a row of 2025 takes 14.0 us instead of 13.0)
            mass[j0 + j] = keep[j] && (!(q.min_p > 0.f) || w >= fmin((double)q.min_p, 1.)) ? sc.wt.mass(w) : 0;
        }
    }
    const uint64_t all = wave_sums<NV>(s, mass);
    draw<NV>(s, mass, 0, all, draw_at(q.u, all), 0, out);
}

// Long rows: chunks of kChunk tokens. The first launch notes each chunk's range; the second, which knows the row's, its bins and
// its ids in the order of the bins (or, where neither k nor p cuts, its kept mass); the third, a workgroup per row, adds
// the bins up, cuts (a bin's tokens by their ids: reading the row again took 28 us of a cut in its bulk), finds the chunk in
// which the draw lies, and draws there.
constexpr int kChunk = 8192, kMostChunks = (1 << 24) / kChunk;
struct Long {
    int chunks, row0;      // chunks of a row; the first row of this launch
    f32x4* range;          // [rows][chunks] largest, least finite logit, NaN
    uint64_t* kept;        // [rows][chunks]
    uint64_t* mass;        // [rows][chunks][kBins]
    uint32_t* cnt;         // 16 bits: where a bin's ids begin, 16 bits: their number
    uint16_t* ids;         // [rows][chunks][kChunk] within the chunk
};

// NV logits of a thread of the chunk from id0 on; past the row -infinity
template <typename T, int NT>
__device__ __forceinline__ void load_chunk(const T* x, int V, int id0, float* l) {
    constexpr int NV = kChunk / NT;
    const int at = id0 + (threadIdx.x >> 6) * NV * 64 + (threadIdx.x & 63);
    if (id0 + kChunk <= V) {
#pragma unroll
        for (int j = 0; j < NV; j++) l[j] = (float)x[at + 64 * j];
    } else {
#pragma unroll
        for (int j = 0; j < NV; j++) l[j] = at + 64 * j < V ? (float)x[at + 64 * j] : -INFINITY;
    }
}

template <typename T>
__global__ __launch_bounds__(512) void k_sample_range(SampleArgs a, Long g) {
    constexpr int NV = kChunk / 512;
    __shared__ Lds<0, 512> s;
    const int64_t row = g.row0 + blockIdx.y;
    float l[NV], m = -INFINITY, lo = INFINITY;
    load_chunk<T, 512>((const T*)a.x + row * a.x_stride, a.V, blockIdx.x * kChunk, l);
    bool nan = false;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        nan = nan || l[j] != l[j];
        m = fmaxf(m, l[j]);
        lo = l[j] > -INFINITY ? fminf(lo, l[j]) : lo;
    }
    reduce_range(s, m, lo, nan);
    if (threadIdx.x == 0) g.range[(int64_t)blockIdx.y * g.chunks + blockIdx.x] = f32x4{m, lo, nan ? 1.f : 0.f, 0.f};
}

template <class L>
__device__ __forceinline__ void row_range(L& s, const Long& g, float& m, float& lo, bool& nan) {
    m = -INFINITY, lo = INFINITY, nan = false;
    for (int c = threadIdx.x; c < g.chunks; c += L::kThreads) {
        const f32x4 r = g.range[(int64_t)blockIdx.y * g.chunks + c];
        m = fmaxf(m, r[0]), lo = fminf(lo, r[1]), nan = nan || r[2] != 0.f;
    }
    reduce_range(s, m, lo, nan);
}

template <typename T>
__global__ __launch_bounds__(512, 4) void k_sample_bins(SampleArgs a, Long g) {
    constexpr int NV = kChunk / 512;
    __shared__ Lds<0, 512> s;
    __shared__ __attribute__((aligned(16))) uint16_t ids[kChunk];
    const int tid = threadIdx.x, id0 = blockIdx.x * kChunk;
    const int64_t row = g.row0 + blockIdx.y, at = (int64_t)blockIdx.y * g.chunks + blockIdx.x;
    float l[NV], m, lo;
    bool nan;
    load_chunk<T, 512>((const T*)a.x + row * a.x_stride, a.V, id0, l);
    for (int i = tid; i < kBins; i += 512) s.cnt[i] = 0, s.mass[i] = 0;
    const Ask q = ask_of(a, row);
    row_range(s, g, m, lo, nan);
    if (nan || m == -INFINITY || q.greedy) return;
    const Scale sc(m, lo, q.temp, a.unit);
    const int first = id0 + (tid >> 6) * NV * 64 + (tid & 63);
    if (q.by_k || q.by_p) {
        uint32_t bin[NV];                // and the number of the token among its bin's; past the row: none
#pragma unroll
        for (int j = 0; j < NV; j++) {
            bin[j] = first + 64 * j < a.V ? sc.bin(l[j]) : kBins;
            if (bin[j] < kBins) bin[j] |= atomicAdd(&s.cnt[bin[j]], 1u) << 16;
        }
        uint32_t most = kBins - 1;
        if (q.by_k && q.k < kChunk) {    // what the first k of the row cannot hold is left out: all but the chunk's own first k
            find_bin(s, true, (uint64_t)q.k, 0., 0, 0);
            most = (uint32_t)s.found[2];
        } else {
            __syncthreads();
        }
        if (tid < 64) {                  // where each bin's ids begin
            constexpr int E = kBins / 64;
            uint32_t c[E], n = 0;
#pragma unroll
            for (int j = 0; j < E; j++) c[j] = s.cnt[E * tid + j], n += c[j];
            uint32_t o = (uint32_t)scan64(n) - n;
#pragma unroll
            for (int j = 0; j < E; j++) s.cnt[E * tid + j] = o << 16 | c[j], o += c[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const uint32_t b = bin[j] & 0xffff;
            if (b <= most) {
                atomicAdd((ull*)&s.mass[b], (ull)sc.mass(l[j]));
                ids[(s.cnt[b] >> 16) + (bin[j] >> 16)] = (uint16_t)(first - id0 + 64 * j);
            }
            if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);       // (four exponentials' registers at a time)
        }
        __syncthreads();
        for (int i = tid; i < kBins; i += 512) g.cnt[at * kBins + i] = s.cnt[i], g.mass[at * kBins + i] = s.mass[i];
        const int n = ((s.cnt[most] >> 16) + (s.cnt[most] & 0xffff) + 7) / 8;
        for (int i = tid; i < n; i += 512) *(u32x4*)(g.ids + at * kChunk + 8 * i) = *(const u32x4*)(ids + 8 * i);
        return;
    }
    uint64_t mass[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const double w = sc.wt.of(l[j]);
        mass[j] = q.likely(w) ? sc.wt.mass(w) : 0;
        if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    const uint64_t all = wave_sums<NV>(s, mass);
    if (tid == 0) g.kept[at] = all;
}

template <typename T>
__global__ __launch_bounds__(1024) void k_sample_pick(SampleArgs a, Long g) {
    constexpr int NT = 1024, NV = kChunk / NT;
    __shared__ Lds<2048, NT> s;
    __shared__ uint64_t kept[kMostChunks];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.V;
    const int64_t row = g.row0 + blockIdx.y, at0 = (int64_t)blockIdx.y * g.chunks;
    const T* x = (const T*)a.x + row * a.x_stride;
    const Answer out{a.ids + row, a.prob ? a.prob + row : nullptr};
    float m, lo;
    bool nan;
    const Ask q = ask_of(a, row);
    row_range(s, g, m, lo, nan);
    if (nan || m == -INFINITY) {
        if (tid == 0) out.put(-1, nan ? __builtin_nanf("") : 0.f);
        return;
    }
    float l[NV];
    const int first = wave * NV * 64 + lane;
    if (q.greedy) {
        auto least = [&](int v) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) v = min(v, __shfl_xor(v, d));
            __syncthreads();
            if (lane == 0) s.redi[wave] = v;
            __syncthreads();
            for (int w = 0; w < NT / 64; w++) v = min(v, s.redi[w]);
            return v;
        };
        int best = INT32_MAX;
        for (int c = tid; c < g.chunks; c += NT)
            if (g.range[at0 + c][0] == m) best = min(best, c);
        const int id0 = least(best) * kChunk;
        load_chunk<T, NT>(x, V, id0, l);
        best = INT32_MAX;
#pragma unroll
        for (int j = NV - 1; j >= 0; j--)
            if (l[j] == m) best = id0 + first + 64 * j;
        best = least(best);
        if (tid == 0) out.put(best, 1.f);
        return;
    }
    const Scale sc(m, lo, q.temp, a.unit);
    uint64_t last = ~0ull;
    const bool cut = q.by_k || q.by_p;
    if (cut) {
        if (q.min_p > 0.f)
            last = (uint64_t)~least_key(key_of(m), [&](float y) { return q.likely(sc.wt.of(y)); }) << 32 | 0xffffffffull;
        auto fill = [&] {                // the row's bins: two halves of the chunks
            const int b = tid & (kBins - 1), half = tid / kBins;
            uint32_t n = 0;
            uint64_t w = 0;
#pragma unroll 8
            for (int c = half; c < g.chunks; c += NT / kBins) n += g.cnt[(at0 + c) * kBins + b] & 0xffff, w += g.mass[(at0 + c) * kBins + b];
            __syncthreads();
            if (half) s.cnt[b] = n, s.mass[b] = w;
            __syncthreads();
            if (!half) s.cnt[b] += n, s.mass[b] += w;
            __syncthreads();
        };
        auto each = [&](int bin, auto f) {               // a wave per chunk
            for (int c = wave; c < g.chunks; c += NT / 64) {
                const uint32_t w = g.cnt[(at0 + c) * kBins + bin], n = w & 0xffff;
                const uint16_t* ids = g.ids + (at0 + c) * kChunk + (w >> 16);
                for (uint32_t i = lane; i < n; i += 64) {
                    const int id = c * kChunk + ids[i];
                    f((float)x[id], id);
                }
            }
        };
        fill();
        Cut c{~0ull, 0, -1, true, 0};
        uint64_t total = 0;
        if (q.by_k) {
            c = cut_at(s, sc, true, (uint64_t)q.k, 0., each);
            last = c.place < last ? c.place : last;
            total = c.mass;
            if (q.by_p && !c.intact) fill();
        }
        if (q.by_p) {
            if (!q.by_k) {
                const uint64_t v = tid < kBins ? s.mass[tid] : 0;
                total = wave_sums<1>(s, &v);
            }
            c = cut_at(s, sc, false, 0, (double)q.top_p * (double)total, each);
            last = c.place < last ? c.place : last;
        }
        // each chunk's kept mass: bins before the last place's, and what is kept of that one
        const int bin = sc.bin(logit_of(~(uint32_t)(last >> 32)));
        for (int k = wave; k < g.chunks; k += NT / 64) {
            uint64_t v = 0;
#pragma unroll
            for (int i = 0; i < kBins / 64; i++) {
                const int b = 64 * i + lane;
                const uint64_t w = g.mass[(at0 + k) * kBins + b];
                v += b < bin ? w : 0;
            }
            v = sum64(v);
            if (lane == 0) kept[k] = v;
        }
        __syncthreads();
        auto add = [&](uint64_t p, uint64_t w) {
            if (p <= last) atomicAdd((ull*)&kept[(uint32_t)p / kChunk], (ull)w);
        };
        if (c.bin == bin) {
            const uint32_t n = c.held;
            for (uint32_t i = tid; i < n; i += NT) add(s.place[i], s.w[i]);
        } else {
            each(bin, [&](float y, int i) {
                if (sc.bin(y) == bin && place_of(y, i) <= last) add(place_of(y, i), sc.mass(y));
            });
        }
    } else {
        for (int c = tid; c < g.chunks; c += NT) kept[c] = g.kept[at0 + c];
    }
    __syncthreads();
    uint64_t all = 0;
    for (int c = tid; c < g.chunks; c += NT) all += kept[c];
    all = wave_sums<1>(s, &all);
    const uint64_t at = draw_at(q.u, all);
    if (wave == 0) {
        uint64_t ahead = 0;
        for (int c0 = 0; c0 < g.chunks; c0 += 64) {
            const uint64_t run = ahead + scan64(c0 + lane < g.chunks ? kept[c0 + lane] : 0);
            const uint64_t who = __ballot(run > at);
            if (who) {
                const int w = __builtin_ctzll(who);
                if (lane == w) s.found[0] = (uint64_t)(c0 + lane), s.found[1] = run - kept[c0 + lane];
                break;
            }
            ahead = lane64(run, 63);
        }
    }
    __syncthreads();
    const int id0 = (int)s.found[0] * kChunk;
    const uint64_t ahead = s.found[1];
    load_chunk<T, NT>(x, V, id0, l);
    // Without a cut by the comparison that the chunk's mass was kept by and not by a place: weights within 2^-51 of min-p need not
    // fall with the logits, and a draw past what the tokens of this chunk add up to would be none of them. (Loops of their own:
    // one that takes each token's weight and then either test 44.9 us instead of 42.8, 64 rows of 128001 with top-k and top-p)
    uint64_t mass[NV];
    if (cut) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = id0 + first + 64 * j;
            mass[j] = i < V && place_of(l[j], i) <= last ? sc.mass(l[j]) : 0;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const double w = sc.wt.of(l[j]);
            mass[j] = id0 + first + 64 * j < V && q.likely(w) ? sc.wt.mass(w) : 0;
        }
    }
    wave_sums<NV>(s, mass);
    draw<NV>(s, mass, ahead, all, at, id0, out);
}

template <typename T>
void launch_short(const SampleArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)a.rows);
    // (1024 threads for short rows too: one row of 1000 5.9 us instead of 5.3, of 2025 with top-k and top-p 15 instead of 13,
    // 1028 rows with top-k 45 instead of 16)
    if (a.V <= 2048) hipLaunchKernelGGL((k_sample<T, 256, 8>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_sample<T, 1024, 8>), grid, dim3(1024), 0, s, a);
}

constexpr size_t kRowBytes = sizeof(f32x4) + sizeof(uint64_t) + kBins * (sizeof(uint64_t) + sizeof(uint32_t)) + kChunk * sizeof(uint16_t);   // of a chunk

template <typename T>
void launch_long(const SampleArgs& a, const SamplePlan& p, hipStream_t s) {
    for (int r0 = 0; r0 < a.rows; r0 += p.batch) {
        const size_t n = (size_t)std::min(p.batch, a.rows - r0) * p.chunks;
        Long g{p.chunks, r0, (f32x4*)a.ws, nullptr, nullptr, nullptr, nullptr};
        g.ids = (uint16_t*)(g.range + n);
        g.mass = (uint64_t*)(g.ids + n * kChunk);
        g.kept = g.mass + n * kBins;
        g.cnt = (uint32_t*)(g.kept + n);
        const unsigned rows = (unsigned)std::min(p.batch, a.rows - r0);
        hipLaunchKernelGGL(k_sample_range<T>, dim3((unsigned)p.chunks, rows), dim3(512), 0, s, a, g);
        hipLaunchKernelGGL(k_sample_bins<T>, dim3((unsigned)p.chunks, rows), dim3(512), 0, s, a, g);
        hipLaunchKernelGGL(k_sample_pick<T>, dim3(1, rows), dim3(1024), 0, s, a, g);
    }
}

}  // namespace

double sample_unit(int V) {
    int bits = 0;
    while ((1ll << bits) < V) bits++;
    const int s = 62 - bits < 51 ? 62 - bits : 51;
    return (double)(1ull << s);
}

// A row in one workgroup up to 8192 tokens (in chunks instead: one row of 8000 17 us instead of 8, with top-p 27 instead of 18; 64
// rows 29 instead of 20; 1028 rows 71 instead of 40); longer ones in chunks, as many rows at a time as 128 MB of bins and ids hold
SamplePlan sample_plan(const SampleArgs& a) {
    SamplePlan p{};
    if (a.V <= kChunk) return p;
    p.chunks = (a.V + kChunk - 1) / kChunk;
    const size_t per = kRowBytes * p.chunks;
    p.batch = (int)std::min<size_t>({(size_t)a.rows, std::max<size_t>(1, ((size_t)128 << 20) / per), 65535});
    p.ws_bytes = per * p.batch;
    return p;
}

hipError_t launch_sample(const SampleArgs& a, const SamplePlan& p, hipStream_t s) {
    if (p.chunks && a.f16) launch_long<_Float16>(a, p, s);
    else if (p.chunks) launch_long<float>(a, p, s);
    else if (a.f16) launch_short<_Float16>(a, s);
    else launch_short<float>(a, s);
    return hipGetLastError();
}

}  // namespace mgh
