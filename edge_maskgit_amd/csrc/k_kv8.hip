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
#include "k_kv8.h"

namespace mgh {

namespace {

__device__ __forceinline__ uint32_t code_of(_Float16 x, float d, float id) {
    const float a = fabsf((float)x), f = floorf(a * id);
    const int q = (int)f + (fmaf(-(f + 0.5f), d, a) >= 0.f ? 1 : 0);
    return (uint32_t)(128 + ((float)x < 0.f ? -q : q));
}

// One workgroup per touched block, head and sequence. Threads take 16 features of a token of K and two
// features of 8 tokens of V: the 16 bytes that they write. The largest |x| goes by its bits, which put
// NaN above infinity: a block that holds either has that scale, and all its values come out NaN.
__global__ __launch_bounds__(256) void k_kv8_append(Kv8AppendArgs a) {
    __shared__ uint32_t mx[2][4];
    const Kv8& c = a.c;
    const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, D = c.D;
    int len, total;
    if (!spans(c, a.lens, a.fresh, a.S, b, len, total)) return;
    const int t0 = (len & ~(kKvBlock - 1)) + kKvBlock * blockIdx.x;      // the block's first token
    if (total == len || t0 >= total) return;
    const int64_t src = b * a.st[3] + hk * a.st[2];
    _Float16* ring_k = c.k_tail + ((int64_t)b * c.Hkv + hk) * kKvRing * D;
    _Float16* ring_v = c.v_tail + ((int64_t)b * c.Hkv + hk) * D * kKvRing;
    auto in = [&](const void* p, int t, int d) -> _Float16 {
        const int64_t e = src + (int64_t)(t - len) * a.st[1] + d * a.st[0];
        return a.in16 ? ((const _Float16*)p)[e] : (_Float16)((const float*)p)[e];
    };
    if (t0 + kKvBlock <= total) {
        const int64_t page = page_of(c, b, t0 / kKvBlock);
        const bool has_k = tid < 2 * D, has_v = tid < 2 * D;             // 32 D / 16 units each
        _Float16 xk[16], xv[16];
        uint32_t m[2] = {0, 0};
        auto widen = [](uint32_t m, _Float16 x) {
            const uint32_t u = __builtin_bit_cast(uint16_t, x) & 0x7fffu;
            return m > u ? m : u;
        };
        const int kt = t0 + tid / (D / 16), kd = 16 * (tid % (D / 16));
        const int vt = t0 + 8 * (tid & 3), vd = 2 * (tid >> 2);
        if (has_k)
            for (int i = 0; i < 16; i++) {
                xk[i] = kt < len ? ring_k[(kt % kKvRing) * D + kd + i] : in(a.k, kt, kd + i);
                m[0] = widen(m[0], xk[i]);
            }
        if (has_v)
            for (int i = 0; i < 16; i++) {
                const int t = vt + (i & 7), d = vd + (i >> 3);
                xv[i] = t < len ? ring_v[d * kKvRing + t % kKvRing] : in(a.v, t, d);
                m[1] = widen(m[1], xv[i]);
            }
        for (int w = 0; w < 2; w++) {
            for (int i = 1; i < 64; i <<= 1) {
                const uint32_t o = __shfl_xor(m[w], i);
                m[w] = m[w] > o ? m[w] : o;
            }
            if ((tid & 63) == 0) mx[w][tid >> 6] = m[w];
        }
        __syncthreads();
        for (int w = 0; w < 2; w++) {
            uint32_t u = 0;
            for (int i = 0; i < 4; i++) u = u > mx[w][i] ? u : mx[w][i];
            const float top = h2f(u), d = top / 127.f, id = u && u < 0x7c00u ? 127.f / top : 0.f;
            if (page < 0 || !(w ? has_v : has_k)) continue;
            const _Float16* x = w ? xv : xk;
            u32x4 q = {0, 0, 0, 0};
            for (int i = 0; i < 16; i++) q[i >> 2] |= (id > 0.f ? code_of(x[i], d, id) : 128u) << (8 * (i & 3));
            const int64_t at = (page * c.Hkv + hk) * kKvBlock * D + (int64_t)16 * tid;
            *(u32x4*)((w ? c.v : c.k) + at) = q;
            if (tid == 0) c.scales[(page * c.Hkv + hk) * 2 + w] = d;
        }
    }
    if (blockIdx.x) return;
    // the ring, by the workgroup that has read what it held (a slot is a position modulo 64)
    __syncthreads();
    const int r0 = total - kKvRing > len ? total - kKvRing : len;
    for (int i = tid; i < (total - r0) * D; i += 256) {
        const int t = r0 + i / D, d = i % D;
        ring_k[(t % kKvRing) * D + d] = in(a.k, t, d);
        ring_v[d * kKvRing + t % kKvRing] = in(a.v, t, d);
    }
}

// values of tokens [first, first + n) that a sequence has: codes times their scale, or the ring's fp16
__global__ __launch_bounds__(256) void k_kv8_read(Kv8ReadArgs a) {
    const Kv8& c = a.c;
    const int hk = blockIdx.y, b = blockIdx.z, D = c.D;
    const int total = a.lens[b], first = a.first ? a.first[b] : 0;
    const bool fits = total >= 0 && first >= 0 && total <= (int64_t)c.max_blocks * kKvBlock;
    const int64_t row = ((int64_t)b * c.Hkv + hk) * a.n;
    auto put = [&](int i, int d, float k, float v) {
        const int64_t e = (row + i) * D + d;
        if (a.k16) a.k16[e] = (_Float16)k, a.v16[e] = (_Float16)v;
        else a.k[e] = k, a.v[e] = v;
    };
    if (!fits) {                                 // numbers that the cache cannot hold
        for (int i = blockIdx.x * kKvBlock; i < a.n && i < ((int)blockIdx.x + 1) * kKvBlock; i++)
            for (int d = threadIdx.x; d < D; d += 256) put(i, d, __builtin_nanf(""), __builtin_nanf(""));
        return;
    }
    const int64_t t0 = (first & ~(kKvBlock - 1)) + (int64_t)kKvBlock * blockIdx.x;
    if (t0 >= total) return;
    const bool whole = t0 + kKvBlock <= total;
    const int64_t page = whole ? page_of(c, b, (int)(t0 / kKvBlock)) : 0;
    const float nan = __builtin_nanf("");
    const int64_t at = (page < 0 ? 0 : page) * c.Hkv + hk;
    const float dk = whole && page >= 0 ? c.scales[2 * at] : nan, dv = whole && page >= 0 ? c.scales[2 * at + 1] : nan;
    for (int i = threadIdx.x; i < kKvBlock * D; i += 256) {
        const int s = i / D, d = i % D;
        const int64_t t = t0 + s, out = t - first;
        if (out < 0 || out >= a.n || t >= total) continue;
        float k = nan, v = nan;
        if (whole) {
            if (page >= 0) {
                k = (float)(c.k[at * kKvBlock * D + s * D + d] - 128) * dk;
                v = (float)(c.v[at * kKvBlock * D + v_at(s, d)] - 128) * dv;
            }
        } else {
            const int64_t r = ((int64_t)b * c.Hkv + hk) * kKvRing * D;
            k = (float)c.k_tail[r + (t % kKvRing) * D + d];
            v = (float)c.v_tail[r + (int64_t)d * kKvRing + t % kKvRing];
        }
        put((int)out, d, k, v);
    }
}

__global__ void k_kv8_advance(int32_t* lens, const int32_t* fresh, int B, int S) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < B) lens[b] += fresh ? fresh[b] : S;      // (32-bit wrap-around lands on a length that every call refuses)
}

}  // namespace

hipError_t launch_kv8_append(const Kv8AppendArgs& a, hipStream_t s) {
    // blocks that S tokens can touch: the open one and what follows
    const dim3 grid((unsigned)(((int64_t)a.S + 2 * kKvBlock - 2) / kKvBlock), (unsigned)a.c.Hkv, (unsigned)a.c.B);
    hipLaunchKernelGGL(k_kv8_append, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8ReadArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(((int64_t)a.n + 2 * kKvBlock - 2) / kKvBlock), (unsigned)a.c.Hkv, (unsigned)a.c.B);
    hipLaunchKernelGGL(k_kv8_read, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_kv8_advance(int32_t* lens, const int32_t* fresh, int B, int S, hipStream_t s) {
    hipLaunchKernelGGL(k_kv8_advance, dim3((unsigned)((B + 255) / 256)), dim3(256), 0, s, lens, fresh, B, S);
    return hipGetLastError();
}

}  // namespace mgh
