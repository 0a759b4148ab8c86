// k_attn_masked.hip — attention under causal, prefix and document masks with capped or sloped scores: the
// narrow heads of the tiled kernel (k_attn_masked.h), the packing of rows that it does not take as they are,
// and the joining of what a head's keys gave in parts.
#include <algorithm>

#include "k_attn_masked.h"

namespace mgh {

namespace {

// {D, S, H, B} views of any type and strides -> fp16 [B][H][S][D]; blockIdx.y: q, k, v. One thread per 8
// features.
__global__ __launch_bounds__(256) void k_attn_pack(PackArgs p) {
    const PackArgs::View& v = p.v[blockIdx.y];
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int D8 = p.D / 8;
    if (n >= (int64_t)p.B * v.H * v.S * D8) return;
    const int d = 8 * (int)(n % D8);
    const int64_t row = n / D8;
    const int64_t e = row / v.S / v.H * v.st[3] + row / v.S % v.H * v.st[2] + row % v.S * v.st[1] + d * v.st[0];
    f16x8 x;
    if (p.in16) {
        const _Float16* s = (const _Float16*)v.src + e;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = s[i * v.st[0]];
    } else {
        const float* s = (const float*)v.src + e;
        if (v.vec) {
            const f32x4 lo = *(const f32x4*)s, hi = *(const f32x4*)(s + 4);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = (_Float16)(i < 4 ? lo[i] : hi[i - 4]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = (_Float16)s[i * v.st[0]];
        }
    }
    *(f16x8*)(v.dst + row * p.D + d) = x;
}

// a joined row's features d .. d + 3
__device__ __forceinline__ void put_row(const JoinArgs& a, int row, int d, const float* o, float l) {
    const int hb = row / a.R, r = row - hb * a.R, i = r / a.G, g = r - i * a.G, b = hb / a.Hkv;
    const int64_t ro = (int64_t)b * a.ost[3] + (int64_t)((hb - b * a.Hkv) * a.G + g) * a.ost[2] + (int64_t)i * a.ost[1];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    f32x4 v;
#pragma unroll
    for (int x = 0; x < 4; x++) v[x] = l == 0.f ? 0.f : o[x] * inv;
    if (a.vec_o) {
        if (a.o16) *(f16x4*)(a.o16 + ro + d) = __builtin_convertvector(v, f16x4);
        else *(f32x4*)(a.o + ro + d) = v;
        return;
    }
#pragma unroll
    for (int x = 0; x < 4; x++) {
        if (a.o16) a.o16[ro + (d + x) * a.ost[0]] = (_Float16)v[x];
        else a.o[ro + (d + x) * a.ost[0]] = v[x];
    }
}

// Few parts (at most P): half a wave per row, 4 features a lane, no wait for another wave. Bound by bytes where rows are
// many (32768 of 128 features in two parts, 42 MB: 8.9 us, 4.7 TB/s; a wave per row, 2 features a lane, 13.4), else by
// one round trip to memory (32 rows 2.8 us).
template <int P>
__global__ __launch_bounds__(256) void k_attn_join_few(JoinArgs a) {
    const int d = 4 * (threadIdx.x & 31), row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= a.rows) return;
    const f32x2* ml = (const f32x2*)(a.ws + (int64_t)a.splits * a.rows * a.D);
    const float* ws = a.ws + (int64_t)row * a.D + (d < a.D ? d : 0);
    // all loads at once: a part that saw nothing wrote no values, whatever lies there is read and not used
    f32x2 st[P];
    f32x4 part[P];
#pragma unroll
    for (int s = 0; s < P; s++) {
        const int64_t at = (int64_t)min(s, a.splits - 1) * a.rows;
        st[s] = ml[at + row];
        part[s] = *(const f32x4*)(ws + at * a.D);
    }
    if (st[0][1] < 0.f) return;              // not a sequence's row
#pragma unroll
    for (int s = 0; s < P; s++)
        if (s >= a.splits) st[s] = f32x2{kNoScore, 0.f};
    float m = st[0][0], l = 0.f;
#pragma unroll
    for (int s = 1; s < P; s++) m = fmaxf(m, st[s][0]);
    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < P; s++) {
        const float w = st[s][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(st[s][0] - m);
        l = fmaf(w, st[s][1], l);
#pragma unroll
        for (int x = 0; x < 4; x++) o[x] = w == 0.f ? o[x] : fmaf(part[s][x], w, o[x]);
    }
    if (d < a.D) put_row(a, row, d, o, l);
}

// Many: one workgroup per row, the parts' states joined. The weights 2^(m_s - m) go to LDS, then 8 groups of 32
// threads, 4 features each, take every eighth part and add up in order.
__global__ __launch_bounds__(256) void k_attn_join(JoinArgs a) {
    __shared__ float w[kMostSplits], red[8];
    __shared__ __attribute__((aligned(16))) float part[8][128];
    const int tid = threadIdx.x, wave = tid >> 6;
    const int row = blockIdx.x;
    const f32x2* ml = (const f32x2*)(a.ws + (int64_t)a.splits * a.rows * a.D);
    if (ml[row][1] < 0.f) return;            // not a sequence's row
    float m = -INFINITY;
    for (int s = tid; s < a.splits; s += 256) m = fmaxf(m, ml[(int64_t)s * a.rows + row][0]);
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) m = fmaxf(m, __shfl_xor(m, i));
    if ((tid & 63) == 0) red[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float l = 0.f;
    for (int s = tid; s < a.splits; s += 256) {
        const f32x2 x = ml[(int64_t)s * a.rows + row];
        w[s] = x[1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(x[0] - m);
        l = fmaf(w[s], x[1], l);
    }
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) l += __shfl_xor(l, i);
    if ((tid & 63) == 0) red[4 + wave] = l;
    __syncthreads();
    l = red[4] + red[5] + red[6] + red[7];
    const int grp = tid >> 5, d = 4 * (tid & 31);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (d < a.D)
#pragma unroll 4
        for (int s = grp; s < a.splits; s += 8)
            if (w[s] != 0.f) o += *(const f32x4*)(a.ws + ((int64_t)s * a.rows + row) * a.D + d) * w[s];
    *(f32x4*)&part[grp][d] = o;
    __syncthreads();
    if (tid >= 32 || d >= a.D) return;
    for (int i = 1; i < 8; i++) o += *(const f32x4*)&part[i][d];
    const float v[4] = {o[0], o[1], o[2], o[3]};
    put_row(a, row, d, v, l);
}

}  // namespace

hipError_t launch_attn_pack(const PackArgs& p, hipStream_t s) {
    int64_t most = 0;
    for (int i = 0; i < p.n; i++) most = std::max(most, (int64_t)p.B * p.v[i].H * p.v[i].S * (p.D / 8));
    hipLaunchKernelGGL(k_attn_pack, dim3((unsigned)((most + 255) / 256), (unsigned)p.n), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_attn_join(const JoinArgs& a, hipStream_t s) {
    const dim3 waves((unsigned)((a.rows + 7) / 8));
    if (a.splits <= 2) hipLaunchKernelGGL(k_attn_join_few<2>, waves, dim3(256), 0, s, a);
    else if (a.splits <= 4) hipLaunchKernelGGL(k_attn_join_few<4>, waves, dim3(256), 0, s, a);
    else if (a.splits <= 8) hipLaunchKernelGGL(k_attn_join_few<8>, waves, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_attn_join, dim3((unsigned)a.rows), dim3(256), 0, s, a);
    return hipGetLastError();
}

// Two row tiles per wave (each operand read from LDS serves both) where they still give a workgroup per CU: 128
// features, 32 heads of 4097 tokens 332 against 372 us for one, a prefix of 1000 in 8191 capped 638 / 795. Up to 64
// features the LDS is no bound and the gain is small (unmasked 177 / 193 us), while rows that see unlike numbers of
// keys are better shared out in smaller pieces (nine documents 78 / 69, causal 105 / 107) and capped scores wait for
// the VALU anyway (276 / 270): one.
// Too few workgroups for two per CU: the keys in parts (512 x 12345, 256 workgroups: one part 248 us, two 199; one
// token over 8000 keys, 64 workgroups: 1 / 2 / 4 / 8 parts 253 / 136 / 78 / 56 us), of at least 4 chunks (257 tokens, 80
// workgroups of 5 chunks: 12 us whole, 19 in two parts).
MaskedPlan masked_plan(const MaskedAttnArgs& a) {
    const int64_t R = (int64_t)a.Sq * (a.H / a.Hkv), heads = (int64_t)a.Hkv * a.B, nch = (a.Sk + kMaskKeys - 1) / kMaskKeys;
    MaskedPlan p{1, 1, 0};
    const bool even = !a.causal && !a.docs && a.mod.cap2 == 0.f;
    if (heads * ((R + 127) / 128) >= 256 && (a.D > 64 || even)) p.qt = 2;
    const int64_t wgs = heads * ((R + 64 * p.qt - 1) / (64 * p.qt));
    if (wgs < 384) p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / wgs, nch / 4));
    if (p.splits > 1) p.ws_bytes = (size_t)p.splits * heads * R * (a.D + 2) * sizeof(float);
    return p;
}

hipError_t launch_attn_masked(const MaskedAttnArgs& a, const MaskedPlan& p, hipStream_t s) {
    const int dc = a.D / 16;
    const hipError_t e = dc <= 2 ? launch_masked_d<2>(a, p, s) : dc == 3 ? launch_masked_d<3>(a, p, s)
                       : dc == 4 ? launch_masked_d<4>(a, p, s) : launch_attn_masked_wide(a, p, s);
    if (e != hipSuccess || p.splits == 1) return e;
    JoinArgs j{};
    j.ws = a.ws; j.o = a.o; j.o16 = a.o16;
    for (int i = 0; i < 4; i++) j.ost[i] = a.ost[i];
    j.G = a.H / a.Hkv; j.Hkv = a.Hkv; j.D = a.D; j.splits = p.splits;
    j.vec_o = a.vec_o;
    j.R = a.Sq * j.G;
    j.rows = j.R * a.Hkv * a.B;
    return launch_attn_join(j, s);
}

}  // namespace mgh
