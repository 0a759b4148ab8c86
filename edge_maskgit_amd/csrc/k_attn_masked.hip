// k_attn_masked.hip — attention under causal, prefix and document masks with capped or sloped scores.
#include "k_attn_row.h"

namespace mgh {

namespace {

// q, k, v as they come, rounded to fp16
__device__ __forceinline__ float elem(const void* p, bool f16, int64_t e) {
    return f16 ? (float)((const _Float16*)p)[e] : (float)(_Float16)((const float*)p)[e];
}

struct MaskedSrc {
    const MaskedAttnArgs& a;
    int64_t kv;            // element offset of the sequence's and head's first row
    int64_t p;             // the row's position
    int prefix;
    const int32_t* docs;   // the sequence's ids, or null
    int doc;
    __device__ bool seen(int64_t j) const {
        return (!a.causal || j <= p || j < prefix) && (!docs || (docs[j] == doc && doc >= 0));
    }
    __device__ float dot(int64_t j, const float* qs) const {
        const int64_t e = kv + j * a.kvst[1];
        float s = 0.f;
        for (int d = 0; d < a.D; d++) s = fmaf(qs[d], elem(a.k, a.in16, e + d * a.kvst[0]), s);
        return s;
    }
    __device__ float value(int64_t j, int d) const { return elem(a.v, a.in16, kv + j * a.kvst[1] + d * a.kvst[0]); }
};

__global__ __launch_bounds__(256) void k_attn_masked(MaskedAttnArgs a) {
    __shared__ float qs[4][128], pl[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / (a.H / a.Hkv);
    const int64_t i = (int64_t)blockIdx.x * 4 + wave;
    if (i >= a.Sq) return;
    const int64_t p = (int64_t)a.Sk - a.Sq + i;
    const int64_t qe = b * a.qst[3] + h * a.qst[2] + i * a.qst[1];
    for (int d = lane; d < a.D; d += 64) qs[wave][d] = elem(a.q, a.in16, qe + d * a.qst[0]);
    __builtin_amdgcn_wave_barrier();
    MaskedSrc src{a, b * a.kvst[3] + hk * a.kvst[2], p, a.prefix ? a.prefix[b] : 0, a.docs ? a.docs + b * a.doc_stride : nullptr, -1};
    if (src.docs && p >= 0) src.doc = src.docs[p];
    const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    const RowState st = attn_row(src, a.mod, slope2, p, 0, a.Sk, a.D, qs[wave], pl[wave], lane);
    const int64_t oe = b * a.ost[3] + h * a.ost[2] + i * a.ost[1];
    for (int t = 0; t < 2; t++) {
        const int d = lane + 64 * t;
        if (d >= a.D) continue;
        const float o = st.l == 0.f ? 0.f : st.o[t] / st.l;
        if (a.o16) a.o16[oe + d * a.ost[0]] = (_Float16)o;
        else a.o[oe + d * a.ost[0]] = o;
    }
}

}  // namespace

hipError_t launch_attn_masked(const MaskedAttnArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(k_attn_masked, dim3((unsigned)((a.Sq + 3) / 4), (unsigned)a.H, (unsigned)a.B), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace mgh
