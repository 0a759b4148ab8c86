// k_logits.hip — what is done to logits between the output head and the sampling (gfx950).
//
// Per row and token v with n occurrences in the row's history:
//   n > 0: l <- (l > 0 ? l / rep : l rep) - (freq n + pres);   l <- l + bias[v];   not allowed: -inf.
// fp32 arithmetic; fp16 logits are rounded once, when they are stored. One pass: a workgroup takes kChunk
// tokens of a row, counts the history's ids in its range in LDS (whole numbers: the order of the
// atomics changes nothing) and edits its logits. Every workgroup of a row reads the whole history, from
// L2: 4 bytes per id against the 8 bytes per token that it moves from and to memory.
#include "mgh_common.h"
#include "mgh_kernels.h"

namespace mgh {

namespace {

constexpr int kChunk = 4096;

template <bool F16>
__global__ __launch_bounds__(256) void k_logits(LogitsArgs a) {
    __shared__ int n[kChunk];
    const int chunks = (a.V + kChunk - 1) / kChunk;
    const int64_t r = blockIdx.x / chunks;
    const int v0 = (int)(blockIdx.x % chunks) * kChunk, nv = a.V - v0 < kChunk ? a.V - v0 : kChunk;
    const bool counted = a.hist != nullptr;
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (counted) {
        if (a.rep) rep = a.rep[r];
        if (a.freq) freq = a.freq[r];
        if (a.pres) pres = a.pres[r];
        for (int i = threadIdx.x; i < nv; i += 256) n[i] = 0;
        __syncthreads();
        int len = a.hist_len ? a.hist_len[r] : a.max_hist;
        len = len < 0 ? 0 : len > a.max_hist ? a.max_hist : len;
        const int32_t* h = a.hist + r * a.hist_stride;
        for (int i = threadIdx.x; i < len; i += 256) {
            const uint32_t at = (uint32_t)h[i] - (uint32_t)v0;        // ids outside the vocabulary count nowhere
            if (at < (uint32_t)nv) atomicAdd(&n[at], 1);
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < nv; i += 256) {
        const int v = v0 + i;
        float l = F16 ? (float)((const _Float16*)a.x)[r * a.x_stride + v] : ((const float*)a.x)[r * a.x_stride + v];
        if (counted && n[i]) {
            l = l > 0.f ? l / rep : l * rep;
            l -= fmaf(freq, (float)n[i], pres);
        }
        if (a.bias) l += a.bias[r * a.bias_stride + v];
        if (a.allowed && !(a.allowed[r * a.allowed_stride + (v >> 5)] >> (v & 31) & 1)) l = -INFINITY;
        if (F16) ((_Float16*)a.y)[r * a.y_stride + v] = (_Float16)l;
        else ((float*)a.y)[r * a.y_stride + v] = l;
    }
}

}  // namespace

hipError_t launch_logits_process(const LogitsArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.rows * ((a.V + kChunk - 1) / kChunk)));
    if (a.f16) hipLaunchKernelGGL(k_logits<true>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_logits<false>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace mgh
