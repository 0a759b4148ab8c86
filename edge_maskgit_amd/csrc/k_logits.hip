// k_logits.hip — what is done to logits between the output head and the sampling (gfx950).
//
// Per row and token v with n occurrences in the row's history:
//   n > 0: l <- (l > 0 ? l / rep : l rep) - (freq n + pres);   l <- l + bias[v];   not allowed: -inf.
// fp32 arithmetic; fp16 logits are rounded once, when they are stored. One pass: a workgroup takes kChunk
// tokens of a row, counts the history's ids in its range in LDS (whole numbers: the order of the
// atomics changes nothing) and edits its logits. Every workgroup of a row reads the whole history, from
// L2: 4 bytes per id against the 8 bytes per token that it moves from and to memory. Bound by those 8 bytes: 64
// rows of 128001 fp32 logits, 4000 ids, shared bias and a mask per row 16.1 us (4.2 TB/s; chunks of 4096 tokens
// 16.4, of 8192 19.2), one row of 2025 3.4 us (4.2, 5.9).
#include "mgh_common.h"
#include "mgh_kernels.h"

namespace mgh {

namespace {

constexpr int kChunk = kLogitsChunk;

// T: the logits' type. VEC: rows of aligned 16-byte pieces, 4 tokens at a time. Buffer accesses, whose range
// is the row's chunk: no branch per token at the row's end. All of a thread's loads (ids of the history
// first, then its 16 tokens' logits, bias and mask words) are on their way while the counts are cleared; y may be
// x, so the compiler could move none of them before a store.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_logits(LogitsArgs a) {
    __shared__ __attribute__((aligned(16))) int n[kChunk];
    typedef T t4 __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    constexpr int U = kChunk / 1024, EB = sizeof(T);
    const int chunks = (a.V + kChunk - 1) / kChunk, tid = threadIdx.x;
    const int64_t r = blockIdx.x / chunks;
    const int v0 = (int)(blockIdx.x % chunks) * kChunk, nv = a.V - v0 < kChunk ? a.V - v0 : kChunk;
    auto range = [](const void* p, int bytes) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, bytes, 0x00020000); };
    const __amdgpu_buffer_rsrc_t rx = range((const T*)a.x + r * a.x_stride + v0, nv * EB);
    const __amdgpu_buffer_rsrc_t ry = range((T*)a.y + r * a.y_stride + v0, nv * EB);
    const __amdgpu_buffer_rsrc_t rb = range(a.bias + (a.bias ? r * a.bias_stride + v0 : 0), nv * 4);
    const __amdgpu_buffer_rsrc_t rm = range(a.allowed + (a.allowed ? r * a.allowed_stride + (v0 >> 5) : 0), (nv + 31) / 32 * 4);
    const bool counted = a.hist != nullptr;
    // token j of group u of this thread
    auto at = [&](int u, int j) { return VEC ? 1024 * u + 4 * tid + j : 1024 * u + 256 * j + tid; };
    constexpr int HU = 8;                // ids of the history asked for at once
    int len = 0, hv[HU];
    const int32_t* h = nullptr;
    if (counted) {
        h = a.hist + r * a.hist_stride;
        len = a.hist_len ? a.hist_len[r] : a.max_hist;
        len = len < 0 ? 0 : len > a.max_hist ? a.max_hist : len;
        const __amdgpu_buffer_rsrc_t rh = range(h, len < 256 * HU ? 4 * len : 1024 * HU);
#pragma unroll
        for (int k = 0; k < HU; k++) hv[k] = __builtin_amdgcn_raw_buffer_load_b32(rh, 1024 * k + 4 * tid, 0, 0);
    }
    T in[U][4];
    float add[U][4];
    uint32_t keep[U][4];                 // mask words, the token's bit lowest
#pragma unroll
    for (int u = 0; u < U; u++) {
        auto single = [&](int j) {
            if constexpr (EB == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(rx, EB * at(u, j), 0, 0));
            else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(rx, EB * at(u, j), 0, 0));
        };
        if (VEC && at(u, 3) < nv) {
            t4 v;
            if constexpr (EB == 4) v = __builtin_bit_cast(t4, __builtin_amdgcn_raw_buffer_load_b128(rx, EB * at(u, 0), 0, 0));
            else v = __builtin_bit_cast(t4, __builtin_amdgcn_raw_buffer_load_b64(rx, EB * at(u, 0), 0, 0));
#pragma unroll
            for (int j = 0; j < 4; j++) in[u][j] = v[j];
        } else {                         // (a row of aligned pieces may end inside one)
#pragma unroll
            for (int j = 0; j < 4; j++) in[u][j] = single(j);
        }
        if (a.bias)
#pragma unroll
            for (int j = 0; j < 4; j++) add[u][j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rb, 4 * at(u, j), 0, 0));
        if (a.allowed)
#pragma unroll
            for (int j = 0; j < (VEC ? 1 : 4); j++) keep[u][j] = __builtin_amdgcn_raw_buffer_load_b32(rm, at(u, j) >> 5 << 2, 0, 0);
    }
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (counted) {
        if (a.rep) rep = a.rep[r];
        if (a.freq) freq = a.freq[r];
        if (a.pres) pres = a.pres[r];
        for (int i = 4 * tid; i < kChunk; i += 1024) *(i32x4*)&n[i] = i32x4{0, 0, 0, 0};
        stage_sync<63>();                // (loads stay on their way)
        auto count = [&](int v) {
            const uint32_t id = (uint32_t)v - (uint32_t)v0;           // ids outside the vocabulary count nowhere
            if (id < (uint32_t)nv) atomicAdd(&n[id], 1);
        };
#pragma unroll
        for (int k = 0; k < HU; k++)
            if (256 * k + tid < len) count(hv[k]);
#pragma unroll 4
        for (int i = 256 * HU + tid; i < len; i += 256) count(h[i]);
        stage_sync<63>();
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        t4 o;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float l = (float)in[u][j];
            const int c = counted ? n[at(u, j)] : 0;
            if (c) {
                l = l > 0.f ? l / rep : l * rep;
                l -= fmaf(freq, (float)c, pres);
            }
            if (a.bias) l += add[u][j];
            if (a.allowed && !(keep[u][VEC ? 0 : j] >> (at(u, j) & 31) & 1)) l = -INFINITY;
            o[j] = (T)l;
        }
        if (VEC && at(u, 3) < nv) {
            if constexpr (EB == 4) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), ry, EB * at(u, 0), 0, 0);
            else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, o), ry, EB * at(u, 0), 0, 0);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const T v = o[j];        // (a bit cast of the vector's element itself takes element 0)
                if constexpr (EB == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), ry, EB * at(u, j), 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), ry, EB * at(u, j), 0, 0);
            }
        }
    }
}

}  // namespace

hipError_t launch_logits_process(const LogitsArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.rows * ((a.V + kChunk - 1) / kChunk)));
    const int64_t apart = a.rows > 1 ? a.x_stride | a.y_stride : 0;
    const bool vec = apart % 4 == 0 && ((uintptr_t)a.x | (uintptr_t)a.y) % (a.f16 ? 8 : 16) == 0;
    if (a.f16 && vec) hipLaunchKernelGGL((k_logits<_Float16, true>), grid, dim3(256), 0, s, a);
    else if (a.f16) hipLaunchKernelGGL((k_logits<_Float16, false>), grid, dim3(256), 0, s, a);
    else if (vec) hipLaunchKernelGGL((k_logits<float, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_logits<float, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace mgh
