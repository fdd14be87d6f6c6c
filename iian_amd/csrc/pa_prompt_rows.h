// pa_prompt_rows.h - whole-prompt attention, a wave per (token, head): any head
// size up to 1024, any alignment (iian_pa_prompt_attention where the
// matrix-core kernels of pa_prompt.hip do not apply; compiled in
// pa_general.hip).
//
// The wave keeps its query row in LDS as fp32 and walks its prompt's visible
// tokens 64 at a time: lane l dots token l's K row with it, the softmax is
// online over the wave (a reference maximum and a sum), and the lanes then take
// output values l, l + 64, ... over the 64 tokens' V rows, whose probabilities
// come from LDS.  All in fp32.  Bound by its loads: K rows a lane each, V rows
// coalesced.  (One 8192-token prompt at H32/Hkv8/D128, which the matrix cores take
// 0.53 ms for, took it 269 ms: kept for what they do not take.)
#pragma once

#include "pa_common.h"
#include "pa_launch.h"

#include <algorithm>

namespace iian_pa {

constexpr int kRowsWaves = 4;
constexpr int kRowsMaxDim = 1024;
constexpr int kRowsMaxWgs = 1 << 23;   // of 256 threads: a launch holds below 2^32 threads

// The tokens of its prompt (length L) that token i sees: [lo, hi).
__device__ __forceinline__ int2 prompt_window(const PromptParams &p, int t, int i, int L) {
    int hi = p.row_end ? min(max(p.row_end[t], 0), L) : p.causal ? i + 1 : L;
    int lo = p.n_swa > 0 ? max(0, i - p.n_swa + 1) : 0;
    return make_int2(min(lo, hi), hi);
}

// Prompt of token t and its range, by a binary search over query_start_loc
// (clamped into [0, T]); false when t is in none.
__device__ __forceinline__ bool prompt_of(const PromptParams &p, int t, int &s, int &q0, int &q1) {
    int lo = 0, hi = p.S;   // the last prompt that starts at or before t
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (p.qsl[m] <= t) lo = m;
        else hi = m;
    }
    s = lo;
    q0 = min(max(p.qsl[s], 0), p.T);
    q1 = min(max(p.qsl[s + 1], q0), p.T);
    return t >= q0 && t < q1;
}

template <typename T, int NO>
__global__ __launch_bounds__(kRowsWaves * 64) void pa_prompt_rows_kernel(PromptParams p) {
    __shared__ float qs[kRowsWaves][kRowsMaxDim], ps[kRowsWaves][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float cs = p.softcap > 0.f ? p.scale / p.softcap : p.scale * kLog2e;
    // (no workgroup barrier in this kernel)
    for (int64_t unit = (int64_t) blockIdx.x * kRowsWaves + wave; unit < (int64_t) p.T * p.H;
         unit += (int64_t) gridDim.x * kRowsWaves) {
        const int t = (int) (unit / p.H), h = (int) (unit - (int64_t) t * p.H), hk = h / p.gqa;
        int s, q0, q1;
        if (!prompt_of(p, t, s, q0, q1)) continue;
        if (q1 - q0 > p.max_q && t == q0 && h == 0 && lane == 0 && p.err) atomicOr(p.err, 4);
        const int2 w = prompt_window(p, t, t - q0, q1 - q0);
        const T *q = (const T *) p.q + t * p.q_stride + (int64_t) h * p.D;
        for (int e = lane; e < p.D; e += 64) qs[wave][e] = (float) q[e];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        float acc[NO], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int o = 0; o < NO; o++) acc[o] = 0.f;
        for (int c = w.x; c < w.y; c += 64) {
            const int j = c + lane;
            float x = -INFINITY;
            if (j < w.y) {
                const T *k = (const T *) p.k + (q0 + j) * p.k_stride + (int64_t) hk * p.D;
                float d = 0.f;
                for (int e = 0; e < p.D; e++) d += qs[wave][e] * (float) k[e];
                x = d * cs;
                if (p.softcap > 0.f) x = tanhf(x) * (p.softcap * kLog2e);
            }
            float mx = x;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
            const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
            const float alpha = exp2f(m - ref), pr = j < w.y ? exp2f(x - ref) : 0.f;
            m = mn;
            l = l * alpha + pr;
            ps[wave][lane] = pr;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int o = 0; o < NO; o++) acc[o] *= alpha;
            const int n = min(64, w.y - c);
            for (int y = 0; y < n; y++) {
                const T *v = (const T *) p.v + (q0 + c + y) * p.v_stride + (int64_t) hk * p.Dv;
                const float pv = ps[wave][y];
#pragma unroll
                for (int o = 0; o < NO; o++)
                    if (lane + 64 * o < p.Dv) acc[o] += pv * (float) v[lane + 64 * o];
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
        const float inv = l == 0.f ? 0.f : 1.f / l;   // no cell seen, or none with a weight
        T *out = (T *) p.out + t * p.o_stride + (int64_t) h * p.Dv;
#pragma unroll
        for (int o = 0; o < NO; o++)
            if (lane + 64 * o < p.Dv) out[lane + 64 * o] = (T) (acc[o] * inv);
    }
}

template <typename T>
static hipError_t launch_prompt_rows_t(const PromptParams &p, hipStream_t stream) {
    const int64_t wgs = std::min<int64_t>(((int64_t) p.T * p.H + kRowsWaves - 1) / kRowsWaves, kRowsMaxWgs);
    const dim3 grid((unsigned) wgs), wg(kRowsWaves * 64);
    if (p.Dv <= 256) hipLaunchKernelGGL((pa_prompt_rows_kernel<T, 4>), grid, wg, 0, stream, p);
    else hipLaunchKernelGGL((pa_prompt_rows_kernel<T, 16>), grid, wg, 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_prompt_rows(const PromptParams &p, int type, hipStream_t stream) {
    switch (type) {
        case 0: return launch_prompt_rows_t<float>(p, stream);
        case 1: return launch_prompt_rows_t<_Float16>(p, stream);
        case 30: return launch_prompt_rows_t<__bf16>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace iian_pa
