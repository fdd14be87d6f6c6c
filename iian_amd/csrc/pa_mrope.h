// pa_mrope.h - multi-axis RoPE with the heads' RMS norm, fused into the
// slot-mapped KV write (iian_pa_mrope_kv_write; compiled in pa_rope.hip).
//
// Pair j of a head turns by pos[axis[j]][t] * freqs[j].  The angle is reduced
// exactly, in turns: the fraction of a turn per position is a 64-bit fixed-point
// number, and its product with the position, modulo 2^64, is the fraction of the
// angle with no more than |pos| * 2^-54 turns of error (the frequency's own 53
// bits), at position 10^6 as at 1.  What is left is at most an eighth of a turn
// either side of a quadrant, where Taylor sums of degree 8 and 9 reach 3e-8.
//
// The vector form.  A lane moves E elements of each half of a head row (E = 8 of
// a 16-bit row, 4 of an f32 one: one 16-byte access), lpr lanes share a row and
// a wave takes 64/lpr rows per step with kMropeU steps in flight.  A wave has one
// token's rows, or a share of them when the step has few tokens, and its own
// (cos, sin) table in LDS, one or two pairs per lane: nothing waits on another
// wave.  The first rows are requested before the table is computed.
// HBM-bound for prompts (16,384 f16 tokens of H16/Hkv8/D256 112.6 us in the kernel
// trace, 4.8 TB/s of the 5.1 that a copy reaches), latency-bound for decode steps (64 tokens of
// H32/Hkv8/D128 4.0 us).
//
// The row form takes what is left (odd head sizes, partial rotation, unaligned
// rows, Dv != D, Q8_0 blocks that straddle the halves): a wave per head row,
// staged in LDS as fp32.
#pragma once

#include "pa_common.h"
#include "pa_launch.h"

#include <algorithm>

namespace iian_pa {

constexpr int kMropeWaves = 4;
constexpr int kMropeU = 3;              // steps in flight
constexpr int kMropeVecMaxDim = 512;    // largest head of the vector form: 256 pairs in a wave's table
constexpr int kMropeMaxDim = 1024;      // largest head the row form stages
constexpr int kMropeMaxWgs = 1 << 23;   // workgroups of 256 threads: a launch holds below 2^32 threads

typedef __bf16 bf16_t;

__device__ __forceinline__ float mrope_f32(float x) { return x; }
__device__ __forceinline__ float mrope_f32(_Float16 x) { return (float) x; }
__device__ __forceinline__ float mrope_f32(bf16_t x) { return (float) x; }

// (cos, sin) of pos * freq, times mscale.  (The fraction is of |freq|: that of a tiny negative one would round to a whole turn.)
__device__ __forceinline__ float2 mrope_cs(double freq, int pos, float mscale) {
    const double turns = fabs(freq) * 0.15915494309189533576888;   // 1 / (2 pi)
    const double fr = turns - floor(turns);
    const double up = fr * 4294967296.0, hi = floor(up);
    const uint64_t step = ((uint64_t) (uint32_t) hi << 32) | (uint32_t) ((up - hi) * 4294967296.0);
    const uint64_t u = step * (uint64_t) (freq < 0 ? -(int64_t) pos : (int64_t) pos);
    const uint32_t quad = (uint32_t) ((u + (1ull << 61)) >> 62);
    const int32_t rest = (int32_t) ((u - ((uint64_t) quad << 62)) >> 32);   // [-2^29, 2^29) of 2^32 a turn
    const float x = (float) rest * 1.46291807926715968e-9f;                 // 2 pi 2^-32: [-pi/4, pi/4)
    const float y = x * x;
    const float c = 1.f + y * (-0.5f + y * (4.16666667e-2f + y * (-1.38888889e-3f + y * 2.48015873e-5f)));
    const float s = x + x * y * (-1.66666667e-1f + y * (8.33333333e-3f + y * (-1.98412698e-4f + y * 2.75573192e-6f)));
    const bool odd = quad & 1;
    float cq = odd ? s : c, sq = odd ? c : s;
    if ((quad + 1) & 2) cq = -cq;   // quadrants 1 and 2
    if (quad & 2) sq = -sq;         // quadrants 2 and 3
    return make_float2(cq * mscale, sq * mscale);
}

__device__ __forceinline__ int mrope_pos(const MropeParams &p, int j, int t) {
    const int a = min(max(p.axis[j], 0), p.n_axes - 1);
    return p.pos[(int64_t) a * p.T + t];
}

// E values of one head row, 16 bytes.
template <typename T, int E>
struct __attribute__((aligned(16))) MropeVec {
    T v[E];
};

// Values x[0..E) of elements e .. e+E-1 of head h into pool row `slot`.  Q8_0: the
// E-element pieces of a 32-value block are in neighbouring lanes, all of them here.
template <int E>
__device__ __forceinline__ void mrope_store_pool(int type, void *pool, int64_t slot, int Hkv, int h, int D, int e,
                                                 const float *x) {
    const int64_t base = (slot * Hkv + h) * (int64_t) D + e;
    if (type == 1) {
        typedef uint32_t __attribute__((ext_vector_type(E / 2))) vec;
        vec w;
#pragma unroll
        for (int i = 0; i < E / 2; i++) w[i] = pack_f16x2(x[2 * i], x[2 * i + 1]);
        *(vec *) ((_Float16 *) pool + base) = w;
    } else if (type == 0) {
#pragma unroll
        for (int i = 0; i < E; i += 4)
            *(float4 *) ((float *) pool + base + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    } else {
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < E; i++) amax = fmaxf(amax, fabsf(x[i]));
#pragma unroll
        for (int o = 1; o < 32 / E; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
        const float id = amax != 0.f ? 127.f / amax : 0.f;
        uint16_t *blk = (uint16_t *) ((uint8_t *) pool + (slot * Hkv + h) * (int64_t) (D / 32 * 34) + 34 * (e >> 5));
        uint16_t *dst = blk + 1 + ((e & 31) >> 1);
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const int a = min(127, max(-128, (int) __builtin_rintf(x[i] * id))) & 0xff;
            const int b = min(127, max(-128, (int) __builtin_rintf(x[i + 1] * id))) & 0xff;
            dst[i / 2] = (uint16_t) (a | (b << 8));
        }
        if ((e & 31) == 0) blk[0] = __builtin_bit_cast(uint16_t, (_Float16) (amax / 127.f));
    }
}

// Wave u of the launch: token u / shares, rows [share * rows_per, +rows_per) of
// the token's nq q heads, Hkv K heads and (with pools) Hkv V heads.
template <typename T, int E, bool NORM>
__global__ __launch_bounds__(kMropeWaves * 64, 4) void pa_mrope_vec_kernel(MropeParams p, int shares, int rows_per,
                                                                         int lpr_log2) {
    __shared__ __attribute__((aligned(16))) float2 tab[kMropeWaves][kMropeVecMaxDim / 2];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t unit = (int64_t) blockIdx.x * kMropeWaves + wave;
    const int64_t t64 = unit / shares;
    if (t64 >= p.T) return;   // (no workgroup barrier in this kernel)
    const int t = (int) t64, share = (int) (unit - t64 * shares);
    const int D = p.D, half = D >> 1, nq = p.q ? p.H : 0;
    const bool pools = p.k_pool != nullptr;
    const int rpt = nq + p.Hkv * (pools ? 2 : 1);
    const int r0 = share * rows_per, r1 = min(rpt, r0 + rows_per);
    const int i = lane & ((1 << lpr_log2) - 1), sub = lane >> lpr_log2, rps = 64 >> lpr_log2;
    const bool act = E * i < half;
    const bool ne = p.mode != 0;
    MropeVec<T, E> xa[kMropeU], xb[kMropeU];
    auto load = [&](int rb) {
#pragma unroll
        for (int u = 0; u < kMropeU; u++) {
            const int r = rb + u * rps + sub;
            if (r < r1 && act) {
                const T *src = r < nq           ? (const T *) p.q + t * p.q_stride + (int64_t) r * D
                               : r < nq + p.Hkv ? (const T *) p.k + t * p.k_stride + (int64_t) (r - nq) * D
                                                : (const T *) p.v + t * p.v_stride + (int64_t) (r - nq - p.Hkv) * D;
                xa[u] = *(const MropeVec<T, E> *) (src + E * i);
                xb[u] = *(const MropeVec<T, E> *) (src + half + E * i);
            }
        }
    };
    load(r0);
    int64_t slot = -1;
    if (pools) {
        slot = p.slots[t];
        if (slot < 0 || slot >= p.n_cells) {
            if (share == 0 && lane == 0 && p.err) atomicOr(p.err, 1);
            slot = -1;
        }
    }
    float2 *cs = tab[wave];
    if (r0 < nq + p.Hkv) {   // wave-uniform: some row rotates
        for (int j = lane; j < half; j += 64) cs[j] = mrope_cs(p.freqs[j], mrope_pos(p, j, t), p.mscale);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    for (int rb = r0; rb < r1; rb += kMropeU * rps) {
        if (rb != r0) load(rb);
#pragma unroll
        for (int u = 0; u < kMropeU; u++) {
            const int r = rb + u * rps + sub;
            const bool live = r < r1 && act, turns = r < nq + p.Hkv;
            float a[E], b[E];
#pragma unroll
            for (int k = 0; k < E; k++) {
                a[k] = live ? mrope_f32(xa[u].v[k]) : 0.f;
                b[k] = live ? mrope_f32(xb[u].v[k]) : 0.f;
            }
            if constexpr (NORM) {
                // (every lane takes part: the row's lanes are neighbours)
                float ss = 0.f;
#pragma unroll
                for (int k = 0; k < E; k++) ss += a[k] * a[k] + b[k] * b[k];
                for (int o = 1; o < 1 << lpr_log2; o <<= 1) ss += __shfl_xor(ss, o);
                const float *w = r < nq ? p.q_norm : p.k_norm;
                if (live && turns && w) {
                    const float inv = 1.f / sqrtf(ss / (float) D + p.eps);
#pragma unroll
                    for (int k = 0; k < E; k += 4) {
                        const float4 wa = *(const float4 *) (w + E * i + k), wb = *(const float4 *) (w + half + E * i + k);
                        a[k] *= inv * wa.x;
                        a[k + 1] *= inv * wa.y;
                        a[k + 2] *= inv * wa.z;
                        a[k + 3] *= inv * wa.w;
                        b[k] *= inv * wb.x;
                        b[k + 1] *= inv * wb.y;
                        b[k + 2] *= inv * wb.z;
                        b[k + 3] *= inv * wb.w;
                    }
                }
            }
            if (!live) continue;
            if (turns) {
                if (ne) {   // pairs (e, e + half)
#pragma unroll
                    for (int k = 0; k < E; k += 2) {
                        const float4 c = *(const float4 *) &cs[E * i + k];
                        const float a0 = a[k], a1 = a[k + 1], b0 = b[k], b1 = b[k + 1];
                        a[k] = a0 * c.x - b0 * c.y;
                        b[k] = a0 * c.y + b0 * c.x;
                        a[k + 1] = a1 * c.z - b1 * c.w;
                        b[k + 1] = a1 * c.w + b1 * c.z;
                    }
                } else {    // pairs (2e, 2e + 1)
#pragma unroll
                    for (int k = 0; k < E; k += 4) {
                        const float4 ca = *(const float4 *) &cs[(E * i + k) / 2];
                        const float4 cb = *(const float4 *) &cs[(half + E * i + k) / 2];
                        const float a0 = a[k], a1 = a[k + 1], a2 = a[k + 2], a3 = a[k + 3];
                        const float b0 = b[k], b1 = b[k + 1], b2 = b[k + 2], b3 = b[k + 3];
                        a[k] = a0 * ca.x - a1 * ca.y;
                        a[k + 1] = a0 * ca.y + a1 * ca.x;
                        a[k + 2] = a2 * ca.z - a3 * ca.w;
                        a[k + 3] = a2 * ca.w + a3 * ca.z;
                        b[k] = b0 * cb.x - b1 * cb.y;
                        b[k + 1] = b0 * cb.y + b1 * cb.x;
                        b[k + 2] = b2 * cb.z - b3 * cb.w;
                        b[k + 3] = b2 * cb.w + b3 * cb.z;
                    }
                }
                T *dst = r < nq       ? (T *) p.q_out + t * p.qo_stride + (int64_t) r * D
                         : p.k_out != nullptr ? (T *) p.k_out + t * p.ko_stride + (int64_t) (r - nq) * D
                                              : nullptr;
                if (dst) {
                    MropeVec<T, E> ya, yb;
#pragma unroll
                    for (int k = 0; k < E; k++) {
                        ya.v[k] = (T) a[k];
                        yb.v[k] = (T) b[k];
                    }
                    *(MropeVec<T, E> *) (dst + E * i) = ya;
                    *(MropeVec<T, E> *) (dst + half + E * i) = yb;
                }
            }
            if (r >= nq && slot >= 0) {
                const int h = turns ? r - nq : r - nq - p.Hkv;
                const int ty = turns ? p.type_k : p.type_v;
                void *pool = turns ? p.k_pool : p.v_pool;
                mrope_store_pool<E>(ty, pool, slot, p.Hkv, h, D, E * i, a);
                mrope_store_pool<E>(ty, pool, slot, p.Hkv, h, D, half + E * i, b);
            }
        }
    }
}

// A wave per head row, any head size, pairing and alignment.
template <typename T>
__global__ __launch_bounds__(kMropeWaves * 64) void pa_mrope_row_kernel(MropeParams p) {
    __shared__ __attribute__((aligned(16))) float stage[kMropeWaves][kMropeMaxDim];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int nq = p.q ? p.H : 0;
    const bool pools = p.k_pool != nullptr;
    const int64_t rpt = nq + (int64_t) p.Hkv * (pools ? 2 : 1);
    // (no workgroup barrier in this kernel)
    for (int64_t unit = (int64_t) blockIdx.x * kMropeWaves + wave; unit < p.T * rpt;
         unit += (int64_t) gridDim.x * kMropeWaves) {
        const int64_t t = unit / rpt;
        const int r = (int) (unit - t * rpt);
        const int kind = r < nq ? 0 : r < nq + p.Hkv ? 1 : 2;   // q, K, V
        const int h = kind == 0 ? r : kind == 1 ? r - nq : r - nq - p.Hkv;
        const int n = kind == 2 ? p.Dv : p.D, half = p.n_dims >> 1;
        const T *src = kind == 0   ? (const T *) p.q + t * p.q_stride + (int64_t) h * p.D
                       : kind == 1 ? (const T *) p.k + t * p.k_stride + (int64_t) h * p.D
                                   : (const T *) p.v + t * p.v_stride + (int64_t) h * p.Dv;
        int64_t slot = -1;
        if (pools) {
            slot = p.slots[t];
            if (slot < 0 || slot >= p.n_cells) {
                if (r == 0 && lane == 0 && p.err) atomicOr(p.err, 1);
                slot = -1;
            }
        }
        float *x = stage[wave];
        const float *w = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
        float ss = 0.f;
        for (int e = lane; e < n; e += 64) {
            const float v = mrope_f32(src[e]);
            x[e] = v;
            ss += v * v;
        }
        if (w) {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) ss += __shfl_xor(ss, o);
            const float inv = 1.f / sqrtf(ss / (float) n + p.eps);
            for (int e = lane; e < n; e += 64) x[e] *= inv * w[e];
        }
        wave_lds_sync();
        if (kind != 2)
            for (int j = lane; j < half; j += 64) {
                const int e0 = p.mode ? j : 2 * j, e1 = p.mode ? j + half : 2 * j + 1;
                const float2 c = mrope_cs(p.freqs[j], mrope_pos(p, j, (int) t), p.mscale);
                const float x0 = x[e0], x1 = x[e1];
                x[e0] = x0 * c.x - x1 * c.y;
                x[e1] = x0 * c.y + x1 * c.x;
            }
        wave_lds_sync();
        T *dst = kind == 0   ? (T *) p.q_out + t * p.qo_stride + (int64_t) h * p.D
                 : kind == 1 && p.k_out ? (T *) p.k_out + t * p.ko_stride + (int64_t) h * p.D
                                        : nullptr;
        if (dst)
            for (int e = lane; e < n; e += 64) dst[e] = (T) x[e];
        const int ty = kind == 1 ? p.type_k : p.type_v;
        void *pool = kind == 1 ? p.k_pool : p.v_pool;
        const int64_t base = (slot * p.Hkv + h) * (int64_t) n;
        if (kind == 0 || slot < 0) {
        } else if (ty == 0) {
            for (int e = lane; e < n; e += 64) ((float *) pool)[base + e] = x[e];
        } else if (ty == 1) {
            for (int e = lane; e < n; e += 64) ((_Float16 *) pool)[base + e] = (_Float16) x[e];
        } else {
            rope_store_q8_0(x, n, (uint8_t *) pool + (slot * p.Hkv + h) * (int64_t) (n / 32 * 34), lane);
        }
        wave_lds_sync();   // the slice is rewritten by the wave's next row
    }
}

// The vector form: whole heads of one size rotated, rows, weights and pools in
// aligned pieces of E elements that do not straddle the halves.
static bool mrope_vec_ok(const MropeParams &p, int esize, int E) {
    const bool pools = p.k_pool != nullptr;
    if (p.T > kMropeMaxWgs || p.n_dims != p.D || p.D % (2 * E) || p.D > kMropeVecMaxDim || (pools && p.Dv != p.D)) return false;
    if (pools && (p.type_k == 8 || p.type_v == 8) && p.D % 64) return false;
    uintptr_t al = (uintptr_t) p.q | (uintptr_t) p.k | (uintptr_t) p.q_out | (uintptr_t) p.k_out |
                   (uintptr_t) p.q_norm | (uintptr_t) p.k_norm;
    int64_t st = p.k_stride | (p.q ? p.q_stride | p.qo_stride : 0) | (p.k_out ? p.ko_stride : 0);
    if (pools) {
        al |= (uintptr_t) p.v | (p.type_k == 8 ? 0 : (uintptr_t) p.k_pool) | (p.type_v == 8 ? 0 : (uintptr_t) p.v_pool);
        st |= p.v_stride;
    }
    return al % 16 == 0 && (st * esize) % 16 == 0;
}

template <typename T, int E>
static hipError_t launch_mrope_vec(const MropeParams &p, hipStream_t stream) {
    int lpr_log2 = 0;
    while ((2 * E << lpr_log2) < p.D) lpr_log2++;
    const int64_t rpt = (p.q ? p.H : 0) + (int64_t) p.Hkv * (p.k_pool ? 2 : 1), rps = 64 >> lpr_log2;
    // A wave has a whole token when the step has 4096 of them (4 per SIMD), and
    // else a share, down to one step of rows.  (1903 tokens of 48 bf16 rows of 128
    // 12.9 us, 14.1 at 8192, 14.0 at 2048; 512 f32 tokens 6.8, 7.8 and 7.4.)
    const int64_t steps = (rpt + rps - 1) / rps, want = std::max<int64_t>(1, 4096 / p.T);
    const int64_t per = (steps + std::min(steps, want) - 1) / std::min(steps, want), shares = (steps + per - 1) / per;
    const int64_t wgs = (p.T * shares + kMropeWaves - 1) / kMropeWaves;
    if (rpt > INT32_MAX / 2 || wgs > kMropeMaxWgs) return hipErrorInvalidValue;
    if (p.q_norm || p.k_norm)
        hipLaunchKernelGGL((pa_mrope_vec_kernel<T, E, true>), dim3((unsigned) wgs), dim3(kMropeWaves * 64), 0, stream, p,
                           (int) shares, (int) (per * rps), lpr_log2);
    else
        hipLaunchKernelGGL((pa_mrope_vec_kernel<T, E, false>), dim3((unsigned) wgs), dim3(kMropeWaves * 64), 0, stream,
                           p, (int) shares, (int) (per * rps), lpr_log2);
    return hipGetLastError();
}

template <typename T>
static hipError_t launch_mrope_t(const MropeParams &p, hipStream_t stream) {
    if (mrope_vec_ok(p, sizeof(T), 16 / sizeof(T))) return launch_mrope_vec<T, 16 / sizeof(T)>(p, stream);
    const int64_t rpt = (p.q ? p.H : 0) + (int64_t) p.Hkv * (p.k_pool ? 2 : 1);
    if (rpt > INT32_MAX / 2) return hipErrorInvalidValue;
    const int64_t wgs = std::min<int64_t>((p.T * rpt + kMropeWaves - 1) / kMropeWaves, kMropeMaxWgs);
    hipLaunchKernelGGL((pa_mrope_row_kernel<T>), dim3((unsigned) wgs), dim3(kMropeWaves * 64), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_mrope_kv_write(const MropeParams &p, hipStream_t stream) {
    switch (p.type) {
        case 0: return launch_mrope_t<float>(p, stream);
        case 1: return launch_mrope_t<_Float16>(p, stream);
        case 30: return launch_mrope_t<bf16_t>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace iian_pa
