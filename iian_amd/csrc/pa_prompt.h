// pa_prompt.h - whole-prompt attention on the matrix cores (iian_pa_prompt_attention):
// packed prompts, grouped heads, head sizes up to 256; F16, BF16 and F32 rows
// (pa_prompt.hip, pa_prompt_bf16.hip, pa_prompt_f32.hip hold one type each).
//
// A workgroup of 4 waves owns 128 rows r = i*gqa + g (token i, head g of the
// group) of one (prompt, kv head), 32 per wave, and walks the tokens that any of
// them sees in tiles of KT, staged in LDS (two buffers, one barrier per tile: the
// next tile's rows are requested before the tile is computed and written behind
// it).  One pass with a running maximum and sum per row:
//
//   S^T = K Q^T     v_mfma_f32_32x32x16: K rows are the A operand as they lie in
//                   LDS, Q^T stays in registers.  Lane l then holds, of row l%32,
//                   the scores of tokens 8(r/4) + 4(l/32) + r%4: a row is two lanes
//   softmax         exp2 domain; the reference maximum follows only when a tile
//                   passes it by 2^8, so the accumulators are seldom rescaled
//   O^T += V^T P^T  P^T is the S^T registers, rounded to the rows' type; V^T comes
//                   through the transpose read ds_read_b64_tr_b16.  O^T keeps a row
//                   in its lane: rescaling and the final division stay there
//
// F32 rows enter as pairs of f16 terms (hi + lo, 22 bits; three products, the one
// of two lo terms left out): v_mfma_f32_32x32x16_f16 three times does the work of
// the fp32 form at five times its rate.  So that f16's exponents suffice for any
// fp32 value, each row of Q, K and V is scaled by a power of two to a largest value
// in [2^14, 2^15): Q's goes into the row's factor, K's into its token's score, V's
// into its token's probability (kept below f16's range by a reference exponent
// per row, as the maximum is).
//
// Masks are evaluated in tiles that some row of the wave does not see whole.  A
// value that a row does not see has weight zero there, and zero times an
// infinity or NaN must not reach the row: in tiles that some row of the workgroup
// does not see whole, V's non-finite values are left out of the tile, and the rows
// that do see them add them afterwards (fix_v).
#pragma once

#include "pa_common.h"
#include "pa_launch.h"
#include "pa_mfma.h"

#include <algorithm>
#include <type_traits>

namespace iian_pa {

constexpr int kPromptWaves = 4;
constexpr int kPromptThreads = kPromptWaves * 64;
constexpr int kPromptRows = kPromptWaves * 32;   // rows per workgroup

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <int TY>
struct PromptType;   // 1 F16, 30 BF16, 0 F32
template <>
struct PromptType<1> {
    typedef _Float16 T;
};
template <>
struct PromptType<30> {
    typedef __bf16 T;
};
template <>
struct PromptType<0> {
    typedef float T;
};

// TY: rows' type; DK: head size rounded up to 16 dims, DV: to 32.
//
// LDS tiles.  Rows are unpadded, so that tiles of 16-bit rows can be loaded
// straight into LDS (16 consecutive bytes per lane), and the 16-byte pieces of
// row r are permuted by an exclusive or with swz(r) instead: 16 rows read at one
// piece, as QK^T does, and the 4 rows x 64 bytes of a transpose read each fill
// the 64 banks.
template <int TY, int DK, int DV>
struct PromptShape {
    static constexpr int NP = TY == 0 ? 2 : 1;                 // 16-bit terms per value
    static constexpr int KT = TY == 0 || DK > 128 ? 32 : 64;   // tokens per tile
    static constexpr int NH = KT / 32, KS = DK / 16, NO = DV / 32;
    static constexpr int CPR = DK <= 64 ? 8 : DK <= 128 ? 16 : 32;   // 16-byte pieces per row
    static_assert((DV <= 64 ? 8 : DV <= 128 ? 16 : 32) == CPR, "K and V rows of one pitch");
    static constexpr int STRIDE = CPR * 16;
    static constexpr int PLANE = KT * STRIDE, BUF = NP * PLANE;
    static constexpr int PPT = KT * CPR / kPromptThreads;      // pieces per thread and tile
    static_assert(PPT * kPromptThreads == KT * CPR, "pieces divide evenly");
    __device__ static __forceinline__ int swz(int r) {
        return CPR == 8 ? ((r & 2) << 1) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
    }
};

template <int TY>
struct Piece8 {   // 8 dims of one row as they are in memory
    u32x4 a;
};
template <>
struct Piece8<0> {
    f32x4 a, b;
};

// Dims d .. d+7 of a row of D.  ZERO: zero past D and where !live; else the row
// is there and d is below D (pieces may reach past it, VEC rows excepted, whose
// size is whole pieces).
template <int TY, bool VEC, bool ZERO>
__device__ __forceinline__ Piece8<TY> load_piece(const typename PromptType<TY>::T *row, int d, int D, bool live = true) {
    Piece8<TY> x = {};
    if constexpr (VEC) {
        if (!ZERO || (live && d < D)) {
            if constexpr (TY == 0) {
                x.a = *(const f32x4 *) (row + d);
                x.b = *(const f32x4 *) (row + d + 4);
            } else {
                x.a = *(const u32x4 *) (row + d);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const bool ok = d + e < D && (!ZERO || live);
            if constexpr (TY == 0) {
                const float v = ok ? row[d + e] : 0.f;
                if (e < 4) x.a[e] = v;
                else x.b[e - 4] = v;
            } else {
                const uint32_t v = ok ? ((const uint16_t *) row)[d + e] : 0;
                x.a[e / 2] |= v << (16 * (e & 1));
            }
        }
    }
    return x;
}

// lds_load16_s at a wave-uniform LDS base plus a constant.  (A load into LDS wants one wait state behind the write of m0.)
__device__ __forceinline__ void lds_load16_at(const void *sbase, uint32_t voff, uint32_t lds_base, int lds_off) {
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_base), "v"(voff), "s"(sbase), "i"(lds_off)
                 : "m0", "scc");
}

// Exponent e that scales a row's largest magnitude into [2^14, 2^15) as 2^(15 - e)
// times it.  (At least -100, so that the factor is an ordinary number: a row of
// zeros then never sets the reference of V's factors.)
__device__ __forceinline__ int split_exp(float mx) {
    return mx < INFINITY ? mx > 0.f ? max(__builtin_amdgcn_frexp_expf(mx), -100) : -100 : 15;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t) (127 + e) << 23); }

// x = hi + lo to 22 bits, each rounded to nearest.  (The difference's terms pass
// through empty asm: folded into a mixed-precision FMA with a negated operand it
// has come out wrong, see split_f16x8.)
__device__ __forceinline__ void split2(float x, _Float16 &hi, _Float16 &lo) {
    asm volatile("" : "+v"(x));
    hi = (_Float16) x;
    float f = (float) hi;
    asm volatile("" : "+v"(f));
    lo = (_Float16) (x - f);
}

template <int TY>
__device__ __forceinline__ f32x16 prompt_mfma(const u32x4 &a, const u32x4 &b, const f32x16 &c) {
    if constexpr (TY == 30)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two values rounded to nearest, in one instruction.
template <int TY>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    if constexpr (TY == 30) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, b2));
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, h2));
    }
}

// c plus both 16-bit values of x.
template <int TY>
__device__ __forceinline__ float sum2(uint32_t x, float c) {
    if constexpr (TY == 30) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, x), (b2){(__bf16) 1.f, (__bf16) 1.f}, c, false);
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), (h2){(_Float16) 1.f, (_Float16) 1.f}, c, false);
    }
}

// The larger of lanes l and l ^ 32.
__device__ __forceinline__ float max_halves(float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// Zeroes the non-finite 16-bit values of a piece; whether there were any.
template <int TY>
__device__ __forceinline__ bool finite_piece(Piece8<TY> &x) {
    bool bad = false;
    if constexpr (TY == 0) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if ((__float_as_uint(x.a[e]) & 0x7f800000u) == 0x7f800000u) x.a[e] = 0.f, bad = true;
            if ((__float_as_uint(x.b[e]) & 0x7f800000u) == 0x7f800000u) x.b[e] = 0.f, bad = true;
        }
    } else {
        constexpr uint32_t EXP = TY == 30 ? 0x7f80u : 0x7c00u;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if ((x.a[i] & EXP) == EXP) x.a[i] &= 0xffff0000u, bad = true;
            if ((x.a[i] & (EXP << 16)) == EXP << 16) x.a[i] &= 0xffffu, bad = true;
        }
    }
    return bad;
}

// Row block b of the launch: the prompts' blocks in order, each prompt's last
// (which sees the most tokens) first.  Wave-uniform; false past the last.
__device__ __forceinline__ bool find_block(const PromptParams &p, int b, int &s, int &rb, int &q0, int &L) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int s0 = 0; s0 < p.S; s0 += 64) {
        const int si = s0 + lane;
        int a = 0, len = 0, n = 0;
        if (si < p.S) {
            a = min(max(p.qsl[si], 0), p.T);
            len = min(max(p.qsl[si + 1], a), p.T) - a;
            n = (int) (((int64_t) min(len, p.max_q) * p.gqa + kPromptRows - 1) / kPromptRows);
        }
        const int sum = wave_incl_scan(n);
        const int total = __builtin_amdgcn_readlane(sum, 63);
        if (b < base + total) {
            const uint64_t m = __ballot(base + sum > b);
            const int at = __builtin_ctzll(m);
            s = s0 + at;
            q0 = __builtin_amdgcn_readlane(a, at);
            L = __builtin_amdgcn_readlane(len, at);
            rb = base + __builtin_amdgcn_readlane(sum, at) - 1 - b;   // the last block first
            return true;
        }
        base += total;
    }
    return false;
}

template <int TY, int DK, int DV, bool VEC>
__global__ __launch_bounds__(kPromptThreads) __attribute__((amdgpu_waves_per_eu(DK <= 128 ? 2 : 1))) void
pa_prompt_kernel(PromptParams p) {
    using SH = PromptShape<TY, DK, DV>;
    using T = typename PromptType<TY>::T;
    constexpr bool F32 = TY == 0, DMA = VEC && !F32;   // 16-bit tiles go straight into LDS
    constexpr int NP = SH::NP, KT = SH::KT, NH = SH::NH, KS = SH::KS, NO = SH::NO, NS = 16 * NH, CPR = SH::CPR;
    __shared__ __attribute__((aligned(16))) char lds_k[2][SH::BUF];
    __shared__ __attribute__((aligned(16))) char lds_v[2][SH::BUF];
    __shared__ __attribute__((aligned(16))) float k_up[2][F32 ? KT : 1];   // F32: 2^(e - 15) of each K row
    __shared__ __attribute__((aligned(16))) float v_up[2][F32 ? KT : 1];   // and of each V row
    __shared__ int bad_v;   // some tile that is not seen whole had non-finite values of V (left out of it)
    __shared__ int wave_end[2][kPromptWaves];

    const int hk = blockIdx.x % p.Hkv;
    int s, rb, q0, L;
    if (!find_block(p, blockIdx.x / p.Hkv, s, rb, q0, L)) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 31, h = lane >> 5;
    if (rb == 0 && hk == 0 && tid == 0 && L > p.max_q && p.err) atomicOr(p.err, 4);
    const int rows = min(L, p.max_q) * p.gqa;   // (the host holds tokens times heads below 2^31)
    const int wg0 = rb * kPromptRows, row0 = wg0 + 32 * wave;

    // ---- the wave's rows: token i of the lane's row, and the tokens it sees, [lo, end) ----
    const int row = row0 + n;
    const bool live = row < rows;
    const int i = live ? row / p.gqa : 0, head = hk * p.gqa + (live ? row - i * p.gqa : 0);
    const int64_t t = q0 + i;
    int end = 0;
    if (live) end = p.row_end ? min(max(p.row_end[t], 0), L) : p.causal ? i + 1 : L;
    const int lo = p.n_swa > 0 ? max(0, i - p.n_swa + 1) : 0;
    // of the wave: the tokens that all of its rows see, [w_lo_all, w_end_all), and that any sees, [w_lo, w_end)
    const int last = min(row0 + 31, rows - 1), i_first = row0 / p.gqa, i_last = last / p.gqa;
    // of the workgroup: its tiles start in [g_lo, g_end), and all of its rows see [g_lo_all, g_end_all)
    const int g_first = wg0 / p.gqa, g_last = (min(wg0 + kPromptRows, rows) - 1) / p.gqa;
    int w_end, w_end_all, g_end, g_end_all;
    if (p.row_end) {
        int mx = end, mn = live ? end : INT32_MAX;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            mx = max(mx, __shfl_xor(mx, o));
            mn = min(mn, __shfl_xor(mn, o));
        }
        w_end = __builtin_amdgcn_readfirstlane(mx);
        w_end_all = __builtin_amdgcn_readfirstlane(mn);
        if (lane == 0) wave_end[0][wave] = mx, wave_end[1][wave] = mn;
        __syncthreads();
        mx = 0, mn = INT32_MAX;
#pragma unroll
        for (int w = 0; w < kPromptWaves; w++) mx = max(mx, wave_end[0][w]), mn = min(mn, wave_end[1][w]);
        g_end = __builtin_amdgcn_readfirstlane(mx);
        g_end_all = __builtin_amdgcn_readfirstlane(mn);
    } else {
        w_end = row0 >= rows ? 0 : p.causal ? i_last + 1 : L;
        w_end_all = p.causal ? i_first + 1 : L;
        g_end = p.causal ? g_last + 1 : L;
        g_end_all = p.causal ? g_first + 1 : L;
    }
    const int w_lo = p.n_swa > 0 ? max(0, i_first - p.n_swa + 1) : 0;
    const int w_lo_all = p.n_swa > 0 ? max(0, i_last - p.n_swa + 1) : 0;
    const int g_lo = (p.n_swa > 0 ? max(0, g_first - p.n_swa + 1) : 0) / KT * KT;
    const int g_lo_all = p.n_swa > 0 ? max(0, g_last - p.n_swa + 1) : 0;

    // ---- staging: piece (row r, 8 dims) of a tile per thread and step; rows past the prompt's end
    // are its last one again, dims past the head's its last ones (never seen, never stored) ----
    const T *kb = (const T *) p.k + q0 * p.k_stride + (int64_t) hk * p.D;
    const T *vb = (const T *) p.v + q0 * p.v_stride + (int64_t) hk * p.Dv;
    const int pr0 = tid / CPR;   // a thread's pieces: rows pr0 + x * (threads / CPR), at one place of the row
    auto piece_row = [&](int x) __attribute__((always_inline)) { return pr0 + x * (kPromptThreads / CPR); };
    auto piece_dim = [&](int x, int D) __attribute__((always_inline)) { return min(((tid % CPR) ^ SH::swz(piece_row(x))) * 8, (D - 1) & ~7); };
    const uint32_t lk0 = lds_addr(lds_k[0]), lv0 = lds_addr(lds_v[0]);
    Piece8<TY> ks[DMA ? 1 : SH::PPT], vs[DMA ? 1 : SH::PPT];
    // 16-bit rows: byte offsets of a thread's pieces from the tile's first row
    uint32_t kvo[SH::PPT], vvo[SH::PPT];
    if constexpr (DMA) {
#pragma unroll
        for (int x = 0; x < SH::PPT; x++) {
            kvo[x] = (piece_row(x) * (uint32_t) p.k_stride + piece_dim(x, p.D)) * 2;
            vvo[x] = (piece_row(x) * (uint32_t) p.v_stride + piece_dim(x, p.Dv)) * 2;
        }
    }
    const uint32_t lkw = __builtin_amdgcn_readfirstlane(lk0 + wave * 1024), lvw = __builtin_amdgcn_readfirstlane(lv0 + wave * 1024);
    // K rows ck .. of a tile into buffer bk, V rows cv .. into bv (none from g_end on)
    auto load_rows = [&](const T *base, int64_t stride, const uint32_t (&vo)[SH::PPT], uint32_t lds, int D, int c0) __attribute__((always_inline)) {
        const T *from = base + c0 * stride;
        if (c0 + KT <= L) {
#pragma unroll
            for (int x = 0; x < SH::PPT; x++) lds_load16_at(from, vo[x], lds, x * kPromptThreads * 16);
        } else {
#pragma unroll
            for (int x = 0; x < SH::PPT; x++) {
                const uint32_t r = min(piece_row(x), L - 1 - c0);
                lds_load16_at(from, (r * (uint32_t) stride + piece_dim(x, D)) * 2, lds, x * kPromptThreads * 16);
            }
        }
    };
    auto load_tile = [&](int ck, int bk, int cv, int bv) __attribute__((always_inline)) {
        if constexpr (DMA) {
            if (ck < g_end) load_rows(kb, p.k_stride, kvo, lkw + bk * SH::BUF, p.D, ck);
            if (cv < g_end) load_rows(vb, p.v_stride, vvo, lvw + bv * SH::BUF, p.Dv, cv);
        } else {
#pragma unroll
            for (int x = 0; x < SH::PPT; x++) {
                const int64_t jk = min(ck + piece_row(x), L - 1), jv = min(cv + piece_row(x), L - 1);
                if (ck < g_end) ks[x] = load_piece<TY, VEC, false>(kb + jk * p.k_stride, piece_dim(x, p.D), p.D);
                if (cv < g_end) vs[x] = load_piece<TY, VEC, false>(vb + jv * p.v_stride, piece_dim(x, p.Dv), p.Dv);
            }
        }
    };
    // F32: the scale of a row's pieces, which are in CPR neighbouring lanes
    auto row_scale = [&](const Piece8<TY> &x, float *up) __attribute__((always_inline)) {
        float m = 0.f;
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; e++) m = fmaxf(m, fmaxf(fabsf(x.a[e]), fabsf(x.b[e])));
#pragma unroll
            for (int o = 1; o < CPR; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        }
        const int ex = split_exp(m);
        if (tid % CPR == 0) *up = pow2(ex - 15);
        return pow2(15 - ex);
    };
    auto put_piece = [&](const Piece8<TY> &x, char *at, float up) __attribute__((always_inline)) {
        if constexpr (F32) {
            f16x8 hi, lw;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                _Float16 a, b;
                split2((e < 4 ? x.a[e] : x.b[e - 4]) * up, a, b);
                hi[e] = a;
                lw[e] = b;
            }
            *(f16x8 *) at = hi;
            *(f16x8 *) (at + SH::PLANE) = lw;
        } else {
            *(u32x4 *) at = x.a;
        }
    };
    // (workgroup-uniform) some row of the workgroup does not see all of the tile
    auto partial = [&](int64_t c0) __attribute__((always_inline)) { return c0 < g_lo_all || c0 + KT > g_end_all; };
    auto put_tile = [&](int ck, int bk, int cv, int bv) __attribute__((always_inline)) {
        if constexpr (!DMA) {
            bool bad = false;
            const bool part = partial(cv);
#pragma unroll
            for (int x = 0; x < SH::PPT; x++) {
                const int at = (tid + x * kPromptThreads) * 16, r = piece_row(x);
                float up = 1.f;
                if (ck < g_end) {
                    if constexpr (F32) up = row_scale(ks[x], &k_up[bk][r]);
                    put_piece(ks[x], lds_k[bk] + at, up);
                }
                if (cv < g_end) {
                    if (part) bad |= finite_piece<TY>(vs[x]);
                    if constexpr (F32) up = row_scale(vs[x], &v_up[bv][r]);
                    put_piece(vs[x], lds_v[bv] + at, up);
                }
            }
            if (bad) bad_v = 1;
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
    };

    // the first tile (and K of the second) is on its way while Q is loaded
    if (tid == 0) bad_v = 0;
    if constexpr (!DMA) __syncthreads();
    load_tile(g_lo, 0, g_lo, 0);
    if constexpr (DMA) load_tile(g_lo + KT, 1, INT32_MAX, 0);

    // ---- Q: dims 16 ks + 8h .. + 7 of the lane's row (negated for a negative scale) ----
    u32x4 qr[NP][KS];
    // of the product; above zero, so that a masked score stays -inf (a scale of zero takes Q as zero instead)
    float cs = p.scale == 0.f ? 1.f : fabsf(p.softcap > 0.f ? p.scale / p.softcap : p.scale * kLog2e);
    {
        const T *qp = (const T *) p.q + t * p.q_stride + (int64_t) head * p.D;
        if constexpr (!F32) {
            const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                qr[0][k] = load_piece<TY, VEC, true>(qp, 16 * k + 8 * h, p.D, live).a;
#pragma unroll
                for (int e = 0; e < 4; e++) qr[0][k][e] = p.scale == 0.f ? 0 : qr[0][k][e] ^ sign;
            }
        } else {
            Piece8<0> x[KS];
            float mx = 0.f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                x[k] = load_piece<TY, VEC, true>(qp, 16 * k + 8 * h, p.D, live);
#pragma unroll
                for (int e = 0; e < 4; e++) mx = fmaxf(mx, fmaxf(fabsf(x[k].a[e]), fabsf(x[k].b[e])));
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const int ex = split_exp(mx);
            const float up = p.scale == 0.f ? 0.f : p.scale < 0.f ? -pow2(15 - ex) : pow2(15 - ex);
            cs *= pow2(ex - 15);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                f16x8 hi, lw;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    _Float16 a, b;
                    split2((e < 4 ? x[k].a[e] : x[k].b[e - 4]) * up, a, b);
                    hi[e] = a;
                    lw[e] = b;
                }
                qr[0][k] = __builtin_bit_cast(u32x4, hi);
                qr[NP - 1][k] = __builtin_bit_cast(u32x4, lw);
            }
        }
        cs = fmaxf(cs, 1e-37f);
        // Q is here: no wait for it (and with it for the tile in flight) inside the loop
#pragma unroll
        for (int k = 0; k < KS; k++) {
            asm volatile("" : "+v"(qr[0][k]));
            if constexpr (F32) asm volatile("" : "+v"(qr[NP - 1][k]));
        }
    }

    f32x16 o[NO];
#pragma unroll
    for (int m = 0; m < NO; m++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[m][r] = 0.f;
    float m_ref = -0x1p127f, l = 0.f;   // reference maximum (log2 units, below any score) and the lane's part of the sum
    float v_ref = 0x1p-126f;            // F32: power of two that V's factors are taken relative to

    // lane's LDS byte offsets.  K row n (+ 32 hh), piece 2k + h; V transpose reads: rows 4h + (lane%16)/4 (+ 8, + 16 st),
    // dims 32m + 16((lane/16)%2) + 4(lane%4): piece 4m + 2((lane/16)%2) + (lane%4)/2, 8 bytes into it for odd lanes.  The
    // exclusive or does not mix with the constants added, so a base per distinct pattern is kept: swz(n) is K's; rows r and
    // r + 8 (r + 16 is r again) are V's.
    const int vrow = 4 * h + ((lane & 15) >> 2), vpiece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    uint32_t koff[KS], voff[2][NO];
#pragma unroll
    for (int k = 0; k < KS; k++) koff[k] = lk0 + n * SH::STRIDE + 16 * ((2 * k + h) ^ SH::swz(n));
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int m = 0; m < NO; m++)
            voff[e][m] = lv0 + (vrow + 8 * e) * SH::STRIDE + 16 * ((4 * m + vpiece) ^ SH::swz(vrow + 8 * e)) + 8 * (lane & 1);

    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    // The tile loop.  K is a tile ahead of V: while the weights of tile i are computed and its V multiplied, the matrix
    // cores also take the scores of tile i + 1 into the other score registers, so that vector and matrix work of one
    // wave overlap.  F32 has no registers for that, and takes tile i's scores at its start (AHEAD = 0).
    constexpr int AHEAD = F32 ? 0 : 1;
    constexpr int NQ = KS * NH;   // products of a tile's scores, and of its V (triples of them, F32)
    static_assert(NQ == NO * (NS / 8), "as many products with K as with V");
    u32x4 kr[3][NP], vr[3][NP];   // operands, read two products ahead
    auto read_k = [&](int q, int buf) __attribute__((always_inline)) {
        const int k = q / NH, hh = q % NH;
#pragma unroll
        for (int e = 0; e < NP; e++)
            kr[q % 3][e] = *(const lds_u32x4 *) (uintptr_t) (koff[k] + buf * SH::BUF + e * SH::PLANE + hh * 32 * SH::STRIDE);
    };
    auto mul_k = [&](int q, int buf, f32x16 (&sc)[NH]) __attribute__((always_inline)) {
        const int k = q / NH, hh = q % NH;
        if (q + 2 < NQ) read_k(q + 2, buf);
        if (k == 0)
#pragma unroll
            for (int r = 0; r < 16; r++) sc[hh][r] = 0.f;
        sc[hh] = prompt_mfma<TY>(kr[q % 3][0], qr[0][k], sc[hh]);
        if constexpr (F32) {
            sc[hh] = prompt_mfma<TY>(kr[q % 3][NP - 1], qr[0][k], sc[hh]);
            sc[hh] = prompt_mfma<TY>(kr[q % 3][0], qr[NP - 1][k], sc[hh]);
        }
    };
    auto scores = [&](int buf, f32x16 (&sc)[NH]) __attribute__((always_inline)) {
        read_k(0, buf);
        read_k(1, buf);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            mul_k(q, buf, sc);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto read_v = [&](int q, int buf) __attribute__((always_inline)) {
        const int st = q / NO, m = q % NO;
#pragma unroll
        for (int e = 0; e < NP; e++) {
            const uint32_t off = buf * SH::BUF + e * SH::PLANE + 16 * st * SH::STRIDE;
            vr[q % 3][e] = __builtin_bit_cast(u32x4, lds_tr_b16x8_at(voff[0][m] + off, voff[1][m] + off));
        }
    };
    // Tile c0, whose V is in buffer `buf` and whose scores are sc; with AHEAD, the next tile's scores into nx.
    auto tile = [&](int c0, auto buf_, f32x16 (&sc)[NH], f32x16 (&nx)[NH]) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_)::value;
        const int k_at = c0 + (AHEAD + 1) * KT, v_at = c0 + KT;   // what is loaded while this tile is computed
        load_tile(k_at, buf ^ 1 ^ AHEAD, v_at, buf ^ 1);
        if (DMA && partial(c0)) {
            bool bad = false;
#pragma unroll
            for (int x = 0; x < SH::PPT; x++) {
                Piece8<TY> v;
                u32x4 *at = (u32x4 *) (lds_v[buf] + (tid + x * kPromptThreads) * 16);
                if constexpr (!F32) {
                    v.a = *at;
                    if (finite_piece<TY>(v)) *at = v.a, bad = true;
                }
            }
            if (bad) bad_v = 1;
            __syncthreads();
        }
        if (c0 < w_end && c0 + KT > w_lo) {   // wave-uniform: some row sees some of the tile
            if constexpr (!AHEAD) scores(buf, sc);
            // ---- softmax ----
            float x[NS];
            float cx = cs;   // x times cx is the score in log2 units
#pragma unroll
            for (int j = 0; j < NS; j++) {
                x[j] = sc[j / 16][j % 16];
                if constexpr (F32) x[j] *= k_up[buf][(j / 16) * 32 + 8 * (j % 16 / 4) + 4 * h + j % 4];
            }
            if (p.softcap > 0.f) {
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    if constexpr (F32) x[j] = tanhf(x[j] * cs);
                    else x[j] = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x[j] * (cs * (2.f * kLog2e))));
                }
                cx = p.softcap * kLog2e;
            }
            if (c0 < w_lo_all || c0 + KT > w_end_all) {   // wave-uniform
                const int a = lo - c0 - 4 * h, b = end - c0 - 4 * h;
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    const int key = (j / 16) * 32 + 8 * (j % 16 / 4) + j % 4;
                    x[j] = key >= a && key < b ? x[j] : -INFINITY;
                }
            }
            if constexpr (AHEAD) {
                read_k(0, buf ^ 1);
                read_k(1, buf ^ 1);
#pragma unroll
                for (int q = 0; q < NQ / 4; q++) mul_k(q, buf ^ 1, nx);
            }
            float mx = x[0];
#pragma unroll
            for (int j = 1; j < NS; j++) mx = fmaxf(mx, x[j]);
            mx = max_halves(mx) * cx;
            if (__any(mx > m_ref + kRescaleSlack)) {
                const float mn = mx > m_ref + kRescaleSlack ? mx : m_ref;
                const float alpha = __builtin_amdgcn_exp2f(m_ref - mn);
                m_ref = mn;
                l *= alpha;
#pragma unroll
                for (int m = 0; m < NO; m++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[m][r] *= alpha;
            }
            const float ref = m_ref;
            u32x4 pr[NP][NS / 8];
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], cx, -ref));
                    l += x[j];
                }
                // V's factors: of the tokens with a weight, at most 2^6 times the row's reference
                float vf[NS], top = 0.f;
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    vf[j] = v_up[buf][(j / 16) * 32 + 8 * (j % 16 / 4) + 4 * h + j % 4];
                    top = fmaxf(top, x[j] != 0.f ? vf[j] : 0.f);
                }
                top = max_halves(top);
                if (__any(top > v_ref * 64.f)) {
                    const float vn = top > v_ref * 64.f ? top : v_ref;
                    const float beta = v_ref / vn;
                    v_ref = vn;
#pragma unroll
                    for (int m = 0; m < NO; m++)
#pragma unroll
                        for (int r = 0; r < 16; r++) o[m][r] *= beta;
                }
                const float inv = 1.f / v_ref;
#pragma unroll
                for (int st = 0; st < NS / 8; st++) {
                    f16x8 hi, lw;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        _Float16 a, b;
                        // (a token of no weight may have any factor)
                        split2(x[8 * st + e] != 0.f ? x[8 * st + e] * (vf[8 * st + e] * inv) : 0.f, a, b);
                        hi[e] = a;
                        lw[e] = b;
                    }
                    pr[0][st] = __builtin_bit_cast(u32x4, hi);
                    pr[NP - 1][st] = __builtin_bit_cast(u32x4, lw);
                }
            }
            // ---- O^T += V^T P^T, the next 16 tokens' probabilities beside the products of 16 ----
            // (the sum is of the rounded probabilities, as the products are)
            auto weigh = [&](int st, int e) __attribute__((always_inline)) {   // pair e of the 16 tokens st
                x[8 * st + 2 * e] = __builtin_amdgcn_exp2f(fmaf(x[8 * st + 2 * e], cx, -ref));
                x[8 * st + 2 * e + 1] = __builtin_amdgcn_exp2f(fmaf(x[8 * st + 2 * e + 1], cx, -ref));
                pr[0][st][e] = pack2<TY>(x[8 * st + 2 * e], x[8 * st + 2 * e + 1]);
                l = sum2<TY>(pr[0][st][e], l);
            };
            read_v(0, buf);
            read_v(1, buf);
            if constexpr (!F32) {
#pragma unroll
                for (int e = 0; e < 4; e++) weigh(0, e);
#pragma unroll
                for (int q = NQ / 4; q < NQ / 2; q++) mul_k(q, buf ^ 1, nx);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                const int st = q / NO, m = q % NO;
                if (q + 2 < NQ) read_v(q + 2, buf);
                o[m] = prompt_mfma<TY>(vr[q % 3][0], pr[0][st], o[m]);
                if constexpr (F32) {
                    o[m] = prompt_mfma<TY>(vr[q % 3][NP - 1], pr[0][st], o[m]);
                    o[m] = prompt_mfma<TY>(vr[q % 3][0], pr[NP - 1][st], o[m]);
                } else {
                    if (q % 2 == 0) mul_k(NQ / 2 + q / 2, buf ^ 1, nx);
                    if (st + 1 < NS / 8) {
#pragma unroll
                        for (int e = 4 * m / NO; e < 4 * (m + 1) / NO; e++) weigh(st + 1, e);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else if constexpr (AHEAD) {
            scores(buf ^ 1, nx);
        }
        put_tile(k_at, buf ^ 1 ^ AHEAD, v_at, buf ^ 1);
        __syncthreads();
    };
    f32x16 s0[NH], s1[NH];
    put_tile(g_lo, 0, g_lo, 0);
    __syncthreads();
    if constexpr (AHEAD) {
        if constexpr (!DMA) load_tile(g_lo + KT, 1, INT32_MAX, 0);
        scores(0, s0);
        if constexpr (!DMA) put_tile(g_lo + KT, 1, INT32_MAX, 0);
        __syncthreads();
    }
    for (int c0 = g_lo; c0 < g_end; c0 += 2 * KT) {
        tile(c0, std::integral_constant<int, 0>(), s0, s1);
        if (c0 + KT >= g_end) break;
        tile(c0 + KT, std::integral_constant<int, 1>(), s1, s0);
    }

    // ---- V's non-finite values, left out of the tiles, for the rows that see them ----
    if (bad_v)
        for (int j = g_lo; j < min(g_end, L); j++) {
            if (!partial(j / KT * KT)) continue;
            const T *vr = vb + (int64_t) j * p.v_stride;
            const bool sees = j >= lo && j < end;
#pragma unroll
            for (int m = 0; m < NO; m++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int d = 32 * m + 8 * (r / 4) + 4 * h + r % 4;
                    const float v = sees && d < p.Dv ? (float) vr[d] : 0.f;
                    o[m][r] += (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? v : 0.f;
                }
        }

    // ---- rows out ----
    l += __shfl_xor(l, 32);
    float inv = l == 0.f ? 0.f : 1.f / l;
    if (!live) return;
    if constexpr (F32) inv *= v_ref;   // (an empty row: 0 * 2^-126)
    T *out = (T *) p.out + t * p.o_stride + (int64_t) head * p.Dv;
#pragma unroll
    for (int m = 0; m < NO; m++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int d = 32 * m + 8 * b + 4 * h;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = o[m][4 * b + e] * inv;
            if (VEC && d < p.Dv) {
                if constexpr (F32) *(float4 *) (out + d) = make_float4(y[0], y[1], y[2], y[3]);
                else *(u32x2 *) (out + d) = u32x2{pack2<TY>(y[0], y[1]), pack2<TY>(y[2], y[3])};
            } else if (!VEC) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (d + e < p.Dv) out[d + e] = (T) y[e];
            }
        }
}

template <int TY, int DK, int DV>
static hipError_t launch_prompt_d(const PromptParams &p, bool vec, hipStream_t stream) {
    // blocks of the launch: at most one more than whole ones for each prompt
    const int64_t rows = (int64_t) p.T * p.gqa, per = ((int64_t) p.max_q * p.gqa + kPromptRows - 1) / kPromptRows;
    const int64_t blocks = std::min(rows / kPromptRows + p.S, per * p.S) * p.Hkv;
    if (blocks > (1 << 23)) return hipErrorInvalidValue;   // 256 threads each: a launch holds below 2^32
    const dim3 grid((unsigned) blocks), wg(kPromptThreads);
    if (vec) hipLaunchKernelGGL((pa_prompt_kernel<TY, DK, DV, true>), grid, wg, 0, stream, p);
    else hipLaunchKernelGGL((pa_prompt_kernel<TY, DK, DV, false>), grid, wg, 0, stream, p);
    return hipGetLastError();
}

// Rows of whole aligned pieces of 16 bytes.
template <int TY>
static bool prompt_vec(const PromptParams &p) {
    const int64_t es = TY == 0 ? 4 : 2;
    const uintptr_t al = (uintptr_t) p.q | (uintptr_t) p.k | (uintptr_t) p.v | (uintptr_t) p.out;
    // (a tile's rows are addressed by 32-bit offsets)
    if (std::max(p.k_stride, p.v_stride) >= 1 << 24) return false;
    return al % 16 == 0 && ((p.q_stride | p.k_stride | p.v_stride | p.o_stride) * es) % 16 == 0 && p.D % 8 == 0 && p.Dv % 8 == 0;
}

}  // namespace iian_pa
