// pa_prompt.h - whole-prompt attention on the matrix cores (iian_pa_prompt_attention):
// packed prompts, grouped heads, head sizes up to 256; F16, BF16 and F32 rows
// (pa_prompt.hip, pa_prompt_bf16.hip, pa_prompt_f32.hip hold one type each).
//
// A workgroup of 4 waves owns 128 rows r = i*gqa + g (token i, head g of the
// group) of one (prompt, kv head), 32 per wave, and walks the tokens that any of
// them sees in tiles of 32, staged in LDS two tiles ahead (one ahead through
// registers), one barrier per tile.  Calls with fewer workgroups than that fills
// the chip with split the tokens instead (KW > 1): KW waves share 32 rows, each
// takes every KW-th tile, and their results are joined in LDS at the end.  Head
// size 256 has 8 waves and 256 rows (its O and Q leave room for two waves per
// SIMD, the Q pieces that do not fit wait in LDS), F32 rows 8 waves in small
// calls.  One pass with a running maximum and sum per row:
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
// that do see them add them after the loop.
//
// What bounds it (calls, and PMC of the same): one prompt of 8192 f16 tokens at
// H32/Hkv8/D128 526 us, 1.04 PFLOP/s, matrix cores 59% busy at the 1.6 GHz that the
// card's power allows (397 us with zeros as data).  16 prompts of 100 to 2000
// tokens 80 us: the latencies before and behind a workgroup's loop, a third of its
// cycles, hidden by two others.  D256: LDS, of which 8 waves read 336 KB a tile.
// F32: the conversion into terms.
#pragma once

#include "pa_common.h"
#include "pa_launch.h"
#include "pa_mfma.h"

#include <algorithm>
#include <type_traits>

namespace iian_pa {

constexpr int kPromptCus = 256;   // an MI355X

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

// TY: rows' type; DK: head size rounded up to 16 dims, DV: to 32; VEC: rows of
// whole aligned 16-byte pieces; KW: waves that share their rows; NW: waves of a
// workgroup.
//
// LDS tiles.  Rows are unpadded, so that tiles of 16-bit rows can be loaded
// straight into LDS (16 consecutive bytes per lane), and the 16-byte pieces of
// row r are permuted by an exclusive or with swz(r) instead: 16 rows read at one
// piece, as QK^T does, and the 4 rows x 64 bytes of a transpose read each fill
// the 64 banks.
template <int TY, int DK, int DV, bool VEC, int KW, int NW>
struct PromptShape {
    static constexpr int NP = TY == 0 ? 2 : 1;             // 16-bit terms per value
    static constexpr bool DMA = VEC && TY != 0;            // tiles go straight into LDS
    static constexpr int KT = 32, TT = KT * KW;            // tokens per wave and tile, and per workgroup's
    static constexpr int THREADS = NW * 64, ROWS = 32 * (NW / KW);   // of a workgroup
    static constexpr int KS = DK / 16, NO = DV / 32, NS = 16;
    static constexpr int CPR = DK <= 64 ? 8 : DK <= 128 ? 16 : 32;   // 16-byte pieces per row
    static_assert((DV <= 64 ? 8 : DV <= 128 ? 16 : 32) == CPR, "K and V rows of one pitch");
    static constexpr int STRIDE = CPR * 16;
    static constexpr int PLANE = TT * STRIDE, BUF = NP * PLANE;
    // three buffers (loads two tiles ahead) where three workgroups of them fit a CU's 160 KB of LDS
    static constexpr int NB = DMA && BUF * 6 <= 49152 ? 3 : 2;
    static constexpr int PPT = TT * CPR / THREADS;  // pieces per thread and tile
    static_assert(PPT * THREADS == TT * CPR, "pieces divide evenly");
    // Q pieces (of KS) that wait in LDS instead of registers: with 8 waves of head size 256, O and half of Q fit the 256
    // registers that two waves per SIMD have
    // (F32 at 256: of Q's lo terms, as many as LDS has room for)
    static constexpr int QL = DK <= 128 ? 0 : TY == 0 ? 7 : NW == 8 ? KS * 5 / 8 : 0;
    // waves per SIMD asked of the register allocator
    static constexpr int WAVES = DK > 128 ? NW / 4 : TY == 0 || (KW > 1 && DK > 64) ? 2 : 3;
    static constexpr int RD = TY == 0 && DK > 128 ? 2 : 3;   // operands held: read RD - 1 products ahead
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

// The larger of lanes l and l ^ 32.
__device__ __forceinline__ float max_halves(float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// x[2i], x[2i+1] = hi + lo to 22 bits, each rounded to nearest, into element i of
// hi and lo (packed f16).  (The differences' terms pass through empty asm: folded
// into a mixed-precision FMA with a negated operand they have come out wrong,
// see split_f16x8.)
__device__ __forceinline__ void split2(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    asm volatile("" : "+v"(x0), "+v"(x1));
    const h2 h = __builtin_convertvector((f2){x0, x1}, h2);
    float f0 = (float) h[0], f1 = (float) h[1];
    asm volatile("" : "+v"(f0), "+v"(f1));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x0 - f0, x1 - f1}, h2));
}

// Largest |x| of a piece, and of the pieces of CPR neighbouring lanes.
__device__ __forceinline__ float piece_max(const Piece8<0> &x) {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) m = fmaxf(fmaxf(m, fabsf(x.a[e])), fabsf(x.b[e]));   // (one instruction each)
    return m;
}
template <int CPR>
__device__ __forceinline__ float lanes_max(float m) {
    auto with = [&](auto ctrl) __attribute__((always_inline)) {
        return fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), decltype(ctrl)::value, 0xf, 0xf, true)));
    };
    m = with(std::integral_constant<int, 0xb1>());    // quad_perm [1, 0, 3, 2]
    m = with(std::integral_constant<int, 0x4e>());    // quad_perm [2, 3, 0, 1]
    m = with(std::integral_constant<int, 0x141>());   // row_half_mirror: the other quad of 8 lanes
    if constexpr (CPR >= 16) m = with(std::integral_constant<int, 0x140>());   // row_mirror: the other 8 of 16
    if constexpr (CPR >= 32) m = fmaxf(m, __shfl_xor(m, 16));
    return m;
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

// Whether a 16-bit piece holds non-finite values.
template <int TY>
__device__ __forceinline__ bool any_bad(const u32x4 &a) {
    typedef uint16_t h2 __attribute__((ext_vector_type(2)));
    constexpr uint32_t EXP = TY == 30 ? 0x7f807f80u : 0x7c007c00u;
    auto e = [&](int i) { return __builtin_bit_cast(h2, a[i] & EXP); };
    const h2 m = __builtin_elementwise_max(__builtin_elementwise_max(e(0), e(1)), __builtin_elementwise_max(e(2), e(3)));
    return m[0] == (uint16_t) EXP || m[1] == (uint16_t) EXP;
}

// Zeroes the non-finite values of a piece; whether there were any.
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

// r / gqa by the host's multiplier (2^32 / gqa + 1: at most one too many for r
// below 2^31; 0 for gqa = 1).
__device__ __forceinline__ int token_of_row(const PromptParams &p, int r) {
    if (p.gqa_mul == 0) return r;
    const int q = (int) __umulhi((uint32_t) r, p.gqa_mul);
    return q * p.gqa > r ? q - 1 : q;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int lane_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);    // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast 31 into rows 2 and 3
    return v;
}

struct PromptBlock {
    int s, rb, q0, L;   // prompt, row block, first token, tokens
};

// Row block b of the launch, in an order that starts the longest work first:
// with up to 64 prompts, causal ones by row block, the last of any prompt first
// (a row block's work grows with its place in the prompt), others by the
// prompt's length.  More prompts: in order, each prompt's last block first.
// Wave-uniform; false past the last block.
template <int ROWS>
__device__ __forceinline__ bool find_block(const PromptParams &p, int b, PromptBlock &out) {
    const int lane = threadIdx.x & 63;
    auto blocks = [&](int from, int to, int &a, int &len) {
        a = min(max(from, 0), p.T);
        len = min(max(to, a), p.T) - a;
        return (int) ((uint32_t) (min(len, p.max_q) * p.gqa + ROWS - 1) / ROWS);   // (the host holds tokens times heads below 2^31)
    };
    auto prompt = [&](int s, int &a, int &len) { return blocks(p.qsl[s], p.qsl[s + 1], a, len); };
    int a = 0, len = 0, n = 0, s0 = 0;
    if (p.S <= 64) {
        if (lane < p.S) n = prompt(lane, a, len);
        if (p.S > 1) {
            int at, rb;
            if (p.causal || p.row_end) {
                // the largest row block index r with more than b blocks at r or above
                // (the sum over prompts of max(0, n - lo) is above b, at hi it is not)
                int lo = 0, above = 0, hi = (int) ((uint32_t) (p.max_q * p.gqa + ROWS - 1) / ROWS);
                if (b >= __builtin_amdgcn_readlane(lane_scan(n), 63)) return false;
                while (hi - lo > 1) {
                    const int m = (lo + hi) >> 1, c = __builtin_amdgcn_readlane(lane_scan(max(0, n - m)), 63);
                    if (c > b) lo = m;
                    else hi = m, above = c;
                }
                uint64_t m = __ballot(n > lo);
                for (int k = b - above; k > 0; k--) m &= m - 1;
                at = __builtin_ctzll(m);
                rb = lo;
            } else {
                int before = 0;   // blocks of longer prompts, and of earlier ones as long
                for (int j = 0; j < p.S; j++) {
                    const int nj = __builtin_amdgcn_readlane(n, j);
                    before += nj > n || (nj == n && j < lane) ? nj : 0;
                }
                const uint64_t m = __ballot(b >= before && b < before + n);
                if (!m) return false;
                at = __builtin_ctzll(m);
                rb = b - __builtin_amdgcn_readlane(before, at);
            }
            out = {at, rb, __builtin_amdgcn_readlane(a, at), __builtin_amdgcn_readlane(len, at)};
            return true;
        }
    } else {
        // the lane's share of the prompts, then the prompts of the share that holds b
        const int per = (p.S + 63) / 64;
        int sum = 0;
        for (int s = lane * per, last = min(p.S, (lane + 1) * per); s < last; s += 8) {
            int at[9];   // (together: one wait for the nine)
#pragma unroll
            for (int j = 0; j < 9; j++) at[j] = p.qsl[min(s + j, last)];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (s + j < last) sum += blocks(at[j], at[j + 1], a, len);
        }
        const int scan = lane_scan(sum);
        const uint64_t m = __ballot(scan > b);
        if (!m) return false;
        const int at = __builtin_ctzll(m);
        b -= __builtin_amdgcn_readlane(scan, at) - __builtin_amdgcn_readlane(sum, at);
        s0 = at * per;
        n = 0;
        if (s0 + lane < p.S) n = prompt(s0 + lane, a, len);
    }
    for (;;) {
        const int scan = lane_scan(n), all = __builtin_amdgcn_readlane(scan, 63);
        if (b < all) {
            const int at = __builtin_ctzll(__ballot(scan > b));
            out = {s0 + at, __builtin_amdgcn_readlane(scan, at) - 1 - b, __builtin_amdgcn_readlane(a, at),
                   __builtin_amdgcn_readlane(len, at)};
            return true;
        }
        b -= all;
        s0 += 64;
        if (s0 >= p.S) return false;
        n = 0;
        if (s0 + lane < p.S) n = prompt(s0 + lane, a, len);
    }
}

template <int TY, int DK, int DV, bool VEC, int KW, int NW>
__global__ __launch_bounds__(NW * 64)
    __attribute__((amdgpu_waves_per_eu(PromptShape<TY, DK, DV, VEC, KW, NW>::WAVES))) void pa_prompt_kernel(PromptParams p) {
    using SH = PromptShape<TY, DK, DV, VEC, KW, NW>;
    using T = typename PromptType<TY>::T;
    constexpr bool F32 = TY == 0, DMA = SH::DMA;
    constexpr int NP = SH::NP, KT = SH::KT, TT = SH::TT, NB = SH::NB, KS = SH::KS, NO = SH::NO, NS = SH::NS, CPR = SH::CPR;
    constexpr int ROWS = SH::ROWS;
    // K and V tiles; in the end the waves' results that are joined
    constexpr int JOIN = KW > 1 ? NW * (NO * 16 + 2) * 64 * 4 : 0;
    __shared__ __attribute__((aligned(16))) char lds[std::max(2 * NB * SH::BUF, JOIN)];
    char *const lds_k = lds, *const lds_v = lds + NB * SH::BUF;
    __shared__ __attribute__((aligned(16))) float k_up[NB][F32 ? TT : 1];   // F32: 2^(e - 15) of each K row
    __shared__ __attribute__((aligned(16))) float v_up[NB][F32 ? TT : 1];   // and of each V row
    __shared__ __attribute__((aligned(16))) u32x4 q_lds[std::max(1, NW * SH::QL * 64)];   // each lane's own Q pieces
    __shared__ int bad_v;   // some tile that is not seen whole had non-finite values of V (left out of it)
    __shared__ int wave_end[2][NW];

    const int hk = blockIdx.x % p.Hkv;
    PromptBlock blk;
    if (!find_block<ROWS>(p, blockIdx.x / p.Hkv, blk)) return;
    const int q0 = blk.q0, L = blk.L;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 31, h = lane >> 5;
    if (blk.rb == 0 && hk == 0 && tid == 0 && L > p.max_q && p.err) atomicOr(p.err, 4);
    const int rows = min(L, p.max_q) * p.gqa;   // (the host holds tokens times heads below 2^31)
    if ((uint32_t) blk.rb > (uint32_t) rows / ROWS) return;   // (counts of an out-of-order query_start_loc may pass 32 bits)
    const int wg0 = blk.rb * ROWS, row0 = wg0 + 32 * (wave / KW), kg = wave % KW;

    // ---- the wave's rows: token i of the lane's row, and the tokens it sees, [lo, end) ----
    const int row = row0 + n;
    const bool live = row < rows;
    auto token_of = [&](int r) { return token_of_row(p, r); };
    const int i = live ? token_of(row) : 0, head = hk * p.gqa + (live ? row - i * p.gqa : 0);
    const int64_t t = q0 + i;
    int end = 0;
    if (live) end = p.row_end ? min(max(p.row_end[t], 0), L) : p.causal ? i + 1 : L;
    const int lo = p.n_swa > 0 ? max(0, i - p.n_swa + 1) : 0;
    // of the wave: the tokens that all of its rows see, [w_lo_all, w_end_all), and that any sees, [w_lo, w_end)
    const int i_first = token_of(row0), i_last = token_of(min(row0 + 31, rows - 1));
    // of the workgroup: its tiles start in [g_lo, g_end), and all of its rows see [g_lo_all, g_end_all)
    const int g_first = token_of(wg0), g_last = token_of(min(wg0 + ROWS, rows) - 1);
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
        for (int w = 0; w < NW; w++) mx = max(mx, wave_end[0][w]), mn = min(mn, wave_end[1][w]);
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
    const int g_lo = (p.n_swa > 0 ? max(0, g_first - p.n_swa + 1) : 0) / TT * TT;
    const int g_lo_all = p.n_swa > 0 ? max(0, g_last - p.n_swa + 1) : 0;

    // ---- staging: piece (row r, 8 dims) of a tile per thread and step; rows past the prompt's end
    // are its last one again, dims past the head's its last ones (never seen, never stored) ----
    const T *kb = (const T *) p.k + q0 * p.k_stride + (int64_t) hk * p.D;
    const T *vb = (const T *) p.v + q0 * p.v_stride + (int64_t) hk * p.Dv;
    const int pr0 = tid / CPR;   // a thread's pieces: rows pr0 + x * (threads / CPR), at one place of the row
    auto piece_row = [&](int x) __attribute__((always_inline)) { return pr0 + x * (SH::THREADS / CPR); };
    auto piece_dim = [&](int x, int D) __attribute__((always_inline)) { return min(((tid % CPR) ^ SH::swz(piece_row(x))) * 8, (D - 1) & ~7); };
    const uint32_t lk0 = lds_addr(lds_k), lv0 = lds_addr(lds_v);
    Piece8<TY> st[DMA ? 1 : SH::PPT], st0[DMA ? 1 : SH::PPT];   // of K or of V, on their way through registers (st0: the first K)
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
    // 16-bit rows c0 .. of a tile into LDS; nothing from g_end on.
    auto load_tile = [&](int c0, int buf) __attribute__((always_inline)) {
        if (c0 >= g_end) return;
        const T *const kt = kb + c0 * p.k_stride, *const vt = vb + c0 * p.v_stride;
        const uint32_t lk = lkw + buf * SH::BUF, lv = lvw + buf * SH::BUF;
        if (c0 + TT <= L) {
#pragma unroll
            for (int x = 0; x < SH::PPT; x++) {
                lds_load16_at(kt, kvo[x], lk, x * SH::THREADS * 16);
                lds_load16_at(vt, vvo[x], lv, x * SH::THREADS * 16);
            }
        } else {
#pragma unroll
            for (int x = 0; x < SH::PPT; x++) {
                const uint32_t r = min(piece_row(x), L - 1 - c0);
                lds_load16_at(kt, (r * (uint32_t) p.k_stride + piece_dim(x, p.D)) * 2, lk, x * SH::THREADS * 16);
                lds_load16_at(vt, (r * (uint32_t) p.v_stride + piece_dim(x, p.Dv)) * 2, lv, x * SH::THREADS * 16);
            }
        }
    };
    // The others through registers, K and V in turn: rows c0 .. of a tile of K or V into st.
    auto load_rows = [&](auto &st, const T *base, int64_t stride, int D, int c0) __attribute__((always_inline)) {
        if (c0 >= g_end) return;
#pragma unroll
        for (int x = 0; x < SH::PPT; x++)
            st[x] = load_piece<TY, VEC, false>(base + (int64_t) min(c0 + piece_row(x), L - 1) * stride, piece_dim(x, D), D);
    };
    // F32: the scale of a row's pieces, which are in CPR neighbouring lanes
    auto row_scale = [&](const Piece8<TY> &x, float *up) __attribute__((always_inline)) {
        int ex = 0;
        if constexpr (F32) ex = split_exp(lanes_max<CPR>(piece_max(x)));
        if (tid % CPR == 0) *up = pow2(ex - 15);
        return pow2(15 - ex);
    };
    auto put_piece = [&](const Piece8<TY> &x, char *at, float up) __attribute__((always_inline)) {
        if constexpr (F32) {
            u32x4 hi, lw;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const f32x4 &y = e < 2 ? x.a : x.b;
                uint32_t a, b;
                split2(y[2 * (e & 1)] * up, y[2 * (e & 1) + 1] * up, a, b);
                hi[e] = a;
                lw[e] = b;
            }
            *(u32x4 *) at = hi;
            *(u32x4 *) (at + SH::PLANE) = lw;
        } else {
            *(u32x4 *) at = x.a;
        }
    };
    // (workgroup-uniform) some row of the workgroup does not see all of the tile
    auto partial = [&](int c0) __attribute__((always_inline)) { return c0 < g_lo_all || c0 + TT > g_end_all; };
    // st, rows c0 .. of K or V, into LDS
    auto put_rows = [&](auto &st, char *lds_at, float *ups, int c0, bool v) __attribute__((always_inline)) {
        if (c0 >= g_end) return;
        const bool part = v && partial(c0);
        bool bad = false;
#pragma unroll
        for (int x = 0; x < SH::PPT; x++) {
            float up = 1.f;
            if (part) bad |= finite_piece<TY>(st[x]);
            if constexpr (F32) up = row_scale(st[x], &ups[piece_row(x)]);
            put_piece(st[x], lds_at + (tid + x * SH::THREADS) * 16, up);
        }
        if (bad) bad_v = 1;
    };
    // The wait for a tile behind which `newer` ones may still be on their way.
    auto wait_tile = [&](bool newer) __attribute__((always_inline)) {
        if (newer) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * SH::PPT) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };

    // the first tiles are on their way while Q is loaded
    if (tid == 0) bad_v = 0;
    if constexpr (DMA) {
        load_tile(g_lo, 0);
        if constexpr (NB == 3) load_tile(g_lo + TT, 1);
    } else {
        __syncthreads();
        load_rows(st0, kb, p.k_stride, p.D, g_lo);
        load_rows(st, vb, p.v_stride, p.Dv, g_lo);
    }

    // ---- Q: dims 16 ks + 8h .. + 7 of the lane's row (negated for a negative scale) ----
    constexpr int QL = SH::QL, QR = KS - QL;   // the last QL pieces (F32: of the lo terms) in LDS
    u32x4 qh[F32 ? KS : QR], qlo[F32 ? QR : 1];
    u32x4 *const ql = q_lds + wave * QL * 64 + lane;
    // of the product; above zero, so that a masked score stays -inf (a scale of zero takes Q as zero instead)
    float cs = p.scale == 0.f ? 1.f : fabsf(p.softcap > 0.f ? p.scale / p.softcap : p.scale * kLog2e);
    {
        const T *qp = (const T *) p.q + t * p.q_stride + (int64_t) head * p.D;
        if constexpr (!F32) {
            const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                u32x4 x = load_piece<TY, VEC, true>(qp, 16 * k + 8 * h, p.D, live).a;
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = p.scale == 0.f ? 0 : x[e] ^ sign;
                if (k < QR) qh[k] = x;
                else ql[(k - QR) * 64] = x;
            }
        } else {
            Piece8<0> x[KS];
            float mx = 0.f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                x[k] = load_piece<TY, VEC, true>(qp, 16 * k + 8 * h, p.D, live);
                mx = fmaxf(mx, piece_max(x[k]));
            }
            const int ex = split_exp(max_halves(mx));
            const float up = p.scale == 0.f ? 0.f : p.scale < 0.f ? -pow2(15 - ex) : pow2(15 - ex);
            cs *= pow2(ex - 15);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                u32x4 lw;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const f32x4 &y = e < 2 ? x[k].a : x[k].b;
                    uint32_t a, b;
                    split2(y[2 * (e & 1)] * up, y[2 * (e & 1) + 1] * up, a, b);
                    qh[k][e] = a;
                    lw[e] = b;
                }
                if (k < QR) qlo[k < QR ? k : 0] = lw;
                else ql[(k - QR) * 64] = lw;
            }
        }
        cs = fmaxf(cs, 1e-37f);
        // Q is here: no wait for it (and with it for the tile in flight) inside the loop
#pragma unroll
        for (int k = 0; k < (F32 ? KS : QR); k++) asm volatile("" : "+v"(qh[k]));
        if constexpr (F32)
#pragma unroll
            for (int k = 0; k < QR; k++) asm volatile("" : "+v"(qlo[k]));
    }

    f32x16 o[NO];
#pragma unroll
    for (int m = 0; m < NO; m++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[m][r] = 0.f;
    float m_ref = -0x1p127f, l = 0.f;   // reference maximum (log2 units, below any score) and the lane's part of the sum
    float v_ref = 0x1p-126f, v_inv = 0x1p126f;   // F32: power of two that V's factors are taken relative to, and one over it

    // lane's LDS byte offsets.  K row n, piece 2k + h; V transpose reads: rows 4h + (lane%16)/4 (+ 8, + 16 st),
    // dims 32m + 16((lane/16)%2) + 4(lane%4): piece 4m + 2((lane/16)%2) + (lane%4)/2, 8 bytes into it for odd lanes.  The
    // exclusive or does not mix with the constants added, so a base per distinct pattern is kept: swz(n) is K's; rows r and
    // r + 8 (r + 16 is r again) are V's.
    const int vrow = 4 * h + ((lane & 15) >> 2), vpiece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    // (opaque: kept as they are, so that what is added below is a constant of the read)
    // (the exclusive or stays within 16 pieces, 256 bytes: past them the patterns come again)
    constexpr int KP = KS < 8 ? KS : 8, VP = NO < 4 ? NO : 4;
    uint32_t koff[KP], voff[2][VP];
#pragma unroll
    for (int k = 0; k < KP; k++) koff[k] = opaque(lk0 + (KT * kg + n) * SH::STRIDE + 16 * ((2 * k + h) ^ SH::swz(n)));
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int m = 0; m < VP; m++)
            voff[e][m] = opaque(lv0 + (KT * kg + vrow + 8 * e) * SH::STRIDE + 16 * ((4 * m + vpiece) ^ SH::swz(vrow + 8 * e)) + 8 * (lane & 1));

    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    // ---- the tile loop ----
    // Operands are read ahead of their products; the scheduling barriers keep the compiler from pulling each read down to its
    // product, where the wave would wait for it.
    constexpr int NQ = NO * (NS / 8);   // products (triples of them, F32) of a tile with V; KS with K
    constexpr int RD = SH::RD;
    u32x4 kr[RD][NP], vr[RD][NP], qv[RD];
    auto read_k = [&](int k, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < NP; e++)
            kr[k % RD][e] = *(const lds_u32x4 *) (uintptr_t) (koff[k % KP] + k / KP * 256 + buf * SH::BUF + e * SH::PLANE);
        if (k >= QR) qv[k % RD] = ql[(k - QR) * 64];
    };
    auto read_v = [&](int q, int buf) __attribute__((always_inline)) {
        const int st = q / NO, m = q % NO;
#pragma unroll
        for (int e = 0; e < NP; e++) {
            const uint32_t off = buf * SH::BUF + e * SH::PLANE + 16 * st * SH::STRIDE + m / VP * 256;
            vr[q % RD][e] = __builtin_bit_cast(u32x4, lds_tr_b16x8_at(voff[0][m % VP] + off, voff[1][m % VP] + off));
        }
    };
    // Tile c0 of the workgroup, in buffer buf_; the wave's part of it begins at cw.  Into buffer `ahead` another is loaded
    // meanwhile: the one after next (NB = 3), or the next.
    auto tile = [&](int c0, auto buf_) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_)::value, ahead = (buf + NB - 1) % NB;
        if constexpr (!DMA) {
            load_rows(st, kb, p.k_stride, p.D, c0 + TT);
        } else {
            load_tile(c0 + (NB - 1) * TT, ahead);
            if (partial(c0)) {
                char *const at = lds_v + buf * SH::BUF + tid * 16;
                bool bad = false;
#pragma unroll
                for (int x = 0; x < SH::PPT; x++) bad |= any_bad<TY>(*(const u32x4 *) (at + x * SH::THREADS * 16));
                if (bad) {
                    for (int x = 0; x < SH::PPT; x++) {
                        Piece8<TY> v = {*(const u32x4 *) (at + x * SH::THREADS * 16)};
                        finite_piece<TY>(v);
                        *(u32x4 *) (at + x * SH::THREADS * 16) = v.a;
                    }
                    bad_v = 1;
                }
                __syncthreads();
            }
        }
        const int cw = c0 + KT * kg;
        float x[NS], cx = cs, ref;   // x times cx is the score in log2 units, against ref
        u32x4 pr[NP][NS / 8];
        auto weights = [&]() __attribute__((always_inline)) {
            // ---- scores ----
            f32x16 sc;
#pragma unroll
            for (int r = 0; r < 16; r++) sc[r] = 0.f;
#pragma unroll
            for (int k = 0; k < RD - 1; k++) read_k(k, buf);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                if (k + RD - 1 < KS) read_k(k + RD - 1, buf);
                sc = prompt_mfma<TY>(kr[k % RD][0], F32 || k < QR ? qh[F32 || k < QR ? k : 0] : qv[k % RD], sc);
                if constexpr (F32) {
                    sc = prompt_mfma<TY>(kr[k % RD][NP - 1], qh[k], sc);
                    sc = prompt_mfma<TY>(kr[k % RD][0], k < QR ? qlo[k < QR ? k : 0] : qv[k % RD], sc);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            // ---- softmax ----
#pragma unroll
            for (int j = 0; j < NS; j++) {
                x[j] = sc[j];
                if constexpr (F32) x[j] *= k_up[buf][KT * kg + 8 * (j / 4) + 4 * h + j % 4];
            }
            if (p.softcap > 0.f) {
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    if constexpr (F32) x[j] = tanhf(x[j] * cs);
                    else x[j] = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x[j] * (cs * (2.f * kLog2e))));
                }
                cx = p.softcap * kLog2e;
            }
            if (cw < w_lo_all || cw + KT > w_end_all) {   // wave-uniform
                const int a = lo - cw - 4 * h, b = end - cw - 4 * h;
#pragma unroll
                for (int j = 0; j < NS; j++) {
                    const int key = 8 * (j / 4) + j % 4;
                    x[j] = key >= a && key < b ? x[j] : -INFINITY;
                }
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
            ref = m_ref;
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
                    vf[j] = v_up[buf][KT * kg + 8 * (j / 4) + 4 * h + j % 4];
                    top = fmaxf(top, vf[j]);
                }
                if (__any(top > v_ref * 64.f)) {   // (of all the tile's tokens: seldom)
                    top = 0.f;
#pragma unroll
                    for (int j = 0; j < NS; j++) top = fmaxf(top, x[j] != 0.f ? vf[j] : 0.f);
                    top = max_halves(top);
                    const float vn = top > v_ref * 64.f ? top : v_ref;
                    const float beta = v_ref * (1.f / vn);   // (powers of two)
                    v_ref = vn;
                    v_inv = 1.f / vn;
#pragma unroll
                    for (int m = 0; m < NO; m++)
#pragma unroll
                        for (int r = 0; r < 16; r++) o[m][r] *= beta;
                }
#pragma unroll
                for (int st = 0; st < NS / 8; st++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        // (a token of no weight may have any factor: kept finite)
                        const int j = 8 * st + 2 * e;
                        uint32_t a, b;
                        split2(x[j] * fminf(vf[j] * v_inv, 0x1p100f), x[j + 1] * fminf(vf[j + 1] * v_inv, 0x1p100f), a, b);
                        pr[0][st][e] = a;
                        pr[NP - 1][st][e] = b;
                    }
            }
        };
        auto products = [&]() __attribute__((always_inline)) {
            // ---- O^T += V^T P^T, the next 16 tokens' probabilities beside the products of 16 ----
            // (the sum is of the rounded probabilities, as the products are)
            auto weigh = [&](int st, int e) __attribute__((always_inline)) {   // pair e of the 16 tokens st
                x[8 * st + 2 * e] = __builtin_amdgcn_exp2f(fmaf(x[8 * st + 2 * e], cx, -ref));
                x[8 * st + 2 * e + 1] = __builtin_amdgcn_exp2f(fmaf(x[8 * st + 2 * e + 1], cx, -ref));
                pr[0][st][e] = pack2<TY>(x[8 * st + 2 * e], x[8 * st + 2 * e + 1]);
                l = sum2<TY>(pr[0][st][e], l);
            };
#pragma unroll
            for (int q = 0; q < RD - 1; q++) read_v(q, buf);
            if constexpr (!F32) {
#pragma unroll
                for (int e = 0; e < 4; e++) weigh(0, e);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                const int st = q / NO, m = q % NO;
                if (q + RD - 1 < NQ) read_v(q + RD - 1, buf);
                o[m] = prompt_mfma<TY>(vr[q % RD][0], pr[0][st], o[m]);
                if constexpr (F32) {
                    o[m] = prompt_mfma<TY>(vr[q % RD][NP - 1], pr[0][st], o[m]);
                    o[m] = prompt_mfma<TY>(vr[q % RD][0], pr[NP - 1][st], o[m]);
                } else if (st + 1 < NS / 8) {
#pragma unroll
                    for (int e = 4 * m / NO; e < 4 * (m + 1) / NO; e++) weigh(st + 1, e);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const bool sees = cw < w_end && cw + KT > w_lo;   // wave-uniform: some row sees some of it
        if constexpr (DMA) {
            if (sees) {
                weights();
                products();
            }
            wait_tile(NB == 3 && c0 + 2 * TT < g_end);
        } else {
            if (sees) weights();
            put_rows(st, lds_k + ahead * SH::BUF, k_up[ahead], c0 + TT, false);
            load_rows(st, vb, p.v_stride, p.Dv, c0 + TT);
            if (sees) products();
            put_rows(st, lds_v + ahead * SH::BUF, v_up[ahead], c0 + TT, true);
        }
        __syncthreads();
    };
    if constexpr (DMA) {
        wait_tile(NB == 3 && g_lo + TT < g_end);
    } else {
        put_rows(st0, lds_k, k_up[0], g_lo, false);
        put_rows(st, lds_v, v_up[0], g_lo, true);
    }
    __syncthreads();
    for (int c0 = g_lo; c0 < g_end; c0 += NB * TT) {
        tile(c0, std::integral_constant<int, 0>());
        if (c0 + TT >= g_end) break;
        tile(c0 + TT, std::integral_constant<int, 1>());
        if constexpr (NB == 3) {
            if (c0 + 2 * TT >= g_end) break;
            tile(c0 + 2 * TT, std::integral_constant<int, 2>());
        }
    }

    l += __shfl_xor(l, 32);
    // ---- KW > 1: the waves' results joined; each wave then has every KW-th 32 dims of its rows ----
    if constexpr (KW > 1) {
        float *const mine = (float *) lds + (wave * (NO * 16 + 2)) * 64 + lane;
        if constexpr (F32) {   // in units of their own rows' V
#pragma unroll
            for (int m = 0; m < NO; m++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[m][r] *= v_ref;
        }
        // (the loop ended with a barrier: the tiles are read)
#pragma unroll
        for (int m = 0; m < NO; m++)
#pragma unroll
            for (int r = 0; r < 16; r++) mine[(m * 16 + r) * 64] = o[m][r];
        mine[NO * 16 * 64] = m_ref;
        mine[(NO * 16 + 1) * 64] = l;
        __syncthreads();
        const float *const first = (const float *) lds + (wave / KW * KW * (NO * 16 + 2)) * 64 + lane;
        float f[KW], top = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int w = 0; w < KW; w++) top = fmaxf(top, first[(w * (NO * 16 + 2) + NO * 16) * 64]);
#pragma unroll
        for (int w = 0; w < KW; w++) {
            f[w] = __builtin_amdgcn_exp2f(first[(w * (NO * 16 + 2) + NO * 16) * 64] - top);
            l += f[w] * first[(w * (NO * 16 + 2) + NO * 16 + 1) * 64];
        }
#pragma unroll
        for (int m = 0; m < NO; m++) {
            if (m % KW != kg) continue;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < KW; w++) sum += f[w] * first[(w * (NO * 16 + 2) + m * 16 + r) * 64];
                o[m][r] = sum;
            }
        }
    }

    // ---- V's non-finite values, left out of the tiles, for the rows that see them ----
    // (each value by the one wave that stores its place)
    if (bad_v)
        for (int j = g_lo; j < min(g_end, L); j++) {
            if (!partial(j / TT * TT)) continue;
            const T *vr = vb + (int64_t) j * p.v_stride;
            const bool sees = j >= lo && j < end;
            int Dv = p.Dv;   // (opaque: a comparison per value held over the whole kernel would take all scalar registers)
            asm volatile("" : "+s"(Dv));
#pragma unroll
            for (int m = 0; m < NO; m++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    if (KW > 1 && m % KW != kg) continue;
                    const int d = 32 * m + 8 * (r / 4) + 4 * h + r % 4;
                    const float v = sees && d < Dv ? (float) vr[d] : 0.f;
                    o[m][r] += (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? v : 0.f;
                }
        }

    // ---- rows out ----
    float inv = l == 0.f ? 0.f : 1.f / l;
    if constexpr (F32 && KW == 1) inv *= v_ref;   // (an empty row: 0 * 2^-126)
    T *out = (T *) p.out + t * p.o_stride + (int64_t) head * p.Dv;
    if constexpr (VEC && KW == 1) {
        // Through the wave's part of LDS (the tiles are read: the loop ended with a barrier), so that a store writes whole
        // rows, 16 bytes a lane, instead of 4 values in each of 64 places.  128 bytes of the rows at a time.
        constexpr int ES = sizeof(T), MB = 4 / ES, RB = 128 + 16, LPR = 8, RPI = 64 / LPR;   // row pitch, lanes per row, rows per store
        static_assert(32 * RB * NW <= sizeof(lds), "the rows fit");
        char *const my = lds + wave * 32 * RB;
        const int last = min(31, rows - 1 - row0);
        // (a row's place: its own lane knows it)
        const int64_t place = t * p.o_stride + (int64_t) head * p.Dv;
#pragma unroll
        for (int m0 = 0; m0 < NO; m0 += MB) {
#pragma unroll
            for (int m = m0; m < (NO < m0 + MB ? NO : m0 + MB); m++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    char *at = my + n * RB + (32 * (m - m0) + 8 * b + 4 * h) * ES;
                    float y[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = o[m][4 * b + e] * inv;
                    if constexpr (F32) *(float4 *) at = make_float4(y[0], y[1], y[2], y[3]);
                    else *(u32x2 *) at = u32x2{pack2<TY>(y[0], y[1]), pack2<TY>(y[2], y[3])};
                }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int x = 0; x < 32 / RPI; x++) {
                const int r = x * RPI + lane / LPR, d = 32 * m0 + lane % LPR * (16 / ES);
                const int64_t to = __shfl(place, r);
                const u32x4 y = *(const u32x4 *) (my + r * RB + lane % LPR * 16);
                if (r <= last && d < p.Dv && d < 32 * NO) *(u32x4 *) ((T *) p.out + to + d) = y;
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    } else {
        if (!live) return;
#pragma unroll
        for (int m = 0; m < NO; m++)
#pragma unroll
            for (int b = 0; b < 4; b++) {
                if (KW > 1 && m % KW != kg) continue;
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
}

constexpr int64_t kPromptMaxBlocks = 1 << 22;   // of at most 512 threads: a launch holds below 2^32

// Row blocks of `rows` rows that the launch may have: at most one more than whole ones for each prompt.
inline int64_t prompt_blocks(const PromptParams &p, int rows) {
    const int64_t all = (int64_t) p.T * p.gqa, per = ((int64_t) p.max_q * p.gqa + rows - 1) / rows;
    return std::min(all / rows + p.S, per * p.S) * p.Hkv;
}

// All prompts of at most 64 tokens, two tiles.
inline bool prompt_short(const PromptParams &p) { return p.max_q <= 64 && p.T <= 64 * (int64_t) p.S; }

template <int TY, int DK, int DV, bool VEC, int KW, int NW>
static hipError_t launch_prompt_k(const PromptParams &p, hipStream_t stream) {
    const int64_t blocks = prompt_blocks(p, PromptShape<TY, DK, DV, VEC, KW, NW>::ROWS);
    hipLaunchKernelGGL((pa_prompt_kernel<TY, DK, DV, VEC, KW, NW>), dim3((unsigned) blocks), dim3(NW * 64), 0, stream, p);
    return hipGetLastError();
}

// KW4, KW2: whether waves may share rows by four, by two (LDS holds their tiles).
// They do in calls whose workgroups then still run at once, two on a CU (one at head
// size 256): one 512-token prompt, H32/Hkv8/D128 bf16, 13 us, 17 with KW = 1, by
// four at H14/Hkv2/D64 8, 9 with KW = 2 and 13 with KW = 1 (by four saves nothing
// from head size 80 on).  Not up to 64 tokens, where joining costs more than the
// second tile (one token 5.3 us, 6.0 with KW = 2; 16 prompts of 64 8 and 11).
// Longer causal prompts share by two up to twice that (three times at head size
// 64), since their last row blocks see the most tokens and are the call's critical
// path, the less the more tokens there are beside them: with more than two such
// prompts' up to 5/4 (twice).  Prompts of 900 and 300 tokens 20 us, 26 with KW = 1, one of
// 2048 48 and 54, at H20/Hkv20/D96 31 and 46, one of 4096 at H14/Hkv2/D64 48 and 71, 4 of
// 1000 19 and 23; slower beyond, for shorter ones and those that see all: one of
// 2600, D128, 77 and 74, 3 of 600 26 and 21, 4 of 512 25 and 21, one that sees all of 2048
// 83 and 73; D256, H16/Hkv8: one of 2048 70 and 90, 4 of 1000 89 and 56.
//
// NW8: whether workgroups have 8 waves (head size 256) where every CU then still
// has one (4 prompts of 1000 tokens, H16/Hkv8, 57 us, 61 with 4 waves; 2 images of
// 2048 123 and 178; below, one causal prompt of 2048 95 and 89) and the longest prompt
// has rows for more than 4 of them (64 prompts of 30 tokens 24 us, 21 with 4 waves).
template <int TY, int DK, int DV, bool KW4, bool KW2, bool NW8 = false>
static hipError_t launch_prompt_d(const PromptParams &p, bool vec, hipStream_t stream) {
    if (!vec) return launch_prompt_k<TY, DK, DV, false, 1, 4>(p, stream);
    if (!prompt_short(p)) {
        constexpr int at_once = (DK <= 128 ? 2 : 1) * kPromptCus;
        const bool critical = (p.causal || p.row_end) && p.max_q >= 600, few = p.T <= 2 * (int64_t) p.max_q;
        if constexpr (KW4)
            if (prompt_blocks(p, 32) <= at_once) return launch_prompt_k<TY, DK, DV, true, 4, 4>(p, stream);
        if constexpr (KW2)
            if (prompt_blocks(p, 64) <= at_once * (!critical ? 4 : DK <= 64 ? few ? 12 : 8 : few ? 8 : 5) / 4)
                return launch_prompt_k<TY, DK, DV, true, 2, 4>(p, stream);
    }
    if constexpr (NW8)
        if (prompt_blocks(p, 256) >= kPromptCus && (int64_t) p.max_q * p.gqa > 128)
            return launch_prompt_k<TY, DK, DV, true, 1, 8>(p, stream);
    return launch_prompt_k<TY, DK, DV, true, 1, 4>(p, stream);
}

// Rows of whole aligned pieces of 16 bytes.
template <int TY>
static bool prompt_vec(const PromptParams &p) {
    const int64_t es = TY == 0 ? 4 : 2;
    const uintptr_t al = (uintptr_t) p.q | (uintptr_t) p.k | (uintptr_t) p.v | (uintptr_t) p.out;
    // (a tile's rows are addressed by 32-bit offsets)
    if (std::max(p.k_stride, p.v_stride) > 1 << 22) return false;
    return al % 16 == 0 && ((p.q_stride | p.k_stride | p.v_stride | p.o_stride) * es) % 16 == 0 && p.D % 8 == 0 && p.Dv % 8 == 0;
}

}  // namespace iian_pa
