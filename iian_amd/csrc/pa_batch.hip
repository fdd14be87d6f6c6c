// pa_batch.hip - device-side batch metadata of one engine step.
//
// Engine::step builds its UBatch on the host by expanding every scheduled
// request's block table into absolute cells, one entry per context token
// (src/iian/engine.cpp:491-535; cell_of, include/iian/kv_cache.h:135-137):
// O(sum of context lengths) host work and transfer per step.  This kernel
// builds the arrays iian_pa_attention and iian_pa_kv_write read straight from
// the per-request state the scheduler already holds - the block ids of each
// request (KVRequestState::block_ids, kv_cache.h:93-97), its computed-token
// count and its new-token count - so the host uploads sum(blocks) + 3S
// integers instead of sum(context) cells.
//
// One workgroup per request s:
//   query_start_loc[s]  prefix sum of the new-token counts before s (each
//                       workgroup sums them itself: no second pass)
//   seq_lens[s]         num_computed + n_new
//   block_tables[s][b]  the request's block ids for the blocks its context
//                       uses, 0 after them (the padding PagedBatch uses)
//   pos[t], slots[t]    for its new tokens: pos = num_computed + i, slot =
//                       cell_of(pos) (engine.cpp:508-513)
#include "pa_common.h"
#include "pa_launch.h"

#include <algorithm>

namespace iian_pa {

__global__ __launch_bounds__(256) void pa_build_batch_kernel(BatchParams p) {
    __shared__ int part[4];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int acc = 0;
    for (int i = tid; i < s; i += 256) acc += max(p.n_new[i], 0);
    acc = wave_sum_i(acc);
    if (lane == 0) part[wave] = acc;
    __syncthreads();
    const int q0 = part[0] + part[1] + part[2] + part[3];

    const int nc = p.num_computed[s], nn = p.n_new[s];
    const int off = p.block_off[s], nb = p.block_off[s + 1] - off;
    bool bad = nc < 0 || nn < 0 || nb < 0;
    const int L = max(nc, 0) + max(nn, 0);
    const int used = (L + p.block_size - 1) / p.block_size;
    // the request's blocks must cover its context and fit the table row
    bad |= used > nb || used > p.max_blocks;
    if (tid == 0) {
        p.seq_lens[s] = L;
        p.qsl[s] = q0;
        if (s == p.S - 1) {
            p.qsl[p.S] = q0 + max(nn, 0);
            bad |= q0 + max(nn, 0) != p.T;
        }
        if (bad && p.err) atomicOr(p.err, 8);
    }
    const int have = min(used, max(nb, 0));
    for (int b = tid; b < p.max_blocks; b += 256) {
        int32_t id = 0;
        if (b < have) {
            id = p.block_ids[off + b];
            if ((uint32_t) id >= (uint32_t) p.num_blocks && p.err) atomicOr(p.err, 2);
        }
        p.block_tables[(int64_t) s * p.max_blocks + b] = id;
    }
    for (int i = tid; i < nn; i += 256) {
        const int t = q0 + i;
        if (t >= p.T) {   // more new tokens than the caller's n_tokens (flagged above)
            if (p.err) atomicOr(p.err, 8);
            break;
        }
        const int ps = max(nc, 0) + i;
        const int b = ps / p.block_size;
        int64_t slot = -1;   // no block for this token: iian_pa_kv_write skips and flags slot -1
        if (b < max(nb, 0)) slot = (int64_t) p.block_ids[off + b] * p.block_size + (ps - b * p.block_size);
        else if (p.err) atomicOr(p.err, 1);
        p.pos[t] = ps;
        p.slots[t] = slot;
    }
    // Tokens past the last request's (the counts sum to less than n_tokens,
    // flagged above): slot -1, so a KV write of n_tokens rows skips them
    // instead of writing to whatever the buffers held.
    if (s == p.S - 1)
        for (int t = q0 + max(nn, 0) + tid; t < p.T; t += 256) {
            p.pos[t] = 0;
            p.slots[t] = -1;
        }
}

// Sliding-window block freeing (the reference's planned "free out-of-window
// blocks", docs/ROADMAP.md:33).  On a layer with window n_swa, a query at
// position q sees cells c > q - n_swa (src/iian/paged_attn.cpp:124), and the
// kernels start reading at that bound rounded down to a multiple of kTile.
// A sequence's later steps only have larger positions, so every block that
// ends at or before align_down(min_pos - n_swa + 1, kTile) is never read again
// by any kernel of this library: n_free[s] counts those leading blocks, and
// their table entries may be overwritten (with -1 here) and the blocks
// reused.  One wave per sequence.
__global__ __launch_bounds__(256) void pa_swa_free_kernel(const int32_t *__restrict__ qsl,
                                                          const int32_t *__restrict__ pos, int32_t S, int32_t T,
                                                          int32_t n_swa, int32_t block_size, int32_t *n_free,
                                                          int32_t *block_tables, int32_t max_blocks) {
    const int s = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (s >= S) return;
    const int q0 = min(max(qsl[s], 0), T), q1 = min(max(qsl[s + 1], q0), T);
    int mn = INT32_MAX;
    for (int t = q0 + lane; t < q1; t += 64) mn = min(mn, pos[t]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mn = min(mn, __shfl_xor(mn, o));
    int nf = 0;
    if (q1 > q0 && n_swa > 0) nf = (max(0, mn - n_swa + 1) & ~(kTile - 1)) / block_size;
    if (lane == 0) n_free[s] = nf;
    if (block_tables)
        for (int b = lane; b < min(nf, max_blocks); b += 64) block_tables[(int64_t) s * max_blocks + b] = -1;
}

// Positions on three axes of a step's new tokens (iian_pa_mrope_positions).
//
// Workgroup (s, c) takes the c-th share of request s' new tokens.  It needs the
// token and position prefix sums over the request's runs up to them: kRunsPer
// runs per thread, loaded together and summed, a scan over the wave's lanes by
// lane permutes and one over the waves, so a round covers 2048 runs and a request of
// 2000 takes one.  The prefixes and the runs go to LDS, where each of the share's
// tokens finds its run by a binary search.  Every share scans for itself: a
// request's runs are a few KB and stay in L2, while a scan in a launch of its
// own would cost the launch.  Sums are held at INT32_MAX (adding and holding is
// associative), so 32 bits suffice.  Latency-bound: query_start_loc and
// span_off, then the runs, the search, the stores (kernel trace: 48 decoding
// requests of 12 runs 4.6 us, 131,072 tokens of 4 requests of 2000 runs 9.0; with
// 64-bit sums and the run read again from memory 6.4 and 10.1).
constexpr int kRunsPer = 8;
constexpr int kRunsRound = 256 * kRunsPer;
constexpr uint32_t kMost = INT32_MAX;

struct RunExtent {
    uint32_t tokens, advance;   // at most kMost
    bool bad;
};

__device__ __forceinline__ uint32_t hold(uint64_t v) { return (uint32_t) min(v, (uint64_t) kMost); }
__device__ __forceinline__ uint32_t sum_held(uint32_t a, uint32_t b) { return min(a + b, kMost); }   // (both at most kMost)

// Tokens and position advance of a run.
__device__ __forceinline__ RunExtent run_extent(const int4 &r) {
    RunExtent e = {0, 0, false};
    const bool grid = r.y != 0 || r.z != 0;
    if (r.x < 0 || (grid && (r.y <= 0 || r.z <= 0))) {
        e.bad = true;
    } else if (!grid) {
        e.tokens = e.advance = r.x;
    } else if (r.x > 0) {
        const uint64_t tokens = (uint64_t) r.x * hold((uint64_t) (uint32_t) r.y * (uint32_t) r.z);
        const uint64_t time = (uint64_t) (r.x - 1) * (uint32_t) max(r.w, 1) + 1;
        e.tokens = hold(tokens);
        e.advance = max(hold(time), (uint32_t) max(r.y, r.z));
        e.bad = r.w < 1 || tokens > kMost || time > kMost;
    }
    return e;
}

// Inclusive held sums over the wave's lanes.
__device__ __forceinline__ uint32_t scan_held(uint32_t v) {
    v = sum_held(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));    // row_shr 1, 2, 4, 8
    v = sum_held(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));
    v = sum_held(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));
    v = sum_held(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));
    v = sum_held(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));   // row_bcast 15 into rows 1 and 3
    v = sum_held(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));   // row_bcast 31 into rows 2 and 3
    return v;
}

__global__ __launch_bounds__(256) void pa_mrope_positions_kernel(MropePosParams p) {
    __shared__ uint32_t wave_sum[2][4];
    // of the round's runs: tokens before each, and behind the last; position before it, h, w (0 for text) and step
    __shared__ uint32_t tok[kRunsRound + 1];
    __shared__ __attribute__((aligned(16))) int4 info[kRunsRound];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int f0 = p.span_off[s], f1 = p.span_off[s + 1];
    const int nc = p.num_computed[s];
    const int q0 = min(max(p.qsl[s], 0), p.T), q1 = min(max(p.qsl[s + 1], q0), p.T);
    const int nn = q1 - q0;
    // shares of whole waves
    const int64_t per = ((int64_t) nn + gridDim.y - 1) / gridDim.y + 63 & ~(int64_t) 63;
    const int i0 = (int) min(blockIdx.y * per, (int64_t) nn), i1 = (int) min(i0 + per, (int64_t) nn);
    const int b0 = min(max(f0, 0), p.n_spans), b1 = min(max(f1, b0), p.n_spans);
    bool bad = nc < 0 || f0 != b0 || f1 != b1;
    if (i0 >= i1 && blockIdx.y != 0) return;   // (the first share flags a request, whether it has new tokens or not)
    const uint32_t r0 = (uint32_t) max(nc, 0) + i0, r1 = (uint32_t) max(nc, 0) + i1;   // the share's tokens of the request
    uint32_t tok0 = 0, at0 = 0;   // before the round
    uint32_t done = r0;           // tokens written so far
    auto put = [&](uint32_t r, uint64_t pt, uint64_t ph, uint64_t pw, uint64_t end) {
        const int t = q0 + (int) (r - max(nc, 0));
        bad |= max(max(pt, ph), max(pw, end)) > kMost;
        p.pos[t] = (int32_t) hold(pt);
        p.pos[(int64_t) p.T + t] = (int32_t) hold(ph);
        p.pos[2 * (int64_t) p.T + t] = (int32_t) hold(pw);
        if (p.row_end) p.row_end[t] = (int32_t) hold(end);
    };
    for (int b = b0; b < b1 && done < r1; b += kRunsRound) {
        const int n = min(kRunsRound, b1 - b);
        int4 run[kRunsPer];
        RunExtent e[kRunsPer];
        uint32_t ts = 0, as = 0;
#pragma unroll
        for (int k = 0; k < kRunsPer; k++) {
            const int j = tid * kRunsPer + k;
            run[k] = j < n ? p.spans[b + j] : make_int4(0, 0, 0, 1);
        }
#pragma unroll
        for (int k = 0; k < kRunsPer; k++) {
            e[k] = run_extent(run[k]);
            bad |= e[k].bad;
            ts = sum_held(ts, e[k].tokens);
            as = sum_held(as, e[k].advance);
        }
        const uint32_t tp = scan_held(ts), ap = scan_held(as);
        if (lane == 63) {
            wave_sum[0][wave] = tp;
            wave_sum[1][wave] = ap;
        }
        // (held sums do not subtract: what is before the lane is the lane's below)
        uint32_t tw = __shfl_up(tp, 1), aw = __shfl_up(ap, 1);
        if (lane == 0) tw = aw = 0;
        __syncthreads();
        uint32_t tb = tok0, ab = at0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            if (w < wave) {
                tb = sum_held(tb, wave_sum[0][w]);
                ab = sum_held(ab, wave_sum[1][w]);
            }
            tok0 = sum_held(tok0, wave_sum[0][w]);
            at0 = sum_held(at0, wave_sum[1][w]);
        }
        tw = sum_held(tw, tb);
        aw = sum_held(aw, ab);
        if (tid * kRunsPer < n) {
#pragma unroll
            for (int k = 0; k < kRunsPer; k++) {
                tok[tid * kRunsPer + k] = tw;
                info[tid * kRunsPer + k] = make_int4((int) aw, run[k].y, run[k].y > 0 ? run[k].z : 0, max(run[k].w, 1));
                tw = sum_held(tw, e[k].tokens);
                aw = sum_held(aw, e[k].advance);
            }
        }
        if (tid == 0) tok[n] = tok0;
        __syncthreads();
        const uint32_t stop = min(r1, tok0);   // the round's runs hold tokens up to tok0
        for (uint32_t r = done + tid; r < stop; r += 256) {
            // the last run that starts at or before token r: it holds r, since the
            // runs of no tokens behind it start where the next one does
            int lo = 0, hi = n;
            while (hi - lo > 1) {
                const int m = (lo + hi) >> 1;
                if (tok[m] <= r) lo = m;
                else hi = m;
            }
            const int4 g = info[lo];
            const uint32_t i = r - tok[lo];
            const uint64_t base = (uint32_t) g.x;
            if (g.z > 0) {
                const uint32_t w = (uint32_t) g.z, h = (uint32_t) g.y, row = i / w, it = row / h;
                put(r, base + (uint64_t) it * (uint32_t) g.w, base + (row - it * h), base + (i - row * w),
                    p.grid_full ? (uint64_t) tok[lo + 1] : (uint64_t) r + 1);
            } else {
                put(r, base + i, base + i, base + i, (uint64_t) r + 1);
            }
        }
        done = max(done, stop);
        __syncthreads();   // the prefixes are rewritten by the next round
    }
    for (uint32_t r = done + tid; r < r1; r += 256) {
        const uint64_t at = (uint64_t) at0 + (r - tok0);
        put(r, at, at, at, (uint64_t) r + 1);
    }
    if (bad && p.err) atomicOr(p.err, 8);
}

hipError_t launch_mrope_positions(const MropePosParams &p, hipStream_t stream) {
    // Shares per request: one per 512 tokens of the step, up to 64 (a single
    // request may hold them all); a share of no tokens ends at once.
    const int shares = std::min(64, std::max(1, (p.T + 511) / 512));
    hipLaunchKernelGGL(pa_mrope_positions_kernel, dim3(p.S, shares), dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_swa_free(const int32_t *qsl, const int32_t *pos, int32_t S, int32_t T, int32_t n_swa,
                           int32_t block_size, int32_t *n_free, int32_t *block_tables, int32_t max_blocks,
                           hipStream_t stream) {
    hipLaunchKernelGGL(pa_swa_free_kernel, dim3((S + 3) / 4), dim3(256), 0, stream, qsl, pos, S, T, n_swa, block_size,
                       n_free, block_tables, max_blocks);
    return hipGetLastError();
}

hipError_t launch_build_batch(const BatchParams &p, hipStream_t stream) {
    hipLaunchKernelGGL(pa_build_batch_kernel, dim3(p.S), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace iian_pa
