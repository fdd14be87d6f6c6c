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
// runs per thread, loaded together and summed, a wave scan over the threads and
// one over the waves, so a round covers 2048 runs and a request of 2000 takes
// one.  The prefixes go to LDS, where each of the share's tokens finds its run
// by a binary search.  Every share scans for itself: a request's runs are a few
// KB and stay in L2, while a scan in a launch of its own would cost the launch.
// Latency-bound: query_start_loc and span_off, then the runs, then the store.
constexpr int kRunsPer = 8;
constexpr int kRunsRound = 256 * kRunsPer;

struct RunExtent {
    int64_t tokens, advance;
    bool bad;
};

// Tokens and position advance of a run, each below 2^31 (a larger one is held
// at INT32_MAX: prefix sums of 2^31 runs stay within 64 bits).
__device__ __forceinline__ RunExtent run_extent(const int4 &r) {
    RunExtent e = {0, 0, false};
    const bool grid = r.y != 0 || r.z != 0;
    if (r.x < 0 || (grid && (r.y <= 0 || r.z <= 0))) {
        e.bad = true;
    } else if (!grid) {
        e.tokens = e.advance = r.x;
    } else if (r.x > 0) {
        const int64_t plane = min((int64_t) r.y * r.z, (int64_t) INT32_MAX);
        e.tokens = min(r.x * plane, (int64_t) INT32_MAX);
        const int64_t time = (int64_t) (r.x - 1) * max(r.w, 1) + 1;
        e.advance = min(max(time, (int64_t) max(r.y, r.z)), (int64_t) INT32_MAX);
        e.bad = r.w < 1 || r.x * plane > INT32_MAX || time > INT32_MAX;
    }
    return e;
}

__global__ __launch_bounds__(256) void pa_mrope_positions_kernel(MropePosParams p) {
    __shared__ int64_t wave_sum[2][4];
    // tokens and position before each run of the round, and after the last
    __shared__ int32_t tok[kRunsRound + 1], at[kRunsRound + 1];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int q0 = min(max(p.qsl[s], 0), p.T), q1 = min(max(p.qsl[s + 1], q0), p.T);
    const int nn = q1 - q0;
    // shares of whole waves
    const int64_t per = ((int64_t) nn + gridDim.y - 1) / gridDim.y + 63 & ~(int64_t) 63;
    const int i0 = (int) min(blockIdx.y * per, (int64_t) nn), i1 = (int) min(i0 + per, (int64_t) nn);
    const int f0 = p.span_off[s], f1 = p.span_off[s + 1];
    const int nc = p.num_computed[s];
    const int b0 = min(max(f0, 0), p.n_spans), b1 = min(max(f1, b0), p.n_spans);
    bool bad = nc < 0 || f0 != b0 || f1 != b1;
    const bool first = blockIdx.y == 0;   // flags each request once, whether it has new tokens or not
    if (i0 >= i1 && !first) return;
    const int64_t r0 = (int64_t) max(nc, 0) + i0, r1 = (int64_t) max(nc, 0) + i1;   // the share's tokens of the request
    int64_t tok0 = 0, at0 = 0;   // before the round
    int64_t done = r0;           // tokens written so far
    auto put = [&](int64_t r, int64_t pt, int64_t ph, int64_t pw, int64_t end) {
        const int t = q0 + (int) (r - max(nc, 0));
        bad |= pt > INT32_MAX || ph > INT32_MAX || pw > INT32_MAX || end > INT32_MAX;
        p.pos[t] = (int32_t) min(pt, (int64_t) INT32_MAX);
        p.pos[(int64_t) p.T + t] = (int32_t) min(ph, (int64_t) INT32_MAX);
        p.pos[2 * (int64_t) p.T + t] = (int32_t) min(pw, (int64_t) INT32_MAX);
        if (p.row_end) p.row_end[t] = (int32_t) min(end, (int64_t) INT32_MAX);
    };
    for (int b = b0; b < b1 && done < r1; b += kRunsRound) {
        const int n = min(kRunsRound, b1 - b);
        int4 run[kRunsPer];
        int64_t ts = 0, as = 0;
#pragma unroll
        for (int k = 0; k < kRunsPer; k++) {
            const int j = tid * kRunsPer + k;
            run[k] = j < n ? p.spans[b + j] : make_int4(0, 0, 0, 1);
        }
#pragma unroll
        for (int k = 0; k < kRunsPer; k++) {
            const RunExtent e = run_extent(run[k]);
            bad |= e.bad;
            ts += e.tokens;
            as += e.advance;
        }
        int64_t tp = ts, ap = as;   // inclusive scans over the wave's lanes
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t x = __shfl_up(tp, o), y = __shfl_up(ap, o);
            if (lane >= o) {
                tp += x;
                ap += y;
            }
        }
        if (lane == 63) {
            wave_sum[0][wave] = tp;
            wave_sum[1][wave] = ap;
        }
        __syncthreads();
        int64_t tw = tok0, aw = at0;
        for (int w = 0; w < 4; w++) {
            if (w < wave) {
                tw += wave_sum[0][w];
                aw += wave_sum[1][w];
            }
            tok0 += wave_sum[0][w];
            at0 += wave_sum[1][w];
        }
        tw += tp - ts;
        aw += ap - as;
#pragma unroll
        for (int k = 0; k < kRunsPer; k++) {
            tok[tid * kRunsPer + k] = (int32_t) min(tw, (int64_t) INT32_MAX);
            at[tid * kRunsPer + k] = (int32_t) min(aw, (int64_t) INT32_MAX);
            const RunExtent e = run_extent(run[k]);
            tw += e.tokens;
            aw += e.advance;
        }
        if (tid == 255) {
            tok[kRunsRound] = (int32_t) min(tw, (int64_t) INT32_MAX);
            at[kRunsRound] = (int32_t) min(aw, (int64_t) INT32_MAX);
        }
        __syncthreads();
        const int64_t stop = min(r1, tok0);   // the round's runs hold tokens up to tok0
        for (int64_t r = done + tid; r < stop; r += 256) {
            // the last run that starts at or before token r: it holds r, since the
            // runs of no tokens behind it start where the next one does
            int lo = 0, hi = kRunsRound;
            while (hi - lo > 1) {
                const int m = (lo + hi) >> 1;
                if (tok[m] <= r) lo = m;
                else hi = m;
            }
            const int4 g = p.spans[b + min(lo, n - 1)];
            const uint32_t i = (uint32_t) (r - tok[lo]);
            const int64_t base = at[lo];
            if (g.y > 0 && g.z > 0) {
                const uint32_t w = (uint32_t) g.z, h = (uint32_t) g.y, row = i / w, it = row / h;
                put(r, base + (int64_t) it * max(g.w, 1), base + (row - it * h), base + (i - row * w),
                    p.grid_full ? (int64_t) tok[lo + 1] : r + 1);
            } else {
                put(r, base + i, base + i, base + i, r + 1);
            }
        }
        done = max(done, stop);
        __syncthreads();   // the prefixes are rewritten by the next round
    }
    for (int64_t r = done + tid; r < r1; r += 256) put(r, at0 + (r - tok0), at0 + (r - tok0), at0 + (r - tok0), r + 1);
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
