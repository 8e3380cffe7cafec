// The pass plan of the paged cache, built on the GPU from the sequences' lengths: page allotment,
// slot map, positions, and the work lists of the append and attention kernels.
//
// One workgroup: prefix sums over the sequences (new tokens, allotted and released pages, touched pages,
// row blocks) stay in LDS, then every list is written by all threads, each entry finding its sequence
// by binary search in the sums. No other workgroup takes part, so there is nothing to wait for
// across the GPU, and state may be updated in place.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8_params.h"

namespace clef_hip {
namespace kv8 {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64, kPlanSums = 5;

// Exclusive prefix sums of N values per thread over the workgroup; total[] gets the sums. Two barriers.
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*waves)[N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int own[N];
#pragma unroll
    for (int i = 0; i < N; i++) own[i] = v[i];
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int up = __shfl_up(v[i], d);
            if (lane >= d) v[i] += up;
        }
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; i++) waves[wave][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        int before = 0, all = 0;
        for (int w = 0; w < kPlanWaves; w++) {
            const int s = waves[w][i];
            before += w < wave ? s : 0;
            all += s;
        }
        v[i] += before - own[i];
        total[i] = all;
    }
    __syncthreads();
}

// The last r with sums[r] <= j (sums[0] = 0, n entries before the total).
__device__ __forceinline__ int find(const int *sums, int n, int j) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= j) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(kPlanThreads) void kv8_plan_kernel(PlanParams p) {
    __shared__ int cu[kPlanSums][kMaxSeq + 1], len[kMaxSeq], held[kMaxSeq], waves[kPlanWaves][kPlanSums], bad;
    int *const cu_q = cu[0], *const cu_add = cu[1], *const cu_rel = cu[2], *const cu_app = cu[3], *const cu_blk = cu[4];
    const int tid = threadIdx.x, n = p.n_seq;
    const int n_free = p.state[0];
    int status = (unsigned)n_free > (unsigned)p.n_pages ? CLEF_HIP_KV8_BAD_STATE : 0;
    int base[kPlanSums] = {0, 0, 0, 0, 0};
    if (tid == 0) bad = 0;   // the scans' barriers come before its first use
    for (int r0 = 0; r0 < n; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int v[kPlanSums] = {0, 0, 0, 0, 0}, total[kPlanSums];
        if (r < n) {
            int L = p.state[2 + 2 * r], h = p.state[3 + 2 * r], q = p.new_lens[r];
            if (h < 0 || h > p.max_pages || L < 0 || (long)L > (long)h * PAGE) {
                status |= CLEF_HIP_KV8_BAD_STATE;
                L = h = 0;
            }
            if (q < 0) v[2] = h;
            else if (q > p.T) status |= CLEF_HIP_KV8_ROWS;
            else if (q > 0) {
                const int need = (L + q + PAGE - 1) / PAGE;
                if (need > p.max_pages) status |= CLEF_HIP_KV8_TOO_LONG;
                v[0] = q;
                v[1] = max(need - h, 0);
                v[3] = need - L / PAGE;
                v[4] = (q * p.group + p.l.bm - 1) / p.l.bm;
            }
            len[r] = L;
            held[r] = h;
        }
        block_scan(v, total, waves);
#pragma unroll
        for (int i = 0; i < kPlanSums; i++) {
            if (r < n) cu[i][r] = base[i] + v[i];
            base[i] += total[i];
        }
    }
    if (tid < kPlanSums) cu[tid][n] = base[tid];
    const int n_tok = base[0], n_add = base[1], n_rel = base[2], n_app = base[3], n_blk = base[4];
    if (n_tok > p.T) status |= CLEF_HIP_KV8_ROWS;
    if (n_free + n_rel > p.n_pages) status |= CLEF_HIP_KV8_BAD_STATE;
    if (n_add > n_free + n_rel) status |= CLEF_HIP_KV8_NO_PAGES;
    if (status) atomicOr(&bad, status);
    __syncthreads();
    status = bad;
    // every page that changes hands is looked at before anything is written
    auto released = [&](int j) {
        const int r = find(cu_rel, n, j);
        return p.tables[(size_t)r * p.max_pages + j - cu_rel[r]];
    };
    if (!status) {
        for (int j = tid; j < n_rel; j += kPlanThreads)
            if ((unsigned)released(j) >= (unsigned)p.n_pages) atomicOr(&bad, CLEF_HIP_KV8_BAD_STATE);
        for (int j = n_rel + tid; j < n_add; j += kPlanThreads)
            if ((unsigned)p.free_pages[n_free + n_rel - 1 - j] >= (unsigned)p.n_pages) atomicOr(&bad, CLEF_HIP_KV8_BAD_STATE);
        __syncthreads();
        status = bad;
    }
    const bool good = status == 0;
    if (good) {
        // released pages go on top of the stack, then the allotted ones come off it
        for (int j = tid; j < n_rel; j += kPlanThreads) p.free_pages[n_free + j] = released(j);
        __threadfence_block();
        __syncthreads();
        for (int j = tid; j < n_add; j += kPlanThreads) {
            const int r = find(cu_add, n, j);
            p.tables[(size_t)r * p.max_pages + held[r] + j - cu_add[r]] = p.free_pages[n_free + n_rel - 1 - j];
        }
        __threadfence_block();
        __syncthreads();
    }
    for (int r = tid; r < n; r += kPlanThreads) {
        const bool gone = cu_rel[r + 1] > cu_rel[r] || p.new_lens[r] < 0;
        const int L = len[r], h = held[r];
        p.state_out[2 + 2 * r] = !good ? p.state[2 + 2 * r] : gone ? 0 : L + cu_q[r + 1] - cu_q[r];
        p.state_out[3 + 2 * r] = !good ? p.state[3 + 2 * r] : gone ? 0 : h + cu_add[r + 1] - cu_add[r];
        p.cu_q[r] = good ? cu_q[r] : 0;
    }
    // slot and position of each row; rows behind the last sequence have none
    int2 *const tok = (int2 *)(p.work + p.l.tok);
    for (int i = tid; i < p.T; i += kPlanThreads) {
        int slot = -1, pos = 0;
        int2 where = {0, 0};
        if (good && i < n_tok) {
            const int r = find(cu_q, n, i), at = len[r] + i - cu_q[r];
            const int page = p.tables[(size_t)r * p.max_pages + at / PAGE];
            if ((unsigned)page < (unsigned)p.n_pages) slot = page * PAGE + at % PAGE;
            pos = at + (p.pos_off ? p.pos_off[r] : 0);
            where = make_int2(cu_blk[r], i - cu_q[r]);
        }
        p.slots[i] = slot;
        tok[i] = where;
        if (p.pos3) {
            p.pos3[3 * (size_t)i] = pos;
            p.pos3[3 * (size_t)i + 1] = pos;
            p.pos3[3 * (size_t)i + 2] = pos;
        }
    }
    if (good) {
        int4 *const app = (int4 *)(p.work + p.l.app);
        for (int j = tid; j < n_app; j += kPlanThreads) {
            const int r = find(cu_app, n, j), L = len[r], q = cu_q[r + 1] - cu_q[r];
            const int pg = L / PAGE + j - cu_app[r], lo = max(L, pg * PAGE), hi = min(L + q, (pg + 1) * PAGE);
            app[j] = make_int4(p.tables[(size_t)r * p.max_pages + pg], cu_q[r] + lo - L, (lo - pg * PAGE) | (hi - lo) << 8, cu_q[r]);
        }
    }
    // blocks, in two rounds: the pages of all of them set the chunk, then each block's items are placed
    auto block = [&](int b, int &r, int &row0, int &rows) {
        r = find(cu_blk, n, b);
        row0 = (b - cu_blk[r]) * p.l.bm;
        const int q = cu_q[r + 1] - cu_q[r];
        rows = min(p.l.bm, q * p.group - row0);
        return (len[r] + (row0 + rows - 1) / p.group) / PAGE + 1;   // pages up to its last token's own key
    };
    int n_items = 0, n_slots = 0;
    if (good && n_blk) {
        int r, row0, rows;
        long mine = 0;
        for (int b = tid; b < n_blk; b += kPlanThreads) mine += block(b, r, row0, rows);
        // pages can pass 2^31 over all blocks: the sum is kept in units of 2^8 pages, rounded up
        int v[1] = {(int)((mine + 255) >> 8)}, total[1];
        const bool small = !__syncthreads_or(mine >= (1 << 18));
        if (small) v[0] = (int)mine;
        block_scan(v, total, (int(*)[1])waves);
        const long W = small ? (long)total[0] : (long)total[0] << 8;
        int C = (int)max((long)p.l.least, (W + p.l.budget - 1) / p.l.budget);
        // a block below 1.5 chunks stays whole, others are cut into the nearest number of pieces
        auto pieces = [&](int pages) { return max(1, (2 * pages + C) / (2 * C)); };
        // few blocks: the chunk grows until the items fit the budget, which is one round of workgroups
        for (int again = 0; again < 4 && 2 * n_blk <= p.l.budget; again++) {
            int c[1] = {0}, all[1];
            if (tid < n_blk) c[0] = pieces(block(tid, r, row0, rows));
            block_scan(c, all, (int(*)[1])waves);
            if (all[0] <= p.l.budget) break;
            C = max(C + 1, (int)((long)C * all[0] / p.l.budget));
        }
        int at = 0, at_slot = 0;
        for (int b0 = 0; b0 < n_blk; b0 += kPlanThreads) {
            const int b = b0 + tid;
            int pages = 0, c[2] = {0, 0}, sum[2];
            if (b < n_blk) {
                pages = block(b, r, row0, rows);
                c[0] = pieces(pages);
                c[1] = c[0] > 1 ? c[0] : 0;
            }
            const int items = c[0], cut = c[1];
            block_scan(c, sum, (int(*)[2])waves);
            if (b < n_blk) {
                const int first = at + c[0], slot = at_slot + c[1], q0 = cu_q[r], q = cu_q[r + 1] - q0;
                ((int4 *)(p.work + p.l.blk))[b] = make_int4(first, items, row0, slot);
                int4 *const it = (int4 *)(p.work + p.l.items);
                for (int k = 0; k < items; k++) {   // the pages split evenly over the items
                    const int pg0 = (int)((long)pages * k / items), pg1 = (int)((long)pages * (k + 1) / items);
                    it[2 * (first + k)] = make_int4(r, q0, len[r], len[r] + q);
                    it[2 * (first + k) + 1] = make_int4(row0, rows | (cut ? slot + k + 1 : 0) << 8, pg0, pg1);
                }
            }
            at += sum[0];
            at_slot += sum[1];
        }
        n_items = at;
        n_slots = at_slot;
    }
    if (tid == 0) {
        p.cu_q[n] = good ? n_tok : 0;
        p.state_out[0] = good ? n_free + n_rel - n_add : n_free;
        p.state_out[1] = status;
        int32_t *h = p.work;
        h[H_MAGIC] = kPlanMagic;
        h[H_SEQ] = n;
        h[H_ROWS] = p.T;
        h[H_GROUP] = p.group;
        h[H_BM] = p.l.bm;
        h[H_STATUS] = status;
        h[H_TOKENS] = good ? n_tok : 0;
        h[H_APPEND] = good ? n_app : 0;
        h[H_ITEMS] = n_items;
        h[H_BLOCKS] = good ? n_blk : 0;
        h[H_SPLIT] = n_slots;
    }
}

}  // namespace kv8
}  // namespace clef_hip
