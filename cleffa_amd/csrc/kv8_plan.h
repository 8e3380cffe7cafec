// The pass plan of the paged cache, built on the GPU from the sequences' lengths: page allotment,
// slot map, positions, and the work lists of the append and attention kernels.
//
// One workgroup: prefix sums over the sequences (new tokens, allotted and released pages, touched pages,
// row blocks) stay in LDS, then every list is written by all threads, each entry finding its sequence
// by binary search in the sums. No other workgroup takes part, so there is nothing to wait for
// across the GPU, and state may be updated in place. Bound by latency: the pages that sequences take are read
// into LDS (and looked at) before anything is written, so that after the one barrier behind that no list waits
// for another's stores; a wave's part of a sum is VALU only (DPP).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8_params.h"

namespace clef_hip {
namespace kv8 {

constexpr int kPlanSums = 5;
constexpr int kMaxFresh = kMaxRows / PAGE + 1 + kMaxSeq;   // pages a pass can take: n / 64 + 1 for a sequence of n
constexpr int kChunks = 8;                                 // chunk lengths tried at once

// Inclusive sum over the lanes up to this one: within rows of 16, then rows' last lanes onto the next rows.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);   // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);   // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);   // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1, 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2, 3
    return v;
}
__device__ __forceinline__ int row_scan(int v) {   // the same within rows of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    return v;
}
// Exclusive prefix sums of N values per thread over the workgroup; total[] gets the sums. Two barriers.
template <int WAVES, int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*waves)[WAVES]) {
    static_assert(WAVES <= 16 && !(WAVES & (WAVES - 1)), "a row of lanes holds the waves' sums");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int own[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        own[i] = v[i];
        v[i] = wave_scan(v[i]);
    }
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; i++) waves[i][wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int all = row_scan(waves[i][lane & (WAVES - 1)]);
        total[i] = __builtin_amdgcn_readlane(all, WAVES - 1);
        v[i] += (wave ? __builtin_amdgcn_readlane(all, (wave - 1) & 15) : 0) - own[i];
    }
    __syncthreads();
}

// The last r with sums[r] <= j (sums[0] = 0, n entries before the total).
__device__ __forceinline__ int find(const int *sums, int n, int j) {
    int r = 0;
    for (int step = 1 << (31 - __clz(n)); step; step >>= 1)
        if (r + step < n && sums[r + step] <= j) r += step;
    return r;
}

// Slot, position and token entry of a pass row; rows behind the last sequence have none.
__device__ __forceinline__ void put_row(const PlanParams &p, int i, bool there, int at, int page, int r, int token, int block) {
    const int pos = there ? at + (p.pos_off ? p.pos_off[r] : 0) : 0;
    p.slots[i] = (unsigned)page < (unsigned)p.n_pages ? page * PAGE + at % PAGE : -1;
    ((int2 *)(p.work + p.l.tok))[i] = there ? make_int2(block, token) : make_int2(0, 0);
    if (p.pos3) {
        int32_t *dst = p.pos3 + 3 * (size_t)i;
        dst[0] = pos;
        dst[1] = pos;
        dst[2] = pos;
    }
}

// The rows of larger passes: their stores alone would keep one CU busy for 20 us at 16,800 rows (all of the plan
// then took 31 us). Each workgroup takes 256 rows and searches the sequences' first rows in LDS.
constexpr int kRowThreads = 256;
__global__ __launch_bounds__(kRowThreads) void kv8_plan_rows_kernel(PlanParams p) {
    __shared__ int cu_q[kMaxSeq];
    const int n = p.n_seq, n_tok = p.work[H_TOKENS], i = blockIdx.x * kRowThreads + threadIdx.x;
    for (int r = threadIdx.x; r < n; r += kRowThreads) cu_q[r] = p.cu_q[r];
    __syncthreads();
    if (i >= p.T) return;
    const bool there = i < n_tok;
    const int r = find(cu_q, n, i), token = i - cu_q[r];
    int at = 0, page = -1, block = 0;
    if (there) {   // the state is the one after the pass
        at = p.state_out[2 + 2 * r] - (p.cu_q[r + 1] - cu_q[r]) + token;
        page = p.tables[(size_t)r * p.max_pages + at / PAGE];
        block = p.work[p.l.seq_blk + r];
    }
    put_row(p, i, there, at, page, r, token, block);
}

// THREADS: 256 for small passes (an instruction of 16 waves takes four times as long as one of four: 64 sequences of
// a token each 10.2 us with 1,024 threads), 1,024 for others.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv8_plan_kernel(PlanParams p) {
    constexpr int kPlanThreads = THREADS, kPlanWaves = THREADS / 64;
    __shared__ int cu[kPlanSums][kMaxSeq + 1], len[kMaxSeq], held[kMaxSeq], fresh[kMaxFresh], waves[kChunks][kPlanWaves], bad, bad_page, most;
    int *const cu_q = cu[0], *const cu_add = cu[1], *const cu_rel = cu[2], *const cu_app = cu[3], *const cu_blk = cu[4];
    const int tid = threadIdx.x, n = p.n_seq;
    const int n_free = p.state[0];
    const int magic = p.work[H_MAGIC], kept = p.work[H_FAILED];
    const int failed = kept & -(int)(magic == kPlanMagic);   // a buffer's first plan has none before it
    int status = (unsigned)n_free > (unsigned)p.n_pages ? CLEF_HIP_KV8_BAD_STATE : 0;
    int base[kPlanSums] = {0, 0, 0, 0, 0};
    if (tid == 0) bad = bad_page = most = 0;   // the scans' barriers come before their first use
    for (int r0 = 0; r0 < n; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int v[kPlanSums] = {0, 0, 0, 0, 0}, total[kPlanSums];
        if (r < n) {
            int L = p.state[2 + 2 * r], h = p.state[3 + 2 * r];
            const int q = p.new_lens[r];
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
    // The stack after the pages that come back are pushed: those lie above its old top. The pages that go out come
    // off its top, into LDS; every page that changes hands is looked at before anything is written. Its finding has a
    // word of its own: the one before may still be read, and all waves must take the same way past the barrier below.
    auto released = [&](int j) {
        const int r = find(cu_rel, n, j);
        return p.tables[(size_t)r * p.max_pages + j - cu_rel[r]];
    };
    if (!status) {
        bool odd = false;
        for (int j = tid; j < n_add; j += kPlanThreads) {
            const int at = n_free + n_rel - 1 - j, page = at < n_free ? p.free_pages[at] : released(at - n_free);
            fresh[j] = page;
            odd |= (unsigned)page >= (unsigned)p.n_pages;
        }
        for (int j = tid; j < n_rel; j += kPlanThreads) odd |= (unsigned)released(j) >= (unsigned)p.n_pages;
        if (odd) atomicOr(&bad_page, CLEF_HIP_KV8_BAD_STATE);
        __syncthreads();
        status = bad_page;
    }
    const bool good = status == 0;
    // the table's entry, also of pages that are only now written there
    auto page_of = [&](int r, int pg) {
        const int h = held[r];
        return pg < h ? p.tables[(size_t)r * p.max_pages + pg] : fresh[min(cu_add[r] + pg - h, kMaxFresh - 1)];
    };
    int4 *const app = (int4 *)(p.work + p.l.app);
    int app_r = 0, app_pg = 0, app_page = 0;
    auto app_look = [&](int j) {
        app_r = find(cu_app, n, j);
        app_pg = len[app_r] / PAGE + j - cu_app[app_r];
        app_page = page_of(app_r, app_pg);
    };
    auto app_put = [&](int j) {
        const int L = len[app_r], q = cu_q[app_r + 1] - cu_q[app_r];
        const int lo = max(L, app_pg * PAGE), hi = min(L + q, (app_pg + 1) * PAGE);
        app[j] = make_int4(app_page, cu_q[app_r] + lo - L, (lo - app_pg * PAGE) | (hi - lo) << 8, cu_q[app_r]);
    };
    const bool app_first = good && tid < n_app;
    if (app_first) app_look(tid);   // its load runs beside the rows'
    if (p.T <= kPlanThreads) {
        const int i = tid, r = find(cu_q, n, i);
        if (i < p.T) {
            const bool there = good && i < n_tok;
            const int at = len[r] + i - cu_q[r];
            put_row(p, i, there, at, there ? page_of(r, at / PAGE) : -1, r, i - cu_q[r], cu_blk[r]);
        }
    } else   // the rows are another kernel's, which finds a sequence's first block here
        for (int r = tid; r < n; r += kPlanThreads) p.work[p.l.seq_blk + r] = cu_blk[r];
    if (app_first) app_put(tid);
    if (good) {
        for (int j = tid + kPlanThreads; j < n_app; j += kPlanThreads) {
            app_look(j);
            app_put(j);
        }
        for (int j = tid; j < n_add; j += kPlanThreads) {
            const int r = find(cu_add, n, j);
            p.tables[(size_t)r * p.max_pages + held[r] + j - cu_add[r]] = fresh[j];
        }
        for (int j = tid; j < n_rel; j += kPlanThreads) p.free_pages[n_free + j] = released(j);
    }
    for (int r = tid; r < n; r += kPlanThreads) {
        const bool gone = p.new_lens[r] < 0;
        const int L = len[r], h = held[r];
        p.state_out[2 + 2 * r] = !good ? p.state[2 + 2 * r] : gone ? 0 : L + cu_q[r + 1] - cu_q[r];
        p.state_out[3 + 2 * r] = !good ? p.state[3 + 2 * r] : gone ? 0 : h + cu_add[r + 1] - cu_add[r];
        p.cu_q[r] = good ? cu_q[r] : 0;
    }
    // blocks, in two rounds: the pages of all of them set the chunk, then each block's items are placed
    auto block = [&](int b, int &r, int &row0, int &rows) {
        r = find(cu_blk, n, b);
        row0 = (b - cu_blk[r]) * p.l.bm;
        const int q = cu_q[r + 1] - cu_q[r];
        rows = min(p.l.bm, q * p.group - row0);
        return (len[r] + (row0 + rows - 1) / p.group) / PAGE + 1;   // pages up to its last token's own key
    };
    int n_items = 0;
    if (good && n_blk) {
        int r = 0, row0 = 0, rows = 0;
        const int pages0 = tid < n_blk ? block(tid, r, row0, rows) : 0;   // of the thread's first block
        long mine = pages0;
        for (int b = tid + kPlanThreads; b < n_blk; b += kPlanThreads) {
            int r1, row1, rows1;
            mine += block(b, r1, row1, rows1);
        }
        // pages can pass 2^31 over all blocks: the sum is kept in units of 2^8 pages, rounded up
        const bool small = n_blk <= kPlanThreads;   // below 2^16 pages a thread
        int v[1] = {small ? (int)mine : (int)((mine + 255) >> 8)}, total[1];
        block_scan(v, total, waves);
        const long W = small ? (long)total[0] : (long)total[0] << 8;
        int C = (int)min(max((long)p.l.least, (W + p.l.budget - 1) / p.l.budget), 2L * kMaxTablePages);
        // a block below 1.5 chunks stays whole, others are cut into the nearest number of pieces
        auto pieces = [](int pages, int chunk) { return max(1, (2 * pages + chunk) / (2 * chunk)); };
        if (2 * n_blk <= p.l.budget && n_blk <= kPlanThreads) {
            // few blocks: of chunks up to twice as long, the first whose items are one round of workgroups
            int c[kChunks], all[kChunks];
#pragma unroll
            for (int k = 0; k < kChunks; k++) {   // (in floats: near enough to choose by)
                const float chunk = (float)(C + (C * k + kChunks - 2) / (kChunks - 1));
                c[k] = tid < n_blk ? max(1, (int)((float)pages0 * __builtin_amdgcn_rcpf(chunk) + 0.5f)) : 0;
            }
            block_scan(c, all, waves);
            int best = kChunks - 1;
#pragma unroll
            for (int k = kChunks - 2; k >= 0; k--)
                if (all[k] <= p.l.budget) best = k;
            C += (C * best + kChunks - 2) / (kChunks - 1);
        }
        // first items of the blocks, in LDS where they fit (the fresh pages have been written), so that all threads
        // place the items; else each thread its blocks'
        const bool in_lds = n_blk < kMaxFresh;
        int4 *const it = (int4 *)(p.work + p.l.items);
        auto place = [&](int at_item, int k, int items, int pages, int r, int row0, int rows, int slot) {   // the pages split evenly
            const int q0 = cu_q[r];
            it[2 * at_item] = make_int4(r, q0, len[r], len[r] + cu_q[r + 1] - q0);
            it[2 * at_item + 1] = make_int4(row0, rows | (items > 1 ? slot + k + 1 : 0) << 8, (int)((unsigned)pages * k / (unsigned)items),
                                            (int)((unsigned)pages * (k + 1) / (unsigned)items));
        };
        int at = 0, at_slot = 0;
        for (int b0 = 0; b0 < n_blk; b0 += kPlanThreads) {
            const int b = b0 + tid;
            int pages = pages0, c[2] = {0, 0}, sum[2];
            if (b < n_blk) {
                if (b0) pages = block(b, r, row0, rows);
                c[0] = pieces(pages, C);
                c[1] = c[0] > 1 ? c[0] : 0;
            }
            const int items = c[0];
            block_scan(c, sum, waves);
            if (b < n_blk) {
                const int first = at + c[0], slot = at_slot + c[1];
                ((int4 *)(p.work + p.l.blk))[b] = make_int4(first, items, row0, slot);
                if (items > 1) atomicMax(&most, items);
                if (in_lds) fresh[b] = first | slot << 16;   // at most 2^14, 2^11
                else
                    for (int k = 0; k < items; k++) place(first + k, k, items, pages, r, row0, rows, slot);
            }
            at += sum[0];
            at_slot += sum[1];
        }
        if (in_lds) {
            if (tid == 0) fresh[n_blk] = at;
            __syncthreads();
            for (int j = tid; j < at; j += kPlanThreads) {
                int b = 0;
                for (int step = 1 << (31 - __clz(n_blk)); step; step >>= 1)
                    if (b + step < n_blk && (fresh[b + step] & 0xffff) <= j) b += step;
                const int e = fresh[b], first = e & 0xffff;
                const int pages = block(b, r, row0, rows);
                place(j, j - first, (fresh[b + 1] & 0xffff) - first, pages, r, row0, rows, e >> 16);
            }
        }
        n_items = at;
    }
    __syncthreads();
    if (tid == 0) {
        p.cu_q[n] = good ? n_tok : 0;
        p.state_out[0] = good ? n_free + n_rel - n_add : n_free;
        p.state_out[1] = status;
        int32_t *h = p.work;
        h[H_MAGIC] = kPlanMagic;
        h[H_SEQ] = n;
        h[H_ROWS] = p.T;
        h[H_SHAPE] = p.l.shape;
        h[H_TABLE] = p.max_pages;
        h[H_TOKENS] = good ? n_tok : 0;
        h[H_APPEND] = good ? n_app : 0;
        h[H_ITEMS] = n_items;
        h[H_MOST] = most;   // items of the most cut block
        h[H_STATUS] = status;
        h[H_FAILED] = failed | status;
    }
}

}  // namespace kv8
}  // namespace clef_hip
