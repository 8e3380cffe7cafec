// The 8-bit paged prefix cache: its formats, the pass plan's layout and the kernels' argument
// blocks (internal; the interface is documented in include/clef_hip_attn.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "clef_hip_attn.h"

namespace clef_hip {
namespace kv8 {

constexpr int HD = 256;                        // head dim
constexpr int PAGE = CLEF_HIP_KV8_PAGE;        // tokens per page
constexpr int PAGE_BYTES = PAGE * HD;          // codes of one page and kv head, K or V
constexpr int kMaxSeq = CLEF_HIP_KV8_MAX_SEQ;
constexpr int kMaxRows = CLEF_HIP_KV8_MAX_ROWS;
constexpr int kMaxTablePages = 1 << 16;        // entries of a table row: token indexes stay below 2^22
constexpr int kMaxGroup = 128;                 // q heads per kv head
constexpr int32_t kPlanMagic = 0x4b563850;     // 'KV8P'

// Plan header words. A failed plan leaves counts of 0, so the kernels that follow do nothing.
enum { H_MAGIC, H_SEQ, H_ROWS, H_SHAPE, H_TABLE, H_TOKENS, H_APPEND, H_ITEMS, H_MOST,
       H_STATUS = CLEF_HIP_KV8_PLAN_STATUS, H_FAILED = CLEF_HIP_KV8_PLAN_FAILED, H_WORDS = 16 };

// Where the parts of a plan buffer lie (in int32) and how many entries each can need:
//  the first block of each sequence (of passes whose rows a second kernel writes);
//  append items {page, pass row of its first new token, slot of that token in the page | count << 8, first
//  pass row of its sequence}, one for each page that a sequence's new tokens touch: at most one per
//  token and (n - 1) / 64 + 2 per sequence of n;
//  token entries {first block of the token's sequence, index in the sequence};
//  block entries {first item, items, first row, split slot of the first item}: BM rows of a sequence,
//  a row being one q head of the kv group for one token (token-major);
//  attention items {sequence, its first pass row, its cached tokens, its keys, first row, rows |
//  (split slot + 1) << 8, first page, end page}: a block's rows over a run of its pages.
// A block of p pages makes max(1, floor(p / C + 1/2)) items, C at least W / budget, W the pages of all
// blocks: items <= blocks + budget, and those of cut blocks (split slots; p >= 1.5 C) <= 4 W / (3 C) < 2 budget.
struct Layout {
    int bm, shape, budget, least, max_app, max_blk, max_items, max_slots;
    long seq_blk, app, tok, blk, items, ints;
    size_t ws_bytes;
};
inline Layout layout(int n_seq, int T, int nh, int nkv, int max_new, int n_cu) {
    Layout l;
    const int G = nh / nkv;
    const long rows = (long)(max_new > 0 && max_new < T ? max_new : T) * G;
    // Blocks of 16 rows for single tokens (one of 24/4 heads on 4,091 9.7 us, with blocks of 32 13.2, of 128 22.5; 64 sequences of
    // 4,000 tokens 99, 97, 159; at 30 rows of them 155, with blocks of 32 100). Of 32, rather than 128 that share the conversion
    // of a page, for up to 64 rows a sequence (the same 64, 48 rows: 160 against 163) and for passes of up to 8,192
    // (row, head) pairs, whose blocks of 128 would leave CUs idle or each page to few of them: 270 rows 24/4 on 4,091
    // tokens 24.7 against 30.3, 8 x 192 rows on 2,000 30.5 against 37.5, 512 tokens 16/16 on 8,000 86.3 against 85.5; most is
    // lost behind one very long text (1,536 rows on 30,000 tokens 251 against 211). Above: 64 x 96 rows on 4,000 175 against
    // 164, 16 x 128 tokens 16/16 on 4,000 209 against 170.
    l.bm = rows <= 16 ? 16 : rows <= 64 || (long)T * nh <= 8192 ? 32 : 128;
    l.shape = G | nkv << 8 | l.bm << 20;   // what the lists go by beside n_seq and T
    l.budget = ((l.bm == 16 ? 2 : 1) * n_cu + nkv - 1) / nkv;   // items of one round of workgroups, two or one to a CU
    l.least = 4;
    const long app = (long)T / PAGE + 2L * n_seq;
    l.max_app = (int)(app < T ? app : T);
    l.max_blk = (int)((long)T * G / l.bm) + (n_seq < T ? n_seq : T);
    l.max_items = l.max_blk + l.budget;
    l.max_slots = 2 * l.budget;
    l.seq_blk = H_WORDS;
    l.app = (l.seq_blk + n_seq + 3) / 4 * 4;
    l.tok = l.app + 4L * l.max_app;
    l.blk = (l.tok + 2L * T + 3) / 4 * 4;
    l.items = (l.blk + 4L * l.max_blk + 7) / 8 * 8;
    l.ints = l.items + 8L * l.max_items;
    l.ws_bytes = (size_t)l.max_slots * nkv * l.bm * (HD + 2) * sizeof(float);
    return l;
}

struct PlanParams {
    int n_seq, max_pages, n_pages, T, group;
    Layout l;
    int32_t *tables, *free_pages;
    const int32_t *state, *new_lens, *pos_off;
    int32_t *state_out, *cu_q, *slots, *pos3, *work;
};

struct Params {
    const uint16_t *qkv;
    const float *q_norm, *k_norm, *inv_freq;
    const int32_t *pos3, *tables, *plan;
    uint8_t *k_pages, *v_pages;
    float *k_scale, *v_scale, *partial;
    void *out;
    int32_t *ovf;
    int nh, nkv, group, n_rot, row, T, n_seq, max_pages, n_pages, gate, out_type;
    float eps, scale_log2, f16_lim;
    Layout l;
};

// A plan is run only with the sizes it was made for: list entries, items and split slots stay within those sizes.
// One wait for all five words (&& would load each after the one before).
__device__ __forceinline__ bool plan_fits(int magic, int seq, int rows, int shape, int table, const Params &p) {
    return ((magic ^ kPlanMagic) | (seq ^ p.n_seq) | (rows ^ p.T) | (shape ^ p.l.shape) | (table ^ p.max_pages)) == 0;
}
// Whether list entry i of h[count] is one of a plan that fits. Its words a, b come with the header's, not behind the
// check of them (one trip to memory for two: one token 7.1 -> 6.8 us): named together, all are loaded before. The host
// has checked that the buffer is as long as this call's layout, so they lie within it whatever the header says.
__device__ __forceinline__ bool plan_has(const Params &p, int count, int i, int4 &a, int4 &b) {
    const int32_t *h = p.plan;
    int magic = h[H_MAGIC], seq = h[H_SEQ], rows = h[H_ROWS], shape = h[H_SHAPE], table = h[H_TABLE], n = h[count];
    asm volatile("" : "+s"(a.x), "+s"(a.y), "+s"(a.z), "+s"(a.w), "+s"(b.x), "+s"(b.y), "+s"(b.z), "+s"(b.w),
                      "+s"(magic), "+s"(seq), "+s"(rows), "+s"(shape), "+s"(table), "+s"(n));
    return plan_fits(magic, seq, rows, shape, table, p) && i < n;
}

}  // namespace kv8
}  // namespace clef_hip
