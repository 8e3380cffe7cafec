// Grouped-query attention of a pass's new tokens over the 8-bit paged cache, with the Q prologue
// (RMSNorm, rotary) and the sigmoid gate fused in.
//
// Rows are (token, q head of the kv group), token-major, so that the q heads that share a kv head share its
// pages: one token of 24/4 heads is 6 rows of a 16-row matrix tile. Per 16-row tile and 64-token page
//   S^T = K . Q^T     v_mfma_f32_16x16x32_f16: A = K codes as f16 (exact), B = Q (f16)
//   O^T += V^T . P^T  v_mfma_f32_16x16x32_f16: A = V codes as f16 (exact), B = 2^15 P (f16)
// The page's K scale multiplies the f32 scores together with the softmax scale, at no cost per element. The
// accumulated O is kept in units of the current page's V scale times 2^-15: where that changes, so does the factor
// that rescales O for a new maximum. P in f16 rounds by 2^-11 of itself (bf16: 2^-8); 2^15 P keeps that down
// to P = 2^-29, and what falls below 2^-40 of the row's largest weight is lost. Units of 2^-64 to 2^8 leave O
// within 2^113 and 2^-100. Row r of A tile t (of four that make up 64
// rows) is token / dim 16 (r / 4) + 4 t + r % 4: then a lane's 16 scores of a page are 16 consecutive tokens,
// which are the k indexes of the next product's B operand with no exchange, and its 16 outputs of a dim
// group are consecutive dims. A lane reads 16-byte pieces (row, 16 dims or tokens) of the page, each two
// operands' worth.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "bf16_ops.h"
#include "kv8_pages.h"
#include "kv8_params.h"
#include "text_ops.h"

namespace clef_hip {
namespace kv8 {

typedef __attribute__((ext_vector_type(4))) float f32x4;
constexpr float kNone = -1e30f;   // a running maximum before any key: below every score, and finite

__device__ __forceinline__ f16x8 codes_f16(unsigned a, unsigned b) {
    const f16x2 x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false), y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true);
    const f16x2 z = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false), w = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true);
    return f16x8{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}
// The first n bytes of a word (n below 0 or above 4: none, all).
__device__ __forceinline__ unsigned keep_bytes(int n) { return n <= 0 ? 0u : ~0u >> 8 * (4 - min(n, 4)); }

// One q row as the B operand of its 16-row tile: lane (row, g) takes dims 64c + 16g + e, e < 16, as operands
// 2c (e < 8) and 2c + 1. Two steps, so that other loads can go out between them: the row as it is, then norm and
// rotary in f32 and f16 with split16's saturation (flagged).
struct QRow {
    u32x4 w[8];
    float pos[3];
};
__device__ __forceinline__ void load_q(const Params &p, int t, int head, int g, QRow &r) {
    const uint16_t *src = p.qkv + (size_t)t * p.row + (size_t)head * 2 * HD + 16 * g;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        r.w[2 * c] = *(const u32x4 *)(src + 64 * c);
        r.w[2 * c + 1] = *(const u32x4 *)(src + 64 * c + 8);
    }
    if (p.n_rot)
#pragma unroll
        for (int i = 0; i < 3; i++) r.pos[i] = (float)p.pos3[3 * (size_t)t + i];
}
__device__ __forceinline__ float other_half(float x) {   // lane ^ 32's value
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ void make_q(const Params &p, const QRow &r, int g, f16x8 (&q)[8], int32_t *flag) {
    float x[4][16];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < 4; c++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[c][2 * i] = bf_lo(r.w[2 * c][i]);
            x[c][2 * i + 1] = bf_hi(r.w[2 * c][i]);
            x[c][8 + 2 * i] = bf_lo(r.w[2 * c + 1][i]);
            x[c][9 + 2 * i] = bf_hi(r.w[2 * c + 1][i]);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) ss += x[c][i] * x[c][i];
    }
    if (p.q_norm) {
        const float inv = rsqrtf(text::xrow_sum(ss) / (float)HD + p.eps);
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 w = *(const float4 *)(p.q_norm + 64 * c + 16 * g + i);
                x[c][i] *= inv * w.x;
                x[c][i + 1] *= inv * w.y;
                x[c][i + 2] *= inv * w.z;
                x[c][i + 3] *= inv * w.w;
            }
    }
    if (p.n_rot) {
        // dims 16g + e of the first 64: pair (16g + e) % 32, whose other half lane ^ 32 holds; the two lanes share
        // their 16 pairs' sin and cos, eight each
        float sn[16], cn[16];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int i = 16 * (g & 1) + 8 * (g >> 1) + e;
            const int axis = i % 3;
            rope_sincos((axis == 0 ? r.pos[0] : axis == 1 ? r.pos[1] : r.pos[2]) * p.inv_freq[i], &sn[e], &cn[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float s1 = other_half(sn[e]), c1 = other_half(cn[e]), s0 = sn[e], c0 = cn[e];
            sn[e] = g < 2 ? s0 : s1;
            sn[e + 8] = g < 2 ? s1 : s0;
            cn[e] = g < 2 ? c0 : c1;
            cn[e + 8] = g < 2 ? c1 : c0;
        }
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float o = other_half(x[0][e]);
            x[0][e] = g < 2 ? x[0][e] * cn[e] - o * sn[e] : x[0][e] * cn[e] + o * sn[e];
        }
    }
    bool bad = false;
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            bad |= saturate(x[c][i], p.f16_lim);
            q[2 * c + (i >> 3)][i & 7] = (_Float16)x[c][i];
        }
    if (bad && flag) __hip_atomic_store(flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sixteen finished outputs (dims d0 ..) of a row: times the gate's sigmoid, converted and stored.
__device__ __forceinline__ void finish16(const Params &p, int t, int head, int d0, float (&o)[16], int32_t *flag) {
    if (p.gate) {
        const uint16_t *src = p.qkv + (size_t)t * p.row + (size_t)head * 2 * HD + HD + d0;
        const u32x4 a = *(const u32x4 *)src, b = *(const u32x4 *)(src + 8);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            o[2 * i] *= sigmoidf(bf_lo(a[i]));
            o[2 * i + 1] *= sigmoidf(bf_hi(a[i]));
            o[8 + 2 * i] *= sigmoidf(bf_lo(b[i]));
            o[9 + 2 * i] *= sigmoidf(bf_hi(b[i]));
        }
    }
    const size_t idx = ((size_t)t * p.nh + head) * HD + d0;
    store_out8(p.out, idx, o, p.out_type, p.f16_lim, flag);
    store_out8(p.out, idx + 8, o + 8, p.out_type, p.f16_lim, flag);
}

// Partial results of a cut block: [split slot][kv head][row][256] unnormalised outputs, then
// [split slot][kv head][row][2] running maximum (log2 units) and sum.
__device__ __forceinline__ size_t partial_row(const Params &p, int slot, int kh, int row) {
    return ((size_t)slot * p.nkv + kh) * p.l.bm + row;
}
__device__ __forceinline__ float *partial_ml(const Params &p) {
    return p.partial + (size_t)p.l.max_slots * p.nkv * p.l.bm * HD;
}

// Few rows (decoding): a workgroup takes an item's 16 MT rows over its pages, wave w the pages w, w + 4, ...
// Bound by memory: each page is read once, straight into registers, 4 KB pieces (four 1 KB loads) in a ring of
// four that K and V share: as a piece is used up, the one four later is loaded into its registers, so 16 KB a
// wave are always in flight, and with 16 rows two workgroups fit a CU, one's prologue and joins behind the
// other's stream. Page numbers and scales of a wave's next 64 pages are held one per lane. The four waves'
// results join through LDS.
constexpr int kRowsThreads = 256, kRowsWaves = 4;
template <int MT>
__global__ __launch_bounds__(kRowsThreads, MT == 1 ? 2 : 1) void kv8_attn_rows_kernel(Params p) {
    constexpr int BM = 16 * MT, OS = HD + 4;   // LDS row stride of the outputs
    __shared__ float os[kRowsWaves][16][OS], ml[kRowsWaves][BM][2];
    const int32_t *h = p.plan;
    const int item = blockIdx.x / p.nkv, kh = blockIdx.x - item * p.nkv;
    const int4 *it = (const int4 *)(p.plan + p.l.items) + 2 * item;
    const int4 e0 = it[0], e1 = it[1];
    if (!plan_fits(h, p.n_seq, p.T, p.group, p.l.bm) || item >= h[H_ITEMS]) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q16 = lane & 15, g = lane >> 4;
    const int lofs = (16 * (q16 >> 2) + (q16 & 3)) * 64 + 16 * g;   // the lane's piece of tile 0
    const int seq = e0.x, q0 = e0.y, L = e0.z, n_keys = e0.w, row0 = e1.x, rows = e1.y & 0xff, slot = (e1.y >> 8) - 1;
    const int pg0 = e1.z, pg1 = e1.w;
    const int32_t *table = p.tables + (size_t)seq * p.max_pages;
    QRow raw[MT];
    int last[MT];   // the last key the lane's row sees
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int fr = row0 + min(16 * m + q16, rows - 1), t = fr / p.group, head = kh * p.group + fr - t * p.group;
        load_q(p, q0 + t, head, g, raw[m]);
        last[m] = L + t;
    }
    // the wave's pages i = 0, 1, ... are pg0 + wave + 4 i; lane j holds number and scales of page (i & ~63) + j
    const int n_mine = (pg1 - pg0 - wave + kRowsWaves - 1) / kRowsWaves;   // 0 or less: none
    unsigned ids = 0;
    float kss = 0.f, vss = 0.f;
    auto look_up = [&](int i0) {
        const int pg = pg0 + wave + kRowsWaves * (i0 + lane);
        ids = pg < pg1 ? (unsigned)table[pg] : 0u;
        if (ids >= (unsigned)p.n_pages) ids = 0;
        ids = ids * p.nkv + kh;
        kss = p.k_scale[ids];
        vss = p.v_scale[ids];
        asm volatile("" : "+v"(kss), "+v"(vss));   // waited for here: the loop's waits are for its own loads
    };
    u32x4 ring[4][4];
    auto load = [&](const uint8_t *pages, unsigned at, int c) {
        const uint8_t *src = pages + (size_t)at * PAGE_BYTES + 4096 * c + lofs;
#pragma unroll
        for (int t = 0; t < 4; t++) ring[c][t] = *(const u32x4 *)(src + 256 * t);
    };
    unsigned at = 0;
    if (n_mine > 0) {
        look_up(0);
        at = __builtin_amdgcn_readlane(ids, 0);
#pragma unroll
        for (int c = 0; c < 4; c++) load(p.k_pages, at, c);
    }
    f16x8 q[MT][8];
#pragma unroll
    for (int m = 0; m < MT; m++) make_q(p, raw[m], g, q[m], p.ovf ? p.ovf + q0 : nullptr);
    f32x4 o[MT][16];
    float mx[MT], sum[MT];
    int unit = 0;   // o is in units of 2^(unit - 15)
#pragma unroll
    for (int m = 0; m < MT; m++) {
        mx[m] = kNone;
        sum[m] = 0.f;
#pragma unroll
        for (int d = 0; d < 16; d++) o[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // Only a wave's last page can hold keys that a row does not see or that are not there: an item's rows are of at
    // most 32 tokens, whose keys lie in its last two pages. It runs apart, so that the others' loads are unconditional
    // (the compiler's waits would otherwise count on none being in flight).
    auto page = [&](int i, auto more_t) {
        constexpr bool MORE = decltype(more_t)::value;
        const int pg = pg0 + wave + kRowsWaves * i;
        const float kf = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kss), i & 63)) * p.scale_log2;
        const int ev = (int)(__builtin_amdgcn_readlane(__float_as_uint(vss), i & 63) >> 23) - 127;   // the V scale is 2^ev
        f32x4 s[MT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int t = 0; t < 4; t++) s[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; c++) {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const u32x4 w = ring[c][t];
                const f16x8 a = codes_f16(w[0], w[1]), b = codes_f16(w[2], w[3]);
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    s[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[m][2 * c], s[m][t], 0, 0, 0);
                    s[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, q[m][2 * c + 1], s[m][t], 0, 0, 0);
                }
            }
            load(p.v_pages, at, c);
            __builtin_amdgcn_sched_barrier(0);   // pieces are used, and asked for, in this order
        }
        const int key0 = pg * PAGE + 16 * g;
        f16x8 pb[MT][2];
#pragma unroll
        for (int m = 0; m < MT; m++) {
            if (!MORE && (pg + 1) * PAGE > L + 1) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (key0 + 4 * t + e > last[m]) s[m][t][e] = -INFINITY;
            }
            float top = s[m][0][0];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) top = fmaxf(top, s[m][t][e]);
            const float now = fmaxf(mx[m], text::xrow_max(top) * kf);
            const float f = __builtin_amdgcn_exp2f(mx[m] - now);
            mx[m] = now;
            float add = 0.f;
            const float shift = 15.f - now;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[m][t][e], kf, shift));
                    add += x;
                    pb[m][t >> 1][4 * (t & 1) + e] = (_Float16)x;
                }
            sum[m] = sum[m] * f + add;
            const float fo = ldexpf(f, unit - ev);
            if (__any(fo != 1.f))
#pragma unroll
                for (int d = 0; d < 16; d++) o[m][d] *= fo;
        }
        unit = ev;
        unsigned next = 0;
        if constexpr (MORE) {
            if (((i + 1) & 63) == 0) look_up(i + 1);
            next = __builtin_amdgcn_readlane(ids, (i + 1) & 63);
        } else if ((pg + 1) * PAGE > n_keys) {   // V codes behind the last key may be NaN, whose product with 0 is NaN
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const unsigned keep = keep_bytes(n_keys - key0 - 4 * w);
#pragma unroll
                for (int d = 0; d < 16; d++) ring[d >> 2][d & 3][w] &= keep;
            }
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const u32x4 w = ring[c][t];
                const f16x8 a = codes_f16(w[0], w[1]), b = codes_f16(w[2], w[3]);
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    o[m][4 * c + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pb[m][0], o[m][4 * c + t], 0, 0, 0);
                    o[m][4 * c + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, pb[m][1], o[m][4 * c + t], 0, 0, 0);
                }
            }
            if constexpr (MORE) load(p.k_pages, next, c);
            __builtin_amdgcn_sched_barrier(0);
        }
        at = next;
    };
    for (int i = 0; i + 1 < n_mine; i++) page(i, std::true_type{});
    if (n_mine > 0) page(n_mine - 1, std::false_type{});
    // join the waves: each scales its outputs to the common maximum and to units of 1 (sums are of 2^15 P)
#pragma unroll
    for (int m = 0; m < MT; m++) {
        sum[m] = text::xrow_sum(sum[m]);
        if (g == 0) {
            ml[wave][16 * m + q16][0] = mx[m];
            ml[wave][16 * m + q16][1] = sum[m];
        }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; m++) {
        float top = kNone;
#pragma unroll
        for (int w = 0; w < kRowsWaves; w++) top = fmaxf(top, ml[w][16 * m + q16][0]);
        const float f = ldexpf(__builtin_amdgcn_exp2f(mx[m] - top), unit);
#pragma unroll
        for (int d = 0; d < 16; d++) *(f32x4 *)&os[wave][q16][64 * (d >> 2) + 16 * g + 4 * (d & 3)] = o[m][d] * f;
        __syncthreads();
        const int r = tid >> 4, d0 = 16 * (tid & 15), row = 16 * m + r;
        if (row < rows) {
            float x[16], l = 0.f;
            float mrow = kNone;
#pragma unroll
            for (int w = 0; w < kRowsWaves; w++) mrow = fmaxf(mrow, ml[w][row][0]);
#pragma unroll
            for (int w = 0; w < kRowsWaves; w++) l += ml[w][row][1] * __builtin_amdgcn_exp2f(ml[w][row][0] - mrow);
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = os[0][r][d0 + i] + os[1][r][d0 + i] + os[2][r][d0 + i] + os[3][r][d0 + i];
            if (slot < 0) {
                const int fr = row0 + row, t = fr / p.group, head = kh * p.group + fr - t * p.group;
                const float inv = 1.f / l;
#pragma unroll
                for (int i = 0; i < 16; i++) x[i] *= inv;
                finish16(p, q0 + t, head, d0, x, p.ovf ? p.ovf + q0 : nullptr);
            } else {
                const size_t pr = partial_row(p, slot, kh, row);
                float *dst = p.partial + pr * HD + d0;
#pragma unroll
                for (int i = 0; i < 16; i += 4) *(f32x4 *)(dst + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
                if ((tid & 15) == 0) *(float2 *)(partial_ml(p) + 2 * pr) = make_float2(mrow, l);
            }
        }
        if (m + 1 < MT) __syncthreads();
    }
}

// Many rows (prompts, questions): 128 rows an item, 16 MT per wave, the pages shared through LDS. Pages come in as
// they are by DMA (global_load_lds), already in operand order, three stages of 32 KB ahead of one barrier a
// page; every wave turns the codes it needs into f16 after the read. Codes in LDS halve its traffic against
// f16 tiles (8 waves x 32 KB a page: 2,048 clocks, as long as the page's matrix products), for 256 conversions
// per wave and page.
constexpr int kTileStages = 3, kTileStage = 2 * PAGE_BYTES;
typedef __attribute__((address_space(3))) void lds_ptr;
template <int OFF>
__device__ __forceinline__ u32x4 lds_read(unsigned addr) {
    u32x4 r;
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(OFF) : "memory");
    return r;
}
template <int N>
__device__ __forceinline__ void lds_wait(u32x4 (&r)[4]) {
    asm volatile("s_waitcnt lgkmcnt(%4)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]) : "i"(N));
}
template <int C>
__device__ __forceinline__ void lds_piece(u32x4 (&r)[4], unsigned addr) {
    r[0] = lds_read<4096 * C>(addr);
    r[1] = lds_read<4096 * C + 1024>(addr);
    r[2] = lds_read<4096 * C + 2048>(addr);
    r[3] = lds_read<4096 * C + 3072>(addr);
}

template <int MT>
__global__ __launch_bounds__(512 / MT, 2 / MT) void kv8_attn_tile_kernel(Params p) {
    constexpr int WAVES = 8 / MT, PIECES = 32 / WAVES, NS = kTileStages;
    __shared__ __attribute__((aligned(16))) uint8_t stage[NS * kTileStage];
    const int32_t *h = p.plan;
    const int item = blockIdx.x / p.nkv, kh = blockIdx.x - item * p.nkv;
    const int4 *it = (const int4 *)(p.plan + p.l.items) + 2 * item;
    const int4 e0 = it[0], e1 = it[1];
    if (!plan_fits(h, p.n_seq, p.T, p.group, p.l.bm) || item >= h[H_ITEMS]) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q16 = lane & 15, g = lane >> 4;
    const int seq = e0.x, q0 = e0.y, L = e0.z, n_keys = e0.w, row0 = e1.x, rows = e1.y & 0xff, slot = (e1.y >> 8) - 1;
    const int pg0 = e1.z, n_pages = e1.w - e1.z;
    const int32_t *table = p.tables + (size_t)seq * p.max_pages;
    const int w0 = 16 * MT * wave;   // the wave's first row in the block
    const bool active = w0 < rows;
    QRow raw[MT];
    int last[MT], head[MT], tok[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int fr = row0 + min(w0 + 16 * m + q16, rows - 1);
        tok[m] = fr / p.group;
        head[m] = kh * p.group + fr - tok[m] * p.group;
        load_q(p, q0 + tok[m], head[m], g, raw[m]);
        last[m] = L + tok[m];
    }
    // keys that every row of the wave sees, and the last that any sees
    const int all_see = L + (row0 + min(w0, rows - 1)) / p.group, any_sees = L + (row0 + min(w0 + 16 * MT, rows) - 1) / p.group;
    unsigned ids = 0;   // lane j: page (i & ~63) + j
    float kss = 0.f, vss = 0.f;
    auto look_up = [&](int i0) {
        const int i = i0 + lane;
        ids = i < n_pages ? (unsigned)table[pg0 + i] : 0u;
        if (ids >= (unsigned)p.n_pages) ids = 0;
        ids = ids * p.nkv + kh;
    };
    unsigned pofs[PIECES];   // the lane's byte in the page of each piece its wave loads
#pragma unroll
    for (int j = 0; j < PIECES; j++) {
        const int piece = (wave * PIECES + j) & 15;
        pofs[j] = (piece >> 2) * 4096 + (piece & 3) * 256 + (16 * (q16 >> 2) + (q16 & 3)) * 64 + 16 * g;
    }
    auto fill = [&](int i) {   // page i into its stage; i & 63 must lie in the looked-up run
        const size_t at = (size_t)__builtin_amdgcn_readlane(ids, i & 63) * PAGE_BYTES;
        const uint8_t *src = (wave * PIECES < 16 ? p.k_pages : p.v_pages) + at;
        uint8_t *dst = stage + (i % NS) * kTileStage + wave * PIECES * 1024;
#pragma unroll
        for (int j = 0; j < PIECES; j++) {
            unsigned off = pofs[j];
            asm volatile("" : "+v"(off));
            __builtin_amdgcn_global_load_lds((const void *)(src + off), (lds_ptr *)(dst + 1024 * j), 16, 0, 0);
        }
    };
    look_up(0);
    const unsigned ids0 = ids;
    kss = p.k_scale[ids0];
    vss = p.v_scale[ids0];
    for (int i = 0; i < NS - 1 && i < n_pages; i++) fill(i);
    f16x8 q[MT][8];
#pragma unroll
    for (int m = 0; m < MT; m++) make_q(p, raw[m], g, q[m], p.ovf ? p.ovf + q0 : nullptr);
    asm volatile("" : "+v"(kss), "+v"(vss));
    f32x4 o[MT][16];
    float mx[MT], sum[MT];
    int unit = 0;   // o is in units of 2^(unit - 15)
#pragma unroll
    for (int m = 0; m < MT; m++) {
        mx[m] = kNone;
        sum[m] = 0.f;
#pragma unroll
        for (int d = 0; d < 16; d++) o[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const unsigned lds0 = (unsigned)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)stage + 16 * lane;
    for (int i = 0; i < n_pages; i++) {
        if (i && (i & 63) == 0) {   // the scales of this page's run (its numbers were looked up with the fills)
            const int j = i + lane;
            unsigned id = j < n_pages ? (unsigned)table[pg0 + j] : 0u;
            if (id >= (unsigned)p.n_pages) id = 0;
            kss = p.k_scale[(size_t)id * p.nkv + kh];
            vss = p.v_scale[(size_t)id * p.nkv + kh];
            asm volatile("" : "+v"(kss), "+v"(vss));   // waited for here, or every page would wait for all fills
        }
        // the page has come once at most the fills of the pages behind it are in flight, in every wave
        if (i + 1 < n_pages) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(PIECES * (NS - 2)) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int ahead = i + NS - 1;   // its stage held page i - 1, which every wave is done with
        if (ahead < n_pages) {
            if ((ahead & 63) == 0) look_up(ahead);
            fill(ahead);
        }
        const int pg = pg0 + i;
        if (active && pg * PAGE <= any_sees) {
            const unsigned kl = lds0 + (i % NS) * kTileStage;
            u32x4 r[2][4];
            f32x4 s[MT][4];
            lds_piece<0>(r[0], kl);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < 4; t++) s[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            auto k_step = [&](auto c) {
                constexpr int C = decltype(c)::value;
                lds_piece<C + 1>(r[(C + 1) & 1], kl);   // behind K piece 3 lies V piece 0
                lds_wait<4>(r[C & 1]);
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const u32x4 w = r[C & 1][t];
                    const f16x8 a = codes_f16(w[0], w[1]), b = codes_f16(w[2], w[3]);
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        s[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[m][2 * C], s[m][t], 0, 0, 0);
                        s[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, q[m][2 * C + 1], s[m][t], 0, 0, 0);
                    }
                }
            };
            text::static_for<4>(k_step);
            const float kf = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kss), i & 63)) * p.scale_log2;
            const int ev = (int)(__builtin_amdgcn_readlane(__float_as_uint(vss), i & 63) >> 23) - 127;
            const int key0 = pg * PAGE + 16 * g;
            f16x8 pb[MT][2];
#pragma unroll
            for (int m = 0; m < MT; m++) {
                if ((pg + 1) * PAGE > all_see + 1) {
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (key0 + 4 * t + e > last[m]) s[m][t][e] = -INFINITY;
                }
                float top = s[m][0][0];
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) top = fmaxf(top, s[m][t][e]);
                const float now = fmaxf(mx[m], text::xrow_max(top) * kf);
                const float f = __builtin_amdgcn_exp2f(mx[m] - now);
                mx[m] = now;
                float add = 0.f;
                const float shift = 15.f - now;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x = __builtin_amdgcn_exp2f(fmaf(s[m][t][e], kf, shift));
                        add += x;
                        pb[m][t >> 1][4 * (t & 1) + e] = (_Float16)x;
                    }
                sum[m] = sum[m] * f + add;
                const float fo = ldexpf(f, unit - ev);
                if (__any(fo != 1.f))
#pragma unroll
                    for (int d = 0; d < 16; d++) o[m][d] *= fo;
            }
            unit = ev;
            const bool tail = (pg + 1) * PAGE > n_keys;
            auto v_step = [&](auto c) {
                constexpr int C = decltype(c)::value;
                if constexpr (C < 3) {
                    lds_piece<C + 5>(r[(C + 1) & 1], kl);
                    lds_wait<4>(r[C & 1]);
                } else lds_wait<0>(r[C & 1]);
                if (tail) {   // V codes behind the last key, which may be NaN
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const unsigned keep = keep_bytes(n_keys - key0 - 4 * w);
#pragma unroll
                        for (int t = 0; t < 4; t++) r[C & 1][t][w] &= keep;
                    }
                }
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const u32x4 w = r[C & 1][t];
                    const f16x8 a = codes_f16(w[0], w[1]), b = codes_f16(w[2], w[3]);
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        o[m][4 * C + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pb[m][0], o[m][4 * C + t], 0, 0, 0);
                        o[m][4 * C + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, pb[m][1], o[m][4 * C + t], 0, 0, 0);
                    }
                }
            };
            text::static_for<4>(v_step);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int row = w0 + 16 * m + q16;
        const float l = text::xrow_sum(sum[m]);
        if (row >= rows) continue;
        const float f = slot < 0 ? ldexpf(1.f / l, unit) : ldexpf(1.f, unit);
        const size_t pr = slot < 0 ? 0 : partial_row(p, slot, kh, row);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            float x[16];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[4 * t + e] = o[m][4 * c + t][e] * f;
            if (slot < 0) finish16(p, q0 + tok[m], head[m], 64 * c + 16 * g, x, p.ovf ? p.ovf + q0 : nullptr);
            else
#pragma unroll
                for (int t = 0; t < 4; t++) *(f32x4 *)(p.partial + pr * HD + 64 * c + 16 * g + 4 * t) = f32x4{x[4 * t], x[4 * t + 1], x[4 * t + 2], x[4 * t + 3]};
        }
        if (slot >= 0 && g == 0) *(float2 *)(partial_ml(p) + 2 * pr) = make_float2(mx[m], l);
    }
}

// Joins the items of cut blocks. Workgroup unit (pass row, q head): wave w takes items w, w + 4, ..., a lane
// four dims; the items are added in a fixed order, so results do not change from run to run.
constexpr int kJoinThreads = 256, kJoinWaves = kJoinThreads / 64;
__global__ __launch_bounds__(kJoinThreads) void kv8_join_kernel(Params p) {
    __shared__ float os[kJoinWaves][HD], ls[kJoinWaves];
    const int32_t *h = p.plan;
    if (!plan_fits(h, p.n_seq, p.T, p.group, p.l.bm) || h[H_SPLIT] == 0) return;
    const int units = h[H_TOKENS] * p.nh, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int t = u / p.nh, head = u - t * p.nh, kh = head / p.group;
        const int2 tok = ((const int2 *)(p.plan + p.l.tok))[t];
        const int fr = tok.y * p.group + head - kh * p.group, b = tok.x + fr / p.l.bm;
        const int4 blk = ((const int4 *)(p.plan + p.l.blk))[b];
        const int n = blk.y, row = fr - blk.z;
        if (n <= 1) continue;   // the whole workgroup skips it
        const int q0 = t - tok.y;
        const float *ml = partial_ml(p);
        float top = kNone;
        for (int k = lane; k < n; k += 64) top = fmaxf(top, ml[2 * partial_row(p, blk.w + k, kh, row)]);
#pragma unroll
        for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
#pragma unroll 4
        for (int k = wave; k < n; k += kJoinWaves) {
            const size_t pr = partial_row(p, blk.w + k, kh, row);
            const float2 e = *(const float2 *)(ml + 2 * pr);
            const f32x4 x = *(const f32x4 *)(p.partial + pr * HD + 4 * lane);
            const float f = __builtin_amdgcn_exp2f(e.x - top);
            l += e.y * f;
            o += x * f;
        }
        *(f32x4 *)&os[wave][4 * lane] = o;
        if (lane == 0) ls[wave] = l;
        __syncthreads();
        if (tid < 16) {
            float x[16];
            const float inv = 1.f / (ls[0] + ls[1] + ls[2] + ls[3]);
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = (os[0][16 * tid + i] + os[1][16 * tid + i] + os[2][16 * tid + i] + os[3][16 * tid + i]) * inv;
            finish16(p, t, head, 16 * tid, x, p.ovf ? p.ovf + q0 : nullptr);
        }
        __syncthreads();
    }
}

}  // namespace kv8
}  // namespace clef_hip
