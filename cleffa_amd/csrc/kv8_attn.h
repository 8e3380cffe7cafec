// Grouped-query attention of a pass's new tokens over the 8-bit paged cache, with the Q prologue
// (RMSNorm, rotary) and the sigmoid gate fused in.
//
// Rows are (token, q head of the kv group), token-major, so that the q heads that share a kv head share its
// pages: one token of 24/4 heads is 6 rows of a 16-row matrix tile. Per 16-row tile and 64-token page
//   S^T = K . Q^T     v_mfma_f32_16x16x32_f16: A = K codes as f16 (exact), B = Q (f16)
//   O^T += V^T . P^T  v_mfma_f32_16x16x32_f16: A = V codes as f16 (exact), B = P (f16)
// The page's K scale multiplies the f32 scores in the instruction that takes the maximum off, its V scale is a unit of O or
// goes into the exponent of P: neither costs an instruction per element. P in f16 rounds by 2^-11 of itself (bf16:
// 2^-8); against the row's largest it is held from 2^3 on, which keeps that down to P = 2^-17, with steps of
// 2^-27 below. Units of 2^-64 to 2^8 leave O within 2^113 and 2^-100. Row r of A tile t (of four that make up 64
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

// The running maximum m is one that later pages may pass by up to 2^8: it, and what has been summed under it, is
// only moved for a page that passes it by more (most pages of most rows do not, which saves the products that
// rescale O). Likewise the unit of O, a V scale 2^unit, stays for pages whose scale is within 2^2 of it: the
// difference goes into P's exponent. P is then held as 2^(5 + ev - unit) P in f16, 2^15 at most.
constexpr float kPUnit = 5.f, kSlack = 8.f;
constexpr int kUnitSlack = 2;
constexpr float kPMost = 8192.f;   // 2^(5 + 8): a weight as large as the slack allows, of a page in its own unit
__device__ __forceinline__ float pow2(int e) { return ldexpf(1.f, e); }
// Maxima are of q . k with the K scale in it, a power of two, so they are exact images of the scores they came from; the
// softmax scale times log2 e comes behind the difference from m. (A rounded product as m, and the weights from the exact
// one, would part by half a step of m: 2^16 in a weight from scores of 2^28 on.)
__device__ __forceinline__ float weight(float s, float k_scale, float m, float scale_log2, float unit) {
    return __builtin_amdgcn_exp2f(fmaf(fmaf(s, k_scale, -m), scale_log2, unit));
}
// Moves m for a page whose largest score top passes it by more than the slack; returns the factor that sums under the old m take.
__device__ __forceinline__ float new_max(float &m, float top, float slack, float scale_log2) {
    const float now = (top - m) * scale_log2 > slack ? top : m;
    const float f = __builtin_amdgcn_exp2f((m - now) * scale_log2);
    m = now;
    return f;
}

__device__ __forceinline__ f16x8 codes_f16(unsigned a, unsigned b) {
    const f16x2 x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false), y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true);
    const f16x2 z = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false), w = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true);
    return f16x8{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}
// The first n bytes of a word (n below 0 or above 4: none, all).
__device__ __forceinline__ unsigned keep_bytes(int n) { return n <= 0 ? 0u : ~0u >> 8 * (4 - min(n, 4)); }

// The q rows of an item: RMSNorm and rotary in f32, then f16 with split16's saturation (flagged), into LDS rows of QS.
// The workgroup's waves share them, 16 lanes a row, lane j of them dims 64c + 4j + e, e < 4: few loads, of whole lines
// (a wave that made the operands of its own 16 rows spent 8,000 clocks on loading them, 29 loads of 16 bytes a lane).
// Loads and arithmetic are apart, so that other loads can go out between them.
constexpr int QS = HD + 8;
struct QNorm {   // of all rows
    float4 norm[4], freq;
};
struct QPart {
    uint2 w[4];
    int pos[3];
};
__device__ __forceinline__ void load_norm(const Params &p, int j, QNorm &n) {
    if (p.q_norm)
#pragma unroll
        for (int c = 0; c < 4; c++) n.norm[c] = *(const float4 *)(p.q_norm + 64 * c + 4 * j);
    if (p.n_rot) n.freq = *(const float4 *)(p.inv_freq + 4 * (j & 7));   // pairs 4 (j & 7) + e
}
__device__ __forceinline__ void load_part(const Params &p, int t, int head, int j, QPart &r) {
    const uint16_t *src = p.qkv + (size_t)t * p.row + (size_t)head * 2 * HD + 4 * j;
    if (p.n_rot)
#pragma unroll
        for (int i = 0; i < 3; i++) r.pos[i] = p.pos3[3 * (size_t)t + i];
#pragma unroll
    for (int c = 0; c < 4; c++) r.w[c] = *(const uint2 *)(src + 64 * c);
}
__device__ __forceinline__ void make_part(const Params &p, const QNorm &n, const QPart &r, int j, _Float16 *row, int32_t *flag) {
    float x[4][4];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        x[c][0] = bf_lo(r.w[c].x);
        x[c][1] = bf_hi(r.w[c].x);
        x[c][2] = bf_lo(r.w[c].y);
        x[c][3] = bf_hi(r.w[c].y);
#pragma unroll
        for (int i = 0; i < 4; i++) ss += x[c][i] * x[c][i];
    }
    if (p.q_norm) {
        const float inv = rsqrtf(row16_sum(ss) / (float)HD + p.eps);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const float4 w = n.norm[c];
            x[c][0] *= inv * w.x;
            x[c][1] *= inv * w.y;
            x[c][2] *= inv * w.z;
            x[c][3] *= inv * w.w;
        }
    }
    if (p.n_rot) {
        const float freq[4] = {n.freq.x, n.freq.y, n.freq.z, n.freq.w};
        const int ax = j & 7;   // pair 4 ax + e: axis (4 ax + e) % 3 = (ax + e) % 3
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int axis = (ax + e) % 3;
            float sn, cn;
            rope_turns((float)(axis == 0 ? r.pos[0] : axis == 1 ? r.pos[1] : r.pos[2]) * freq[e], &sn, &cn);
            const float o = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x[0][e]), 0x128, 0xf, 0xf, false));   // lane j ^ 8's
            x[0][e] = j < 8 ? x[0][e] * cn - o * sn : x[0][e] * cn + o * sn;
        }
    }
    // split16's saturation: the largest magnitude decides (NaN passes through the maximum and fails the compare)
    float most = 0.f;
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int i = 0; i < 4; i += 2)
            most = __builtin_elementwise_maximum(most, __builtin_elementwise_maximum(fabsf(x[c][i]), fabsf(x[c][i + 1])));
    if (!(most <= p.f16_lim)) {
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) saturate(x[c][i], p.f16_lim);
        if (flag) __hip_atomic_store(flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int c = 0; c < 4; c++) *(uint2 *)(row + 64 * c + 4 * j) = make_uint2(pack_f16(x[c][0], x[c][1]), pack_f16(x[c][2], x[c][3]));
}

// Four finished outputs (dims d0 ..) of a row: times the sigmoid of their gates (loaded ahead), converted and stored.
__device__ __forceinline__ uint2 load_gate(const Params &p, int t, int head, int d0) {
    return p.gate ? *(const uint2 *)(p.qkv + (size_t)t * p.row + (size_t)head * 2 * HD + HD + d0) : make_uint2(0, 0);
}
__device__ __forceinline__ f32x4 gated(f32x4 o, uint2 gate) {
    return f32x4{o[0] * sigmoidf(bf_lo(gate.x)), o[1] * sigmoidf(bf_hi(gate.x)), o[2] * sigmoidf(bf_lo(gate.y)), o[3] * sigmoidf(bf_hi(gate.y))};
}
__device__ __forceinline__ void finish4(const Params &p, int t, int head, int d0, uint2 gate, f32x4 o, int32_t *flag) {
    if (p.gate) o = gated(o, gate);
    store_out4(p.out, ((size_t)t * p.nh + head) * HD + d0, o, p.out_type, p.f16_lim, flag);
}

// Partial results of a cut block: [split slot][kv head][row][256] unnormalised outputs, then
// [split slot][kv head][row][2] running maximum (of q . k) and sum.
__device__ __forceinline__ size_t partial_row(const Params &p, int slot, int kh, int row) {
    return ((size_t)slot * p.nkv + kh) * p.l.bm + row;
}
__device__ __forceinline__ float *partial_ml(const Params &p) {
    return p.partial + (size_t)p.l.max_slots * p.nkv * p.l.bm * HD;
}

// A barrier whose LDS accesses before it are done; loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Few rows (decoding, short questions): a workgroup takes an item's 16 MT rows over its pages, wave w the pages w, w + 4, ...
// Bound by memory: each page is read once, straight into registers, 4 KB pieces (four 1 KB loads) in a ring of
// four that K and V share: as a piece is used up, the one four later is loaded into its registers, so 16 KB a
// wave are always in flight, and with 16 rows two workgroups fit a CU, one's prologue and joins behind the
// other's stream. Page numbers and scales of a wave's next 64 pages are held one per lane. The four waves'
// results join through LDS. One token of 16/4 heads behind 130,000: 48.7 us, 5.5 TB/s; of 64 sequences of 30 to 8,000
// tokens (24/4): 49.8 us, 4.7 TB/s (a large read: 6.4, a large copy: 4.9), where CUs have work for 0.64 of the time. Short ones are bound by the chain of loads: 6.7 us for one
// token on 4,091.
constexpr int kRowsThreads = 256, kRowsWaves = 4;
template <int MT>
__global__ __launch_bounds__(kRowsThreads, MT == 1 ? 2 : 1) void kv8_attn_rows_kernel(Params p) {
    constexpr int BM = 16 * MT, OS = HD + 4;   // LDS row stride of the outputs
    __shared__ __attribute__((aligned(16))) float os[kRowsWaves][16][OS];   // holds the q rows before
    __shared__ float ml[kRowsWaves][BM][2];
    const int item = blockIdx.x / p.nkv, kh = blockIdx.x - item * p.nkv;
    const int4 *it = (const int4 *)(p.plan + p.l.items) + 2 * item;
    int4 e0 = it[0], e1 = it[1];
    if (!plan_has(p, H_ITEMS, item, e0, e1)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q16 = lane & 15, g = lane >> 4;
    const int lofs = (16 * (q16 >> 2) + (q16 & 3)) * 64 + 16 * g;   // the lane's piece of tile 0
    const int seq = e0.x, q0 = e0.y, L = e0.z, n_keys = e0.w, row0 = e1.x, rows = e1.y & 0xff, slot = (e1.y >> 8) - 1;
    const int pg0 = e1.z, pg1 = e1.w;
    const int32_t *table = p.tables + (size_t)seq * p.max_pages;
    // the wave's pages i = 0, 1, ... are pg0 + wave + 4 i; lane j holds number and scales of page (i & ~63) + j (a page
    // behind the item's last: the last's)
    const int n_mine = (pg1 - pg0 - wave + kRowsWaves - 1) / kRowsWaves;   // 0 or less: none
    auto number = [&](int i0) { return (unsigned)table[min(pg0 + wave + kRowsWaves * (i0 + lane), pg1 - 1)]; };
    unsigned ids = number(0);
    // Each wave makes a quarter of the rows. Loads go out in the order of their uses, and none of them conditionally:
    // a wave without a page loads the item's last.
    const int part = lane & 15;
    QNorm norm;
    QPart raw[MT];
    load_norm(p, part, norm);
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int fr = row0 + min(16 * m + 4 * wave + (lane >> 4), rows - 1), t = fr / p.group, head = kh * p.group + fr - t * p.group;
        load_part(p, q0 + t, head, part, raw[m]);
    }
    __builtin_amdgcn_sched_barrier(0);
    float kss, vss;
    auto scales = [&] {
        if (ids >= (unsigned)p.n_pages) ids = 0;
        ids = ids * p.nkv + kh;
        kss = p.k_scale[ids];
        vss = p.v_scale[ids];
    };
    auto landed = [&] { asm volatile("" : "+v"(kss), "+v"(vss)); };   // waited for here: the loop's waits are for its own loads
    u32x4 ring[4][4];
    auto load = [&](const uint8_t *pages, unsigned at, int c) {
        const uint8_t *src = pages + (size_t)at * PAGE_BYTES + 4096 * c + lofs;
#pragma unroll
        for (int t = 0; t < 4; t++) ring[c][t] = *(const u32x4 *)(src + 256 * t);
    };
    scales();
    unsigned at = __builtin_amdgcn_readlane(ids, 0);
#pragma unroll
    for (int c = 0; c < 4; c++) load(p.k_pages, at, c);
    _Float16 *const qs = (_Float16 *)&os[0][0][0];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int r = 16 * m + 4 * wave + (lane >> 4);
        make_part(p, norm, raw[m], part, qs + r * QS, p.ovf ? p.ovf + q0 : nullptr);
    }
    landed();
    lds_barrier();
    f16x8 q[MT][8];
    int last[MT];   // the last key the lane's row sees
#pragma unroll
    for (int m = 0; m < MT; m++) {
#pragma unroll
        for (int c = 0; c < 8; c++) q[m][c] = *(const f16x8 *)(qs + (16 * m + q16) * QS + 64 * (c >> 1) + 16 * g + 8 * (c & 1));
        last[m] = L + (row0 + min(16 * m + q16, rows - 1)) / p.group;
    }
    f32x4 o[MT][16];
    float mx[MT], sum[MT];
    int unit = 0;   // o is in units of 2^(unit - 5)
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
        const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kss), i & 63));
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
        const int now_unit = abs(ev - unit) <= kUnitSlack ? unit : ev;
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
            const float f = new_max(mx[m], text::xrow_max(top) * ks, kSlack, p.scale_log2);
            float add = 0.f;
            const float in_unit = kPUnit + (float)(ev - now_unit);
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = weight(s[m][t][e], ks, mx[m], p.scale_log2, in_unit);
                    add += x;
                    pb[m][t >> 1][4 * (t & 1) + e] = (_Float16)x;
                }
            sum[m] = sum[m] * f + add * pow2(now_unit - ev);
            const float fo = ldexpf(f, unit - now_unit);
            if (__any(fo != 1.f))
#pragma unroll
                for (int d = 0; d < 16; d++) o[m][d] *= fo;
        }
        unit = now_unit;
        unsigned next = 0;
        if constexpr (MORE) {
            if (((i + 1) & 63) == 0) {
                ids = number(i + 1);
                scales();
                landed();
            }
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
    // the lane will finish dims 4 lane .. of rows wave, wave + 4, ...: their gates, and their places in the output
    uint2 gate[MT][4];
    int unit_row[MT][4];
    if (slot < 0)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int fr = row0 + min(16 * m + 4 * i + wave, rows - 1), t = fr / p.group, head = kh * p.group + fr - t * p.group;
                gate[m][i] = load_gate(p, q0 + t, head, 4 * lane);
                unit_row[m][i] = (q0 + t) * p.nh + head;
            }
    // join the waves: each scales its outputs to the common maximum, to units of 1 (sums are of 2^5 P) and, if they
    // are not partial results, by the sum of all
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
        const int own = 16 * m + q16;
        float top = kNone, l = 0.f;
#pragma unroll
        for (int w = 0; w < kRowsWaves; w++) top = fmaxf(top, ml[w][own][0]);
#pragma unroll
        for (int w = 0; w < kRowsWaves; w++) l += ml[w][own][1] * __builtin_amdgcn_exp2f((ml[w][own][0] - top) * p.scale_log2);
        const float f = ldexpf(__builtin_amdgcn_exp2f((mx[m] - top) * p.scale_log2), unit) * (slot < 0 ? 1.f / l : 1.f);
        if (slot >= 0 && wave == 0 && g == 0 && own < rows) *(float2 *)(partial_ml(p) + 2 * partial_row(p, slot, kh, own)) = make_float2(top, l);
#pragma unroll
        for (int d = 0; d < 16; d++) *(f32x4 *)&os[wave][q16][64 * (d >> 2) + 16 * g + 4 * (d & 3)] = o[m][d] * f;
        __syncthreads();
        f32x4 x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] = *(const f32x4 *)&os[0][4 * i + wave][4 * lane];
#pragma unroll
            for (int w = 1; w < kRowsWaves; w++) x[i] += *(const f32x4 *)&os[w][4 * i + wave][4 * lane];
        }
        if (slot < 0 && p.gate)
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = gated(x[i], gate[m][i]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = 16 * m + 4 * i + wave;
            if (row >= rows) break;
            if (slot < 0) store_out4(p.out, (size_t)unit_row[m][i] * HD + 4 * lane, x[i], p.out_type, p.f16_lim, p.ovf ? p.ovf + q0 : nullptr);
            else *(f32x4 *)(p.partial + partial_row(p, slot, kh, row) * HD + 4 * lane) = x[i];
        }
        if (m + 1 < MT) __syncthreads();
    }
}

// Many rows (prompts): 128 rows an item, the pages' codes turned into f16 once and shared through LDS.
// On this chip conversions and the matrix products they feed hardly overlap (four conversions and a product take
// 25 clocks of a SIMD, a product 16), so no wave converts what another has: each of the eight takes an eighth of a
// page, and what is left to the inner loops is products and their LDS reads. Waves w and w + 4 share 32 rows: each
// takes the scores of half of a page's tokens, and O of half of the dims, so that an operand read from LDS serves
// two products and O and Q of 32 rows fit 128 registers, two waves a SIMD; the weights P go through LDS.
// Two phases a page, a barrier behind each: scores and softmax of page i while its V is written to LDS, then
// O += P V while K of page i + 1 is; so one slot of 32 KB is enough for each. Codes come into registers a page ahead.
//
// The maximum of a row is common to its two waves, and no page's own maximum is looked for while weights stay small: a
// wave whose sums of eight weights pass what the slack allows says so in a flag; behind the barrier all waves then
// take the pairs' new maxima and make that page's P again (the first page, and hardly ever after).
// 4 x 512 tokens of 16/4 heads on 2,048 take 92 to 97 us, 800 to 840 TFLOP/s (a large f16 product: 1,209); a page takes 4,500
// clocks of an item. No unit is full: of the time that a CU has work its matrix units are busy for 0.39 (2,050 clocks a page), other
// vector instructions are issued for 0.27, LDS moves data for 0.35 (conflicts 0.003). What bounds it is the turn of the phases: with two
// waves a SIMD and two barriers a page, all waves are in the same one, a wave stands at waits and barriers for 0.29 of
// its time and behind the other's instructions for 0.38.
constexpr int kTileThreads = 512;
struct TileLds {
    u32x4 k[32][64], v[32][64];   // operand [2 (4 c + t) + h][lane]
    u32x4 p[4][2][2][64];         // row group, half of the tokens, tile
    float top[4][2][32], sum[4][2][32];
    int flag[2];
};
// Operand reads and slot writes are issued by hand and waited for by count, so that reads run four operands ahead of
// the products and behind the conversions.
__device__ __forceinline__ unsigned lds_at(const void *ptr) { return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void *)ptr; }
template <int OFF>
__device__ __forceinline__ u32x4 lds_read(unsigned addr) {
    u32x4 r;
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(OFF) : "memory");
    return r;
}
template <int OFF, int STEP>
__device__ __forceinline__ void lds_read4(u32x4 (&r)[4], unsigned addr) {
    r[0] = lds_read<OFF>(addr);
    r[1] = lds_read<OFF + STEP>(addr);
    r[2] = lds_read<OFF + 2 * STEP>(addr);
    r[3] = lds_read<OFF + 3 * STEP>(addr);
}
template <int OFF>
__device__ __forceinline__ void lds_write(unsigned addr, f16x8 v) {
    asm volatile("ds_write_b128 %0, %1 offset:%2" ::"v"(addr), "v"(v), "i"(OFF) : "memory");
}
template <int N>
__device__ __forceinline__ void lds_wait(u32x4 (&r)[4]) {
    asm volatile("s_waitcnt lgkmcnt(%4)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]) : "i"(N));
}
template <int N>
__device__ __forceinline__ void lds_wait2(u32x4 (&r)[4], u32x4 &a, u32x4 &b) {
    asm volatile("s_waitcnt lgkmcnt(%6)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]), "+v"(a), "+v"(b) : "i"(N));
}
__global__ __launch_bounds__(kTileThreads, 2) void kv8_attn_tile_kernel(Params p) {
    __shared__ __attribute__((aligned(16))) TileLds sm;
    const int item = blockIdx.x / p.nkv, kh = blockIdx.x - item * p.nkv;
    const int4 *it = (const int4 *)(p.plan + p.l.items) + 2 * item;
    int4 e0 = it[0], e1 = it[1];
    if (!plan_has(p, H_ITEMS, item, e0, e1)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave & 3, half = wave >> 2;   // rows 32 rg .. 32 rg + 31, half of the tokens or dims
    const int q16 = lane & 15, g = lane >> 4;
    const int seq = e0.x, q0 = e0.y, L = e0.z, n_keys = e0.w, row0 = e1.x, rows = e1.y & 0xff, slot = (e1.y >> 8) - 1;
    const int pg0 = e1.z, n = e1.w - e1.z;
    const int32_t *table = p.tables + (size_t)seq * p.max_pages;
    int32_t *const flag_row = p.ovf ? p.ovf + q0 : nullptr;
    auto row_at = [&](int m, int &t, int &head) {
        const int fr = row0 + min(32 * rg + 16 * m + q16, rows - 1);
        t = fr / p.group;
        head = kh * p.group + fr - t * p.group;
    };
    // lane j: page (i & ~63) + j of the run that is being loaded (ids), or being scored (scales); behind the last: the last
    auto number = [&](int i0) { return (unsigned)table[pg0 + min(i0 + lane, n - 1)]; };
    auto in_pool = [&](unsigned id) { return (id < (unsigned)p.n_pages ? id : 0u) * p.nkv + kh; };
    unsigned ids = number(0);
    // 32 q rows at a time, 16 lanes each; loads go out in the order of their uses, none conditionally
    QNorm norm;
    QPart raw[4];
    load_norm(p, lane & 15, norm);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int fr = row0 + min(32 * k + (tid >> 4), rows - 1), t = fr / p.group;
        load_part(p, q0 + t, kh * p.group + fr - t * p.group, lane & 15, raw[k]);
    }
    __builtin_amdgcn_sched_barrier(0);
    const unsigned lofs = (16 * (q16 >> 2) + (q16 & 3)) * 64 + 16 * g;
    const unsigned pofs = (wave >> 1) * 4096 + (wave & 1) * 512 + lofs;   // pieces 2 wave and 2 wave + 1 of a page
    u32x4 kr[2], vr[2];
    auto load = [&](u32x4 (&r)[2], const uint8_t *pages, unsigned at) {
        const uint8_t *src = pages + (size_t)at * PAGE_BYTES + pofs;
        r[0] = *(const u32x4 *)src;
        r[1] = *(const u32x4 *)(src + 256);
    };
    auto store = [&](unsigned dst, const u32x4 &r) {   // two LDS writes
        lds_write<0>(dst, codes_f16(r[0], r[1]));
        lds_write<1024>(dst, codes_f16(r[2], r[3]));
    };
    const unsigned k_out = lds_at(sm.k[4 * wave]) + 16 * lane, v_out = lds_at(sm.v[4 * wave]) + 16 * lane;
    ids = in_pool(ids);
    float kss = p.k_scale[ids], vss = p.v_scale[ids];
    unsigned id_next = __builtin_amdgcn_readlane(ids, n > 1 ? 1 : 0);   // of page i + 1
    load(kr, p.k_pages, __builtin_amdgcn_readlane(ids, 0));
    load(vr, p.v_pages, __builtin_amdgcn_readlane(ids, 0));
    _Float16 *const qs = (_Float16 *)&sm;   // the rows lie where K, V and P will
#pragma unroll
    for (int k = 0; k < 4; k++) make_part(p, norm, raw[k], lane & 15, qs + (32 * k + (tid >> 4)) * QS, flag_row);
    if (tid < 2) sm.flag[tid] = 0;
    lds_barrier();
    f16x8 q[2][8];
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int c = 0; c < 8; c++) q[m][c] = *(const f16x8 *)(qs + (32 * rg + 16 * m + q16) * QS + 64 * (c >> 1) + 16 * g + 8 * (c & 1));
    lds_barrier();
    store(k_out, kr[0]);
    store(k_out + 2048, kr[1]);
    load(kr, p.k_pages, id_next);
    int last[2];   // the last key that the lane's row of each tile sees
#pragma unroll
    for (int m = 0; m < 2; m++) {
        int t, head;
        row_at(m, t, head);
        last[m] = L + t;
    }
    const int all_see = L + (row0 + min(32 * rg, rows - 1)) / p.group;   // keys up to this one are seen by all of the group's rows
    f32x4 o[2][8], s[2][2];
    float mx[2] = {kNone, kNone}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int d = 0; d < 8; d++) o[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    int unit = 0;   // o is in units of 2^(unit - 5)
    // operand 2 (4 c + t) + h of K: the group's tokens are tiles t = 2 half, 2 half + 1; of V: its dims groups c likewise
    const unsigned k_in = lds_at(sm.k) + 16 * lane + 4096 * half;
    const unsigned v_own = lds_at(sm.v) + 16 * lane + (16384 + 1024) * half, v_other = lds_at(sm.v) + 16 * lane + 16384 * half + 1024 * (half ^ 1);
    const unsigned p_in = lds_at(sm.p[rg][half ^ 1]) + 16 * lane, flag_in = lds_at(sm.flag);
    for (int i = 0; i < n; i++) {
        const int pg = pg0 + i;
        u32x4 r[2][4];
        lds_barrier();   // K of page i is there, V of page i - 1 is used up
        lds_read4<0, 1024>(r[0], k_in);       // dims 0-63: tiles' operands (t, h)
        lds_read4<8192, 1024>(r[1], k_in);    // dims 64-127
        if ((pg + 1) * PAGE > n_keys) {   // V codes behind the last key may be NaN, whose product with 0 is NaN
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const unsigned keep = keep_bytes(n_keys - pg * PAGE - 16 * g - 4 * w);
                vr[0][w] &= keep;
                vr[1][w] &= keep;
            }
        }
        if (i && (i & 63) == 0) {   // the scales of the next run
            const unsigned id = in_pool(number(i));
            kss = p.k_scale[id];
            vss = p.v_scale[id];
            asm volatile("" : "+v"(kss), "+v"(vss));   // waited for here and not at every page
        }
        const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kss), i & 63));
        const int ev = (int)(__builtin_amdgcn_readlane(__float_as_uint(vss), i & 63) >> 23) - 127;   // the V scale is 2^ev
        const int now_unit = abs(ev - unit) <= kUnitSlack ? unit : ev;
        const float in_unit = kPUnit + (float)(ev - now_unit), out_unit = pow2(now_unit - ev);
#pragma unroll
        for (int m = 0; m < 2; m++) s[m][0] = s[m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        // dims 64 c ..: four operands, eight products; V's codes go to LDS between them. Waits count what lies behind
        // the operands: the next four, and the writes of a piece (two)
        auto k_part = [&](auto c_t) {
            constexpr int C = decltype(c_t)::value;
            lds_wait<C == 0 ? 4 : C == 1 ? 6 : C == 2 ? 8 : 2>(r[C & 1]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const f16x8 a = __builtin_bit_cast(f16x8, r[C & 1][e]);
#pragma unroll
                for (int m = 0; m < 2; m++) s[m][e >> 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[m][2 * C + (e & 1)], s[m][e >> 1], 0, 0, 0);
            }
            if constexpr (C < 2) {
                lds_read4<8192 * (C + 2), 1024>(r[C & 1], k_in);
                store(v_out + 2048 * C, vr[C]);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        text::static_for<4>(k_part);
        load(vr, p.v_pages, id_next);
        const int key0 = pg * PAGE + 16 * g + 8 * half;
        if ((pg + 1) * PAGE > all_see + 1)
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (key0 + e > last[m]) s[m][e >> 2][e & 3] = -INFINITY;
        // P of the page from the scores and the maxima: the own half stays in registers, both lie in LDS
        f16x8 pb[2];
        float add[2];
        auto make_p = [&]() {
#pragma unroll
            for (int m = 0; m < 2; m++) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = weight(s[m][e >> 2][e & 3], ks, mx[m], p.scale_log2, in_unit);
                add[m] = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
                pb[m] = __builtin_bit_cast(f16x8, u32x4{pack_f16(x[0], x[1]), pack_f16(x[2], x[3]), pack_f16(x[4], x[5]), pack_f16(x[6], x[7])});
                sm.p[rg][half][m][lane] = __builtin_bit_cast(u32x4, pb[m]);
            }
        };
        make_p();
        // no weight of the page is past the slack while the sums of eight are not
        if (__any(fmaxf(add[0], add[1]) > kPMost)) sm.flag[i & 1] = 1;
        lds_barrier();   // V and P of page i are there, K of it is used up
        u32x4 pr[2];     // the other half's P operands
        unsigned moved;
        asm volatile("ds_read_b32 %0, %1" : "=v"(moved) : "v"(flag_in + 4 * (i & 1)) : "memory");
        pr[0] = lds_read<0>(p_in);
        pr[1] = lds_read<1024>(p_in);
        lds_read4<0, 2048>(r[0], v_own);
        asm volatile("s_waitcnt lgkmcnt(6)" : "+v"(moved));
        if (__builtin_amdgcn_readfirstlane(moved)) {
            lds_wait2<0>(r[0], pr[0], pr[1]);   // no read may land in a register that is used anew
            float top[2];
#pragma unroll
            for (int m = 0; m < 2; m++) {
                top[m] = s[m][0][0];
#pragma unroll
                for (int e = 1; e < 8; e++) top[m] = fmaxf(top[m], s[m][e >> 2][e & 3]);
                top[m] = text::xrow_max(top[m]) * ks;
                if (g == 0) sm.top[rg][half][16 * m + q16] = top[m];
            }
            lds_barrier();
#pragma unroll
            for (int m = 0; m < 2; m++) {
                const float f = new_max(mx[m], fmaxf(sm.top[rg][0][16 * m + q16], sm.top[rg][1][16 * m + q16]), 0.f, p.scale_log2);
                sum[m] *= f;
#pragma unroll
                for (int d = 0; d < 8; d++) o[m][d] *= f;
            }
            make_p();
            lds_barrier();
            pr[0] = lds_read<0>(p_in);
            pr[1] = lds_read<1024>(p_in);
            lds_read4<0, 2048>(r[0], v_own);
        }
        if (unit != now_unit) {
            const float f = pow2(unit - now_unit);
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int d = 0; d < 8; d++) o[m][d] *= f;
        }
        unit = now_unit;
#pragma unroll
        for (int m = 0; m < 2; m++) sum[m] = fmaf(add[m], out_unit, sum[m]);
        lds_read4<8192, 2048>(r[1], v_own);
        // first the own tokens' products (tiles 4 c ..), then the other half's; K's codes go to LDS between them
        auto v_part = [&](auto c_t) {
            constexpr int C = decltype(c_t)::value;
            if constexpr (C == 2) lds_wait2<8>(r[0], pr[0], pr[1]);
            else lds_wait<C == 0 ? 4 : C == 1 ? 6 : 2>(r[C & 1]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const f16x8 a = __builtin_bit_cast(f16x8, r[C & 1][e]);
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    const f16x8 w = C < 2 ? pb[m] : __builtin_bit_cast(f16x8, pr[m]);
                    o[m][4 * (C & 1) + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, w, o[m][4 * (C & 1) + e], 0, 0, 0);
                }
            }
            if constexpr (C < 2) {
                lds_read4<8192 * C, 2048>(r[C & 1], v_other);
                store(k_out + 2048 * C, kr[C]);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        text::static_for<4>(v_part);
        const int ahead = min(i + 2, n - 1);
        if (ahead == i + 2 && (ahead & 63) == 0) ids = in_pool(number(ahead));
        id_next = __builtin_amdgcn_readlane(ids, ahead & 63);
        load(kr, p.k_pages, id_next);
        if (tid == 0) sm.flag[(i + 1) & 1] = 0;
    }
    // The outputs go through LDS, 16 rows of the wave's 128 dims at a time, so that a store takes whole lines: lane dims
    // 4 (lane & 31) .. of rows 2 k + (lane >> 5). (Stored as they lie in registers, 16 bytes of each of 64 rows and dim
    // groups: 13,000 clocks of the 54,000 of a cut block of four pages; now 6,000 of 42,000.)
    int t_own[2], head_own[2], unit_own[2];   // token, q head and output row of the lane's own rows
    uint2 gate[2][8];
    const int d0 = 128 * half + 4 * (lane & 31);
#pragma unroll
    for (int m = 0; m < 2; m++) {
        row_at(m, t_own[m], head_own[m]);
        unit_own[m] = (q0 + t_own[m]) * p.nh + head_own[m];
    }
    auto of_row = [&](int own, int k) {   // what lane 2 k, or 2 k + 1 in the upper half, has of its row
        const int a = __builtin_amdgcn_readlane(own, 2 * k), b = __builtin_amdgcn_readlane(own, 2 * k + 1);
        return lane & 32 ? b : a;
    };
    if (slot < 0)
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int k = 0; k < 8; k++) gate[m][k] = load_gate(p, q0 + of_row(t_own[m], k), of_row(head_own[m], k), d0);
#pragma unroll
    for (int m = 0; m < 2; m++) {
        sum[m] = text::xrow_sum(sum[m]);
        if (g == 0) sm.sum[rg][half][16 * m + q16] = sum[m];
    }
    lds_barrier();
    constexpr int OS = 128 + 4;   // LDS row stride
    float *const os = (float *)&sm + wave * 16 * OS;
#pragma unroll
    for (int m = 0; m < 2; m++) {
        const float l = sm.sum[rg][0][16 * m + q16] + sm.sum[rg][1][16 * m + q16];
        const float f = slot < 0 ? pow2(unit) / l : pow2(unit);
#pragma unroll
        for (int d = 0; d < 8; d++) *(f32x4 *)(os + q16 * OS + 64 * (d >> 2) + 16 * g + 4 * (d & 3)) = o[m][d] * f;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own rows
        const int row0_m = 32 * rg + 16 * m;
        if (slot >= 0 && g == 0 && half == 0 && row0_m + q16 < rows)
            *(float2 *)(partial_ml(p) + 2 * partial_row(p, slot, kh, row0_m + q16)) = make_float2(mx[m], l);
        f32x4 x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = *(const f32x4 *)(os + (2 * k + (lane >> 5)) * OS + 4 * (lane & 31));
        auto put = [&](auto store) {   // one loop of stores for each kind, not a choice at each store
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (row0_m + 2 * k + (lane >> 5) < rows) store(k, x[k]);
        };
        auto finished = [&](auto type) {
            put([&](int k, f32x4 v) {
                store_out4(p.out, (size_t)of_row(unit_own[m], k) * HD + d0, v, decltype(type)::value, p.f16_lim, flag_row);
            });
        };
        if (slot >= 0) {
            float *const dst = p.partial + partial_row(p, slot, kh, row0_m + (lane >> 5)) * HD + d0;
            put([&](int k, f32x4 v) { *(f32x4 *)(dst + 2 * k * HD) = v; });
        } else {
            if (p.gate)
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = gated(x[k], gate[m][k]);
            if (p.out_type == CLEF_HIP_OUT_BF16) finished(std::integral_constant<int, CLEF_HIP_OUT_BF16>{});
            else if (p.out_type == CLEF_HIP_OUT_F16) finished(std::integral_constant<int, CLEF_HIP_OUT_F16>{});
            else finished(std::integral_constant<int, CLEF_HIP_OUT_F32>{});
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// Joins the items of cut blocks. A unit is a pass row's q head; one or four waves take its items in turn (by the
// plan's most cut block: what a wave reads is in flight at once), a lane four dims, and the first of them adds
// them up. The order is fixed, so results do not change from run to run. Bound by its chain of loads (header, token,
// block, partial results): 4.2 us for one token's 24 heads in 16 pieces, 8.2 for 16 heads in 128; the last workgroup of
// a block joining it instead took longer (64 sequences: 109 us for both against 52 + 7 with fences, 60.5 against 59.4
// with write-through stores).
constexpr int kJoinThreads = 256, kJoinWaves = kJoinThreads / 64, kJoinBatch = 8;
__global__ __launch_bounds__(kJoinThreads) void kv8_join_kernel(Params p) {
    __shared__ float os[kJoinWaves][HD], ml[kJoinWaves][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // a unit's wave or waves depend on the header: the token entries of both choices are asked for with it
    const int2 *const toks = (const int2 *)(p.plan + p.l.tok);
    const int2 tok1 = toks[min(((int)blockIdx.x * kJoinWaves + wave) / p.nh, p.T - 1)], tok4 = toks[min((int)blockIdx.x / p.nh, p.T - 1)];
    int4 first = {tok1.x, tok1.y, tok4.x, tok4.y}, head_words = {p.plan[H_MOST], p.plan[H_TOKENS], 0, 0};
    if (!plan_has(p, H_MOST, 1, first, head_words)) return;   // no block is cut
    const int most = head_words.x, units = head_words.y * p.nh;
    const int W = most <= kJoinBatch / 2 ? 1 : kJoinWaves, sub = wave & (W - 1), per = kJoinWaves / W;
    const int rounds = (units + per * (int)gridDim.x - 1) / (per * (int)gridDim.x);
    for (int round = 0; round < rounds; round++) {
        const int u = (round * (int)gridDim.x + (int)blockIdx.x) * per + wave / W;
        const int t = min(u / p.nh, p.T - 1), head = u % p.nh, kh = head / p.group;
        const int2 tok = round ? toks[t] : W == 1 ? make_int2(first.x, first.y) : make_int2(first.z, first.w);
        const int fr = tok.y * p.group + head - kh * p.group, b = tok.x + fr / p.l.bm;
        int4 blk = {0, 0, 0, 0};
        uint2 gate = {0, 0};
        if (u < units) {
            blk = ((const int4 *)(p.plan + p.l.blk))[b];
            gate = load_gate(p, t, head, 4 * lane);
        }
        const int n = __builtin_amdgcn_readfirstlane(blk.y), row = fr - blk.z;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float m = kNone, l = 0.f;
        if (n > 1)
            for (int k0 = sub; k0 < n; k0 += W * kJoinBatch) {
                float2 e[kJoinBatch];
                f32x4 x[kJoinBatch];
#pragma unroll
                for (int j = 0; j < kJoinBatch; j++) {
                    const size_t pr = partial_row(p, blk.w + min(k0 + W * j, n - 1), kh, row);
                    e[j] = *(const float2 *)(partial_ml(p) + 2 * pr);
                    x[j] = *(const f32x4 *)(p.partial + pr * HD + 4 * lane);
                }
                float top = m;
#pragma unroll
                for (int j = 0; j < kJoinBatch; j++) top = fmaxf(top, e[j].x);
                const float f = __builtin_amdgcn_exp2f((m - top) * p.scale_log2);
                o *= f;
                l *= f;
                m = top;
#pragma unroll
                for (int j = 0; j < kJoinBatch; j++) {
                    const float w = k0 + W * j < n ? __builtin_amdgcn_exp2f((e[j].x - top) * p.scale_log2) : 0.f;
                    l += e[j].y * w;
                    o += x[j] * w;
                }
            }
        if (W > 1) {
            *(f32x4 *)&os[wave][4 * lane] = o;
            if (lane == 0) {
                ml[wave][0] = m;
                ml[wave][1] = l;
            }
            __syncthreads();
            if (sub == 0) {
                float top = m;
                for (int w = 1; w < W; w++) top = fmaxf(top, ml[wave + w][0]);
                const float f = __builtin_amdgcn_exp2f((m - top) * p.scale_log2);
                o *= f;
                l *= f;
                for (int w = 1; w < W; w++) {
                    const float g = __builtin_amdgcn_exp2f((ml[wave + w][0] - top) * p.scale_log2);
                    l += ml[wave + w][1] * g;
                    o += *(const f32x4 *)&os[wave + w][4 * lane] * g;
                }
            }
        }
        if (n > 1 && sub == 0) {
            finish4(p, t, head, 4 * lane, gate, o * (1.f / l), p.ovf ? p.ovf + t - tok.y : nullptr);
        }
        if (W > 1) __syncthreads();
    }
}

}  // namespace kv8
}  // namespace clef_hip
