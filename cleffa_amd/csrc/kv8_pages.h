// Writing and reading the pages of the 8-bit prefix cache.
//
// A page holds 64 tokens of a kv head as OCP e4m3 codes, K [4][64][64] (dim group, token, dim) and V
// [256][64] (dim, token), each with one scale 2^e: value = code * 2^e, e the least integer from -64 on with
// max|x| <= 448 * 2^e. A power of two costs a floating-point code nothing (its step is relative), makes
// rescaling exact but for codes that become subnormal, and folds into the attention's arithmetic. Both
// orders give a wave of the attention kernels its matrix operands as whole 16-byte pieces (kv8_attn.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bf16_ops.h"
#include "kv8_params.h"
#include "text_ops.h"

namespace clef_hip {
namespace kv8 {

// 2^e of a page whose largest magnitude is `most`: 448 = 1.75 * 2^8, so e is most's exponent less 8, one
// more where its fraction passes 1.75.
__device__ __forceinline__ float page_scale(float most) {
    const unsigned b = __float_as_uint(most);
    const int e = max((int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0), -64);
    return __uint_as_float((unsigned)(e + 127) << 23);
}
// The exact reciprocal of a scale 2^e, |e| <= 64.
__device__ __forceinline__ float inverse_pow2(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// Four values, already divided by the scale, as e4m3 codes (nearest, ties to even; |x| <= 448 by the scale's choice).
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
// Four codes times f, coded again (f = old scale / new scale, at most 1).
__device__ __forceinline__ unsigned recode4(unsigned w, float f) {
    return codes4(__builtin_amdgcn_cvt_f32_fp8(w, 0) * f, __builtin_amdgcn_cvt_f32_fp8(w, 1) * f,
                  __builtin_amdgcn_cvt_f32_fp8(w, 2) * f, __builtin_amdgcn_cvt_f32_fp8(w, 3) * f);
}

// |x| > lim or NaN saturates to +-65504 (split16's rule for the 16-bit planes); returns whether it did.
__device__ __forceinline__ bool saturate(float &x, float lim) {
    const bool bad = !(fabsf(x) <= lim);
    if (bad) x = copysignf(65504.f, x);
    return bad;
}

// sin and cos of an angle by the hardware functions of revolutions, the fraction exact in two products: 4e-7 off at
// most up to 10^6 (measured over 4 million angles), against 5e-4 of an f16 operand and 6e-2 of a code. That is more
// than the 16-bit path's rope_sincos (1.3 * 2^-24 up to 2^21): of 11,000 keys that rotate to near a border between two codes none within
// 3 * 2^-24 of the pair's magnitudes changed sides, with rope_sincos none within 1 * 2^-24; of 4.2 million codes of a 4,096-token append
// 3, 8 and 3 are not float64's (three seeds), with rope_sincos 2, 5 and 3, with f32 torch 0, 6 and 6. It would take longer:
// that append 13.8 us for 12.0, 4 x 512 tokens on 2,048 94.4 for 92.7. Angles behind 2^24 stay within 7e-6.
__device__ __forceinline__ void rope_turns(float x, float *s, float *c) {
    constexpr double kTurn = 0.15915494309189535;   // 1 / (2 pi)
    constexpr float C1 = (float)kTurn, C2 = (float)(kTurn - (double)C1);
    const float j = __builtin_rintf(x * C1);
    const float r = fmaf(x, C2, fmaf(x, C1, -j));
    *s = __builtin_amdgcn_sinf(r);
    *c = __builtin_amdgcn_cosf(r);
}

// The page's new scale from each thread's largest magnitude; old rows keep the page's scale as a floor.
__device__ __forceinline__ float shared_scale(float most, float before, float *red) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
    __syncthreads();
    return fmaxf(page_scale(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]))), before);
}

// A pass's new tokens into the pages. Workgroup (item, kv head, K or V): the new tokens of one page, which
// lie in consecutive pass rows. The page's rows before them keep their values; where the scale has to
// grow they are coded again. Nothing else of the page is written, and no other workgroup writes it.
constexpr int kAppendThreads = 256;
__global__ __launch_bounds__(kAppendThreads) void kv8_append_kernel(Params p) {
    __shared__ float red[4];
    const int kh = blockIdx.x % p.nkv, item = blockIdx.x / p.nkv, tid = threadIdx.x;
    int4 it = ((const int4 *)(p.plan + p.l.app))[item];   // the grid ends with the list's room
    int4 none = {0, 0, 0, 0};
    if (!plan_has(p, H_APPEND, item, it, none)) return;
    const int page = it.x, t0 = it.y, off = it.z & 0xff, n = it.z >> 8, flag = it.w;
    if ((unsigned)page >= (unsigned)p.n_pages) return;
    const size_t at = (size_t)page * p.nkv + kh;
    bool bad = false;
    float most = 0.f;
    if (blockIdx.y == 0) {
        // K: 16 lanes a row, 16 rows a round; lane k holds dims 8k + e and 32 + 8k + e (e < 8) for k < 4, so
        // that its rotary pairs are its own, and 64 + 16 (k - 4) + e (e < 16) above
        const int k = tid & 15, rr = tid >> 4;
        const int d0 = k < 4 ? 8 * k : 64 + 16 * (k - 4), d1 = k < 4 ? 32 + 8 * k : d0 + 8;
        const uint16_t *src = p.qkv + (size_t)p.nh * 2 * HD + (size_t)kh * HD;
        u32x4 raw[4][2];
        int pos[4][3];
        float w[16], freq[8];
#pragma unroll
        for (int m = 0; m < 4; m++) {
            if (16 * m >= n) break;
            const int t = t0 + min(16 * m + rr, n - 1);
            raw[m][0] = *(const u32x4 *)(src + (size_t)t * p.row + d0);
            raw[m][1] = *(const u32x4 *)(src + (size_t)t * p.row + d1);
            if (p.n_rot)
#pragma unroll
                for (int c = 0; c < 3; c++) pos[m][c] = p.pos3[3 * (size_t)t + c];
        }
        if (p.k_norm)
#pragma unroll
            for (int i = 0; i < 16; i++) w[i] = p.k_norm[(i < 8 ? d0 : d1) + (i & 7)];
        if (p.n_rot)
#pragma unroll
            for (int e = 0; e < 8; e++) freq[e] = p.inv_freq[(8 * k + e) & 31];
        const float before = off ? p.k_scale[at] : 0.f;
        float x[4][16];
#pragma unroll
        for (int m = 0; m < 4; m++) {
            if (16 * m >= n) break;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[m][2 * i] = bf_lo(raw[m][0][i]);
                x[m][2 * i + 1] = bf_hi(raw[m][0][i]);
                x[m][8 + 2 * i] = bf_lo(raw[m][1][i]);
                x[m][9 + 2 * i] = bf_hi(raw[m][1][i]);
            }
            if (p.k_norm) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 16; i++) ss += x[m][i] * x[m][i];
                const float inv = rsqrtf(row16_sum(ss) / (float)HD + p.eps);
#pragma unroll
                for (int i = 0; i < 16; i++) x[m][i] *= inv * w[i];
            }
            if (p.n_rot && k < 4) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int axis = (8 * k + e) % 3;
                    float sn, cn;
                    rope_turns((float)(axis == 0 ? pos[m][0] : axis == 1 ? pos[m][1] : pos[m][2]) * freq[e], &sn, &cn);
                    const float a = x[m][e], b = x[m][e + 8];
                    x[m][e] = a * cn - b * sn;
                    x[m][e + 8] = b * cn + a * sn;
                }
            }
            // split16's saturation: the largest magnitude decides (NaN passes through the maximum and fails the compare)
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i += 2)
                top = __builtin_elementwise_maximum(top, __builtin_elementwise_maximum(fabsf(x[m][i]), fabsf(x[m][i + 1])));
            if (!(top <= p.f16_lim)) {
                bad = true;
                top = 65504.f;
#pragma unroll
                for (int i = 0; i < 16; i++) saturate(x[m][i], p.f16_lim);
            }
            most = fmaxf(most, top);
        }
        const float s = shared_scale(most, before, red), f = inverse_pow2(s);
        uint8_t *pg = p.k_pages + at * PAGE_BYTES;
#pragma unroll
        for (int m = 0; m < 4; m++) {
            const int j = 16 * m + rr;
            if (j >= n) break;
            u32x4 c;
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = codes4(x[m][4 * i] * f, x[m][4 * i + 1] * f, x[m][4 * i + 2] * f, x[m][4 * i + 3] * f);
            uint8_t *row = pg + (size_t)(off + j) * 64;
            *(uint2 *)(row + (d0 >> 6) * 4096 + (d0 & 63)) = make_uint2(c[0], c[1]);
            *(uint2 *)(row + (d1 >> 6) * 4096 + (d1 & 63)) = make_uint2(c[2], c[3]);
        }
        if (off && s > before)
            for (int c = tid; c < PAGE_BYTES / 16; c += kAppendThreads)
                if ((c >> 2 & 63) < off) {
                    u32x4 v = *(u32x4 *)(pg + 16 * c);
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = recode4(v[i], before * f);
                    *(u32x4 *)(pg + 16 * c) = v;
                }
        __syncthreads();   // every thread has read the old scale
        if (tid == 0) p.k_scale[at] = s;
    } else {
        // V: thread (dims 8c .. 8c + 7, tokens 8a .. 8a + 7 of the page): eight rows' 16-byte pieces, stored as
        // eight 8-byte runs of V^T
        const int c = tid & 31, a = tid >> 5;
        const uint16_t *src = p.qkv + (size_t)p.nh * 2 * HD + (size_t)(p.nkv + kh) * HD + 8 * c;
        const int lo = max(off - 8 * a, 0), hi = min(off + n - 8 * a, 8);   // the thread's new tokens
        u32x4 v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] = u32x4{0u, 0u, 0u, 0u};
            if (i >= lo && i < hi) v[i] = *(const u32x4 *)(src + (size_t)(t0 + 8 * a + i - off) * p.row);
        }
        const float before = off ? p.v_scale[at] : 0.f;
        // bf16 magnitudes are ordered as integers are, NaN above all others
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, max(v[i][e] << 16 & 0x7fffffffu, v[i][e] & 0x7fff0000u));
        bad = !(__uint_as_float(top) <= p.f16_lim);
        most = bad ? 65504.f : __uint_as_float(top);
        const float s = shared_scale(most, before, red), f = inverse_pow2(s);
        uint8_t *pg = p.v_pages + at * PAGE_BYTES;
        // old tokens: those of this thread's runs, so that no other thread writes them
        const bool again = off && s > before;
        if (hi > lo || (again && 8 * a < off)) {
            // bytes to write: new ones, and old ones where the scale grew
            const int first = again ? 0 : lo, last = max(hi, min(off - 8 * a, 8));
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[i] = e & 1 ? bf_hi(v[i][e / 2]) : bf_lo(v[i][e / 2]);
                    if (bad) saturate(x[i], p.f16_lim);
                    x[i] *= f;
                }
                uint8_t *run = pg + (8 * c + e) * PAGE + 8 * a;
                uint2 o = make_uint2(codes4(x[0], x[1], x[2], x[3]), codes4(x[4], x[5], x[6], x[7]));
                if (first == 0 && lo > 0) {   // old tokens share the run
                    const uint2 w = *(const uint2 *)run;
                    const uint2 r = make_uint2(recode4(w.x, before * f), recode4(w.y, before * f));
                    const uint64_t keep = lo >= 8 ? ~0ull : (1ull << 8 * lo) - 1;
                    const uint64_t both = ((uint64_t)r.y << 32 | r.x) & keep | ((uint64_t)o.y << 32 | o.x) & ~keep;
                    o = make_uint2((unsigned)both, (unsigned)(both >> 32));
                }
                if (first == 0 && last == 8) *(uint2 *)run = o;
                else
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (i >= first && i < last) run[i] = (uint8_t)((i < 4 ? o.x : o.y) >> 8 * (i & 3));
            }
        }
        __syncthreads();
        if (tid == 0) p.v_scale[at] = s;
    }
    if (bad && p.ovf) __hip_atomic_store(p.ovf + flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct ReadParams {
    const uint8_t *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    const int32_t *tables, *state, *first_page, *cu;
    uint16_t *k_plane, *vt_plane;
    int n_seq, max_pages, n_pages, nkv, kvT;
};

// Eight codes as f16 or bf16 of code * s (the conversion's scale operand is a power of two, as the pages' are);
// f16 values beyond 65504 (only 65536, of a page with e = 8) become 65504.
__device__ __forceinline__ u32x4 to_f16(unsigned a, unsigned b, float s) {
    float x[8];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const unsigned c = w ? b : a;
        x[4 * w] = __builtin_amdgcn_cvt_f32_fp8(c, 0);
        x[4 * w + 1] = __builtin_amdgcn_cvt_f32_fp8(c, 1);
        x[4 * w + 2] = __builtin_amdgcn_cvt_f32_fp8(c, 2);
        x[4 * w + 3] = __builtin_amdgcn_cvt_f32_fp8(c, 3);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = fminf(fmaxf(x[i] * s, -65504.f), 65504.f);
    return u32x4{pack_f16(x[0], x[1]), pack_f16(x[2], x[3]), pack_f16(x[4], x[5]), pack_f16(x[6], x[7])};
}
__device__ __forceinline__ u32x4 to_bf16(unsigned a, unsigned b, float s) {
    u32x4 o;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const unsigned c = w ? b : a;
        o[2 * w] = pack_bf16(__builtin_amdgcn_cvt_f32_fp8(c, 0) * s, __builtin_amdgcn_cvt_f32_fp8(c, 1) * s);
        o[2 * w + 1] = pack_bf16(__builtin_amdgcn_cvt_f32_fp8(c, 2) * s, __builtin_amdgcn_cvt_f32_fp8(c, 3) * s);
    }
    return o;
}

// Pages back into 16-bit planes. Workgroup (piece, kv head): NP pages, N = 64 NP tokens. Piece i belongs to the last
// sequence r with cu[r] / N + r <= i and is its pages NP (i - cu[r] / N - r) and up (from first_page on): sequence r
// has cu[r + 1] / N - cu[r] / N + 1 pieces, enough for its cu[r + 1] - cu[r] rows. The sequence is found by all threads
// counting at once, a search's loads one after the other would take longer than the copy. Bound by memory (a byte
// in, two out): every load and store instruction of a wave covers whole lines, a lane taking eight codes to sixteen
// bytes. Two pages make 256 bytes of a V^T row (79,000 tokens, 4 heads: 120.5 -> 106.6 us, 4.6 TB/s), which small reads
// lack the workgroups for (4,091 tokens: 7.3 -> 9.1 us): the launch takes two from 8 workgroups a CU on.
template <int NP>
__global__ __launch_bounds__(256 * NP) void kv8_read_kernel(ReadParams p) {
    constexpr int kReadThreads = 256 * NP, kReadTokens = PAGE * NP, LANES = 8 * NP;   // lanes a V^T row
    const int kh = blockIdx.x % p.nkv, piece = blockIdx.x / p.nkv, tid = threadIdx.x;
    int r = -1;
    for (int r0 = 0; r0 < p.n_seq; r0 += kReadThreads) {
        const int i = r0 + tid;
        r += __syncthreads_count(i < p.n_seq && p.cu[i] / kReadTokens + i <= piece);
    }
    if (r < 0) return;
    const int row0 = p.cu[r], j = piece - row0 / kReadTokens - r;
    const int first = p.first_page ? p.first_page[r] : 0;
    const long pg = (long)first + NP * j;
    if (j < 0 || row0 < 0 || row0 % 8 || first < 0 || pg >= p.max_pages) return;
    // rows of the piece: the sequence's tokens, the room of its plane rows, the plane's end and the table's bound them
    const long left = (long)min(p.cu[r + 1], p.kvT) - row0 - (long)j * kReadTokens;
    const long have = min((long)p.state[2 + 2 * r], (long)p.max_pages * PAGE) - pg * PAGE;
    const int n = (int)min(min(left, have), (long)kReadTokens);
    if (n <= 0) return;
    const int32_t *table = p.tables + (size_t)r * p.max_pages + pg;
    const unsigned page0 = (unsigned)table[0], page1 = NP > 1 && n > PAGE ? (unsigned)table[1] : page0;
    if (page0 >= (unsigned)p.n_pages || page1 >= (unsigned)p.n_pages) return;
    const size_t at0 = (size_t)page0 * p.nkv + kh, at1 = (size_t)page1 * p.nkv + kh;
    const float ks0 = p.k_scale[at0], ks1 = p.k_scale[at1], vs0 = p.v_scale[at0], vs1 = p.v_scale[at1];
    const size_t base = (size_t)row0 + (size_t)j * kReadTokens;
    // K: thread (token, 8 dims), 32 lanes a row; V: thread (dim, 8 tokens)
    uint2 k[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int id = tid + kReadThreads * i, tok = id >> 5, part = id & 31, t8 = id % LANES;
        k[i] = *(const uint2 *)(p.k_pages + (tok < PAGE ? at0 : at1) * PAGE_BYTES + (part >> 3) * 4096 + (tok & 63) * 64 + (part & 7) * 8);
        v[i] = *(const uint2 *)(p.v_pages + (t8 < 8 ? at0 : at1) * PAGE_BYTES + id / LANES * PAGE + (t8 & 7) * 8);
    }
    uint16_t *const k_dst = p.k_plane + ((size_t)kh * p.kvT + base) * HD;
    uint16_t *const v_dst = p.vt_plane + (size_t)kh * HD * p.kvT + base;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int id = tid + kReadThreads * i, tok = id >> 5, part = id & 31;
        if (tok < n) __builtin_nontemporal_store(to_f16(k[i].x, k[i].y, tok < PAGE ? ks0 : ks1), (u32x4 *)(k_dst + tok * HD + 8 * part));
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int id = tid + kReadThreads * i, d = id / LANES, t0 = 8 * (id % LANES), m = n - t0;
        uint16_t *dst = v_dst + (size_t)d * p.kvT + t0;
        const u32x4 w = to_bf16(v[i].x, v[i].y, t0 < PAGE ? vs0 : vs1);
        if (m >= 8) __builtin_nontemporal_store(w, (u32x4 *)dst);
        else if (m > 0) {   // the last tokens: four, two, one
            if (m & 4) *(uint2 *)dst = make_uint2(w[0], w[1]);
            if (m & 2) *(unsigned *)(dst + (m & 4)) = m & 4 ? w[2] : w[0];
            if (m & 1) dst[m - 1] = (uint16_t)(m & 4 ? (m & 2 ? w[3] : w[2]) : (m & 2 ? w[1] : w[0]));
        }
    }
}

}  // namespace kv8
}  // namespace clef_hip
