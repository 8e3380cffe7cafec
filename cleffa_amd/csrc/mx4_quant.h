// Rows into microscaled 4-bit codes, back into 16 or 32 bits, and codes between this layout and the flat one of files.
#pragma once
#include "mx4_params.h"

namespace clef_hip {
namespace mx4 {

enum XType { X_BF16 = CLEF_HIP_OUT_BF16, X_F16 = CLEF_HIP_OUT_F16, X_F32 = CLEF_HIP_OUT_F32 };

// Scale byte of a block whose largest magnitude has these bits: 2^e the least power of two from 2^-127 on with max < 7 * 2^e.
// 7 = 1.75 * 4, and adding 0.25 to the mantissa carries into the exponent from 1.75 on. An infinity or a NaN takes the
// whole block.
__device__ __forceinline__ int scale_byte(unsigned max_bits) {
    if (max_bits >= 0x7f800000u) return kNanScale;
    const int s = (int)((max_bits + 0x200000u) >> 23) - 2;
    return s < 0 ? 0 : s > kMaxScale ? kMaxScale : s;
}
// The scale as the conversions take it: they read the exponent field alone, 255 as NaN.
__device__ __forceinline__ float scale_value(int s) { return __uint_as_float((unsigned)s << 23); }

// Eight f32 values to eight codes in a word, nearest with ties to even codes, at most 6.
__device__ __forceinline__ unsigned to_codes(const float (&v)[8], float scale) {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
    return r;
}

// Eight values of a row, as they lie in memory and in f32.
template <int TYPE>
struct Values {
    u32x4 w[TYPE == X_F32 ? 2 : 1];
};
template <int TYPE>
__device__ __forceinline__ Values<TYPE> load8(const void *x, size_t at) {
    Values<TYPE> r;
    const u32x4 *from = (const u32x4 *)((const uint8_t *)x + at * (TYPE == X_F32 ? 4 : 2));
    r.w[0] = from[0];
    if constexpr (TYPE == X_F32) r.w[1] = from[1];
    return r;
}
template <int TYPE>
__device__ __forceinline__ void values8(const Values<TYPE> &x, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < (TYPE == X_F32 ? 8 : 4); i++) {
        const unsigned word = x.w[i / 4][i % 4];     // a copy: a cast of the element itself takes element 0
        if constexpr (TYPE == X_F32) {
            v[i] = __uint_as_float(word);
        } else if constexpr (TYPE == X_BF16) {
            v[2 * i] = bf_lo(word);
            v[2 * i + 1] = bf_hi(word);
        } else {
            const f16x2 h = __builtin_bit_cast(f16x2, word);
            v[2 * i] = (float)h[0];
            v[2 * i + 1] = (float)h[1];
        }
    }
}

// The largest of four neighbouring lanes' values, to each of them.
__device__ __forceinline__ unsigned quad_max(unsigned m) {
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));
    return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));
}

// A workgroup makes 16 rows x 512 columns, each of its four waves a tile of 16 x 128: four loads of 4 rows x 256 bytes, a
// block's 32 values in four neighbouring lanes. Codes go through LDS, so that a tile's 1 KB is stored in a row (written there four
// to a bank, 3.9e5 conflict clocks on 1.1e5 instructions, behind the memory).
// Bound by memory: 4,096 x 6,144 f16 values 11.0 us one call behind the other, 5.8 TB/s of what it reads and writes; reading alone takes
// 8.0. Two row tiles a workgroup, for more loads in flight, took 11.5.
constexpr int kQuantThreads = 256;
template <int TYPE>
__global__ __launch_bounds__(kQuantThreads) void mx4_quantise_kernel(QuantParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t sc[GROUP_BYTES];
    __shared__ __attribute__((aligned(16))) uint8_t cd[4 * TILE_BYTES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int rt = blockIdx.x / p.kgroups, kg = blockIdx.x % p.kgroups, kt = 4 * kg + wave;
    const int c = lane & 15, g = c >> 2;
    const int k = kt * KT + 8 * c;
    Values<TYPE> x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int t = ROWS * rt + 4 * i + (lane >> 4);
        Values<TYPE> zero{}, in = zero;
        if (t < p.rows && k < p.K) in = load8<TYPE>(p.x, (size_t)t * p.row + k);
        x[i] = in;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = 4 * i + (lane >> 4);
        float v[8];
        values8<TYPE>(x[i], v);
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
        const int s = scale_byte(quad_max(m));
        *(unsigned *)(cd + wave * TILE_BYTES + 16 * (ROWS * g + r) + 4 * (c & 3)) = s == kNanScale ? 0u : to_codes(v, scale_value(s));
        if ((c & 3) == 0) sc[4 * (ROWS * g + r) + wave] = (uint8_t)s;
    }
    __syncthreads();
    if (ROWS * rt + (lane & 15) >= p.rows) return;       // lane l now has row l % 16
    if (kt < p.ktiles) *(u32x4 *)(p.codes + ((size_t)rt * p.ktiles + kt) * TILE_BYTES + 16 * lane) = *(const u32x4 *)(cd + wave * TILE_BYTES + 16 * lane);
    if (wave == 0) *(unsigned *)(p.scales + ((size_t)rt * p.kgroups + kg) * GROUP_BYTES + 4 * lane) = *(const unsigned *)(sc + 4 * lane);
}

// The values that codes stand for; the same split. Bound by memory: four times as many bytes out as in, stored past the caches, which
// keep what was there (4,096 x 6,144 to bf16 and the quantisation ahead of it 26.6 us with ordinary stores, 21.5 with these).
template <bool F32>
__global__ __launch_bounds__(kQuantThreads) void mx4_values_kernel(QuantParams p) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int rt = blockIdx.x / p.kgroups, kg = blockIdx.x % p.kgroups, kt = 4 * kg + wave;
    // a lane's values of a row: eight of bf16, or two runs of four of f32, 64 apart, so that 16 lanes store whole lines (4,096 x 5,152 17 us; with
    // eight in a row, half of each line a store, 31)
    constexpr int RUNS = F32 ? 2 : 1, V = F32 ? 4 : 8;
    const int c = lane & 15, r0 = lane >> 4;
    unsigned w[4][RUNS];
    float s[4][RUNS];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < RUNS; j++) {
            const int r = 4 * i + r0, k = 64 * j + V * c, place = ROWS * (k / BLOCK) + r;     // in the K tile
            const bool in = ROWS * rt + r < p.rows && KT * kt + k < p.K;
            const uint8_t *codes = p.codes + ((size_t)rt * p.ktiles + kt) * TILE_BYTES + 16 * place + k % BLOCK / 2;
            w[i][j] = !in ? 0u : F32 ? *(const uint16_t *)codes : *(const unsigned *)codes;
            s[i][j] = scale_value(in ? p.scales[((size_t)rt * p.kgroups + kg) * GROUP_BYTES + 4 * place + wave] : 0);
        }
    with_past(p.past, [&](auto PAST) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < RUNS; j++) {
                const int t = ROWS * rt + 4 * i + r0, k = KT * kt + 64 * j + V * c;
                if (t >= p.rows || k >= p.K) continue;
                if constexpr (F32) {
                    typedef __attribute__((ext_vector_type(2))) float f32x2;
                    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][j], s[i][j], 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][j], s[i][j], 1);
                    store_past(PAST, (f32x4 *)((float *)p.y + (size_t)t * p.row + k), f32x4{a[0], a[1], b[0], b[1]});
                } else {
                    u32x4 o;
                    o[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i][j], s[i][j], 0));
                    o[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i][j], s[i][j], 1));
                    o[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i][j], s[i][j], 2));
                    o[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i][j], s[i][j], 3));
                    store_past(PAST, (u32x4 *)((uint16_t *)p.y + (size_t)t * p.row + k), o);
                }
            }
    });
}

// Flat codes and scales into this layout (TO), or back: a thread a block. Blocks beyond K become 0.
template <bool TO>
__global__ __launch_bounds__(256) void mx4_pack_kernel(PackParams p) {
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int blocks = TO ? 16 * p.kgroups : p.K / BLOCK;
    const size_t t = id / blocks;
    const int b = (int)(id % blocks);
    if (t >= (size_t)p.rows) return;
    const size_t rt = t / ROWS;
    const int r = (int)(t % ROWS), kt = b >> 2, g = b & 3;
    uint8_t *codes = p.codes + (rt * p.ktiles + kt) * TILE_BYTES + 16 * (ROWS * g + r);
    uint8_t *scale = p.scales + (rt * p.kgroups + (kt >> 2)) * GROUP_BYTES + 4 * (ROWS * g + r) + (kt & 3);
    uint8_t *flat = p.flat_codes + t * (size_t)(p.K / 2) + 16 * b, *flat_scale = p.flat_scales + t * (size_t)(p.K / BLOCK) + b;
    if constexpr (TO) {
        const bool in = b < p.K / BLOCK;
        if (kt < p.ktiles) *(u32x4 *)codes = in ? *(const u32x4 *)flat : u32x4{0, 0, 0, 0};
        *scale = in ? *flat_scale : 0;
    } else {
        *(u32x4 *)flat = *(const u32x4 *)codes;
        *flat_scale = *scale;
    }
}

}  // namespace mx4
}  // namespace clef_hip
