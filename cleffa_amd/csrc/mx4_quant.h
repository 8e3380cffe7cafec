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
// block's 32 values in four neighbouring lanes. Codes go through LDS, so that a tile's 1 KB is stored in a row.
// Bound by memory: 4,096 x 6,144 f16 values 17.5 us, 3.6 TB/s of what it reads and writes (a large copy: 4.9).
constexpr int kQuantThreads = 256;
// RT: row tiles of a workgroup, whose loads go out together
template <int TYPE, int RT>
__global__ __launch_bounds__(kQuantThreads) void mx4_quantise_kernel(QuantParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t sc[RT][GROUP_BYTES];
    __shared__ __attribute__((aligned(16))) uint8_t cd[RT][4 * TILE_BYTES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int rt0 = blockIdx.x / p.kgroups * RT, kg = blockIdx.x % p.kgroups, kt = 4 * kg + wave;
    const int c = lane & 15, g = c >> 2;
    const int k = kt * KT + 8 * c;
    Values<TYPE> x[RT][4];
#pragma unroll
    for (int n = 0; n < RT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = ROWS * (rt0 + n) + 4 * i + (lane >> 4);
            Values<TYPE> zero{}, in = zero;
            if (t < p.rows && k < p.K) in = load8<TYPE>(p.x, (size_t)t * p.row + k);
            x[n][i] = in;
        }
#pragma unroll
    for (int n = 0; n < RT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 4 * i + (lane >> 4);
            float v[8];
            values8<TYPE>(x[n][i], v);
            unsigned m = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
            const int s = scale_byte(quad_max(m));
            *(unsigned *)(cd[n] + wave * TILE_BYTES + 16 * (ROWS * g + r) + 4 * (c & 3)) = s == kNanScale ? 0u : to_codes(v, scale_value(s));
            if ((c & 3) == 0) sc[n][4 * (ROWS * g + r) + wave] = (uint8_t)s;
        }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < RT; n++) {
        if (ROWS * (rt0 + n) + (lane & 15) >= p.rows) return;       // lane l now has row l % 16
        const size_t rt = rt0 + n;
        if (kt < p.ktiles) *(u32x4 *)(p.codes + (rt * p.ktiles + kt) * TILE_BYTES + 16 * lane) = *(const u32x4 *)(cd[n] + wave * TILE_BYTES + 16 * lane);
        if (wave == 0) *(unsigned *)(p.scales + (rt * p.kgroups + kg) * GROUP_BYTES + 4 * lane) = *(const unsigned *)(sc[n] + 4 * lane);
    }
}

// The values that codes stand for; the same split.
template <bool F32>
__global__ __launch_bounds__(kQuantThreads) void mx4_values_kernel(QuantParams p) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int rt = blockIdx.x / p.kgroups, kg = blockIdx.x % p.kgroups, kt = 4 * kg + wave;
    const int c = lane & 15, g = c >> 2;
    const int k = kt * KT + 8 * c;
    if (k >= p.K) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = 4 * i + (lane >> 4), t = ROWS * rt + r;
        if (t >= p.rows) continue;
        const unsigned w = *(const unsigned *)(p.codes + ((size_t)rt * p.ktiles + kt) * TILE_BYTES + 16 * (ROWS * g + r) + 4 * (c & 3));
        const float s = scale_value(p.scales[((size_t)rt * p.kgroups + kg) * GROUP_BYTES + 4 * (ROWS * g + r) + wave]);
        if constexpr (F32) {
            typedef __attribute__((ext_vector_type(2))) float f32x2;
            const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
            const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
            float *y = (float *)p.y + (size_t)t * p.row + k;
            *(float4 *)y = float4{a[0], a[1], b[0], b[1]};
            *(float4 *)(y + 4) = float4{d[0], d[1], e[0], e[1]};
        } else {
            u32x4 o;
            o[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
            o[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
            o[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
            o[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
            *(u32x4 *)((uint16_t *)p.y + (size_t)t * p.row + k) = o;
        }
    }
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
