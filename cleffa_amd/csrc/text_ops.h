// Arithmetic that the text, vision and paged-cache kernels share: the gate's sigmoid, the rotary
// sin/cos, the output conversion (act16) and sums over parts of a wave.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <utility>

#include "bf16_ops.h"
#include "clef_hip_attn.h"

namespace clef_hip {

// sigmoid(x) = 1 / (1 + 2^(-x log2 e)) with the hardware exp2 and reciprocal (~1 ulp each).
__device__ __forceinline__ float sigmoidf(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-x * 1.4426950408889634f));
}

// sin and cos of a rotary angle (|x| < 2^20), without the memory tables of a general-range
// routine. Cody-Waite reduction by pi/2 in three parts with fma (the parts come from the double
// pi/2 split into floats), then Taylor polynomials on |r| <= pi/4: sin to r^9 (truncation
// < 2e-9), cos to r^10 (< 1e-10); about 1-2 ulp overall for the float angle the caller formed.
__device__ __forceinline__ void rope_sincos(float x, float *s, float *c) {
    constexpr double kHalfPi = 1.5707963267948966;
    constexpr float C1 = (float)kHalfPi;
    constexpr float C2 = (float)(kHalfPi - (double)C1);
    constexpr float C3 = (float)(kHalfPi - (double)C1 - (double)C2);
    const float j = __builtin_rintf(x * 0.63661977236758134f);
    float r = fmaf(-j, C1, x);
    r = fmaf(-j, C2, r);
    r = fmaf(-j, C3, r);
    const float r2 = r * r;
    float ps = fmaf(r2, 1.f / 362880.f, -1.f / 5040.f);
    ps = fmaf(ps, r2, 1.f / 120.f);
    ps = fmaf(ps, r2, -1.f / 6.f);
    const float sr = fmaf(ps * r2, r, r);
    float pc = fmaf(r2, -1.f / 3628800.f, 1.f / 40320.f);
    pc = fmaf(pc, r2, -1.f / 720.f);
    pc = fmaf(pc, r2, 1.f / 24.f);
    pc = fmaf(pc, r2, -0.5f);
    const float cr = fmaf(pc, r2, 1.f);
    const int q = (int)j & 3;   // x = j pi/2 + r
    const float sv = (q & 1) ? cr : sr, cv = (q & 1) ? sr : cr;
    *s = (q & 2) ? -sv : sv;
    *c = ((q + 1) & 2) ? -cv : cv;
}

// Output conversion of the o_proj operand (metal/clef.metal:98-106, act16): bf16, or f16
// that saturates to +-65504 and flags the record when |v| > lim or v is NaN, or plain f32.
__device__ __forceinline__ void store_out8(void *out, size_t idx, const float *v, int out_type,
                                           float lim, int32_t *flag) {
    if (out_type == CLEF_HIP_OUT_BF16) {
        u32x4 w = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                   pack_bf16(v[6], v[7])};
        *(u32x4 *)((uint16_t *)out + idx) = w;
    } else if (out_type == CLEF_HIP_OUT_F16) {
        _Float16 h[8];
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float x = v[j];
            if (!(fabsf(x) <= lim)) {
                bad = true;
                x = copysignf(65504.0f, x);
            }
            h[j] = (_Float16)x;
        }
        if (bad && flag) __hip_atomic_store(flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *(u32x4 *)((uint16_t *)out + idx) = __builtin_bit_cast(u32x4, h);
    } else {
        float *o = (float *)out + idx;
        *(float4 *)o = make_float4(v[0], v[1], v[2], v[3]);
        *(float4 *)(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
}

// act16 of four consecutive output elements of one row (metal/clef.metal:98-106), as store_out8:
// bf16, f16 saturating at +-65504 with the record flag when |v| > lim or NaN, or f32.
typedef float f32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void store_out4(void *out, size_t idx, f32x4_t v, int out_type, float lim, int32_t *flag) {
    if (out_type == CLEF_HIP_OUT_F32) {
        *(f32x4_t *)((float *)out + idx) = v;
        return;
    }
    uint16_t h[4];
    if (out_type == CLEF_HIP_OUT_BF16) {
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = __builtin_bit_cast(uint16_t, (__bf16)v[e]);
    } else {
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float x = v[e];
            if (!(fabsf(x) <= lim)) {
                bad = true;
                x = copysignf(65504.0f, x);
            }
            h[e] = __builtin_bit_cast(uint16_t, (_Float16)x);
        }
        if (bad && flag) __hip_atomic_store(flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    *(uint2 *)((uint16_t *)out + idx) = make_uint2(h[0] | ((unsigned)h[1] << 16), h[2] | ((unsigned)h[3] << 16));
}

__device__ __forceinline__ float row16_sum(float v) {   // sum over the lane's 16-lane row
    v += __builtin_amdgcn_update_dpp(0.f, v, 0x128, 0xf, 0xf, false);   // row_ror:8
    v += __builtin_amdgcn_update_dpp(0.f, v, 0x124, 0xf, 0xf, false);   // row_ror:4
    v += __builtin_amdgcn_update_dpp(0.f, v, 0x4e, 0xf, 0xf, false);    // quad_perm [2,3,0,1]
    v += __builtin_amdgcn_update_dpp(0.f, v, 0xb1, 0xf, 0xf, false);    // quad_perm [1,0,3,2]
    return v;
}

namespace text {
// Sum / max over the four 16-lane rows of a wave (v_permlane16_swap / v_permlane32_swap, VALU
// only, so no LDS traffic). Every lane gets the same bits.
__device__ __forceinline__ float xrow_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float m = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float xrow_sum(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float m = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}
template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F &&f) {
    static_for_impl(f, std::make_integer_sequence<int, N>{});
}
}  // namespace text

}  // namespace clef_hip
