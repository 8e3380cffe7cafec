// Y = X . W^T (+ residual) with W in microscaled 4 bits and X in the same or in bf16.
#pragma once
#include <utility>

#include "mx4_params.h"

namespace clef_hip {
namespace mx4 {

typedef __attribute__((ext_vector_type(8))) int i32x8;

__device__ __forceinline__ i32x8 operand(u32x4 c) { return i32x8{(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0}; }
// 16 x 16 outputs, 128 deep: A = 16 rows of W (columns of Y), B = 16 rows of X. Lane l's accumulators are columns
// 4 (l / 16) .. + 3 of row l % 16. The scales are the low bytes of sw and sx.
__device__ __forceinline__ f32x4 mfma4(u32x4 w, u32x4 x, f32x4 acc, int sw, int sx) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(x), acc, 4, 4, 0, sw, 0, sx);
}
// Eight codes as bf16, exactly (but for magnitudes beyond bf16).
__device__ __forceinline__ bf16x8 widen(unsigned c, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
    return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// The sums of a workgroup's W waves, each of MT x NT tiles of 16 x 16, added in order through LDS and stored.
template <int MT, int NT, int W>
__device__ __forceinline__ void join_waves(const GemmParams &p, const f32x4 (&acc)[MT][NT], f32x4 (*part)[MT * NT][64], int t0, int n0) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) part[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int u = wave; u < MT * NT; u += W) {
        f32x4 s = part[0][u][lane];
#pragma unroll
        for (int w = 1; w < W; w++) s += part[w][u][lane];
        const int t = 16 * (t0 + u / NT) + (lane & 15), c = 16 * (n0 + u % NT) + 4 * (lane >> 4);
        if (t < p.T && c < p.N) store4(p, t, c, s);
    }
}

// Few 4-bit rows: MT x NT tiles of 16 rows and 16 columns a workgroup, whose W waves share the K tiles and add their sums in LDS in a
// fixed order. Operands come straight from memory into D buffers of a K tile each. Nothing holds the loads where they are written: the
// compiler moves the last buffer's down to their products, so that D - 1 K tiles are in flight, and with D = 2 none behind the second of
// two. 45 rows x 14,336 x 5,120 read 39 MB in 9.9 us, and 16 rows x 5,120 x 6,144 16.8 MB in 5.1: latency, of the five or six K tiles of a wave one after
// the other. What deeper or pinned loads would give is not measured.
template <int MT, int NT, int W, int D>
__global__ __launch_bounds__(64 * W) void mx4_rows_kernel(GemmParams p) {
    __shared__ f32x4 part[W][MT * NT][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int n_tiles = ceil_div(p.N, 16), t_tiles = ceil_div(p.T, 16), nb = ceil_div(n_tiles, NT);
    const int n0 = (blockIdx.x % nb) * NT, t0 = (blockIdx.x / nb) * MT;
    const int k_lo = p.w.ktiles * wave / W, k_hi = p.w.ktiles * (wave + 1) / W;
    struct Ops {
        u32x4 w[NT], x[MT];
        int ws[NT], xs[MT];
    };
    auto load = [&](Ops &o, int kt) __attribute__((always_inline)) {
        kt = min(kt, k_hi - 1);
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int nt = min(n0 + j, n_tiles - 1);
            o.w[j] = *(const u32x4 *)(p.w.tile(nt, kt) + 16 * lane);
            o.ws[j] = *(const int *)(p.w.group(nt, kt >> 2) + 4 * lane);
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const int tt = min(t0 + i, t_tiles - 1);
            o.x[i] = *(const u32x4 *)(p.x.tile(tt, kt) + 16 * lane);
            o.xs[i] = *(const int *)(p.x.group(tt, kt >> 2) + 4 * lane);
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (k_lo < k_hi) {
        Ops ops[D];
#pragma unroll
        for (int d = 0; d < D; d++) load(ops[d], k_lo + d);
        for (int kt = k_lo; kt < k_hi; kt += D) {
#pragma unroll
            for (int d = 0; d < D; d++) {
                const int sh = 8 * (kt + d & 3);
                if (kt + d < k_hi) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int i = 0; i < MT; i++)
                            acc[i][n] = mfma4(ops[d].w[n], ops[d].x[i], acc[i][n], (unsigned)ops[d].ws[n] >> sh, (unsigned)ops[d].xs[i] >> sh);
                }
                load(ops[d], kt + d + D);
            }
        }
    }
    join_waves<MT, NT, W>(p, acc, part, t0, n0);
}

}  // namespace mx4
}  // namespace clef_hip
