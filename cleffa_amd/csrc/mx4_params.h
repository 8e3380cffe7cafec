// Microscaled 4-bit matrices: their layout and the kernels' argument blocks (internal; the interface is documented in
// include/clef_hip_attn.h).
//
// A matrix [rows][K] holds e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one scale 2^(s - 127) for each 32
// of a row. It lies in the order in which a wave feeds the scaled matrix instruction 16x16x128, whose lane l takes
// 32 codes along K of row l % 16, block l / 16, and their scale:
//   codes   [row tile of 16][K tile of 128][block 4][row 16][16 bytes]: a tile is 1 KB, lane l's 16 bytes at 16 l, the lower
//           four bits of a byte first;
//   scales  [row tile of 16][K group of 512][block 4][row 16][K tile 4] bytes: lane l's word at 4 l holds its scales for the
//           four tiles of a group, which the instruction selects from by byte.
// So every load of codes is 1 KB in a row and every load of scales 256 bytes; copied into LDS as they are, lanes read 16
// bytes each in order, without bank conflicts or a swizzle. Both operands of a product have this layout. Rows of the last
// row tile beyond the matrix are never used; codes beyond K are 0.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "bf16_ops.h"
#include "clef_hip_attn.h"

namespace clef_hip {
namespace mx4 {

constexpr int BLOCK = CLEF_HIP_MX4_BLOCK;     // values that share a scale
constexpr int ROWS = 16, KT = 128, KG = 512;  // a tile's rows and columns, columns of a scale group
constexpr int TILE_BYTES = ROWS * KT / 2, GROUP_BYTES = ROWS * KG / BLOCK;
constexpr int kMaxScale = 252;                // 6 * 2^(252 - 127) is the largest finite value
constexpr int kNanScale = 255;

__host__ __device__ inline int ceil_div(int a, int b) { return a / b + (a % b != 0); }

struct Matrix {
    const uint8_t *codes, *scales;
    int rows, ktiles, kgroups;
    __device__ const uint8_t *tile(int rt, int kt) const { return codes + ((size_t)rt * ktiles + kt) * TILE_BYTES; }
    __device__ const uint8_t *group(int rt, int kg) const { return scales + ((size_t)rt * kgroups + kg) * GROUP_BYTES; }
};

struct QuantParams {
    const void *x;
    void *y;
    uint8_t *codes, *scales;
    int rows, K, ktiles, kgroups;
    long row;                 // elements between rows of x or y
};

struct PackParams {
    uint8_t *flat_codes, *flat_scales;   // [rows][K / 2], [rows][K / 32]
    uint8_t *codes, *scales;
    int rows, K, ktiles, kgroups;
};

struct GemmParams {
    Matrix w, x;              // x.codes NULL: xb
    const uint16_t *xb;       // [T][x_row] bf16
    long x_row, y_row, r_row;
    void *y;
    const float *residual;
    int T, N, K, y_bf16;
    int vec;                  // y (and the residual) allow stores of four columns at a time
};

// Four consecutive columns of a row, all inside the matrix, at addresses that allow it: residual, rounding, store.
__device__ __forceinline__ void store4_whole(const GemmParams &p, int t, int c, float v0, float v1, float v2, float v3) {
    if (p.y_bf16) {
        *(u32x2 *)((uint16_t *)p.y + (size_t)t * p.y_row + c) = u32x2{pack_bf16(v0, v1), pack_bf16(v2, v3)};
        return;
    }
    float4 o = {v0, v1, v2, v3};
    if (p.residual) {
        const float4 r = *(const float4 *)(p.residual + (size_t)t * p.r_row + c);
        o = {v0 + r.x, v1 + r.y, v2 + r.z, v3 + r.w};
    }
    *(float4 *)((float *)p.y + (size_t)t * p.y_row + c) = o;
}
// Anywhere, c inside the matrix.
__device__ __forceinline__ void store4(const GemmParams &p, int t, int c, float v0, float v1, float v2, float v3) {
    const int n = p.N - c;
    if (p.vec && n >= 4) return store4_whole(p, t, c, v0, v1, v2, v3);
    const float v[4] = {v0, v1, v2, v3};
    for (int i = 0; i < 4 && i < n; i++) {
        if (p.y_bf16) ((uint16_t *)p.y)[(size_t)t * p.y_row + c + i] = f2bf(v[i]);
        else ((float *)p.y)[(size_t)t * p.y_row + c + i] = v[i] + (p.residual ? p.residual[(size_t)t * p.r_row + c + i] : 0.f);
    }
}

}  // namespace mx4
}  // namespace clef_hip
