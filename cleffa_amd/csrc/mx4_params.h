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
    bool past;                // of y: store_past
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
    bool past;                // of y: store_past
};

// Vectors at any element's address: the memory takes them, and odd row strides keep their wide stores.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// Up to four consecutive columns of a row, c inside the matrix: residual, rounding, store.
__device__ __forceinline__ void store4(const GemmParams &p, int t, int c, f32x4 v) {
    const int n = p.N - c;
    if (p.y_bf16) {
        uint16_t *y = (uint16_t *)p.y + (size_t)t * p.y_row + c;
        if (n >= 4) *(u32x2_any *)y = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        else
            for (int i = 0; i < n; i++) y[i] = f2bf(i == 0 ? v[0] : i == 1 ? v[1] : v[2]);
        return;
    }
    float *y = (float *)p.y + (size_t)t * p.y_row + c;
    const float *r = p.residual ? p.residual + (size_t)t * p.r_row + c : nullptr;
    if (n >= 4) {
        if (r) v += *(const f32x4_any *)r;
        *(f32x4_any *)y = v;
    } else {
        for (int i = 0; i < n; i++) y[i] = (i == 0 ? v[0] : i == 1 ? v[1] : v[2]) + (r ? r[i] : 0.f);
    }
}

}  // namespace mx4
}  // namespace clef_hip
