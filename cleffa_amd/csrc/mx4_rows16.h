// Few bf16 rows times a 4-bit matrix: MT x NT tiles of 16 rows and 16 columns a workgroup, whose W waves share the K tiles and add their
// sums in LDS in a fixed order. A K tile of 128 is four products 16x16x32, j of them with word j of each lane's 32 codes, widened to
// bf16, and X's eight values at their places, chunk 4 (l / 16) + j of the 16 in a row's 256 bytes.
//
// W comes straight from memory into registers, 1 KB a load. X goes through LDS, each wave's own part of it: a load takes 16 lanes at a
// time, whose addresses it can join; four rows x 256 bytes an instruction are two lines for each 16, where the operands themselves,
// 16 rows x 16 bytes, are sixteen lines (61 x 5,120 x 6,144 took 26 us with them, against 12.3 now). Chunk c of row r lies at c ^ r.
#pragma once
#include "mx4_tile.h"

namespace clef_hip {
namespace mx4 {

// XF: the loads of X for a K tile, four rows each; 4 MT, or less where no more rows are there (the others' outputs are not stored)
template <int MT, int NT, int W, int XF>
__global__ __launch_bounds__(64 * W) void mx4_rows16_kernel(GemmParams p) {
    constexpr int X_BYTES = MT * 16 * 256, STAGE = X_BYTES * W;       // of a wave and K tile, of all waves
    constexpr int PART_BYTES = W * MT * NT * 64 * 16, BYTES = 2 * STAGE > PART_BYTES ? 2 * STAGE : PART_BYTES;
    constexpr int GROUP = 2 * NT + XF;                                // loads of a K tile
    __shared__ __attribute__((aligned(1024))) uint8_t lds[BYTES];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int n_tiles = ceil_div(p.N, 16), nb = ceil_div(n_tiles, NT);
    const int n0 = (blockIdx.x % nb) * NT, t0 = (blockIdx.x / nb) * MT;
    const int ktiles = p.w.ktiles, k_lo = ktiles * wave / W, k_hi = ktiles * (wave + 1) / W;
    const uint8_t *wsrc[NT], *ssrc[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        wsrc[j] = p.w.tile(min(n0 + j, n_tiles - 1), 0);
        ssrc[j] = p.w.group(min(n0 + j, n_tiles - 1), 0);
    }
    const uint8_t *xsrc[XF];         // rows 4 i + lane / 16
#pragma unroll
    for (int i = 0; i < XF; i++) xsrc[i] = (const uint8_t *)(p.xb + (size_t)min(16 * t0 + 4 * i + g, p.T - 1) * p.x_row);
    const uint8_t *zeros = p.w.tile(n_tiles - 1, ktiles - 1) + 3 * 256;   // codes beyond K, where there are any: for X beyond K
    uint8_t *mine = lds + wave * X_BYTES;
    struct Ops {
        u32x4 w[NT];
        unsigned s[NT];
    };
    // the loads of K tile kt, of which there are always as many: beyond the wave's last they take one address in all lanes
    auto load = [&](Ops &o, int kt, int stage) CLEF_INLINE {
        const bool live = kt < k_hi;
        kt = live ? kt : k_hi - 1;
        const int at = live ? lane : 0;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            o.w[j] = *(const u32x4 *)(wsrc[j] + (size_t)kt * TILE_BYTES + 16 * at);
            o.s[j] = *(const unsigned *)(ssrc[j] + (size_t)(kt >> 2) * GROUP_BYTES + 4 * at);
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < XF; i++) {
            const int chunk = l16 ^ (4 * (i & 3) + g);
            const uint8_t *from = live && KT * kt + 8 * chunk < p.K ? xsrc[i] + (size_t)kt * 256 + 16 * chunk : zeros;
            __builtin_amdgcn_global_load_lds((const void *)from, (lds_void4 *)(mine + stage * STAGE + i * 1024), 16, 0, 0);
        }
        asm volatile("" ::: "memory");
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const unsigned base = lds_address(mine) + l16 * 256;
    auto k_tile = [&](Ops &o, int kt, int stage) CLEF_INLINE {
        // the next K tile's may stay in flight. On every other K tile they do not: the compiler waits for W by a count of its own, which it
        // takes over the ways around the loop's skip and the loads of X, and that is none.
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(GROUP) : "memory");
        u32x4 x[4 * MT];
        for_each<4>([&](auto J) CLEF_INLINE {
            constexpr int j = decltype(J)::value;
            const unsigned at = base + stage * STAGE + ((4 * g + j) ^ l16) * 16;
            for_each<MT>([&](auto I) CLEF_INLINE { x[decltype(I)::value * 4 + j] = lds_read16<decltype(I)::value * 4096>(at); });
        });
        lds_wait(x);
        const int sh = 8 * (kt & 3);
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float scale = __uint_as_float((o.s[n] >> sh & 255u) << 23);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned codes = o.w[n][j];
                const bf16x8 w = widen(codes, scale);
#pragma unroll
                for (int i = 0; i < MT; i++)
                    acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, __builtin_bit_cast(bf16x8, x[i * 4 + j]), acc[i][n], 0, 0, 0);
            }
        }
        load(o, kt + 2, stage);
    };
    if (k_lo < k_hi) {
        Ops o0, o1;
        load(o0, k_lo, 0);
        load(o1, k_lo + 1, 1);
        for (int kt = k_lo; kt < k_hi; kt += 2) {
            k_tile(o0, kt, 0);
            if (kt + 1 < k_hi) k_tile(o1, kt + 1, 1);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    join_waves<MT, NT, W>(p, acc, (f32x4(*)[MT * NT][64])lds, t0, n0);
}

}  // namespace mx4
}  // namespace clef_hip
