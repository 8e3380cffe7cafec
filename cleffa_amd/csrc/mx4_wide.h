// The product of bf16 rows with a 4-bit matrix in tiles, operands through LDS: codes are widened to bf16 in registers, exactly,
// and multiplied by the 16-bit matrix instruction 32x32x16.
//
// K goes by tiles of 128, two halves of four steps of 16. Lane l holds 32 codes of row l % 32 of W, block 2 half + l / 32, in four words
// of eight; step j takes word j, and of X the eight values at the same places: chunk 4 (2 half + l / 32) + j of the 16 in a row's
// 256 bytes. X's rows lie in LDS with chunk c of row r at c ^ (r % 16), so that 16 rows' chunks are on distinct banks.
// A code takes a quarter of a value's bytes, so a wave's part of the tile is wide in columns: 64 rows x 128 columns read 16 KB of X
// and 8 KB of W a K tile.
//
// Bound by the matrix units: 4,096 x 14,336 x 5,120 takes 432 to 455 us on different chips, 1.32 to 1.39 PFLOP/s, where the products
// alone ran at 1.65 in a loop without any loads and library products of 16-bit operands at 1.21 (8,192 cubed) and 1.27 (this one). Widening
// issues between the products, while the matrix unit works.
#pragma once
#include "mx4_tile.h"

namespace clef_hip {
namespace mx4 {

template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int PER_CU_>
struct WideCfg {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, PER_CU = PER_CU_;
    static constexpr int WAVES_N = BN / WN, WAVES = BM / WM * WAVES_N, THREADS = 64 * WAVES;
    static constexpr int MT = WM / 32, NT = WN / 32;
    static constexpr int W_TILES = BN / 16, W_FILLS = W_TILES / WAVES, X_FILLS = BM / 4 / WAVES, FILLS = W_FILLS + X_FILLS;
    static constexpr int S_FILLS = (W_TILES / 4 + WAVES - 1) / WAVES;
    static constexpr int X_AT = W_TILES * TILE_BYTES, STAGE_BYTES = X_AT + BM * 256, SCALES_AT = STAGES * STAGE_BYTES;
    static constexpr int OUT_ROW = out_row(NT);
    static constexpr int LDS_BYTES = SCALES_AT + W_TILES * GROUP_BYTES > WAVES * 32 * OUT_ROW ? SCALES_AT + W_TILES * GROUP_BYTES : WAVES * 32 * OUT_ROW;
    static_assert(W_TILES % WAVES == 0 && W_TILES % 4 == 0 && BM / 4 % WAVES == 0, "fills divide over the waves");
    static_assert(STAGES >= 2 && STAGES <= 4, "scales arrive with the K tile in front of theirs or before");
    static_assert(MT == 2 && (NT == 2 || NT == 4), "operands of a wave's tile");
    static_assert(PER_CU * LDS_BYTES <= 160 * 1024, "LDS");
};

// One wait for what a step has read: two operands of X and the codes of a half.
template <int NT>
__device__ __forceinline__ void lds_wait(u32x4 (&x)[2], u32x4 (&w)[NT]) {
    if constexpr (NT == 2) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(x[0]), "+v"(x[1]), "+v"(w[0]), "+v"(w[1])::"memory");
    else asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(x[0]), "+v"(x[1]), "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3])::"memory");
}
template <int NT>
__device__ __forceinline__ void lds_wait(u32x4 (&x)[2], u32x4 (&w)[NT], unsigned (&s)[2][NT]) {
    if constexpr (NT == 2)
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(x[0]), "+v"(x[1]), "+v"(w[0]), "+v"(w[1]), "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[1][0]), "+v"(s[1][1])::"memory");
    else
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(x[0]), "+v"(x[1]), "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]), "+v"(s[0][0]), "+v"(s[0][1]),
                     "+v"(s[0][2]), "+v"(s[0][3]), "+v"(s[1][0]), "+v"(s[1][1]), "+v"(s[1][2]), "+v"(s[1][3])::"memory");
}

template <typename C>
__global__ __launch_bounds__(C::THREADS, C::WAVES / 4 * C::PER_CU) void mx4_wide_kernel(GemmParams p) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS_BYTES];
    constexpr int MT = C::MT, NT = C::NT, P = MT * NT, STAGES = C::STAGES, FILLS = C::FILLS, S_FILLS = C::S_FILLS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn;
    if (!tile_of(blockIdx.x, ceil_div(p.T, C::BM), ceil_div(p.N, C::BN), &tm, &tn)) return;
    const int wm = wave / C::WAVES_N, wn = wave % C::WAVES_N;
    const int ktiles = p.w.ktiles, kgroups = p.w.kgroups;
    const int w_last = ceil_div(p.N, 16) - 1;

    // fills: this wave's tiles of W, then four rows of X an instruction; rows beyond the matrix are its last one again
    const uint8_t *wsrc[C::W_FILLS];
#pragma unroll
    for (int f = 0; f < C::W_FILLS; f++) wsrc[f] = p.w.tile(min(tn * C::W_TILES + wave * C::W_FILLS + f, w_last), 0);
    const uint8_t *xsrc[C::X_FILLS];
#pragma unroll
    for (int f = 0; f < C::X_FILLS; f++)
        xsrc[f] = (const uint8_t *)(p.xb + (size_t)min(tm * C::BM + 4 * (wave * C::X_FILLS + f) + (lane >> 4), p.T - 1) * p.x_row);
    const uint8_t *ssrc[S_FILLS];
    int s_at[S_FILLS];
#pragma unroll
    for (int f = 0; f < S_FILLS; f++) {
        s_at[f] = min(wave * S_FILLS + f, C::W_TILES / 4 - 1);
        ssrc[f] = p.w.group(min(tn * C::W_TILES + 4 * s_at[f] + (lane >> 4), w_last), 0) + 16 * (lane & 15);
    }
    // values of X beyond K come from the codes beyond K of W's last K tile, which are zeros
    const uint8_t *zeros = p.w.tile(w_last, ktiles - 1) + (4 - 1) * 256;
    unsigned at = 16 * lane;
    auto fill_one = [&](int kt, unsigned stage, int f) CLEF_INLINE {
        kt = min(kt, ktiles - 1);
        if (f < C::W_FILLS) {
            asm volatile("" : "+v"(at));
            __builtin_amdgcn_global_load_lds((const void *)(wsrc[f] + (size_t)kt * TILE_BYTES + at),
                                             (lds_void4 *)(lds + stage + (wave * C::W_FILLS + f) * TILE_BYTES), 16, 0, 0);
        } else {
            const int i = f - C::W_FILLS, row = 4 * (wave * C::X_FILLS + i);
            const int chunk = (lane & 15) ^ ((row & 15) + (lane >> 4));
            const uint8_t *from = KT * kt + 8 * chunk < p.K ? xsrc[i] + (size_t)kt * 256 + 16 * chunk : zeros;
            __builtin_amdgcn_global_load_lds((const void *)from, (lds_void4 *)(lds + stage + C::X_AT + row * 256), 16, 0, 0);
        }
    };
    auto fill_scales = [&](int kg) CLEF_INLINE {
#pragma unroll
        for (int f = 0; f < S_FILLS; f++)
            __builtin_amdgcn_global_load_lds((const void *)(ssrc[f] + (size_t)min(kg, kgroups - 1) * GROUP_BYTES),
                                             (lds_void4 *)(lds + C::SCALES_AT + s_at[f] * 1024), 16, 0, 0);
    };

    const unsigned wbase = lds_address(lds) + wn * (C::WN / 16) * TILE_BYTES + (lane >> 4 & 1) * 1024 + (lane >> 5) * 256 + (lane & 15) * 16;
    const unsigned sbase = lds_address(lds) + C::SCALES_AT + wn * (C::WN / 16) * GROUP_BYTES + (lane >> 4 & 1) * GROUP_BYTES + (lane >> 5) * 64 + (lane & 15) * 4;
    // chunk 8 half + 4 (lane / 32) + j of row lane % 32 (rows 32 apart have the same place)
    unsigned xbase[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        xbase[i] = lds_address(lds) + C::X_AT + (wm * C::WM + (lane & 31)) * 256 + ((((i & 4) << 1) + 4 * (lane >> 5) + (i & 3)) ^ (lane & 15)) * 16;
    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x16{};
    u32x4 x[4][2];                          // X of this step, the next one, and that behind it, which is read
    u32x4 w[2][NT];                         // codes of two halves
    u32x4 wide[2][NT];                      // W of two steps, widened
    unsigned s[2][NT], s_next[2][NT];       // scales of the halves, a byte for each of four K tiles
    auto read_x = [&](auto STEP, unsigned stage) CLEF_INLINE {   // step 0 .. 7 of a K tile
        constexpr int st = decltype(STEP)::value;
        x[st & 3][0] = lds_read16<0>(xbase[st] + stage);
        x[st & 3][1] = lds_read16<32 * 256>(xbase[st] + stage);
    };
    auto read_w = [&](auto H, unsigned stage) CLEF_INLINE {
        for_each<NT>([&](auto I) CLEF_INLINE { w[decltype(H)::value][decltype(I)::value] = lds_read16<decltype(I)::value * 2048 + decltype(H)::value * 512>(wbase + stage); });
    };
    auto read_scales = [&]() CLEF_INLINE {
        for_each<2 * NT>([&](auto I) CLEF_INLINE {
            constexpr int h = decltype(I)::value / NT, i = decltype(I)::value % NT;
            s_next[h][i] = lds_read4<i * 512 + h * 128>(sbase);
        });
    };
    // two of the four words that step st (of the K tile at pos) takes of part j of W
    auto widen2 = [&](auto POS, auto STEP, int j, int part) CLEF_INLINE {
        constexpr int st = decltype(STEP)::value, h = st / 4, pos = decltype(POS)::value;
        const float scale = __uint_as_float((s[h][j] >> (8 * pos) & 255u) << 23);
        const unsigned codes = w[h][j][st % 4];
        u32x4 &o = wide[st & 1][j];
        if (part == 0) {
            o[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
            o[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
        } else {
            o[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
            o[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
        }
    };
    constexpr std::integral_constant<int, 0> i0;
    constexpr std::integral_constant<int, 1> i1;
    unsigned stage = 0;
    auto after = [&](unsigned st) CLEF_INLINE { return st == (STAGES - 1) * C::STAGE_BYTES ? 0u : st + C::STAGE_BYTES; };
    // K tile kt at POS of its group. X of a step is read two steps before, so that after the sixth step nothing more is read of this K
    // tile, and its buffer takes kt + STAGES with the last two steps. Reads stand behind a step's first product and the barrier behind
    // some of its step's: with reads and barrier ahead of the products 4,096 x 14,336 x 5,120 took 452 us, against 432 on the same chip.
    auto k_tile = [&](int kt, auto POS) CLEF_INLINE {
        constexpr int pos = decltype(POS)::value, next = (pos + 1) & 3;
        const unsigned here = stage;
        for_each<8>([&](auto STEP) CLEF_INLINE {
            constexpr int st = decltype(STEP)::value;
            constexpr std::integral_constant<int, (st + 1) & 7> st_next;
            constexpr std::integral_constant<int, st == 7 ? next : pos> pos_next;
            // between the products the next step's W is widened, X and codes are read, fills go out; the barriers keep them there
            for_each<P>([&](auto Q) CLEF_INLINE {
                constexpr int q = decltype(Q)::value, i = q % MT, j = q / MT, first = st == 6 ? P / 4 : 0;
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, wide[st & 1][j]), __builtin_bit_cast(bf16x8, x[st & 3][i]), acc[i][j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (q == first) {
                    if constexpr (st == 6) {
                        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"((STAGES - 2) * FILLS + (next >= 2 && next < STAGES ? S_FILLS : 0)) : "memory");
                        if constexpr (next == 1) fill_scales((kt >> 2) + 1);
                        stage = after(stage);
                    }
                    read_x(std::integral_constant<int, (st + 2) & 7>{}, stage);
                }
                if constexpr (q == first + 1) {
                    if constexpr (st == 6) read_w(i0, stage);
                    if constexpr (st == 6 && next == 0) read_scales();
                    if constexpr (st == 1) read_w(i1, stage);
                }
                widen2(pos_next, st_next, j, i);
                constexpr int at = (st - 6) * P + q - P / 4 - 1, n = 2 * P - P / 4 - 1;    // of the products behind the barrier
                if constexpr (st >= 6 && at >= 0) {
#pragma unroll
                    for (int f = at * FILLS / n; f < (at + 1) * FILLS / n; f++) fill_one(kt + STAGES, here, f);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (st == 6 && next == 0) {
                lds_wait(x[(st + 2) & 3], w[0], s_next);
#pragma unroll
                for (int i = 0; i < 2 * NT; i++) s[i / NT][i % NT] = s_next[i / NT][i % NT];
            } else if constexpr (st == 6) lds_wait(x[(st + 2) & 3], w[0]);
            else lds_wait(x[(st + 2) & 3], w[1]);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    fill_scales(0);
    for (int q = 0; q < STAGES; q++)
#pragma unroll
        for (int f = 0; f < FILLS; f++) fill_one(q, q * C::STAGE_BYTES, f);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"((STAGES - 1) * FILLS) : "memory");
    read_w(i0, 0);
    read_scales();
    read_x(i0, 0);
    lds_wait(x[0], w[0], s_next);
    read_x(i1, 0);
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) s[i / NT][i % NT] = s_next[i / NT][i % NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        widen2(i0, i0, j, 0);
        widen2(i0, i0, j, 1);
    }
    lds_wait(x[1], w[0]);
    int kt = 0;
    for (; kt + 4 <= ktiles; kt += 4) for_each<4>([&](auto POS) CLEF_INLINE { k_tile(kt + decltype(POS)::value, POS); });
    for_each<3>([&](auto POS) CLEF_INLINE {
        if (kt + decltype(POS)::value < ktiles) k_tile(kt + decltype(POS)::value, POS);
    });
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // the last fills
    __syncthreads();
    store_tile<MT, NT>(p, acc, lds + wave * 32 * C::OUT_ROW, tm * C::BM + wm * C::WM, tn * C::BN + wn * C::WN);
}

}  // namespace mx4
}  // namespace clef_hip
