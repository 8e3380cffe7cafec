// The product of two 4-bit matrices in tiles of BM rows and BN columns a workgroup, operands through LDS.
//
// The matrix instruction 32x32x64 takes from lane l 32 codes of row l % 32, block l / 32. Tiles of codes (16 rows x 128) go to
// LDS as they lie in memory, 1 KB an instruction; a lane's 16 bytes of rows 32 i .. + 31, half h of the K tile, are at
// 2048 i + 512 h + 1024 (l / 16 % 2) + 256 (l / 32) + 16 (l % 16): 256 bytes in a row for each 16 lanes, all banks once.
// Scales of four K tiles go to LDS together and from there into a register for each operand, of which the instruction
// takes a byte; those reads, four bytes a lane, meet two ways, rows 16 and on 256 bytes behind the others (counted: 3.4e6 conflict
// clocks on 6.4e6 LDS instructions of 4,096 x 14,336 x 5,120). So the loop takes four K tiles at a time, one straight line of code: over branches the compiler would move the
// products behind the waits.
//
// Bound by the matrix units and LDS together. A K tile of 256 x 256 is 1,024 clocks of a CU's products; its waves' operands are 96 KB
// of LDS reads and 32 KB of fills, at 128 bytes a clock as many again. The products alone ran at 6.3 PFLOP/s, on such data, in a loop
// without any loads, the chip at 1.8 of its 2.4 GHz for its power. 4,096 x 14,336 x 5,120 takes 139 to 144 us in tiles of 256 x 128, two
// workgroups a CU (4.2 to 4.3 PFLOP/s; 149 on one chip), 142 to 149 in tiles of 256 x 256, 162 to 164 in 128 x 128; 3,000 x 10,240 x 4,096 66 to 68
// in 256 x 128 and 61 to 67 in 256 x 256. Four waves of 128 x 128 read a third less of LDS, but nothing runs while they wait: 149 us where
// eight took 144.
#pragma once
#include <utility>

#include "mx4_gemm.h"

namespace clef_hip {
namespace mx4 {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((address_space(3))) void lds_void4;
// of the kernels' lambdas: what is left a call keeps its operands in memory
#define CLEF_INLINE __attribute__((always_inline))

__device__ __forceinline__ unsigned lds_address(const void *p) {
    return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}
template <int OFF>
__device__ __forceinline__ u32x4 lds_read16(unsigned addr) {
    u32x4 r;
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(OFF) : "memory");
    return r;
}
template <int OFF>
__device__ __forceinline__ unsigned lds_read4(unsigned addr) {
    unsigned r;
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(OFF) : "memory");
    return r;
}
template <typename F, int... I>
__device__ __forceinline__ void for_each_impl(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void for_each(F &&f) {
    for_each_impl(f, std::make_integer_sequence<int, N>{});
}
// Waits for all LDS reads in one statement that names what they fill, codes and scales, so that no copy or use of it comes before.
template <int F>
__device__ __forceinline__ void lds_wait(u32x4 (&r)[F]) {
    static_assert(F == 3 || F == 4 || F == 6 || F == 8, "operands of a wave's tile");
    if constexpr (F == 3) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2])::"memory");
    else if constexpr (F == 4) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3])::"memory");
    else if constexpr (F == 6)
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]), "+v"(r[4]), "+v"(r[5])::"memory");
    else
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]), "+v"(r[4]), "+v"(r[5]), "+v"(r[6]), "+v"(r[7])::"memory");
}
template <int F>
__device__ __forceinline__ void lds_wait(u32x4 (&r)[F], unsigned (&s)[2][F]) {
    static_assert(F == 3 || F == 4 || F == 6, "operands of a wave's tile");
    if constexpr (F == 3)
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[0][2]), "+v"(s[1][0]), "+v"(s[1][1]),
                     "+v"(s[1][2])::"memory");
    else if constexpr (F == 4)
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]), "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[0][2]), "+v"(s[0][3]),
                     "+v"(s[1][0]), "+v"(s[1][1]), "+v"(s[1][2]), "+v"(s[1][3])::"memory");
    else
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]), "+v"(r[4]), "+v"(r[5]), "+v"(s[0][0]), "+v"(s[0][1]),
                     "+v"(s[0][2]), "+v"(s[0][3]), "+v"(s[0][4]), "+v"(s[0][5]), "+v"(s[1][0]), "+v"(s[1][1]), "+v"(s[1][2]), "+v"(s[1][3]),
                     "+v"(s[1][4]), "+v"(s[1][5])::"memory");
}

// Between what lanes write to LDS and what other lanes of the wave read or overwrite of it. The hardware takes a wave's LDS instructions in order,
// so this costs none: it keeps the compiler from moving them across, which it may where it sees that a lane's own addresses differ.
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wave's outputs, rows t0 .. and columns c0 ..: lane l's accumulators of a 32 x 32 part are columns 8 (e / 4) + 4 (l / 32) + e % 4 of row
// l % 32. 32 rows at a time go through `mine`, LDS of the wave's own, so that stores take whole lines, past the caches where rows of Y
// begin at them: 4,096 x 14,336 x 5,120 148 us with ordinary stores, 140 past the caches (on one chip), which W and X then have to themselves; 2,000 x 6,389
// x 160, where they do not, 12.3 and 16.6.
constexpr int out_row(int NT) { return 32 * NT * 4 + 16; }
template <int MT, int NT>
__device__ __forceinline__ void store_tile(const GemmParams &p, const f32x16 (&acc)[MT][NT], uint8_t *mine, int t_first, int c0) {
    constexpr int WN = 32 * NT, OUT_ROW = out_row(NT);
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int t0 = t_first + 32 * i;
        wave_lds_order();        // the rows before have been read
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                *(f32x4 *)(mine + (lane & 31) * OUT_ROW + (32 * j + 8 * e + 4 * (lane >> 5)) * 4) =
                    f32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
        wave_lds_order();
        // V columns a lane, 16 bytes of Y; the columns before N that are fewer come after, one by one
        if (p.y_bf16) {
            constexpr int LANES = WN / 8, ROWS_I = 64 / LANES;    // lanes of a row, rows of an instruction
            const int c = c0 + 8 * (lane % LANES), t = t0 + lane / LANES;
            const uint8_t *from = mine + lane / LANES * OUT_ROW + 32 * (lane % LANES);
            uint16_t *to = (uint16_t *)p.y + (size_t)t * p.y_row + c;
            const int rows = c + 8 <= p.N ? p.T - t : 0;
            with_past(p.past, [&](auto PAST) CLEF_INLINE {
#pragma unroll
                for (int r = 0; r < 32; r += ROWS_I) {
                    const f32x4 a = *(const f32x4 *)(from + r * OUT_ROW), b = *(const f32x4 *)(from + r * OUT_ROW + 16);
                    if (r < rows)
                        store_past(PAST, (u32x4_any *)(to + (size_t)r * p.y_row), u32x4{pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]), pack_bf16(b[0], b[1]), pack_bf16(b[2], b[3])});
                }
            });
            if (c0 + WN > p.N && p.N % 8) {
#pragma unroll 1
                for (int r = 0; r < 32; r += ROWS_I)
                    for (int k = 0; k < 8; k += 4)
                        if (t + r < p.T && c + 8 > p.N && c + k < p.N) store4(p, t + r, c + k, *(const f32x4 *)(from + r * OUT_ROW + 4 * k));
            }
            continue;
        }
        constexpr int LANES = WN / 4, ROWS_I = 64 / LANES;
        const int c = c0 + 4 * (lane % LANES), t = t0 + lane / LANES;
        const uint8_t *from = mine + lane / LANES * OUT_ROW + 16 * (lane % LANES);
        const int rows = c + 4 <= p.N ? p.T - t : 0;
        f32x4 v[32 / ROWS_I];
#pragma unroll
        for (int r = 0; r < 32 / ROWS_I; r++) {
            f32x4 z{0.f, 0.f, 0.f, 0.f};
            if (p.residual && r * ROWS_I < rows) z = *(const f32x4_any *)(p.residual + (size_t)(t + r * ROWS_I) * p.r_row + c);   // all loads together
            v[r] = z;
        }
#pragma unroll
        for (int r = 0; r < 32 / ROWS_I; r++) v[r] += *(const f32x4 *)(from + r * ROWS_I * OUT_ROW);
        with_past(p.past, [&](auto PAST) CLEF_INLINE {
#pragma unroll
            for (int r = 0; r < 32 / ROWS_I; r++)
                if (r * ROWS_I < rows) store_past(PAST, (f32x4_any *)((float *)p.y + (size_t)(t + r * ROWS_I) * p.y_row + c), v[r]);
        });
        if (c0 + WN > p.N && p.N % 4) {
#pragma unroll 1
            for (int r = 0; r < 32; r += ROWS_I)
                if (t + r < p.T && c + 4 > p.N && c < p.N) store4(p, t + r, c, *(const f32x4 *)(from + r * OUT_ROW));
        }
    }
}

// Tile, a wave's part of it, K tiles in LDS at a time, workgroups a CU.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int PER_CU_>
struct TileCfg {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, PER_CU = PER_CU_;
    static constexpr int WAVES_N = BN / WN, WAVES = BM / WM * WAVES_N, THREADS = 64 * WAVES;
    static constexpr int MT = WM / 32, NT = WN / 32, FR = MT + NT;
    static constexpr int W_TILES = BN / 16, X_TILES = BM / 16, TILES = W_TILES + X_TILES, FILLS = TILES / WAVES, S_FILLS = (TILES / 4 + WAVES - 1) / WAVES;
    static constexpr int STAGE_BYTES = TILES * TILE_BYTES, SCALES_AT = STAGES * STAGE_BYTES;
    static constexpr int OUT_ROW = out_row(NT);
    static constexpr int LDS_BYTES = SCALES_AT + TILES * GROUP_BYTES > WAVES * 32 * OUT_ROW ? SCALES_AT + TILES * GROUP_BYTES : WAVES * 32 * OUT_ROW;
    static_assert(TILES % WAVES == 0 && W_TILES % 4 == 0 && X_TILES % 4 == 0, "fills divide over the waves");
    static_assert(STAGES >= 2 && STAGES <= 4, "scales arrive with the K tile in front of theirs or before");
    static_assert(PER_CU * LDS_BYTES <= 160 * 1024, "LDS");
};

// Workgroup b to its tile: XCD b % 8 takes columns of tiles b % 8, + 8, .. and goes through them row of tiles by row of tiles, so
// that the tiles that run on it together share rows of X and W in its L2.
__device__ __forceinline__ bool tile_of(int b, int m_tiles, int n_tiles, int *tm, int *tn) {
    const int x = b & 7, j = b >> 3, cnt = (n_tiles - x + 7) >> 3;
    if (cnt <= 0 || j >= cnt * m_tiles) return false;
    *tm = j / cnt;
    *tn = x + 8 * (j % cnt);
    return true;
}

template <typename C>
__global__ __launch_bounds__(C::THREADS, C::WAVES / 4 * C::PER_CU) void mx4_tile_kernel(GemmParams p) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS_BYTES];
    constexpr int MT = C::MT, NT = C::NT, FR = C::FR, P = MT * NT, STAGES = C::STAGES, FILLS = C::FILLS, S_FILLS = C::S_FILLS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn;
    if (!tile_of(blockIdx.x, ceil_div(p.T, C::BM), ceil_div(p.N, C::BN), &tm, &tn)) return;
    const int wm = wave / C::WAVES_N, wn = wave % C::WAVES_N;
    const int ktiles = p.w.ktiles, kgroups = p.w.kgroups;
    const int w_last = ceil_div(p.N, 16) - 1, x_last = ceil_div(p.T, 16) - 1;

    // This wave's fills: tiles wave * FILLS .. of W's and then X's; tiles beyond the matrix are its last one again. Scales: four
    // tiles an instruction, the last four again where they do not divide over the waves.
    const int first = wave * FILLS;
    const uint8_t *src[FILLS];
#pragma unroll
    for (int f = 0; f < FILLS; f++) {
        const int t = first + f;
        src[f] = t < C::W_TILES ? p.w.tile(min(tn * C::W_TILES + t, w_last), 0) : p.x.tile(min(tm * C::X_TILES + t - C::W_TILES, x_last), 0);
    }
    const uint8_t *ssrc[S_FILLS];
    int s_at[S_FILLS];
#pragma unroll
    for (int f = 0; f < S_FILLS; f++) {
        s_at[f] = min(wave * S_FILLS + f, C::TILES / 4 - 1);
        const int t = 4 * s_at[f] + (lane >> 4);
        ssrc[f] = (t < C::W_TILES ? p.w.group(min(tn * C::W_TILES + t, w_last), 0) : p.x.group(min(tm * C::X_TILES + t - C::W_TILES, x_last), 0)) + 16 * (lane & 15);
    }
    // K tile and group beyond the last are the last again, into buffers that nothing reads
    unsigned at = 16 * lane;
    auto fill_one = [&](int kt, unsigned stage, int f) CLEF_INLINE {
        asm volatile("" : "+v"(at));
        __builtin_amdgcn_global_load_lds((const void *)(src[f] + (size_t)min(kt, ktiles - 1) * TILE_BYTES + at),
                                         (lds_void4 *)(lds + stage + (first + f) * TILE_BYTES), 16, 0, 0);
    };
    auto fill_scales = [&](int kg) CLEF_INLINE {
#pragma unroll
        for (int f = 0; f < S_FILLS; f++)
            __builtin_amdgcn_global_load_lds((const void *)(ssrc[f] + (size_t)min(kg, kgroups - 1) * GROUP_BYTES),
                                             (lds_void4 *)(lds + C::SCALES_AT + s_at[f] * 1024), 16, 0, 0);
    };

    const unsigned base = lds_address(lds) + (lane >> 4 & 1) * 1024 + (lane >> 5) * 256 + (lane & 15) * 16;
    const unsigned wbase = base + wn * (C::WN / 16) * TILE_BYTES, xbase = base + (C::W_TILES + wm * (C::WM / 16)) * TILE_BYTES;
    const unsigned sbase = lds_address(lds) + C::SCALES_AT + (lane >> 4 & 1) * GROUP_BYTES + (lane >> 5) * 64 + (lane & 15) * 4;
    const unsigned wsbase = sbase + wn * (C::WN / 16) * GROUP_BYTES, xsbase = sbase + (C::W_TILES + wm * (C::WM / 16)) * GROUP_BYTES;
    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x16{};
    u32x4 r0[FR], r1[FR];
    unsigned s[2][FR], s_next[2][FR];       // scales of the halves' operands, a byte for each of four K tiles
    // operand i of a half, NT of W and then MT of X
    auto read = [&](u32x4 (&r)[FR], unsigned stage, auto H, auto I) CLEF_INLINE {
        constexpr int h = decltype(H)::value, i = decltype(I)::value, j = i < NT ? i : i - NT;
        r[i] = lds_read16<j * 2048 + h * 512>((i < NT ? wbase : xbase) + stage);
    };
    auto read_scales = [&]() CLEF_INLINE {
        for_each<2 * FR>([&](auto I) CLEF_INLINE {
            constexpr int h = decltype(I)::value / FR, i = decltype(I)::value % FR, j = i < NT ? i : i - NT;
            s_next[h][i] = lds_read4<j * 512 + h * 128>(i < NT ? wsbase : xsbase);
        });
    };
    auto take_scales = [&]() CLEF_INLINE {
#pragma unroll
        for (int i = 0; i < 2 * FR; i++) s[i / FR][i % FR] = s_next[i / FR][i % FR];
    };
    // product Q of half H of K tile POS of four
    auto product = [&](u32x4 (&r)[FR], auto POS, auto H, auto Q) CLEF_INLINE {
        constexpr int i = decltype(Q)::value / NT, j = decltype(Q)::value % NT, h = decltype(H)::value, pos = decltype(POS)::value;
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(r[j]), operand(r[NT + i]), acc[i][j], 4, 4, pos, (int)s[h][j], pos, (int)s[h][NT + i]);
    };
    // Products FROM .. of a half, reads of the next half's operands between them, so that the matrix unit has work while
    // reads are issued and in flight (behind the first half of the products: there is time left for them to arrive); and fills F0 .. F1,
    // which issue as fast as addresses are taken, 16 clocks each for all of the CU's waves.
    auto step = [&](auto POS, u32x4 (&now)[FR], auto H, auto FROM, u32x4 (&next)[FR], unsigned stage, auto H_NEXT, int fill_kt, unsigned fill_stage, auto F0, auto F1) CLEF_INLINE {
        constexpr int from = decltype(FROM)::value, n = P - from, early = n > 1 ? n / 2 : 1, per = (FR + early - 1) / early, f0 = decltype(F0)::value, nf = decltype(F1)::value - f0;
        for_each<n>([&](auto Q) CLEF_INLINE {
            constexpr int q = decltype(Q)::value;
            product(now, POS, H, std::integral_constant<int, q + from>{});
            __builtin_amdgcn_sched_barrier(0);
            for_each<per>([&](auto Z) CLEF_INLINE {
                if constexpr (q * per + decltype(Z)::value < FR) read(next, stage, H_NEXT, std::integral_constant<int, q * per + decltype(Z)::value>{});
            });
#pragma unroll
            for (int f = f0 + q * nf / n; f < f0 + (q + 1) * nf / n; f++) fill_one(fill_kt, fill_stage, f);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    constexpr std::integral_constant<int, 0> first_half, zero;
    constexpr std::integral_constant<int, 1> second_half;
    constexpr std::integral_constant<int, FILLS / 2> some_fills;
    constexpr std::integral_constant<int, FILLS> all_fills;
    constexpr std::integral_constant<int, P / 4> some;      // products ahead of the barrier
    // K tile kt, at POS of its group, and the first operands of the next. Behind the barrier kt + 1 may be read, and kt's buffer,
    // which every wave has left, takes kt + STAGES: half of it now, the rest with the next tile's first products. The scales of a group,
    // which every wave has in registers by its second tile, make room there for the next group's, which arrive ahead of its codes.
    unsigned stage = 0;                                     // of kt
    auto after = [&](unsigned st) CLEF_INLINE { return st == (STAGES - 1) * C::STAGE_BYTES ? 0u : st + C::STAGE_BYTES; };
    auto k_tile = [&](int kt, auto POS) CLEF_INLINE {
        constexpr int pos = decltype(POS)::value, next = (pos + 1) & 3;
        const unsigned before = stage == 0 ? (STAGES - 1) * C::STAGE_BYTES : stage - C::STAGE_BYTES;
        step(POS, r0, first_half, zero, r1, stage, second_half, kt + STAGES - 1, before, some_fills, all_fills);
        lds_wait(r1);
        __builtin_amdgcn_sched_barrier(0);
        for_each<decltype(some)::value>([&](auto Q) CLEF_INLINE { product(r1, POS, second_half, Q); });
        __builtin_amdgcn_sched_barrier(0);
        // in flight may stay what was issued behind kt + 1's codes: those of STAGES - 2 tiles, and scales where they went between
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"((STAGES - 2) * FILLS + (next >= 2 && next < STAGES ? S_FILLS : 0)) : "memory");
        if constexpr (next == 1) fill_scales((kt >> 2) + 1);
        if constexpr (next == 0) read_scales();
        const unsigned here = stage;
        stage = after(stage);
        step(POS, r1, second_half, some, r0, stage, first_half, kt + STAGES, here, zero, some_fills);
        if constexpr (next == 0) {
            lds_wait(r0, s_next);
            take_scales();
        } else {
            lds_wait(r0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    fill_scales(0);
    for (int q = 0; q < STAGES - 1; q++)
#pragma unroll
        for (int f = 0; f < FILLS; f++) fill_one(q, q * C::STAGE_BYTES, f);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"((STAGES - 2) * FILLS) : "memory");
    for_each<FR>([&](auto I) CLEF_INLINE { read(r0, 0, first_half, I); });
    read_scales();
    lds_wait(r0, s_next);
    take_scales();
#pragma unroll
    for (int f = 0; f < FILLS / 2; f++) fill_one(STAGES - 1, (STAGES - 1) * C::STAGE_BYTES, f);
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
