// Which form of the 4-bit product takes T rows of X and N rows of W (host only).
#pragma once

namespace clef_hip {
namespace mx4 {

// The compute units of the chips this library is built for (gfx950): forms are chosen for them.
constexpr int kCus = 256;

// X in 4 bits: row and column tiles of 16 a workgroup, or tiles of rows x columns
enum Form4 { ROWS_1X1, ROWS_1X2, ROWS_2X2, ROWS_2X4, ROWS_4X4, TILE_64X128, TILE_128X128, TILE_256X128, TILE_256X256, FORMS4 };
constexpr const char *kForms4[FORMS4] = {"rows 1x1", "rows 1x2", "rows 2x2", "rows 2x4", "rows 4x4", "tile 64x128", "tile 128x128", "tile 256x128", "tile 256x256"};
// X in bf16; _FEW: at most four rows, a quarter of the loads of X; _W4: four waves, two workgroups a CU, else eight and one
enum Form16 { ROWS16_1X1_FEW, ROWS16_1X1, ROWS16_1X2_FEW, ROWS16_1X2, ROWS16_1X4_FEW, ROWS16_1X4, ROWS16_2X4, ROWS16_2X4_W4, WIDE_64X256, WIDE_128X256, FORMS16 };
constexpr const char *kForms16[FORMS16] = {"rows 1x1 few", "rows 1x1", "rows 1x2 few", "rows 1x2", "rows 1x4 few", "rows 1x4", "rows 2x4", "rows 2x4/4", "tile 64x256", "tile 128x256"};

inline long groups_of(int a, int b) { return a / b + (a % b != 0); }
inline long blocks_of(int T, int N, int bm, int bn) { return groups_of(T, bm) * groups_of(N, bn); }
// The time of n tiles, two a CU at a time, of which a round takes `full` and one of no more than a CU each `half`.
inline float rounds(long n, float half, float full) {
    const long r = n % (2 * kCus);
    return (float)(n / (2 * kCus)) * full + (r == 0 ? 0.f : r <= kCus ? half : full);
}

// Where a form's workgroups make no more than one for each CU, its K loop is the time, and the smallest
// tile wins; else the rounds of workgroups count. Measured in us (three weights in turn, K 6,144 at N 5,120, 5,120 at 14,336):
//   4 bits, rows forms MT x NT row and column tiles of 16: N 5,120, 16 rows: 1x2 5.1, 2x2 6.0, 1x1 6.0; 32 rows: 2x2 6.2, 1x2 6.8; 64 rows: 2x4 7.1,
//     1x2 8.9; 128 rows: 4x4 9.5, tiles 64 x 128 10.5; 256 rows: tiles 64 x 128 10.8, 4x4 17.3. N 14,336, 16 rows: 2x4 8.6, 1x1 9.1; 96 rows: tiles
//     64 x 128 10.2, 4x4 17.1. One row at N 34,816: tiles 64 x 128 21.4, 2x4 20.1.
//   bf16 rows: N 5,120, 16 rows: 1x2 7.2, 1x4 9.2; 48 rows: 1x4 9.8, 1x2 11.8; 64 rows: 2x4 12.5, 1x4 13.9; 128 rows: 2x4 of four waves (two
//     workgroups a CU) 20, of eight 23; tiles of 64 x 256 33 up to 256 rows. N 14,336, 96 rows: 2x4 of four waves 28.1, tiles of 64 x 256 27.8; 128 rows
//     33 and 28. The rule loses at one row of more than 16,384 columns: N 20,480 17.7 (1x4 in two rounds 13.1), N 34,816 37 (20).
inline Form4 form4(int T, int N) {
    if (blocks_of(T, N, 16, 16) <= kCus) return ROWS_1X1;
    if (blocks_of(T, N, 16, 32) <= kCus) return ROWS_1X2;
    if (blocks_of(T, N, 32, 32) <= kCus) return ROWS_2X2;
    if (blocks_of(T, N, 32, 64) <= kCus) return ROWS_2X4;
    if (blocks_of(T, N, 64, 64) <= kCus) return ROWS_4X4;
    // rounds of 40 K tiles, us, on two chips: 256 rows x 14,336 small 16.3 to 16.7, middle 13.2 to 13.6, large 17.2 to 17.6, square 25; 512 rows 32, 25, 23,
    // 28; 2,048 rows 116, 82 to 85, 78 to 80, 71 to 75; 4,096 rows 218 to 223, 162 to 164, 141 to 149, 143 to 149; 3,000 x 10,240 x 4,096 95, 71 to 75,
    // 66 to 68, 61 to 67; 1,160 x 5,120 x 6,144 27 to 28, 25.4 to 26.0, 24.7 to 25.0, 32; 2,048 rows 45, 40, 40 to 42, 38 to 39
    const float small = rounds(blocks_of(T, N, 64, 128), 10.5f, 16.7f), middle = rounds(blocks_of(T, N, 128, 128), 13.f, 24.5f);
    const float large = rounds(blocks_of(T, N, 256, 128), 20.f, 41.f);
    const float square = 36.f * (float)((blocks_of(T, N, 256, 256) + kCus - 1) / kCus);
    if (square < large && square < middle && square < small) return TILE_256X256;
    if (small <= middle && small <= large) return TILE_64X128;
    return middle <= large ? TILE_128X128 : TILE_256X128;
}

inline Form16 form16(int T, int N) {
    const bool few = T <= 4;
    if (blocks_of(T, N, 16, 16) <= kCus) return few ? ROWS16_1X1_FEW : ROWS16_1X1;
    if (blocks_of(T, N, 16, 32) <= kCus) return few ? ROWS16_1X2_FEW : ROWS16_1X2;
    if (blocks_of(T, N, 16, 64) <= kCus) return few ? ROWS16_1X4_FEW : ROWS16_1X4;
    if (blocks_of(T, N, 32, 64) <= kCus) return ROWS16_2X4;
    if (blocks_of(T, N, 32, 64) <= 2 * kCus) return ROWS16_2X4_W4;
    // rounds of 40 K tiles, us, on two chips: 256 rows x 14,336 small 33 to 34, large 48; 512 rows 68 to 70, 61 to 64; 2,048 rows 242, 241; 4,096 rows
    // 455 to 480, 441 to 455
    const float large = 58.f * (float)((blocks_of(T, N, 128, 256) + kCus - 1) / kCus);
    return rounds(blocks_of(T, N, 64, 256), 31.f, 64.f) <= large ? WIDE_64X256 : WIDE_128X256;
}

}  // namespace mx4
}  // namespace clef_hip
