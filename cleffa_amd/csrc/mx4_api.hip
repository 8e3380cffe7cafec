// C ABI of the microscaled 4-bit matrices: argument checks and launches. Documented in include/clef_hip_attn.h.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "clef_hip_attn.h"
#include "mx4_forms.h"
#include "mx4_gemm.h"
#include "mx4_params.h"
#include "mx4_quant.h"
#include "mx4_rows16.h"
#include "mx4_tile.h"
#include "mx4_wide.h"
#include "ranges.h"

using namespace clef_hip;

namespace {

bool fail(char *err, size_t errlen, const char *fmt, ...) {
    if (err && errlen) {
        int n = snprintf(err, errlen, "hip: ");
        if (n < 0) n = 0;
        if ((size_t)n < errlen) {
            va_list ap;
            va_start(ap, fmt);
            vsnprintf(err + n, errlen - (size_t)n, fmt, ap);
            va_end(ap);
        }
    }
    return false;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

bool launch_ok(const char *what, char *err, size_t errlen) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(err, errlen, "%s launch failed: %s", what, hipGetErrorString(e));
    return true;
}

// A launch holds fewer than 2^32 threads: of rows / 16 x K / 512 workgroups of 256, fewer than 2^24.
bool shape_ok(const char *what, int rows, int K, char *err, size_t errlen) {
    if (rows < 0 || rows > CLEF_HIP_MX4_MAX) return fail(err, errlen, "%s: %d rows, 0 to %d are supported", what, rows, CLEF_HIP_MX4_MAX);
    if (K <= 0 || K > CLEF_HIP_MX4_MAX || K % mx4::BLOCK)
        return fail(err, errlen, "%s: rows of %d values, multiples of %d up to %d are supported", what, K, mx4::BLOCK, CLEF_HIP_MX4_MAX);
    if ((long)mx4::ceil_div(rows, mx4::ROWS) * mx4::ceil_div(K, mx4::KG) >= (1L << 24))
        return fail(err, errlen, "%s: %d x %d values are too many", what, rows, K);
    return true;
}

bool matrix_ok(const char *what, const uint8_t *codes, const uint8_t *scales, char *err, size_t errlen) {
    if (!codes || !scales || !aligned16(codes) || !aligned16(scales))
        return fail(err, errlen, "%s codes and scales must be 16-byte aligned device pointers", what);
    return true;
}

// Y and the residual by rows, each row from its first to its last value.
Rows rows_of(const void *p, int n, long row, long values, long size) { return Rows{(uintptr_t)p, n, n > 1 ? row * size : 0, values * size}; }
// Whether the residual is Y itself, or none of its values one of Y's.
bool apart(const clef_hip_mx4_gemm_args *a) {
    return (a->y == a->residual && (a->T == 1 || a->y_row == a->r_row)) || !meet(rows_of(a->y, a->T, a->y_row, a->N, 4), rows_of(a->residual, a->T, a->r_row, a->N, 4));
}
// Whether rows have bytes of a matrix's buffers.
bool meets_matrix(const Rows &y, const uint8_t *codes, const uint8_t *scales, int rows, int K) {
    const size_t tiles = (size_t)mx4::ceil_div(rows, mx4::ROWS);
    return meets(y, (uintptr_t)codes, (uintptr_t)codes + tiles * mx4::ceil_div(K, mx4::KT) * mx4::TILE_BYTES) ||
           meets(y, (uintptr_t)scales, (uintptr_t)scales + tiles * mx4::ceil_div(K, mx4::KG) * mx4::GROUP_BYTES);
}

// x of a quantisation or of values: rows not too far apart, and outside of the matrix.
bool rows_ok(const char *what, const clef_hip_mx4_rows_args *a, char *err, size_t errlen) {
    const int size = a->type == CLEF_HIP_OUT_F32 ? 4 : 2;
    if (!span_ok(a->rows, a->row, size)) return fail(err, errlen, "%s: rows too far apart", what);
    if (meets_matrix(rows_of(a->x, a->rows, a->row, a->K, size), a->codes, a->scales, a->rows, a->K)) return fail(err, errlen, "%s: x overlaps codes or scales", what);
    return true;
}

mx4::Matrix matrix(const uint8_t *codes, const uint8_t *scales, int rows, int K) {
    return mx4::Matrix{codes, scales, rows, mx4::ceil_div(K, mx4::KT), mx4::ceil_div(K, mx4::KG)};
}

template <int TYPE>
void launch_quantise(const mx4::QuantParams &p, hipStream_t s) {
    hipLaunchKernelGGL(mx4::mx4_quantise_kernel<TYPE>, dim3((unsigned)(mx4::ceil_div(p.rows, mx4::ROWS) * p.kgroups)), dim3(mx4::kQuantThreads), 0, s, p);
}

template <int MT, int NT>
void launch_rows(const mx4::GemmParams &p, hipStream_t s) {
    constexpr int W = 8, D = MT == 1 ? 3 : 2;
    hipLaunchKernelGGL((mx4::mx4_rows_kernel<MT, NT, W, D>), dim3((unsigned)mx4::blocks_of(p.T, p.N, 16 * MT, 16 * NT)), dim3(64 * W), 0, s, p);
}
template <int MT, int NT, int W, int XF>
void launch_rows16(const mx4::GemmParams &p, hipStream_t s) {
    hipLaunchKernelGGL((mx4::mx4_rows16_kernel<MT, NT, W, XF>), dim3((unsigned)mx4::blocks_of(p.T, p.N, 16 * MT, 16 * NT)), dim3(64 * W), 0, s, p);
}

template <typename C>
dim3 tile_grid(const mx4::GemmParams &p) {
    return dim3((unsigned)(8 * mx4::ceil_div(mx4::ceil_div(p.N, C::BN), 8) * mx4::ceil_div(p.T, C::BM)));
}
template <typename C>
void launch_tile(const mx4::GemmParams &p, hipStream_t s) {
    hipLaunchKernelGGL(mx4::mx4_tile_kernel<C>, tile_grid<C>(p), dim3(C::THREADS), 0, s, p);
}
template <typename C>
void launch_wide(const mx4::GemmParams &p, hipStream_t s) {
    hipLaunchKernelGGL(mx4::mx4_wide_kernel<C>, tile_grid<C>(p), dim3(C::THREADS), 0, s, p);
}

void launch4(const mx4::GemmParams &p, hipStream_t s) {
    switch (mx4::form4(p.T, p.N)) {
    case mx4::ROWS_1X1: return launch_rows<1, 1>(p, s);
    case mx4::ROWS_1X2: return launch_rows<1, 2>(p, s);
    case mx4::ROWS_2X2: return launch_rows<2, 2>(p, s);
    case mx4::ROWS_2X4: return launch_rows<2, 4>(p, s);
    case mx4::ROWS_4X4: return launch_rows<4, 4>(p, s);
    case mx4::TILE_64X128: return launch_tile<mx4::TileCfg<64, 128, 64, 32, 4, 2>>(p, s);
    case mx4::TILE_128X128: return launch_tile<mx4::TileCfg<128, 128, 64, 64, 4, 2>>(p, s);
    // eight waves; with four, where each CU has one: 425 x 10,240 x 4,096 17.0 us, with eight 16.0
    case mx4::TILE_256X128: return launch_tile<mx4::TileCfg<256, 128, 64, 64, 3, 2>>(p, s);
    // eight waves, one workgroup a CU
    default: return launch_tile<mx4::TileCfg<256, 256, 128, 64, 4, 1>>(p, s);
    }
}

void launch16(const mx4::GemmParams &p, hipStream_t s) {
    switch (mx4::form16(p.T, p.N)) {
    case mx4::ROWS16_1X1_FEW: return launch_rows16<1, 1, 8, 1>(p, s);
    case mx4::ROWS16_1X1: return launch_rows16<1, 1, 8, 4>(p, s);
    case mx4::ROWS16_1X2_FEW: return launch_rows16<1, 2, 8, 1>(p, s);
    case mx4::ROWS16_1X2: return launch_rows16<1, 2, 8, 4>(p, s);
    case mx4::ROWS16_1X4_FEW: return launch_rows16<1, 4, 8, 1>(p, s);
    case mx4::ROWS16_1X4: return launch_rows16<1, 4, 8, 4>(p, s);
    case mx4::ROWS16_2X4: return launch_rows16<2, 4, 8, 8>(p, s);
    case mx4::ROWS16_2X4_W4: return launch_rows16<2, 4, 4, 8>(p, s);
    case mx4::WIDE_64X256: return launch_wide<mx4::WideCfg<64, 256, 64, 64, 2, 2>>(p, s);      // two workgroups a CU
    default: return launch_wide<mx4::WideCfg<128, 256, 64, 128, 2, 1>>(p, s);                  // one
    }
}

}  // namespace

extern "C" {

bool clef_hip_mx4_sizes(int rows, int K, size_t *code_bytes, size_t *scale_bytes, char *err, size_t errlen) {
    if (!shape_ok("4-bit matrix", rows, K, err, errlen)) return false;
    const size_t rt = (size_t)mx4::ceil_div(rows, mx4::ROWS);
    if (code_bytes) *code_bytes = rt * mx4::ceil_div(K, mx4::KT) * mx4::TILE_BYTES;
    if (scale_bytes) *scale_bytes = rt * mx4::ceil_div(K, mx4::KG) * mx4::GROUP_BYTES;
    return true;
}

bool clef_hip_mx4_quantise(const clef_hip_mx4_rows_args *a, void *stream, char *err, size_t errlen) {
    if (!a) return fail(err, errlen, "null quantise arguments");
    if (!shape_ok("quantise", a->rows, a->K, err, errlen)) return false;
    if (a->type < CLEF_HIP_OUT_BF16 || a->type > CLEF_HIP_OUT_F32) return fail(err, errlen, "quantise: bad type %d", a->type);
    if (a->row < a->K || a->row % 8) return fail(err, errlen, "quantise: row %ld must be >= %d and a multiple of 8", a->row, a->K);
    if (a->rows == 0) return true;
    if (!matrix_ok("quantise:", a->codes, a->scales, err, errlen)) return false;
    if (!a->x || !aligned16(a->x)) return fail(err, errlen, "quantise: x must be a 16-byte aligned device pointer");
    if (!rows_ok("quantise", a, err, errlen)) return false;
    mx4::QuantParams p{a->x, nullptr, a->codes, a->scales, a->rows, a->K, mx4::ceil_div(a->K, mx4::KT), mx4::ceil_div(a->K, mx4::KG), a->row, false};
    if (a->type == CLEF_HIP_OUT_BF16) launch_quantise<mx4::X_BF16>(p, (hipStream_t)stream);
    else if (a->type == CLEF_HIP_OUT_F16) launch_quantise<mx4::X_F16>(p, (hipStream_t)stream);
    else launch_quantise<mx4::X_F32>(p, (hipStream_t)stream);
    return launch_ok("mx4_quantise", err, errlen);
}

bool clef_hip_mx4_values(const clef_hip_mx4_rows_args *a, void *stream, char *err, size_t errlen) {
    if (!a) return fail(err, errlen, "null values arguments");
    if (!shape_ok("values", a->rows, a->K, err, errlen)) return false;
    if (a->type != CLEF_HIP_OUT_BF16 && a->type != CLEF_HIP_OUT_F32) return fail(err, errlen, "values: bad type %d (bf16 and f32 hold every value)", a->type);
    if (a->row < a->K || a->row % 8) return fail(err, errlen, "values: row %ld must be >= %d and a multiple of 8", a->row, a->K);
    if (a->rows == 0) return true;
    if (!matrix_ok("values:", a->codes, a->scales, err, errlen)) return false;
    if (!a->x || !aligned16(a->x)) return fail(err, errlen, "values: x must be a 16-byte aligned device pointer");
    if (!rows_ok("values", a, err, errlen)) return false;
    mx4::QuantParams p{nullptr, a->x, a->codes, a->scales, a->rows, a->K, mx4::ceil_div(a->K, mx4::KT), mx4::ceil_div(a->K, mx4::KG), a->row,
                       whole_lines(a->x, a->row * (a->type == CLEF_HIP_OUT_F32 ? 4 : 2))};
    const dim3 grid((unsigned)((long)mx4::ceil_div(a->rows, mx4::ROWS) * p.kgroups)), block(mx4::kQuantThreads);
    if (a->type == CLEF_HIP_OUT_BF16) hipLaunchKernelGGL(mx4::mx4_values_kernel<false>, grid, block, 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(mx4::mx4_values_kernel<true>, grid, block, 0, (hipStream_t)stream, p);
    return launch_ok("mx4_values", err, errlen);
}

bool clef_hip_mx4_pack(int rows, int K, uint8_t *flat_codes, uint8_t *flat_scales, uint8_t *codes, uint8_t *scales, int to_flat,
                       void *stream, char *err, size_t errlen) {
    if (!shape_ok("pack", rows, K, err, errlen)) return false;
    if (rows == 0) return true;
    if (!matrix_ok("pack:", codes, scales, err, errlen)) return false;
    if (!flat_codes || !flat_scales || !aligned16(flat_codes)) return fail(err, errlen, "pack: flat codes must be a 16-byte aligned device pointer, flat scales a device pointer");
    if (meets_matrix(rows_of(flat_codes, 1, 0, (long)rows * (K / 2), 1), codes, scales, rows, K) ||
        meets_matrix(rows_of(flat_scales, 1, 0, (long)rows * (K / mx4::BLOCK), 1), codes, scales, rows, K))
        return fail(err, errlen, "pack: flat codes or scales overlap the matrix");
    mx4::PackParams p{flat_codes, flat_scales, codes, scales, rows, K, mx4::ceil_div(K, mx4::KT), mx4::ceil_div(K, mx4::KG)};
    const size_t blocks = (size_t)rows * (to_flat ? K / mx4::BLOCK : 16 * p.kgroups);
    const dim3 grid((unsigned)((blocks + 255) / 256));
    if (to_flat) hipLaunchKernelGGL(mx4::mx4_pack_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(mx4::mx4_pack_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, p);
    return launch_ok("mx4_pack", err, errlen);
}

bool clef_hip_mx4_gemm(const clef_hip_mx4_gemm_args *a, void *stream, char *err, size_t errlen) {
    if (!a) return fail(err, errlen, "null 4-bit product arguments");
    if (!shape_ok("4-bit product: W", a->N, a->K, err, errlen) || !shape_ok("4-bit product: X", a->T, a->K, err, errlen)) return false;
    if (a->N == 0) return fail(err, errlen, "4-bit product: W has no rows");
    if (a->y_type != CLEF_HIP_GEMM_Y_F32 && a->y_type != CLEF_HIP_GEMM_Y_BF16) return fail(err, errlen, "4-bit product: bad y_type %d", a->y_type);
    if (a->residual && a->y_type != CLEF_HIP_GEMM_Y_F32) return fail(err, errlen, "4-bit product: a residual needs an f32 Y");
    if (a->y_row < a->N || (a->residual && a->r_row < a->N)) return fail(err, errlen, "4-bit product: rows of Y and the residual must hold %d values", a->N);
    const int y_size = a->y_type == CLEF_HIP_GEMM_Y_BF16 ? 2 : 4;
    if (!span_ok(a->T, a->y_row, y_size) || (a->residual && !span_ok(a->T, a->r_row, 4)) || (a->x_bf16 && !span_ok(a->T, a->x_row, 2)))
        return fail(err, errlen, "4-bit product: rows too far apart");
    if (!a->x_codes != !a->x_scales) return fail(err, errlen, "4-bit product: x_codes and x_scales must both be set or both be NULL");
    if (!a->x_codes == !a->x_bf16) return fail(err, errlen, "4-bit product: X must be given in 4 bits or in bf16");
    if (a->T == 0) return true;
    if (!matrix_ok("4-bit product: W", a->w_codes, a->w_scales, err, errlen)) return false;
    if (a->x_codes && !matrix_ok("4-bit product: X", a->x_codes, a->x_scales, err, errlen)) return false;
    if (a->x_bf16 && (!aligned16(a->x_bf16) || a->x_row < a->K || a->x_row % 8))
        return fail(err, errlen, "4-bit product: X must be 16-byte aligned, its row %ld >= %d and a multiple of 8", a->x_row, a->K);
    if (!a->y || (uintptr_t)a->y % y_size || ((uintptr_t)a->residual & 3u))
        return fail(err, errlen, "4-bit product: Y and the residual must be aligned device pointers");
    if (a->residual && !apart(a)) return fail(err, errlen, "4-bit product: the residual may be Y itself, but not overlap it otherwise");
    const Rows y = rows_of(a->y, a->T, a->y_row, a->N, y_size);
    if (meets_matrix(y, a->w_codes, a->w_scales, a->N, a->K)) return fail(err, errlen, "4-bit product: Y overlaps W");
    if (a->x_codes ? meets_matrix(y, a->x_codes, a->x_scales, a->T, a->K) : meet(y, rows_of(a->x_bf16, a->T, a->x_row, a->K, 2)))
        return fail(err, errlen, "4-bit product: Y overlaps X");
    mx4::GemmParams p;
    p.w = matrix(a->w_codes, a->w_scales, a->N, a->K);
    p.x = matrix(a->x_codes, a->x_scales, a->T, a->K);
    p.xb = a->x_bf16; p.x_row = a->x_row; p.y = a->y; p.y_row = a->y_row; p.residual = a->residual; p.r_row = a->r_row;
    p.T = a->T; p.N = a->N; p.K = a->K; p.y_bf16 = a->y_type == CLEF_HIP_GEMM_Y_BF16;
    p.past = whole_lines(a->y, a->y_row * (p.y_bf16 ? 2 : 4));
    if (p.xb) launch16(p, (hipStream_t)stream);
    else launch4(p, (hipStream_t)stream);
    return launch_ok("mx4_gemm", err, errlen);
}

}  // extern "C"
