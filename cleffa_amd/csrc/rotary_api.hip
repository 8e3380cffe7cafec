// C ABI of the rotary operator: frequency tables, argument checks and launches. Documented in include/clef_hip_attn.h.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "clef_hip_attn.h"
#include "ranges.h"
#include "rotary.h"

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

bool group_ok(const char *what, const clef_hip_rotary_heads *g, int T, int hd, int size, int out_size, char *err, size_t errlen) {
    if (g->heads < 0 || g->heads > 4096) return fail(err, errlen, "rotary: %d %s heads", g->heads, what);
    if (g->heads == 0 || T == 0) return true;
    if (!g->x || !g->out || (uintptr_t)g->x % size || (uintptr_t)g->out % out_size || ((uintptr_t)g->norm & 3u))
        return fail(err, errlen, "rotary: %s, its output and norm must be aligned device pointers", what);
    if ((T > 1 && (g->x_row < 0 || g->out_row < 0)) || (g->heads > 1 && (g->x_head < 0 || g->out_head < 0)))
        return fail(err, errlen, "rotary: negative %s strides", what);
    if (!span_ok(T, g->x_row, size) || !span_ok(T, g->out_row, size) || !span_ok(g->heads, g->x_head, size) || !span_ok(g->heads, g->out_head, size))
        return fail(err, errlen, "rotary: %s too far apart", what);
    // rows of heads, or heads of rows
    const long row = T > 1 ? g->out_row : LONG_MAX, head = g->heads > 1 ? g->out_head : LONG_MAX;
    const bool by_row = head >= hd && (T == 1 || row >= (g->heads - 1) * g->out_head + hd);
    const bool by_head = row >= hd && (g->heads == 1 || head >= (T - 1) * g->out_row + hd);
    if (!by_row && !by_head) return fail(err, errlen, "rotary: heads or rows of the %s output overlap", what);
    if (g->x == g->out && size != out_size) return fail(err, errlen, "rotary: %s in place needs outputs of the same type", what);
    if (g->x == g->out && ((T > 1 && g->x_row != g->out_row) || (g->heads > 1 && g->x_head != g->out_head)))
        return fail(err, errlen, "rotary: %s in place needs the same strides", what);
    return true;
}

// whether all of a group's runs of v values of `size` bytes, `out_size` of its outputs, start at multiples of their size
bool runs_ok(const clef_hip_rotary_heads *g, int T, int v, int size, int out_size) {
    if (g->heads == 0) return true;
    if ((uintptr_t)g->x % (v * size) || (uintptr_t)g->out % (v * out_size)) return false;
    if (g->heads > 1 && (g->x_head % v || g->out_head % v)) return false;
    return T <= 1 || (g->x_row % v == 0 && g->out_row % v == 0);
}

// Whether outputs have bytes of heads that are read, or of each other; heads turned in place are their own outputs.
bool overlap(const clef_hip_rotary_args *a, int size, int out_size) {
    const auto heads = [&](const void *p, const clef_hip_rotary_heads &g, long row, long head, long size) {
        return Heads{(uintptr_t)p, a->T, g.heads && a->T > 1 ? row * size : 0, g.heads, g.heads > 1 ? head * size : 0, a->hd * size};
    };
    const Heads q = heads(a->q.x, a->q, a->q.x_row, a->q.x_head, size), k = heads(a->k.x, a->k, a->k.x_row, a->k.x_head, size);
    const Heads qo = heads(a->q.out, a->q, a->q.out_row, a->q.out_head, out_size), ko = heads(a->k.out, a->k, a->k.out_row, a->k.out_head, out_size);
    return (a->q.x != a->q.out && meet(qo, q)) || (a->k.x != a->k.out && meet(ko, k)) || meet(qo, k) || meet(ko, q) || meet(qo, ko);
}

rotary::Group group(const clef_hip_rotary_heads *g, int out_size) {
    return rotary::Group{g->x, g->out, g->norm, g->x_row, g->x_head, g->out_row, g->out_head, g->heads,
                         whole_lines(g->out, g->out_row * out_size) && whole_lines(g->out, g->out_head * out_size)};
}

template <int TYPE, int OUT, int V, int L, int I, bool HALF>
void launch_tokens(const rotary::Params &p, hipStream_t s) {
    if (p.T <= 512) hipLaunchKernelGGL((rotary::rotary_kernel<TYPE, OUT, V, L, I, 1, HALF>), dim3((unsigned)p.T), dim3(rotary::kThreads), 0, s, p);
    else hipLaunchKernelGGL((rotary::rotary_kernel<TYPE, OUT, V, L, I, 4, HALF>), dim3((unsigned)((p.T + 3) / 4)), dim3(rotary::kThreads), 0, s, p);
}
template <int TYPE, int OUT, int V, int L, int I>
void launch(rotary::Params &p, hipStream_t s) {
    p.q_units = (p.q.heads + 64 / L - 1) / (64 / L);
    p.units = p.q_units + (p.k.heads + 64 / L - 1) / (64 / L);
    if (p.half) launch_tokens<TYPE, OUT, V, L, I, true>(p, s);
    else launch_tokens<TYPE, OUT, V, L, I, false>(p, s);
}
// L: the least power of two of lanes that holds a head in pairs of runs of V
template <int TYPE, int OUT, int V>
void launch_runs(rotary::Params &p, hipStream_t s) {
    const int pairs = (p.hd + 2 * V - 1) / (2 * V);
    if (pairs <= 4) launch<TYPE, OUT, V, 4, 1>(p, s);
    else if (pairs <= 8) launch<TYPE, OUT, V, 8, 1>(p, s);
    else if (pairs <= 16) launch<TYPE, OUT, V, 16, 1>(p, s);
    else if constexpr (V <= 4) {
        if (pairs <= 32) launch<TYPE, OUT, V, 32, 1>(p, s);
        else if constexpr (V <= 2) {
            if (pairs <= 64) launch<TYPE, OUT, V, 64, 1>(p, s);
            else launch<TYPE, OUT, V, 64, 2>(p, s);
        }
    }
}
template <int TYPE, int OUT>
void launch_type(rotary::Params &p, int v, hipStream_t s) {
    if constexpr (TYPE != CLEF_HIP_OUT_F32) {
        if (v == 8) return launch_runs<TYPE, OUT, 8>(p, s);
    }
    if (v == 4) launch_runs<TYPE, OUT, 4>(p, s);
    else if (v == 2) launch_runs<TYPE, OUT, 2>(p, s);
    else launch_runs<TYPE, OUT, 1>(p, s);
}

}  // namespace

extern "C" {

bool clef_hip_rotary_freqs(int n_rot, double theta, int scaling, double factor, double original, double low, double high, double *freq,
                           char *err, size_t errlen) {
    if (n_rot <= 0 || n_rot % 2 || n_rot > rotary::kMaxHd) return fail(err, errlen, "rotary: n_rot %d must be even, 2 to %d", n_rot, rotary::kMaxHd);
    if (!(theta > 1.) || !isfinite(theta)) return fail(err, errlen, "rotary: bad theta");
    if (scaling < CLEF_HIP_ROTARY_NONE || scaling > CLEF_HIP_ROTARY_PARTS) return fail(err, errlen, "rotary: bad scaling %d", scaling);
    if (scaling != CLEF_HIP_ROTARY_NONE && (!(factor >= 1.) || !isfinite(factor))) return fail(err, errlen, "rotary: the scaling factor must be at least 1");
    if (scaling == CLEF_HIP_ROTARY_BASE && n_rot == 2) return fail(err, errlen, "rotary: a changed base needs more than one pair");
    if (scaling == CLEF_HIP_ROTARY_PARTS && (!(original > 0.) || !isfinite(original) || !(low >= 0.) || !(high > low) || !isfinite(high)))
        return fail(err, errlen, "rotary: scaling by parts needs an original length and 0 <= low < high");
    if (!freq) return fail(err, errlen, "rotary: missing freq");
    const double tau = 6.283185307179586476925;
    const double base = scaling == CLEF_HIP_ROTARY_BASE ? theta * pow(factor, (double)n_rot / (n_rot - 2)) : theta;
    if (!isfinite(base)) return fail(err, errlen, "rotary: theta %g scaled by %g is too large", theta, factor);
    for (int j = 0; j < n_rot / 2; j++) {
        double f = pow(base, -2. * j / n_rot);
        if (scaling == CLEF_HIP_ROTARY_LINEAR) f /= factor;
        if (scaling == CLEF_HIP_ROTARY_PARTS) {
            const double keep = fmin(1., fmax(0., (original * f / tau - low) / (high - low)));
            f = keep * f + (1. - keep) * f / factor;
        }
        freq[j] = f / tau;
    }
    return true;
}

bool clef_hip_rotary(const clef_hip_rotary_args *a, void *stream, char *err, size_t errlen) {
    if (!a) return fail(err, errlen, "null rotary arguments");
    if (a->T < 0 || a->T > CLEF_HIP_ROTARY_ROWS) return fail(err, errlen, "rotary: %d rows, 0 to %d are supported", a->T, CLEF_HIP_ROTARY_ROWS);
    if (a->hd <= 0 || a->hd > rotary::kMaxHd || a->hd % 2) return fail(err, errlen, "rotary: head dim %d must be even, 2 to %d", a->hd, rotary::kMaxHd);
    if (a->n_rot <= 0 || a->n_rot % 2 || a->n_rot > a->hd) return fail(err, errlen, "rotary: n_rot %d must be even, 2 to the head dim", a->n_rot);
    if (a->layout != CLEF_HIP_ROTARY_HALF && a->layout != CLEF_HIP_ROTARY_INTERLEAVED) return fail(err, errlen, "rotary: bad layout %d", a->layout);
    if (a->axes < 1 || a->axes > 4) return fail(err, errlen, "rotary: %d position axes, 1 to 4 are supported", a->axes);
    if (a->type < CLEF_HIP_OUT_BF16 || a->type > CLEF_HIP_OUT_F32) return fail(err, errlen, "rotary: bad type %d", a->type);
    if (!(a->eps >= 0.f) || !isfinite(a->magnitude)) return fail(err, errlen, "rotary: bad eps or magnitude");
    if (a->bf16_out != 0 && (a->bf16_out != 1 || a->type != CLEF_HIP_OUT_F32)) return fail(err, errlen, "rotary: bf16_out %d goes with f32 heads", a->bf16_out);
    const int size = a->type == CLEF_HIP_OUT_F32 ? 4 : 2, out_size = a->bf16_out ? 2 : size;
    if (!group_ok("q", &a->q, a->T, a->hd, size, out_size, err, errlen) || !group_ok("k", &a->k, a->T, a->hd, size, out_size, err, errlen)) return false;
    if (a->T == 0 || a->q.heads + a->k.heads == 0) return true;
    if (!a->pos || !a->freq || ((uintptr_t)a->pos & 3u) || ((uintptr_t)a->freq & 7u)) return fail(err, errlen, "rotary: pos and freq must be aligned device pointers");
    if (overlap(a, size, out_size)) return fail(err, errlen, "rotary: an output overlaps the other one, or heads that are read");
    rotary::Params p;
    p.q = group(&a->q, out_size); p.k = group(&a->k, out_size); p.pos = a->pos; p.freq = a->freq;
    p.T = a->T; p.hd = a->hd; p.n_rot = a->n_rot; p.half = a->layout == CLEF_HIP_ROTARY_HALF; p.axes = a->axes;
    p.eps = a->eps; p.magnitude = a->magnitude;
    // the longest runs that heads divide into and that pointers and strides allow
    int v = 16 / size;
    while (v > 1 && (a->hd % v || (p.half && (a->n_rot / 2) % v) || !runs_ok(&a->q, a->T, v, size, out_size) || !runs_ok(&a->k, a->T, v, size, out_size))) v /= 2;
    const hipStream_t s = (hipStream_t)stream;
    if (a->type == CLEF_HIP_OUT_BF16) launch_type<CLEF_HIP_OUT_BF16, CLEF_HIP_OUT_BF16>(p, v, s);
    else if (a->type == CLEF_HIP_OUT_F16) launch_type<CLEF_HIP_OUT_F16, CLEF_HIP_OUT_F16>(p, v, s);
    else if (a->bf16_out) launch_type<CLEF_HIP_OUT_F32, CLEF_HIP_OUT_BF16>(p, v, s);
    else launch_type<CLEF_HIP_OUT_F32, CLEF_HIP_OUT_F32>(p, v, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(err, errlen, "rotary launch failed: %s", hipGetErrorString(e));
    return true;
}

}  // extern "C"
