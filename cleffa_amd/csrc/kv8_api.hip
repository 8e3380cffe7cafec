// C ABI of the 8-bit paged prefix cache: argument checks and launches. Documented in
// include/clef_hip_attn.h.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "clef_hip_attn.h"
#include "kv8_attn.h"
#include "kv8_pages.h"
#include "kv8_params.h"
#include "kv8_plan.h"

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

// The compute units of the chips this library is built for (gfx950): plans and workspaces are sized for
// them, so that a plan buffer's size needs no device.
constexpr int kCus = 256;

bool sizes_ok(int n_seq, int T, int nh, int nkv, char *err, size_t errlen) {
    if (nh <= 0 || nkv <= 0 || nh % nkv || nh / nkv > kv8::kMaxGroup) return fail(err, errlen, "bad head counts nh=%d nkv=%d", nh, nkv);
    if (nkv > 1024) return fail(err, errlen, "nkv %d too large", nkv);
    if (n_seq <= 0 || n_seq > kv8::kMaxSeq) return fail(err, errlen, "%d sequences: 1 to %d are supported", n_seq, kv8::kMaxSeq);
    if (T < 0 || T > kv8::kMaxRows) return fail(err, errlen, "%d pass rows: at most %d are supported", T, kv8::kMaxRows);
    return true;
}

bool pool_ok(int max_pages, int n_pages, int nkv, char *err, size_t errlen) {
    if (max_pages <= 0 || max_pages > kv8::kMaxTablePages)
        return fail(err, errlen, "table rows of %d pages: 1 to %d are supported", max_pages, kv8::kMaxTablePages);
    if (n_pages <= 0 || n_pages > INT32_MAX / CLEF_HIP_KV8_PAGE || (long)n_pages * nkv > INT32_MAX)
        return fail(err, errlen, "pool of %d pages", n_pages);
    return true;
}

bool fill(const clef_hip_kv8_args *a, bool core, kv8::Params *q, char *err, size_t errlen) {
    if (!a) return fail(err, errlen, "null 8-bit cache arguments");
    if (a->hd != kv8::HD) return fail(err, errlen, "the 8-bit cache supports hd 256 only (got %d)", a->hd);
    if (!sizes_ok(a->n_seq, a->T, a->nh, a->nkv, err, errlen) || !pool_ok(a->max_pages, a->n_pages, a->nkv, err, errlen)) return false;
    if (a->n_rot != 0 && a->n_rot != 64) return fail(err, errlen, "unsupported n_rot %d", a->n_rot);
    const long need_row = 2L * a->nh * a->hd + 2L * a->nkv * a->hd;
    if (a->row < need_row || a->row % 8) return fail(err, errlen, "qkv row %d must be >= %ld and a multiple of 8", a->row, need_row);
    if (a->T && (!a->qkv || !aligned16(a->qkv))) return fail(err, errlen, "qkv must be a 16-byte aligned device pointer");
    if (!aligned16(a->q_norm) || !aligned16(a->k_norm)) return fail(err, errlen, "norm weights must be 16-byte aligned");
    if (!a->k_norm != !a->q_norm) return fail(err, errlen, "q_norm and k_norm must both be set or both be NULL");
    if (a->T && a->n_rot && (!a->pos3 || !a->inv_freq)) return fail(err, errlen, "rotary needs pos3 and inv_freq");
    if (a->n_rot && !aligned16(a->inv_freq)) return fail(err, errlen, "inv_freq must be 16-byte aligned");
    if (!a->k_pages || !a->v_pages || !aligned16(a->k_pages) || !aligned16(a->v_pages)) return fail(err, errlen, "K / V pages must be 16-byte aligned device pointers");
    if (!a->k_scale || !a->v_scale) return fail(err, errlen, "missing page scales");
    if (!a->tables) return fail(err, errlen, "missing page tables");
    if (!a->plan || !aligned16(a->plan)) return fail(err, errlen, "plan must be a 16-byte aligned device pointer");
    if (!(a->eps >= 0.f)) return fail(err, errlen, "bad eps");
    q->l = kv8::layout(a->n_seq, a->T, a->nh, a->nkv, a->max_new, kCus);
    if (core) {
        if (a->T && (!a->out || !aligned16(a->out))) return fail(err, errlen, "out must be a 16-byte aligned device pointer");
        if (a->out_type < CLEF_HIP_OUT_BF16 || a->out_type > CLEF_HIP_OUT_F32) return fail(err, errlen, "bad out_type %d", a->out_type);
        if (!(a->scale > 0.f)) return fail(err, errlen, "bad scale");
        if (!a->workspace || !aligned16(a->workspace)) return fail(err, errlen, "workspace must be a 16-byte aligned device pointer");
        if (a->workspace_bytes < q->l.ws_bytes) return fail(err, errlen, "workspace of %zu bytes, %zu are needed", a->workspace_bytes, q->l.ws_bytes);
    }
    // the kernels load their list entries, at offsets by these sizes, together with the plan's header
    if (a->plan_ints < (size_t)q->l.ints) return fail(err, errlen, "plan of %zu int32, %ld are needed", a->plan_ints, q->l.ints);
    q->qkv = a->qkv; q->q_norm = a->q_norm; q->k_norm = a->k_norm; q->inv_freq = a->inv_freq; q->pos3 = a->pos3;
    q->tables = a->tables; q->plan = a->plan;
    q->k_pages = a->k_pages; q->v_pages = a->v_pages; q->k_scale = a->k_scale; q->v_scale = a->v_scale;
    q->partial = (float *)a->workspace; q->out = a->out; q->ovf = a->ovf;
    q->nh = a->nh; q->nkv = a->nkv; q->group = a->nh / a->nkv; q->n_rot = a->n_rot; q->row = a->row; q->T = a->T;
    q->n_seq = a->n_seq; q->max_pages = a->max_pages; q->n_pages = a->n_pages; q->gate = a->gate; q->out_type = a->out_type;
    q->eps = a->eps; q->scale_log2 = a->scale * 1.4426950408889634f;
    q->f16_lim = (a->f16_lim > 0.f && a->f16_lim <= 65504.f) ? a->f16_lim : 65504.f;
    return true;
}

}  // namespace

extern "C" {

bool clef_hip_kv8_sizes(int n_seq, int T, int nh, int nkv, int max_new, size_t *plan_ints, size_t *workspace_bytes,
                        char *err, size_t errlen) {
    if (!sizes_ok(n_seq, T, nh, nkv, err, errlen)) return false;
    const kv8::Layout l = kv8::layout(n_seq, T, nh, nkv, max_new, kCus);
    if (plan_ints) *plan_ints = (size_t)l.ints;
    if (workspace_bytes) *workspace_bytes = l.ws_bytes;
    return true;
}

bool clef_hip_kv8_plan(const clef_hip_kv8_plan_args *a, void *stream, char *err, size_t errlen) {
    if (!a) return fail(err, errlen, "null plan arguments");
    if (!sizes_ok(a->n_seq, a->T, a->nh, a->nkv, err, errlen) || !pool_ok(a->max_pages, a->n_pages, a->nkv, err, errlen)) return false;
    if (!a->tables || !a->free_pages || !a->state || !a->state_out || !a->new_lens || !a->cu_q || (a->T && !a->slots))
        return fail(err, errlen, "missing page tables, free pages, state, lengths, cu_q or slots");
    if (!a->plan || !aligned16(a->plan)) return fail(err, errlen, "plan must be a 16-byte aligned device pointer");
    kv8::PlanParams p;
    p.l = kv8::layout(a->n_seq, a->T, a->nh, a->nkv, a->max_new, kCus);
    if (a->plan_ints < (size_t)p.l.ints) return fail(err, errlen, "plan of %zu int32, %ld are needed", a->plan_ints, p.l.ints);
    p.n_seq = a->n_seq; p.max_pages = a->max_pages; p.n_pages = a->n_pages; p.T = a->T; p.group = a->nh / a->nkv;
    p.tables = a->tables; p.free_pages = a->free_pages; p.state = a->state; p.state_out = a->state_out;
    p.new_lens = a->new_lens; p.pos_off = a->pos_off; p.cu_q = a->cu_q; p.slots = a->slots; p.pos3 = a->pos3; p.work = a->plan;
    if (a->n_seq <= 256 && a->T <= 256) hipLaunchKernelGGL(kv8::kv8_plan_kernel<256>, dim3(1), dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(kv8::kv8_plan_kernel<1024>, dim3(1), dim3(1024), 0, (hipStream_t)stream, p);
    if (!launch_ok("kv8_plan", err, errlen)) return false;
    if (a->T <= 1024) return true;
    hipLaunchKernelGGL(kv8::kv8_plan_rows_kernel, dim3((unsigned)((a->T + kv8::kRowThreads - 1) / kv8::kRowThreads)), dim3(kv8::kRowThreads), 0, (hipStream_t)stream, p);
    return launch_ok("kv8_plan", err, errlen);
}

bool clef_hip_kv8_append(const clef_hip_kv8_args *a, void *stream, char *err, size_t errlen) {
    kv8::Params p;
    if (!fill(a, false, &p, err, errlen)) return false;
    if (a->T == 0) return true;
    hipLaunchKernelGGL(kv8::kv8_append_kernel, dim3((unsigned)(p.l.max_app * p.nkv), 2), dim3(kv8::kAppendThreads), 0, (hipStream_t)stream, p);
    return launch_ok("kv8_append", err, errlen);
}

bool clef_hip_kv8_attention(const clef_hip_kv8_args *a, void *stream, char *err, size_t errlen) {
    kv8::Params p;
    if (!fill(a, true, &p, err, errlen)) return false;
    if (a->T == 0) return true;
    // a workgroup for every item the plan may hold: the plan's counts are on the device
    const unsigned grid = (unsigned)(p.l.max_items * p.nkv);
    if (p.l.bm == 16) hipLaunchKernelGGL(kv8::kv8_attn_rows_kernel<1>, dim3(grid), dim3(kv8::kRowsThreads), 0, (hipStream_t)stream, p);
    else if (p.l.bm == 128) hipLaunchKernelGGL(kv8::kv8_attn_tile_kernel, dim3(grid), dim3(kv8::kTileThreads), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(kv8::kv8_attn_rows_kernel<2>, dim3(grid), dim3(kv8::kRowsThreads), 0, (hipStream_t)stream, p);
    if (!launch_ok("kv8_attn", err, errlen)) return false;
    const long wgs = (long)p.T * p.nh;   // if every unit takes all of a workgroup's waves
    hipLaunchKernelGGL(kv8::kv8_join_kernel, dim3((unsigned)(wgs < 8L * kCus ? wgs : 8L * kCus)), dim3(kv8::kJoinThreads), 0, (hipStream_t)stream, p);
    return launch_ok("kv8_join", err, errlen);
}

bool clef_hip_kv8_read(const clef_hip_kv8_read_args *a, void *stream, char *err, size_t errlen) {
    if (!a) return fail(err, errlen, "null read arguments");
    if (a->hd != kv8::HD) return fail(err, errlen, "the 8-bit cache supports hd 256 only (got %d)", a->hd);
    if (!sizes_ok(a->n_seq, 0, a->nkv, a->nkv, err, errlen) || !pool_ok(a->max_pages, a->n_pages, a->nkv, err, errlen)) return false;
    if (!a->k_pages || !a->v_pages || !aligned16(a->k_pages) || !aligned16(a->v_pages)) return fail(err, errlen, "K / V pages must be 16-byte aligned device pointers");
    if (!a->k_scale || !a->v_scale) return fail(err, errlen, "missing page scales");
    if (!a->tables || !a->state || !a->cu) return fail(err, errlen, "missing page tables, state or cu");
    if (a->kvT < 0 || a->kvT % 8) return fail(err, errlen, "kvT %d must be a multiple of 8", a->kvT);
    if ((long)a->kvT * a->hd * 2 >= (1L << 32)) return fail(err, errlen, "kvT %d too large for 32-bit plane offsets", a->kvT);
    if (a->kvT == 0) return true;
    if (!a->k_plane || !a->vt_plane || !aligned16(a->k_plane) || !aligned16(a->vt_plane)) return fail(err, errlen, "K / V^T planes must be 16-byte aligned");
    kv8::ReadParams p;
    p.k_pages = a->k_pages; p.v_pages = a->v_pages; p.k_scale = a->k_scale; p.v_scale = a->v_scale;
    p.tables = a->tables; p.state = a->state; p.first_page = a->first_page; p.cu = a->cu;
    p.k_plane = a->k_plane; p.vt_plane = a->vt_plane;
    p.n_seq = a->n_seq; p.max_pages = a->max_pages; p.n_pages = a->n_pages; p.nkv = a->nkv; p.kvT = a->kvT;
    const long pages = (long)a->kvT / CLEF_HIP_KV8_PAGE + a->n_seq;
    if (pages * a->nkv < 8L * kCus)
        hipLaunchKernelGGL(kv8::kv8_read_kernel<1>, dim3((unsigned)(pages * a->nkv)), dim3(256), 0, (hipStream_t)stream, p);
    else
        hipLaunchKernelGGL(kv8::kv8_read_kernel<2>, dim3((unsigned)(((long)a->kvT / (2 * CLEF_HIP_KV8_PAGE) + a->n_seq) * a->nkv)), dim3(512), 0,
                           (hipStream_t)stream, p);
    return launch_ok("kv8_read", err, errlen);
}

}  // extern "C"
