// Rotation of q and k heads by their positions, RMSNorm ahead of it where the model has one. Documented in
// include/clef_hip_attn.h.
//
// Pair j of a head turns by a = pos * freq_j: (x, y) -> m (x cos a - y sin a, y cos a + x sin a). Frequencies are
// f64 turns a position, so the whole turns drop out exactly and what is left, below one, goes to f32: at position
// 500,000 an FP32 product of position and frequency would be off by up to 0.03 radians.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bf16_ops.h"
#include "clef_hip_attn.h"

namespace clef_hip {
namespace rotary {

constexpr int kThreads = 256, kMaxHd = 256;

struct Group {
    const void *x;
    void *out;
    const float *norm;
    long x_row, x_head, out_row, out_head;
    int heads;
};
struct Params {
    Group q, k;
    const int32_t *pos;
    const double *freq;
    int T, hd, n_rot, half, axes, units;   // units: groups of heads that a wave takes together, of q and then of k
    int q_units;
    float eps, magnitude;
};

template <int TYPE>
__device__ __forceinline__ float get(const void *x, long at) {
    if constexpr (TYPE == CLEF_HIP_OUT_F32) return ((const float *)x)[at];
    else if constexpr (TYPE == CLEF_HIP_OUT_F16) return (float)((const _Float16 *)x)[at];
    else return bf2f(((const uint16_t *)x)[at]);
}
// V values at x + at, V * size a power of two of at most 16 bytes
template <int TYPE, int V>
__device__ __forceinline__ void load(const void *x, long at, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = get<TYPE>(x, at);
    } else if constexpr (TYPE == CLEF_HIP_OUT_F32) {
        typedef __attribute__((ext_vector_type(V))) float fv;
        const fv w = *(const fv *)((const float *)x + at);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = w[i];
    } else {
        typedef __attribute__((ext_vector_type(V))) uint16_t hv;
        const hv w = *(const hv *)((const uint16_t *)x + at);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = TYPE == CLEF_HIP_OUT_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]) : bf2f(w[i]);
    }
}
template <int TYPE, int V>
__device__ __forceinline__ void store(void *x, long at, const float (&v)[V]) {
    if constexpr (TYPE == CLEF_HIP_OUT_F32) {
        typedef __attribute__((ext_vector_type(V))) float fv;
        fv w;
#pragma unroll
        for (int i = 0; i < V; i++) w[i] = v[i];
        *(fv *)((float *)x + at) = w;
    } else {
        typedef __attribute__((ext_vector_type(V))) uint16_t hv;
        hv w;
#pragma unroll
        for (int i = 0; i < V; i++) w[i] = TYPE == CLEF_HIP_OUT_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[i]) : f2bf(v[i]);
        *(hv *)((uint16_t *)x + at) = w;
    }
}

// A lane holds two runs of V dims of a head: in the half layout the runs of V pairs' first and second parts, behind them
// (and in the interleaved layout, whose pairs lie in one run) neighbouring runs. L lanes, a power of two, hold a
// head, I pairs of runs each; a wave takes 64 / L heads of a token at a time, a workgroup TOK tokens.
template <int TYPE, int V, int L, int I, int TOK>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Params p) {
    __shared__ float2 table[TOK][kMaxHd / 2];
    const int half_rot = p.n_rot / 2, t0 = blockIdx.x * TOK;
    for (int i = threadIdx.x; i < TOK * half_rot; i += kThreads) {
        const int t = t0 + i / half_rot, j = i % half_rot;
        if (t < p.T) {
            const double a = (double)p.pos[(long)t * p.axes + j % p.axes] * p.freq[j];
            float s, c;
            sincospif(2.f * (float)(a - rint(a)), &s, &c);
            table[i / half_rot][j] = float2{c * p.magnitude, s * p.magnitude};
        }
    }
    __syncthreads();
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, at = lane % L;
    const int runs = half_rot / V;   // of the half layout: pairs of runs that turn
    for (int u = wave; u < TOK * p.units; u += kThreads / 64) {
        const int tok = u / p.units, unit = u % p.units, t = t0 + tok;
        const bool is_q = unit < p.q_units;
        const Group &gr = is_q ? p.q : p.k;
        const int h = (is_q ? unit : unit - p.q_units) * (64 / L) + lane / L;
        const bool there = t < p.T && h < gr.heads;
        const long xb = (long)t * gr.x_row + (long)h * gr.x_head, ob = (long)t * gr.out_row + (long)h * gr.out_head;
        float a[I][V], b[I][V];
        int da[I], db[I];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < I; i++) {
            const int pr = at + L * i;
            da[i] = p.half && pr < runs ? pr * V : 2 * pr * V;
            db[i] = p.half && pr < runs ? half_rot + pr * V : 2 * pr * V + V;
#pragma unroll
            for (int j = 0; j < V; j++) a[i][j] = b[i][j] = 0.f;
            if (there && da[i] < p.hd) load<TYPE, V>(gr.x, xb + da[i], a[i]);
            if (there && db[i] < p.hd) load<TYPE, V>(gr.x, xb + db[i], b[i]);
#pragma unroll
            for (int j = 0; j < V; j++) sum += a[i][j] * a[i][j] + b[i][j] * b[i][j];
        }
        if (gr.norm) {
#pragma unroll
            for (int d = 1; d < L; d *= 2) sum += __shfl_xor(sum, d);
            const float rs = 1.f / sqrtf(sum / p.hd + p.eps);
#pragma unroll
            for (int i = 0; i < I; i++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    if (da[i] < p.hd) a[i][j] *= rs * gr.norm[da[i] + j];
                    if (db[i] < p.hd) b[i][j] *= rs * gr.norm[db[i] + j];
                }
        }
        const bool in_place = gr.x == gr.out && !gr.norm;   // then what does not turn is there already
#pragma unroll
        for (int i = 0; i < I; i++) {
            if (!there) continue;
            if (p.half) {
                if (da[i] < half_rot) {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float2 cs = table[tok][da[i] + j];
                        const float x = a[i][j], y = b[i][j];
                        a[i][j] = x * cs.x - y * cs.y;
                        b[i][j] = y * cs.x + x * cs.y;
                    }
                } else if (in_place) continue;
            } else if constexpr (V == 1) {
                if (da[i] < p.n_rot) {
                    const float2 cs = table[tok][da[i] / 2];
                    const float x = a[i][0], y = b[i][0];
                    a[i][0] = x * cs.x - y * cs.y;
                    b[i][0] = y * cs.x + x * cs.y;
                } else if (in_place) continue;
            } else {
                if (in_place && da[i] >= p.n_rot) continue;
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    if (da[i] + j < p.n_rot) {
                        const float2 cs = table[tok][(da[i] + j) / 2];
                        const float x = a[i][j], y = a[i][j + 1];
                        a[i][j] = x * cs.x - y * cs.y;
                        a[i][j + 1] = y * cs.x + x * cs.y;
                    }
                    if (db[i] + j < p.n_rot) {
                        const float2 cs = table[tok][(db[i] + j) / 2];
                        const float x = b[i][j], y = b[i][j + 1];
                        b[i][j] = x * cs.x - y * cs.y;
                        b[i][j + 1] = y * cs.x + x * cs.y;
                    }
                }
            }
            if (da[i] < p.hd) store<TYPE, V>(gr.out, ob + da[i], a[i]);
            if (db[i] < p.hd) store<TYPE, V>(gr.out, ob + db[i], b[i]);
        }
    }
}

}  // namespace rotary
}  // namespace clef_hip
