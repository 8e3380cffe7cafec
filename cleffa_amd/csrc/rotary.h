// Rotation of q and k heads by their positions, RMSNorm ahead of it where the model has one. Documented in
// include/clef_hip_attn.h.
//
// Pair j of a head turns by a = pos * freq_j: (x, y) -> m (x cos a - y sin a, y cos a + x sin a). Frequencies are
// f64 turns a position, so the whole turns drop out exactly and what is left, below one, goes to f32: at position
// 500,000 an FP32 product of position and frequency would be off by up to 0.03 radians.
//
// Bound by memory: 4,096 tokens with 36 f32 heads of 128 are 151 MB in 24 us (32 with stores through the caches), with 28 bf16 heads of 256,
// norms and 64 of the dims turned 117 MB in 21 (27); 64 tokens of those by the latency of the loads, the angles and the launch, 4.2.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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
    bool past;                // of out: store_past
};
struct Params {
    Group q, k;
    const int32_t *pos;
    const double *freq;
    int T, hd, n_rot, half, axes, units;   // units: groups of heads that a wave takes together, of q and then of k
    int q_units;
    float eps, magnitude;
};

// a or b, by value: c ? p.a : p.b is a choice between addresses, and would put the argument block on the stack
template <typename T>
__device__ __forceinline__ T pick(bool c, T a, T b) { return c ? a : b; }

// V values of a head as they lie in memory, V * size a power of two of at most 16 bytes
template <int TYPE, int V>
struct Run {
    typedef __attribute__((ext_vector_type(V))) float f32s;
    typedef __attribute__((ext_vector_type(V))) uint16_t u16s;
    using Raw = typename std::conditional<TYPE == CLEF_HIP_OUT_F32, f32s, u16s>::type;
    using Elem = typename std::conditional<TYPE == CLEF_HIP_OUT_F32, float, uint16_t>::type;
    static __device__ __forceinline__ Raw load(const void *x, long at) { return *(const Raw *)((const Elem *)x + at); }
    static __device__ __forceinline__ float value(const Raw &r, int i) {
        const Elem e = r[i];
        if constexpr (TYPE == CLEF_HIP_OUT_F32) return e;
        else if constexpr (TYPE == CLEF_HIP_OUT_F16) return (float)__builtin_bit_cast(_Float16, e);
        else return bf2f(e);
    }
    template <typename PAST>
    static __device__ __forceinline__ void store(PAST past, void *x, long at, const float (&v)[V]) {
        Raw r;
#pragma unroll
        for (int i = 0; i < V; i++) {
            if constexpr (TYPE == CLEF_HIP_OUT_F32) r[i] = v[i];
            else if constexpr (TYPE == CLEF_HIP_OUT_F16) r[i] = __builtin_bit_cast(uint16_t, (_Float16)v[i]);
            else r[i] = f2bf(v[i]);
        }
        store_past(past, (Raw *)((Elem *)x + at), r);
    }
};

// A lane holds two runs of V dims of a head: in the half layout the first and the second dims of V pairs, else (dims that do not turn, and
// all of the interleaved layout, whose pairs lie in one run) runs half of what is left apart, so that neighbouring lanes read
// neighbouring runs. L lanes, a power of two, hold a head, I pairs of runs each; a wave takes 64 / L heads of a token at a time.
// The lane's dims are the same for every head: norm weights are loaded once, cosines and sines once a token.
template <int L>
__device__ __forceinline__ float sum_of(float x) {   // over L lanes, to each of them
    const auto from = [](float v, auto CTRL) {
        return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), decltype(CTRL)::value, 0xf, 0xf, true));
    };
    x += from(x, std::integral_constant<int, 0xb1>{});                          // lane ^ 1
    x += from(x, std::integral_constant<int, 0x4e>{});                          // lane ^ 2
    if constexpr (L >= 8) x += from(x, std::integral_constant<int, 0x141>{});   // 7 - lane of eight: the other four's sum
    if constexpr (L >= 16) x += from(x, std::integral_constant<int, 0x140>{});  // 15 - lane of sixteen
#pragma unroll
    for (int d = 16; d < L; d *= 2) x += __shfl_xor(x, d);
    return x;
}

// OUT: of the outputs, TYPE, or bf16 from f32 heads: those are then rounded here alone, where rows rounded to bf16 ahead of the call make q and k
// twice rounded (errors 1.7e-3 and 2.3e-3, relative, rms: the square root of two).
template <int TYPE, int OUT, int V, int L, int I, int TOK, bool HALF>
__global__ __launch_bounds__(kThreads, 4) void rotary_kernel(Params p) {
    using R = Run<TYPE, V>;
    using O = Run<OUT, V>;
    constexpr int PER_TOK = kThreads / 64 / TOK, U = TOK == 1 ? 2 : 4;   // waves of a token; groups of heads that are loaded together
    __shared__ __attribute__((aligned(16))) float2 table[TOK][kMaxHd / 2];
    const int half_rot = p.n_rot / 2, t0 = blockIdx.x * TOK;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, at = lane % L;
    const int tok = wave / PER_TOK, t = t0 + tok;
    int da[I], db[I];
    const int pairs = HALF ? half_rot / V : 0, rest = p.hd / V - 2 * pairs, apart = (rest + 1) / 2;
#pragma unroll
    for (int i = 0; i < I; i++) {
        const int pr = at + L * i, q = pr - pairs;
        da[i] = pr < pairs ? pr * V : (2 * pairs + q) * V;
        db[i] = pr < pairs ? half_rot + pr * V : q + apart < rest ? (2 * pairs + q + apart) * V : p.hd;
        if (q >= apart) da[i] = db[i] = p.hd;
        if (V == 1 && !HALF) {     // a pair is two runs
            da[i] = min(2 * pr, p.hd);
            db[i] = min(2 * pr + 1, p.hd);
        }
    }
    // the unit's group of heads, as they lie in memory: the first U go out ahead of the angles
    struct Raw {
        typename R::Raw a[I], b[I];
    };
    auto load = [&](int unit) __attribute__((always_inline)) {
        const bool is_q = unit < p.q_units;
        const int h = (is_q ? unit : unit - p.q_units) * (64 / L) + lane / L;
        const void *x = pick(is_q, p.q.x, p.k.x);
        const long xb = (long)t * pick(is_q, p.q.x_row, p.k.x_row) + (long)h * pick(is_q, p.q.x_head, p.k.x_head);
        const bool there = t < p.T && unit < p.units && h < pick(is_q, p.q.heads, p.k.heads);
        Raw r;
#pragma unroll
        for (int i = 0; i < I; i++) {
            typename R::Raw a{}, b{};
            if (there && da[i] < p.hd) a = R::load(x, xb + da[i]);
            if (there && db[i] < p.hd) b = R::load(x, xb + db[i]);
            r.a[i] = a;
            r.b[i] = b;
        }
        return r;
    };
    Raw raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = load(wave % PER_TOK + u * PER_TOK);
    typedef __attribute__((ext_vector_type(V), aligned(4))) float Weights;   // loaded by the run: one by one they took 3.3 us of a small call's 7.3
    auto weights = [&](const float *w, int d) __attribute__((always_inline)) {
        Weights r = (Weights)1.f;
        if (w && d < p.hd) r = *(const Weights *)(w + d);
        return r;
    };
    Weights wq[2][I], wk[2][I];
#pragma unroll
    for (int i = 0; i < I; i++) {
        wq[0][i] = weights(p.q.norm, da[i]);
        wq[1][i] = weights(p.q.norm, db[i]);
        wk[0][i] = weights(p.k.norm, da[i]);
        wk[1][i] = weights(p.k.norm, db[i]);
    }
    for (int i = threadIdx.x; i < TOK * half_rot; i += kThreads) {
        const int tt = t0 + i / half_rot, j = i % half_rot;
        if (tt < p.T) {
            const double a = (double)p.pos[(long)tt * p.axes + j % p.axes] * p.freq[j];
            float s, c;
            sincospif(2.f * (float)(a - rint(a)), &s, &c);
            table[i / half_rot][j] = float2{c * p.magnitude, s * p.magnitude};
        }
    }
    __syncthreads();
    if (t >= p.T) return;
    // of the half layout V pairs' cosines and sines; of the interleaved one V / 2 of run a, V / 2 of run b
    float2 cs[I][V];
#pragma unroll
    for (int i = 0; i < I; i++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            int pair;
            if constexpr (HALF) pair = da[i] < half_rot ? da[i] + j : -1;
            else if constexpr (V == 1) pair = da[i] < p.n_rot ? da[i] / 2 : -1;
            else {
                const int d = j < V / 2 ? da[i] + 2 * j : db[i] + 2 * j - V;
                pair = d < p.n_rot ? d / 2 : -1;
            }
            cs[i][j] = pair >= 0 ? table[tok][pair] : float2{1.f, 0.f};
        }
    const float inv_hd = 1.f / p.hd;
    auto turn = [&](const Raw &r, int unit) __attribute__((always_inline)) {
        const bool is_q = unit < p.q_units;
        const int h = (is_q ? unit : unit - p.q_units) * (64 / L) + lane / L;
        void *out = pick(is_q, p.q.out, p.k.out);
        const long ob = (long)t * pick(is_q, p.q.out_row, p.k.out_row) + (long)h * pick(is_q, p.q.out_head, p.k.out_head);
        const bool there = h < pick(is_q, p.q.heads, p.k.heads), norm = pick(is_q, p.q.norm != nullptr, p.k.norm != nullptr);
        const bool past = pick(is_q, p.q.past, p.k.past);
        const bool in_place = !norm && out == pick(is_q, p.q.x, p.k.x);   // then what does not turn is there already
        float a[I][V], b[I][V], sum = 0.f;
#pragma unroll
        for (int i = 0; i < I; i++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                a[i][j] = R::value(r.a[i], j);
                b[i][j] = R::value(r.b[i], j);
                sum += a[i][j] * a[i][j] + b[i][j] * b[i][j];
            }
        if (norm) {
            const float rs = rsqrtf(sum_of<L>(sum) * inv_hd + p.eps);
#pragma unroll
            for (int i = 0; i < I; i++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    a[i][j] *= rs * pick<float>(is_q, wq[0][i][j], wk[0][i][j]);
                    b[i][j] *= rs * pick<float>(is_q, wq[1][i][j], wk[1][i][j]);
                }
        }
        if (!there) return;
#pragma unroll
        for (int i = 0; i < I; i++) {
            if constexpr (V == 1 || HALF) {
                if (da[i] < (HALF ? half_rot : p.n_rot)) {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float x = a[i][j], y = b[i][j];
                        a[i][j] = x * cs[i][j].x - y * cs[i][j].y;
                        b[i][j] = y * cs[i][j].x + x * cs[i][j].y;
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    const float2 ca = cs[i][j / 2], cb = cs[i][V / 2 + j / 2];
                    if (da[i] + j < p.n_rot) {
                        const float x = a[i][j], y = a[i][j + 1];
                        a[i][j] = x * ca.x - y * ca.y;
                        a[i][j + 1] = y * ca.x + x * ca.y;
                    }
                    if (db[i] + j < p.n_rot) {
                        const float x = b[i][j], y = b[i][j + 1];
                        b[i][j] = x * cb.x - y * cb.y;
                        b[i][j + 1] = y * cb.x + x * cb.y;
                    }
                }
            }
        }
        with_past(past, [&](auto PAST) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < I; i++) {
                if (da[i] < p.hd && !(in_place && da[i] >= p.n_rot)) O::store(PAST, out, ob + da[i], a[i]);
                if (db[i] < p.hd && !(in_place && db[i] >= p.n_rot)) O::store(PAST, out, ob + db[i], b[i]);
            }
        });
    };
    for (int u0 = wave % PER_TOK; u0 < p.units; u0 += U * PER_TOK) {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (u0 + u * PER_TOK < p.units) turn(raw[u], u0 + u * PER_TOK);
        if (u0 + U * PER_TOK < p.units) {
#pragma unroll
            for (int u = 0; u < U; u++) raw[u] = load(u0 + (U + u) * PER_TOK);
        }
    }
}

}  // namespace rotary
}  // namespace clef_hip
