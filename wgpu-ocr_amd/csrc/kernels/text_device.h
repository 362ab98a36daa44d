// Device helpers that the text decoder's kernels share: element types, wavefront sums, scores.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "../text.h"

namespace ocr {

typedef __bf16 bf16;
typedef _Float16 f16;

// A launch's element type as a template argument: with_type(t, [&](auto z) { using T = decltype(z); ... }).
template <class F> void with_type16(int t, F &&f) {
    if (t == T_F16) f(f16{});
    else f(bf16{});
}
template <class F> void with_type(int t, F &&f) {
    if (t == T_F32) f(float{});
    else with_type16(t, f);
}
// A cache's types: codes of 8 bits, each type of its own.
struct e4m3 {
    uint8_t bits;
};
template <class F> void with_cache(int t, F &&f) {
    if (t == T_I8) f(int8_t{});
    else if (t == T_E4M3) f(e4m3{});
    else with_type16(t, f);
}
template <class C> constexpr bool scaled = sizeof(C) == 1;

__device__ inline float to_f32(float v) { return v; }
__device__ inline float to_f32(f16 v) { return float(v); }
__device__ inline float to_f32(bf16 v) { return float(v); }
__device__ inline float to_f32(int8_t v) { return float(v); }
__device__ inline float to_f32(e4m3 v) { return __builtin_amdgcn_cvt_f32_fp8(int(v.bits), 0); }

// The code of a value already divided by its vector's scale (rounded to nearest, ties to even).
template <class C> __device__ inline C code_of(float v) {
    if constexpr (std::is_same_v<C, int8_t>) return int8_t(rintf(v));
    else if constexpr (std::is_same_v<C, e4m3>) return e4m3{uint8_t(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 255)};
    else return C(v);
}
template <class C> constexpr float code_max = std::is_same_v<C, int8_t> ? 127.f : 448.f;
// Vectors whose largest value is under this are held as zeros: 448 over it still is a float.
constexpr float kTinyMax = 1e-30f;

__device__ inline float wave_max(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ inline float wave_sum(float v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// A scaled score through the cap and the distance bias.
__device__ inline float score_of(float s, float cap, float slope, int distance) {
    if (cap > 0.f) s = cap * tanhf(s / cap);
    return s - slope * float(distance);
}

// One query's attention over keys [lo, hi) by one wavefront, by the formula: the scores' maximum
// first, then exp(s - max) and the value sums, all in float32. q: the query's dim values in LDS,
// scaled; kv.k(j, c) and kv.v(j, c): value c of key and value vector j. Scores of minus infinity
// weigh nothing, a query that sees nothing gives zeros. done(c, value) gets each of the outputs.
template <class KV, class Done>
__device__ inline void attend_row(const KV &kv, const float *q, int dim, int lo, int hi, int pos, float cap, float slope, Done &&done) {
    const int lane = threadIdx.x & 63;
    auto score = [&](int j) {
        float s = 0.f;
        for (int c = 0; c < dim; c++) s = __fmaf_rn(q[c], kv.k(j, c), s);
        return score_of(s, cap, slope, pos > j ? pos - j : j - pos);
    };
    float m = -INFINITY;
    for (int j = lo + lane; j < hi; j += 64) m = fmaxf(m, score(j));
    m = wave_max(m);
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int j = j0 + lane;
        float p = 0.f;
        if (j < hi) {
            const float s = score(j);
            p = s == -INFINITY ? 0.f : expf(s - m);
        }
        l += p;
        const int cnt = min(64, hi - j0);
        for (int t = 0; t < cnt; t++) {
            const float w = __shfl(p, t);
            if (w == 0.f) continue;
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (lane + 64 * u < dim) o[u] = __fmaf_rn(w, kv.v(j0 + t, lane + 64 * u), o[u]);
        }
    }
    l = wave_sum(l);
    for (int u = 0; u < 4; u++)
        if (lane + 64 * u < dim) done(lane + 64 * u, l == 0.f ? 0.f : o[u] / l);
}

}  // namespace ocr
