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

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 16-bit values whose type is known at run time (uniform).
__device__ inline float widen16(uint32_t bits, int type) {
    return type == T_F16 ? float(__builtin_bit_cast(f16, uint16_t(bits))) : __uint_as_float(bits << 16);
}
// Eight of them from value i on; aligned: i lies on 16 bytes (uniform).
__device__ inline u32x4 load16x8(const void *p, int64_t i, bool aligned) {
    const uint16_t *x = static_cast<const uint16_t *>(p) + i;
    if (aligned) return *reinterpret_cast<const u32x4 *>(x);
    u32x4 r;
    for (int k = 0; k < 4; k++) r[k] = uint32_t(x[2 * k]) | uint32_t(x[2 * k + 1]) << 16;
    return r;
}
__device__ inline void store16(void *p, int type, int64_t i, float v) {
    if (type == T_F16) static_cast<f16 *>(p)[i] = f16(v);
    else static_cast<bf16 *>(p)[i] = bf16(v);
}

// D[16][16] += A[16][32] B[32][16]: lane l holds A's row and B's column l % 16, values 8 (l / 16) on
// of the 32; of D, column l % 16 and rows 4 (l / 16) on.
__device__ inline f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// D[32][32] += A[32][16] B[16][32]: lane l holds A's row and B's column l % 32, values 8 (l / 32) on of
// the 16; of D, column l % 32 and rows 8 i + 4 (l / 32) + 0 .. 3 in element 4 i on.
__device__ inline f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// Transposing reads of LDS. 16 lanes name 4 rows of 16 values of 16 bits (lanes 4 r to 4 r + 3 the
// four quarters of row r), or 8 rows of 16 bytes (lanes 2 r, 2 r + 1 the halves); each gets its column.
__device__ inline u32x2 lds_read_tr16(const char *p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)p));
}
__device__ inline u32x2 lds_read_tr8(const char *p) {
    typedef int i2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i2 *)p));
}

// Eight codes of an 8-bit cache as float16, exactly.
template <class C> __device__ inline f16x8 widen8(uint32_t a, uint32_t b) {
    f16x2 x[4];
    if constexpr (std::is_same_v<C, int8_t>) {
        // 0x6400 | u is 1024 + u.
        a ^= 0x80808080u, b ^= 0x80808080u;
        const f16x2 off{f16(1152.f), f16(1152.f)};
        x[0] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - off;
        x[1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - off;
        x[2] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - off;
        x[3] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - off;
    } else {
        x[0] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false));
        x[1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true));
        x[2] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false));
        x[3] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true));
    }
    return f16x8{x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
}

// A softmax's reference may lie up to 2^8 under the true maximum before the sums are scaled again.
// Weights in float16 are held as 2^6 times their value relative to it: at most 2^14, within the type,
// and its last step 2^-24 is 2^-30 of the reference. bfloat16 has the range to hold them under one,
// which leaves the sums that of their values. The factor is common to the sums and leaves with them.
constexpr float kSlack = 8.f;
template <class M> constexpr float lift = std::is_same_v<M, f16> ? 6.f : -kSlack;

// 2^x; results under the normal range are zero.
__device__ inline float exp2_f32(float x) { return __builtin_amdgcn_exp2f(x); }
// A score through the cap: most tanh(y) = most (1 - 2 / (e^2y + 1)), off by 2^-23 of the cap; and with the small
// ones off by their own size (text_rules.h).
__device__ inline float large_capped(const Cap &c, float s) {
    return c.most * (1.f - 2.f * __builtin_amdgcn_rcpf(exp2_f32(s * c.inv * 2.8853900817779268f) + 1.f));
}
__device__ inline float capped(const Cap &c, float s) { return fabsf(s) <= c.small ? small_capped(c, s) : large_capped(c, s); }

// The code of a value already divided by its vector's scale (rounded to nearest, ties to even).
template <class C> __device__ inline C code_of(float v) {
    if constexpr (std::is_same_v<C, int8_t>) return int8_t(rintf(v));
    else if constexpr (std::is_same_v<C, e4m3>) return e4m3{uint8_t(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 255)};
    else return C(v);
}
template <class C> constexpr float code_max = std::is_same_v<C, int8_t> ? 127.f : 448.f;
// Vectors whose largest value is under this are held as zeros: 448 over it still is a float.
constexpr float kTinyMax = 1e-30f;

// Over a wavefront, without LDS: each row of 16 lanes, then the rows in order; the last lane has the
// result.
template <int Ctrl, int Rows, class V> __device__ inline V dpp(V old, V v) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v), Ctrl, Rows, 15, false));
}
template <class V, class Op> __device__ inline V wave_reduce(V v, V none, Op &&op) {
    v = op(v, dpp<0x111, 15>(none, v));  // from 1, 2, 4, 8 lanes before
    v = op(v, dpp<0x112, 15>(none, v));
    v = op(v, dpp<0x114, 15>(none, v));
    v = op(v, dpp<0x118, 15>(none, v));
    v = op(v, dpp<0x142, 10>(none, v));  // a row's last lane to the next row (rows 1 and 3)
    v = op(v, dpp<0x143, 12>(none, v));  // lane 31 to rows 2 and 3
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ inline float wave_max(float v) {
    return wave_reduce(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline float wave_sum(float v) {
    return wave_reduce(v, 0.f, [](float a, float b) { return a + b; });
}
// Over groups of W lanes, all of which get the result.
template <int W, class V, class Op> __device__ inline V group_reduce(V v, Op &&op) {
    auto from = [](V x, auto ctrl) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        return __builtin_bit_cast(V, uint32_t(__builtin_amdgcn_update_dpp(u, u, decltype(ctrl)::value, 15, 15, false)));
    };
    v = op(v, from(v, std::integral_constant<int, 0xb1>{}));                          // neighbours
    v = op(v, from(v, std::integral_constant<int, 0x4e>{}));                          // pairs of four
    if constexpr (W > 4) v = op(v, from(v, std::integral_constant<int, 0x141>{}));    // eight, mirrored
    if constexpr (W > 8) v = op(v, from(v, std::integral_constant<int, 0x140>{}));    // sixteen, mirrored
    if constexpr (W > 16) v = op(v, V(__shfl_xor(v, 16)));
    return v;
}
__device__ inline int wave_max_i(int v) {
    return wave_reduce(v, int(0x80000000), [](int a, int b) { return max(a, b); });
}
__device__ inline int wave_min_i(int v) { return -1 - wave_max_i(-1 - v); }

// One query's attention over keys [lo, hi) by one wavefront, by the formula: the scores' maximum
// first, then exp(s - max) and the value sums, all in float32. q: the query's dim values in LDS,
// scaled; kv.k(j, c) and kv.v(j, c): value c of key and value vector j. Scores of minus infinity
// weigh nothing, a query that sees nothing gives zeros. done(c, value) gets each of the outputs.
template <class KV, class Done>
__device__ inline void attend_row(const KV &kv, const float *q, int dim, int lo, int hi, int pos, float cap, float slope, Done &&done) {
    const int lane = threadIdx.x & 63;
    const Cap most = cap_of(cap, 1.f);
    auto score = [&](int j) {
        float s = 0.f;
        for (int c = 0; c < dim; c++) s = __fmaf_rn(q[c], kv.k(j, c), s);
        if (cap > 0.f) s = capped(most, s);
        return s - slope * float(pos > j ? pos - j : j - pos);
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
