// Attention of single tokens over the paged cache.
//
// Every cached vector is needed once for each of the group's query heads, so a step is bound by the
// cache's bytes: a workgroup reads one key head's vectors of a part of a sequence once for all of
// its (up to 16) query heads, and the parts of a sequence are joined afterwards. Products run on the
// matrix cores, 16 queries wide, with keys as rows: S^T = K Q^T, O^T = V^T P^T. A lane of the first's
// result holds four keys of one query, which is what the second takes from it as it is.
// 4 sequences of 131 072 and less over 8 heads of 128 in e4m3 (981 MB): 178 us with the join, 5.5
// TB/s, faster than a large copy. 144 of up to 700 in int8 (71 MB): 25 us; of those 4 pass before the
// first keys are asked for, and the longest sequences end well after the median. Registers for two
// wavefronts a SIMD: for three some are spilled (186 and 27 us, where two took 178 and 24).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

// A head's vectors in a sequence's pages; a position whose page there is not holds zeros.
template <class C> struct PagedKv {
    KvCache c;
    const int32_t *row;
    uint32_t width, head;
    __device__ int64_t slot(int j) const {
        const int32_t p = page_of(row, width, c.page, c.pages, j);
        return p < 0 ? -1 : slot_of(p, c.heads, c.page, head, uint32_t(j) % c.page);
    }
    __device__ float k(int j, int i) const {
        const int64_t s = slot(j);
        return s < 0 ? 0.f : to_f32(static_cast<const C *>(c.k)[s * c.dim + i]) * (scaled<C> ? c.k_scale[s] : 1.f);
    }
    __device__ float v(int j, int i) const {
        const int64_t s = slot(j);
        return s < 0 ? 0.f : to_f32(static_cast<const C *>(c.v)[s * c.dim + i]) * (scaled<C> ? c.v_scale[s] : 1.f);
    }
};

// Vectors that are no whole 16-byte pieces: one wavefront a (sequence, head), by the formula. 144 sequences of 700,
// 4 heads of 72 in int8: 1.3 ms, of 80 by the tiles 28 us.
template <class T, class C> __global__ __launch_bounds__(64) void decode_row_kernel(DecodeArgs a) {
    __shared__ float s_q[256];
    const int64_t r = blockIdx.x;
    const int h = blockIdx.y, dim = a.kv.dim, hk = h / int(a.q_heads / a.kv.heads);
    const T *q = static_cast<const T *>(a.q) + r * a.q_stride + int64_t(h) * dim;
    for (int c = threadIdx.x; c < dim; c += 64) s_q[c] = to_f32(q[c]) * a.scale;
    __syncthreads();
    const int len = clamp_len(a.lens[r], a.table.width, a.kv.page);
    const PagedKv<C> kv{a.kv, a.table.p + r * a.table.width, a.table.width, uint32_t(hk)};
    T *out = static_cast<T *>(a.out) + r * a.out_stride + int64_t(h) * dim;
    attend_row(kv, s_q, dim, 0, len, len - 1, a.cap, a.slopes ? a.slopes[h] : 0.f, [&](int c, float o) { out[c] = T(o); });
}

// What a launch's workgroups share. shift: a page's positions as a power of two, -1 if they are none.
struct DecodePlan {
    uint32_t parts;
    int group, blocks, shift;  // query heads a key head, blocks of 16 of them
    bool q_pieces;
    Cap cap;  // in units of log2
};

// Parts of a sequence joined: part [row][head][parts] holds dim normalised values, then log2 of the
// sum of weights.
constexpr int kPartTail = 4;  // keeps the rows' 16-byte alignment

// T: the queries' type, C: the cache's; products of 8-bit caches in float16, which holds their codes
// exactly.
template <class T, class C, int DP> __global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void decode_kernel(DecodeArgs a, DecodePlan plan, float *part) {
    using M = std::conditional_t<scaled<C>, f16, C>;
    typedef M mvec __attribute__((ext_vector_type(8)));
    constexpr int NU = DP * int(sizeof(C)) / 64;    // 16-byte pieces of a vector that a lane holds
    constexpr int NS = DP / 32;                     // steps of 32 values of the first product
    constexpr int NB = DP / 16;                     // blocks of 16 values of the second
    constexpr int PITCH = DP * int(sizeof(C)) + 16; // a value vector's bytes in LDS: rows start four banks apart
    constexpr int CH = 1024;                        // positions looked up at a time
    constexpr int JOIN = 2 * 16 * (DP + 4) * 4;     // the waves' sums on their way to each other
    constexpr int STAGE = 4 * 32 * PITCH;
    __shared__ __align__(16) char s_mem[STAGE > JOIN ? STAGE : JOIN];
    __shared__ int64_t s_at[CH];  // a position's vector in the pool, negative: none
    __shared__ __align__(16) float s_scale[4][2][32];  // the waves' key and value scales of a tile
    __shared__ float s_ml[2][2][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g4 = lane >> 4;
    const int64_t r = blockIdx.x;
    const uint32_t parts = plan.parts;
    const int hk = plan.blocks == 1 ? blockIdx.y : blockIdx.y / plan.blocks, q0 = (int(blockIdx.y) - hk * plan.blocks) * 16, dim = a.kv.dim;
    const int group = plan.group;
    const int h = hk * group + q0 + n;  // the lane's query head
    const bool real = q0 + n < group;
    // The lane's query, in the order of its key pieces.
    u32x4 raw[NS];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        const int c = sizeof(C) == 1 ? 64 * (s >> 1) + 16 * g4 + 8 * (s & 1) : 32 * s + 8 * g4;
        raw[s] = u32x4{0, 0, 0, 0};
        if (real && c < dim) raw[s] = load16x8(a.q, r * a.q_stride + int64_t(h) * dim + c, plan.q_pieces);
    }
    const int len = clamp_len(a.lens[r], a.table.width, a.kv.page);
    const Parts ps = parts_of(len, parts);
    const int lo = int(blockIdx.z) * ps.each, hi = min(len, lo + ps.each);
    if (parts > 1 && lo >= hi) return;

    const int pieces = dim * int(sizeof(C)) / 16;
    const uint32_t vec_bytes = dim * int(sizeof(C));
    uint32_t off[NU];
#pragma unroll
    for (int u = 0; u < NU; u++) off[u] = 16 * min(4 * u + g4, pieces - 1);
    char *const s_v = s_mem + wave * 32 * PITCH;
    const float slope = a.slopes && real ? a.slopes[h] * 1.4426950408889634f : 0.f;
    // bfloat16 queries over an 8-bit cache are float16 in the products, each over a power of two of its own (below),
    // which is in its lanes' score_scale.
    constexpr bool own_scale = scaled<C> && std::is_same_v<T, bf16>;
    float score_scale = a.scale * 1.4426950408889634f;
    mvec qf[NS];
    f32x4 o[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    float vtop = 0.f, vinv = 0.f;  // a power of two over all value scales so far, and one over it

    for (int c0 = lo; c0 < hi; c0 += CH) {
        if (c0 != lo) __syncthreads();
        const int cn = min(CH, hi - c0);
        for (int i = tid; i < ((cn + 31) & ~31); i += 256) {
            int64_t at = -1;
            if (i < cn) {
                const uint32_t pos = c0 + i, entry = plan.shift >= 0 ? pos >> plan.shift : pos / a.kv.page;
                const int32_t p = page_at(a.table.p + r * a.table.width, a.table.width, a.kv.pages, entry);
                if (p >= 0) at = slot_of(p, a.kv.heads, a.kv.page, hk, pos - entry * a.kv.page);
            }
            s_at[i] = at;
        }
        __syncthreads();
        // A tile's keys, values and scales; where there is no vector or no such piece of it, the
        // pool's first, zeroed when the tile is used. (Past the last tile too: loads under a condition
        // would be waited for where the paths meet.)
        u32x4 kr[2][NU], vr[2][NU];
        float scale_r = 0.f;
        bool none[2];
        auto load = [&](int t0) {
            int64_t at[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                at[t] = s_at[min(t0, CH - 32) + 16 * t + n];
                none[t] = t0 >= cn || at[t] < 0;
                at[t] = none[t] ? 0 : at[t];
            }
            if constexpr (scaled<C>) {
                const int64_t vec = (g4 & 1) ? at[1] : at[0];
                scale_r = (g4 < 2 ? a.kv.k_scale : a.kv.v_scale)[vec];
            }
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int u = 0; u < NU; u++)
                    kr[t][u] = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.kv.k) + at[t] * vec_bytes + off[u]);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int u = 0; u < NU; u++)
                    vr[t][u] = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.kv.v) + at[t] * vec_bytes + off[u]);
        };
        load(wave * 32);
        if (c0 == lo) {
            // The exponent of the query's largest finite value: float16 holds the others to 2^-11 of themselves down
            // to 2^-14 of it, and to 2^-25 of it below.
            if constexpr (own_scale) {
                float top = 0.f;
#pragma unroll
                for (int s = 0; s < NS; s++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float x = fabsf(widen16(raw[s][i >> 1] >> (16 * (i & 1)), T_BF16));
                        top = fmaxf(top, x < INFINITY ? x : 0.f);
                    }
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const int e = top > 0.f ? max(-126, min(126, ilogbf(top))) : 0;
                const float down = ldexpf(1.f, -e);
                score_scale *= ldexpf(1.f, e);
#pragma unroll
                for (int s = 0; s < NS; s++)
#pragma unroll
                    for (int i = 0; i < 8; i++) qf[s][i] = M(widen16(raw[s][i >> 1] >> (16 * (i & 1)), T_BF16) * down);
            } else {
#pragma unroll
                for (int s = 0; s < NS; s++) qf[s] = __builtin_bit_cast(mvec, raw[s]);
            }
        }
        for (int t0 = wave * 32; t0 < cn; t0 += 128) {
            if (pieces < 4 * NU || __any(none[0] || none[1])) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int u = 0; u < NU; u++)
                        if (none[t] || 4 * u + g4 >= pieces) kr[t][u] = vr[t][u] = u32x4{0, 0, 0, 0};
                if (none[g4 & 1]) scale_r = 0.f;
            }
            // The tile's scales: the keys' with the scores' own where that is one for all, the values' over their power of two.
            bool spread = false;  // some value scale is under the span
            if constexpr (scaled<C>) {
                if (__any(g4 >= 2 && fabsf(scale_r) > vtop)) {
                    const float vmax = wave_max(g4 >= 2 ? fabsf(scale_r) : 0.f);
                    const float vn = over_pow2(vmax), f = vtop / vn;
#pragma unroll
                    for (int b = 0; b < NB; b++) o[b] *= f;
                    vtop = vn, vinv = 1.f / vn;
                }
                spread = __any(g4 >= 2 && fabsf(scale_r) < vtop * kScaleSpan && scale_r != 0.f);
                s_scale[wave][g4 >> 1][16 * (g4 & 1) + n] = scale_r * (g4 < 2 ? own_scale ? 1.f : score_scale : vinv);
            }
            f32x4 s[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < NS; st++) {
                    mvec kf;
                    if constexpr (scaled<C>) kf = widen8<C>(kr[t][st >> 1][2 * (st & 1)], kr[t][st >> 1][2 * (st & 1) + 1]);
                    else kf = __builtin_bit_cast(mvec, kr[t][st]);
                    s[t] = mfma16(kf, qf[st], s[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int u = 0; u < NU; u++)
                    *reinterpret_cast<u32x4 *>(s_v + (16 * t + n) * PITCH + 16 * (4 * u + g4)) = vr[t][u];
            load(t0 + 128);
            // Scores in units of log2.
            float sc[2][4];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                f32x4 ks{score_scale, score_scale, score_scale, score_scale};
                if constexpr (scaled<C>) ks = *reinterpret_cast<const f32x4 *>(&s_scale[wave][0][16 * t + 4 * g4]);
#pragma unroll
                for (int i = 0; i < 4; i++) sc[t][i] = (own_scale ? s[t][i] * score_scale : s[t][i]) * ks[i];
            }
            if (a.cap > 0.f) {
                float far = 0.f;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) far = fmaxf(far, fabsf(sc[t][i]));
                if (__any(far > plan.cap.small)) {
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sc[t][i] = capped(plan.cap, sc[t][i]);
                } else {
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sc[t][i] = small_capped(plan.cap, sc[t][i]);
                }
            }
            if (a.slopes) {
                const float d = float(len - 1 - c0 - t0 - 4 * g4);
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) sc[t][i] -= slope * (d - float(16 * t + i));
            }
            if (t0 + 32 > cn) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (t0 + 16 * t + 4 * g4 + i >= cn) sc[t][i] = -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, sc[t][i]);
            if (__any(top > m + kSlack)) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float mn = fmaxf(m, top), f = mn == -INFINITY ? 1.f : exp2_f32(m - mn);
                l *= f;
#pragma unroll
                for (int b = 0; b < NB; b++) o[b] *= f;
                m = mn;
            }
            const float ref = m == -INFINITY ? 0.f : m - lift<M>;
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                w[i] = exp2_f32(sc[i >> 2][i & 3] - ref);
                l += w[i];
            }
            auto value = [&](int b) {  // block b of the tile's values
                if constexpr (scaled<C>) {
                    const int row = (lane & 15) >> 1;
                    const u32x2 x = lds_read_tr8(s_v + (16 * (row >> 2) + 4 * g4 + (row & 3)) * PITCH + 16 * b + 8 * (lane & 1));
                    return widen8<C>(x[0], x[1]);
                } else {
                    const int row = 4 * g4 + ((lane & 15) >> 2);
                    const u32x2 x = lds_read_tr16(s_v + row * PITCH + 32 * b + 8 * (lane & 3));
                    const u32x2 y = lds_read_tr16(s_v + (16 + row) * PITCH + 32 * b + 8 * (lane & 3));
                    return __builtin_bit_cast(mvec, u32x4{x[0], x[1], y[0], y[1]});
                }
            };
            f32x4 vs[2];
            if constexpr (scaled<C>) {
#pragma unroll
                for (int t = 0; t < 2; t++) vs[t] = *reinterpret_cast<const f32x4 *>(&s_scale[wave][1][16 * t + 4 * g4]);
            }
            mvec p;
            if (!scaled<C> || !spread) {
#pragma unroll
                for (int i = 0; i < 8; i++) p[i] = M(scaled<C> ? w[i] * vs[i >> 2][i & 3] : w[i]);
#pragma unroll
                for (int b = 0; b < NB; b++) o[b] = mfma16(value(b), p, o[b]);
            } else {
                // A span at a time (kScaleSpan). 144 sequences whose first vectors have 2^10 times the others' scale, so that a
                // quarter of the tiles come here: 31 us instead of 25.
                float left = NAN;  // scales from here on are done; those that are no numbers are in every span
                for (;;) {
                    float largest = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float x = fabsf(vs[i >> 2][i & 3]);
                        largest = fmaxf(largest, x >= left ? 0.f : x);
                    }
                    largest = wave_max(largest);
                    if (!more_spans(largest)) break;
                    const ScaleSpan span = span_of(largest);
                    const float up = 1.f / span.over;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float x = vs[i >> 2][i & 3];
                        p[i] = M(fabsf(x) >= left || fabsf(x) < span.low ? 0.f : w[i] * (x * up));
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) o[b] += span.over * mfma16(value(b), p, f32x4{0.f, 0.f, 0.f, 0.f});
                    left = span.low;
                }
            }
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    // The weights' most taken out, and the values' scales put in.
    constexpr float most = lift<M> > 0.f ? 0x1p-14f : 1.f;
    const float back = scaled<C> ? vtop * most : most;
#pragma unroll
    for (int b = 0; b < NB; b++) o[b] *= back;
    l *= most;
    // Waves 2 and 3 hand their sums to 0 and 1, then 1 to 0.
    float *const s_o = reinterpret_cast<float *>(s_mem);
#pragma unroll
    for (int step = 2; step >= 1; step >>= 1) {
        __syncthreads();
        if (wave >= step && wave < 2 * step) {
            float *dst = s_o + ((wave - step) * 16 + n) * (DP + 4);
#pragma unroll
            for (int b = 0; b < NB; b++) *reinterpret_cast<f32x4 *>(dst + 16 * b + 4 * g4) = o[b];
            if (g4 == 0) s_ml[wave - step][0][n] = m, s_ml[wave - step][1][n] = l;
        }
        __syncthreads();
        if (wave < step) {
            const float *src = s_o + (wave * 16 + n) * (DP + 4);
            const float m2 = s_ml[wave][0][n], l2 = s_ml[wave][1][n], mn = fmaxf(m, m2);
            const float f = mn == -INFINITY ? 0.f : exp2_f32(m - mn), f2 = mn == -INFINITY ? 0.f : exp2_f32(m2 - mn);
            l = l * f + l2 * f2;
#pragma unroll
            for (int b = 0; b < NB; b++) o[b] = o[b] * f + *reinterpret_cast<const f32x4 *>(src + 16 * b + 4 * g4) * f2;
            m = mn;
        }
    }
    if (wave != 0 || !real) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (part) {
        float *dst = part + ((r * a.q_heads + h) * parts + blockIdx.z) * (dim + kPartTail);
#pragma unroll
        for (int b = 0; b < NB; b++)
            if (16 * b + 4 * g4 < dim) *reinterpret_cast<f32x4 *>(dst + 16 * b + 4 * g4) = o[b] * inv;
        if (g4 == 0) dst[dim] = l == 0.f ? -INFINITY : m + log2f(l);
    } else {
        const int64_t at = r * a.out_stride + int64_t(h) * dim;
#pragma unroll
        for (int b = 0; b < NB; b++)
            for (int i = 0; i < 4; i++)
                if (16 * b + 4 * g4 < dim) store16(a.out, a.type, at + 16 * b + 4 * g4 + i, o[b][i] * inv);
    }
}

// One workgroup a (sequence, head): four values a thread, the parts side by side.
template <int N> __global__ __launch_bounds__(N) void decode_join_kernel(DecodeArgs a, uint32_t parts, const float *part) {
    __shared__ __align__(16) float s_o[N * 4];
    __shared__ float s_l[N];
    const int64_t r = blockIdx.x;
    const int h = blockIdx.y, dim = a.kv.dim, tid = threadIdx.x;
    const int len = clamp_len(a.lens[r], a.table.width, a.kv.page), count = parts_of(len, parts).count;
    const int pitch = dim + kPartTail, lanes = dim / 4, side = N / lanes, c = tid % lanes, k = tid / lanes;
    const float *src = part + (r * a.q_heads + h) * parts * pitch;
    // Each thread's parts are k, k + side, ...: a running maximum over them, then over the threads.
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    if (k < side) {
#pragma unroll 4
        for (int i = k; i < count; i += side) {
            const float lse = src[i * pitch + dim];
            const f32x4 x = *reinterpret_cast<const f32x4 *>(src + i * pitch + 4 * c);
            const float mn = fmaxf(m, lse), f = mn == -INFINITY ? 0.f : exp2_f32(m - mn), w = lse == -INFINITY ? 0.f : exp2_f32(lse - mn);
            o = o * f + x * w;
            l = l * f + w, m = mn;
        }
    }
    s_l[tid] = m;
    __syncthreads();
    float top = -INFINITY;
    for (int i = 0; i < side; i++) top = fmaxf(top, s_l[c + i * lanes]);
    __syncthreads();
    const float f = top == -INFINITY ? 0.f : exp2_f32(m - top);
    s_l[tid] = l * f;
    *reinterpret_cast<f32x4 *>(&s_o[tid * 4]) = o * f;
    __syncthreads();
    if (k != 0) return;
    o = f32x4{0.f, 0.f, 0.f, 0.f}, l = 0.f;
    for (int i = 0; i < side; i++) o += *reinterpret_cast<const f32x4 *>(&s_o[(c + i * lanes) * 4]), l += s_l[c + i * lanes];
    const int64_t at = r * a.out_stride + int64_t(h) * dim + 4 * c;
    for (int i = 0; i < 4; i++) store16(a.out, a.type, at + i, l == 0.f ? 0.f : o[i] / l);
}

template <class T, class C> void launch_tiles(const DecodeArgs &a, uint32_t parts, float *part, hipStream_t s) {
    const int group = int(a.q_heads / a.kv.heads);
    const DecodePlan plan{parts, group, (group + 15) / 16, a.kv.page & (a.kv.page - 1) ? -1 : __builtin_ctz(a.kv.page),
                          reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_stride % 8 == 0, cap_of(a.cap, 1.4426950408889634f)};
    const dim3 grid(a.table.rows, a.kv.heads * plan.blocks, parts);
    if (a.kv.dim <= 64) hipLaunchKernelGGL((decode_kernel<T, C, 64>), grid, dim3(256), 0, s, a, plan, part);
    else if (a.kv.dim <= 128) hipLaunchKernelGGL((decode_kernel<T, C, 128>), grid, dim3(256), 0, s, a, plan, part);
    else hipLaunchKernelGGL((decode_kernel<T, C, 256>), grid, dim3(256), 0, s, a, plan, part);
    OCR_HIP(hipGetLastError());
}

// f(query type, cache type) of the pairs that check_decode lets through.
template <class F> void with_pair(const DecodeArgs &a, F &&f) {
    with_type16(a.type, [&](auto t) {
        with_cache(a.kv.type, [&](auto k) {
            if constexpr (scaled<decltype(k)> || std::is_same_v<decltype(t), decltype(k)>) f(t, k);
        });
    });
}

}  // namespace

void launch_decode(Ctx &c, const DecodeArgs &a, hipStream_t s) {
    const bool pieces = whole_pieces(a.kv);
    // Parts until there are two workgroups for every compute unit; a sequence has as many as its own
    // length gives work to. 4 sequences of 131 072: 256 workgroups 194 us, 384 204, 512 179, 1024
    // 181; 144 of 700: one part (576) 24 us, two 30.
    constexpr uint64_t kWork = 512;
    const uint64_t heads = uint64_t(a.table.rows) * a.kv.heads * ((a.q_heads / a.kv.heads + 15) / 16);
    const uint64_t most = uint64_t(a.table.width) * a.kv.page;
    const uint32_t parts = uint32_t(std::max<uint64_t>(1, std::min<uint64_t>({kMostParts, (kWork + heads - 1) / heads, (most + kLeastPart - 1) / kLeastPart})));
    ProbeScope probe("text_decode", s, 4.0 * a.table.rows * a.table.width * a.kv.page * a.q_heads * a.kv.dim,
                     2.0 * a.table.rows * a.table.width * a.kv.page * a.kv.heads * a.kv.dim * type_bytes(a.kv.type),
                     !pieces ? "text_decode_row" : parts > 1 ? "text_decode_parts" : "text_decode_whole");
    if (!pieces) {
        with_pair(a, [&](auto t, auto k) {
            hipLaunchKernelGGL((decode_row_kernel<decltype(t), decltype(k)>), dim3(a.table.rows, a.q_heads), dim3(64), 0, s, a);
        });
        OCR_HIP(hipGetLastError());
        return;
    }
    DBuf part;
    if (parts > 1) part = DBuf(&c, size_t(a.table.rows) * a.q_heads * parts * (a.kv.dim + kPartTail) * 4, s);
    with_pair(a, [&](auto t, auto k) { launch_tiles<decltype(t), decltype(k)>(a, parts, part.as<float>(), s); });
    if (parts > 1) {
        const dim3 grid(a.table.rows, a.q_heads);
        if (parts <= 8) hipLaunchKernelGGL(decode_join_kernel<64>, grid, dim3(64), 0, s, a, parts, part.as<float>());
        else hipLaunchKernelGGL(decode_join_kernel<256>, grid, dim3(256), 0, s, a, parts, part.as<float>());
        OCR_HIP(hipGetLastError());
    }
}

}  // namespace ocr
