// How much of the attention each key got, added up: of a prompt's queries and of single tokens.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

// A query's scores by the formula: their maximum and the sum of e^(s - max), one wavefront. kv.k as in attend_row.
template <class KV> struct RowScores {
    const KV &kv;
    const float *q;
    int dim, pos;
    Cap most;
    float cap, slope;
    __device__ float operator()(int j) const {
        float s = 0.f;
        for (int c = 0; c < dim; c++) s = __fmaf_rn(q[c], kv.k(j, c), s);
        if (cap > 0.f) s = capped(most, s);
        return s - slope * float(pos > j ? pos - j : j - pos);
    }
    __device__ float2 sums(int lo, int hi) const {
        const int lane = threadIdx.x & 63;
        float m = -INFINITY, l = 0.f;
        for (int j = lo + lane; j < hi; j += 64) m = fmaxf(m, (*this)(j));
        m = wave_max(m);
        for (int j = lo + lane; j < hi; j += 64) {
            const float s = (*this)(j);
            l += s == -INFINITY ? 0.f : expf(s - m);
        }
        l = wave_sum(l);
        return {m, l == 0.f ? 0.f : 1.f / l};
    }
};

template <class T> struct DenseK {
    const T *p;
    int64_t stride;
    __device__ float k(int j, int c) const { return to_f32(p[j * stride + c]); }
};

// Every query's maximum and one over its sum.
template <class T> __global__ __launch_bounds__(64) void row_sums_kernel(AttentionArgs a, float2 *sums) {
    __shared__ float s_q[256];
    const int i = blockIdx.x, h = blockIdx.y, dim = a.dim, hk = h / int(a.q_heads / a.kv_heads);
    const T *q = static_cast<const T *>(a.q) + i * a.q_stride + int64_t(h) * dim;
    for (int c = threadIdx.x; c < dim; c += 64) s_q[c] = to_f32(q[c]) * a.scale;
    __syncthreads();
    const KeyRange r = key_range(i, int(a.n), a.docs, int(a.ndocs), a.prefix);
    const DenseK<T> kv{static_cast<const T *>(a.k) + int64_t(hk) * dim, a.k_stride};
    const float2 x = RowScores<DenseK<T>>{kv, s_q, dim, i, cap_of(a.cap, 1.f), a.cap, a.slopes ? a.slopes[h] : 0.f}.sums(r.lo, r.hi);
    if (threadIdx.x == 0) sums[int64_t(i) * a.q_heads + h] = x;
}

// A key's weights by the formula, one wavefront a (key, head): the lanes take its queries.
template <class T> __global__ __launch_bounds__(64) void weights_row_kernel(AttentionArgs a, Weights w, const float2 *sums) {
    __shared__ float s_k[256];
    const int j = blockIdx.x, hk = blockIdx.y, dim = a.dim, group = int(a.q_heads / a.kv_heads);
    const QueryRange r = query_range(j, int(a.n), a.docs, int(a.ndocs), a.prefix, int(w.window));
    if (r.doc < 0 || uint32_t(r.place) >= w.most) return;
    const T *k = static_cast<const T *>(a.k) + j * a.k_stride + int64_t(hk) * dim;
    for (int c = threadIdx.x; c < dim; c += 64) s_k[c] = to_f32(k[c]);
    __syncthreads();
    const Cap most = cap_of(a.cap, 1.f);
    float sum = 0.f;
    for (int g = 0; g < group; g++) {
        const int h = hk * group + g;
        const float slope = a.slopes ? a.slopes[h] : 0.f;
        for (int i = r.lo + int(threadIdx.x); i < r.hi; i += 64) {
            const T *q = static_cast<const T *>(a.q) + i * a.q_stride + int64_t(h) * dim;
            float s = 0.f;
            for (int c = 0; c < dim; c++) s = __fmaf_rn(to_f32(q[c]) * a.scale, s_k[c], s);
            if (a.cap > 0.f) s = capped(most, s);
            s -= slope * float(i > j ? i - j : j - i);
            const float2 x = sums[int64_t(i) * a.q_heads + h];
            sum += s == -INFINITY ? 0.f : expf(s - x.x) * x.y;
        }
    }
    sum = wave_sum(sum);
    if (threadIdx.x == 0) w.p[(int64_t(r.doc) * a.kv_heads + hk) * w.most + r.place] += sum;
}

// Keys of a sequence's pages; a position whose page there is not holds zeros.
template <class C> struct PagedK {
    KvCache c;
    const int32_t *row;
    uint32_t width, head;
    __device__ float k(int j, int i) const {
        const int32_t p = page_of(row, width, c.page, c.pages, j);
        if (p < 0) return 0.f;
        const int64_t s = slot_of(p, c.heads, c.page, head, uint32_t(j) % c.page);
        return to_f32(static_cast<const C *>(c.k)[s * c.dim + i]) * (scaled<C> ? c.k_scale[s] : 1.f);
    }
};

// A single token's weights by the formula: one wavefront a (sequence, key head).
template <class T, class C> __global__ __launch_bounds__(64) void single_weights_row_kernel(DecodeArgs a, Weights w) {
    __shared__ float s_q[256];
    __shared__ float2 s_sums[1024];  // of the key head's query heads
    const int64_t r = blockIdx.x;
    const int hk = blockIdx.y, dim = a.kv.dim, group = int(a.q_heads / a.kv.heads), lane = threadIdx.x;
    const int len = clamp_len(a.lens[r], a.table.width, a.kv.page);
    const PagedK<C> kv{a.kv, a.table.p + r * a.table.width, a.table.width, uint32_t(hk)};
    const T *const q0 = static_cast<const T *>(a.q) + r * a.q_stride + int64_t(hk) * group * dim;
    const Cap most = cap_of(a.cap, 1.f);
    const auto slope = [&](int g) { return a.slopes ? a.slopes[hk * group + g] : 0.f; };
    for (int g = 0; g < group; g++) {
        __syncthreads();
        for (int c = lane; c < dim; c += 64) s_q[c] = to_f32(q0[g * dim + c]) * a.scale;
        __syncthreads();
        const float2 x = RowScores<PagedK<C>>{kv, s_q, dim, len - 1, most, a.cap, slope(g)}.sums(0, len);
        if (lane == 0) s_sums[g] = x;
    }
    for (int j0 = 0; j0 < len && uint32_t(j0) < w.most; j0 += 64) {
        const int j = j0 + lane;
        float sum = 0.f;
        for (int g = 0; g < group; g++) {
            __syncthreads();
            for (int c = lane; c < dim; c += 64) s_q[c] = to_f32(q0[g * dim + c]) * a.scale;
            __syncthreads();
            if (j >= len) continue;
            const float s = RowScores<PagedK<C>>{kv, s_q, dim, len - 1, most, a.cap, slope(g)}(j);
            sum += s == -INFINITY ? 0.f : expf(s - s_sums[g].x) * s_sums[g].y;
        }
        if (j < len && uint32_t(j) < w.most) w.p[(r * a.kv.heads + hk) * w.most + j] += sum;
    }
}

}  // namespace

void launch_attention_weights(Ctx &c, const AttentionArgs &a, const Weights &w, hipStream_t s) {
    launch_attention(a, s);
    ProbeScope probe("text_weights", s, 2.0 * a.n * a.n * a.q_heads * a.dim, 2.0 * a.n * (a.q_heads + a.kv_heads) * a.dim, "text_weights_row");
    DBuf sums(&c, size_t(a.n) * a.q_heads * sizeof(float2), s);
    with_type16(a.type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((row_sums_kernel<T>), dim3(a.n, a.q_heads), dim3(64), 0, s, a, sums.as<float2>());
        hipLaunchKernelGGL((weights_row_kernel<T>), dim3(a.n, a.kv_heads), dim3(64), 0, s, a, w, sums.as<float2>());
    });
    OCR_HIP(hipGetLastError());
}

void launch_decode_weights(Ctx &c, const DecodeArgs &a, const Weights &w, hipStream_t s) {
    launch_decode(c, a, s);
    ProbeScope probe("text_weights", s, 2.0 * a.table.rows * w.most * a.q_heads * a.kv.dim, 8.0 * a.table.rows * w.most * a.kv.heads, "text_weights_row");
    with_type16(a.type, [&](auto t) {
        with_cache(a.kv.type, [&](auto k) {
            if constexpr (scaled<decltype(k)> || std::is_same_v<decltype(t), decltype(k)>)
                hipLaunchKernelGGL((single_weights_row_kernel<decltype(t), decltype(k)>), dim3(a.table.rows, a.kv.heads), dim3(64), 0, s, a, w);
        });
    });
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
