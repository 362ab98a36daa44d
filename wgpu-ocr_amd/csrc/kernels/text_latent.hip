// Latent attention over the paged cache of latent vectors: their writing, and single tokens' attention.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

// One wavefront a token.
template <class T, class O> __global__ __launch_bounds__(64) void latent_append_kernel(LatentAppendArgs a) {
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x, rank = a.c.rank, rot = a.c.rot, width = rank + rot;
    const T *x = static_cast<const T *>(a.x) + t * a.stride;
    const int seq = a.seq[t], pos = a.pos[t];
    int page = -1;
    if (seq >= 0 && seq < int(a.table.rows)) page = page_of(a.table.p + size_t(seq) * a.table.width, a.table.width, a.c.page, a.c.pages, pos);
    O *const held = page < 0 ? nullptr : static_cast<O *>(a.c.p) + (int64_t(page) * a.c.page + uint32_t(pos) % a.c.page) * width;
    O *const out = a.out ? static_cast<O *>(a.out) + t * width : nullptr;
    auto put = [&](int c, float v) {
        const O y = O(v);
        if (held) held[c] = y;
        if (out) out[c] = y;
    };
    float r = 1.f;
    if (a.norm) {
        float ss = 0.f;
        for (int c = lane; c < rank; c += 64) ss = __fmaf_rn(to_f32(x[c]), to_f32(x[c]), ss);
        r = 1.f / sqrtf(wave_sum(ss) / float(rank) + a.eps);
    }
    for (int c = lane; c < rank; c += 64) put(c, a.norm ? to_f32(x[c]) * r * a.norm[c] : to_f32(x[c]));
    for (int e = lane; e < rot / 2; e += 64) {
        const int i = rank + (a.adjacent ? 2 * e : e), j = i + (a.adjacent ? 1 : rot / 2);
        const float2 turn = turn_of(a, t, e, rot);
        const float p = to_f32(x[i]), q = to_f32(x[j]);
        put(i, p * turn.x - q * turn.y);
        put(j, q * turn.x + p * turn.y);
    }
}

// By the formula, one wavefront a (sequence, head): a running maximum over 64 positions at a time.
template <class T> __global__ __launch_bounds__(64) void latent_row_kernel(LatentDecodeArgs a) {
    __shared__ float s_q[kMostRank + kMostLatentRot];
    const int64_t r = blockIdx.x;
    const int h = blockIdx.y, lane = threadIdx.x, rank = a.c.rank, width = rank + int(a.c.rot);
    const T *q = static_cast<const T *>(a.q) + r * a.q_stride + int64_t(h) * width;
    for (int c = lane; c < width; c += 64) s_q[c] = to_f32(q[c]) * a.scale;
    __syncthreads();
    const int len = clamp_len(a.lens[r], a.table.width, a.c.page);
    auto vec = [&](int j) -> const T * {
        const int32_t p = page_of(a.table.p + r * a.table.width, a.table.width, a.c.page, a.c.pages, j);
        return p < 0 ? nullptr : static_cast<const T *>(a.c.p) + (int64_t(p) * a.c.page + uint32_t(j) % a.c.page) * width;
    };
    float m = -INFINITY, l = 0.f, o[kMostRank / 64];
#pragma unroll
    for (int u = 0; u < int(kMostRank / 64); u++) o[u] = 0.f;
    for (int j0 = 0; j0 < len; j0 += 64) {
        const int j = j0 + lane;
        float s = -INFINITY;
        if (j < len) {
            const T *c = vec(j);
            s = 0.f;
            if (c)
                for (int e = 0; e < width; e++) s = __fmaf_rn(s_q[e], to_f32(c[e]), s);
        }
        const float mn = fmaxf(m, wave_max(s)), f = mn == -INFINITY ? 1.f : expf(m - mn);
        const float p = s == -INFINITY ? 0.f : expf(s - mn);
        l = l * f + p;
        m = mn;
#pragma unroll
        for (int u = 0; u < int(kMostRank / 64); u++) o[u] *= f;
        const int count = min(64, len - j0);
        for (int t = 0; t < count; t++) {
            const float w = __shfl(p, t);
            const T *c = vec(j0 + t);
            if (w == 0.f || !c) continue;
#pragma unroll
            for (int u = 0; u < int(kMostRank / 64); u++)
                if (lane + 64 * u < rank) o[u] = __fmaf_rn(w, to_f32(c[lane + 64 * u]), o[u]);
        }
    }
    l = wave_sum(l);
    T *out = static_cast<T *>(a.out) + r * a.out_stride + int64_t(h) * rank;
#pragma unroll
    for (int u = 0; u < int(kMostRank / 64); u++)
        if (lane + 64 * u < rank) out[lane + 64 * u] = T(l == 0.f ? 0.f : o[u] / l);
}

}  // namespace

void launch_latent_append(const LatentAppendArgs &a, hipStream_t s) {
    const double values = double(a.n) * (a.c.rank + a.c.rot);
    ProbeScope probe("latent_append", s, 6 * values, values * (type_bytes(a.type) + 2));
    with_type(a.type, [&](auto t) {
        with_type16(a.c.type, [&](auto o) { hipLaunchKernelGGL((latent_append_kernel<decltype(t), decltype(o)>), dim3(a.n), dim3(64), 0, s, a); });
    });
    OCR_HIP(hipGetLastError());
}

void launch_latent_decode(Ctx &, const LatentDecodeArgs &a, hipStream_t s) {
    const double vecs = double(a.table.rows) * a.table.width * a.c.page;
    ProbeScope probe("latent_decode", s, 2.0 * vecs * a.heads * (2 * a.c.rank + a.c.rot), 2.0 * vecs * (a.c.rank + a.c.rot), "latent_decode_row");
    with_type16(a.c.type, [&](auto t) { hipLaunchKernelGGL((latent_row_kernel<decltype(t)>), dim3(a.table.rows, a.heads), dim3(64), 0, s, a); });
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
