// The text decoder's cache: a step's projections normed, rotated and written into pages, pages read
// back, beams' pages reordered.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

// One wavefront a (token, head): lane l holds values l, l + 64, ... of the head's vector.
template <class T, class O, class C> __global__ __launch_bounds__(64) void append_kernel(AppendArgs a) {
    __shared__ float s_x[256];
    const int lane = threadIdx.x, dim = a.kv.dim, heads = a.kv.heads;
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y;
    const int kind = h < int(a.q_heads) ? 0 : h < int(a.q_heads) + heads ? 1 : 2;  // q, k, v
    const T *src = static_cast<const T *>(a.qkv) + t * a.stride + int64_t(h) * dim;
    const int pos = a.pos[t];
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; u++) x[u] = lane + 64 * u < dim ? to_f32(src[lane + 64 * u]) : 0.f;
    const float *norm = kind == 0 ? a.q_norm : a.k_norm;
    if (kind < 2 && norm) {
        float ss = 0.f;
        for (int u = 0; u < 4; u++) ss += x[u] * x[u];
        const float r = 1.f / sqrtf(wave_sum(ss) / float(dim) + a.eps);
        for (int u = 0; u < 4; u++)
            if (lane + 64 * u < dim) x[u] = x[u] * r * norm[lane + 64 * u];
    }
    if (kind < 2 && a.rot) {
        for (int u = 0; u < 4; u++) s_x[lane + 64 * u] = x[u];
        __syncthreads();
        const int half = a.rot / 2;
        for (int u = 0; u < 4; u++) {
            const int c = lane + 64 * u;
            if (c >= int(a.rot)) continue;
            const int i = a.adjacent ? c >> 1 : c % half;
            const bool second = a.adjacent ? c & 1 : c >= half;
            const int other = a.adjacent ? c ^ 1 : second ? c - half : c + half;
            const double turns = double(pos) * (exp2(-2.0 * i / double(a.rot) * a.log2_theta) * 0.15915494309189533577);
            float sn, cs;
            sincospif(2.f * float(turns - rint(turns)), &sn, &cs);
            x[u] = second ? x[u] * cs + s_x[other] * sn : x[u] * cs - s_x[other] * sn;
        }
    }
    if (kind == 0) {
        O *dst = static_cast<O *>(a.q) + (t * a.q_heads + h) * dim;
        for (int u = 0; u < 4; u++)
            if (lane + 64 * u < dim) dst[lane + 64 * u] = O(x[u]);
        return;
    }
    const int hk = h - int(a.q_heads) - (kind == 2 ? heads : 0);
    if (kind == 1 && a.k) {
        O *dst = static_cast<O *>(a.k) + (t * heads + hk) * dim;
        for (int u = 0; u < 4; u++)
            if (lane + 64 * u < dim) dst[lane + 64 * u] = O(x[u]);
    }
    const int seq = a.seq[t];
    if (seq < 0 || seq >= int(a.table.rows)) return;
    const int page = page_of(a.table.p + size_t(seq) * a.table.width, a.table.width, a.kv.page, a.kv.pages, pos);
    if (page < 0) return;
    const int64_t slot = slot_of(page, heads, a.kv.page, hk, pos % a.kv.page);
    C *dst = static_cast<C *>(kind == 1 ? a.kv.k : a.kv.v) + slot * dim;
    float inv = 1.f;
    if constexpr (scaled<C>) {
        float m = 0.f, bad = 0.f;
        for (int u = 0; u < 4; u++) m = fmaxf(m, fabsf(x[u])), bad += x[u] * 0.f;
        m = wave_max(m);
        bad = wave_sum(bad);
        inv = m > kTinyMax ? code_max<C> / m : 0.f;
        float scale = m > kTinyMax ? m / code_max<C> : 0.f;
        if (!(bad == 0.f)) inv = 0.f, scale = NAN;  // a value that is not finite: the whole vector reads as NaN
        if (lane == 0) (kind == 1 ? a.kv.k_scale : a.kv.v_scale)[slot] = scale;
        if (!(bad == 0.f))
            for (int u = 0; u < 4; u++) x[u] = 0.f;
    }
    for (int u = 0; u < 4; u++)
        if (lane + 64 * u < dim) dst[lane + 64 * u] = code_of<C>(x[u] * inv);
}

template <class C, class O> __global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
    const int dim = a.kv.dim, heads = a.kv.heads;
    const int64_t pos = blockIdx.x, seq = blockIdx.y;
    const bool there = pos < clamp_len(a.lens[seq], a.table.width, a.kv.page);
    const int page = there ? page_of(a.table.p + seq * a.table.width, a.table.width, a.kv.page, a.kv.pages, pos) : -1;
    const int64_t out = (seq * a.most + pos) * heads * dim;
    for (int i = threadIdx.x; i < heads * dim; i += 256) {
        float k = 0.f, v = 0.f;
        if (page >= 0) {
            const int64_t slot = slot_of(page, heads, a.kv.page, i / dim, pos % a.kv.page);
            k = to_f32(static_cast<const C *>(a.kv.k)[slot * dim + i % dim]);
            v = to_f32(static_cast<const C *>(a.kv.v)[slot * dim + i % dim]);
            if constexpr (scaled<C>) k *= a.kv.k_scale[slot], v *= a.kv.v_scale[slot];
        }
        static_cast<O *>(a.k)[out + i] = O(k);
        static_cast<O *>(a.v)[out + i] = O(v);
    }
}

// One workgroup a (sequence, head): the head's part of a copied page, the first also the table's row.
// P: what a thread copies at once.
template <class P> __global__ __launch_bounds__(256) void fork_kernel(ForkArgs a) {
    const uint32_t r = blockIdx.x, h = blockIdx.y, w = r % a.beams, g = r - w;
    const Fork f = fork_of(a.parents + g, a.beams, w, a.lens + g, a.table.width, a.kv.page);
    const int32_t p = a.parents[r];
    const bool ok = p >= 0 && uint32_t(p) < a.beams;
    const int32_t *from = a.table.p + size_t(g + (ok ? p : 0)) * a.table.width;
    if (h == 0) {
        int32_t *to = a.table_out + size_t(r) * a.table.width;
        const uint32_t cols = ok ? f.full + (f.tail > 0) : 0;
        for (uint32_t i = threadIdx.x; i < a.table.width; i += 256)
            to[i] = i >= cols ? -1 : i == f.full && f.copy ? a.spare[r] : from[i];
        if (threadIdx.x == 0) a.lens_out[r] = f.len, a.used[r] = f.copy;
    }
    if (!f.copy) return;
    const int32_t src = from[f.full], dst = a.spare[r];
    if (src < 0 || uint32_t(src) >= a.kv.pages || dst < 0 || uint32_t(dst) >= a.kv.pages || src == dst) return;
    const bool coded = a.kv.type == T_I8 || a.kv.type == T_E4M3;
    const size_t vec = size_t(a.kv.dim) * (coded ? 1 : 2);
    const int64_t s0 = slot_of(src, a.kv.heads, a.kv.page, h, 0), d0 = slot_of(dst, a.kv.heads, a.kv.page, h, 0);
    const P *ks = reinterpret_cast<const P *>(static_cast<const char *>(a.kv.k) + s0 * vec), *vs = reinterpret_cast<const P *>(static_cast<const char *>(a.kv.v) + s0 * vec);
    P *kd = reinterpret_cast<P *>(static_cast<char *>(a.kv.k) + d0 * vec), *vd = reinterpret_cast<P *>(static_cast<char *>(a.kv.v) + d0 * vec);
    const uint32_t n = uint32_t(f.tail * vec / sizeof(P));
    uint32_t i = threadIdx.x;
    for (; i + 768 < n; i += 1024) {  // all on their way before the first is written
        P x[4], y[4];
#pragma unroll
        for (int u = 0; u < 4; u++) x[u] = ks[i + 256 * u], y[u] = vs[i + 256 * u];
#pragma unroll
        for (int u = 0; u < 4; u++) kd[i + 256 * u] = x[u], vd[i + 256 * u] = y[u];
    }
    for (; i < n; i += 256) kd[i] = ks[i], vd[i] = vs[i];
    if (coded)
        for (uint32_t e = threadIdx.x; e < f.tail; e += 256)
            a.kv.k_scale[d0 + e] = a.kv.k_scale[s0 + e], a.kv.v_scale[d0 + e] = a.kv.v_scale[s0 + e];
}

}  // namespace

void launch_append(const AppendArgs &a, hipStream_t s) {
    const double values = double(a.n) * (a.q_heads + 2 * a.kv.heads) * a.kv.dim;
    ProbeScope probe("text_append", s, 10 * values, values * (type_bytes(a.type) + 2));
    const dim3 grid(a.n, a.q_heads + 2 * a.kv.heads);
    with_type(a.type, [&](auto t) {
        with_type16(a.out_type, [&](auto o) {
            with_cache(a.kv.type, [&](auto c) {
                hipLaunchKernelGGL((append_kernel<decltype(t), decltype(o), decltype(c)>), grid, dim3(64), 0, s, a);
            });
        });
    });
    OCR_HIP(hipGetLastError());
}

void launch_read(const ReadArgs &a, hipStream_t s) {
    const double values = 2.0 * a.table.rows * a.most * a.kv.heads * a.kv.dim;
    ProbeScope probe("text_read", s, values, values * (type_bytes(a.kv.type) + 2));
    const dim3 grid(a.most, a.table.rows);
    with_cache(a.kv.type, [&](auto c) {
        with_type16(a.type, [&](auto o) { hipLaunchKernelGGL((read_kernel<decltype(c), decltype(o)>), grid, dim3(256), 0, s, a); });
    });
    OCR_HIP(hipGetLastError());
}

void launch_fork(const ForkArgs &a, hipStream_t s) {
    ProbeScope probe("text_fork", s, 0, 8.0 * a.table.rows * a.table.width);
    const dim3 grid(a.table.rows, a.kv.heads);
    if (whole_pieces(a.kv)) hipLaunchKernelGGL(fork_kernel<u32x4>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(fork_kernel<uint8_t>, grid, dim3(256), 0, s, a);
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
