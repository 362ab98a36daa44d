// Attention of single tokens over the paged cache.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

// A head's vectors in a sequence's pages; a position whose page there is not holds minus infinity's
// worth: its key scores nothing.
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

}  // namespace

void launch_decode(Ctx &, const DecodeArgs &a, hipStream_t s) {
    ProbeScope probe("text_decode", s, 4.0 * a.table.rows * a.table.width * a.kv.page * a.q_heads * a.kv.dim,
                     2.0 * a.table.rows * a.table.width * a.kv.page * a.kv.heads * a.kv.dim * type_bytes(a.kv.type));
    with_type16(a.type, [&](auto t) {
        with_cache(a.kv.type, [&](auto c) {
            hipLaunchKernelGGL((decode_row_kernel<decltype(t), decltype(c)>), dim3(a.table.rows, a.q_heads), dim3(64), 0, s, a);
        });
    });
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
