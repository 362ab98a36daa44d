// Attention over a packed row of documents: scores capped by a tanh, a bias that falls with the
// distance, document and prefix masks.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

template <class T> struct DenseKv {
    const T *kp, *vp;
    int64_t ks, vs;
    __device__ float k(int j, int c) const { return to_f32(kp[j * ks + c]); }
    __device__ float v(int j, int c) const { return to_f32(vp[j * vs + c]); }
};

// One wavefront a (token, head), by the formula.
template <class T> __global__ __launch_bounds__(64) void attention_row_kernel(AttentionArgs a) {
    __shared__ float s_q[256];
    const int64_t i = blockIdx.x;
    const int h = blockIdx.y, dim = a.dim, hk = h / int(a.q_heads / a.kv_heads);
    const T *q = static_cast<const T *>(a.q) + i * a.q_stride + int64_t(h) * dim;
    for (int c = threadIdx.x; c < dim; c += 64) s_q[c] = to_f32(q[c]) * a.scale;
    __syncthreads();
    const KeyRange r = key_range(int(i), int(a.n), a.docs, int(a.ndocs), a.prefix);
    const DenseKv<T> kv{static_cast<const T *>(a.k) + int64_t(hk) * dim, static_cast<const T *>(a.v) + int64_t(hk) * dim, a.k_stride, a.v_stride};
    T *out = static_cast<T *>(a.out) + i * a.out_stride + int64_t(h) * dim;
    attend_row(kv, s_q, dim, r.lo, r.hi, int(i), a.cap, a.slopes ? a.slopes[h] : 0.f, [&](int c, float o) { out[c] = T(o); });
}

}  // namespace

void launch_attention(const AttentionArgs &a, hipStream_t s) {
    ProbeScope probe("text_attention", s, 2.0 * a.n * a.n * a.q_heads * a.dim, 4.0 * a.n * (a.q_heads + a.kv_heads) * a.dim);
    with_type16(a.type, [&](auto t) {
        hipLaunchKernelGGL((attention_row_kernel<decltype(t)>), dim3(a.n, a.q_heads), dim3(64), 0, s, a);
    });
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
