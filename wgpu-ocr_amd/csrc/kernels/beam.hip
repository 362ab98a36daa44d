// A step of beam search: log-softmax of every beam's logits, the best of all beams' continuations.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

// A continuation: larger score first, then the lower index.
struct Cand {
    double score;
    int at;
};
__device__ inline bool before(const Cand &a, const Cand &b) { return a.score > b.score || (a.score == b.score && a.at < b.at); }
__device__ inline Cand wave_best(Cand c) {
    for (int o = 32; o; o >>= 1) {
        const Cand d{__shfl_xor(c.score, o), __shfl_xor(c.at, o)};
        if (before(d, c)) c = d;
    }
    return c;
}

// One workgroup a beam: its best `beams` continuations in order.
template <class T> __global__ __launch_bounds__(256) void beam_rows_kernel(BeamArgs a, Cand *cand) {
    __shared__ double s_d[4];
    __shared__ float s_m[4];
    __shared__ Cand s_c[4];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, v = a.vocab;
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    const double cum = a.scores[row];
    const bool over = a.finished && a.finished[row];
    auto logit = [&](int t) {  // NaN weighs nothing
        const float f = to_f32(x[t]);
        return f == f ? f : -INFINITY;
    };
    float m = -INFINITY;
    for (int t = threadIdx.x; t < v; t += 256) m = fmaxf(m, logit(t));
    m = wave_max(m);
    if (lane == 0) s_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    double sum = 0;
    for (int t = threadIdx.x; t < v; t += 256) sum += exp(double(logit(t)) - double(m));
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) s_d[wave] = sum;
    __syncthreads();
    const double lse = double(m) + log(s_d[0] + s_d[1] + s_d[2] + s_d[3]);
    auto score = [&](int t) {
        const double s = over ? (t == a.eos ? cum : -INFINITY) : cum + (double(logit(t)) - lse);
        return s == s ? s : -INFINITY;
    };
    Cand last{INFINITY, -1};
    for (int k = 0; k < int(a.beams); k++) {
        Cand best{-INFINITY, 0x7fffffff};
        for (int t = threadIdx.x; t < v; t += 256) {
            const Cand c{score(t), t};
            if (before(last, c) && before(c, best)) best = c;
        }
        best = wave_best(best);
        __syncthreads();
        if (lane == 0) s_c[wave] = best;
        __syncthreads();
        for (int o = 0; o < 4; o++)
            if (before(s_c[o], best)) best = s_c[o];
        if (threadIdx.x == 0) cand[row * a.beams + k] = best;
        last = best;
    }
}

// One wavefront a group.
__global__ __launch_bounds__(64) void beam_groups_kernel(BeamArgs a, const Cand *cand) {
    const int g = blockIdx.x, w = a.beams, n = w * w, lane = threadIdx.x;
    struct Pick {
        Cand c;
        int beam;
    };
    int fin[2] = {0, 0};
    Cand last{INFINITY, -1};
    int last_beam = -1;
    for (int k = 0; k < w; k++) {
        Cand best{-INFINITY, 0x7fffffff};
        int beam = w;
        auto better = [](const Cand &c, int cb, const Cand &d, int db) {
            return c.score > d.score || (c.score == d.score && (cb < db || (cb == db && c.at < d.at)));
        };
        for (int i = lane; i < n; i += 64) {
            const Cand c = cand[int64_t(g) * n + i];
            if (c.at == 0x7fffffff) continue;
            if (better(last, last_beam, c, i / w) && better(c, i / w, best, beam)) best = c, beam = i / w;
        }
        for (int o = 32; o; o >>= 1) {
            const Cand d{__shfl_xor(best.score, o), __shfl_xor(best.at, o)};
            const int db = __shfl_xor(beam, o);
            if (better(d, db, best, beam)) best = d, beam = db;
        }
        if (lane == k) fin[0] = (a.finished && a.finished[g * w + beam]) || (a.eos >= 0 && best.at == a.eos);
        if (lane == 0) {
            a.parents[g * w + k] = beam;
            a.tokens[g * w + k] = best.at;
        }
        if (lane == k) fin[1] = __float_as_int(float(best.score));
        last = best, last_beam = beam;
    }
    if (lane < w) {  // every score and flag of the group has been read: the outputs may be the inputs
        a.out_scores[g * w + lane] = __int_as_float(fin[1]);
        if (a.out_finished) a.out_finished[g * w + lane] = fin[0];
    }
}

}  // namespace

void launch_beam(Ctx &c, const BeamArgs &a, hipStream_t s) {
    const int rows = int(a.groups * a.beams);
    ProbeScope probe("beam_select", s, 3.0 * rows * a.vocab, double(rows) * a.vocab * type_bytes(a.type));
    DBuf cand(&c, size_t(rows) * a.beams * sizeof(Cand), s);
    with_type(a.type, [&](auto t) {
        hipLaunchKernelGGL((beam_rows_kernel<decltype(t)>), dim3(rows), dim3(256), 0, s, a, cand.as<Cand>());
    });
    OCR_HIP(hipGetLastError());
    hipLaunchKernelGGL(beam_groups_kernel, dim3(a.groups), dim3(64), 0, s, a, cand.as<Cand>());
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
