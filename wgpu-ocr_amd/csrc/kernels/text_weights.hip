// How much of the attention each key got from a prompt's queries, added up (single tokens': text_decode.hip).
//
// The attention itself leaves every query's reference and one over its sum, so a weight is e^(s - reference) times that:
// the scores are made a second time, S = Q K^T with the queries as rows, so that a lane has one key and sums its
// column in a register, without maximum, rescaling or atomics.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "text_device.h"
#include "text_tile.h"

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

// The documents' offsets, few ones in LDS: the search for a key's document is six loads one after another for 36 of them.
constexpr int kFewDocs = 256;
__device__ inline const int32_t *offsets_here(const AttentionArgs &a, int32_t *s_docs) {
    if (!a.docs || a.ndocs >= kFewDocs) return a.docs;
    for (uint32_t i = threadIdx.x; i <= a.ndocs; i += blockDim.x) s_docs[i] = a.docs[i];
    __syncthreads();
    return s_docs;
}

// 32 KB keys a wavefront, held in registers, over tiles of 64 queries of one head that come into LDS by DMA while the tile
// before is worked on. A workgroup's 128 KB keys of a key head; slice: one of its query heads, and one of `cuts` parts of the queries.
// part [slice][kv_heads][n]. CAPPED: with a cap or slopes.
// Two documents of up to 5000, 32 query heads over 8 of 128, bf16: 165 us, the matrix cores busy a quarter of it; an exponential, two
// fused products and a wait for LDS a score are some 24 cycles of a wavefront. 32 keys a wavefront 239 us.
template <class T, int DP, bool CAPPED, int KB> __global__ __launch_bounds__(256) void prompt_weights_kernel(AttentionArgs a, int window, int tiles, int cuts, float *part) {
    typedef T tvec __attribute__((ext_vector_type(8)));
    constexpr int PW = DP <= 64 ? 64 : DP <= 128 ? 128 : 256, QT = PW == 256 ? 32 : 64, KS = DP / 16;
    using TQ = Tile<PW, QT>;
    constexpr int BUF = TQ::BYTES + 2 * 256;  // the queries, their references and their sums' inverses
    __shared__ __align__(16) char s_q[2 * BUF];
    __shared__ int s_lo[4], s_hi[4];
    __shared__ int32_t s_docs[kFewDocs];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int group = int(a.q_heads / a.kv_heads), slices = group * cuts;
    // Dies take key heads in turn; a die's workgroups go through a head's keys before the next slice, whose queries stay in its level-two cache.
    const int hk = int(blockIdx.x % a.kv_heads), rest = int(blockIdx.x / a.kv_heads), tile = rest % tiles, slice = rest / tiles;
    const int h = hk * group + slice / cuts, cut = slice % cuts, dim = a.dim, pieces = dim / 8;
    if (slice >= slices) return;
    int j[KB], lo[KB], hi[KB];  // the lane's keys, and the queries that see them
#pragma unroll
    for (int t = 0; t < KB; t++) j[t] = tile * (128 * KB) + 32 * (KB * wave + t) + (lane & 31);
    tvec kf[KB][KS];
    {
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0;
#pragma unroll
        for (int t = 0; t < KB; t++) {
            const char *k = static_cast<const char *>(a.k) + (int64_t(min(j[t], int(a.n) - 1)) * a.k_stride + int64_t(hk) * dim) * 2;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                u32x4 x{0, 0, 0, 0};
                if (2 * s + half < pieces) x = *reinterpret_cast<const u32x4 *>(k + 16 * (2 * s + half));
                kf[t][s] = __builtin_bit_cast(tvec, x ^ flip);
            }
        }
    }
    const int32_t *const docs = offsets_here(a, s_docs);
    int wlo = 0x7fffffff, whi = 0, flo = 0, fhi = 0x7fffffff;  // some key is seen by those in [wlo, whi), all by those in [flo, fhi)
#pragma unroll
    for (int t = 0; t < KB; t++) {
        QueryRange r{0, 0, -1, 0};
        if (j[t] < int(a.n)) r = query_range(j[t], int(a.n), docs, int(a.ndocs), a.prefix, window);
        const bool seen = r.lo < r.hi;
        lo[t] = seen ? r.lo : 0, hi[t] = seen ? r.hi : 0;
        wlo = min(wlo, seen ? r.lo : 0x7fffffff), whi = max(whi, hi[t]);
        flo = max(flo, lo[t]), fhi = min(fhi, hi[t]);
    }
    wlo = wave_min_i(wlo), whi = wave_max_i(whi), flo = wave_max_i(flo), fhi = wave_min_i(fhi);
    if (lane == 0) s_lo[wave] = wlo, s_hi[wave] = whi;
    const TQ tq(a.q_stride, pieces);
    if (pieces < TQ::PP) {  // pieces that no copy writes count nothing
        for (int x = tid; x < 2 * BUF / 16; x += 256) *reinterpret_cast<u32x4 *>(s_q + 16 * x) = u32x4{0, 0, 0, 0};
    }
    __syncthreads();
    int qlo = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3])), qhi = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
    qlo = __builtin_amdgcn_readfirstlane(qlo), qhi = __builtin_amdgcn_readfirstlane(qhi);
    float sum[KB][4] = {};
    if (qlo < qhi) {
        // This part's tiles of queries.
        const int t0 = qlo / QT, t1 = (qhi + QT - 1) / QT, each = (t1 - t0 + cuts - 1) / cuts;
        const int i0 = (t0 + cut * each) * QT, i1 = min(qhi, (t0 + (cut + 1) * each) * QT);
        const char *const qbase = static_cast<const char *>(a.q) + int64_t(h) * dim * 2;
        const float *const sums = a.sums + 2 * int64_t(h) * sums_pitch(a.n);
        const unsigned lds0 = lds_addr(s_q);
        auto copy = [&](int i, int buf) {
            tq.copy(qbase + int64_t(i) * tq.step, lds0 + buf * BUF + wave * 1024, int(a.n) - i);
            // Sixteen lanes for the references, sixteen for the inverses.
            if (wave == 0 && lane < 32)
                dma16s_to(sums + i, unsigned(((lane >> 4) * sums_pitch(a.n) + 4 * (lane & 15) % QT) * 4), lds0 + buf * BUF + TQ::BYTES);
        };
        int qoff[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) qoff[s] = (lane & 31) * PW * 2 + ((2 * s + half) ^ TQ::swap_of(lane & 15)) * 16;
        const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);
        const float slope = CAPPED && a.slopes ? a.slopes[h] * 1.4426950408889634f : 0.f;
        const SmallCap small(fabsf(a.scale), CAPPED && a.cap > 0.f ? a.cap : 1.f);
        const Cap cap = cap_of(a.cap, 1.4426950408889634f);
        // 32 queries from i on.
        auto turn = [&](int i, const char *s_b, int u) __attribute__((always_inline)) {
            if (i >= whi || i + 32 <= wlo) return;
            f32x16 s[KB];
#pragma unroll
            for (int t = 0; t < KB; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[t][e] = 0.f;
#pragma unroll
            for (int st = 0; st < KS; st++) {
                const tvec q = *reinterpret_cast<const tvec *>(s_b + qoff[st] + u * 32 * PW * 2);
#pragma unroll
                for (int t = 0; t < KB; t++) s[t] = mfma32(q, kf[t][st], s[t]);
            }
            if constexpr (CAPPED) {
                float top = 0.f;
                if (a.cap > 0.f) {
#pragma unroll
                    for (int t = 0; t < KB; t++)
#pragma unroll
                        for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(s[t][e]));
                }
                const bool large = a.cap > 0.f && __any(top > small.most);
#pragma unroll
                for (int t = 0; t < KB; t++) {
                    if (large) {
#pragma unroll
                        for (int e = 0; e < 16; e++) s[t][e] = capped(cap, s[t][e] * c);
                    } else if (a.cap > 0.f) {
#pragma unroll
                        for (int e = 0; e < 16; e++) s[t][e] *= small.factor(s[t][e]);
                    } else {
                        s[t] *= c;
                    }
                    if (a.slopes) {
                        const float d = float(i + 4 * half - j[t]);
#pragma unroll
                        for (int e = 0; e < 16; e++) s[t][e] -= slope * fabsf(d + float(8 * (e / 4) + e % 4));
                    }
                }
            }
            auto add = [&](auto whole) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const f32x4 ref = *reinterpret_cast<const f32x4 *>(s_b + TQ::BYTES + (32 * u + 2 * e + 4 * half) * 4);
                    const f32x4 inv = *reinterpret_cast<const f32x4 *>(s_b + TQ::BYTES + 256 + (32 * u + 2 * e + 4 * half) * 4);
#pragma unroll
                    for (int t = 0; t < KB; t++)
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const float p = exp2_f32(CAPPED ? s[t][e + x] - ref[x] : __fmaf_rn(s[t][e + x], c, -ref[x]));
                            // What is not seen may be anything, and so may its query's sum.
                            if constexpr (decltype(whole)::value) sum[t][x] = __fmaf_rn(p, inv[x], sum[t][x]);
                            else sum[t][x] += unsigned(i + 4 * half + 2 * e + x - lo[t]) < unsigned(hi[t] - lo[t]) ? p * inv[x] : 0.f;
                        }
                }
            };
            if (i >= flo && i + 32 <= fhi) add(std::true_type{});
            else add(std::false_type{});
        };
        auto step = [&](int i, auto which) __attribute__((always_inline)) {
            constexpr int buf = decltype(which)::value;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            lds_barrier();  // the tile is there, and all have left the other buffer
            if (i + QT < i1) copy(i + QT, buf ^ 1);
#pragma unroll
            for (int u = 0; u < QT / 32; u++) turn(i + 32 * u, s_q + buf * BUF, u);
        };
        if (i0 < i1) copy(i0, 0);
        for (int i = i0; i < i1; i += 2 * QT) {
            step(i, std::integral_constant<int, 0>{});
            if (i + QT < i1) step(i + QT, std::integral_constant<int, 1>{});
        }
    }
#pragma unroll
    for (int t = 0; t < KB; t++) {
        float all = (sum[t][0] + sum[t][1]) + (sum[t][2] + sum[t][3]);
        all += __shfl_xor(all, 32);
        if (half == 0 && j[t] < int(a.n)) part[(int64_t(slice) * a.kv_heads + hk) * a.n + j[t]] = all;
    }
}

// The slices' sums of every key, in order, to its place.
__global__ __launch_bounds__(256) void prompt_weights_join_kernel(AttentionArgs a, Weights w, int slices, const float *part) {
    __shared__ int32_t s_docs[kFewDocs];
    const int j = int(blockIdx.x * 256 + threadIdx.x), hk = blockIdx.y;
    float sum = 0.f;
    if (j < int(a.n)) {
#pragma unroll 4
        for (int x = 0; x < slices; x++) sum += part[(int64_t(x) * a.kv_heads + hk) * a.n + j];
    }
    const int32_t *const docs = offsets_here(a, s_docs);
    if (j >= int(a.n)) return;
    const QueryRange r = query_range(j, int(a.n), docs, int(a.ndocs), a.prefix, int(w.window));
    if (r.doc < 0 || uint32_t(r.place) >= w.most) return;
    w.p[(int64_t(r.doc) * a.kv_heads + hk) * w.most + r.place] += sum;
}

template <class T, int DP, bool CAPPED> void launch_keys(const AttentionArgs &a, int window, int tiles, int cuts, bool many, float *part, hipStream_t s) {
    const dim3 grid(unsigned(tiles) * a.q_heads * unsigned(cuts));
    if (many && DP <= 128) hipLaunchKernelGGL((prompt_weights_kernel<T, DP, CAPPED, DP <= 128 ? 2 : 1>), grid, dim3(256), 0, s, a, window, tiles, cuts, part);
    else hipLaunchKernelGGL((prompt_weights_kernel<T, DP, CAPPED, 1>), grid, dim3(256), 0, s, a, window, tiles, cuts, part);
}
template <class T, bool CAPPED> void launch_dims(const AttentionArgs &a, int window, int tiles, int cuts, bool many, float *part, hipStream_t s) {
    if (a.dim <= 32) launch_keys<T, 32, CAPPED>(a, window, tiles, cuts, many, part, s);
    else if (a.dim <= 64) launch_keys<T, 64, CAPPED>(a, window, tiles, cuts, many, part, s);
    else if (a.dim <= 96) launch_keys<T, 96, CAPPED>(a, window, tiles, cuts, many, part, s);
    else if (a.dim <= 128) launch_keys<T, 128, CAPPED>(a, window, tiles, cuts, many, part, s);
    else launch_keys<T, 256, CAPPED>(a, window, tiles, cuts, many, part, s);
}

}  // namespace

void launch_attention_weights(Ctx &c, const AttentionArgs &args, const Weights &w, hipStream_t s) {
    AttentionArgs a = args;
    const bool pieces = attention_tiles(a);
    DBuf sums(&c, pieces ? 2 * size_t(a.q_heads) * sums_pitch(a.n) * 4 : size_t(a.n) * a.q_heads * sizeof(float2), s);
    if (pieces) a.sums = sums.as<float>();
    launch_attention(a, s);
    ProbeScope probe("text_weights", s, 2.0 * a.n * a.n * a.q_heads * a.dim, 2.0 * a.n * (a.q_heads + a.kv_heads) * a.dim,
                     pieces ? "text_weights_tiles" : "text_weights_row");
    if (pieces) {
        // The queries cut until every compute unit has two workgroups: 36 documents of up to 130, 4 key heads of 4, 11.0 us with the
        // join; four workgroups 13.2, one 12.1.
        const bool many = a.dim <= 128 && int64_t((a.n + 255) / 256) * a.q_heads >= 512;  // 64 keys a wavefront
        const int keys = many ? 256 : 128, tiles = int((a.n + keys - 1) / keys), group = int(a.q_heads / a.kv_heads);
        const int64_t mine = int64_t(tiles) * a.q_heads, most = (a.n + 255) / 256;
        const int cuts = int(std::max<int64_t>(1, std::min<int64_t>({16, (512 + mine - 1) / mine, most})));
        DBuf part(&c, size_t(group) * cuts * a.kv_heads * a.n * 4, s);
        with_type16(a.type, [&](auto t) {
            if (a.cap > 0.f || a.slopes) launch_dims<decltype(t), true>(a, int(w.window), tiles, cuts, many, part.as<float>(), s);
            else launch_dims<decltype(t), false>(a, int(w.window), tiles, cuts, many, part.as<float>(), s);
        });
        hipLaunchKernelGGL(prompt_weights_join_kernel, dim3((a.n + 255) / 256, a.kv_heads), dim3(256), 0, s, a, w, group * cuts, part.as<float>());
        OCR_HIP(hipGetLastError());
        return;
    }
    with_type16(a.type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((row_sums_kernel<T>), dim3(a.n, a.q_heads), dim3(64), 0, s, a, sums.as<float2>());
        hipLaunchKernelGGL((weights_row_kernel<T>), dim3(a.n, a.kv_heads), dim3(64), 0, s, a, w, sums.as<float2>());
    });
    OCR_HIP(hipGetLastError());
}

void launch_single_weights_row(const DecodeArgs &a, const Weights &w, hipStream_t s) {
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
