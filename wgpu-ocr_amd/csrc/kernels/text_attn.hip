// Attention over a packed row of documents: scores capped by a tanh, a bias that falls with the
// distance, document and prefix masks.
//
// One pass over the keys with the running maximum and sum of the softmax. Both products have the
// keys as rows: S^T = K Q^T, O^T = V^T P^T, so that a lane holds all of its share of a query's
// scores and hands them to the second product from the registers they are in: of 32 x 32 results, lane
// l has column l % 32 and rows 8 i + 4 (l / 32) + 0 .. 3, and as the second product's 16 keys a step it
// gives rows 8 i .. 8 i + 15 in that order, which the value side follows. Values come transposed out
// of LDS by its transposing reads.
//
// Two documents of 5000 and less, 32 heads of 128, causal: 250 us, 940 TFLOP/s (the library's large
// product 1226): the matrix cores are busy 48 % of the clock's cycles (1.9 GHz under this load; 38 % of 2.4)
// and vector instructions take 25 % of the wavefronts' time, at two wavefronts a SIMD. Tried and no faster: the next tile's first product among this one's
// exponentials (260), eight wavefronts over tiles of 128 keys (249), priorities by phase or wavefront
// (250 to 256), the weights' sums by dot products (257).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "lds_dma.h"
#include "text_device.h"

namespace ocr {

namespace {

template <class T> struct DenseKv {
    const T *kp, *vp;
    int64_t ks, vs;
    __device__ float k(int j, int c) const { return to_f32(kp[j * ks + c]); }
    __device__ float v(int j, int c) const { return to_f32(vp[j * vs + c]); }
};

// Token i, head h by one wavefront, by the formula; s_q: 256 floats of the wavefront's own.
template <class T> __device__ inline void attention_row(const AttentionArgs &a, int64_t i, int h, float *s_q) {
    const int dim = a.dim, hk = h / int(a.q_heads / a.kv_heads);
    const T *q = static_cast<const T *>(a.q) + i * a.q_stride + int64_t(h) * dim;
    for (int c = threadIdx.x & 63; c < dim; c += 64) s_q[c] = to_f32(q[c]) * a.scale;
    __builtin_amdgcn_wave_barrier();
    const KeyRange r = key_range(int(i), int(a.n), a.docs, int(a.ndocs), a.prefix);
    const DenseKv<T> kv{static_cast<const T *>(a.k) + int64_t(hk) * dim, static_cast<const T *>(a.v) + int64_t(hk) * dim, a.k_stride, a.v_stride};
    T *out = static_cast<T *>(a.out) + i * a.out_stride + int64_t(h) * dim;
    attend_row(kv, s_q, dim, r.lo, r.hi, int(i), a.cap, a.slopes ? a.slopes[h] : 0.f, [&](int c, float o) { out[c] = T(o); });
    __builtin_amdgcn_wave_barrier();
}

// Vectors that do not lie on 16-byte pieces. 109 tokens, 8 heads of 64: 35 us (tiles: 6); 2929, 16 of
// 128: 14 ms (66 us).
template <class T> __global__ __launch_bounds__(64) void attention_row_kernel(AttentionArgs a) {
    __shared__ float s_q[256];
    attention_row<T>(a, blockIdx.x, blockIdx.y, s_q);
}

// What scores go through besides the scale: nothing, a fine cap, the distance's bias and perhaps a fine cap, or any cap
// and perhaps the bias.
//
// A tile with a score past 0.35 of the cap takes the exponential's form, for all of its scores where the cap
// is fine (kFineCap). Score by score it costs more: a page of 2929 tokens with scores past the cap: 104 us, so 135.
enum Scores { kPlain, kCapped, kBias, kAny };

// cap tanh(s / cap) of unscaled scores as s times a polynomial of their squares (tanh_ratio, its powers
// of scale / cap in the factors), which lasts to 0.35 of the cap. In units of log2; the exponential's and the reciprocal's way takes half again as long.
struct SmallCap {
    float k[4], most;
    __device__ SmallCap(float scale, float cap) {
        const float y = scale / cap, t = y * y;
        k[0] = scale * 1.4426950408889634f;
        float power = k[0];
#pragma unroll
        for (int e = 1; e < 4; e++) power *= t, k[e] = kTanhPart[e] * power;
        // Where the powers leave float32: as far as those that are left reach (the fourth power's part under 2^-25 of
        // the score, the square's), and no score's square is infinite.
        most = y >= 1e3f ? -1.f : fabsf(k[3]) >= 1e-36f ? kSmallTanh / y : fminf((fabsf(k[1]) >= 1e-36f ? 0.02f : 3e-4f) / y, 1e18f);
    }
    __device__ float factor(float s) const {
        const float t = s * s;
        return __fmaf_rn(__fmaf_rn(__fmaf_rn(k[3], t, k[2]), t, k[1]), t, k[0]);
    }
};

// 32 queries of one head a wavefront over tiles of KT keys that come into LDS by DMA while the tile
// before is worked on. DP: the head's values rounded up to 32. QW: of the four wavefronts, those with
// queries of their own; where it is two, the other two take the same queries over the other half of
// each tile's keys, and their sums are joined at the end.
template <class T, int DP, Scores KIND, int QW> __global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void attention_tile_kernel(AttentionArgs a, int tiles) {
    typedef T tvec __attribute__((ext_vector_type(8)));
    constexpr int PW = DP <= 64 ? 64 : DP <= 128 ? 128 : 256;  // a vector's values in LDS
    constexpr int PP = PW / 8;                                 // its 16-byte pieces
    constexpr int KT = PW == 256 ? 32 : 64, KB = KT / 32 * QW / 4;  // a tile's keys, blocks of 32 of a wavefront's part
    static_assert(KB >= 1, "a wavefront's part of a tile");
    constexpr int KS = DP / 16, NB = DP / 32;
    constexpr int TILE = KT * PW * 2;
    constexpr int ND = KT * PP / 256;  // copies a lane for a tile's keys
    __shared__ __align__(16) char s_kv[2][2][TILE];
    __shared__ int s_lo[4], s_hi[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int qw = wave % QW, part = wave / QW * KB * 32;  // its queries, the first of its keys of a tile
    const HeadTile w = head_tile(blockIdx.x, tiles, a.q_heads, a.kv_heads, PW == 128 ? 32 : 0);
    if (w.head < 0) return;
    const int h = w.head, hk = h / int(a.q_heads / a.kv_heads), dim = a.dim;
    const int i = w.tile * (32 * QW) + 32 * qw + (lane & 31);
    const KeyRange r = key_range(i, int(a.n), a.docs, int(a.ndocs), a.prefix);
    const bool sees = r.lo < r.hi;
    // The wavefront's keys: some query sees those in [wlo, whi), all do those in [flo, fhi).
    const int wlo = wave_min_i(sees ? r.lo : 0x7fffffff), whi = wave_max_i(sees ? r.hi : 0);
    const int flo = wave_max_i(sees ? r.lo : 0), fhi = wave_min_i(sees ? r.hi : 0x7fffffff);
    if (lane == 0) s_lo[wave] = wlo, s_hi[wave] = whi;

    const int pieces = dim / 8;
    tvec qf[KS];
    {
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0;
        const char *q = static_cast<const char *>(a.q) + (int64_t(min(i, int(a.n) - 1)) * a.q_stride + int64_t(h) * dim) * 2;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            u32x4 x{0, 0, 0, 0};
            if (2 * s + half < pieces) x = *reinterpret_cast<const u32x4 *>(q + 16 * (2 * s + half));
            qf[s] = __builtin_bit_cast(tvec, x ^ flip);
        }
    }
    if (pieces < PP) {  // pieces that no copy writes count nothing
        for (int x = tid; x < 4 * KT * PP; x += 256) *reinterpret_cast<u32x4 *>(&s_kv[0][0][0] + 16 * x) = u32x4{0, 0, 0, 0};
    }
    __syncthreads();
    int jlo = s_lo[0], jhi = s_hi[0];
#pragma unroll
    for (int x = 1; x < 4; x++) jlo = min(jlo, s_lo[x]), jhi = max(jhi, s_hi[x]);
    jlo = __builtin_amdgcn_readfirstlane(jlo), jhi = __builtin_amdgcn_readfirstlane(jhi);
    if (jlo >= jhi) jlo = jhi = 0;  // nothing is seen: jlo is the largest int, and tiles on from it none

    // Copies: a lane's pieces of a tile lie in LDS in order, each row's exchanged so that the reads
    // below touch every bank (swap_of), by the choice of the piece that the lane copies.
    auto swap_of = [](int row) { return PP == 8 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3); };
    const char *kbase = static_cast<const char *>(a.k) + (int64_t(jlo) * a.k_stride + int64_t(hk) * dim) * 2;
    const char *vbase = static_cast<const char *>(a.v) + (int64_t(jlo) * a.v_stride + int64_t(hk) * dim) * 2;
    const unsigned lds0 = lds_addr(&s_kv[0][0][0]) + wave * 1024;
    const unsigned kstep = unsigned(a.k_stride * 2), vstep = unsigned(a.v_stride * 2);
    auto row_of = [&](int d) { return ((4 * d + wave) * 64 + lane) / PP; };
    auto piece_of = [&](int d) { return ((4 * d + wave) * 64 + lane) % PP ^ swap_of(row_of(d)); };
    unsigned kat[ND], vat[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) kat[d] = row_of(d) * kstep + 16 * piece_of(d), vat[d] = row_of(d) * vstep + 16 * piece_of(d);
    auto copy = [&](int j0, int buf) {
        const char *kb = kbase + int64_t(j0 - jlo) * kstep, *vb = vbase + int64_t(j0 - jlo) * vstep;
        const unsigned to = lds0 + buf * 2 * TILE;
        if (j0 + KT <= jhi && pieces == PP) {
#pragma unroll
            for (int d = 0; d < ND; d++) {
                dma16s_to(kb, kat[d], to + d * 4096);
                dma16s_to(vb, vat[d], to + TILE + d * 4096);
            }
            return;
        }
#pragma unroll
        for (int d = 0; d < ND; d++) {  // past the last row: that again
            const unsigned over = unsigned(max(0, row_of(d) - (jhi - 1 - j0)));
            if (piece_of(d) < pieces) {
                dma16s_to(kb, kat[d] - over * kstep, to + d * 4096);
                dma16s_to(vb, vat[d] - over * vstep, to + TILE + d * 4096);
            }
        }
    };
    int koff[KS], voff[NB][2];
#pragma unroll
    for (int s = 0; s < KS; s++) koff[s] = (lane & 31) * PW * 2 + ((2 * s + half) ^ swap_of(lane & 15)) * 16;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int row = 4 * half + ((lane & 15) >> 2) + 8 * e;
            voff[b][e] = row * PW * 2 + ((4 * b + 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ swap_of(row)) * 16 + 8 * (lane & 1);
        }

    f32x16 o[NB];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[b][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);  // not 0: masked scores stay minus infinity
    const float slope = KIND >= kBias && a.slopes ? a.slopes[h] * 1.4426950408889634f : 0.f;

    const SmallCap small(fabsf(a.scale), KIND != kPlain && a.cap > 0.f ? a.cap : 1.f);
    const Cap cap = cap_of(a.cap, 1.4426950408889634f);

    // 32 KB keys from jw on, in LDS at sk, and their values at sv.
    auto turn = [&](int jw, const char *sk, const char *sv) __attribute__((always_inline)) {
        if (jw >= whi || jw + 32 * KB <= wlo) return;
        f32x16 s[KB];
#pragma unroll
        for (int t = 0; t < KB; t++) {
#pragma unroll
            for (int e = 0; e < 16; e++) s[t][e] = 0.f;
#pragma unroll
            for (int st = 0; st < KS; st++)
                s[t] = mfma32(*reinterpret_cast<const tvec *>(sk + koff[st] + t * 32 * PW * 2), qf[st], s[t]);
        }
        // Scores in units of log2 over `unit`, in place.
        constexpr bool scaled_later = KIND == kPlain;
        const float unit = scaled_later ? c : 1.f;
        if (!scaled_later) {
            float top = 0.f;
            if (a.cap > 0.f) {
#pragma unroll
                for (int t = 0; t < KB; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(s[t][e]));
            }
            if (a.cap > 0.f && __any(top > small.most)) {
#pragma unroll
                for (int t = 0; t < KB; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[t][e] = KIND == kAny ? capped(cap, s[t][e] * c) : large_capped(cap, s[t][e] * c);
            } else if (a.cap > 0.f) {
#pragma unroll
                for (int t = 0; t < KB; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[t][e] *= small.factor(s[t][e]);
            } else {
#pragma unroll
                for (int t = 0; t < KB; t++) s[t] *= c;
            }
            if (KIND == kBias || (KIND == kAny && a.slopes)) {
                const float d = float(i - jw - 4 * half);
#pragma unroll
                for (int t = 0; t < KB; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[t][e] -= slope * fabsf(d - float(32 * t + 8 * (e / 4) + e % 4));
            }
        }
        if (jw < flo || jw + 32 * KB > fhi) {
            const unsigned first = unsigned(jw + 4 * half - r.lo), count = unsigned(r.hi - r.lo);
#pragma unroll
            for (int t = 0; t < KB; t++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (first + unsigned(32 * t + 8 * (e / 4) + e % 4) >= count) s[t][e] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int t = 0; t < KB; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, s[t][e]);
        top *= unit;
        if (__any(top > m + kSlack)) {
            const float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32))), f = mn == -INFINITY ? 1.f : exp2_f32(m - mn);
            l *= f;
#pragma unroll
            for (int b = 0; b < NB; b++) o[b] *= f;
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.f : m - lift<T>;
        tvec p[KB][2];
#pragma unroll
        for (int t = 0; t < KB; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float x = exp2_f32(scaled_later ? __fmaf_rn(s[t][e], unit, -ref) : s[t][e] - ref);
                l += x;
                p[t][e / 8][e % 8] = T(x);
            }
#pragma unroll
        for (int t = 0; t < KB; t++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const u32x2 x = lds_read_tr16(sv + voff[b][0] + (32 * t + 16 * u) * PW * 2);
                    const u32x2 y = lds_read_tr16(sv + voff[b][1] + (32 * t + 16 * u) * PW * 2);
                    o[b] = mfma32(__builtin_bit_cast(tvec, u32x4{x[0], x[1], y[0], y[1]}), p[t][u], o[b]);
                }
    };
    auto step = [&](int j0, auto which) __attribute__((always_inline)) {
        constexpr int buf = decltype(which)::value;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();  // the tile is there, and all have left the other buffer
        if (j0 + KT < jhi) copy(j0 + KT, buf ^ 1);
        turn(j0 + part, s_kv[buf][0] + part * PW * 2, s_kv[buf][1] + part * PW * 2);
    };
    if (jlo < jhi) copy(jlo, 0);
    for (int j0 = jlo; j0 < jhi; j0 += 2 * KT) {
        step(j0, std::integral_constant<int, 0>{});
        if (j0 + KT < jhi) step(j0 + KT, std::integral_constant<int, 1>{});
    }
    l += __shfl_xor(l, 32);
    if constexpr (QW < 4) {
        static_assert(2 * 64 * (16 * NB + 2) * 4 <= int(sizeof(s_kv)), "the sums' way");
        __syncthreads();
        float *const s_o = reinterpret_cast<float *>(&s_kv[0][0][0]) + qw * 64 * (16 * NB + 2) + lane;
        if (wave >= QW) {
#pragma unroll
            for (int e = 0; e < 16 * NB; e++) s_o[64 * e] = o[e / 16][e % 16];
            s_o[64 * 16 * NB] = m, s_o[64 * (16 * NB + 1)] = l;
        }
        __syncthreads();
        if (wave < QW) {
            const float m2 = s_o[64 * 16 * NB], l2 = s_o[64 * (16 * NB + 1)], mn = fmaxf(m, m2);
            const float f = mn == -INFINITY ? 1.f : exp2_f32(m - mn), f2 = mn == -INFINITY ? 1.f : exp2_f32(m2 - mn);
            l = l * f + l2 * f2;
#pragma unroll
            for (int e = 0; e < 16 * NB; e++) o[e / 16][e % 16] = o[e / 16][e % 16] * f + s_o[64 * e] * f2;
        }
    }
    // A value that is not finite spoils the sums of every query of its tile, also where the mask
    // gives it no weight: those queries again, by the formula.
    float bad = 0.f;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) bad += o[b][e] * 0.f;
    const unsigned long long spoilt = wave < QW ? __ballot(sees && !(bad == 0.f)) : 0;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (wave < QW && i < int(a.n) && !((spoilt >> (lane & 31) | spoilt >> ((lane & 31) + 32)) & 1)) {
        T *out = static_cast<T *>(a.out) + int64_t(i) * a.out_stride + int64_t(h) * dim;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int col = 32 * b + 2 * e + 4 * half;
                typedef T t4 __attribute__((ext_vector_type(4)));
                if (col < dim)
                    *reinterpret_cast<t4 *>(out + col) = sees ? t4{T(o[b][e] * inv), T(o[b][e + 1] * inv), T(o[b][e + 2] * inv), T(o[b][e + 3] * inv)}
                                                              : t4{T(0.f), T(0.f), T(0.f), T(0.f)};
            }
    }
    __syncthreads();
    for (unsigned todo = unsigned(spoilt | spoilt >> 32); todo; todo &= todo - 1)
        attention_row<T>(a, w.tile * (32 * QW) + 32 * qw + __builtin_ctz(todo), h, reinterpret_cast<float *>(&s_kv[0][0][0]) + 256 * wave);
}

template <class T, int DP, Scores KIND, int QW> void launch_tiles(const AttentionArgs &a, hipStream_t s) {
    const int tiles = int((a.n + 32 * QW - 1) / (32 * QW));
    hipLaunchKernelGGL((attention_tile_kernel<T, DP, KIND, QW>), dim3(unsigned(head_blocks(tiles, a.q_heads, a.kv_heads))), dim3(256), 0, s, a, tiles);
}
// Tiles of 64 queries while those of 128 would leave compute units empty, but they bring every key
// from level two twice as often. 36 documents of up to 130 tokens, 16 heads of 64 (336 tiles of
// 128; four workgroups of it fit a compute unit): 11.9 us with 64 queries, 12.9 with 128; one of
// 2929, 16 heads of 128 (368 tiles; two fit): 103 and 87 us.
bool few_tiles(const AttentionArgs &a) {
    return a.dim <= 128 && int64_t((a.n + 127) / 128) * a.q_heads <= (a.dim <= 64 ? 768 : 256);
}
template <class T, Scores KIND> void launch_dims(const AttentionArgs &a, bool few, hipStream_t s) {
    if (a.dim <= 32) few ? launch_tiles<T, 32, KIND, 2>(a, s) : launch_tiles<T, 32, KIND, 4>(a, s);
    else if (a.dim <= 64) few ? launch_tiles<T, 64, KIND, 2>(a, s) : launch_tiles<T, 64, KIND, 4>(a, s);
    else if (a.dim <= 96) few ? launch_tiles<T, 96, KIND, 2>(a, s) : launch_tiles<T, 96, KIND, 4>(a, s);
    else if (a.dim <= 128) few ? launch_tiles<T, 128, KIND, 2>(a, s) : launch_tiles<T, 128, KIND, 4>(a, s);
    else launch_tiles<T, 256, KIND, 4>(a, s);
}

}  // namespace

void launch_attention(const AttentionArgs &a, hipStream_t s) {
    // Whole 16-byte pieces, and rows of a tile within 32 bits of each other.
    bool pieces = a.dim % 8 == 0 && head_blocks((a.n + 63) / 64, a.q_heads, a.kv_heads) < 1 << 24;
    for (const void *p : {a.q, a.k, a.v, static_cast<const void *>(a.out)}) pieces = pieces && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int64_t st : {a.q_stride, a.k_stride, a.v_stride, a.out_stride}) pieces = pieces && st % 8 == 0 && st < 1 << 24;
    const bool few = few_tiles(a);
    ProbeScope probe("text_attention", s, 2.0 * a.n * a.n * a.q_heads * a.dim, 4.0 * a.n * (a.q_heads + a.kv_heads) * a.dim,
                     !pieces ? "text_attention_row" : few ? "text_attention_64" : "text_attention_128");
    with_type16(a.type, [&](auto t) {
        using T = decltype(t);
        if (!pieces) hipLaunchKernelGGL((attention_row_kernel<T>), dim3(a.n, a.q_heads), dim3(64), 0, s, a);
        else if (cap_of(a.cap, 1.4426950408889634f).most > kFineCap) launch_dims<T, kAny>(a, few, s);
        else if (a.slopes) launch_dims<T, kBias>(a, few, s);
        else if (a.cap > 0.f) launch_dims<T, kCapped>(a, few, s);
        else launch_dims<T, kPlain>(a, few, s);
    });
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
