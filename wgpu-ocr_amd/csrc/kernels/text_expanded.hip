// Latent attention over a packed row of documents, with keys and values expanded: a key is a head's own part and one
// that all heads share.
//
// The prompt attention's form (text_attn.hip): one pass over the keys with the running maximum and sum of the
// softmax, S^T = K Q^T and O^T = V^T P^T on the matrix cores, a lane's scores going into the second product from the
// registers they are in. Keys' own and shared parts are two tiles in LDS, so no key is put together in memory.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "text_device.h"
#include "text_tile.h"

namespace ocr {

namespace {

// A key of its own part and the part that all heads share.
template <class T> struct SharedKv {
    const T *kp, *rp, *vp;
    int64_t ks, rs, vs;
    int key;
    __device__ float k(int j, int c) const { return to_f32(c < key ? kp[j * ks + c] : rp[j * rs + c - key]); }
    __device__ float v(int j, int c) const { return to_f32(vp[j * vs + c]); }
};

// Token i, head h by one wavefront, by the formula; s_q: kRowFloats floats of the wavefront's own.
constexpr int kRowFloats = 256 + kMostLatentRot;
template <class T> __device__ inline void expanded_row(const LatentAttentionArgs &a, int64_t i, int h, float *s_q) {
    const int width = a.key + a.rot;
    const T *q = static_cast<const T *>(a.q) + i * a.q_stride + int64_t(h) * width;
    for (int c = threadIdx.x & 63; c < width; c += 64) s_q[c] = to_f32(q[c]) * a.scale;
    __builtin_amdgcn_wave_barrier();
    const KeyRange r = key_range(int(i), int(a.n), a.docs, int(a.ndocs), a.prefix);
    const SharedKv<T> kv{static_cast<const T *>(a.k) + h * a.k_head, static_cast<const T *>(a.r), static_cast<const T *>(a.v) + h * a.v_head,
                         a.k_stride, a.r_stride, a.v_stride, int(a.key)};
    T *out = static_cast<T *>(a.out) + i * a.out_stride + int64_t(h) * a.value;
    attend_row(kv, s_q, width, r.lo, r.hi, int(i), 0.f, 0.f, [&](int c, float o) { out[c] = T(o); }, int(a.value));
    __builtin_amdgcn_wave_barrier();
}

// Sizes that the tiles do not take.
template <class T> __global__ __launch_bounds__(64) void expanded_row_kernel(LatentAttentionArgs a) {
    __shared__ float s_q[kRowFloats];
    expanded_row<T>(a, blockIdx.x, blockIdx.y, s_q);
}

// 32 queries of one head a wavefront over tiles of 64 keys that come into LDS by DMA while the tile before is worked
// on. DK, DR, DV: the key's own and shared values and the value's, rounded up. QW: of the four wavefronts, those with queries of
// their own; where it is two, the other two take the same queries over the other half of each tile's keys.
// Two documents of up to 5000, 32 heads of 128 + 64 and 128, bf16 (292 GFLOP): 329 to 343 us, 850 to 890 TFLOP/s, where a large product
// reaches 1213: matrix cores and exponentials take turns. 36 documents of up to 130, 12 heads of 64 + 32: 11 us, half of it before the first products.
template <class T, int DK, int DR, int DV, int QW> __global__ __launch_bounds__(256, 2) void expanded_tile_kernel(LatentAttentionArgs a, int tiles) {
    typedef T tvec __attribute__((ext_vector_type(8)));
    constexpr int KT = 64, KB = KT / 32 * QW / 4;
    constexpr int KS = DK / 16, RS = DR / 16, NB = DV / 32;
    using TK = Tile<DK, KT>;
    using TR = Tile<64, KT>;
    using TV = Tile<DV, KT>;
    constexpr int BUF = TK::BYTES + TR::BYTES + TV::BYTES;  // the widest: 40 KB, two workgroups fill a compute unit's LDS
    __shared__ __align__(16) char s_kv[2 * BUF];
    int *const s_lo = reinterpret_cast<int *>(s_kv), *const s_hi = s_lo + 4;  // before the first copies
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int qw = wave % QW, part = wave / QW * KB * 32;
    const HeadTile w = head_tile(blockIdx.x, tiles, a.heads, a.heads, 32);
    if (w.head < 0) return;
    const int h = w.head, key = a.key, rot = a.rot, value = a.value, width = key + rot;
    const int i = w.tile * (32 * QW) + 32 * qw + (lane & 31);
    const KeyRange r = key_range(i, int(a.n), a.docs, int(a.ndocs), a.prefix);
    const bool sees = r.lo < r.hi;
    const int wlo = wave_min_i(sees ? r.lo : 0x7fffffff), whi = wave_max_i(sees ? r.hi : 0);
    const int flo = wave_max_i(sees ? r.lo : 0), fhi = wave_min_i(sees ? r.hi : 0x7fffffff);
    if (lane == 0) s_lo[wave] = wlo, s_hi[wave] = whi;

    tvec qf[KS + RS];
    {
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0;
        const char *q = static_cast<const char *>(a.q) + (int64_t(min(i, int(a.n) - 1)) * a.q_stride + int64_t(h) * width) * 2;
#pragma unroll
        for (int s = 0; s < KS + RS; s++) {
            const int c = s < KS ? 2 * s + half : 2 * (s - KS) + half, first = s < KS ? 0 : key / 8, count = (s < KS ? key : rot) / 8;
            u32x4 x{0, 0, 0, 0};
            if (c < count) x = *reinterpret_cast<const u32x4 *>(q + 16 * (first + c));
            qf[s] = __builtin_bit_cast(tvec, x ^ flip);
        }
    }
    __syncthreads();
    int jlo = s_lo[0], jhi = s_hi[0];
#pragma unroll
    for (int x = 1; x < 4; x++) jlo = min(jlo, s_lo[x]), jhi = max(jhi, s_hi[x]);
    jlo = __builtin_amdgcn_readfirstlane(jlo), jhi = __builtin_amdgcn_readfirstlane(jhi);
    if (jlo >= jhi) jlo = jhi = 0;  // nothing is seen
    __syncthreads();
    const TK tk(a.k_stride, key / 8);
    const TR tr(a.r_stride, rot / 8);
    const TV tv(a.v_stride, value / 8);
    if (tk.pieces < TK::PP || tr.pieces < TR::PP || tv.pieces < TV::PP) {  // pieces that no copy writes count nothing
        for (int x = tid; x < 2 * BUF / 16; x += 256) *reinterpret_cast<u32x4 *>(s_kv + 16 * x) = u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    const char *kbase = static_cast<const char *>(a.k) + int64_t(h) * a.k_head * 2, *rbase = static_cast<const char *>(a.r);
    const char *vbase = static_cast<const char *>(a.v) + int64_t(h) * a.v_head * 2;
    const unsigned lds0 = lds_addr(s_kv) + wave * 1024;
    auto copy = [&](int j0, int buf) {
        const unsigned to = lds0 + buf * BUF;
        tk.copy(kbase + int64_t(j0) * tk.step, to, jhi - j0);
        tr.copy(rbase + int64_t(j0) * tr.step, to + TK::BYTES, jhi - j0);
        tv.copy(vbase + int64_t(j0) * tv.step, to + TK::BYTES + TR::BYTES, jhi - j0);
    };
    int koff[KS], roff[RS], voff[NB][2];
#pragma unroll
    for (int s = 0; s < KS; s++) koff[s] = (lane & 31) * DK * 2 + ((2 * s + half) ^ TK::swap_of(lane & 15)) * 16;
#pragma unroll
    for (int s = 0; s < RS; s++) roff[s] = TK::BYTES + (lane & 31) * 128 + ((2 * s + half) ^ TR::swap_of(lane & 15)) * 16;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int row = 4 * half + ((lane & 15) >> 2) + 8 * e;
            voff[b][e] = TK::BYTES + TR::BYTES + row * DV * 2 + ((4 * b + 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ TV::swap_of(row)) * 16 + 8 * (lane & 1);
        }

    f32x16 o[NB];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[b][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);  // not 0: masked scores stay minus infinity

    // Every product's LDS read is asked for four products before it, in an order that is kept: left to itself the compiler reads,
    // waits and multiplies one after another (364 us where this takes 341, two ahead 343).
    constexpr int kAhead = 4;
    // 32 KB keys from jw on; s: the buffer, at the wavefront's part of it.
    auto turn = [&](int jw, const char *s_b) __attribute__((always_inline)) {
        if (jw >= whi || jw + 32 * KB <= wlo) return;
        f32x16 s[KB];
#pragma unroll
        for (int t = 0; t < KB; t++) {
#pragma unroll
            for (int e = 0; e < 16; e++) s[t][e] = 0.f;
        }
        auto key_read = [&](int x) __attribute__((always_inline)) {
            const int t = x / (KS + RS), st = x % (KS + RS);
            return *reinterpret_cast<const tvec *>(st < KS ? s_b + koff[st < KS ? st : 0] + (part + t * 32) * DK * 2 : s_b + roff[st < KS ? 0 : st - KS] + (part + t * 32) * 128);
        };
        {
            tvec k[kAhead];
#pragma unroll
            for (int x = 0; x < kAhead; x++) k[x] = key_read(x);
#pragma unroll
            for (int x = 0; x < KB * (KS + RS); x++) {
                s[x / (KS + RS)] = mfma32(k[x % kAhead], qf[x % (KS + RS)], s[x / (KS + RS)]);
                if (x + kAhead < KB * (KS + RS)) k[x % kAhead] = key_read(x + kAhead);
                __builtin_amdgcn_sched_barrier(0);
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
        top *= c;
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
                const float x = exp2_f32(__fmaf_rn(s[t][e], c, -ref));
                l += x;
                p[t][e / 8][e % 8] = T(x);
            }
        auto value_read = [&](int x) __attribute__((always_inline)) {
            const int t = x / (2 * NB), u = x / NB % 2, b = x % NB;
            const u32x2 y = lds_read_tr16(s_b + voff[b][0] + (part + 32 * t + 16 * u) * DV * 2);
            const u32x2 z = lds_read_tr16(s_b + voff[b][1] + (part + 32 * t + 16 * u) * DV * 2);
            return __builtin_bit_cast(tvec, u32x4{y[0], y[1], z[0], z[1]});
        };
        tvec v[kAhead];
#pragma unroll
        for (int x = 0; x < kAhead; x++) v[x] = value_read(x);
#pragma unroll
        for (int x = 0; x < KB * 2 * NB; x++) {
            o[x % NB] = mfma32(v[x % kAhead], p[x / (2 * NB)][x / NB % 2], o[x % NB]);
            if (x + kAhead < KB * 2 * NB) v[x % kAhead] = value_read(x + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto step = [&](int j0, auto which) __attribute__((always_inline)) {
        constexpr int buf = decltype(which)::value;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();  // the tile is there, and all have left the other buffer
        if (j0 + KT < jhi) copy(j0 + KT, buf ^ 1);
        turn(j0 + part, s_kv + buf * BUF);
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
        float *const s_o = reinterpret_cast<float *>(s_kv) + qw * 64 * (16 * NB + 2) + lane;
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
    // A value that is not finite spoils the sums of every query of its tile, also where the mask gives it no weight:
    // those queries again, by the formula.
    float bad = 0.f;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) bad += o[b][e] * 0.f;
    const unsigned long long spoilt = wave < QW ? __ballot(sees && !(bad == 0.f)) : 0;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (wave < QW && i < int(a.n) && !((spoilt >> (lane & 31) | spoilt >> ((lane & 31) + 32)) & 1)) {
        T *out = static_cast<T *>(a.out) + int64_t(i) * a.out_stride + int64_t(h) * value;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int col = 32 * b + 2 * e + 4 * half;
                typedef T t4 __attribute__((ext_vector_type(4)));
                if (col < value)
                    *reinterpret_cast<t4 *>(out + col) = sees ? t4{T(o[b][e] * inv), T(o[b][e + 1] * inv), T(o[b][e + 2] * inv), T(o[b][e + 3] * inv)}
                                                              : t4{T(0.f), T(0.f), T(0.f), T(0.f)};
            }
    }
    __syncthreads();
    for (unsigned todo = unsigned(spoilt | spoilt >> 32); todo; todo &= todo - 1)
        expanded_row<T>(a, w.tile * (32 * QW) + 32 * qw + __builtin_ctz(todo), h, reinterpret_cast<float *>(s_kv) + kRowFloats * wave);
}

template <class T, int DK, int DR, int DV, int QW> void launch_tiles(const LatentAttentionArgs &a, hipStream_t s) {
    const int tiles = int((a.n + 32 * QW - 1) / (32 * QW));
    hipLaunchKernelGGL((expanded_tile_kernel<T, DK, DR, DV, QW>), dim3(unsigned(head_blocks(tiles, a.heads, a.heads))), dim3(256), 0, s, a, tiles);
}
// Tiles of 64 queries while those of 128 would leave compute units empty.
template <class T, int DK, int DR, int DV> void launch_queries(const LatentAttentionArgs &a, bool few, hipStream_t s) {
    few ? launch_tiles<T, DK, DR, DV, 2>(a, s) : launch_tiles<T, DK, DR, DV, 4>(a, s);
}
template <class T, int DK, int DR> void launch_values(const LatentAttentionArgs &a, bool few, hipStream_t s) {
    a.value <= 64 ? launch_queries<T, DK, DR, 64>(a, few, s) : launch_queries<T, DK, DR, 128>(a, few, s);
}
template <class T, int DK> void launch_keys(const LatentAttentionArgs &a, bool few, hipStream_t s) {
    a.rot <= 32 ? launch_values<T, DK, 32>(a, few, s) : launch_values<T, DK, 64>(a, few, s);
}

}  // namespace

void launch_latent_attention(const LatentAttentionArgs &a, hipStream_t s) {
    const double n = a.n;
    // Whole 16-byte pieces, and rows of a tile within 32 bits of each other.
    bool pieces = a.key <= 128 && a.rot <= 64 && a.value <= 128 && (a.key | a.rot | a.value) % 8 == 0 &&
                  head_blocks((a.n + 63) / 64, a.heads, a.heads) < 1 << 24;
    for (const void *p : {a.q, a.k, a.r, a.v, static_cast<const void *>(a.out)}) pieces = pieces && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int64_t st : {a.q_stride, a.k_stride, a.k_head, a.rot ? a.r_stride : 0, a.v_stride, a.v_head, a.out_stride}) pieces = pieces && st % 8 == 0 && st < 1 << 24;
    // Until every compute unit has a workgroup of 128 queries, 64 a workgroup: 36 documents of up to 130 11.6 us and 12.1, two of up
    // to 5000 425 and 375.
    const bool few = int64_t((a.n + 127) / 128) * a.heads <= 256;
    ProbeScope probe("latent_attention", s, n * n * a.heads * (a.key + a.rot + a.value), 4.0 * n * a.heads * (a.key + a.value),
                     !pieces ? "latent_attention_row" : few ? "latent_attention_64" : "latent_attention_128");
    with_type16(a.type, [&](auto t) {
        using T = decltype(t);
        if (!pieces) hipLaunchKernelGGL((expanded_row_kernel<T>), dim3(a.n, a.heads), dim3(64), 0, s, a);
        else a.key <= 64 ? launch_keys<T, 64>(a, few, s) : launch_keys<T, 128>(a, few, s);
    });
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
