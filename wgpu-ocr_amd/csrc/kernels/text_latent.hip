// Latent attention over the paged cache of latent vectors: their writing, and single tokens' attention.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "lds_dma.h"
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

// Which tiles of which sequences are whose: lens scanned 64 sequences at a time by every wavefront.
struct LatentPlan {
    int runs;    // workgroups that share the tiles
    int groups;  // of 16 heads
};
// f(first sequence of a 64, its lane's tiles, tiles before the lane's sequence) until it answers true; the tiles of all.
template <class F> __device__ inline int64_t scan_tiles(const LatentDecodeArgs &a, F &&f) {
    const int lane = threadIdx.x & 63;
    int64_t before = 0;
    for (uint32_t r0 = 0; r0 < a.table.rows; r0 += 64) {
        const int mine = r0 + lane < a.table.rows ? latent_tiles(clamp_len(a.lens[r0 + lane], a.table.width, a.c.page)) : 0;
        int64_t upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int64_t x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        if (f(r0, mine, before + upto - mine)) break;
        before += __shfl(upto, 63);
    }
    return before;
}

// 16 heads a wavefront, HB wavefronts over the same tiles of 32 positions, whose vectors come into LDS by DMA, SLOTS - 1
// tiles ahead. RC: the rank rounded up (the rotated part to 64). Each run of tiles goes through its sequences one after another.
//
// S^T = C Q^T, O^T = C^T P^T: the vectors are keys, row by row, and values, through the transposing reads, from one
// copy in LDS. A row's pieces are exchanged so that the reads of 16 rows touch every bank.
template <class T, int RC, int HB, int SLOTS> __global__ __launch_bounds__(64 * HB, HB < 4 ? 1 : 2) void latent_tile_kernel(LatentDecodeArgs a, LatentPlan plan, float *part) {
    typedef T tvec __attribute__((ext_vector_type(8)));
    constexpr int DP = RC + 64, PP = DP / 8, PB = DP * 2, TILE = kLatentTile * PB;
    constexpr int NS = DP / 32, NB = RC / 16;
    constexpr int PER = PP / 8;  // copies of a wavefront for eight rows
    constexpr int CH = HB == 8 ? 1024 : 512;  // positions looked up at a time
    __shared__ __align__(16) char s_c[SLOTS * TILE];
    __shared__ int64_t s_at[CH];  // a position's vector in the pool, in bytes; negative: none
    __shared__ int s_gaps;        // whether some of them are none
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g4 = lane >> 4;
    const int rank = a.c.rank, width = rank + int(a.c.rot), pieces = width / 8;
    const int h = (int(blockIdx.y) * HB + wave) * 16 + n;
    const bool real = h < int(a.heads);
    const int64_t total = scan_tiles(a, [](uint32_t, int, int64_t) { return false; });
    const int64_t each = latent_run(total, plan.runs), g = blockIdx.x;
    int64_t x = g * each;
    const int64_t x1 = min(total, x + each);
    if (x >= x1) return;
    // The sequence of tile x, and its own first tile.
    int64_t r = 0, start = 0;
    scan_tiles(a, [&](uint32_t r0, int mine, int64_t before) {
        const unsigned long long here = __ballot(before <= x && x < before + mine);
        if (!here) return false;
        const int at = __builtin_ctzll(here);
        r = r0 + at, start = __shfl(before, at);
        return true;
    });

    const unsigned lds0 = lds_addr(s_c);
    // Eight rows' (group 0 .. 3) copy k of the tile at position t0 of the lookup.
    auto copy_one = [&](int t0, int slot, int group, int k, int from) __attribute__((always_inline)) {
        const int row = (64 * k + from) / PP, piece = (64 * k + from) % PP ^ (row >> 1);
        int64_t at = s_at[t0 + 8 * group + row];
        at = at < 0 ? 0 : at;
        const int p = min(piece ^ (group & 1) * 4, pieces - 1);
        dma16_to(static_cast<const char *>(a.c.p) + at + 16 * p, lds0 + slot * TILE + group * 8 * PB + k * 1024);
    };
    auto copy = [&](int t0, int slot) __attribute__((always_inline)) {
        int from = lane;  // rows and pieces are worked out each time: held, they would push the sums out of the registers
        asm volatile("" : "+v"(from));
        if constexpr (HB == 8) {  // two wavefronts share eight rows
            constexpr int FIRST = (PER + 1) / 2;
            if (wave & 1) {
#pragma unroll
                for (int k = FIRST; k < PER; k++) copy_one(t0, slot, wave >> 1, k, from);
            } else {
#pragma unroll
                for (int k = 0; k < FIRST; k++) copy_one(t0, slot, wave >> 1, k, from);
            }
        } else {
#pragma unroll
            for (int y = 0; y < 4 / HB; y++)
#pragma unroll
                for (int k = 0; k < PER; k++) copy_one(t0, slot, wave * (4 / HB) + y, k, from);
        }
    };
    // Waits until all but the copies of `ahead` tiles are there.
    auto arrived = [&](bool ahead) __attribute__((always_inline)) {
        if (!ahead || SLOTS == 2) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else if constexpr (HB == 8) {
            constexpr int FIRST = (PER + 1) / 2;
            if (wave & 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((SLOTS - 2) * (PER - FIRST)) : "memory");
            else asm volatile("s_waitcnt vmcnt(%0)" ::"n"((SLOTS - 2) * FIRST) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((SLOTS - 2) * PER * 4 / HB) : "memory");
        }
    };
    // Reads: piece 4 st + g4 of row 16 t + n, values 16 b on of rows 4 g4 .. and 16 + 4 g4 ...
    const int kat[2] = {n * PB + (g4 ^ (n >> 1)) * 16, n * PB + ((4 + g4) ^ (n >> 1)) * 16};
    int vat[4];
    {
        const int row = 4 * g4 + ((lane & 15) >> 2);
#pragma unroll
        for (int b = 0; b < 4; b++) vat[b] = row * PB + ((2 * b + ((lane & 3) >> 1)) ^ (row >> 1)) * 16 + 8 * (lane & 1);
    }
    const float c = a.scale * 1.4426950408889634f;

    for (; x < x1; r++) {
        const int len = clamp_len(a.lens[r], a.table.width, a.c.page), tiles = latent_tiles(len);
        if (tiles == 0) continue;
        const int64_t first = x - start, count = min(int64_t(tiles) - first, x1 - x);
        const int lo = int(first) * kLatentTile, hi = int(min(int64_t(len), (first + count) * kLatentTile));
        tvec qf[NS];
#pragma unroll
        for (int st = 0; st < NS; st++) {
            u32x4 y{0, 0, 0, 0};
            if (real && 32 * st + 8 * g4 < width)
                y = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.q) + (r * a.q_stride + int64_t(h) * width + 32 * st + 8 * g4) * 2);
            qf[st] = __builtin_bit_cast(tvec, y);
        }
        f32x4 o[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        for (int c0 = lo; c0 < hi; c0 += CH) {
            const int cn = min(CH, hi - c0), nt = latent_tiles(cn);
            __syncthreads();  // all have left the lookup and the tiles
            if (tid == 0) s_gaps = 0;
            __syncthreads();
            for (int i = tid; i < nt * kLatentTile; i += 64 * HB) {
                const int pos = c0 + min(i, cn - 1);  // past the last: that again, which is finite if it is
                const int32_t p = page_of(a.table.p + r * a.table.width, a.table.width, a.c.page, a.c.pages, pos);
                s_at[i] = p < 0 ? -1 : (int64_t(p) * a.c.page + uint32_t(pos) % a.c.page) * width * 2;
                if (p < 0) s_gaps = 1;
            }
            __syncthreads();
            const bool gaps = s_gaps;
            for (int t = 0; t < SLOTS - 1 && t < nt; t++) copy(t * kLatentTile, t);
            int slot = 0;
            for (int t = 0; t < nt; t++) {
                arrived(t + SLOTS - 2 < nt);
                lds_barrier();  // the tile is there, and all have left the one before
                if (gaps) {     // no page: zeros
                    for (int i = tid; i < kLatentTile * PP; i += 64 * HB)
                        if (s_at[t * kLatentTile + i / PP] < 0) *reinterpret_cast<u32x4 *>(s_c + slot * TILE + 16 * i) = u32x4{0, 0, 0, 0};
                    lds_barrier();
                }
                if (t + SLOTS - 1 < nt) copy((t + SLOTS - 1) * kLatentTile, slot == 0 ? SLOTS - 1 : slot - 1);
                const char *const s_t = s_c + slot * TILE;
                slot = slot == SLOTS - 1 ? 0 : slot + 1;
                f32x4 s[2];
#pragma unroll
                for (int u = 0; u < 2; u++) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < NS; st++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
                        s[u] = mfma16(*reinterpret_cast<const tvec *>(s_t + kat[st & 1] + (st / 2) * 128 + u * 16 * PB), qf[st], s[u]);
                float sc[8];
#pragma unroll
                for (int i = 0; i < 8; i++) sc[i] = s[i >> 2][i & 3] * c;  // in units of log2
                if ((t + 1) * kLatentTile > cn) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (t * kLatentTile + 16 * (i >> 2) + 4 * g4 + (i & 3) >= cn) sc[i] = -INFINITY;
                }
                float top = sc[0];
#pragma unroll
                for (int i = 1; i < 8; i++) top = fmaxf(top, sc[i]);
                if (__any(top > m + kSlack)) {
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float mn = fmaxf(m, top), f = mn == -INFINITY ? 1.f : exp2_f32(m - mn);
                    l *= f;
#pragma unroll
                    for (int b = 0; b < NB; b++) o[b] *= f;
                    m = mn;
                }
                const float ref = m == -INFINITY ? 0.f : m - lift<T>;
                tvec p;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float w = exp2_f32(sc[i] - ref);
                    l += w;
                    p[i] = T(w);
                }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const u32x2 y = lds_read_tr16(s_t + vat[b & 3] + (b / 4) * 128), z = lds_read_tr16(s_t + vat[b & 3] + (b / 4) * 128 + 16 * PB);
                    o[b] = mfma16(__builtin_bit_cast(tvec, u32x4{y[0], y[1], z[0], z[1]}), p, o[b]);
                }
            }
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (real && count == tiles) {
            T *out = static_cast<T *>(a.out) + r * a.out_stride + int64_t(h) * rank;
            typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (16 * b + 4 * g4 < rank)
                    *reinterpret_cast<t4 *>(out + 16 * b + 4 * g4) = t4{T(o[b][0] * inv), T(o[b][1] * inv), T(o[b][2] * inv), T(o[b][3] * inv)};
        } else if (real) {
            float *dst = part + (part_place(g, start, each) * a.heads + h) * (rank + kPartTail);
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (16 * b + 4 * g4 < rank) *reinterpret_cast<f32x4 *>(dst + 16 * b + 4 * g4) = o[b] * inv;
            // The weights carry 2^lift.
            if (g4 == 0) dst[rank] = l == 0.f ? -INFINITY : (m - lift<T>) + log2f(l);
        }
        x += count, start += tiles;
    }
}

// One workgroup a (sequence, head): the parts of sequences that several runs have; zeros for empty ones.
template <class T> __global__ __launch_bounds__(256) void latent_join_kernel(LatentDecodeArgs a, LatentPlan plan, const float *part) {
    const int64_t r = blockIdx.x;
    const int h = blockIdx.y, rank = a.c.rank, tiles = latent_tiles(clamp_len(a.lens[r], a.table.width, a.c.page));
    int64_t start = 0;
    const int64_t total = scan_tiles(a, [&](uint32_t r0, int, int64_t before) {
        if (r - r0 < 64) start = __shfl(before, int(r - r0) & 63);
        return false;
    });
    const int64_t each = latent_run(total, plan.runs);
    const Runs runs = tiles ? runs_of(start, tiles, each) : Runs{0, -1};
    const int count = int(runs.last - runs.first + 1);
    if (count == 1) return;
    T *out = static_cast<T *>(a.out) + r * a.out_stride + int64_t(h) * rank;
    join_parts<256>(count, rank, [&](int i) { return part + (part_place(runs.first + i, start, each) * a.heads + h) * (rank + kPartTail); }, [&](int c, f32x4 o) {
        for (int i = 0; i < 4; i++) out[c + i] = T(o[i]);
    });
}

template <class T, int RC, int HB, int SLOTS> void launch_tiles(const LatentDecodeArgs &a, const LatentPlan &plan, float *part, hipStream_t s) {
    hipLaunchKernelGGL((latent_tile_kernel<T, RC, HB, SLOTS>), dim3(plan.runs, (plan.groups + HB - 1) / HB), dim3(64 * HB), 0, s, a, plan, part);
}
// f(rank class, wavefronts): the least that hold the rank and the heads.
template <class T> void launch_heads(const LatentDecodeArgs &a, const LatentPlan &plan, float *part, hipStream_t s) {
    const int gr = plan.groups;
    if (a.c.rank <= 128) gr <= 1 ? launch_tiles<T, 128, 1, 4>(a, plan, part, s) : gr <= 2 ? launch_tiles<T, 128, 2, 4>(a, plan, part, s) : gr <= 4 ? launch_tiles<T, 128, 4, 4>(a, plan, part, s) : launch_tiles<T, 128, 8, 4>(a, plan, part, s);
    else if (a.c.rank <= 256) gr <= 1 ? launch_tiles<T, 256, 1, 3>(a, plan, part, s) : gr <= 2 ? launch_tiles<T, 256, 2, 3>(a, plan, part, s) : gr <= 4 ? launch_tiles<T, 256, 4, 3>(a, plan, part, s) : launch_tiles<T, 256, 8, 4>(a, plan, part, s);
    else gr <= 1 ? launch_tiles<T, 512, 1, 2>(a, plan, part, s) : gr <= 2 ? launch_tiles<T, 512, 2, 2>(a, plan, part, s) : gr <= 4 ? launch_tiles<T, 512, 4, 2>(a, plan, part, s) : launch_tiles<T, 512, 8, 4>(a, plan, part, s);
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

void launch_latent_decode(Ctx &c, const LatentDecodeArgs &a, hipStream_t s) {
    const double vecs = double(a.table.rows) * a.table.width * a.c.page;
    bool pieces = a.c.rank % 8 == 0 && a.c.rot % 8 == 0 && a.c.rot <= 64 && a.q_stride % 8 == 0 && a.out_stride % 8 == 0;
    for (const void *p : {static_cast<const void *>(a.c.p), a.q, static_cast<const void *>(a.out)}) pieces = pieces && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    ProbeScope probe("latent_decode", s, 2.0 * vecs * a.heads * (2 * a.c.rank + a.c.rot), 2.0 * vecs * (a.c.rank + a.c.rot),
                     pieces ? "latent_decode_runs" : "latent_decode_row");
    if (!pieces) {
        with_type16(a.c.type, [&](auto t) { hipLaunchKernelGGL((latent_row_kernel<decltype(t)>), dim3(a.table.rows, a.heads), dim3(64), 0, s, a); });
        OCR_HIP(hipGetLastError());
        return;
    }
    // A workgroup of 128 heads fills a compute unit, of fewer two do.
    LatentPlan plan{0, int((a.heads + 15) / 16)};
    const int64_t most = int64_t(a.table.rows) * latent_tiles(int(a.table.width * a.c.page));
    const int64_t units = plan.groups > 4 ? 256 : 512;
    plan.runs = int(std::max<int64_t>(1, std::min<int64_t>(units / ((plan.groups + 7) / 8), (most + kLeastRun - 1) / kLeastRun)));
    DBuf part(&c, size_t(2) * plan.runs * a.heads * (a.c.rank + kPartTail) * 4, s);
    with_type16(a.c.type, [&](auto t) {
        using T = decltype(t);
        launch_heads<T>(a, plan, part.as<float>(), s);
        hipLaunchKernelGGL((latent_join_kernel<T>), dim3(a.table.rows, a.heads), dim3(256), 0, s, a, plan, part.as<float>());
    });
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
