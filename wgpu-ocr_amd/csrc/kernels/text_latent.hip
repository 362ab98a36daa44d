// Latent attention over the paged cache of latent vectors: their writing, and single tokens' attention.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "lds_dma.h"
#include "text_device.h"

namespace ocr {

namespace {

// One wavefront a token, a chain of loads (token, page, vector): 64 tokens 9 us beside a cache of 377 MB, one 2.6. With the vector's
// loads all at once 8.4 and 2.9.
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
        before += lane_value(upto, 63);
    }
    return before;
}

// One run of tiles by W wavefronts of 16 heads each over the same tiles of 32 positions, whose vectors come into LDS by
// DMA, up to three tiles ahead. RC: the rank rounded up (the rotated part to 64). Each run goes through its sequences
// one after another.
//
// S^T = C Q^T, O^T = C^T P^T: the vectors are keys, row by row, and values, through the transposing reads, from one
// copy in LDS, rows of an odd number of 128 bytes whose pieces of 16 are exchanged by the row's last three bits: 16 rows' reads touch
// every bank both ways. Every product's LDS read is asked for PF products before it, in an order that is kept: left to
// itself the compiler reads, waits and multiplies one after another (163 us where this takes 147). The exponentials go among
// the next tile's first products, the copies among the second ones. A wavefront of rank 512 has a SIMD's registers for itself:
// 128 for sums, 72 for the query. 64 sequences of 2048 to 8191 positions, 128 heads, rank
// 512 + 64, bf16 (377 MB, 91 GFLOP): 118 us without the copies, 128 without the second products.
template <class T, int RC, int W> __global__ __launch_bounds__(64 * W, 1) void latent_tile_kernel(LatentDecodeArgs a, LatentPlan plan, float *part) {
    typedef T tvec __attribute__((ext_vector_type(8)));
    typedef T t4 __attribute__((ext_vector_type(4)));
    constexpr int DP = RC + 64, PP = DP / 8, PB = DP * 2, TILE = kLatentTile * PB, SLOTS = 4;
    constexpr int NS = DP / 32, NB = RC / 16, PF = 4;
    constexpr int MINE = kLatentTile * PP / 64 / W;  // a wavefront's copies of a tile
    static_assert(kLatentTile * PP % (64 * W) == 0, "whole copies");
    constexpr int CH = 2048;  // positions looked up at a time
    __shared__ __align__(16) char s_c[SLOTS * TILE];
    __shared__ int32_t s_at[CH];  // a position's vector in the pool, negative: none
    __shared__ int s_gaps;        // whether some of them are none
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g4 = lane >> 4;
    const int rank = a.c.rank, width = rank + int(a.c.rot), pieces = width / 8;
    // Workgroups of the same run and other heads are eight apart: on one die, whose level-two cache then reads the tiles once.
    const int shares = (plan.groups + W - 1) / W, share = int(blockIdx.x / 8 % shares);
    const int h = (share * W + wave) * 16 + n;
    const bool real = h < int(a.heads);
    const int64_t total = scan_tiles(a, [](uint32_t, int, int64_t) { return false; });
    const int64_t each = latent_run(total, plan.runs), run = blockIdx.x / (8 * shares) * 8 + blockIdx.x % 8;
    int64_t x = run * each;
    const int64_t x1 = min(total, x + each);
    if (x >= x1) return;
    // The sequence of tile x, and its own first tile.
    int64_t r = 0, start = 0;
    scan_tiles(a, [&](uint32_t r0, int mine, int64_t before) {
        const unsigned long long here = __ballot(before <= x && x < before + mine);
        if (!here) return false;
        const int at = __builtin_ctzll(here);
        r = r0 + at, start = lane_value(before, at);
        return true;
    });

    // Copies: the wavefront's j-th of a tile takes 64 of its pieces. Where its lane's row lies is looked up AHEAD copies before.
    const unsigned lds0 = lds_addr(s_c);
    constexpr int AHEAD = std::min(MINE, 6);
    struct Rows {
        int at[AHEAD];
    };
    auto row_at = [&](int t, int j) __attribute__((always_inline)) { return s_at[t * kLatentTile + (64 * (wave + W * j) + lane) / PP]; };
    auto look = [&](int t) __attribute__((always_inline)) {
        Rows r;
#pragma unroll
        for (int j = 0; j < AHEAD; j++) r.at[j] = row_at(t, j);
        return r;
    };
    auto copy = [&](int t, int j, Rows &rows) __attribute__((always_inline)) {
        int from = 64 * (wave + W * j) + lane;
        asm volatile("" : "+v"(from));  // worked out each time: held, they would take as many registers as there are copies
        const int row = from / PP, piece = min((from - row * PP) ^ (row & 7), pieces - 1);
        dma16_to(static_cast<const char *>(a.c.p) + uint64_t(uint32_t(max(rows.at[j % AHEAD], 0))) * uint32_t(width * 2) + uint32_t(16 * piece),
                 lds0 + t % SLOTS * TILE + (wave + W * j) * 1024);
        if (j + AHEAD < MINE) rows.at[j % AHEAD] = row_at(t, j + AHEAD);
    };
    // Waits until at most `tiles` tiles' copies are on their way (40 at most: the wait's number has six bits).
    auto wait_for = [&](auto tiles) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(decltype(tiles)::value * MINE) : "memory");
    };
    // Reads. Keys: rows n and 16 + n, piece 4 st + g4; values: columns 16 b on, of the rows whose scores the lane has.
    const int kat[2] = {n * PB + (g4 ^ (n & 7)) * 16, n * PB + ((4 + g4) ^ (n & 7)) * 16};
    int vat[4];
    {
        const int row = 4 * g4 + (n >> 2);
#pragma unroll
        for (int b = 0; b < 4; b++) vat[b] = row * PB + ((2 * b + (n >> 1 & 1)) ^ (row & 7)) * 16 + 8 * (n & 1);
    }
    const float c = a.scale * 1.4426950408889634f;

    for (; x < x1; r++) {
        const int len = __builtin_amdgcn_readfirstlane(clamp_len(a.lens[r], a.table.width, a.c.page)), tiles = latent_tiles(len);
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
        struct Scores {
            f32x4 s[2];
        };
        // f(i): other work among the products.
        auto scores = [&](const char *s_t, auto &&f) __attribute__((always_inline)) {
            Scores z{};
            auto read = [&](int i) { return *reinterpret_cast<const tvec *>(s_t + kat[i / 2 & 1] + i / 4 * 128 + i % 2 * 16 * PB); };
            tvec k[PF];
#pragma unroll
            for (int i = 0; i < PF; i++) k[i] = read(i);
#pragma unroll
            for (int i = 0; i < 2 * NS; i++) {
                z.s[i % 2] = mfma16(k[i % PF], qf[i / 2], z.s[i % 2]);
                if (i + PF < 2 * NS) k[i % PF] = read(i + PF);
                f(i);
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("" : "+v"(z.s[0]), "+v"(z.s[1]));  // here, and not where they are used, with all that was read held until then
            return z;
        };
        // Adds tile t by its scores z, which it makes the next one's (NEXT: there is one; else only `left` positions of this one may
        // be there). MORE: and tile t + 3 is asked for.
        auto turn = [&](Scores &z, int t, int left, auto next_, auto more_) __attribute__((always_inline)) {
            constexpr bool NEXT = decltype(next_)::value, MORE = decltype(more_)::value;
            const char *const s_t = s_c + t % SLOTS * TILE;
            Rows rows;
            if constexpr (MORE) rows = look(t + 3);
            float sc[8];  // in units of log2
#pragma unroll
            for (int i = 0; i < 8; i++) sc[i] = z.s[i / 4][i % 4] * c;
            if (!NEXT && left < kLatentTile) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (16 * (i / 4) + 4 * g4 + i % 4 >= left) sc[i] = -INFINITY;
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
            auto weight = [&](int i) __attribute__((always_inline)) {
                if (i >= 8) return;
                const float w = exp2_f32(sc[i] - ref);
                l += w;
                p[i] = T(w);
            };
            if constexpr (NEXT) {
                z = scores(s_c + (t + 1) % SLOTS * TILE, weight);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) weight(i);
            }
            auto read = [&](int b) __attribute__((always_inline)) {
                const char *const at = s_t + vat[b % 4] + b / 4 * 128;
                const u32x2 y = lds_read_tr16(at), v = lds_read_tr16(at + 16 * PB);
                return __builtin_bit_cast(tvec, u32x4{y[0], y[1], v[0], v[1]});
            };
            tvec v[PF];
#pragma unroll
            for (int i = 0; i < PF; i++) v[i] = read(i);
#pragma unroll
            for (int i = 0; i < NB; i++) {
                o[i] = mfma16(v[i % PF], p, o[i]);
                if (i + PF < NB) v[i % PF] = read(i + PF);
                if constexpr (MORE) {
#pragma unroll
                    for (int j = 0; j < MINE; j++)
                        if (j * NB / MINE == i) copy(t + 3, j, rows);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        for (int c0 = lo; c0 < hi; c0 += CH) {
            const int cn = min(CH, hi - c0), nt = latent_tiles(cn);
            __syncthreads();  // all have left the lookup and the tiles
            if (tid == 0) s_gaps = 0;
            __syncthreads();
            for (int i = tid; i < nt * kLatentTile; i += 64 * W) {
                const int pos = c0 + min(i, cn - 1);  // past the last: that again, which is finite if it is
                const int32_t p = page_of(a.table.p + r * a.table.width, a.table.width, a.c.page, a.c.pages, pos);
                s_at[i] = p < 0 ? -1 : int32_t(p * a.c.page + uint32_t(pos) % a.c.page);
                if (p < 0) s_gaps = 1;
            }
            __syncthreads();
            const bool gaps = __builtin_amdgcn_readfirstlane(s_gaps);
            // After a wait for tile t: all wavefronts' pieces are there, and all have left tile t - 2.
            auto arrived = [&](int t) __attribute__((always_inline)) {
                lds_barrier();
                if (!gaps) return;
                char *const s_t = s_c + t % SLOTS * TILE;  // no page: zeros
                for (int i = tid; i < kLatentTile * PP; i += 64 * W)
                    if (s_at[t * kLatentTile + i / PP] < 0) *reinterpret_cast<u32x4 *>(s_t + 16 * i) = u32x4{0, 0, 0, 0};
                lds_barrier();
            };
            for (int t = 0; t < 3 && t < nt; t++) {
                Rows rows = look(t);
#pragma unroll
                for (int j = 0; j < MINE; j++) copy(t, j, rows);
            }
            if (nt >= 3) wait_for(std::integral_constant<int, 2>{});
            else wait_for(std::integral_constant<int, 0>{});
            arrived(0);
            Scores z = scores(s_c, [](int) {});
            int t = 0;
            for (; t + 3 < nt; t++) {
                wait_for(std::integral_constant<int, 1>{});  // tiles t + 1 and t + 2 are on their way
                arrived(t + 1);
                turn(z, t, kLatentTile, std::true_type{}, std::true_type{});
            }
            for (; t + 1 < nt; t++) {
                wait_for(std::integral_constant<int, 0>{});
                arrived(t + 1);
                turn(z, t, kLatentTile, std::true_type{}, std::false_type{});
            }
            turn(z, t, cn - t * kLatentTile, std::false_type{}, std::false_type{});
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (real && count == tiles) {
            T *out = static_cast<T *>(a.out) + r * a.out_stride + int64_t(h) * rank;
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (16 * b + 4 * g4 < rank)
                    *reinterpret_cast<t4 *>(out + 16 * b + 4 * g4) = t4{T(o[b][0] * inv), T(o[b][1] * inv), T(o[b][2] * inv), T(o[b][3] * inv)};
        } else if (real) {
            float *dst = part + (part_place(run, start, each) * a.heads + h) * (rank + kPartTail);
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (16 * b + 4 * g4 < rank) *reinterpret_cast<f32x4 *>(dst + 16 * b + 4 * g4) = o[b] * inv;
            // The weights carry 2^lift.
            if (g4 == 0) dst[rank] = l == 0.f ? -INFINITY : (m - lift<T>) + log2f(l);
        }
        x += count, start += tiles;
    }
}

// One workgroup a sequence and `each_heads` heads: the parts of sequences that several runs have; zeros for empty ones. 64 sequences
// of 128 heads: 18 us for four heads of a workgroup, 21 for one, 22 for eight.
template <class T> __global__ __launch_bounds__(256) void latent_join_kernel(LatentDecodeArgs a, LatentPlan plan, int each_heads, const float *part) {
    const int64_t r = blockIdx.x;
    const int rank = a.c.rank, tiles = latent_tiles(clamp_len(a.lens[r], a.table.width, a.c.page));
    int64_t start = 0;
    const int64_t total = scan_tiles(a, [&](uint32_t r0, int, int64_t before) {
        if (r >= r0 && r - r0 < 64) start = lane_value(before, int(r - r0));
        return false;
    });
    const int64_t each = latent_run(total, plan.runs);
    const Runs runs = tiles ? runs_of(start, tiles, each) : Runs{0, -1};
    const int count = int(runs.last - runs.first + 1);
    if (count == 1) return;
    const int h1 = min(int(a.heads), int(blockIdx.y + 1) * each_heads);
    for (int h = int(blockIdx.y) * each_heads; h < h1; h++) {
        T *out = static_cast<T *>(a.out) + r * a.out_stride + int64_t(h) * rank;
        join_parts<256>(count, rank, [&](int i) { return part + (part_place(runs.first + i, start, each) * a.heads + h) * (rank + kPartTail); }, [&](int c, f32x4 o) {
            for (int i = 0; i < 4; i++) out[c + i] = T(o[i]);
        });
        __syncthreads();
    }
}

template <class T, int RC, int W> void launch_tiles(const LatentDecodeArgs &a, const LatentPlan &plan, float *part, hipStream_t s) {
    const unsigned shares = (plan.groups + W - 1) / W;
    hipLaunchKernelGGL((latent_tile_kernel<T, RC, W>), dim3((plan.runs + 7) / 8 * 8 * shares), dim3(64 * W), 0, s, a, plan, part);
}
// The wavefronts that hold the heads, up to 64 of them.
template <class T, int RC> void launch_heads(const LatentDecodeArgs &a, const LatentPlan &plan, float *part, hipStream_t s) {
    // One wavefront has not the registers for a whole tile of rank 512's copies: of two the second has no heads.
    if (RC < 512 && plan.groups <= 1) launch_tiles<T, RC, RC < 512 ? 1 : 2>(a, plan, part, s);
    else if (plan.groups <= 2) launch_tiles<T, RC, 2>(a, plan, part, s);
    else launch_tiles<T, RC, 4>(a, plan, part, s);
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
    bool pieces = a.c.rank % 8 == 0 && a.c.rot % 8 == 0 && a.c.rot <= 64 && a.q_stride % 8 == 0 && a.out_stride % 8 == 0 &&
                  uint64_t(a.c.pages) * a.c.page < 0x80000000u;
    for (const void *p : {static_cast<const void *>(a.c.p), a.q, static_cast<const void *>(a.out)}) pieces = pieces && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    ProbeScope probe("latent_decode", s, 2.0 * vecs * a.heads * (2 * a.c.rank + a.c.rot), 2.0 * vecs * (a.c.rank + a.c.rot),
                     pieces ? "latent_decode_runs" : "latent_decode_row");
    if (!pieces) {
        with_type16(a.c.type, [&](auto t) { hipLaunchKernelGGL((latent_row_kernel<decltype(t)>), dim3(a.table.rows, a.heads), dim3(64), 0, s, a); });
        OCR_HIP(hipGetLastError());
        return;
    }
    // A workgroup for every compute unit, whose LDS four tiles of rank 512 or 256 fill. Two: 24 sequences of up to 4000, 64 heads of rank 256
    // 42 us for 32; of up to 6000 of rank 128, which leave room for it, 29 for 27, and 3 of up to 20 000 with 16 heads 20 for 21.
    LatentPlan plan{0, int((a.heads + 15) / 16)};
    const int64_t most = int64_t(a.table.rows) * latent_tiles(int(a.table.width * a.c.page)), units = 256;
    plan.runs = int(std::max<int64_t>(1, std::min<int64_t>(units / ((plan.groups + 3) / 4), (most + kLeastRun - 1) / kLeastRun)));
    DBuf part(&c, size_t(2) * plan.runs * a.heads * (a.c.rank + kPartTail) * 4, s);
    const int each = int(std::max<int64_t>(1, std::min<int64_t>(4, int64_t(a.table.rows) * a.heads / 1024)));  // heads of a workgroup that joins
    with_type16(a.c.type, [&](auto t) {
        using T = decltype(t);
        if (a.c.rank <= 128) launch_heads<T, 128>(a, plan, part.as<float>(), s);
        else if (a.c.rank <= 256) launch_heads<T, 256>(a, plan, part.as<float>(), s);
        else launch_heads<T, 512>(a, plan, part.as<float>(), s);
        hipLaunchKernelGGL((latent_join_kernel<T>), dim3(a.table.rows, (a.heads + each - 1) / each), dim3(256), 0, s, a, plan, each, part.as<float>());
    });
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
