// Eviction from the paged cache: of each sequence's cached tokens the most attended stay, and those of them that
// lie past the new length move into the places that became free.
//
// Only what has to move does, so a cache that is a few tokens over its size costs the reading of its weights and a few
// vectors. The threshold that the kept ones reach is found eight bits of their keys at a time (weight_key: an order of
// unsigned numbers), in counts of 256 bins; places are then numbered by masks of 64 of them, so that the lists of free
// places and of moved vectors are in order without a sort. 64 pairs of a sequence and a head, 16 500 places kept down to 2048:
// 29 us for the choice (64 compute units, a third of it vector instructions, the rest waits between the passes), 33 for the moves.
// 144 of 528 places, 512 kept: 9 us, one launch, a chain of lengths, weights, four counts and the moves.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "lds_dma.h"
#include "text_device.h"

namespace ocr {

namespace {

struct Move {
    int32_t to, from;
};

// Vectors of one (sequence, head) moved by `count` threads, of which this is `tid`; P: what a thread copies at once.
template <class P> __device__ inline void move_vectors(const EvictArgs &a, int64_t r, uint32_t h, const Move *moves, int n, int tid, int count) {
    const int32_t *const row = a.table.p + r * a.table.width;
    const bool scales = a.kv.type == T_I8 || a.kv.type == T_E4M3;
    const int pieces = int(a.kv.dim * (scales ? 1 : 2) / sizeof(P)), each = 2 * pieces;  // keys' and values'
    auto slot = [&](int p) -> int64_t {
        const int32_t page = page_of(row, a.table.width, a.kv.page, a.kv.pages, p);
        return page < 0 ? -1 : slot_of(page, a.kv.heads, a.kv.page, h, uint32_t(p) % a.kv.page);
    };
    constexpr int U = 4;
    int i = tid / each, e = tid - i * each;
    const int di = count / each, de = count - di * each;
    while (i < n) {
        P v[U];
        P *to[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            to[u] = nullptr;
            if (i < n) {
                const int c = e < pieces ? e : e - pieces;
                const Move m = moves[i];
                const int64_t src = slot(m.from), dst = slot(m.to);
                if (src >= 0 && dst >= 0) {
                    P *const pool = static_cast<P *>(e < pieces ? a.kv.k : a.kv.v);
                    v[u] = pool[src * pieces + c];
                    to[u] = pool + dst * pieces + c;
                    if (scales && c == 0) {
                        float *const s = e < pieces ? a.kv.k_scale : a.kv.v_scale;
                        s[dst] = s[src];
                    }
                }
            }
            i += di, e += de;
            if (e >= each) e -= each, i++;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (to[u]) *to[u] = v[u];
    }
}

constexpr int kMostMovesHere = 1024;

// One workgroup of N threads a (sequence, head): which stay, the lists of moves, the weights and positions. KEYS: how many
// places' keys fit in LDS (0: they are made again each time). HERE: the vectors are moved as well, in pieces P.
template <int N, int KEYS, bool HERE, class P> __global__ __launch_bounds__(N) void evict_kernel(EvictArgs a, Move *moves_all, int32_t *counts, int cap) {
    constexpr int W = N / 64, U = 4, COPIES = 8;
    constexpr int RUNS = KEYS ? KEYS / 64 : 512;  // of 64 places, numbered at a time
    __shared__ uint32_t s_key[KEYS ? KEYS : 1];
    __shared__ __align__(16) int s_bins[256 * COPIES];
    __shared__ __align__(16) int s_sum[256];
    __shared__ unsigned long long s_stay[RUNS], s_same[RUNS];
    __shared__ int s_to[RUNS], s_from[RUNS];
    __shared__ Move s_moves[HERE ? kMostMovesHere : 1];
    __shared__ uint32_t s_prefix;
    __shared__ int s_want, s_over, s_moved;
    const uint32_t heads = a.kv.heads, h = blockIdx.x % heads;
    const int64_t r = blockIdx.x / heads, base = int64_t(blockIdx.x) * a.most;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = min(clamp_len(a.lens[r], a.table.width, a.kv.page), int(a.most)), left = min(n, int(a.keep)), newest = a.newest[r];
    auto position_of = [&](int p, int32_t held) { return held_position(held, p, n, newest); };
    auto key_of = [&](int p, int32_t held, float w) { return is_protected(position_of(p, held), newest, a.first, a.recent) ? kProtected : weight_key(w); };
    auto place = [&](int to, int from) {  // the weight and position of one place at another
        const float w = a.weights[base + from];
        const int32_t pos = int32_t(position_of(from, a.held[base + from]));
        a.weights_out[base + to] = w, a.held_out[base + to] = pos;
    };
    // f(first place, the lane's key) over 64 places every `step` from p0 on, U of them at a time with their loads together;
    // with first_ the keys are made and kept.
    auto keys = [&](int p0, int p1, int step, auto first_, auto &&f) __attribute__((always_inline)) {
        constexpr bool MAKE = decltype(first_)::value || KEYS == 0;
        for (; p0 < p1; p0 += U * step) {
            uint32_t k[U];
            if constexpr (MAKE) {
                int32_t held[U];
                float w[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int p = min(p0 + u * step + lane, n - 1);
                    held[u] = a.held[base + p], w[u] = a.weights[base + p];
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int p = min(p0 + u * step + lane, n - 1);
                    k[u] = key_of(p, held[u], w[u]);
                    if (KEYS) s_key[p] = k[u];
                }
            } else {
#pragma unroll
                for (int u = 0; u < U; u++) k[u] = s_key[min(p0 + u * step + lane, n - 1)];
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (p0 + u * step < p1) f(p0 + u * step, k[u]);
        }
    };
    if (h == 0 && tid == 0) a.lens_out[r] = left;
    Move *const moves = HERE ? s_moves : moves_all + int64_t(blockIdx.x) * cap;
    int moved = 0;
    if (n <= left) {
        for (int p = tid; p < n; p += N) place(p, p);
    } else {
        // The least key that stays: `prefix` above the bits that are still open, of whose places `want` stay.
        uint32_t prefix = 0;
        int want = left, shift = 24;
        bool all = false;  // every key of the prefix stays
        for (;; shift -= 8) {
            for (int i = tid; i < 64 * COPIES; i += N) reinterpret_cast<u32x4 *>(s_bins)[i] = u32x4{0, 0, 0, 0};
            __syncthreads();
            auto count = [&](int p0, uint32_t k) __attribute__((always_inline)) {
                if (p0 + lane < n && (shift == 24 || k >> ((shift + 8) & 31) == prefix)) atomicAdd(&s_bins[(k >> shift & 255) * COPIES + lane % COPIES], 1);
            };
            if (shift == 24) keys(wave * 64, n, N, std::true_type{}, count);
            else keys(wave * 64, n, N, std::false_type{}, count);
            __syncthreads();
            if (tid < 256) {
                const u32x4 *const copies = reinterpret_cast<const u32x4 *>(s_bins + tid * COPIES);
                const u32x4 x = copies[0] + copies[1];
                s_sum[255 - tid] = int((x[0] + x[1]) + (x[2] + x[3]));
            }
            lds_barrier();
            if (wave == 0) {  // lane l has the bins 255 - 4 l down to 252 - 4 l
                const u32x4 c = *reinterpret_cast<const u32x4 *>(s_sum + 4 * lane);
                const int sum = int((c[0] + c[1]) + (c[2] + c[3]));
                int upto = sum;
#pragma unroll
                for (int d = 1; d < 64; d *= 2) {
                    const int x = __shfl_up(upto, d);
                    if (lane >= d) upto += x;
                }
                int before = upto - sum;
                if (before < want && want <= upto) {
                    int u = 0, here = int(c[0]);
#pragma unroll
                    for (int x = 1; x < 4; x++)
                        if (before + here < want) before += here, here = int(c[x]), u = x;
                    s_prefix = prefix << 8 | uint32_t(255 - 4 * lane - u);
                    s_want = want - before;
                    s_over = here == want - before;
                }
            }
            __syncthreads();
            prefix = s_prefix, want = s_want, all = s_over;
            if (shift == 0 || all) break;
        }
        const uint32_t least = prefix << shift;
        // Masks of the places over and at the least key, then wavefront 0 numbers their runs: keys over it stay, and of the
        // equal ones the first `want` (`all`: every key of the prefix counts as over).
        int ties = 0, past = 0;
        for (int x0 = 0; x0 * 64 < n; x0 += RUNS) {
            const int runs = min(RUNS, (n + 63) / 64 - x0);
            keys(64 * (x0 + wave), 64 * (x0 + runs), N, std::false_type{}, [&](int p0, uint32_t k) __attribute__((always_inline)) {
                const bool in = p0 + lane < n;
                const unsigned long long over = __ballot(in && (k > least || (all && k == least))), same = __ballot(in && !all && k == least);
                if (lane == 0) s_stay[p0 / 64 - x0] = over, s_same[p0 / 64 - x0] = same;
            });
            __syncthreads();
            // Of the places of run x, those under the new length.
            auto under = [&](int x) { return 64 * x >= left ? 0ull : left - 64 * x >= 64 ? ~0ull : (1ull << (left - 64 * x)) - 1; };
            if (wave == 0)
                for (int x = 0; x < runs; x += 64) {
                    const bool in = x + lane < runs;
                    unsigned long long same = in ? s_same[x + lane] : 0, stay = in ? s_stay[x + lane] : 0;
                    auto before = [&](int mine, int &sum) {  // of this lane, and the sum goes up by all
                        int upto = mine;
#pragma unroll
                        for (int d = 1; d < 64; d *= 2) {
                            const int y = __shfl_up(upto, d);
                            if (lane >= d) upto += y;
                        }
                        const int at = sum + upto - mine;
                        sum += __builtin_amdgcn_readlane(upto, 63);
                        return at;
                    };
                    const int open = want - before(__popcll(same), ties);  // of the equal ones, these stay
                    const unsigned long long some = __ballot(open > 0 && __popcll(same) > open);  // one run at most
                    if (some) {
                        const int l = __builtin_ctzll(some), first = __builtin_amdgcn_readlane(open, l);
                        const unsigned long long m = lane_value(same, l), kept = __ballot(m >> lane & 1 && __popcll(m & ((1ull << lane) - 1)) < first);
                        if (lane == l) same = kept;
                    }
                    if (open > 0) stay |= same;
                    const unsigned long long u = under(x0 + x + lane);
                    const int to = before(in ? __popcll(u & ~stay) : 0, moved), from = before(in ? __popcll(stay & ~u) : 0, past);
                    if (in) s_stay[x + lane] = stay, s_to[x + lane] = to, s_from[x + lane] = from;
                }
            __syncthreads();
            for (int x = wave; x < runs; x += W) {
                const unsigned long long stay = s_stay[x], u = under(x0 + x), gaps = u & ~stay, out = stay & ~u, below = (1ull << lane) - 1;
                const int p = 64 * (x0 + x) + lane;
                if (gaps >> lane & 1) moves[s_to[x] + __popcll(gaps & below)].to = p;
                if (out >> lane & 1) moves[s_from[x] + __popcll(out & below)].from = p;
                if (u & stay & 1ull << lane) place(p, p);
            }
            __syncthreads();
        }
        if (tid == 0) s_moved = moved;
        __syncthreads();
        moved = s_moved;
    }
    if (!HERE && tid == 0) counts[blockIdx.x] = moved;
    // The arrays may be the old ones: what moved is read from past the new length, what is left there is cleared after.
    for (int i = tid; i < moved; i += N) place(moves[i].to, moves[i].from);
    __syncthreads();
    for (int p = left + tid; p < int(a.most); p += N) a.weights_out[base + p] = 0.f, a.held_out[base + p] = -1;
    if (HERE) move_vectors<P>(a, r, h, moves, moved, tid, N);
}

// The moves of blockIdx.x's (sequence, head), shared by the workgroups of blockIdx.y: 16 KB of keys each, and of values, if all that
// may move does. 64 pairs, some 1800 vectors of 256 bytes each (118 MB read and written): 33 us, of 32 KB 45, of 64 61, of 8 34.
template <class P> __global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a, const Move *moves, const int32_t *counts, int cap) {
    move_vectors<P>(a, blockIdx.x / a.kv.heads, blockIdx.x % a.kv.heads, moves + int64_t(blockIdx.x) * cap, counts[blockIdx.x],
                    int(blockIdx.y * 256 + threadIdx.x), int(gridDim.y * 256));
}

}  // namespace

void launch_evict(Ctx &c, const EvictArgs &a, hipStream_t s) {
    const uint32_t pairs = a.table.rows * a.kv.heads;
    const uint64_t places = std::min<uint64_t>(a.most, uint64_t(a.table.width) * a.kv.page);
    const uint64_t cap = std::max<uint64_t>(1, std::min<uint64_t>(a.keep, places > a.keep ? places - a.keep : 0));  // moves of one of them, at most
    const size_t vec = size_t(a.kv.dim) * type_bytes(a.kv.type);
    const bool pieces = whole_pieces(a.kv), here = cap * vec <= 32768 && cap <= kMostMovesHere;
    ProbeScope probe("text_evict", s, 4.0 * pairs * places, 16.0 * pairs * places, here ? "text_evict_one" : "text_evict_two");
    DBuf moves(&c, here ? 16 : size_t(pairs) * cap * sizeof(Move), s), counts(&c, size_t(pairs) * 4, s);
    Move *const list = moves.as<Move>();
    int32_t *const count = counts.as<int32_t>();
    // Keys in LDS as long as they fit: 16 500 places of 64 pairs 29 us, made again each time 37. Few places take little LDS and so
    // several workgroups a compute unit; 144 pairs of 528, which need but one, take 9.7 us either way. Short lists of moves are
    // worked off in the same launch: 144 of 16 moves 9.7 us, in one of their own 9.3 and 2.5.
    auto with = [&](auto here_, auto piece) {
        using P = decltype(piece);
        constexpr bool HERE = decltype(here_)::value;
        if (places <= 4096) hipLaunchKernelGGL((evict_kernel<256, 4096, HERE, P>), dim3(pairs), dim3(256), 0, s, a, list, count, int(cap));
        else if (places <= 32768 - 4096) hipLaunchKernelGGL((evict_kernel<1024, 32768 - 4096, HERE, P>), dim3(pairs), dim3(1024), 0, s, a, list, count, int(cap));
        else hipLaunchKernelGGL((evict_kernel<1024, 0, HERE, P>), dim3(pairs), dim3(1024), 0, s, a, list, count, int(cap));
    };
    if (here) {
        if (pieces) with(std::true_type{}, u32x4{});
        else with(std::true_type{}, uint8_t{});
    } else {
        with(std::false_type{}, u32x4{});
        const dim3 grid(pairs, unsigned(std::min<uint64_t>(1024, (cap * vec + 16383) / 16384)));
        if (pieces) hipLaunchKernelGGL((evict_move_kernel<u32x4>), grid, dim3(256), 0, s, a, list, count, int(cap));
        else hipLaunchKernelGGL((evict_move_kernel<uint8_t>), grid, dim3(256), 0, s, a, list, count, int(cap));
    }
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
