// Eviction from the paged cache: of each sequence's cached tokens the most attended stay, and those of them that
// lie past the new length move into the places that became free.
//
// Only what has to move does, so a cache that is a few tokens over its size costs the reading of its weights and a few
// vectors. The threshold that the kept ones reach is found eight bits of their keys at a time (weight_key: an order of
// unsigned numbers), in counts of 256 bins; places are then numbered by the wavefronts' masks, each wavefront a run of
// places, so that the lists of free places and of moved vectors are in order without a sort.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
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

// One workgroup of N threads a (sequence, head): which stay, the lists of moves, the weights and positions. KEYS: how many
// places' keys fit in LDS (0: they are made again each time). P: the vectors' pieces if they are moved here too.
template <int N, int KEYS, class P> __global__ __launch_bounds__(N) void evict_kernel(EvictArgs a, Move *moves_all, int32_t *counts, int cap, bool move_here) {
    constexpr int W = N / 64;
    __shared__ uint32_t s_key[KEYS ? KEYS : 1];
    __shared__ int s_bins[256];
    __shared__ int s_count[3][W];  // the wavefronts' equal keys, free places, moved vectors
    __shared__ uint32_t s_prefix;
    __shared__ int s_want, s_over;
    const uint32_t heads = a.kv.heads, h = blockIdx.x % heads;
    const int64_t r = blockIdx.x / heads, base = int64_t(blockIdx.x) * a.most;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = min(clamp_len(a.lens[r], a.table.width, a.kv.page), int(a.most)), left = min(n, int(a.keep)), newest = a.newest[r];
    auto position = [&](int p) { return held_position(a.held[base + p], p, n, newest); };
    auto make = [&](int p) { return is_protected(position(p), newest, a.first, a.recent) ? kProtected : weight_key(a.weights[base + p]); };
    auto key = [&](int p) { return KEYS ? s_key[p] : make(p); };
    if (h == 0 && tid == 0) a.lens_out[r] = left;
    int moved = 0;
    Move *const moves = moves_all + int64_t(blockIdx.x) * cap;
    if (n > left) {
        if (KEYS)
            for (int p = tid; p < n; p += N) s_key[p] = make(p);
        // The least key that stays: `prefix` above the bits that are still open, of whose places `want` stay.
        uint32_t prefix = 0;
        int want = left, shift = 24;
        bool all = false;  // every key of the prefix stays
        for (;; shift -= 8) {
            for (int b = tid; b < 256; b += N) s_bins[b] = 0;
            __syncthreads();
            for (int p0 = wave * 64; p0 < n; p0 += N) {
                const int p = p0 + lane;
                const uint32_t k = p < n ? key(p) : 0;
                const bool in = p < n && (shift == 24 || k >> ((shift + 8) & 31) == prefix);
                const uint32_t bin = k >> shift & 255;
                const unsigned long long some = __ballot(in);
                if (!some) continue;
                // Keys of one bin (protected places, weights of zero) are added at once.
                const int first = __builtin_ctzll(some);
                const uint32_t common = __builtin_amdgcn_readlane(bin, first);
                const unsigned long long alike = __ballot(in && bin == common);
                if (lane == first) atomicAdd(&s_bins[common], __popcll(alike));
                if (in && bin != common) atomicAdd(&s_bins[bin], 1);
            }
            __syncthreads();
            if (wave == 0) {  // lane l has the bins 255 - 4 l down to 252 - 4 l
                int c[4], sum = 0;
#pragma unroll
                for (int u = 0; u < 4; u++) c[u] = s_bins[255 - 4 * lane - u], sum += c[u];
                int upto = sum;
#pragma unroll
                for (int d = 1; d < 64; d *= 2) {
                    const int x = __shfl_up(upto, d);
                    if (lane >= d) upto += x;
                }
                int before = upto - sum;
                if (before < want && want <= upto) {
                    int u = 0;
                    while (before + c[u] < want) before += c[u++];
                    s_prefix = prefix << 8 | uint32_t(255 - 4 * lane - u);
                    s_want = want - before;
                    s_over = c[u] == want - before;
                }
            }
            __syncthreads();
            prefix = s_prefix, want = s_want, all = s_over;
            if (shift == 0 || all) break;
        }
        const uint32_t least = prefix << shift;
        // Runs of 64 places a wavefront; keys over the least stay, and of the equal ones the first `want`.
        const int runs = (n + 63) / 64, each = (runs + W - 1) / W, r0 = min(wave * each, runs), r1 = min(r0 + each, runs);
        int equal = 0;  // before this wavefront's
        if (!all) {
            int mine = 0;
            for (int x = r0; x < r1; x++) {
                const int p = 64 * x + lane;
                mine += __popcll(__ballot(p < n && key(p) == least));
            }
            if (lane == 0) s_count[0][wave] = mine;
            __syncthreads();
            for (int w = 0; w < wave; w++) equal += s_count[0][w];
        }
        // f(run, mask of the places that stay)
        auto sweep = [&](auto &&f) {
            int ties = equal;
            for (int x = r0; x < r1; x++) {
                const int p = 64 * x + lane;
                const uint32_t k = p < n ? key(p) : 0;
                unsigned long long stay;
                if (all) {
                    stay = __ballot(p < n && k >= least);
                } else {
                    const unsigned long long same = __ballot(p < n && k == least);
                    const int tie = ties + __popcll(same & ((1ull << lane) - 1));
                    stay = __ballot(p < n && (k > least || (k == least && tie < want)));
                    ties += __popcll(same);
                }
                f(x, stay);
            }
        };
        // Of the places of run x, those under the new length.
        auto under = [&](int x) { return 64 * x >= left ? 0ull : left - 64 * x >= 64 ? ~0ull : (1ull << (left - 64 * x)) - 1; };
        int free_places = 0, past = 0;
        sweep([&](int x, unsigned long long stay) { free_places += __popcll(under(x) & ~stay), past += __popcll(stay & ~under(x)); });
        if (lane == 0) s_count[1][wave] = free_places, s_count[2][wave] = past;
        __syncthreads();
        int to = 0, from = 0;
        for (int w = 0; w < W; w++) {
            if (w < wave) to += s_count[1][w], from += s_count[2][w];
            moved += s_count[1][w];
        }
        sweep([&](int x, unsigned long long stay) {
            const unsigned long long below = (1ull << lane) - 1, gaps = under(x) & ~stay, out = stay & ~under(x);
            if (gaps >> lane & 1) moves[to + __popcll(gaps & below)].to = 64 * x + lane;
            if (out >> lane & 1) moves[from + __popcll(out & below)].from = 64 * x + lane;
            to += __popcll(gaps), from += __popcll(out);
        });
    }
    if (tid == 0) counts[blockIdx.x] = moved;
    // In this order they may be the old arrays: what stays, what moves (read from past the new length), what is left.
    for (int p = tid; p < left; p += N) {
        const float w = a.weights[base + p];
        const int32_t pos = int32_t(position(p));
        a.weights_out[base + p] = w, a.held_out[base + p] = pos;
    }
    __syncthreads();
    for (int i = tid; i < moved; i += N) {
        const Move m = moves[i];
        const float w = a.weights[base + m.from];
        const int32_t pos = int32_t(position(m.from));
        a.weights_out[base + m.to] = w, a.held_out[base + m.to] = pos;
    }
    if (move_here) move_vectors<P>(a, r, h, moves, moved, tid, N);
    __syncthreads();
    for (int p = left + tid; p < int(a.most); p += N) a.weights_out[base + p] = 0.f, a.held_out[base + p] = -1;
}

// The moves of blockIdx.x's (sequence, head), shared by the workgroups of blockIdx.y.
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
    const bool pieces = whole_pieces(a.kv), move_here = cap * vec <= 32768;
    ProbeScope probe("text_evict", s, 4.0 * pairs * places, 16.0 * pairs * places, move_here ? "text_evict_one" : "text_evict_two");
    DBuf moves(&c, size_t(pairs) * cap * sizeof(Move), s), counts(&c, size_t(pairs) * 4, s);
    Move *const list = moves.as<Move>();
    int32_t *const count = counts.as<int32_t>();
    auto with = [&](auto piece) {
        using P = decltype(piece);
        if (places <= 4096) hipLaunchKernelGGL((evict_kernel<256, 4096, P>), dim3(pairs), dim3(256), 0, s, a, list, count, int(cap), move_here);
        else if (places <= 32768) hipLaunchKernelGGL((evict_kernel<1024, 32768, P>), dim3(pairs), dim3(1024), 0, s, a, list, count, int(cap), move_here);
        else hipLaunchKernelGGL((evict_kernel<1024, 0, P>), dim3(pairs), dim3(1024), 0, s, a, list, count, int(cap), move_here);
        if (!move_here)
            hipLaunchKernelGGL((evict_move_kernel<P>), dim3(pairs, unsigned(std::min<uint64_t>(1024, (cap * vec + 32767) / 32768))), dim3(256), 0, s, a,
                               list, count, int(cap));
    };
    if (pieces) with(u32x4{});
    else with(uint8_t{});
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
