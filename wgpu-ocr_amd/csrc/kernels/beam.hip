// A step of beam search: log-softmax of every beam's logits, the best of all beams' continuations.
//
// The logits are read once: a wavefront takes a block of a row, keeps it in registers, and writes
// the maxima of the block's four parts and the sum of its exponentials. What can be among a row's
// best `beams` lies in the parts whose maximum is at least the beams-th largest of the maxima, so the
// second kernel, one workgroup a group and a wavefront a beam, reads only those again. Values order as 32-bit keys
// (order_of); the beams-th largest of a set of keys is found bit by bit with ballots.
//
// Continuations order by their float64 scores, then by beam and token. Within a beam that is the logits'
// order wherever different logits score differently, which all do but next to nothing beside the log-sum or
// under a score of 10^9 and more; a row's best are found by their logits, and settle_ties looks for that.
//
// 64 groups of 8 beams: the second kernel takes 21 us, 5 to the row's sums, 7 to its best and 2 to
// the group's; one chain of latencies, on 64 of the compute units.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

constexpr int kChunk = 2048;       // logits that a wavefront holds: four times eight a lane
constexpr int kPart = 512;         // a part of a chunk: eight a lane
constexpr int kMostBlocks = 128;   // blocks of a row
constexpr int kHeld = kMostBlocks * 4 / 64;  // parts' maxima that a lane of the second kernel holds
constexpr int kOneLaunch = kChunk; // rows up to here need no first kernel
constexpr int kRough = 20;         // bits of a threshold that need not be exact
constexpr int kList = 256;         // continuations that a wavefront sorts

// Keys that order as the values do; NaN as minus infinity, the zeros alike.
__device__ inline uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x == x ? x + 0.f : -INFINITY);
    return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}

// Eight logits from index i on, all in the row, as they are in memory (rows lie on no more than a
// logit's size, which global loads take at any width). ONCE: the caches need not keep them, which
// gives 54.6 us instead of 64.8 where the first kernel says so, 55.5 where the second does as well.
template <class T> struct Raw {
    u32x4 x[8 * sizeof(T) / 16];
};
template <bool ONCE, class T> __device__ inline Raw<T> load_raw(const T *row, int i) {
    typedef uint32_t loose __attribute__((ext_vector_type(4), aligned(2)));
    Raw<T> r;
#pragma unroll
    for (int k = 0; k < int(8 * sizeof(T) / 16); k++) {
        const loose *p = reinterpret_cast<const loose *>(reinterpret_cast<const char *>(row + i) + 16 * k);
        r.x[k] = ONCE ? __builtin_nontemporal_load(p) : *p;
    }
    return r;
}
template <class T> __device__ inline void values(const Raw<T> &r, float *x) {
#pragma unroll
    for (int k = 0; k < 8; k++) {
        if constexpr (sizeof(T) == 4) x[k] = __uint_as_float(r.x[k / 4][k % 4]);
        else x[k] = widen16(r.x[0][k / 2] >> (16 * (k % 2)), std::is_same_v<T, f16> ? T_F16 : T_BF16);
    }
}
// The same at a row's end: minus infinity past the last.
template <class T> __device__ inline void last_values(const T *row, int i, int vocab, float *x) {
    T v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = row[min(i + k, vocab - 1)];
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = i + k < vocab ? to_f32(v[k]) : -INFINITY;
}

__device__ inline unsigned long long uniform(unsigned long long x) {
    return uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(x >> 32)))) << 32 | uint32_t(__builtin_amdgcn_readfirstlane(int(x)));
}

// Whether a beam's continuations have scores of their own: not if it is finished, or no score.
__device__ inline bool is_open(const BeamArgs &a, int64_t row) {
    return !(a.finished && a.finished[row]) && fabsf(a.scores[row]) < INFINITY;
}

struct Block {
    float part[4];  // the parts' largest logits (never NaN)
    float top, sum; // the largest of all, the sum of e^(x - top)
};
// A chunk's logits: eight of each part a lane, minus infinity past the row's end.
template <class T> __device__ inline void load_chunk(const T *row, int c, int vocab, float (*x)[8]) {
    const int lane = threadIdx.x & 63;
    if (c + kChunk <= vocab) {
        Raw<T> raw[4];
#pragma unroll
        for (int u = 0; u < 4; u++) raw[u] = load_raw<true>(row, c + kPart * u + 8 * lane);
#pragma unroll
        for (int u = 0; u < 4; u++) values(raw[u], x[u]);
        return;
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
#pragma unroll
        for (int k = 0; k < 8; k++) x[u][k] = -INFINITY;
        if (c + kPart * u < vocab) last_values(row, c + kPart * u + 8 * lane, vocab, x[u]);
    }
}
// A chunk added to a block (its sum still a lane's). Sums in float32: 32 terms a lane and chunk.
__device__ inline void add_chunk(const float (*x)[8], Block &b) {
    float top = b.top;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        float t = -INFINITY;
#pragma unroll
        for (int k = 0; k < 8; k++) t = fmaxf(t, x[u][k]);
        b.part[u] = fmaxf(b.part[u], wave_max(t));
        top = fmaxf(top, b.part[u]);
    }
    if (top == -INFINITY) return;
    b.sum *= exp2_f32((b.top - top) * 1.4426950408889634f);
    b.top = top;
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float e = exp2_f32((x[u][k] - top) * 1.4426950408889634f);
            b.sum += x[u][k] == x[u][k] ? e : 0.f;
        }
}
constexpr Block kNoBlock{{-INFINITY, -INFINITY, -INFINITY, -INFINITY}, -INFINITY, 0.f};

// A wavefront a block of a row. 512 rows of 128 000 bfloat16 values, a sixth of them finished: 24 us,
// 4.7 TB/s.
template <class T> __global__ __launch_bounds__(256) void beam_blocks_kernel(BeamArgs a, int blocks, int size, Block *out) {
    const int64_t row = blockIdx.x;
    const int b = blockIdx.y * 4 + (threadIdx.x >> 6), v = a.vocab;
    if (b >= blocks || !is_open(a, row)) return;
    Block s = kNoBlock;
    for (int c = b * size; c < min(v, (b + 1) * size); c += kChunk) {
        float x[4][8];
        load_chunk(static_cast<const T *>(a.logits) + row * a.stride, c, v, x);
        add_chunk(x, s);
    }
    s.sum = wave_sum(s.sum);
    if ((threadIdx.x & 63) == 0) out[row * blocks + b] = s;
}

// The n-th largest of all lanes' keys as far as `bits` of it go, the others zero: at least n keys
// reach it. count(t) says how many keys are t or more. Never under minus infinity's key.
template <class Count> __device__ inline uint32_t nth_largest(int n, int bits, Count &&count) {
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 32 - bits; bit--) {
        const uint32_t next = t | 1u << bit;
        if (count(next) >= n) t = next;
    }
    return max(t, kNothing);
}

// f(x, at) over a row's parts (sel: one bit a part, of blocks of `size`, all within `words`) in order,
// four at a time: a lane's eight logits of each, minus infinity past the row's end and for NaN, and
// the part's first index, vocab if there is none.
template <class T, class F> __device__ inline void each_part(const T *row, int vocab, int size, const unsigned long long *sel, int words, F &&f) {
    const int lane = threadIdx.x & 63;
    int at[4] = {vocab, vocab, vocab, vocab}, held = 0;
    auto flush = [&](bool whole) {
        float x[4][8];
        if (whole) {
            Raw<T> raw[4];
#pragma unroll
            for (int u = 0; u < 4; u++) raw[u] = load_raw<false>(row, (u < held ? at[u] : at[0]) + 8 * lane);
#pragma unroll
            for (int u = 0; u < 4; u++) values(raw[u], x[u]);
        } else {
            last_values(row, at[0] + 8 * lane, vocab, x[0]);
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (u >= held || x[u][k] != x[u][k]) x[u][k] = -INFINITY;
        f(x, at);
        held = 0;
        at[0] = at[1] = at[2] = at[3] = vocab;
    };
    for (int w = 0; w < words; w++)
        for (unsigned long long bits = uniform(sel[w]); bits;) {
            const int b = 16 * w + __builtin_ctzll(bits) / 4, first = 4 * (b - 16 * w), end = min(vocab, (b + 1) * size);
            const unsigned parts = unsigned(bits >> first) & 15;
            bits &= ~(15ull << first);
            for (int c = b * size; c < end; c += kChunk)
                for (unsigned p = parts; p; p &= p - 1) {
                    const int i = c + kPart * __builtin_ctz(p);
                    if (i >= vocab) break;
                    const bool last = i + kPart > vocab;
                    if (held == 4 || (last && held)) flush(true);
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        if (u == held) at[u] = i;
                    held++;
                    if (last) flush(false);
                }
        }
    if (held) flush(true);
}

// A row's best `want` keys in order into top (the wavefront's own LDS, as list and keys): a logit's
// key, then the index, lower ones larger. each(f): each_part over what can be among them; threshold:
// a key that at least `want` of the row reach, 0 if none is known.
template <class T, class Each>
__device__ inline void row_best(const T *row, int vocab, Each &&each, uint32_t threshold, int want, uint32_t *list, uint64_t *keys, uint64_t *top) {
    const int lane = threadIdx.x & 63;
    float t = value_of(threshold);
    int greater, n;
#pragma unroll 1
    for (int round = threshold ? 0 : 1;; round++) {
        if (round == 1) {  // of the lanes' largest
            uint32_t best = 0;
            each([&](const float (*x)[8], const int *at) {
                float m = -INFINITY;
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int k = 0; k < 8; k++) m = fmaxf(m, x[u][k]);
                if (at[0] + 8 * lane < vocab) best = max(best, order_of(m));
            });
            t = value_of(max(threshold, nth_largest(want, kRough, [&](uint32_t key) { return __popcll(__ballot(best >= key)); })));
        } else if (round == 2) {  // the exact one, which fewer than `want` exceed
            t = value_of(nth_largest(want, 32, [&](uint32_t key) {
                int c = 0;
                each([&](const float (*x)[8], const int *at) {
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int k = 0; k < 8; k++) c += at[u] + 8 * lane + k < vocab && order_of(x[u][k]) >= key;
                });
                for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o);
                return c;
            }));
        }
        greater = 0, n = 0;
        each([&](const float (*x)[8], const int *at) {
            unsigned over = 0, same = 0;  // a bit a logit
#pragma unroll
            for (int u = 0; u < 4; u++) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    over |= unsigned(x[u][k] > t) << (8 * u + k);
                    same |= unsigned(x[u][k] == t) << (8 * u + k);
                }
            }
            for (unsigned long long g; (g = __ballot(over)) != 0; over &= over - 1) {
                const int place = greater + __popcll(g & ((1ull << lane) - 1)), k = __builtin_ctz(over | 1u << 31);
                if (over && place < kList - int(kMostBeams)) list[place] = (k < 16 ? k < 8 ? at[0] : at[1] : k < 24 ? at[2] : at[3]) + 8 * lane + k % 8;
                greater += __popcll(g);
            }
            // Of those that equal the threshold the `want` lowest indices.
#pragma unroll 1
            for (int u = 0; u < 4 && n < want && __ballot(same); u++, same >>= 8) {
                const int i = (u < 2 ? u == 0 ? at[0] : at[1] : u == 2 ? at[2] : at[3]) + 8 * lane;
                unsigned mine = same & (vocab - i >= 8 ? 255u : (1u << max(vocab - i, 0)) - 1);
                if (!__ballot(mine)) continue;
                int before = n, all = n;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const unsigned long long g = __ballot(mine >> k & 1);
                    before += __popcll(g & ((1ull << lane) - 1)), all += __popcll(g);
                }
                for (; mine && before < want; mine &= mine - 1, before++) list[kList - 1 - before] = i + __builtin_ctz(mine);
                n = min(all, want);
            }
        });
        if (greater <= kList - int(kMostBeams)) break;
    }
    __builtin_amdgcn_wave_barrier();
    // Their places by counting.
    const int total = greater + n;
    for (int i = lane; i < total; i += 64) {
        const uint32_t at = list[i < greater ? i : kList - 1 - (i - greater)];
        keys[i] = uint64_t(order_of(to_f32(row[at]))) << 32 | uint32_t(~at);
    }
    __builtin_amdgcn_wave_barrier();
    for (int i = lane; i < total; i += 64) {
        const uint64_t key = keys[i];
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < total; j++) place += keys[j] > key;
        if (place < want) top[place] = key;
    }
    for (int i = total + lane; i < want; i += 64) top[i] = 0;  // fewer tokens than beams
}

// A row's `need` lowest tokens with logits in [lo, hi], of which there are that many: into top, as
// keys of `hi`.
template <class T> __device__ inline void lowest_of(const T *row, int vocab, uint32_t lo, uint32_t hi, int need, uint64_t *top) {
    const int lane = threadIdx.x & 63;
    const float least = value_of(lo), most = value_of(hi);
    for (int c = 0, n = 0; c < vocab && n < need; c += kChunk) {
        float x[4][8];
        load_chunk(row, c, vocab, x);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            unsigned mine = 0;  // a bit a logit; what is past the row's end is minus infinity, under every `lo`
#pragma unroll
            for (int k = 0; k < 8; k++) mine |= unsigned(x[u][k] >= least && x[u][k] <= most) << k;
            if (!__ballot(mine)) continue;
            int before = n, all = n;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const unsigned long long g = __ballot(mine >> k & 1);
                before += __popcll(g & ((1ull << lane) - 1)), all += __popcll(g);
            }
            for (; mine && before < need; mine &= mine - 1, before++)
                top[before] = uint64_t(hi) << 32 | uint32_t(~(c + kPart * u + 8 * lane + __builtin_ctz(mine)));
            n = min(all, need);
        }
    }
}

// A row's best `want` (at most 32) keys, found by their logits, brought into the order of scores, then
// tokens: where different logits score alike the lower tokens come first, those too that are not among
// the best by logits.
template <class T> __device__ inline void settle_ties(const T *row, int vocab, double cum, LogSum lse, int want, uint64_t *top) {
    const int lane = threadIdx.x & 63;
    const uint64_t mine = lane < want ? top[lane] : 0;
    const double s = score_of_key(uint32_t(mine >> 32), cum, lse);
    const uint32_t last = uint32_t(__builtin_amdgcn_readlane(int(mine >> 32), want - 1));
    const double least = score_of_key(last, cum, lse);
    // The next logit under the last one's: what scores as that may be anywhere in the row.
    if (last > kNothing && score_of_key(last - 1, cum, lse) == least) {
        const int first = __builtin_ctzll(__ballot(lane < want && s == least));
        const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(mine >> 32), first));
        lowest_of(row, vocab, lowest_alike(last, cum, lse), hi, want - first, top + first);
        __builtin_amdgcn_wave_barrier();
    }
    const uint64_t key = lane < want ? top[lane] : 0;
    const uint64_t next = __shfl_down(key, 1);
    const double after = __shfl_down(s, 1);  // the scores in order are what they were
    if (!__any(lane + 1 < want && s == after && uint32_t(key) < uint32_t(next))) return;  // ~token: the lower is the larger
    int place = 0;
    for (int j = 0; j < want; j++) {
        const double d = __shfl(s, j);
        const uint32_t t = uint32_t(__shfl(int(uint32_t(key)), j));
        place += d > s || (d == s && t > uint32_t(key));
    }
    __builtin_amdgcn_wave_barrier();
    if (lane < want) top[place] = key;
}

template <class T, bool ONE> __global__ __launch_bounds__(512) void beam_groups_kernel(BeamArgs a, int blocks, int size, const Block *stats) {
    __shared__ uint32_t s_list[8][kList];
    __shared__ uint64_t s_keys[8][kList], s_top[kMostBeams * kMostBeams];
    __shared__ double s_score[kMostBeams * kMostBeams];
    __shared__ int s_place[kMostBeams * kMostBeams];
    __shared__ unsigned long long s_sel[8][kHeld];
    const int64_t g = blockIdx.x;
    const int w = a.beams, v = a.vocab, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, want = min(w, v);
    for (int beam = wave; beam < w; beam += waves) {
        const int64_t r = g * w + beam;
        const T *row = static_cast<const T *>(a.logits) + r * a.stride;
        uint64_t *const top = s_top + beam * w;
        const double cum = a.scores[r];
        const bool over = a.finished && a.finished[r];
        float m = -INFINITY;
        double sum = 0.0;
        float x[4][8];        // a row of one chunk
        uint32_t key[kHeld];  // of the parts' maxima, 0 where there is no part
        const int words = (4 * blocks + 63) / 64;
        // All of the row's loads before the first is looked at.
        float t[kMostBlocks / 64], bs[kMostBlocks / 64], held[kHeld];
        if constexpr (ONE) {
            load_chunk(row, 0, v, x);
        } else {
#pragma unroll
            for (int k = 0; k < kMostBlocks / 64; k++) {
                const Block *b = stats + r * blocks + min(64 * k + lane, blocks - 1);
                t[k] = b->top, bs[k] = b->sum;
            }
#pragma unroll
            for (int k = 0; k < kHeld; k++) {
                const int part = min(64 * k + lane, 4 * blocks - 1);
                held[k] = stats[r * blocks + part / 4].part[part % 4];
            }
        }
        bool open = is_open(a, r);
        if (open) {
            if constexpr (ONE) {
                Block s = kNoBlock;
                add_chunk(x, s);
                m = s.top, sum = wave_sum(s.sum);
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (x[u][k] != x[u][k]) x[u][k] = -INFINITY;
            } else {
                float best = -INFINITY;
#pragma unroll
                for (int k = 0; k < kMostBlocks / 64; k++) {
                    if (64 * k + lane >= blocks) t[k] = -INFINITY;
                    best = fmaxf(best, t[k]);
                }
#pragma unroll
                for (int k = 0; k < kHeld; k++) key[k] = 64 * k + lane < 4 * blocks ? order_of(held[k]) : 0;
                m = wave_max(best);
#pragma unroll
                for (int k = 0; k < kMostBlocks / 64; k++)
                    if (64 * k < blocks && t[k] > -INFINITY) sum += double(bs[k]) * exp(double(t[k]) - double(m));
                for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
            }
            open = m > -INFINITY && m < INFINITY;
        }
        // The blocks' sums are float32 (off by some 2^-23, each its own way), what joins them, and what
        // decides between beams, float64.
        const LogSum lse = open ? log_sum(m, log(sum)) : LogSum{0.0, 0.0};
        if (open) {
            uint32_t t = 0;
            if constexpr (ONE) {
                const int at[4] = {0, min(kPart, v), min(2 * kPart, v), min(3 * kPart, v)};
                row_best(row, v, [&](auto &&f) { f(x, at); }, 0, want, s_list[wave], s_keys[wave], top);
            } else {
                uint32_t most = 0;
#pragma unroll
                for (int k = 0; k < kHeld; k++) most = max(most, key[k]);
                t = nth_largest(want, kRough, [&](uint32_t x) { return __popcll(__ballot(most >= x)); });
#pragma unroll
                for (int k = 0; k < kHeld; k++) {
                    const unsigned long long in = __ballot(key[k] >= t && key[k]);
                    if (lane == 0) s_sel[wave][k] = in;
                }
                __builtin_amdgcn_wave_barrier();
                row_best(row, v, [&](auto &&f) { each_part(row, v, size, s_sel[wave], words, f); }, t, want, s_list[wave], s_keys[wave], top);
            }
            __builtin_amdgcn_wave_barrier();
            settle_ties(row, v, cum, lse, want, top);
            for (int i = want + lane; i < w; i += 64) top[i] = 0;
        } else {
            // A finished beam's only continuation is its end; what scores nothing comes in order.
            const bool kept = over && fabs(cum) < INFINITY;
            for (int i = lane; i < w; i += 64) {
                const int at = !kept ? i : i == 0 ? a.eos : i - 1 + (i - 1 >= a.eos);
                top[i] = at >= 0 && at < v ? uint64_t(kept && i == 0) << 32 | uint32_t(~at) : 0;
            }
        }
        __builtin_amdgcn_wave_barrier();
        for (int i = lane; i < w; i += 64) {
            double s = -INFINITY;
            if (open) {
                if (top[i]) s = score_of_key(uint32_t(top[i] >> 32), cum, lse);
            } else if (top[i] >> 32) {
                s = cum;
            }
            s_score[beam * w + i] = s == s ? s : -INFINITY;
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // The group's best by counting those before each, list by list: the lists are in order, ties go
    // to the lower beam, then the lower token. No two count alike, so every place gets one.
    for (int c = threadIdx.x; c < w * w; c += blockDim.x) s_place[c] = 0;
    __syncthreads();
    for (int x = threadIdx.x; x < w * w * w; x += blockDim.x) {
        const int o = x / (w * w), c = x - o * w * w, beam = c / w;
        if (!s_top[c]) continue;
        const int before = o == beam ? c - beam * w : before_other(s_score + o * w, want, s_score[c], o < beam);
        if (before) atomicAdd(&s_place[c], before);
    }
    __syncthreads();
    // All of the group's inputs have been read but the flags of the winners.
    for (int c = threadIdx.x; c < w * w; c += blockDim.x) {
        const int place = s_place[c], beam = c / w, at = int(~uint32_t(s_top[c]));
        if (!s_top[c] || place >= w) continue;
        const bool over = a.finished && a.finished[g * w + beam];
        s_list[0][place] = uint32_t(c) << 1 | uint32_t(over || (a.eos >= 0 && at == a.eos));
        a.parents[g * w + place] = beam;
        a.tokens[g * w + place] = at;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < w; k += blockDim.x) {
        const uint32_t x = uint32_t(s_list[0][k]);
        a.out_scores[g * w + k] = float(s_score[x >> 1]);
        if (a.out_finished) a.out_finished[g * w + k] = x & 1;
    }
}

}  // namespace

void launch_beam(Ctx &c, const BeamArgs &a, hipStream_t s) {
    const int64_t rows = int64_t(a.groups) * a.beams;
    const size_t bytes = type_bytes(a.type);
    // Blocks of whole chunks, few enough for the second kernel's registers.
    const int chunks = int((a.vocab + kChunk - 1) / kChunk), size = (chunks + kMostBlocks - 1) / kMostBlocks * kChunk;
    const int blocks = int((a.vocab + size - 1) / size);
    const bool two = a.vocab > kOneLaunch;
    ProbeScope probe("beam_select", s, 3.0 * rows * a.vocab, double(rows) * a.vocab * bytes, two ? "beam_select_two" : "beam_select_one");
    DBuf stats;
    if (two) stats = DBuf(&c, size_t(rows) * blocks * sizeof(Block), s);
    with_type(a.type, [&](auto t) {
        using T = decltype(t);
        if (two) {
            hipLaunchKernelGGL((beam_blocks_kernel<T>), dim3(unsigned(rows), (blocks + 3) / 4), dim3(256), 0, s, a, blocks, size, stats.as<Block>());
            OCR_HIP(hipGetLastError());
        }
        const dim3 threads(64 * std::min(a.beams, 8u));
        if (two) hipLaunchKernelGGL((beam_groups_kernel<T, false>), dim3(a.groups), threads, 0, s, a, blocks, size, static_cast<const Block *>(stats.as<Block>()));
        else hipLaunchKernelGGL((beam_groups_kernel<T, true>), dim3(a.groups), threads, 0, s, a, blocks, size, static_cast<const Block *>(nullptr));
    });
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
