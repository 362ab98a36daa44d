// The text decoder's cache: a step's projections normed, rotated and written into pages, pages read
// back, beams' pages reordered. All are bound by the bytes they move: a lane takes eight values of a
// vector at a time, and as many lanes as it has eights (a power of two) share it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

constexpr int kAppendTokens = 4, kReadTokens = 16;  // tokens of a workgroup

// The instructions for reciprocals are off by up to a step, which moves codes over their borders; one Newton step on
// the float32 remainder brings a division's half step back, in four instructions instead of ten.
__device__ inline float root_reciprocal(float x) {
    const float r = __builtin_amdgcn_rsqf(x), h = x * r;
    return __fmaf_rn(__fmaf_rn(-h, r, 1.f), 0.5f * r, r);
}
// A vector's largest magnitude over its code, and the other way round (scale: the first of the two, from
// 2e-33 to 3e36, whose reciprocal is normal).
template <class C> __device__ inline float over_code_max(float m) {
    constexpr float part = 1.f / code_max<C>;
    const float s = m * part;
    return __fmaf_rn(__fmaf_rn(-s, code_max<C>, m), part, s);
}
template <class C> __device__ inline float code_max_over(float m, float scale) {
    const float r = __builtin_amdgcn_rcpf(scale);
    return __fmaf_rn(__fmaf_rn(-m, r, code_max<C>), r * (1.f / code_max<C>), r);
}


// Vectors that are no whole eights, or whose rotated halves are not: one wavefront a (token, head), lane l holds values l,
// l + 64, ... of the head's vector. 20 000 tokens of 48 heads of 64 with 36 values rotated: 324 us (all 64: 64).
template <class T, class O, class C> __global__ __launch_bounds__(64) void append_row_kernel(AppendArgs a) {
    __shared__ float s_x[256];
    const int lane = threadIdx.x, dim = a.kv.dim, heads = a.kv.heads;
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y;
    const int kind = h < int(a.q_heads) ? 0 : h < int(a.q_heads) + heads ? 1 : 2;  // q, k, v
    const T *src = static_cast<const T *>(a.qkv) + t * a.stride + int64_t(h) * dim;
    const int pos = a.pos[t];
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; u++) x[u] = lane + 64 * u < dim ? to_f32(src[lane + 64 * u]) : 0.f;
    const float *norm = kind == 0 ? a.q_norm : a.k_norm;
    if (kind < 2 && norm) {
        float ss = 0.f;
        for (int u = 0; u < 4; u++) ss += x[u] * x[u];
        const float r = 1.f / sqrtf(wave_sum(ss) / float(dim) + a.eps);
        for (int u = 0; u < 4; u++)
            if (lane + 64 * u < dim) x[u] = x[u] * r * norm[lane + 64 * u];
    }
    if (kind < 2 && a.rot) {
        for (int u = 0; u < 4; u++) s_x[lane + 64 * u] = x[u];
        __syncthreads();
        const int half = a.rot / 2;
        for (int u = 0; u < 4; u++) {
            const int c = lane + 64 * u;
            if (c >= int(a.rot)) continue;
            const int i = a.adjacent ? c >> 1 : c % half;
            const bool second = a.adjacent ? c & 1 : c >= half;
            const int other = a.adjacent ? c ^ 1 : second ? c - half : c + half;
            const float2 r = turn_of(a, t, i, a.rot);
            const float cs = r.x, sn = r.y;
            x[u] = second ? x[u] * cs + s_x[other] * sn : x[u] * cs - s_x[other] * sn;
        }
    }
    if (kind == 0) {
        O *dst = static_cast<O *>(a.q) + (t * a.q_heads + h) * dim;
        for (int u = 0; u < 4; u++)
            if (lane + 64 * u < dim) dst[lane + 64 * u] = O(x[u]);
        return;
    }
    const int hk = h - int(a.q_heads) - (kind == 2 ? heads : 0);
    if (kind == 1 && a.k) {
        O *dst = static_cast<O *>(a.k) + (t * heads + hk) * dim;
        for (int u = 0; u < 4; u++)
            if (lane + 64 * u < dim) dst[lane + 64 * u] = O(x[u]);
    }
    const int seq = a.seq[t];
    if (seq < 0 || seq >= int(a.table.rows)) return;
    const int page = page_of(a.table.p + size_t(seq) * a.table.width, a.table.width, a.kv.page, a.kv.pages, pos);
    if (page < 0) return;
    const int64_t slot = slot_of(page, heads, a.kv.page, hk, pos % a.kv.page);
    C *dst = static_cast<C *>(kind == 1 ? a.kv.k : a.kv.v) + slot * dim;
    float inv = 1.f;
    if constexpr (scaled<C>) {
        float m = 0.f, bad = 0.f;
        for (int u = 0; u < 4; u++) m = fmaxf(m, fabsf(x[u])), bad += x[u] * 0.f;
        m = wave_max(m);
        bad = wave_sum(bad);
        inv = m > kTinyMax ? code_max<C> / m : 0.f;
        float scale = m > kTinyMax ? m / code_max<C> : 0.f;
        if (!(bad == 0.f)) inv = 0.f, scale = NAN;  // a value that is not finite: the whole vector reads as NaN
        if (lane == 0) (kind == 1 ? a.kv.k_scale : a.kv.v_scale)[slot] = scale;
        if (!(bad == 0.f))
            for (int u = 0; u < 4; u++) x[u] = 0.f;
    }
    for (int u = 0; u < 4; u++)
        if (lane + 64 * u < dim) dst[lane + 64 * u] = code_of<C>(x[u] * inv);
}

// Outputs that the level-two caches (eight of 4 MiB) cannot hold are stored past them: what is left
// there at a kernel's end is written out before the next one starts. 144 sequences' 88 MB read back:
// 25 us for the step, 33 with ordinary stores; a prompt's 380 MB 149 and 157.
constexpr double kHeld = 32.0 * (1 << 20);

// N (four or eight) values at p, which lies on no more than a value's size. ONCE: the caches need not
// keep them (a prompt's projections: 147 us for writing and reading, 151 without; codes read back so: 32
// instead of 25 for 144 sequences, whose neighbouring heads share lines).
template <class T, int N> struct Some {
    uint32_t x[N * sizeof(T) / 4];
};
template <class T, int N> struct loose_of {
    static constexpr int words = N * sizeof(T) / 4 < 4 ? N * sizeof(T) / 4 : 4;
    typedef uint32_t type __attribute__((ext_vector_type(words), aligned(sizeof(T))));
};
template <class T, int N, bool ONCE = false> __device__ inline Some<T, N> load_some(const T *p) {
    using L = loose_of<T, N>;
    Some<T, N> r;
#pragma unroll
    for (int k = 0; k < int(N * sizeof(T) / 4) / L::words; k++) {
        const typename L::type *from = reinterpret_cast<const typename L::type *>(p) + k, y = ONCE ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
        for (int e = 0; e < L::words; e++) r.x[L::words * k + e] = y[e];
    }
    return r;
}
template <class T, int N> __device__ inline void store_some(T *p, const Some<T, N> &r, bool past) {
    using L = loose_of<T, N>;
    typename L::type y;
#pragma unroll
    for (int e = 0; e < L::words; e++) y[e] = r.x[e];
    if (past) {
        asm volatile("" ::: "memory");  // on both sides: else the compiler makes one ordinary store of the two
        __builtin_nontemporal_store(y, reinterpret_cast<typename L::type *>(p));
        asm volatile("" ::: "memory");
    } else {
        *reinterpret_cast<typename L::type *>(p) = y;
    }
}
template <class T, int N> __device__ inline float value_at(const Some<T, N> &r, int k) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.x[k]);
    else if constexpr (sizeof(T) == 2) return widen16(r.x[k / 2] >> (16 * (k % 2)), std::is_same_v<T, f16> ? T_F16 : T_BF16);
    else return to_f32(__builtin_bit_cast(T, uint8_t(r.x[k / 4] >> (8 * (k % 4)))));
}
// Values rounded to T (codes: already divided by the vector's scale).
template <class T, int N> __device__ inline Some<T, N> some_of(const float *x) {
    Some<T, N> r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < N; k++) r.x[k] = __float_as_uint(x[k]);
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = 0; k < N / 2; k++)
            r.x[k] = uint32_t(__builtin_bit_cast(uint16_t, T(x[2 * k]))) | uint32_t(__builtin_bit_cast(uint16_t, T(x[2 * k + 1]))) << 16;
    } else if constexpr (std::is_same_v<T, e4m3>) {
#pragma unroll
        for (int k = 0; k < N / 4; k++) {
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * k], x[4 * k + 1], 0, false);
            r.x[k] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * k + 2], x[4 * k + 3], lo, true);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N / 4; k++) {
            r.x[k] = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) r.x[k] |= uint32_t(uint8_t(code_of<int8_t>(x[4 * k + e]))) << (8 * e);
        }
    }
    return r;
}

// `each` tokens a workgroup, W lanes a vector. The tokens' turns and places are looked up once for
// all heads; a group of lanes takes a vector after the other, the next two on their way. A lane has
// two fours of a vector: those that it rotates with each other where pairs are halves apart, two
// neighbours otherwise. A prompt of 23 600 tokens of 48 bfloat16 heads of 128 into e4m3: 532 MB in
// 108 to 119 us, 4.5 to 4.9 TB/s (a large copy reaches 5.2); with the rotation's other half from a neighbouring
// lane and the compiler's divisions, the two together, 157, bound by vector instructions.
template <class T, class O, class C, int W> __global__ __launch_bounds__(256) void append_kernel(AppendArgs a, int each, bool past) {
    __shared__ __align__(16) float s_cos[kAppendTokens][128], s_sin[kAppendTokens][128];
    __shared__ __align__(16) float s_norm[2][8 * W];
    __shared__ int64_t s_vec[kAppendTokens];  // head 0's vector in the pool, negative: none
    const int tid = threadIdx.x, c = tid % W, dim = a.kv.dim, heads = a.kv.heads, all = a.q_heads + 2 * heads, half = a.rot / 2;
    const int64_t t0 = int64_t(blockIdx.x) * each;
    const int n = int(min<int64_t>(each, a.n - t0));
    const bool in = 8 * c < dim, turns = 8 * c < int(a.rot), apart = turns && !a.adjacent;
    const int at[2] = {!in ? 0 : apart ? 4 * c : 8 * c, !in ? 0 : apart ? half + 4 * c : 8 * c + 4};
    // A group's vectors: every G-th of the tokens' heads.
    constexpr int G = 256 / W;
    const int dt = G / all, dh = G - dt * all;
    struct Item {
        int t, h;
    };
    auto after = [&](Item i) {
        i.t += dt, i.h += dh;
        if (i.h >= all) i.h -= all, i.t++;
        return i;
    };
    struct Vec {
        Some<T, 4> x[2];
    };
    const T *const base = static_cast<const T *>(a.qkv) + t0 * a.stride;
    auto load = [&](Item i) {
        const T *src = base + (i.t < n ? i.t * a.stride + uint32_t(i.h * dim) : 0);
        return Vec{load_some<T, 4, true>(src + at[0]), load_some<T, 4, true>(src + at[1])};
    };
    Item item{tid / W / all, tid / W % all}, ahead = after(item);
    Vec next[2] = {load(item), load(ahead)};
    for (int k = tid; k < 2 * dim; k += 256) {
        const float *w = k < dim ? a.q_norm : a.k_norm;
        s_norm[k >= dim][k < dim ? k : k - dim] = w ? w[k < dim ? k : k - dim] : 1.f;
    }
    for (int x = tid; x < n * half; x += 256) {
        const int t = x / half, i = x - t * half;
        const float2 r = turn_of(a, t0 + t, i, a.rot);
        s_cos[t][i] = r.x, s_sin[t][i] = r.y;
    }
    if (tid < n) {
        const int seq = a.seq[t0 + tid], pos = a.pos[t0 + tid];
        int page = -1;
        if (seq >= 0 && seq < int(a.table.rows)) page = page_of(a.table.p + size_t(seq) * a.table.width, a.table.width, a.kv.page, a.kv.pages, pos);
        s_vec[tid] = page < 0 ? -1 : slot_of(page, heads, a.kv.page, 0, uint32_t(pos) % a.kv.page);
    }
    __syncthreads();
    auto store = [&](auto *dst, const float *x) {
        using D = std::remove_pointer_t<decltype(dst)>;
        if (!in) return;
        if (apart) {
            store_some(dst + at[0], some_of<D, 4>(x), past);
            store_some(dst + at[1], some_of<D, 4>(x + 4), past);
        } else {
            store_some(dst + at[0], some_of<D, 8>(x), past);
        }
    };
    for (; item.t < n; item = after(item)) {
        const int t = item.t, h = item.h;
        const int kind = h < int(a.q_heads) ? 0 : h < int(a.q_heads) + heads ? 1 : 2;  // q, k, v
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = value_at(next[0].x[k / 4], k % 4);
        if (dim < 8 * W && !in)
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = 0.f;
        ahead = after(ahead);
        next[0] = next[1];
        next[1] = load(ahead);
        if (kind < 2) {
            if (kind == 0 ? a.q_norm : a.k_norm) {
                float ss = 0.f;
#pragma unroll
                for (int k = 0; k < 8; k++) ss = __fmaf_rn(x[k], x[k], ss);
                ss = group_reduce<W>(ss, [](float a, float b) { return a + b; });
                const float ms = ss * (1.f / float(dim)) + a.eps;
                const float r = ms > 1e-30f ? root_reciprocal(ms) : 1.f / sqrtf(ms);  // the instruction takes no subnormals
                const f32x4 w0 = *reinterpret_cast<const f32x4 *>(&s_norm[kind][at[0]]), w1 = *reinterpret_cast<const f32x4 *>(&s_norm[kind][at[1]]);
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = x[k] * r * (k < 4 ? w0[k] : w1[k - 4]);
            }
            if (turns) {
                const f32x4 cs = *reinterpret_cast<const f32x4 *>(&s_cos[t][4 * c]), sn = *reinterpret_cast<const f32x4 *>(&s_sin[t][4 * c]);
                auto turn = [](float &p, float &q, float c, float s) {
                    const float y = p;
                    p = y * c - q * s;
                    q = q * c + y * s;
                };
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (!a.adjacent) turn(x[k], x[4 + k], cs[k], sn[k]);
                    else if (8 * c + 2 * k < int(a.rot)) turn(x[2 * k], x[2 * k + 1], cs[k], sn[k]);
                }
            }
        }
        const int hk = h - int(a.q_heads) - (kind == 2 ? heads : 0);
        if (kind == 0) {
            store(static_cast<O *>(a.q) + ((t0 + t) * a.q_heads + h) * dim, x);
            continue;
        }
        if (kind == 1 && a.k) store(static_cast<O *>(a.k) + ((t0 + t) * heads + hk) * dim, x);
        const int64_t vec = s_vec[t] + int64_t(hk) * a.kv.page;
        if (s_vec[t] < 0) continue;
        if constexpr (scaled<C>) {
            uint32_t top = 0;  // of the magnitudes' bits: infinities and NaN come above every number
#pragma unroll
            for (int k = 0; k < 8; k++) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
            top = group_reduce<W>(top, [](uint32_t a, uint32_t b) { return max(a, b); });
            const float m = __uint_as_float(top);
            const bool fine = top < 0x7f800000u, some = fine && m > kTinyMax;
            const float scale = over_code_max<C>(m), inv = code_max_over<C>(m, scale);
            if (c == 0) (kind == 1 ? a.kv.k_scale : a.kv.v_scale)[vec] = some ? scale : fine ? 0.f : NAN;
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] *= inv;
            if (!some)
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = 0.f;
        }
        store(static_cast<C *>(kind == 1 ? a.kv.k : a.kv.v) + vec * dim, x);
    }
}

// Vectors that are no whole eights: one workgroup a position of a sequence. 20 000 positions of 8 heads of 60: 31 us (of 64:
// 11).
template <class C, class O> __global__ __launch_bounds__(256) void read_row_kernel(ReadArgs a) {
    const int dim = a.kv.dim, heads = a.kv.heads;
    for (int64_t block = blockIdx.x; block < int64_t(a.most) * a.table.rows; block += gridDim.x) {
        const int64_t seq = block / a.most, pos = block - seq * a.most;
        const bool there = pos < clamp_len(a.lens[seq], a.table.width, a.kv.page);
        const int page = there ? page_of(a.table.p + seq * a.table.width, a.table.width, a.kv.page, a.kv.pages, pos) : -1;
        const int64_t out = block * heads * dim;
        for (int i = threadIdx.x; i < heads * dim; i += 256) {
            float k = 0.f, v = 0.f;
            if (page >= 0) {
                const int64_t slot = slot_of(page, heads, a.kv.page, i / dim, pos % a.kv.page);
                k = to_f32(static_cast<const C *>(a.kv.k)[slot * dim + i % dim]);
                v = to_f32(static_cast<const C *>(a.kv.v)[slot * dim + i % dim]);
                if constexpr (scaled<C>) k *= a.kv.k_scale[slot], v *= a.kv.v_scale[slot];
            }
            static_cast<O *>(a.k)[out + i] = O(k);
            static_cast<O *>(a.v)[out + i] = O(v);
        }
    }
}

// kReadTokens positions of a sequence a workgroup, W lanes a vector, two vectors' keys and values on
// their way at a time. Eight prompts of 4096, 8 heads of 128 from e4m3: 181 MB in 43 us, 4.2 TB/s; with
// ordinary stores 38, and 8 more until the next kernel starts.
template <class C, class O, int W> __global__ __launch_bounds__(256) void read_kernel(ReadArgs a, bool past) {
    __shared__ int64_t s_vec[kReadTokens];
    const int tid = threadIdx.x, c = tid % W, dim = a.kv.dim, heads = a.kv.heads;
    const int64_t blocks = (int64_t(a.most) + kReadTokens - 1) / kReadTokens;
    constexpr int G = 256 / W;
    for (int64_t block = blockIdx.x; block < blocks * a.table.rows; block += gridDim.x) {
        const int64_t seq = block / blocks, p0 = (block - seq * blocks) * kReadTokens;
        const int n = int(min<int64_t>(kReadTokens, a.most - p0)), items = n * heads;
        if (tid < n) {
            int64_t vec = -1;
            if (p0 + tid < clamp_len(a.lens[seq], a.table.width, a.kv.page)) {
                const int32_t page = page_of(a.table.p + seq * a.table.width, a.table.width, a.kv.page, a.kv.pages, p0 + tid);
                if (page >= 0) vec = slot_of(page, heads, a.kv.page, 0, uint32_t(p0 + tid) % a.kv.page);
            }
            s_vec[tid] = vec;
        }
        __syncthreads();
        for (int item = tid / W; item < items && 8 * c < dim; item += 2 * G) {
            Some<C, 8> raw[2][2];
            float scale[2][2];
            bool there[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int i = min(item + u * G, items - 1), p = i / heads;
                there[u] = s_vec[p] >= 0;
                const int64_t vec = there[u] ? s_vec[p] + int64_t(i - p * heads) * a.kv.page : 0;
                raw[u][0] = load_some<C, 8>(static_cast<const C *>(a.kv.k) + vec * dim + 8 * c);
                raw[u][1] = load_some<C, 8>(static_cast<const C *>(a.kv.v) + vec * dim + 8 * c);
                scale[u][0] = scaled<C> ? a.kv.k_scale[vec] : 1.f;
                scale[u][1] = scaled<C> ? a.kv.v_scale[vec] : 1.f;
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if (item + u * G >= items) break;
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    float x[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = there[u] ? value_at(raw[u][y], k) * scale[u][y] : 0.f;
                    store_some(static_cast<O *>(y ? a.v : a.k) + ((seq * a.most + p0) * heads + item + u * G) * dim + 8 * c, some_of<O, 8>(x), past);
                }
            }
        }
        __syncthreads();
    }
}

// One workgroup a (sequence, head): the head's part of a copied page, the first also the table's row.
// P: what a thread copies at once. 512 beams, 64-position pages of 4 bfloat16 heads of 128: 12 us, 4.2
// TB/s of the copies; one workgroup a sequence and bytes: 127.
template <class P> __global__ __launch_bounds__(256) void fork_kernel(ForkArgs a) {
    const uint32_t r = blockIdx.x, h = blockIdx.y, w = r % a.beams, g = r - w;
    const Fork f = fork_of(a.parents + g, a.beams, w, a.lens + g, a.table.width, a.kv.page);
    const int32_t p = a.parents[r];
    const bool ok = p >= 0 && uint32_t(p) < a.beams;
    const int32_t *from = a.table.p + size_t(g + (ok ? p : 0)) * a.table.width;
    if (h == 0) {
        int32_t *to = a.table_out + size_t(r) * a.table.width;
        const uint32_t cols = ok ? f.full + (f.tail > 0) : 0;
        for (uint32_t i = threadIdx.x; i < a.table.width; i += 256)
            to[i] = i >= cols ? -1 : i == f.full && f.copy ? a.spare[r] : from[i];
        if (threadIdx.x == 0) a.lens_out[r] = f.len, a.used[r] = f.copy;
    }
    if (!f.copy) return;
    const int32_t src = from[f.full], dst = a.spare[r];
    if (src < 0 || uint32_t(src) >= a.kv.pages || dst < 0 || uint32_t(dst) >= a.kv.pages || src == dst) return;
    const bool coded = a.kv.type == T_I8 || a.kv.type == T_E4M3;
    const size_t vec = size_t(a.kv.dim) * (coded ? 1 : 2);
    const int64_t s0 = slot_of(src, a.kv.heads, a.kv.page, h, 0), d0 = slot_of(dst, a.kv.heads, a.kv.page, h, 0);
    const P *ks = reinterpret_cast<const P *>(static_cast<const char *>(a.kv.k) + s0 * vec), *vs = reinterpret_cast<const P *>(static_cast<const char *>(a.kv.v) + s0 * vec);
    P *kd = reinterpret_cast<P *>(static_cast<char *>(a.kv.k) + d0 * vec), *vd = reinterpret_cast<P *>(static_cast<char *>(a.kv.v) + d0 * vec);
    const uint32_t n = uint32_t(f.tail * vec / sizeof(P));
    uint32_t i = threadIdx.x;
    if (!a.kv.v) {  // latent vectors
        for (; i < n; i += 256) kd[i] = ks[i];
        return;
    }
    for (; i + 768 < n; i += 1024) {  // all on their way before the first is written
        P x[4], y[4];
#pragma unroll
        for (int u = 0; u < 4; u++) x[u] = ks[i + 256 * u], y[u] = vs[i + 256 * u];
#pragma unroll
        for (int u = 0; u < 4; u++) kd[i + 256 * u] = x[u], vd[i + 256 * u] = y[u];
    }
    for (; i < n; i += 256) kd[i] = ks[i], vd[i] = vs[i];
    if (coded)
        for (uint32_t e = threadIdx.x; e < f.tail; e += 256)
            a.kv.k_scale[d0 + e] = a.kv.k_scale[s0 + e], a.kv.v_scale[d0 + e] = a.kv.v_scale[s0 + e];
}

// `each` tokens a workgroup: their turns are looked up once for all heads, then a thread takes two fours of a vector at a
// time, the two that turn with each other where pairs are halves apart, or two neighbours; in place only those that turn.
// The first kRotateBatch are asked for before the turns. 65 521 tokens of 16 heads of 80 in bf16 (335 MB): 81 us (4.1 TB/s),
// 77 of them without the turns; four of a thread at a time 95, and past the caches, loads and stores, 101.
constexpr int kRotateTokens = 8, kRotateBatch = 2;
template <class T> __global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a, int each, bool in_place) {
    __shared__ __align__(16) float s_cos[kRotateTokens][128], s_sin[kRotateTokens][128];
    __shared__ double s_step[128];
    const int tid = threadIdx.x, half = a.rot / 2, turning = a.rot / 8, lanes = in_place ? turning : a.dim / 8;
    const int heads = a.heads;
    struct Item {
        int t, h, c;
    };
    auto item_at = [&](int x) {
        const int v = x / lanes, t = v / heads;
        return Item{t, v - t * heads, x - v * lanes};
    };
    const Item step = item_at(256);
    auto after = [&](Item i) {
        i.t += step.t, i.h += step.h, i.c += step.c;
        if (i.c >= lanes) i.c -= lanes, i.h++;
        if (i.h >= heads) i.h -= heads, i.t++;
        return i;
    };
    // An item's two fours.
    auto places = [&](Item i, int *at) {
        if (i.c < turning) {
            at[0] = a.first + (a.adjacent ? 8 : 4) * i.c;
            at[1] = a.adjacent ? at[0] + 4 : at[0] + half;
        } else {
            const int c = 8 * (i.c - turning);
            at[0] = c < int(a.first) ? c : c + int(a.rot);
            at[1] = at[0] + 4;
        }
    };
    const int64_t t0 = int64_t(blockIdx.x) * each;
    const int n = int(min<int64_t>(each, a.n - t0)), items = n * heads * lanes;
    int pos[kRotateTokens / 2];  // of the thread's turns, half of at most 256 values
#pragma unroll
    for (int u = 0; u < kRotateTokens / 2; u++) {
        const int x = tid + 256 * u, t = half ? x / half : n;
        if (t < n) pos[u] = a.at[(t0 + t) * a.axes.count + a.axes.axis[x - t * half]];
    }
    const T *const x0 = static_cast<const T *>(a.x) + t0 * a.x_stride;
    T *const y0 = static_cast<T *>(a.out) + t0 * a.out_stride;
    struct Vec {
        Some<T, 4> x[2];
    };
    auto load = [&](Item i) {
        if (i.t >= n) i = Item{0, 0, 0};
        int at[2];
        places(i, at);
        const T *src = x0 + i.t * a.x_stride + i.h * a.x_head;
        return Vec{load_some<T, 4>(src + at[0]), load_some<T, 4>(src + at[1])};
    };
    Item item = item_at(tid);
    Vec next[kRotateBatch];
    auto load_batch = [&](Item i) {
#pragma unroll
        for (int u = 0; u < kRotateBatch; u++) next[u] = load(i), i = after(i);
    };
    load_batch(item);
    for (int i = tid; i < half; i += 256) s_step[i] = turns_a_step(a, i, a.rot);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kRotateTokens / 2; u++) {
        const int x = tid + 256 * u, t = half ? x / half : n, i = x - t * half;
        if (t >= n) break;
        const float2 r = turned(double(pos[u]) * s_step[i]);
        s_cos[t][i] = r.x, s_sin[t][i] = a.back ? -r.y : r.y;
    }
    __syncthreads();
    for (int done = tid; done < items; done += 256 * kRotateBatch) {
#pragma unroll
        for (int u = 0; u < kRotateBatch; u++, item = after(item)) {
            if (item.t >= n) break;
            int at[2];
            places(item, at);
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = value_at(next[u].x[k / 4], k % 4);
            if (item.c < turning) {
                const f32x4 cs = *reinterpret_cast<const f32x4 *>(&s_cos[item.t][4 * item.c]), sn = *reinterpret_cast<const f32x4 *>(&s_sin[item.t][4 * item.c]);
                auto turn = [](float &p, float &q, float c, float s) {
                    const float y = p;
                    p = y * c - q * s;
                    q = q * c + y * s;
                };
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (!a.adjacent) turn(x[k], x[4 + k], cs[k], sn[k]);
                    else turn(x[2 * k], x[2 * k + 1], cs[k], sn[k]);
                }
            }
            T *dst = y0 + item.t * a.out_stride + item.h * a.out_head;
            store_some(dst + at[0], some_of<T, 4>(x), false);
            store_some(dst + at[1], some_of<T, 4>(x + 4), false);
        }
        if (done + 256 * kRotateBatch < items) load_batch(item);
    }
}

// A thread a pair, or a value that is not rotated: sizes that are no eights.
template <class T> __global__ __launch_bounds__(256) void rotate_row_kernel(RotateArgs a) {
    const uint32_t half = a.rot / 2, each = a.dim - half;  // a vector's items
    const T *const x = static_cast<const T *>(a.x);
    T *const y = static_cast<T *>(a.out);
    for (int64_t t = blockIdx.x; t < a.n; t += gridDim.x) {
        for (uint32_t item = threadIdx.x; item < a.heads * each; item += 256) {
            const uint32_t h = item / each, e = item - h * each;
            const T *from = x + t * a.x_stride + h * a.x_head;
            T *to = y + t * a.out_stride + h * a.out_head;
            if (e >= half) {
                const uint32_t c = e - half < a.first ? e - half : e + half;
                if (from != to) to[c] = from[c];
                continue;
            }
            const uint32_t i = a.first + (a.adjacent ? 2 * e : e), j = i + (a.adjacent ? 1 : half);
            float2 r = turned(double(a.at[t * a.axes.count + a.axes.axis[e]]) * turns_a_step(a, e, a.rot));
            if (a.back) r.y = -r.y;
            const float p = to_f32(from[i]), q = to_f32(from[j]);
            to[i] = T(p * r.x - q * r.y);
            to[j] = T(q * r.x + p * r.y);
        }
    }
}

// f(lanes of a vector): the power of two that holds its eights.
template <class F> void with_lanes(uint32_t dim, F &&f) {
    if (dim <= 32) f(std::integral_constant<int, 4>{});
    else if (dim <= 64) f(std::integral_constant<int, 8>{});
    else if (dim <= 128) f(std::integral_constant<int, 16>{});
    else f(std::integral_constant<int, 32>{});
}

}  // namespace

void launch_append(const AppendArgs &a, hipStream_t s) {
    const double values = double(a.n) * (a.q_heads + 2 * a.kv.heads) * a.kv.dim;
    const bool eights = a.kv.dim % 8 == 0 && (a.adjacent || a.rot % 8 == 0);
    ProbeScope probe("text_append", s, 10 * values, values * (type_bytes(a.type) + 2), eights ? "text_append_eights" : "text_append_row");
    // Four tokens a workgroup share their lookups once that leaves work for every compute unit.
    const int each = a.n >= 4096 ? kAppendTokens : 1;
    const bool past = double(a.n) * a.kv.dim * (2.0 * a.q_heads + 2.0 * a.kv.heads * type_bytes(a.kv.type)) > kHeld;
    with_type(a.type, [&](auto t) {
        with_type16(a.out_type, [&](auto o) {
            with_cache(a.kv.type, [&](auto c) {
                using T = decltype(t);
                using O = decltype(o);
                using C = decltype(c);
                if (!eights) {
                    hipLaunchKernelGGL((append_row_kernel<T, O, C>), dim3(a.n, a.q_heads + 2 * a.kv.heads), dim3(64), 0, s, a);
                    return;
                }
                with_lanes(a.kv.dim, [&](auto w) {
                    hipLaunchKernelGGL((append_kernel<T, O, C, decltype(w)::value>), dim3((a.n + each - 1) / each), dim3(256), 0, s, a, each, past);
                });
            });
        });
    });
    OCR_HIP(hipGetLastError());
}

void launch_rotate(const RotateArgs &a, hipStream_t s) {
    const double values = double(a.n) * a.heads * a.dim;
    const bool in_place = a.x == a.out, eights = a.dim % 8 == 0 && a.first % 8 == 0 && a.rot % 8 == 0 && a.x_stride < 1 << 30 && a.out_stride < 1 << 30;
    ProbeScope probe("text_rotate", s, 3 * values, 2 * values * type_bytes(a.type), eights ? "text_rotate_eights" : "text_rotate_row");
    const uint32_t lanes = in_place ? a.rot / 8 : a.dim / 8;
    if (eights && lanes == 0) return;  // in place, and nothing turns
    // Many tokens share the frequencies' and turns' way: 65 521 of 16 heads of 80 84 us, a workgroup each 199; few go over all compute units.
    const int each = a.n >= 2048 ? int(std::min<uint32_t>(kRotateTokens, std::max<uint32_t>(1, 2048 / (a.heads * lanes)))) : 1;
    with_type(a.type, [&](auto t) {
        using T = decltype(t);
        if (eights) hipLaunchKernelGGL((rotate_kernel<T>), dim3((a.n + each - 1) / each), dim3(256), 0, s, a, each, in_place);
        else hipLaunchKernelGGL((rotate_row_kernel<T>), dim3(std::min<uint32_t>(a.n, 1 << 22)), dim3(256), 0, s, a);
    });
    OCR_HIP(hipGetLastError());
}

void launch_read(const ReadArgs &a, hipStream_t s) {
    const double values = 2.0 * a.table.rows * a.most * a.kv.heads * a.kv.dim;
    const bool eights = a.kv.dim % 8 == 0;
    ProbeScope probe("text_read", s, values, values * (type_bytes(a.kv.type) + 2), eights ? "text_read_eights" : "text_read_row");
    // Workgroups go on to further positions past what a grid holds.
    const auto grid = [](int64_t blocks) { return dim3(unsigned(std::min<int64_t>(blocks, 1 << 22))); };
    with_cache(a.kv.type, [&](auto c) {
        with_type16(a.type, [&](auto o) {
            using C = decltype(c);
            using O = decltype(o);
            if (!eights) {
                hipLaunchKernelGGL((read_row_kernel<C, O>), grid(int64_t(a.most) * a.table.rows), dim3(256), 0, s, a);
                return;
            }
            const int64_t blocks = (int64_t(a.most) + kReadTokens - 1) / kReadTokens * a.table.rows;
            with_lanes(a.kv.dim, [&](auto w) { hipLaunchKernelGGL((read_kernel<C, O, decltype(w)::value>), grid(blocks), dim3(256), 0, s, a, 2 * values > kHeld); });
        });
    });
    OCR_HIP(hipGetLastError());
}

void launch_fork(const ForkArgs &a, hipStream_t s) {
    const bool pieces = whole_pieces(a.kv);
    ProbeScope probe("text_fork", s, 0, 8.0 * a.table.rows * a.table.width, pieces ? "text_fork_pieces" : "text_fork_bytes");
    const dim3 grid(a.table.rows, a.kv.heads);
    if (pieces) hipLaunchKernelGGL(fork_kernel<u32x4>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(fork_kernel<uint8_t>, grid, dim3(256), 0, s, a);
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
