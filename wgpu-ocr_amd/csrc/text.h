// The text decoder's operators (kernels/text_*.hip, kernels/beam.hip): a paged cache of keys and
// values that is quantised as it is written, attention over packed prompts and of single tokens over
// the cache, beam search. The reference has no counterpart: its recognisers end in CTC.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "text_rules.h"

namespace ocr {

class Ctx;

// Element types, as in the C ABI.
enum Type : int { T_F32 = 0, T_F16 = 1, T_BF16 = 2, T_I8 = 3, T_E4M3 = 4 };
inline size_t type_bytes(int t) { return t == T_F32 ? 4 : t == T_F16 || t == T_BF16 ? 2 : 1; }

// Keys and values [pages][heads][page][dim], and for the 8-bit types a scale a vector.
struct KvCache {
    void *k, *v;
    float *k_scale, *v_scale;
    uint32_t pages, heads, page, dim;
    int type;
};

// Whether its vectors are whole 16-byte pieces.
inline bool whole_pieces(const KvCache &c) {
    return c.dim * type_bytes(c.type) % 16 == 0 && reinterpret_cast<uintptr_t>(c.k) % 16 == 0 && reinterpret_cast<uintptr_t>(c.v) % 16 == 0;
}

// Every sequence's pages: rows of width entries, a negative one where there is none.
struct PageTable {
    const int32_t *p;
    uint32_t rows, width;
};

struct AppendArgs {
    KvCache kv;
    PageTable table;
    const int32_t *seq, *pos;
    const void *qkv;
    int type;
    uint32_t n, q_heads;
    int64_t stride;
    const float *q_norm, *k_norm;
    float eps;
    uint32_t rot;
    double log2_theta;
    int adjacent;
    void *q, *k;
    int out_type;
    const int32_t *at = nullptr;  // with axes: [n][axes.count] positions that the rotation goes by
    AxisMap axes{};
};

// Positions of several axes, as in the C ABI (ocr_axes).
struct Axes {
    const int32_t *at;
    uint32_t count;
    uint32_t pairs[4];
    int in_turn, own;
};

struct RotateArgs {
    const void *x;
    void *out;
    int type;
    uint32_t n, heads, dim;
    int64_t x_stride, x_head, out_stride, out_head;
    uint32_t first, rot;
    double log2_theta;
    int adjacent, back;
    const int32_t *at;
    AxisMap axes;
};

// What attention adds up: weights [sequences or documents][key heads][most]; window: a document's last queries that
// count (0: all of them).
struct Weights {
    float *p;
    uint32_t most, window;
};

struct EvictArgs {
    KvCache kv;
    PageTable table;
    const int32_t *lens, *newest;
    const float *weights;
    const int32_t *held;
    uint32_t most, keep, first, recent;
    float *weights_out;
    int32_t *held_out, *lens_out;
};

// A pool of latent vectors [pages][page][rank + rot].
struct LatentCache {
    void *p;
    uint32_t pages, page, rank, rot;
    int type;
};

struct LatentAppendArgs {
    LatentCache c;
    PageTable table;
    const int32_t *seq, *pos;
    const void *x;
    int type;
    uint32_t n;
    int64_t stride;
    const float *norm;
    float eps;
    double log2_theta;
    int adjacent;
    void *out;
    const int32_t *at;
    AxisMap axes;
};

struct LatentDecodeArgs {
    LatentCache c;
    PageTable table;
    const int32_t *lens;
    const void *q;
    void *out;
    uint32_t heads;
    int64_t q_stride, out_stride;
    float scale;
};

struct LatentAttentionArgs {
    const void *q, *k, *r, *v;
    void *out;
    int type;
    uint32_t n, heads, key, rot, value;
    int64_t q_stride, k_stride, k_head, r_stride, v_stride, v_head, out_stride;
    const int32_t *docs;
    uint32_t ndocs;
    const int32_t *prefix;
    float scale;
};
constexpr uint32_t kMostRank = 512, kMostLatentRot = 128;
// Of a sequence, where kernels count on past the last one in 32 bits.
constexpr uint32_t kMostPlaces = 1u << 30;

struct ReadArgs {
    KvCache kv;
    PageTable table;
    const int32_t *lens;
    uint32_t most;
    int type;
    void *k, *v;
};

struct AttentionArgs {
    const void *q, *k, *v;
    void *out;
    int type;
    uint32_t n, q_heads, kv_heads, dim;
    int64_t q_stride, k_stride, v_stride, out_stride;
    const int32_t *docs;
    uint32_t ndocs;
    const int32_t *prefix;
    float scale, cap;
    const float *slopes;
    float *sums = nullptr;  // the tiles' kernels: every query's reference and one over its sum of weights, [q_heads][2][sums_pitch(n)]
};
OCR_HD int64_t sums_pitch(uint32_t n) { return (int64_t(n) + 63) / 64 * 64; }

struct DecodeArgs {
    KvCache kv;
    PageTable table;
    const int32_t *lens;
    const void *q;
    void *out;
    int type;
    uint32_t q_heads;
    int64_t q_stride, out_stride;
    float scale, cap;
    const float *slopes;
};

struct ForkArgs {
    KvCache kv;
    PageTable table;
    const int32_t *lens, *parents;
    uint32_t beams;
    const int32_t *spare;
    int32_t *table_out, *lens_out, *used;
};

struct BeamArgs {
    const void *logits;
    int type;
    uint32_t groups, beams, vocab;
    int64_t stride;
    const float *scores;
    const int32_t *finished;
    int32_t eos;
    float *out_scores;
    int32_t *parents, *tokens, *out_finished;
};
constexpr uint32_t kMostBeams = 32;

// Checks of the arguments, without a GPU (ocr::Error); false where there is nothing to do.
bool check_append(const AppendArgs &a);
bool check_read(const ReadArgs &a);
bool check_attention(const AttentionArgs &a);
bool check_decode(const DecodeArgs &a);
bool check_fork(const ForkArgs &a);
bool check_beam(const BeamArgs &a);
void check_axes(const Axes &x, uint32_t rot, uint32_t n);
bool check_rotate(const RotateArgs &a);
bool check_weights(const Weights &w, uint32_t rows);
// That weights to be added to lie beside what the (checked) attention reads and writes.
void check_apart(const Weights &w, const AttentionArgs &a);
void check_apart(const Weights &w, const DecodeArgs &a);
bool check_evict(const EvictArgs &a);
bool check_latent_append(const LatentAppendArgs &a);
bool check_latent_decode(const LatentDecodeArgs &a);
bool check_latent_fork(const LatentCache &c, const ForkArgs &a);
bool check_latent_attention(const LatentAttentionArgs &a);

// The launches (arguments checked), queued on s.
void launch_append(const AppendArgs &a, hipStream_t s);
void launch_read(const ReadArgs &a, hipStream_t s);
void launch_rotate(const RotateArgs &a, hipStream_t s);
void launch_attention(const AttentionArgs &a, hipStream_t s);
bool attention_tiles(const AttentionArgs &a);  // whether launch_attention takes the tiles' kernels
void launch_attention_weights(Ctx &c, const AttentionArgs &a, const Weights &w, hipStream_t s);
void launch_decode(Ctx &c, const DecodeArgs &a, hipStream_t s);
void launch_decode_weights(Ctx &c, const DecodeArgs &a, const Weights &w, hipStream_t s);
void launch_single_weights_row(const DecodeArgs &a, const Weights &w, hipStream_t s);  // the weights alone, by the formula
void launch_evict(Ctx &c, const EvictArgs &a, hipStream_t s);
void launch_latent_append(const LatentAppendArgs &a, hipStream_t s);
void launch_latent_decode(Ctx &c, const LatentDecodeArgs &a, hipStream_t s);
void launch_latent_attention(const LatentAttentionArgs &a, hipStream_t s);
void launch_fork(const ForkArgs &a, hipStream_t s);
void launch_beam(Ctx &c, const BeamArgs &a, hipStream_t s);

}  // namespace ocr
