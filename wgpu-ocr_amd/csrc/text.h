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
};

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
};

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

// The launches (arguments checked), queued on s.
void launch_append(const AppendArgs &a, hipStream_t s);
void launch_read(const ReadArgs &a, hipStream_t s);
void launch_attention(const AttentionArgs &a, hipStream_t s);
void launch_decode(Ctx &c, const DecodeArgs &a, hipStream_t s);
void launch_fork(const ForkArgs &a, hipStream_t s);
void launch_beam(Ctx &c, const BeamArgs &a, hipStream_t s);

}  // namespace ocr
