// Argument checks of the text decoder's operators. Whatever a kernel cannot find out for itself is
// refused here; page numbers, lengths and positions live in device memory and are checked by the
// kernels (text_rules.h).
#include "text.h"

#include <cmath>
#include <cstring>
#include <string>

#include "common.h"

namespace ocr {

namespace {

void need(const void *p, const char *what) {
    if (!p) fail(std::string(what) + " is NULL");
}
void need_type(int t, bool f32, const char *what) {
    if (t == T_F16 || t == T_BF16 || (f32 && t == T_F32)) return;
    fail(std::string(what) + ": type " + std::to_string(t) + (f32 ? " is not float32, float16 or bfloat16" : " is not float16 or bfloat16"));
}
void aligned(const void *p, size_t to, const char *what) {
    if (reinterpret_cast<uintptr_t>(p) % to) fail(std::string(what) + " is not aligned to its values");
}
void check_cache(const KvCache &kv) {
    need(kv.k, "cache keys");
    need(kv.v, "cache values");
    if (kv.type != T_F16 && kv.type != T_BF16 && kv.type != T_I8 && kv.type != T_E4M3)
        fail("cache: type " + std::to_string(kv.type) + " is not float16, bfloat16, int8 or e4m3");
    if (kv.pages == 0 || kv.heads == 0 || kv.page == 0 || kv.dim == 0) fail("cache: empty");
    if (kv.dim > 256) fail("cache: heads of " + std::to_string(kv.dim) + " values (at most 256)");
    if (kv.page > 1024) fail("cache: pages of " + std::to_string(kv.page) + " positions (at most 1024)");
    if (kv.heads > 1024) fail("cache: " + std::to_string(kv.heads) + " heads (at most 1024)");
    if (kv.pages > 0x7fffffffu) fail("cache: more pages than a table can name");
    if (kv.type == T_I8 || kv.type == T_E4M3) {
        need(kv.k_scale, "cache key scales");
        need(kv.v_scale, "cache value scales");
        aligned(kv.k_scale, 4, "cache key scales");
        aligned(kv.v_scale, 4, "cache value scales");
    }
    aligned(kv.k, type_bytes(kv.type), "cache keys");
    aligned(kv.v, type_bytes(kv.type), "cache values");
}
void check_table(const PageTable &t, uint32_t page) {
    if (t.rows == 0) return;  // nothing of it is read, and an empty array may have no address
    need(t.p, "page table");
    aligned(t.p, 4, "page table");
    if (t.width == 0) fail("page table: no columns");
    if (int64_t(t.width) * page > 0x7fffffffll) fail("page table: more positions than a length can hold");
    if (t.rows > 0x7fffffffu) fail("page table: too many rows");
}
void check_heads(uint32_t q_heads, uint32_t kv_heads) {
    if (q_heads == 0 || q_heads > 1024 || q_heads % kv_heads)
        fail(std::to_string(q_heads) + " query heads over " + std::to_string(kv_heads) + " key heads");
}
void check_scores(float scale, float cap) {
    if (!std::isfinite(scale)) fail("the scores' scale is not finite");
    if (!std::isfinite(cap) || cap < 0) fail("the scores' cap is negative or not finite");
}
void check_stride(int64_t stride, int64_t row, const char *what) {
    if (stride < row) fail(std::string(what) + ": rows of " + std::to_string(row) + " values every " + std::to_string(stride));
    if (stride > (int64_t(1) << 40)) fail(std::string(what) + ": stride too large");
}
bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

}  // namespace

bool check_append(const AppendArgs &a) {
    check_cache(a.kv);
    check_table(a.table, a.kv.page);
    check_heads(a.q_heads, a.kv.heads);
    need_type(a.type, true, "projections");
    need_type(a.out_type, false, "queries");
    check_stride(a.stride, int64_t(a.q_heads + 2 * a.kv.heads) * a.kv.dim, "projections");
    if (a.rot > a.kv.dim || a.rot % 2) fail("rotation of " + std::to_string(a.rot) + " of " + std::to_string(a.kv.dim) + " values");
    if (a.rot && !std::isfinite(a.log2_theta)) fail("the rotation's base is not a positive number");
    if (!(a.eps >= 0) || !std::isfinite(a.eps)) fail("the norms' epsilon is negative or not finite");
    if (a.n > 0x7fffffffu) fail("too many tokens");
    if (a.n == 0) return false;
    need(a.seq, "sequence numbers");
    need(a.pos, "positions");
    need(a.qkv, "projections");
    need(a.q, "queries");
    for (const void *p : {static_cast<const void *>(a.seq), static_cast<const void *>(a.pos), static_cast<const void *>(a.q_norm),
                          static_cast<const void *>(a.k_norm)})
        aligned(p, 4, "an array of 4-byte values");
    aligned(a.qkv, type_bytes(a.type), "projections");
    aligned(a.q, 2, "queries");
    aligned(a.k, 2, "keys");
    const size_t in = (size_t(a.n - 1) * a.stride + size_t(a.q_heads + 2 * a.kv.heads) * a.kv.dim) * type_bytes(a.type);
    if (overlap(a.q, size_t(a.n) * a.q_heads * a.kv.dim * 2, a.qkv, in) ||
        (a.k && overlap(a.k, size_t(a.n) * a.kv.heads * a.kv.dim * 2, a.qkv, in)))
        fail("queries or keys overlap the projections");
    return true;
}

bool check_read(const ReadArgs &a) {
    check_cache(a.kv);
    check_table(a.table, a.kv.page);
    need_type(a.type, false, "values read");
    if (a.table.rows == 0 || a.most == 0) return false;
    need(a.lens, "lengths");
    need(a.k, "keys");
    need(a.v, "values");
    aligned(a.lens, 4, "lengths");
    aligned(a.k, 2, "keys");
    aligned(a.v, 2, "values");
    if (a.most > 0x7fffffffu) fail("too many positions");
    return true;
}

bool check_attention(const AttentionArgs &a) {
    need_type(a.type, false, "attention");
    if (a.kv_heads == 0 || a.dim == 0 || a.dim > 256) fail("attention: heads of " + std::to_string(a.dim) + " values (1 to 256)");
    check_heads(a.q_heads, a.kv_heads);
    check_scores(a.scale, a.cap);
    check_stride(a.q_stride, int64_t(a.q_heads) * a.dim, "queries");
    check_stride(a.k_stride, int64_t(a.kv_heads) * a.dim, "keys");
    check_stride(a.v_stride, int64_t(a.kv_heads) * a.dim, "values");
    check_stride(a.out_stride, int64_t(a.q_heads) * a.dim, "outputs");
    if (a.n > 0x3fffffffu) fail("attention: too many tokens");
    if (a.docs && a.ndocs > 0x3fffffffu) fail("attention: too many documents");
    if (a.n == 0) return false;
    need(a.q, "queries");
    need(a.k, "keys");
    need(a.v, "values");
    need(a.out, "outputs");
    for (const void *p : {a.q, a.k, a.v, static_cast<const void *>(a.out)}) aligned(p, 2, "queries, keys, values or outputs");
    for (const void *p : {static_cast<const void *>(a.docs), static_cast<const void *>(a.prefix), static_cast<const void *>(a.slopes)})
        aligned(p, 4, "an array of 4-byte values");
    const size_t row_q = size_t(a.q_heads) * a.dim, row_k = size_t(a.kv_heads) * a.dim;
    const size_t n1 = a.n - 1, no = (n1 * a.out_stride + row_q) * 2;
    if (overlap(a.out, no, a.q, (n1 * a.q_stride + row_q) * 2) || overlap(a.out, no, a.k, (n1 * a.k_stride + row_k) * 2) ||
        overlap(a.out, no, a.v, (n1 * a.v_stride + row_k) * 2))
        fail("attention: the outputs overlap an input");
    return true;
}

bool check_decode(const DecodeArgs &a) {
    check_cache(a.kv);
    check_table(a.table, a.kv.page);
    check_heads(a.q_heads, a.kv.heads);
    need_type(a.type, false, "queries");
    check_scores(a.scale, a.cap);
    check_stride(a.q_stride, int64_t(a.q_heads) * a.kv.dim, "queries");
    check_stride(a.out_stride, int64_t(a.q_heads) * a.kv.dim, "outputs");
    if ((a.kv.type == T_F16 || a.kv.type == T_BF16) && a.kv.type != a.type)
        fail("a 16-bit cache is read by queries of its own type");
    if (a.table.rows == 0) return false;
    need(a.lens, "lengths");
    need(a.q, "queries");
    need(a.out, "outputs");
    aligned(a.lens, 4, "lengths");
    aligned(a.slopes, 4, "slopes");
    aligned(a.q, 2, "queries");
    aligned(a.out, 2, "outputs");
    const size_t n1 = a.table.rows - 1, row = size_t(a.q_heads) * a.kv.dim;
    if (overlap(a.out, (n1 * a.out_stride + row) * 2, a.q, (n1 * a.q_stride + row) * 2)) fail("the outputs overlap the queries");
    return true;
}

bool check_fork(const ForkArgs &a) {
    check_cache(a.kv);
    check_table(a.table, a.kv.page);
    if (a.beams == 0 || a.beams > kMostBeams || a.table.rows % a.beams)
        fail("fork: " + std::to_string(a.table.rows) + " sequences in groups of " + std::to_string(a.beams) + " beams (at most " +
             std::to_string(kMostBeams) + ")");
    if (a.table.rows == 0) return false;
    need(a.lens, "lengths");
    need(a.parents, "parents");
    need(a.spare, "spare pages");
    need(a.table_out, "the new table");
    need(a.lens_out, "the new lengths");
    need(a.used, "used");
    for (const void *p : {static_cast<const void *>(a.lens), static_cast<const void *>(a.parents), static_cast<const void *>(a.spare),
                          static_cast<const void *>(a.table_out), static_cast<const void *>(a.lens_out), static_cast<const void *>(a.used)})
        aligned(p, 4, "an array of 4-byte values");
    const size_t rows = a.table.rows, cells = rows * a.table.width * 4;
    if (overlap(a.table_out, cells, a.table.p, cells) || overlap(a.lens_out, rows * 4, a.lens, rows * 4))
        fail("fork: the new table or lengths overlap the old ones");
    return true;
}

bool check_beam(const BeamArgs &a) {
    need_type(a.type, true, "logits");
    if (a.beams == 0 || a.beams > kMostBeams) fail("beam search: " + std::to_string(a.beams) + " beams (1 to " + std::to_string(kMostBeams) + ")");
    if (a.vocab == 0 || a.vocab > (1u << 28)) fail("beam search: a vocabulary of " + std::to_string(a.vocab));
    if (a.eos >= 0 && uint32_t(a.eos) >= a.vocab) fail("beam search: the end token is not in the vocabulary");
    if (a.finished && a.eos < 0) fail("beam search: finished beams need an end token");
    check_stride(a.stride, a.vocab, "logits");
    if (uint64_t(a.groups) * a.beams > 0x7fffffffu) fail("beam search: too many beams");
    if (a.groups == 0) return false;
    need(a.logits, "logits");
    need(a.scores, "scores");
    need(a.out_scores, "new scores");
    need(a.parents, "parents");
    need(a.tokens, "tokens");
    aligned(a.logits, type_bytes(a.type), "logits");
    for (const void *p : {static_cast<const void *>(a.scores), static_cast<const void *>(a.finished), static_cast<const void *>(a.out_scores),
                          static_cast<const void *>(a.parents), static_cast<const void *>(a.tokens), static_cast<const void *>(a.out_finished)})
        aligned(p, 4, "an array of 4-byte values");
    return true;
}

}  // namespace ocr
