// The text decoder's rules and argument checks on the CPU: page numbers and lengths that lie outside
// the buffers, the keys that a token sees, forks, and every refusal.
#include <cmath>
#include <cstdio>
#include <string>
#include <vector>

#include "common.h"
#include "text.h"

static int failures = 0;
static void check(bool ok, const char *what) {
    if (ok) return;
    std::printf("FAILED: %s\n", what);
    failures++;
}
void ocr::fail(const std::string &msg) { throw Error(msg); }

using namespace ocr;

template <class F> static void refused(F &&f, const char *what) {
    try {
        f();
    } catch (const Error &e) {
        check(std::string(e.what()).size() > 4, what);
        return;
    }
    check(false, what);
}
// `good` passes; with each change it is refused.
template <class A, class Check> struct Refusals {
    A good;
    Check fn;
    template <class M> void operator()(const char *what, M &&change) {
        A a = good;
        change(a);
        refused([&] { fn(a); }, what);
    }
};

static void pages() {
    const int32_t row[4] = {2, -1, 9, 0};
    check(page_of(row, 4, 16, 5, 0) == 2 && page_of(row, 4, 16, 5, 15) == 2, "a page");
    check(page_of(row, 4, 16, 5, 16) == -1 && page_of(row, 4, 16, 5, 32) == -1, "a negative page and one past the pool");
    check(page_of(row, 4, 16, 5, 63) == 0 && page_of(row, 4, 16, 5, 64) == -1 && page_of(row, 4, 16, 5, -1) == -1, "positions outside the table");
    check(page_of(row, 4, 16, 9, 32) == -1 && page_of(row, 4, 16, 10, 32) == 9, "the pool's last page");
    check(slot_of(2000000000, 8, 64, 7, 63) == (int64_t(2000000000) * 8 + 7) * 64 + 63, "slots past 32 bits");
    check(clamp_len(-5, 4, 16) == 0 && clamp_len(64, 4, 16) == 64 && clamp_len(65, 4, 16) == 64, "lengths");
    check(clamp_len(0x7fffffff, 0x1ffffff, 64) == 0x7fffffc0, "the longest length");
}

static void ranges() {
    const int32_t docs[5] = {2, 5, 5, 9, 12}, prefix[4] = {0, 7, 2, 99};
    auto is = [&](int i, int lo, int hi, const int32_t *p) {
        const KeyRange r = key_range(i, 14, docs, 4, p);
        return hi <= lo ? r.hi <= r.lo : r.lo == lo && r.hi == hi;
    };
    check(is(0, 0, 0, prefix) && is(1, 0, 0, prefix), "before the first document");
    check(is(2, 2, 3, prefix) && is(4, 2, 5, prefix), "causal");
    check(is(5, 5, 7, prefix) && is(6, 5, 7, prefix) && is(7, 5, 8, prefix), "prefix, after an empty document");
    check(is(9, 9, 12, prefix) && is(11, 9, 12, prefix), "a prefix longer than its document");
    check(is(12, 0, 0, prefix) && is(13, 0, 0, prefix) && is(14, 0, 0, prefix) && is(-1, 0, 0, prefix), "after the last document");
    check(is(7, 5, 8, nullptr), "no prefix");
    const KeyRange all = key_range(3, 10, nullptr, 1, nullptr);
    check(all.lo == 0 && all.hi == 4, "no documents");
    // Offsets and prefixes that make no sense stay inside the row.
    const int32_t bad[4] = {-2000000000, 7, 3, 2000000000};
    const int32_t wild[3] = {0x7fffffff, -5, 0x7fffffff};
    for (int i = 0; i < 10; i++) {
        const KeyRange r = key_range(i, 10, bad, 3, wild);
        check(r.hi <= r.lo || (r.lo >= 0 && r.hi <= 10), "offsets that do not rise");
    }
    check(key_range(0, 10, bad, 0, nullptr).hi == 0, "no document at all");
}

static void forks() {
    const int32_t parents[4] = {1, 1, 3, -1}, lens[4] = {5, 33, 7, 32};
    const Fork a = fork_of(parents, 4, 0, lens, 4, 16), b = fork_of(parents, 4, 1, lens, 4, 16), c = fork_of(parents, 4, 2, lens, 4, 16),
               d = fork_of(parents, 4, 3, lens, 4, 16);
    check(a.len == 33 && a.full == 2 && a.tail == 1 && !a.copy, "the first child keeps the page");
    check(b.len == 33 && b.tail == 1 && b.copy, "the second child copies it");
    check(c.len == 32 && c.full == 2 && c.tail == 0 && !c.copy, "a whole last page is shared");
    check(d.len == 0 && d.full == 0 && !d.copy, "a parent outside the group");
    const int32_t four[1] = {4}, big[1] = {100};
    check(fork_of(four, 1, 0, lens, 4, 16).len == 0, "a parent past the group");
    const int32_t zero[1] = {0};
    check(fork_of(zero, 1, 0, big, 4, 16).len == 64, "a length past the table");
}

static void refusals() {
    alignas(64) static char mem[1 << 16];
    auto at = [&](size_t o) { return static_cast<void *>(mem + o); };
    auto ints = [&](size_t o) { return reinterpret_cast<int32_t *>(mem + o); };
    auto floats = [&](size_t o) { return reinterpret_cast<float *>(mem + o); };
    const KvCache kv{at(0), at(4096), floats(8192), floats(8448), 4, 2, 16, 8, T_I8};
    const PageTable table{ints(9000), 3, 5};

    AppendArgs ap{kv, table, ints(9216), ints(9472), at(10240), T_F32, 4, 4, 64, nullptr, nullptr, 1e-6f, 8, 13.f, 0, at(20480), nullptr, T_F16};
    check(check_append(ap), "append");
    Refusals<AppendArgs, bool (*)(const AppendArgs &)> r{ap, check_append};
    r("keys NULL", [](AppendArgs &a) { a.kv.k = nullptr; });
    r("scales NULL", [](AppendArgs &a) { a.kv.v_scale = nullptr; });
    r("cache type", [](AppendArgs &a) { a.kv.type = T_F32; });
    r("no pages", [](AppendArgs &a) { a.kv.pages = 0; });
    r("pages past a table's numbers", [](AppendArgs &a) { a.kv.pages = 0x80000000u; });
    r("long heads", [](AppendArgs &a) { a.kv.dim = 257, a.stride = 8 * 257; });
    r("long pages", [](AppendArgs &a) { a.kv.page = 1025; });
    r("misaligned scales", [&](AppendArgs &a) { a.kv.k_scale = reinterpret_cast<float *>(mem + 8193); });
    r("table NULL", [](AppendArgs &a) { a.table.p = nullptr; });
    r("table of no columns", [](AppendArgs &a) { a.table.width = 0; });
    r("table past 2^31 positions", [](AppendArgs &a) { a.table.width = 0x8000000; });
    r("query heads", [](AppendArgs &a) { a.q_heads = 3; });
    r("no query heads", [](AppendArgs &a) { a.q_heads = 0; });
    r("projection type", [](AppendArgs &a) { a.type = T_I8; });
    r("query type", [](AppendArgs &a) { a.out_type = T_F32; });
    r("stride", [](AppendArgs &a) { a.stride = 63; });
    r("odd rotation", [](AppendArgs &a) { a.rot = 5; });
    r("rotation past the head", [](AppendArgs &a) { a.rot = 10; });
    r("rotation's base", [](AppendArgs &a) { a.log2_theta = std::log2(-1.0); });
    r("epsilon", [](AppendArgs &a) { a.eps = -1.f; });
    r("epsilon NaN", [](AppendArgs &a) { a.eps = NAN; });
    r("positions NULL", [](AppendArgs &a) { a.pos = nullptr; });
    r("queries NULL", [](AppendArgs &a) { a.q = nullptr; });
    r("projections NULL", [](AppendArgs &a) { a.qkv = nullptr; });
    r("misaligned projections", [&](AppendArgs &a) { a.qkv = at(10242); });
    r("queries over the projections", [&](AppendArgs &a) { a.q = at(10240 + 1008); });
    r("keys over the projections", [&](AppendArgs &a) { a.k = at(10240); });
    r("too many tokens", [](AppendArgs &a) { a.n = 0x80000000u; });
    ap.n = 0, ap.q = nullptr, ap.qkv = nullptr;
    check(!check_append(ap), "nothing to append");

    ReadArgs rd{kv, table, ints(9216), 7, T_BF16, at(20480), at(24576)};
    check(check_read(rd), "read");
    Refusals<ReadArgs, bool (*)(const ReadArgs &)> q{rd, check_read};
    q("lengths NULL", [](ReadArgs &a) { a.lens = nullptr; });
    q("outputs NULL", [](ReadArgs &a) { a.v = nullptr; });
    q("output type", [](ReadArgs &a) { a.type = T_E4M3; });
    q("too many positions", [](ReadArgs &a) { a.most = 0x80000000u; });
    rd.most = 0;
    check(!check_read(rd), "nothing to read");

    AttentionArgs at_{at(0), at(4096), at(8192), at(16384), T_F16, 8, 4, 2, 16, 64, 32, 32, 64, ints(30000), 2, ints(30100), 1.f, 0.f, nullptr};
    check(check_attention(at_), "attention");
    Refusals<AttentionArgs, bool (*)(const AttentionArgs &)> t{at_, check_attention};
    t("type", [](AttentionArgs &a) { a.type = T_F32; });
    t("no heads", [](AttentionArgs &a) { a.kv_heads = 0; });
    t("heads that do not divide", [](AttentionArgs &a) { a.q_heads = 5, a.q_stride = a.out_stride = 80; });
    t("no values", [](AttentionArgs &a) { a.dim = 0; });
    t("long heads", [](AttentionArgs &a) { a.dim = 257; });
    t("stride of q", [](AttentionArgs &a) { a.q_stride = 63; });
    t("stride of v", [](AttentionArgs &a) { a.v_stride = -32; });
    t("wild stride", [](AttentionArgs &a) { a.k_stride = int64_t(1) << 41; });
    t("scale", [](AttentionArgs &a) { a.scale = INFINITY; });
    t("cap", [](AttentionArgs &a) { a.cap = -1.f; });
    t("cap NaN", [](AttentionArgs &a) { a.cap = NAN; });
    t("keys NULL", [](AttentionArgs &a) { a.k = nullptr; });
    t("odd address", [&](AttentionArgs &a) { a.v = mem + 8193; });
    t("outputs over the queries", [&](AttentionArgs &a) { a.out = at(1022); });
    t("outputs over the values", [&](AttentionArgs &a) { a.out = at(8192 + 510); });
    t("too many tokens", [](AttentionArgs &a) { a.n = 0x40000000u; });
    at_.n = 0;
    check(!check_attention(at_), "no tokens");

    DecodeArgs de{kv, table, ints(9216), at(20480), at(24576), T_F16, 4, 32, 32, 1.f, 30.f, nullptr};
    check(check_decode(de), "decode");
    Refusals<DecodeArgs, bool (*)(const DecodeArgs &)> d{de, check_decode};
    d("type", [](DecodeArgs &a) { a.type = T_F32; });
    d("a float16 cache with bfloat16 queries", [](DecodeArgs &a) { a.kv.type = T_F16, a.type = T_BF16; });
    d("heads that do not divide", [](DecodeArgs &a) { a.q_heads = 5, a.q_stride = a.out_stride = 40; });
    d("lengths NULL", [](DecodeArgs &a) { a.lens = nullptr; });
    d("outputs over the queries", [&](DecodeArgs &a) { a.out = at(20480 + 62); });
    d("scale NaN", [](DecodeArgs &a) { a.scale = NAN; });
    de.table.rows = 0;
    check(!check_decode(de), "no sequences");

    ForkArgs fo{kv, {ints(9000), 6, 5}, ints(9216), ints(9472), 3, ints(9600), ints(9700), ints(9900), ints(9952)};
    check(check_fork(fo), "fork");
    Refusals<ForkArgs, bool (*)(const ForkArgs &)> f{fo, check_fork};
    f("groups that do not divide", [](ForkArgs &a) { a.beams = 4; });
    f("no beams", [](ForkArgs &a) { a.beams = 0; });
    f("many beams", [](ForkArgs &a) { a.table.rows = a.beams = 33; });
    f("spare NULL", [](ForkArgs &a) { a.spare = nullptr; });
    f("table over the old one", [](ForkArgs &a) { a.table_out = const_cast<int32_t *>(a.table.p) + 29; });
    f("lengths over the old ones", [](ForkArgs &a) { a.lens_out = const_cast<int32_t *>(a.lens); });

    BeamArgs be{at(0), T_F32, 2, 3, 10, 10, floats(1024), ints(2048), 2, floats(1024), ints(4096), ints(5120), ints(2048)};
    check(check_beam(be), "beam search, scores in place");
    Refusals<BeamArgs, bool (*)(const BeamArgs &)> b{be, check_beam};
    b("type", [](BeamArgs &a) { a.type = T_I8; });
    b("no beams", [](BeamArgs &a) { a.beams = 0; });
    b("many beams", [](BeamArgs &a) { a.beams = 33; });
    b("no vocabulary", [](BeamArgs &a) { a.vocab = 0; });
    b("large vocabulary", [](BeamArgs &a) { a.vocab = (1u << 28) + 1, a.stride = a.vocab; });
    b("end token outside", [](BeamArgs &a) { a.eos = 10; });
    b("finished without an end token", [](BeamArgs &a) { a.eos = -1; });
    b("stride", [](BeamArgs &a) { a.stride = 9; });
    b("parents NULL", [](BeamArgs &a) { a.parents = nullptr; });
    b("too many groups", [](BeamArgs &a) { a.groups = 0x7fffffffu; });
    be.groups = 0;
    check(!check_beam(be), "no groups");
}

int main() {
    pages();
    ranges();
    forks();
    refusals();
    if (!failures) std::printf("all checks passed\n");
    return failures != 0;
}
