// The rules and argument checks of the text decoder's further operators on the CPU: axes of positions, whose weights a key
// gets, what an eviction keeps, how latent vectors are shared out, and every refusal.
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

static void axes() {
    const uint32_t p[4] = {3, 1, 0, 2};
    const AxisMap b = axis_map(4, p, false, false), t = axis_map(4, p, true, true);
    const int block[6] = {0, 0, 0, 1, 3, 3}, block_at[6] = {0, 1, 2, 0, 0, 1}, turn[6] = {0, 1, 3, 0, 3, 0}, turn_at[6] = {0, 0, 0, 1, 1, 2};
    for (int i = 0; i < 6; i++) {
        check(b.axis[i] == block[i] && b.place[i] == block_at[i], "axes in blocks");
        check(t.axis[i] == turn[i] && t.place[i] == turn_at[i], "axes in turn, an empty one among them");
    }
    check(b.count == 4 && !b.own && t.own && t.pairs[0] == 3 && t.pairs[2] == 0, "the axes' numbers");
    const uint32_t all[4] = {128, 0, 0, 0}, last[4] = {0, 0, 0, 128};
    for (const bool in_turn : {false, true}) {
        const AxisMap x = axis_map(1, all, in_turn, false), y = axis_map(4, last, in_turn, false);
        check(x.axis[127] == 0 && x.place[127] == 127 && x.pairs[0] == 128, "the most pairs of one axis");
        check(y.axis[0] == 3 && y.place[127] == 127, "the most pairs of the last axis");
    }
}

// Whoever sees a key by key_range is in its query_range, for every key, document, prefix and window.
static void queries() {
    const int32_t docs[5] = {2, 5, 5, 9, 12}, prefix[4] = {0, 7, 2, 99}, wild[4] = {-3, 0x7fffffff, -0x7fffffff, 3};
    const int n = 14;
    for (const int32_t *pre : {static_cast<const int32_t *>(nullptr), prefix, wild})
        for (const int window : {0, 1, 2, 3, 4, 100, 0x7fffffff})
            for (int j = 0; j < n; j++) {
                const QueryRange r = query_range(j, n, docs, 4, pre, window);
                const int d = j < 2 ? -1 : j < 5 ? 0 : j < 9 ? 2 : j < 12 ? 3 : -1;
                check(r.doc == d, "a key's document");
                if (d < 0) {
                    check(r.hi <= r.lo, "a key of no document");
                    continue;
                }
                check(r.place == j - docs[d], "a key's place");
                for (int i = 0; i < n; i++) {
                    const KeyRange k = key_range(i, n, docs, 4, pre);
                    const bool sees = k.lo <= j && j < k.hi, late = window == 0 || i >= docs[d + 1] - window;
                    check((r.lo <= i && i < r.hi) == (sees && late), "the queries that see a key");
                }
            }
    const QueryRange one = query_range(3, 10, nullptr, 1, nullptr, 4);
    check(one.lo == 6 && one.hi == 10 && one.doc == 0 && one.place == 3, "no documents");
    // Offsets that make no sense stay inside the row, documents among those there are.
    const int32_t bad[4] = {-2000000000, 7, 3, 2000000000}, far[3] = {0x7fffffff, -5, 0x7fffffff};
    for (int j = 0; j < 10; j++) {
        const QueryRange r = query_range(j, 10, bad, 3, far, 0x7fffffff);
        check(r.hi <= r.lo || (r.lo >= 0 && r.hi <= 10), "offsets that do not rise");
        check(r.doc >= -1 && r.doc < 3 && r.place >= 0 && r.place < 10, "its place");
    }
    check(query_range(0, 10, bad, 0, nullptr, 0).doc == -1, "no document at all");
}

static void keys() {
    const float up[] = {-INFINITY, -0x1.fffffep127f, -1.f, -0x1p-149f, 0.f, 0x1p-149f, 0x1p-126f, 0.5f, 1.f, 0x1.fffffep127f, INFINITY};
    for (size_t i = 1; i < sizeof up / sizeof *up; i++) check(weight_key(up[i - 1]) < weight_key(up[i]), "weights' order");
    check(weight_key(-0.f) == weight_key(0.f), "the zeros");
    check(weight_key(NAN) == 0 && weight_key(-NAN) == 0 && weight_key(-INFINITY) > 0, "NaN is least");
    check(weight_key(INFINITY) < kProtected, "protected ones are over all");
    check(held_position(7, 3, 10, 99) == 7 && held_position(0, 3, 10, 99) == 0, "a position that is held");
    check(held_position(-1, 9, 10, 99) == 99 && held_position(-5, 0, 10, 99) == 90, "a position by its place");
    check(held_position(-1, 0, 0x7fffffff, -0x7fffffff - 1) == -0x80000000ll - 0x7ffffffe, "positions past 32 bits");
    check(is_protected(3, 99, 4, 0) && !is_protected(4, 99, 4, 0), "the first positions");
    check(is_protected(96, 99, 0, 4) && !is_protected(95, 99, 0, 4), "the last positions");
    check(!is_protected(0, 99, 0, 0) && !is_protected(99, 99, 0, 0), "none protected");
    check(is_protected(100, 99, 0, 0), "a position after the newest is recent");
    check(!is_protected(0x7fffffff, 0x7fffffff, 0, 0) && is_protected(0x7fffffff, 0x7fffffff, 0, 1), "the last number");
    check(is_protected(-5, 0x7fffffff, 0, 0xffffffffu), "recent past the first");
}

// Every tile of every sequence is in one run's part, no two parts of a run share a place, and runs are equal.
static void runs() {
    check(latent_tiles(0) == 0 && latent_tiles(1) == 1 && latent_tiles(32) == 1 && latent_tiles(33) == 2 && latent_tiles(0x7fffffff) == 0x4000000, "tiles");
    const std::vector<std::vector<int>> cases{{0}, {1}, {5}, {1000}, {0, 3, 0, 1, 7, 0}, {1, 1, 1, 1, 1, 1, 1}, {100, 1, 100}, {64, 64, 64, 64}, {257, 3, 3, 3}};
    for (const auto &c : cases)
        for (const int n : {1, 2, 3, 7, 256}) {
            int64_t total = 0;
            for (int t : c) total += t;
            const int64_t each = latent_run(total, n);
            check(each >= kLeastRun && each * n >= total, "runs hold all tiles");
            std::vector<int> used(2 * n, 0);
            int64_t start = 0;
            for (int t : c) {
                if (t == 0) continue;
                const Runs r = runs_of(start, t, each);
                check(r.first >= 0 && r.first <= r.last && r.last < n, "a sequence's runs");
                check(r.first * each <= start && (r.last + 1) * each >= start + t, "they hold it");
                if (r.last > r.first)
                    for (int64_t g = r.first; g <= r.last; g++) {
                        const int64_t at = part_place(g, start, each);
                        check(at >= 2 * g && at < 2 * g + 2 && !used[at], "a part's place is its own");
                        used[at] = 1;
                    }
                start += t;
            }
        }
    check(latent_run(int64_t(1) << 40, 256) == int64_t(1) << 32, "runs past 32 bits");
}

static void refusals() {
    alignas(64) static char mem[1 << 17];
    auto at = [&](size_t o) { return static_cast<void *>(mem + o); };
    auto ints = [&](size_t o) { return reinterpret_cast<int32_t *>(mem + o); };
    auto floats = [&](size_t o) { return reinterpret_cast<float *>(mem + o); };

    Axes ax{ints(0), 3, {4, 2, 2, 0}, 0, 0};
    check_axes(ax, 16, 5);
    auto axis = [&](const char *what, auto &&change, uint32_t rot = 16, uint32_t n = 5) {
        Axes x = ax;
        change(x);
        refused([&] { check_axes(x, rot, n); }, what);
    };
    axis("no axes", [](Axes &x) { x.count = 0; });
    axis("five axes", [](Axes &x) { x.count = 5; });
    axis("too few pairs", [](Axes &x) { x.pairs[0] = 3; });
    axis("pairs of an axis that is not there", [](Axes &x) { x.pairs[2] = 0, x.pairs[3] = 2; });
    axis("pairs that sum past 32 bits", [](Axes &x) { x.pairs[0] = 0xffffffffu, x.pairs[1] = 7, x.pairs[2] = 2; });
    axis("positions NULL", [](Axes &x) { x.at = nullptr; });
    axis("odd positions", [&](Axes &x) { x.at = reinterpret_cast<int32_t *>(mem + 2); });
    ax.at = nullptr;
    check_axes(ax, 16, 0);

    RotateArgs ro{at(0), at(32768), T_F16, 3, 4, 24, 100, 24, 96, 24, 8, 16, 13.f, 0, 0, ints(0), {}};
    check(check_rotate(ro), "rotation");
    Refusals<RotateArgs, bool (*)(const RotateArgs &)> r{ro, check_rotate};
    r("type", [](RotateArgs &a) { a.type = T_I8; });
    r("no heads", [](RotateArgs &a) { a.heads = 0; });
    r("many heads", [](RotateArgs &a) { a.heads = 4097, a.x_stride = a.out_stride = 4097 * 24; });
    r("no values", [](RotateArgs &a) { a.dim = 0; });
    r("long heads", [](RotateArgs &a) { a.dim = a.x_head = a.out_head = 1025, a.x_stride = a.out_stride = 4100; });
    r("odd rotation", [](RotateArgs &a) { a.rot = 15; });
    r("rotation past the head", [](RotateArgs &a) { a.first = 9; });
    r("rotation that wraps", [](RotateArgs &a) { a.first = 0xfffffff8u; });
    r("base", [](RotateArgs &a) { a.log2_theta = -INFINITY; });
    r("heads of the inputs", [](RotateArgs &a) { a.x_head = 23; });
    r("heads of the outputs", [](RotateArgs &a) { a.out_head = 0; });
    r("stride", [](RotateArgs &a) { a.x_stride = 95; });
    r("wild stride", [](RotateArgs &a) { a.out_stride = (int64_t(1) << 40) + 1; });
    r("inputs NULL", [](RotateArgs &a) { a.x = nullptr; });
    r("outputs NULL", [](RotateArgs &a) { a.out = nullptr; });
    r("odd address", [&](RotateArgs &a) { a.x = mem + 1; });
    r("outputs over the inputs", [&](RotateArgs &a) { a.out = at(2); });
    r("in place with other strides", [](RotateArgs &a) { a.out = const_cast<void *>(a.x); });
    r("too many tokens", [](RotateArgs &a) { a.n = 0x80000000u; });
    ro.out = const_cast<void *>(ro.x), ro.out_stride = 100;
    check(check_rotate(ro), "rotation in place");
    ro.n = 0, ro.x = nullptr;
    check(!check_rotate(ro), "no tokens to rotate");

    const AttentionArgs att{at(0), at(4096), at(8192), at(16384), T_F16, 8, 4, 2, 16, 64, 32, 32, 64, ints(30000), 2, ints(30100), 1.f, 0.f, nullptr};
    const KvCache kv{at(0), at(4096), floats(8192), floats(8448), 4, 2, 16, 8, T_I8};
    const PageTable table{ints(9000), 3, 5};
    const DecodeArgs de{kv, table, ints(9216), at(10240), at(12288), T_F16, 4, 32, 32, 1.f, 0.f, nullptr};
    check(check_attention(att) && check_decode(de), "attention");
    check(check_weights({floats(40000), 7, 0}, 3) && !check_weights({nullptr, 0, 0}, 3) && !check_weights({nullptr, 7, 0}, 0), "weights");
    refused([&] { check_weights({nullptr, 7, 0}, 3); }, "weights NULL");
    refused([&] { check_weights({reinterpret_cast<float *>(mem + 2), 7, 0}, 3); }, "odd weights");
    refused([&] { check_weights({floats(40000), 0x80000000u, 0}, 3); }, "too many places");
    refused([&] { check_weights({floats(40000), 7, 0x80000000u}, 3); }, "window");
    check_apart(Weights{floats(40000), 7, 0}, att), check_apart(Weights{floats(40000), 7, 0}, de);
    for (const size_t o : {size_t(0), size_t(4096), size_t(8192), size_t(16384 + 8 * 128 - 4), size_t(16384 - 2 * 2 * 7 * 4 + 4)})
        refused([&] { check_apart(Weights{floats(o), 7, 0}, att); }, "weights over what attention reads or writes");
    check_apart(Weights{floats(16384 - 2 * 2 * 7 * 4), 7, 0}, att);
    for (const size_t o : {size_t(9216), size_t(10240), size_t(12288 + 188)})
        refused([&] { check_apart(Weights{floats(o), 7, 0}, de); }, "weights over what single tokens' attention reads or writes");

    const EvictArgs ev{kv, table, ints(9100), ints(9200), floats(20480), ints(24576), 80, 40, 4, 16, floats(28672), ints(32768), ints(9300)};
    check(check_evict(ev), "eviction");
    Refusals<EvictArgs, bool (*)(const EvictArgs &)> e{ev, check_evict};
    e("cache", [](EvictArgs &a) { a.kv.v = nullptr; });
    e("table", [](EvictArgs &a) { a.table.p = nullptr; });
    e("no places", [](EvictArgs &a) { a.most = 0; });
    e("too many places", [](EvictArgs &a) { a.most = 0x80000000u; });
    e("places that a step past the last would leave 32 bits", [](EvictArgs &a) { a.most = 0x7ffffff0u; });
    e("nothing to keep", [](EvictArgs &a) { a.keep = a.first = a.recent = 0; });
    e("too many to keep", [](EvictArgs &a) { a.keep = 0x80000000u; });
    e("more protected than kept", [](EvictArgs &a) { a.recent = 37; });
    e("protected past 32 bits", [](EvictArgs &a) { a.recent = 0xffffffffu; });
    e("lengths NULL", [](EvictArgs &a) { a.lens = nullptr; });
    e("newest NULL", [](EvictArgs &a) { a.newest = nullptr; });
    e("weights NULL", [](EvictArgs &a) { a.weights = nullptr; });
    e("positions NULL", [](EvictArgs &a) { a.held = nullptr; });
    e("new weights NULL", [](EvictArgs &a) { a.weights_out = nullptr; });
    e("new positions NULL", [](EvictArgs &a) { a.held_out = nullptr; });
    e("new lengths NULL", [](EvictArgs &a) { a.lens_out = nullptr; });
    e("odd weights", [&](EvictArgs &a) { a.weights = reinterpret_cast<float *>(mem + 20481); });
    e("new weights over part of the old", [](EvictArgs &a) { a.weights_out = const_cast<float *>(a.weights) + 1; });
    e("new positions over part of the old", [](EvictArgs &a) { a.held_out = const_cast<int32_t *>(a.held) + 1; });
    e("new weights over the positions", [](EvictArgs &a) { a.weights_out = reinterpret_cast<float *>(const_cast<int32_t *>(a.held)); });
    e("new weights over the new positions", [](EvictArgs &a) { a.weights_out = reinterpret_cast<float *>(a.held_out) + 3; });
    e("new lengths over the old", [](EvictArgs &a) { a.lens_out = const_cast<int32_t *>(a.lens); });
    e("new lengths over the newest", [](EvictArgs &a) { a.lens_out = const_cast<int32_t *>(a.newest) + 2; });
    e("new lengths over the weights", [](EvictArgs &a) { a.lens_out = reinterpret_cast<int32_t *>(a.weights_out) + 5; });
    EvictArgs same = ev;
    same.weights_out = const_cast<float *>(ev.weights), same.held_out = const_cast<int32_t *>(ev.held);
    check(check_evict(same), "eviction in place");
    same.table.rows = 0, same.lens = nullptr;
    check(!check_evict(same), "no sequences to evict from");

    const LatentCache lc{at(0), 4, 16, 24, 8, T_BF16};
    const LatentAppendArgs la{lc, table, ints(9100), ints(9200), at(40960), T_F32, 3, 40, floats(9300), 1e-6f, 13.f, 0, at(61440), nullptr, {}};
    check(check_latent_append(la), "latent append");
    Refusals<LatentAppendArgs, bool (*)(const LatentAppendArgs &)> l{la, check_latent_append};
    l("cache NULL", [](LatentAppendArgs &a) { a.c.p = nullptr; });
    l("cache type", [](LatentAppendArgs &a) { a.c.type = T_I8; });
    l("no pages", [](LatentAppendArgs &a) { a.c.pages = 0; });
    l("pages past a table's numbers", [](LatentAppendArgs &a) { a.c.pages = 0x80000000u; });
    l("empty pages", [](LatentAppendArgs &a) { a.c.page = 0; });
    l("long pages", [](LatentAppendArgs &a) { a.c.page = 1025; });
    l("no rank", [](LatentAppendArgs &a) { a.c.rank = 0; });
    l("large rank", [](LatentAppendArgs &a) { a.c.rank = 513, a.stride = 521; });
    l("odd rotation", [](LatentAppendArgs &a) { a.c.rot = 7; });
    l("large rotation", [](LatentAppendArgs &a) { a.c.rot = 130, a.stride = 154; });
    l("odd cache", [&](LatentAppendArgs &a) { a.c.p = mem + 1; });
    l("table NULL", [](LatentAppendArgs &a) { a.table.p = nullptr; });
    l("projection type", [](LatentAppendArgs &a) { a.type = T_E4M3; });
    l("stride", [](LatentAppendArgs &a) { a.stride = 31; });
    l("base", [](LatentAppendArgs &a) { a.log2_theta = NAN; });
    l("epsilon", [](LatentAppendArgs &a) { a.eps = -1.f; });
    l("epsilon NaN", [](LatentAppendArgs &a) { a.eps = NAN; });
    l("sequences NULL", [](LatentAppendArgs &a) { a.seq = nullptr; });
    l("positions NULL", [](LatentAppendArgs &a) { a.pos = nullptr; });
    l("projections NULL", [](LatentAppendArgs &a) { a.x = nullptr; });
    l("odd projections", [&](LatentAppendArgs &a) { a.x = mem + 40962; });
    l("odd norm", [&](LatentAppendArgs &a) { a.norm = reinterpret_cast<float *>(mem + 9301); });
    l("outputs over the projections", [&](LatentAppendArgs &a) { a.out = at(40960 + 440); });
    l("too many tokens", [](LatentAppendArgs &a) { a.n = 0x80000000u; });
    LatentAppendArgs none = la;
    none.n = 0, none.x = nullptr;
    check(!check_latent_append(none), "no latent tokens");

    const LatentDecodeArgs ld{lc, table, ints(9100), at(40960), at(61440), 4, 128, 96, 1.f};
    check(check_latent_decode(ld), "latent attention of single tokens");
    Refusals<LatentDecodeArgs, bool (*)(const LatentDecodeArgs &)> d{ld, check_latent_decode};
    d("cache", [](LatentDecodeArgs &a) { a.c.p = nullptr; });
    d("positions that a step past the last would leave 32 bits", [](LatentDecodeArgs &a) { a.table.width = 0x7ffffffu; });
    d("no heads", [](LatentDecodeArgs &a) { a.heads = 0; });
    d("many heads", [](LatentDecodeArgs &a) { a.heads = 1025, a.q_stride = 1025 * 32, a.out_stride = 1025 * 24; });
    d("scale", [](LatentDecodeArgs &a) { a.scale = NAN; });
    d("stride of the queries", [](LatentDecodeArgs &a) { a.q_stride = 127; });
    d("stride of the outputs", [](LatentDecodeArgs &a) { a.out_stride = 95; });
    d("lengths NULL", [](LatentDecodeArgs &a) { a.lens = nullptr; });
    d("queries NULL", [](LatentDecodeArgs &a) { a.q = nullptr; });
    d("outputs NULL", [](LatentDecodeArgs &a) { a.out = nullptr; });
    d("odd address", [&](LatentDecodeArgs &a) { a.q = mem + 40961; });
    d("outputs over the queries", [&](LatentDecodeArgs &a) { a.out = at(40960 + 766); });
    LatentDecodeArgs rows = ld;
    rows.table.rows = 0, rows.q = nullptr;
    check(!check_latent_decode(rows), "no sequences");

    const ForkArgs fo{{at(0), nullptr, nullptr, nullptr, 4, 1, 16, 32, T_BF16}, {ints(9000), 6, 5}, ints(9216), ints(9300), 3, ints(9400), ints(9600), ints(9800), ints(9900)};
    auto forked = [&](const LatentCache &c, const ForkArgs &f) { return check_latent_fork(c, f); };
    check(forked(lc, fo), "latent fork");
    LatentCache bad = lc;
    bad.rot = 3;
    refused([&] { forked(bad, fo); }, "a fork's cache");
    ForkArgs fork = fo;
    fork.table_out = const_cast<int32_t *>(fo.table.p) + 29;
    refused([&] { forked(lc, fork); }, "a fork's table over the old one");
    fork = fo, fork.spare = nullptr;
    refused([&] { forked(lc, fork); }, "a fork's spare pages NULL");

    const LatentAttentionArgs lp{at(0), at(8192), at(16384), at(8192 + 32), at(32768), T_F16, 8, 3, 16, 4, 12, 60, 84, 28, 10, 84, 28, 36, ints(60000), 2, ints(60100), 1.f};
    check(check_latent_attention(lp), "latent attention of prompts");
    Refusals<LatentAttentionArgs, bool (*)(const LatentAttentionArgs &)> p{lp, check_latent_attention};
    p("type", [](LatentAttentionArgs &a) { a.type = T_F32; });
    p("no keys", [](LatentAttentionArgs &a) { a.key = 0; });
    p("long keys", [](LatentAttentionArgs &a) { a.key = 257, a.k_head = 257, a.k_stride = a.q_stride = 1000; });
    p("no values", [](LatentAttentionArgs &a) { a.value = 0; });
    p("long values", [](LatentAttentionArgs &a) { a.value = 257, a.v_head = 257, a.v_stride = a.out_stride = 1000; });
    p("long shared keys", [](LatentAttentionArgs &a) { a.rot = 129, a.r_stride = 129, a.q_stride = 1000; });
    p("no heads", [](LatentAttentionArgs &a) { a.heads = 0; });
    p("many heads", [](LatentAttentionArgs &a) { a.heads = 1025, a.q_stride = a.k_stride = a.v_stride = a.out_stride = 100000; });
    p("scale", [](LatentAttentionArgs &a) { a.scale = INFINITY; });
    p("stride of q", [](LatentAttentionArgs &a) { a.q_stride = 59; });
    p("heads of k", [](LatentAttentionArgs &a) { a.k_head = 15; });
    p("stride of k", [](LatentAttentionArgs &a) { a.k_stride = 71; });
    p("heads of v", [](LatentAttentionArgs &a) { a.v_head = 11; });
    p("stride of v", [](LatentAttentionArgs &a) { a.v_stride = 67; });
    p("stride of r", [](LatentAttentionArgs &a) { a.r_stride = 3; });
    p("stride of the outputs", [](LatentAttentionArgs &a) { a.out_stride = 35; });
    p("too many tokens", [](LatentAttentionArgs &a) { a.n = 0x40000000u; });
    p("too many documents", [](LatentAttentionArgs &a) { a.ndocs = 0x40000000u; });
    p("queries NULL", [](LatentAttentionArgs &a) { a.q = nullptr; });
    p("keys NULL", [](LatentAttentionArgs &a) { a.k = nullptr; });
    p("shared keys NULL", [](LatentAttentionArgs &a) { a.r = nullptr; });
    p("values NULL", [](LatentAttentionArgs &a) { a.v = nullptr; });
    p("outputs NULL", [](LatentAttentionArgs &a) { a.out = nullptr; });
    p("odd address", [&](LatentAttentionArgs &a) { a.r = mem + 16385; });
    p("odd offsets", [&](LatentAttentionArgs &a) { a.docs = reinterpret_cast<int32_t *>(mem + 60002); });
    p("outputs over the queries", [&](LatentAttentionArgs &a) { a.out = at(900); });
    p("outputs over the keys", [&](LatentAttentionArgs &a) { a.out = at(8192 + 84 * 2 * 7); });
    p("outputs over the shared keys", [&](LatentAttentionArgs &a) { a.out = at(16384 + 140); });
    LatentAttentionArgs plain = lp;
    plain.rot = 0, plain.r = nullptr, plain.r_stride = 0;
    check(check_latent_attention(plain), "no shared keys");
    plain.n = 0, plain.q = nullptr;
    check(!check_latent_attention(plain), "no tokens");
}

int main() {
    axes();
    queries();
    keys();
    runs();
    refusals();
    if (!failures) std::printf("all checks passed\n");
    return failures != 0;
}
