// The rules of the text decoder's operators that kernels and host share, free of HIP calls so that
// they run on the CPU too: where a cached vector lies, which keys a prompt's token sees, what a
// fork of a beam's pages does, how a launch is cut.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define OCR_HD __host__ __device__ inline
#else
#define OCR_HD inline
#endif

namespace ocr {

// The page that holds position pos of a sequence (its row of the table, width entries), or -1 where
// there is none: a position outside the table, an entry that names no page of the pool.
OCR_HD int32_t page_at(const int32_t *row, uint32_t width, uint32_t pages, uint32_t entry) {
    if (entry >= width) return -1;
    const int32_t p = row[entry];
    return p >= 0 && uint32_t(p) < pages ? p : -1;
}
OCR_HD int32_t page_of(const int32_t *row, uint32_t width, uint32_t page, uint32_t pages, int64_t pos) {
    if (pos < 0 || pos >= int64_t(width) * page) return -1;
    return page_at(row, width, pages, uint32_t(pos) / page);  // within 31 bits: width * page is (check_table)
}

// Vector index of (page p, head, slot) in a pool laid out [pages][heads][page].
OCR_HD int64_t slot_of(int32_t p, uint32_t heads, uint32_t page, uint32_t head, uint32_t slot) {
    return (int64_t(p) * heads + head) * page + slot;
}

// Positions of a sequence that there are: its length within its table.
OCR_HD int32_t clamp_len(int32_t len, uint32_t width, uint32_t page) {
    const int64_t most = int64_t(width) * page;
    return len < 0 ? 0 : int64_t(len) > most ? int32_t(most) : len;
}

// Keys [lo, hi) that token i of a packed row sees. docs: ndocs + 1 rising offsets, prefix: each document's tokens that
// all of it sees (null: none). Every token of a document sees those before it, itself and the
// document's prefix; tokens outside every document see nothing. Offsets that do not rise give some
// range inside [0, n).
struct KeyRange {
    int lo, hi;
};
OCR_HD KeyRange key_range(int i, int n, const int32_t *docs, int ndocs, const int32_t *prefix) {
    if (i < 0 || i >= n) return {0, 0};
    int a = 0, b = n, pre = 0;
    if (docs) {
        // The last document that starts at or before i.
        int lo = 0, hi = ndocs;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (docs[mid] <= i) lo = mid + 1;
            else hi = mid;
        }
        if (lo == 0 || docs[lo] <= i) return {0, 0};
        a = docs[lo - 1] < 0 ? 0 : docs[lo - 1];
        b = docs[lo] > n ? n : docs[lo];
        if (prefix) pre = prefix[lo - 1];
    } else if (prefix) {
        pre = prefix[0];
    }
    int top = i + 1;
    if (pre > 0 && pre > top - a) top = pre < b - a ? a + pre : b;
    return {a, top < b ? top : b};
}

// The queries [lo, hi) of a packed row that see key j: those of its document from itself on, all of them where the
// document's prefix holds it; with `window` > 0 only the document's last `window` of them. doc, place: the
// key's document and its place in it (doc -1: in none, which nothing sees).
struct QueryRange {
    int lo, hi, doc, place;
};
OCR_HD QueryRange query_range(int j, int n, const int32_t *docs, int ndocs, const int32_t *prefix, int window) {
    int a = 0, b = n, d = 0;
    if (docs) {
        int lo = 0, hi = ndocs;  // the last document that starts at or before j
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (docs[mid] <= j) lo = mid + 1;
            else hi = mid;
        }
        if (lo == 0 || docs[lo] <= j) return {0, 0, -1, 0};
        d = lo - 1;
        a = docs[d] < 0 ? 0 : docs[d];
        b = docs[lo] > n ? n : docs[lo];
    }
    int first = prefix && j - a < prefix[d] ? a : j;
    if (window > 0 && b - window > first) first = b - window;
    return {first, b, d, j - a};
}

// A row of a reordered table: what beam w of a group takes from its parent. len: the parent's
// length; full pages are shared, a part-filled last page goes to the first child and is copied for
// the others.
struct Fork {
    int32_t len;
    uint32_t full, tail;  // whole pages, slots of the last one
    bool copy;
};
OCR_HD Fork fork_of(const int32_t *parents, uint32_t beams, uint32_t w, const int32_t *lens, uint32_t width, uint32_t page) {
    Fork f{0, 0, 0, false};
    const int32_t p = parents[w];
    if (p < 0 || uint32_t(p) >= beams) return f;
    f.len = clamp_len(lens[p], width, page);
    f.full = uint32_t(f.len) / page;
    f.tail = uint32_t(f.len) % page;
    bool first = true;
    for (uint32_t e = 0; e < w; e++) first = first && parents[e] != p;
    f.copy = f.tail > 0 && !first;
    return f;
}

// The axis of each of a rotation's pairs, its place among that axis' pairs, and how many those are: `pairs`
// of each of `count` axes in blocks, or of one axis after another in turn as long as each has some.
struct AxisMap {
    uint8_t axis[128], place[128];
    uint8_t pairs[4];
    uint8_t count, own;  // no axes: 0; own: each axis has the whole range of frequencies
};
OCR_HD AxisMap axis_map(uint32_t count, const uint32_t *pairs, bool in_turn, bool own) {
    AxisMap m{};
    m.count = uint8_t(count), m.own = own;
    int at = 0;
    for (uint32_t k = 0; k < count; k++) m.pairs[k] = uint8_t(pairs[k]);
    for (uint32_t round = 0; round < (in_turn ? 128u : count); round++)
        for (uint32_t x = 0; x < (in_turn ? count : pairs[round]); x++) {
            const uint32_t a = in_turn ? x : round, place = in_turn ? round : x;
            if (place >= pairs[a] || at >= 128) continue;
            m.axis[at] = uint8_t(a), m.place[at] = uint8_t(place);
            at++;
        }
    return m;
}

// What an eviction orders a cached token by, the largest first: protected ones, then the others by their
// weight (as floats order, the zeros alike), NaN last. Equal ones go by their place, the lowest first.
constexpr uint32_t kProtected = 0xffffffffu;
OCR_HD uint32_t weight_key(float w) {
    if (w != w) return 0;
    const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w);
    return u >> 31 ? ~u : u | 0x80000000u;  // minus infinity's is 0x007fffff, infinity's 0xff800000
}
// The position of the token at place p of n: what is held, or, where that is negative, as far before the
// newest as its place is before the last.
OCR_HD int64_t held_position(int32_t held, int p, int n, int32_t newest) { return held >= 0 ? held : int64_t(newest) - (n - 1 - p); }
OCR_HD bool is_protected(int64_t pos, int32_t newest, uint32_t first, uint32_t recent) {
    return pos < int64_t(first) || pos > int64_t(newest) - int64_t(recent);
}

// tanh(y) / y by powers of u = y^2, interpolated at the Chebyshev points of [0, 0.35^2]: up to there off by
// 7.0e-8 (2^-23.8), evaluated in float32 by 1.6e-7 (2^-22.6).
constexpr float kSmallTanh = 0.35f;
constexpr float kTanhPart[4] = {1.f, -0.3333241939544678f, 0.13295751810073853f, -0.04895563796162605f};
OCR_HD float tanh_ratio(float u) {
    return __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(kTanhPart[3], u, kTanhPart[2]), u, kTanhPart[1]), u, kTanhPart[0]);
}
// A cap on scores, in their unit: most tanh(s / most). Scores up to `small` go by the ratio above, whose error is
// theirs; what is left of the difference 1 - 2 / (e^2y + 1) there would have the cap's. Caps that are no float in
// the scores' unit, and reciprocals that are none, are the largest that are: nothing that is not beyond 10^30 can tell.
struct Cap {
    float most, inv, small;
};
// Up to here (in units of log2: a cap of 88) that error, 2^-16, is a thirtieth of a float16 weight's own rounding: one
// form may do for all scores of a prompt's tile.
constexpr float kFineCap = 128.f;
OCR_HD Cap cap_of(float cap, float unit) {
    const float most = __builtin_fminf(cap * unit, 0x1.fffffep127f);
    return {most, most > 0.f ? __builtin_fminf(1.f / most, 1e30f) : 0.f, kSmallTanh * most};
}
OCR_HD float small_capped(const Cap &c, float s) {
    const float y = s * c.inv;
    return s * tanh_ratio(y * y);
}

// Logits as 32-bit keys that order as they do (the zeros next to each other); minus infinity's key.
constexpr uint32_t kNothing = 0x007fffffu;
OCR_HD float value_of(uint32_t key) { return __builtin_bit_cast(float, key ^ (key >> 31 ? 0x80000000u : 0xffffffffu)); }

// A row's log-sum: its largest logit and the log of the sum of e^(x - top), and what their sum lost, which is all of
// the second beside a large first (a row whose mask's lowest value leaves nothing).
struct LogSum {
    double whole, lost;
};
OCR_HD LogSum log_sum(double top, double rest) {
    const double whole = top + rest, b = whole - top;
    return {whole, (top - (whole - b)) + (rest - b)};
}
// A continuation's score: the beam's, and the logit of this key less the row's log-sum.
OCR_HD double score_of_key(uint32_t key, double cum, LogSum lse) {
    return key > kNothing ? cum + (double(value_of(key)) - lse.whole - lse.lost) : -__builtin_inf();
}
// The least key whose score is that of `key` (over minus infinity's): scores rise with the keys, but
// not every step, since a large score absorbs logits, and a log-sum small ones.
OCR_HD uint32_t lowest_alike(uint32_t key, double cum, LogSum lse) {
    const double s = score_of_key(key, cum, lse);
    uint32_t under = kNothing;
    while (key - under > 1) {
        const uint32_t mid = under + (key - under) / 2;
        if (score_of_key(mid, cum, lse) == s) key = mid;
        else under = mid;
    }
    return key;
}
// How many of a beam's n continuations, whose scores fall, come before one of another beam that
// scores s. lower: the list's beam comes before that other one, so its equal scores do. Within its own list a
// continuation's place is where it stands, whatever its score: the places of all are different.
OCR_HD int before_other(const double *list, int n, double s, bool lower) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] > s || (lower && list[mid] == s)) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// How a sequence of len positions is cut for single-token attention: at most `parts` parts of at
// least kLeastPart positions, whole tiles of 32.
constexpr int kLeastPart = 256;
constexpr uint32_t kMostParts = 128;
struct Parts {
    int count, each;
};
OCR_HD Parts parts_of(int len, uint32_t parts) {
    if (len <= 0) return {0, kLeastPart};
    const int want = int((uint32_t(len) + parts - 1) / parts);
    const int each = want <= kLeastPart ? kLeastPart : (want + 31) & ~31;
    return parts == 1 ? Parts{1, len} : Parts{int((uint32_t(len) + uint32_t(each) - 1) / uint32_t(each)), each};
}

// How single-token attention over latent vectors is cut: all sequences' tiles of kLatentTile positions one after
// another, in equal runs, so that sequences of unlike lengths leave no workgroup idle. A run ends in the middle of at most two
// sequences, so it has two places for parts: 0 for a sequence that an earlier run began, 1 for one that goes on after it.
constexpr int kLatentTile = 32, kLeastRun = 2;
OCR_HD int latent_tiles(int len) { return int((uint32_t(len) + kLatentTile - 1) / kLatentTile); }
OCR_HD int64_t latent_run(int64_t total, int runs) {
    const int64_t each = (total + runs - 1) / runs;
    return each < kLeastRun ? kLeastRun : each;
}
// Runs [first, last] that have tiles of a sequence whose first tile is `start`.
struct Runs {
    int64_t first, last;
};
OCR_HD Runs runs_of(int64_t start, int tiles, int64_t each) { return {start / each, (start + tiles - 1) / each}; }
// The place of run g's part of it.
OCR_HD int64_t part_place(int64_t g, int64_t start, int64_t each) { return 2 * g + (start >= g * each ? 1 : 0); }

// The power of two over a positive number, at most 2^126.
OCR_HD float over_pow2(float x) {
    const uint32_t u = (__builtin_bit_cast(uint32_t, x) & 0x7f800000u) + 0x00800000u;
    return __builtin_bit_cast(float, u < 0x7e800000u ? u : 0x7e800000u);
}
// Value scales (over the largest so far) that single-token attention's float16 weights hold at once: a
// weight 2^-16 of the largest keeps eight bits under the least of them. Tiles of more take them a span at
// a time, the largest first, each over a power of two of its own; those under the last span are nothing.
// A span begins at its largest scale, so that each holds one and the next lies lower.
constexpr float kScaleSpan = 0x1p-6f, kLastSpan = 0x1p-120f;
struct ScaleSpan {
    float over, low;  // the power of two, the least scale
};
OCR_HD bool more_spans(float largest) { return largest >= kLastSpan; }
OCR_HD ScaleSpan span_of(float largest) { return {over_pow2(largest), over_pow2(largest) * kScaleSpan}; }

// Which tile of queries and which head workgroup x of a prompt's attention takes. Workgroups go to
// the eight compute dies in turn, each with a level-two cache of its own, so a die gets the query
// heads of as few key heads as there are; later tiles, which see more of their document, come first.
// Workgroups past the last have head -1.
struct HeadTile {
    int tile, head;
};
// Piece y of a die's n, the heaviest first, where each of its compute units holds two workgroups: if n
// lies between one and two for each of `units` (0: no matter), some units get two and the others
// one. The y-th workgroup goes to unit y % units, so the light pieces are put where the pairs are, the
// lightest with the heaviest of them, and the heavy ones have a unit each. 46 pieces of 32 to 46 tiles
// for 32 units: 84 us, in order 88.
OCR_HD uint32_t paired(uint32_t y, uint32_t n, uint32_t units) {
    if (n <= units || n > 2 * units) return y;
    const uint32_t pairs = n - units;
    return y < pairs ? n - 1 - y : y - pairs;
}
OCR_HD int64_t head_blocks(int64_t tiles, uint32_t q_heads, uint32_t kv_heads) {
    const int64_t group = q_heads / kv_heads;
    if (8 % kv_heads == 0) {
        const int64_t sharing = 8 / kv_heads;
        return 8 * ((group * tiles + sharing - 1) / sharing);
    }
    return tiles * q_heads;
}
OCR_HD HeadTile head_tile(uint32_t x, int tiles, uint32_t q_heads, uint32_t kv_heads, uint32_t units = 0) {
    const uint32_t group = q_heads / kv_heads, die = x % 8;
    uint32_t hk, at;  // the key head, the place among its group * tiles pieces
    if (8 % kv_heads == 0) {
        const uint32_t sharing = 8 / kv_heads;
        hk = die % kv_heads, at = paired(x / 8, (group * uint32_t(tiles) + sharing - 1) / sharing, units) * sharing + die / kv_heads;
        if (at >= group * uint32_t(tiles)) return {0, -1};
    } else if (kv_heads % 8 == 0) {
        at = x / 8 % (group * uint32_t(tiles));
        hk = x / 8 / (group * uint32_t(tiles)) * 8 + die;
    } else {
        hk = x % kv_heads, at = x / kv_heads;
    }
    return {tiles - 1 - int(at / group), int(hk * group + at % group)};
}

}  // namespace ocr
