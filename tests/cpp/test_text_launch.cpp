// How the text decoder's launches are cut, on the CPU: every piece of work is somebody's, once.
#include <cstdio>
#include <set>
#include <utility>

#include "text_rules.h"

using namespace ocr;

static int failures = 0;
static void check(bool ok, const char *what, long a, long b, long c) {
    if (ok) return;
    std::printf("FAILED: %s (%ld, %ld, %ld)\n", what, a, b, c);
    failures++;
}

static void parts() {
    for (uint32_t most : {1u, 2u, 3u, 16u, 127u, 128u})
        for (int len : {-5, 0, 1, 31, 32, 33, 255, 256, 257, 511, 512, 513, 8191, 8193, 131072, 1000003, 0x7fffffc0}) {
            const Parts p = parts_of(len, most);
            check(p.count >= 0 && p.count <= int(most), "count", len, most, p.count);
            check((p.count == 0) == (len <= 0), "a part where there is something", len, most, p.count);
            if (len <= 0) continue;
            check(int64_t(p.count) * p.each >= len && int64_t(p.count - 1) * p.each < len, "the parts hold the sequence", len, most, p.each);
            check(most == 1 || (p.each >= kLeastPart && p.each % 32 == 0), "whole tiles", len, most, p.each);
        }
}

static void heads() {
    for (int tiles : {1, 2, 7, 23, 64})
        for (uint32_t kv : {1u, 2u, 3u, 4u, 5u, 6u, 7u, 8u, 12u, 16u, 24u})
            for (uint32_t group : {1u, 2u, 3u, 8u, 17u})
            for (uint32_t units : {0u, 4u, 32u}) {
                const uint32_t q = kv * group;
                std::set<std::pair<int, int>> seen;
                const int64_t n = head_blocks(tiles, q, kv);
                check(n >= int64_t(tiles) * q && n < int64_t(tiles) * q + 64, "workgroups", tiles, kv, group);
                for (int64_t x = 0; x < n; x++) {
                    const HeadTile t = head_tile(uint32_t(x), tiles, q, kv, units);
                    if (t.head < 0) continue;
                    check(t.head < int(q) && t.tile >= 0 && t.tile < tiles && seen.insert({t.head, t.tile}).second, "a tile twice or none", tiles, kv, group);
                    // With eight key heads or a divisor of eight, a die has as few as there are.
                    if (kv == 8) check(t.head / int(group) == int(x % 8), "the die's key head", tiles, kv, group);
                }
                check(seen.size() == size_t(tiles) * q, "every tile", tiles, kv, group);
            }
}

// Between one and two pieces for each unit: the pairs (y and y + units) are of the lighter ones, the
// lightest with the heaviest of them.
static void pairs() {
    for (uint32_t units : {1u, 4u, 32u})
        for (uint32_t n = 1; n <= 3 * units; n++) {
            std::set<uint32_t> seen;
            for (uint32_t y = 0; y < n; y++) check(paired(y, n, units) < n && seen.insert(paired(y, n, units)).second, "a piece twice", y, n, units);
            if (n <= units || n > 2 * units) {
                for (uint32_t y = 0; y < n; y++) check(paired(y, n, units) == y, "the heaviest first", y, n, units);
                continue;
            }
            for (uint32_t y = 0; y < units; y++) {
                const bool two = y + units < n;
                check(two == (paired(y, n, units) >= units) || n == 2 * units, "the light ones in pairs", y, n, units);
                if (two) check(paired(y, n, units) + paired(y + units, n, units) == n - 1 + 2 * units - n, "of like sums", y, n, units);
            }
        }
}

int main() {
    parts();
    pairs();
    heads();
    if (!failures) std::printf("all checks passed\n");
    return failures != 0;
}
