// Spans of value scales on the CPU: every scale that counts is in one span, and there is an end.
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <random>
#include <vector>

#include "text_rules.h"

using namespace ocr;

static int failures = 0;
static void check(bool ok, const char *what, double a, double b) {
    if (ok) return;
    std::printf("FAILED: %s (%g, %g)\n", what, a, b);
    failures++;
}

// The kernel's loop over a tile's scales (as multiples of the largest so far).
static void spans(const std::vector<float> &scale) {
    std::vector<int> taken(scale.size(), 0);
    float left = NAN;
    int rounds = 0;
    for (; rounds < 100; rounds++) {
        float largest = 0.f;
        for (float x : scale) largest = std::fmax(largest, x >= left ? 0.f : x);
        if (!more_spans(largest)) break;
        const ScaleSpan s = span_of(largest);
        check(std::isfinite(s.over) && std::isfinite(1.f / s.over) && s.low > 0 && s.low < largest, "a span", s.over, s.low);
        for (size_t i = 0; i < scale.size(); i++) {
            const float x = scale[i];
            if (x >= left || x < s.low) continue;
            taken[i]++;
            check(!(x / s.over > 1.f) || std::isinf(x), "under its power of two", x, s.over);
            check(!(x / s.over < kScaleSpan), "within a span of it", x, s.over);
        }
        left = s.low;
    }
    check(rounds <= 50, "an end", rounds, 0);
    for (size_t i = 0; i < scale.size(); i++)
        check(std::isnan(scale[i]) ? taken[i] == rounds : scale[i] >= 2 * kLastSpan ? taken[i] == 1 : taken[i] <= 1, "taken once", scale[i], taken[i]);
}

int main() {
    std::mt19937 rng(5);
    std::uniform_real_distribution<float> u(0.f, 1.f);
    for (float least : {0.f, 0x1p-149f, 0x1p-140f, 0x1p-132f, 0x1p-127f, 0x1p-126f, 0x1p-121f, 0x1p-120f, 0x1p-119f, 0x1p-60f, 0x1p-7f, 0x1p-6f, 0.9f})
        for (int round = 0; round < 50; round++) {
            std::vector<float> s(32, least);
            for (int i = 0; i < 8; i++) s[rng() % 32] = std::ldexp(u(rng), -int(rng() % 150));
            s[rng() % 32] = 1.f;
            spans(s);
            s[rng() % 32] = NAN;
            spans(s);
            s[rng() % 32] = INFINITY;
            spans(s);
        }
    spans(std::vector<float>(32, 0.f));
    spans(std::vector<float>(32, 0x1p-149f));
    spans(std::vector<float>(32, NAN));
    if (!failures) std::printf("all checks passed\n");
    return failures != 0;
}
