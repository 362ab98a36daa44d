// The scores' cap on the CPU: how far the small scores' ratio is off, and caps at the ends of float32.
#include <cfloat>
#include <cmath>
#include <cstdio>
#include <initializer_list>

#include "text_rules.h"

using namespace ocr;

static int failures = 0;
static void check(bool ok, const char *what, double a, double b) {
    if (ok) return;
    std::printf("FAILED: %s (%g, %g)\n", what, a, b);
    failures++;
}

int main() {
    double formula = 0, float32 = 0;
    for (int i = 1; i <= 200000; i++) {
        const double y = 0.35 * i / 200000, u = y * y, want = std::tanh(y) / y;
        const double p = double(kTanhPart[0]) + u * (double(kTanhPart[1]) + u * (double(kTanhPart[2]) + u * double(kTanhPart[3])));
        const float yf = float(y);
        formula = std::fmax(formula, std::fabs(p - want));
        float32 = std::fmax(float32, std::fabs(double(yf * tanh_ratio(yf * yf)) / std::tanh(double(yf)) - 1));
    }
    std::printf("off by %.2e, in float32 by %.2e\n", formula, float32);
    check(formula <= 7.0e-8, "the ratio", formula, 0);
    check(float32 <= 1.6e-7, "the ratio in float32", float32, 0);

    const float log2e = 1.4426950408889634f;
    for (float cap : {1e-40f, 1e-30f, 1e-3f, 1.f, 30.f, 1e6f, 1e20f, 1e37f, 2.4e38f, FLT_MAX}) {
        const Cap c = cap_of(cap, log2e);
        check(c.most > 0 && c.most <= FLT_MAX && c.inv > 0 && c.inv <= 1e30f && c.small > 0 && c.small < c.most, "finite constants", cap, c.most);
        for (float s : {0.f, 1e-3f, -1.f, 7.f, -300.f, 1e10f})
            if (std::fabs(s) <= c.small) {
                const double want = double(c.most) * std::tanh(double(s) / double(c.most));
                // The ratio's error, the product's rounding and the square's, which is a third of its size at most.
                check(std::fabs(small_capped(c, s) - want) <= 2.5e-7 * std::fabs(want), "a small score", cap, s);
            }
    }
    check(cap_of(0.f, log2e).inv == 0.f, "no cap", 0, 0);
    if (!failures) std::printf("all checks passed\n");
    return failures != 0;
}
