// The order of a beam search's continuations on the CPU: scores that absorb logits, places that are
// all different.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
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

static uint32_t key_of(float x) {
    uint32_t u;
    x += 0.f;
    std::memcpy(&u, &x, 4);
    return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}

static void keys() {
    const float row[] = {-INFINITY, -3.4e38f, -1.f, -1e-45f, 0.f, 1e-45f, 1e-17f, 2.f, 3.4e38f};
    for (int i = 0; i < 9; i++) {
        check(value_of(key_of(row[i])) == row[i], "a key's value", row[i], value_of(key_of(row[i])));
        check(i == 0 || key_of(row[i - 1]) < key_of(row[i]), "keys order as the values", row[i], 0);
    }
    check(key_of(-INFINITY) == kNothing && key_of(-0.f) == key_of(0.f), "minus infinity and the zeros", 0, 0);
}

// The least logit of a score, by walking down from it or, where that is far, by its neighbours.
static void alike() {
    for (double cum : {0.0, -20.0, -1e9, -1e20, -1e30, -3.4028234663852886e38, 3.4028234663852886e38})
        for (float x : {0.f, 1e-17f, -1e-17f, 9.f, -9.f, 1e6f, -3e38f, 3e38f}) {
            const LogSum lse = log_sum(std::max(0.f, x), std::log(97.0));
            const uint32_t k = key_of(x), low = lowest_alike(k, cum, lse);
            const double s = score_of_key(k, cum, lse);
            check(low > kNothing && low <= k && score_of_key(low, cum, lse) == s, "the least scores alike", cum, x);
            check(score_of_key(low - 1, cum, lse) < s, "the next one less", cum, x);
        }
    check(lowest_alike(key_of(9.f), -20.0, log_sum(9.0, 1.0)) == key_of(9.f), "ordinary logits differ", 0, 0);
    for (float x : {-3.4028235e38f, 3.4028235e38f, 1e20f})
        check(score_of_key(key_of(x), -2.0, log_sum(x, std::log(97.0))) == -2.0 - std::log(97.0), "a row of equal logits", x, 0);
    // What an ordinary sum loses is under its last bit, and logits that it absorbs stay alike.
    for (double top : {-3.0, 0.0, 1.25, 40.0}) {
        const LogSum l = log_sum(top, std::log(20001.0));
        check(std::fabs(l.lost) <= 0x1p-53 * std::fabs(l.whole), "what the sum lost", top, l.lost);
        check(score_of_key(key_of(1e-17f), -1.0, l) == score_of_key(key_of(1.2e-16f), -1.0, l), "absorbed logits", top, 0);
    }
    check(lowest_alike(key_of(9.f), -1e30, log_sum(9.0, 1.0)) < key_of(-1e12f), "a large score absorbs them", 0, 0);
}

// Every continuation's place among all is another one, and the one that sorting gives.
static void places() {
    std::mt19937 rng(3);
    for (int round = 0; round < 400; round++) {
        const int w = 1 + int(rng() % 32), kinds = 1 + int(rng() % 6);
        std::vector<double> score(w * w);
        for (int b = 0; b < w; b++) {
            for (int i = 0; i < w; i++) score[b * w + i] = rng() % 8 == 0 ? -INFINITY : round % 2 ? -1e30 : -double(rng() % kinds);
            std::sort(score.begin() + b * w, score.begin() + b * w + w, [](double x, double y) { return x > y; });
        }
        std::vector<int> want(w * w);
        for (int c = 0; c < w * w; c++) want[c] = c;
        std::stable_sort(want.begin(), want.end(), [&](int x, int y) { return score[x] > score[y]; });
        std::vector<char> taken(w * w, 0);
        for (int c = 0; c < w * w; c++) {
            int place = 0;
            for (int o = 0; o < w; o++) place += o == c / w ? c % w : before_other(&score[o * w], w, score[c], o < c / w);
            check(!taken[place], "a place for two", w, place);
            taken[place] = 1;
            check(want[place] == c, "the place of a sorted row", w, place);
        }
    }
}

int main() {
    keys();
    alike();
    places();
    if (!failures) std::printf("all checks passed\n");
    return failures != 0;
}
