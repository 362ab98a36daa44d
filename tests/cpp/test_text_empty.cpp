// Calls over no sequences and no tokens on the CPU: empty arrays have no address, and there is nothing to do.
#include <cstdio>
#include <string>

#include "common.h"
#include "text.h"

static int failures = 0;
void ocr::fail(const std::string &msg) { throw Error(msg); }

using namespace ocr;

template <class A> static void nothing(bool (*fn)(const A &), const A &a, bool want, const char *what) {
    try {
        if (fn(a) == want) return;
        std::printf("FAILED: %s\n", what);
    } catch (const Error &e) {
        std::printf("FAILED: %s: %s\n", what, e.what());
    }
    failures++;
}

int main() {
    alignas(64) static char mem[1 << 16];
    auto at = [&](size_t o) { return static_cast<void *>(mem + o); };
    auto ints = [&](size_t o) { return reinterpret_cast<int32_t *>(mem + o); };
    const KvCache kv{at(0), at(4096), nullptr, nullptr, 4, 2, 16, 8, T_F16};
    for (uint32_t width : {5u, 0u}) {
        const PageTable none{nullptr, 0, width};
        nothing(check_read, ReadArgs{kv, none, nullptr, 7, T_F16, nullptr, nullptr}, false, "read");
        nothing(check_decode, DecodeArgs{kv, none, nullptr, nullptr, nullptr, T_F16, 4, 32, 32, 1.f, 0.f, nullptr}, false, "decode");
        nothing(check_fork, ForkArgs{kv, none, nullptr, nullptr, 3, nullptr, nullptr, nullptr, nullptr}, false, "fork");
        AppendArgs a{kv, none, nullptr, nullptr, nullptr, T_F32, 0, 4, 64, nullptr, nullptr, 1e-6f, 8, 13.f, 0, nullptr, nullptr, T_F16};
        nothing(check_append, a, false, "append of no tokens");
        // Tokens of no sequence: their queries are wanted all the same.
        a.n = 2, a.seq = ints(9216), a.pos = ints(9472), a.qkv = at(10240), a.q = at(20480);
        nothing(check_append, a, true, "append to no sequence");
    }
    if (!failures) std::printf("all checks passed\n");
    return failures != 0;
}
