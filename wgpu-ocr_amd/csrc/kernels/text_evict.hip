// Eviction from the paged cache: of each sequence's cached tokens the most attended stay, the rest makes room.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../runtime.h"
#include "text_device.h"

namespace ocr {

namespace {

// One workgroup a (sequence, head): each place's rank by counting, then the moves one after another.
__global__ __launch_bounds__(256) void evict_row_kernel(EvictArgs a, uint8_t *kept_all, bool scales) {
    const uint32_t heads = a.kv.heads, h = blockIdx.x % heads;
    const int64_t r = blockIdx.x / heads, base = int64_t(blockIdx.x) * a.most;
    const int tid = threadIdx.x;
    const int32_t *const row = a.table.p + r * a.table.width;
    const int n = min(clamp_len(a.lens[r], a.table.width, a.kv.page), int(a.most)), left = min(n, int(a.keep)), newest = a.newest[r];
    uint8_t *const kept = kept_all + base;
    auto position = [&](int p) { return held_position(a.held[base + p], p, n, newest); };
    auto key = [&](int p) { return is_protected(position(p), newest, a.first, a.recent) ? kProtected : weight_key(a.weights[base + p]); };
    for (int p = tid; p < n; p += 256) {
        const uint32_t k = key(p);
        int before = 0;
        for (int o = 0; o < n; o++) {
            const uint32_t x = key(o);
            before += x > k || (x == k && o < p);
        }
        kept[p] = before < left;
    }
    __syncthreads();
    const size_t vec = size_t(a.kv.dim) * (scales ? 1 : 2);
    auto slot = [&](int p) -> int64_t {
        const int32_t page = page_of(row, a.table.width, a.kv.page, a.kv.pages, p);
        return page < 0 ? -1 : slot_of(page, heads, a.kv.page, h, uint32_t(p) % a.kv.page);
    };
    int to = 0, from = left;
    for (;;) {
        while (to < left && kept[to]) to++;
        while (from < n && !kept[from]) from++;
        if (to >= left || from >= n) break;
        const int64_t src = slot(from), dst = slot(to);
        if (src >= 0 && dst >= 0) {
            for (size_t e = tid; e < vec; e += 256) {
                static_cast<uint8_t *>(a.kv.k)[dst * vec + e] = static_cast<const uint8_t *>(a.kv.k)[src * vec + e];
                static_cast<uint8_t *>(a.kv.v)[dst * vec + e] = static_cast<const uint8_t *>(a.kv.v)[src * vec + e];
            }
            if (scales && tid == 0) a.kv.k_scale[dst] = a.kv.k_scale[src], a.kv.v_scale[dst] = a.kv.v_scale[src];
        }
        if (tid == 0) {
            const float w = a.weights[base + from];
            const int32_t pos = int32_t(position(from));
            a.weights_out[base + to] = w, a.held_out[base + to] = pos;
        }
        to++, from++;
    }
    __syncthreads();
    for (int p = tid; p < int(a.most); p += 256) {
        if (p < left && !kept[p]) continue;
        const float w = p < left ? a.weights[base + p] : 0.f;
        const int32_t pos = p < left ? int32_t(position(p)) : -1;
        a.weights_out[base + p] = w, a.held_out[base + p] = pos;
    }
    if (h == 0 && tid == 0) a.lens_out[r] = left;
}

}  // namespace

void launch_evict(Ctx &c, const EvictArgs &a, hipStream_t s) {
    const bool scales = a.kv.type == T_I8 || a.kv.type == T_E4M3;
    const size_t cells = size_t(a.table.rows) * a.kv.heads * a.most;
    ProbeScope probe("text_evict", s, 4.0 * cells, 16.0 * cells);
    DBuf kept(&c, cells, s);
    hipLaunchKernelGGL(evict_row_kernel, dim3(a.table.rows * a.kv.heads), dim3(256), 0, s, a, kept.as<uint8_t>(), scales);
    OCR_HIP(hipGetLastError());
}

}  // namespace ocr
