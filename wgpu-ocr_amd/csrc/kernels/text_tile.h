// Tiles of rows in LDS that come by DMA, for the matrix-core kernels of prompts.
#pragma once

#include "lds_dma.h"

namespace ocr {

// A tile of KT rows of PW values in LDS: every lane's copies of it, and where its pieces lie. Each row's pieces are
// exchanged so that the reads of 16 rows touch every bank.
template <int PW, int KT> struct Tile {
    static constexpr int PP = PW / 8, BYTES = KT * PW * 2, ND = KT * PP / 256;
    static __device__ int swap_of(int row) { return PP == 8 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3); }
    unsigned at[ND], step;
    int pieces;
    __device__ int row_of(int d) const { return ((4 * d + int(threadIdx.x >> 6)) * 64 + int(threadIdx.x & 63)) / PP; }
    __device__ int piece_of(int d) const { return ((4 * d + int(threadIdx.x >> 6)) * 64 + int(threadIdx.x & 63)) % PP ^ swap_of(row_of(d)); }
    __device__ Tile(int64_t stride, int pieces_) : step(unsigned(stride * 2)), pieces(pieces_) {
#pragma unroll
        for (int d = 0; d < ND; d++) at[d] = row_of(d) * step + 16 * piece_of(d);
    }
    // Rows from `base` on to LDS byte `to` (the wavefront's first piece); `rows` of them there are, past the last: that again.
    __device__ __attribute__((always_inline)) void copy(const char *base, unsigned to, int rows) const {
        if (rows >= KT && pieces == PP) {
#pragma unroll
            for (int d = 0; d < ND; d++) dma16s_to(base, at[d], to + d * 4096);
            return;
        }
#pragma unroll
        for (int d = 0; d < ND; d++)
            if (piece_of(d) < pieces) dma16s_to(base, at[d] - unsigned(max(0, row_of(d) - (rows - 1))) * step, to + d * 4096);
    }
};

}  // namespace ocr
