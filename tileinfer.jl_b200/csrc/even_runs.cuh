// A numbered list of U equal units of work shared out as one run to each of G resident blocks (G at most U, so no run is empty): with q = U / G and
// r = U mod G, the first r blocks take q + 1 units, the others q. An item is a stretch of units that add up to one result; the blocks that share one
// leave parts. A block has at most two parts, of the item that its run begins inside of (or at) and of the one that it ends inside of: slots 2 c and
// 2 c + 1. U is below 2^31.
#pragma once
#include "common.cuh"

struct Runs {
    unsigned q, r;
    __device__ __forceinline__ Runs(unsigned U, unsigned G) : q(U / G), r(U % G) {}
    __device__ __forceinline__ unsigned low(unsigned c) const { return c * q + min(c, r); }
    __device__ __forceinline__ unsigned owner(unsigned u) const {
        const unsigned longer = r * (q + 1);
        return u < longer ? u / (q + 1) : r + (u - longer) / q;
    }
    // The slot of block c's part of the item that begins at unit u0.
    __device__ __forceinline__ unsigned slot(unsigned c, unsigned u0) const { return 2 * c + (low(c) >= u0 ? 0 : 1); }
};
