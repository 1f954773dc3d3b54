// A numbered list of U equal units of work shared out as one run to each of G resident blocks (G at most U, so no run is empty): block c takes
// [U c / G, U (c + 1) / G). An item is a stretch of units that add up to one result; the blocks that share one leave parts. A block has at most two
// parts, of the item that its run begins inside of (or at) and of the one that it ends inside of: slots 2 c and 2 c + 1.
#pragma once
#include "common.cuh"

__device__ __forceinline__ long long run_low(long long U, int c, int G) { return U * c / G; }
__device__ __forceinline__ int run_owner(long long U, long long u, int G) { return (int)(((u + 1) * G - 1) / U); }
// The slot of block c's part of the item that begins at unit u0.
__device__ __forceinline__ int run_slot(long long U, int c, int G, long long u0) { return 2 * c + (run_low(U, c, G) >= u0 ? 0 : 1); }
