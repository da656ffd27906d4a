// escat_experts.h -- shared by the units of the experts' products (escat_experts_plan / _rows / _grad.hip); not part of the ABI
#ifndef ESCAT_EXPERTS_H
#define ESCAT_EXPERTS_H
#include "escat_dev.h"
#include "escat_half.h"

// Pairs = (row, slot) with a routed expert, sorted by expert, stable.  Of the plan (device memory, int32):
struct EPlan {
    int *count;       // E      pairs of each expert
    int *first;       // E + 1  its first sorted position; first[E] = routed pairs
    int *n_tiles;     // 1      tiles of XM sorted positions, none across two experts
    int *tile;        // 2 x max_tiles: expert, first position
    int *pair;        // P      sorted position -> pair
    int *pos;         // P      pair -> sorted position, -1 = not routed
    int *row;         // P      sorted position -> row of the activations (pair / k)
    int *hist;        // E x blocks: scratch of the sort
};
#define XM 128                                    // sorted positions of a tile (rows of activations)
#define XN 128                                    // features of a tile
#define PLAN_CHUNK 2048                           // pairs of a workgroup of the sort

struct EDims { int64_t rows; int d, h, o, E, k; };

static inline int64_t plan_blocks(int64_t P) { return (P + PLAN_CHUNK - 1) / PLAN_CHUNK; }
static inline int64_t plan_max_tiles(int64_t P, int E) { return P / XM + (E < P ? E : P) + 1; }
static inline int64_t plan_ints(int64_t P, int E)
{
    return (int64_t)E + (E + 1) + 1 + 2 * plan_max_tiles(P, E) + 3 * P + E * plan_blocks(P) + 64;
}
static inline EPlan plan_view(void *mem, int64_t P, int E)
{
    EPlan p; int *q = (int *)mem;
    p.count = q; q += E; p.first = q; q += E + 1; p.n_tiles = q; q += 1; p.tile = q; q += 2 * plan_max_tiles(P, E);
    p.pair = q; q += P; p.pos = q; q += P; p.row = q; q += P; p.hist = q;
    return p;
}

// workgroups of a launch go round the eight XCDs one by one, each with its own L2: give each XCD a run of neighbouring work items
// (neighbours share the expert's weights and the rows).  A permutation of [0, n).
__device__ __forceinline__ int xcd_swizzle(int b, int n)
{
    const int per = n >> 3, rest = n & 7, x = b & 7, i = b >> 3;
    return x * per + (x < rest ? x : rest) + i;
}
#endif
