// escat_experts.h -- shared by the units of the experts' products (escat_experts_plan / _rows / _grad.hip); not part of the ABI
#ifndef ESCAT_EXPERTS_H
#define ESCAT_EXPERTS_H
#include "escat_dev.h"
#include "escat_half.h"

// How rows meet experts.  A tile is 128 items that share a key, and the products of a tile go to `per` experts, the digits of its key:
//
//   by pair         items = (row, slot) pairs, key = the pair's expert, per = 1: each pair's result is kept in fp32 and the k of a row are
//                   added by a pass of their own.
//   by combination  items = rows, key = the sorted k experts of a row as digits to the base E + 1 (E: routed nowhere), per = k: the k products
//                   of a tile's rows end in the same accumulators, and results are written once, in their own type.
//
// By combination moves less memory (no fp32 results of pairs written and read again) but cuts the rows into C(E + k - 1, k) groups, pads each
// to whole tiles, and a tile walks k experts one after the other: taken with 2048 rows or more to a group and at most 1024 keys.  One number for
// all: with 8 experts bf16 crosses over near 1024 rows (8 % left there) and fp32 near 2048 (1 % either way).  Forward and backward by
// combination / by pair, us, 256 wide, at 512, 1024, 2048, 4096 rows to a group:
//   bf16, 8 experts, k = 2   205/184  255/277  379/444  610/769       fp32   512/457  781/764  1415/1405  2573/2638
//   bf16, 4 experts, k = 3   203/150  251/236  336/377  527/644       fp32   439/347  701/629  1177/1154  2208/2204
// k = 1 is always its case, the two are the same there.
struct EDims { int64_t rows; int d, h, o, E, k; };
static inline int combo_keys(int64_t rows, int E, int k)        // number of keys by combination, 0 = by pair
{
    int64_t keys = 1, groups = 1;
    for (int j = 0; j < k; ++j) { keys *= E + 1; if (keys > 1025) return 0; }
    if (k == 1) return (int)keys;
    if (keys > 1024) return 0;
    for (int j = 0; j < k; ++j) groups = groups * (E + j) / (j + 1);         // multisets of k experts
    return rows >= 2048 * groups ? (int)keys : 0;
}

// A position is item * per + digit; of the plan (device memory, int32):
struct EPlan {
    int per, base;    // base: E + 1 by combination, 0 by pair (the key is the expert)
    int keys;
    int *count;       // keys      items of each key
    int *first;       // keys + 1  its first item in sorted order; first[keys] = all items
    int *n_tiles;     // 1         tiles of XM items, none across two keys
    int *tile;        // 4 x max_tiles: key, first item, items, 0
    int *pair;        // P         position -> pair
    int *row;         // P         position -> row of the activations
    int *pos;         // P         pair -> position, -1 = not routed
    int *hist;        // keys x blocks: scratch of the sort
};
#define XM 128                                    // items of a tile (rows of activations)
#define XN 128                                    // features of a tile
#define PLAN_CHUNK 2048                           // items of a workgroup of the sort

static inline int64_t plan_items(int64_t rows, int k, int combo) { return combo ? rows : rows * k; }
static inline int64_t plan_blocks(int64_t items) { return (items + PLAN_CHUNK - 1) / PLAN_CHUNK; }
static inline int64_t plan_max_tiles(int64_t items, int keys) { return items / XM + (keys < items ? keys : items) + 1; }
static inline EPlan plan_view(void *mem, int64_t rows, int k, int E, int combo, int64_t *ints)
{
    EPlan p; int *q = (int *)mem;
    const int64_t items = plan_items(rows, k, combo), P = rows * k;
    p.per = combo ? k : 1; p.base = combo ? E + 1 : 0; p.keys = combo ? combo : E;
    p.count = q; q += p.keys; p.first = q; q += p.keys + 1; p.n_tiles = q; q += 1;
    q += (4 - (q - (int *)mem) % 4) % 4;
    p.tile = q; q += 4 * plan_max_tiles(items, p.keys);
    p.pair = q; q += P; p.row = q; q += P; p.pos = q; q += P;
    p.hist = q; q += p.keys * plan_blocks(items);
    if (ints) *ints = q - (int *)mem;
    return p;
}
// the plan of a routing, as escat_experts_plan lays it out
static inline EPlan plan_of(void *mem, int64_t rows, int k, int E) { return plan_view(mem, rows, k, E, combo_keys(rows, E, k), nullptr); }
static inline int64_t plan_ints(int64_t rows, int k, int E) { int64_t n; plan_view(nullptr, rows, k, E, combo_keys(rows, E, k), &n); return n; }

// Whether a training forward leaves u in fp32 next to the hidden rows: 8 bytes an element written and read (2 ps at 4.8 TB/s), or 2 d operations once more
// (0.033 d ps at the 60 TFLOP/s that fp32 tiles reach; 0.003 d with 16-bit operands).  Forward and backward, kept / computed again, us:
//   fp32  32768 rows, k = 2 of 8 experts, d -> 256 -> 256: d = 32 518/507  64 528/528  128 555/577  256 669/734;  8192 rows, 16 of 1024 -> 1024 -> 1024 1988/2296
//   bf16  d -> 256 -> 256: 262144 rows of 256 1061/1001  131072 of 512 742/727  65536 of 768 660/685  of 1024 800/837;  8192 rows, 64 of 1024 -> 2048 -> 1024 897/945
static inline bool keeps_u(int type, int d) { return d > (type == ESCAT_F32 ? 64 : 640); }

// expert of digit j of a key; E (base - 1): none
__device__ __forceinline__ int key_digit(const EPlan &p, int key, int j)
{
    if (p.base == 0) return key;
    for (int i = p.per - 1; i > j; --i) key /= p.base;
    return key % p.base;
}

// workgroups of a launch go round the eight XCDs one by one, each with its own L2: give each XCD a run of neighbouring work items
// (neighbours share the expert's weights and the rows).  A permutation of [0, n).
__device__ __forceinline__ int xcd_swizzle(int b, int n)
{
    const int per = n >> 3, rest = n & 7, x = b & 7, i = b >> 3;
    return x * per + (x < rest ? x : rest) + i;
}
#endif
