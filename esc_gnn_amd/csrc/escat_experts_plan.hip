// escat_experts_plan.hip -- sorts the rows or (row, slot) pairs of a routing by expert (escat_experts.h): what every product of the experts
// goes by.
//
// A stable counting sort without atomics on memory, so that the order of the sums over an expert's rows is the same every
// time: a histogram per chunk of 2048 items, one workgroup that scans keys x chunks, a second pass over the items that ranks them (a wave
// ranks 64 items at once: lanes with the same key find each other by one ballot per bit of the key).
#include "escat_experts.h"

#define PT 256
#define PW (PT / 64)

// what is sorted: `n` items.  base = 0: item i has key experts[i] (one in [0, keys), else left out).  Else item i is a row of k experts.
struct Items { const int *experts; int64_t n; int k, base, keys; };

__device__ __forceinline__ int valid(int e, int E) { return e >= 0 && e < E ? e : E; }

// digit that entry i of a row's experts becomes: its rank among them
__device__ __forceinline__ int rank_of(const int *ex, int i, int k, int E)
{
    const int e = valid(ex[i], E);
    int r = 0;
    for (int j = 0; j < k; ++j) { const int o = valid(ex[j], E); r += o < e || (o == e && j < i); }
    return r;
}

__device__ __forceinline__ int key_of(const Items &it, int64_t i)
{
    if (i >= it.n) return -1;
    if (it.base == 0) { const int e = it.experts[i]; return e >= 0 && e < it.keys ? e : -1; }
    const int E = it.base - 1;
    const int *ex = it.experts + i * it.k;
    if (it.k == 1) return valid(ex[0], E);
    int key = 0;
    for (int j = 0; j < it.k; ++j) {
        int v = valid(ex[j], E);
        for (int q = it.k - 1 - rank_of(ex, j, it.k, E); q > 0; --q) v *= it.base;
        key += v;
    }
    return key;
}

// lanes of the wave that hold the same e (e >= 0); `bits` = bits of E - 1
__device__ __forceinline__ uint64_t same_lanes(int e, int bits)
{
    uint64_t m = ~0ull;
    for (int b = 0; b < bits; ++b) {
        const bool one = (e >> b) & 1;
        const uint64_t v = __ballot(one);
        m &= one ? v : ~v;
    }
    return m & __ballot(e >= 0);
}

#define PSTEPS (PLAN_CHUNK / PT)
// keys of the thread's items, all asked for at once; counts of the chunk's waves in LDS: cnt[wave][key]
__device__ __forceinline__ void wave_counts(const Items &it, int64_t c0, int bits, int *cnt, int (&key)[PSTEPS])
{
    const int E = it.keys;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (it.n > 0 && it.base && it.k <= 4) {                  // (places behind the last item read it again) a row's experts in registers, sorted there: no load waits for another
        const int Eb = it.base - 1;
        int v[PSTEPS][4];
#pragma unroll
        for (int s = 0; s < PSTEPS; ++s) {
            const int64_t i = c0 + wave * (PLAN_CHUNK / PW) + s * 64 + lane, at = (i < it.n ? i : it.n - 1) * it.k;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[s][j] = it.experts[at + (j < it.k ? j : it.k - 1)];
        }
#pragma unroll
        for (int s = 0; s < PSTEPS; ++s) {
            int d[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = j < it.k ? valid(v[s][j], Eb) : 0x7fffffff;
#define ORDER(a, b) { const int lo = min(d[a], d[b]), hi = max(d[a], d[b]); d[a] = lo; d[b] = hi; }
            ORDER(0, 1) ORDER(2, 3) ORDER(0, 2) ORDER(1, 3) ORDER(1, 2)
#undef ORDER
            int k = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) k = j < it.k ? k * it.base + d[j] : k;
            key[s] = c0 + wave * (PLAN_CHUNK / PW) + s * 64 + lane < it.n ? k : -1;
        }
    } else {
#pragma unroll
        for (int s = 0; s < PSTEPS; ++s) key[s] = key_of(it, c0 + wave * (PLAN_CHUNK / PW) + s * 64 + lane);
    }
    for (int i = threadIdx.x; i < PW * E; i += PT) cnt[i] = 0;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < PSTEPS; ++s) {
        const int e = key[s];
        const uint64_t m = same_lanes(e, bits);
        if (e >= 0 && (m & ((1ull << lane) - 1)) == 0) cnt[wave * E + e] += __popcll(m);
    }
    __syncthreads();
}

__global__ void __launch_bounds__(PT) k_plan_hist(const Items it, int bits, int *__restrict__ hist)
{
    const int E = it.keys;
    extern __shared__ int cnt[];
    int key[PSTEPS];
    wave_counts(it, (int64_t)blockIdx.x * PLAN_CHUNK, bits, cnt, key);
    for (int e = threadIdx.x; e < E; e += PT) {
        int s = 0;
#pragma unroll
        for (int w = 0; w < PW; ++w) s += cnt[w * E + e];
        hist[(int64_t)e * gridDim.x + blockIdx.x] = s;
    }
}

__device__ __forceinline__ int wave_scan_incl(int v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) { const int o = __shfl_up(v, m, 64); if (lane >= m) v += o; }
    return v;
}

// counts of the keys -> first positions and tiles, by one workgroup
struct KeyScan { int cnt[1025], first[1026], tfirst[1026]; };
__device__ __forceinline__ void scan_keys(int E, KeyScan &k, const EPlan &p)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    __syncthreads();
    if (wave == 0) {
        int run = 0, trun = 0;
        for (int e0 = 0; e0 < E; e0 += 64) {
            const int v = e0 + lane < E ? k.cnt[e0 + lane] : 0, t = (v + XM - 1) / XM;
            const int inc = wave_scan_incl(v), tinc = wave_scan_incl(t);
            if (e0 + lane < E) { k.first[e0 + lane] = run + inc - v; k.tfirst[e0 + lane] = trun + tinc - t; }
            run += __shfl(inc, 63, 64); trun += __shfl(tinc, 63, 64);
        }
        if (lane == 0) { k.first[E] = run; k.tfirst[E] = trun; *p.n_tiles = trun; }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) { p.count[e] = k.cnt[e]; p.first[e] = k.first[e]; }
    if (threadIdx.x == 0) p.first[E] = k.first[E];
    for (int e = wave; e < E; e += waves)
        for (int t = k.tfirst[e] + lane; t < k.tfirst[e + 1]; t += 64) {
            const int at = (t - k.tfirst[e]) * XM;
            *(int4 *)(p.tile + 4 * t) = make_int4(e, k.first[e] + at, k.cnt[e] - at < XM ? k.cnt[e] - at : XM, 0);
        }
}

// the chunk's items to their places; cnt[wave][key]: the next position of each wave
__device__ __forceinline__ void place_items(const Items &it, int64_t c0, int bits, int *cnt, const int (&key)[PSTEPS], const EPlan &p)
{
    const int E = it.keys;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 0; s < PSTEPS; ++s) {
        const int64_t i = c0 + wave * (PLAN_CHUNK / PW) + s * 64 + lane;
        const int e = key[s];
        const uint64_t m = same_lanes(e, bits), below = m & ((1ull << lane) - 1);
        int at = 0;
        if (e >= 0) at = cnt[wave * E + e] + __popcll(below);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier();      // all lanes have read before one writes
        if (e >= 0 && below == 0) cnt[wave * E + e] += __popcll(m);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier();
        if (i >= it.n) continue;
        if (it.base == 0) {
            p.pos[i] = e >= 0 ? at : -1;
            if (e >= 0) { p.pair[at] = (int)i; p.row[at] = (int)i / it.k; }
        } else {
            const int *ex = it.experts + i * it.k;
            for (int j = 0; j < it.k; ++j) {
                const int v = valid(ex[j], it.base - 1), s2 = at * it.k + (it.k == 1 ? 0 : rank_of(ex, j, it.k, it.base - 1));
                const bool to = v < it.base - 1;
                p.pair[s2] = (int)i * it.k + j; p.row[s2] = (int)i;
                p.pos[i * it.k + j] = to ? s2 : -1;
            }
        }
    }
}

// one workgroup of 1024: hist becomes each chunk's first position within its expert; counts, first positions, tiles
__global__ void __launch_bounds__(1024) k_plan_scan(int E, int blocks, EPlan p)
{
    __shared__ KeyScan k;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = wave; e < E; e += 16) {
        int *h = p.hist + (int64_t)e * blocks;
        int run = 0;
        for (int b0 = 0; b0 < blocks; b0 += 256) {           // four chunks a lane
            const int b = b0 + lane * 4;
            int v[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = b + i < blocks ? h[b + i] : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += v[i];
            const int inc = wave_scan_incl(sum);
            int at = run + inc - sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) { if (b + i < blocks) h[b + i] = at; at += v[i]; }
            run += __shfl(inc, 63, 64);
        }
        if (lane == 0) k.cnt[e] = run;
    }
    scan_keys(E, k, p);
}

__global__ void __launch_bounds__(PT) k_plan_place(const Items it, int bits, EPlan p)
{
    const int E = it.keys;
    extern __shared__ int cnt[];
    const int64_t c0 = (int64_t)blockIdx.x * PLAN_CHUNK;
    int key[PSTEPS];
    wave_counts(it, c0, bits, cnt, key);
    for (int e = threadIdx.x; e < E; e += PT) {               // counts -> the next position of each wave
        int s = p.first[e] + p.hist[(int64_t)e * gridDim.x + blockIdx.x];
#pragma unroll
        for (int w = 0; w < PW; ++w) { const int c = cnt[w * E + e]; cnt[w * E + e] = s; s += c; }
    }
    __syncthreads();
    place_items(it, c0, bits, cnt, key, p);
}

// all of it in one workgroup, for at most one chunk of items: one launch instead of three
__global__ void __launch_bounds__(PT) k_plan_small(const Items it, int bits, EPlan p)
{
    const int E = it.keys;
    extern __shared__ int cnt[];
    __shared__ KeyScan k;
    int key[PSTEPS];
    wave_counts(it, 0, bits, cnt, key);
    for (int e = threadIdx.x; e < E; e += PT) {
        int s = 0;
#pragma unroll
        for (int w = 0; w < PW; ++w) s += cnt[w * E + e];
        k.cnt[e] = s;
    }
    scan_keys(E, k, p);
    for (int e = threadIdx.x; e < E; e += PT) {
        int s = k.first[e];
#pragma unroll
        for (int w = 0; w < PW; ++w) { const int c = cnt[w * E + e]; cnt[w * E + e] = s; s += c; }
    }
    __syncthreads();
    place_items(it, 0, bits, cnt, key, p);
}

__global__ void __launch_bounds__(PT) k_copy_counts(const int *__restrict__ count, int E, int *__restrict__ out)
{
    for (int e = threadIdx.x; e < E; e += PT) out[e] = count[e];
}

// sorts `it` into p (hist in place)
static int run_plan(const Items &it, const EPlan &p, hipStream_t st)
{
    const int blocks = (int)plan_blocks(it.n);
    int bits = 0; while ((1 << bits) < it.keys) ++bits;
    const size_t lds = (size_t)PW * it.keys * 4;
    if (blocks <= 1) { k_plan_small<<<1, PT, lds, st>>>(it, bits, p); CHECK_LAUNCH("escat_experts_plan"); return ESCAT_OK; }
    k_plan_hist<<<blocks, PT, lds, st>>>(it, bits, p.hist);
    CHECK_LAUNCH("escat_experts_plan: histogram");
    k_plan_scan<<<1, 1024, 0, st>>>(it.keys, blocks, p);
    CHECK_LAUNCH("escat_experts_plan: scan");
    k_plan_place<<<blocks, PT, lds, st>>>(it, bits, p);
    CHECK_LAUNCH("escat_experts_plan: place");
    return ESCAT_OK;
}

// Positions of a plan by combination, sorted by expert (for the weights' gradients): by.pair = positions, by.row = their rows.  An expert's
// positions are those of its keys, one run after the other: no second sort (524288 rows, k = 2 of 8 experts: 13 us instead of 29).
// k_by_starts: starts[key * per + digit], where in its expert's positions such a run begins (by.hist, keys x per, holds them); counts and first positions of the experts.
__global__ void __launch_bounds__(1024) k_by_starts(const EPlan p, int E, const EPlan by)
{
    __shared__ int total[1024];                              // (E + 1)^k <= 1024 with k >= 2: 31 experts at most
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = wave; e < E; e += 16) {
        int run = 0;
        for (int k0 = 0; k0 < p.keys; k0 += 64) {
            const int key = k0 + lane, n = key < p.keys ? p.count[key] : 0;
            int times = 0;
            if (n > 0) for (int j = 0; j < p.per; ++j) times += key_digit(p, key, j) == e;
            const int inc = wave_scan_incl(n * times);
            int at = run + inc - n * times;
            if (times > 0) for (int j = 0; j < p.per; ++j) if (key_digit(p, key, j) == e) { by.hist[key * p.per + j] = at; at += n; }
            run += __shfl(inc, 63, 64);
        }
        if (lane == 0) total[e] = run;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int run = 0;
        for (int e = 0; e < E; ++e) { by.count[e] = total[e]; by.first[e] = run; run += total[e]; }
        by.first[E] = run;
    }
}

__global__ void __launch_bounds__(PT) k_by_fill(const EPlan p, int E, const EPlan by)
{
    if ((int)blockIdx.x >= *p.n_tiles) return;
    const int4 tile = *(const int4 *)(p.tile + 4 * blockIdx.x);
    const int key = tile.x, r0 = tile.y, rows = tile.z, r = threadIdx.x % XM;
    for (int j = threadIdx.x / XM; j < p.per; j += PT / XM) {
        const int e = key_digit(p, key, j);
        if (e >= E || r >= rows) continue;
        const int at = by.first[e] + by.hist[key * p.per + j] + r0 - p.first[key] + r, s = (r0 + r) * p.per + j;
        by.pair[at] = s;
        by.row[at] = p.row[s];
    }
}

int escat_experts_plan_by_expert(const EPlan &p, int64_t rows, int E, const EPlan &by, hipStream_t st)
{
    k_by_starts<<<1, 1024, 0, st>>>(p, E, by);
    CHECK_LAUNCH("escat_experts: by expert");
    k_by_fill<<<(unsigned)plan_max_tiles(rows, p.keys), PT, 0, st>>>(p, E, by);
    CHECK_LAUNCH("escat_experts: by expert");
    return ESCAT_OK;
}

static int plan_check(const char *who, int64_t rows, int k, int E)
{
    if (rows < 0 || k < 1 || E < 1) return fail(ESCAT_EINVAL, "%s: rows = %lld, k = %d, experts = %d", who, (long long)rows, k, E);
    if (rows > 0x3fffffff / k || E > ESCAT_ROUTE_MAX_EXPERTS) return fail(ESCAT_ERANGE, "%s: rows * k = %lld * %d (below 2^30), experts = %d (at most %d)", who, (long long)rows, k, E, ESCAT_ROUTE_MAX_EXPERTS);
    return ESCAT_OK;
}

extern "C" size_t escat_experts_plan_bytes(int64_t rows, int k, int E)
{
    return plan_check("escat_experts_plan_bytes", rows, k, E) ? 0 : (size_t)plan_ints(rows, k, E) * 4;
}

extern "C" int escat_experts_plan(const int32_t *experts, int64_t rows, int k, int E, void *plan, size_t plan_bytes, int32_t *counts, void *stream)
{
    int rc = plan_check("escat_experts_plan", rows, k, E); if (rc) return rc;
    if (rows > 0 && !experts) return fail(ESCAT_EINVAL, "escat_experts_plan: experts is null");
    if (counts && k != 1) return fail(ESCAT_EINVAL, "escat_experts_plan: counts are given for k = 1 (k = %d)", k);
    if (((uintptr_t)plan & 15) != 0) return fail(ESCAT_EINVAL, "escat_experts_plan: plan is not aligned to 16 bytes");
    if (!plan || plan_bytes < escat_experts_plan_bytes(rows, k, E)) return fail(ESCAT_EWORKSPACE, "escat_experts_plan: plan of %zu bytes, needs %zu", plan_bytes, escat_experts_plan_bytes(rows, k, E));
    hipStream_t st = (hipStream_t)stream;
    const EPlan p = plan_of(plan, rows, k, E);
    rc = run_plan({experts, p.base ? rows : rows * k, k, p.base, p.keys}, p, st); if (rc) return rc;
    if (counts) { k_copy_counts<<<1, PT, 0, st>>>(p.count, E, counts); CHECK_LAUNCH("escat_experts_plan: counts"); }
    return ESCAT_OK;
}
