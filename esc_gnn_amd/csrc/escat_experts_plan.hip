// escat_experts_plan.hip -- sorts the (row, slot) pairs of a routing by expert: what every product of the experts goes by.
//
// A stable counting sort without atomics on memory, so that the order of the sums over an expert's rows is the same every
// time: a histogram per chunk of 2048 pairs, one workgroup that scans experts x chunks, a second pass over the pairs that ranks them (a wave
// ranks 64 pairs at once: lanes with the same expert find each other by one ballot per bit of the expert's number).
#include "escat_experts.h"

#define PT 256
#define PW (PT / 64)

__device__ __forceinline__ int expert_of(const int *experts, int64_t i, int64_t P, int E)
{
    const int e = i < P ? experts[i] : -1;
    return e >= 0 && e < E ? e : -1;
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

// counts of the chunk's waves in LDS: cnt[wave][E]
__device__ __forceinline__ void wave_counts(const int *experts, int64_t c0, int64_t P, int E, int bits, int *cnt)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < PW * E; i += PT) cnt[i] = 0;
    __syncthreads();
    for (int s = 0; s < PLAN_CHUNK / PT; ++s) {
        const int64_t i = c0 + wave * (PLAN_CHUNK / PW) + s * 64 + lane;
        const int e = expert_of(experts, i, P, E);
        const uint64_t m = same_lanes(e, bits);
        if (e >= 0 && (m & ((1ull << lane) - 1)) == 0) cnt[wave * E + e] += __popcll(m);
    }
    __syncthreads();
}

__global__ void __launch_bounds__(PT) k_plan_hist(const int *__restrict__ experts, int64_t P, int E, int bits, int *__restrict__ hist)
{
    extern __shared__ int cnt[];
    wave_counts(experts, (int64_t)blockIdx.x * PLAN_CHUNK, P, E, bits, cnt);
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

// one workgroup of 1024: hist becomes each chunk's first position within its expert; counts, first positions, tiles
__global__ void __launch_bounds__(1024) k_plan_scan(int E, int blocks, EPlan p)
{
    __shared__ int cnt[1024], first[1025], tfirst[1025];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = wave; e < E; e += 16) {
        int *h = p.hist + (int64_t)e * blocks;
        int run = 0;
        for (int b0 = 0; b0 < blocks; b0 += 64) {
            const int v = b0 + lane < blocks ? h[b0 + lane] : 0;
            const int inc = wave_scan_incl(v);
            if (b0 + lane < blocks) h[b0 + lane] = run + inc - v;
            run += __shfl(inc, 63, 64);
        }
        if (lane == 0) cnt[e] = run;
    }
    __syncthreads();
    if (wave == 0) {
        int run = 0, trun = 0;
        for (int e0 = 0; e0 < E; e0 += 64) {
            const int v = e0 + lane < E ? cnt[e0 + lane] : 0, t = (v + XM - 1) / XM;
            const int inc = wave_scan_incl(v), tinc = wave_scan_incl(t);
            if (e0 + lane < E) { first[e0 + lane] = run + inc - v; tfirst[e0 + lane] = trun + tinc - t; }
            run += __shfl(inc, 63, 64); trun += __shfl(tinc, 63, 64);
        }
        if (lane == 0) { first[E] = run; tfirst[E] = trun; *p.n_tiles = trun; }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += 1024) { p.count[e] = cnt[e]; p.first[e] = first[e]; }
    if (threadIdx.x == 0) p.first[E] = first[E];
    for (int e = wave; e < E; e += 16)
        for (int t = tfirst[e] + lane; t < tfirst[e + 1]; t += 64) { p.tile[2 * t] = e; p.tile[2 * t + 1] = first[e] + (t - tfirst[e]) * XM; }
}

__global__ void __launch_bounds__(PT) k_plan_place(const int *__restrict__ experts, int64_t P, int k, int E, int bits, EPlan p)
{
    extern __shared__ int cnt[];
    const int64_t c0 = (int64_t)blockIdx.x * PLAN_CHUNK;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    wave_counts(experts, c0, P, E, bits, cnt);
    for (int e = threadIdx.x; e < E; e += PT) {               // counts -> the next position of each wave
        int s = p.first[e] + p.hist[(int64_t)e * gridDim.x + blockIdx.x];
#pragma unroll
        for (int w = 0; w < PW; ++w) { const int c = cnt[w * E + e]; cnt[w * E + e] = s; s += c; }
    }
    __syncthreads();
    for (int s = 0; s < PLAN_CHUNK / PT; ++s) {
        const int64_t i = c0 + wave * (PLAN_CHUNK / PW) + s * 64 + lane;
        const int e = expert_of(experts, i, P, E);
        const uint64_t m = same_lanes(e, bits), below = m & ((1ull << lane) - 1);
        int at = 0;
        if (e >= 0) at = cnt[wave * E + e] + __popcll(below);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier();      // all lanes have read before one writes
        if (e >= 0 && below == 0) cnt[wave * E + e] += __popcll(m);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier();
        if (i < P) { p.pos[i] = e >= 0 ? at : -1; if (e >= 0) { p.pair[at] = (int)i; p.row[at] = (int)i / k; } }
    }
}

__global__ void __launch_bounds__(PT) k_copy_counts(const int *__restrict__ count, int E, int *__restrict__ out)
{
    for (int e = threadIdx.x; e < E; e += PT) out[e] = count[e];
}

static int plan_check(const char *who, int64_t P, int E)
{
    if (P < 0 || E < 1) return fail(ESCAT_EINVAL, "%s: pairs = %lld, E = %d", who, (long long)P, E);
    if (P > 0x3fffffff || E > ESCAT_ROUTE_MAX_EXPERTS) return fail(ESCAT_ERANGE, "%s: pairs = %lld (below 2^30), E = %d (at most %d)", who, (long long)P, E, ESCAT_ROUTE_MAX_EXPERTS);
    return ESCAT_OK;
}

extern "C" size_t escat_experts_plan_bytes(int64_t pairs, int E)
{
    return pairs < 0 || E < 1 || E > ESCAT_ROUTE_MAX_EXPERTS ? 0 : (size_t)plan_ints(pairs, E) * 4;
}

extern "C" int escat_experts_plan(const int32_t *experts, int64_t pairs, int k, int E, void *plan, size_t plan_bytes, int32_t *counts, void *stream)
{
    int rc = plan_check("escat_experts_plan", pairs, E); if (rc) return rc;
    if (k < 1) return fail(ESCAT_EINVAL, "escat_experts_plan: k = %d", k);
    if (pairs > 0 && !experts) return fail(ESCAT_EINVAL, "escat_experts_plan: experts is null");
    if (!plan || plan_bytes < escat_experts_plan_bytes(pairs, E)) return fail(ESCAT_EWORKSPACE, "escat_experts_plan: plan of %zu bytes, needs %zu", plan_bytes, escat_experts_plan_bytes(pairs, E));
    hipStream_t st = (hipStream_t)stream;
    const EPlan p = plan_view(plan, pairs, E);
    const int blocks = (int)plan_blocks(pairs);
    int bits = 0; while ((1 << bits) < E) ++bits;
    const size_t lds = (size_t)PW * E * 4;
    if (blocks) { k_plan_hist<<<blocks, PT, lds, st>>>(experts, pairs, E, bits, p.hist); CHECK_LAUNCH("escat_experts_plan: histogram"); }
    k_plan_scan<<<1, 1024, 0, st>>>(E, blocks, p);
    CHECK_LAUNCH("escat_experts_plan: scan");
    if (blocks) { k_plan_place<<<blocks, PT, lds, st>>>(experts, pairs, k, E, bits, p); CHECK_LAUNCH("escat_experts_plan: place"); }
    if (counts) { k_copy_counts<<<1, PT, 0, st>>>(p.count, E, counts); CHECK_LAUNCH("escat_experts_plan: counts"); }
    return ESCAT_OK;
}
