// escat_experts_grad.hip -- gradients of the experts' weights: sums over an expert's rows of outer products,
//
//   dW2_e[o][h] = sum_r dy_r[o] (w h)_r[h]    db2_e[o] = sum_r w_r dy_r[o]    dW1_e[h][d] = sum_r du_r[h] x_r[d]    db1_e[h] = sum_r du_r[h]
//
// as matrix tiles with the rows as the summed index: both operands lie in memory with their features contiguous, so they are staged
// as they are and transposed on the way out of LDS.  A tile of 128 x 128 results sums all of an expert's rows where there are
// tiles enough to fill the chip; otherwise the rows are cut into chunks, whose fp32 results a second kernel adds in order.  The bias
// gradients ride along: a tile's B pieces pass through registers anyway.
#include "escat_experts_tile.h"

struct GradArgs {
    EDims n;
    EPlan p;                   // by pair: items in the order of the sums
    const int *at;             // position of an item's hidden row; NULL: the item itself
    const void *a, *b;         // A: (w h) by position, or x by row; B: dy by row, or du by position
    const float *weights;      // by position: db2's
    void *out, *db;            // (E, N, M), (E, N) of the operands' type
    float *part;               // chunked: [chunk][N * M + N]
    int M, N;                  // A's and B's features
    int chunk;                 // rows of a chunk; 0 = all of an expert's
};

__device__ __forceinline__ int wave_incl(int v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) { const int o = __shfl_up(v, m, 64); if (lane >= m) v += o; }
    return v;
}

// chunk q -> its expert (-1: none) and the number of its chunk; every wave does it for itself
__device__ __forceinline__ int find_chunk(const int *count, int E, int chunk, int q, int &of)
{
    const int lane = threadIdx.x & 63;
    int run = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
        const int v = e0 + lane < E ? (count[e0 + lane] + chunk - 1) / chunk : 0;
        const int inc = run + wave_incl(v);
        const uint64_t hit = __ballot(q < inc);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            of = q - (__shfl(inc, l, 64) - __shfl(v, l, 64));
            return __builtin_amdgcn_readfirstlane(e0 + l);
        }
        run = __shfl(inc, 63, 64);
    }
    return -1;
}

// W2: A by sorted position, B gathered by row and weighted for db; else A gathered by row, B by sorted position
template <typename T, bool W2>
__global__ void __launch_bounds__(XT, 3) k_expert_grad(const GradArgs g)
{
    constexpr int PER = Elem<T>::PER, KB = Elem<T>::KB;
    extern __shared__ __align__(16) char lds[];
    typedef Stage<T, true> SM;
    const int M = g.M, N = g.N, mt = (M + XN - 1) / XN, nt = (N + XN - 1) / XN;
    // Chunks cost the same: each XCD gets a run of them.  Experts do not: their stripes (the tiles that share B's features) go round the XCDs
    // one by one (64 experts of 100 to 500 rows, 1024 x 2048: 172 instead of 220 us)
    const int stripe = ((int)blockIdx.x >> 3) / mt * 8 + (int)(blockIdx.x & 7);
    const int work = g.chunk ? xcd_swizzle(blockIdx.x, gridDim.x) : stripe * mt + ((int)blockIdx.x >> 3) % mt;
    const int q = work / (mt * nt), tile = work - q * mt * nt;
    const int m0 = (tile % mt) * XN, n0 = (tile / mt) * XN;
    int e = q, of = 0;
    if (!g.chunk && e >= g.n.E) return;
    if (g.chunk) { e = find_chunk(g.p.count, g.n.E, g.chunk, q, of); if (e < 0) return; }
    const int end = g.p.first[e + 1], ra = g.p.first[e] + of * g.chunk;
    const int rb = g.chunk && ra + g.chunk < end ? ra + g.chunk : end;

    const int wave = threadIdx.x >> 6, am = (wave & 1) * 64, bn = (wave >> 1) * 64;
    const bool sums = m0 == 0 && g.db != nullptr;
    const int K = rb - ra;
    // the two operands and the items' rows and positions, which are fetched a step ahead of the data
    struct Items {
        const GradArgs &g;
        int ra, rb, k0;
        int row[4], pos[4], row_next[4], pos_next[4];
        __device__ __forceinline__ void fetch()
        {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int s = ra + k0 + SM::row(i) < rb ? ra + k0 + SM::row(i) : rb - 1;
                row_next[i] = g.p.row[s];
                pos_next[i] = g.at ? g.at[s] : s;
            }
            k0 += KB;
        }
    } it{g, ra, rb, 0};
    struct OpA {
        Items &it; const GradArgs &g; ColsKM<T> cols; int K, fk0;
        __device__ __forceinline__ void load(u4 (&r)[4])
        {
#pragma unroll
            for (int i = 0; i < 4; ++i) { it.row[i] = it.row_next[i]; it.pos[i] = it.pos_next[i]; }
            it.fetch();                                       // before the data: memory answers in order, and the next step waits for these
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = load16((const T *)g.a + (int64_t)(W2 ? it.pos[i] : it.row[i]) * g.M + cols.at);
        }
        __device__ __forceinline__ void fix(u4 (&r)[4]) { cols.fix(r, K - fk0, fk0 + KB <= K); fk0 += KB; }
    } A{it, g, ColsKM<T>(m0, M), K, 0};
    struct OpB {
        Items &it; const GradArgs &g; ColsKM<T> cols; int K, fk0; bool sums;
        float w[4], db[PER];
        __device__ __forceinline__ void load(u4 (&r)[4])
        {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r[i] = load16((const T *)g.b + (int64_t)(W2 ? it.row[i] : it.pos[i]) * g.N + cols.at);
                if (W2) w[i] = g.weights[it.pos[i]];
            }
        }
        __device__ __forceinline__ void fix(u4 (&r)[4])
        {
            cols.fix(r, K - fk0, fk0 + KB <= K);
            fk0 += KB;
            if (!sums) return;
            float f[PER];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                to_floats<T>(r[i], f);
#pragma unroll
                for (int z = 0; z < PER; ++z) db[z] = W2 ? fmaf(w[i], f[z], db[z]) : db[z] + f[z];
            }
        }
    } B{it, g, ColsKM<T>(n0, N), K, 0, sums};
#pragma unroll
    for (int i = 0; i < PER; ++i) B.db[i] = 0.f;
    acc_t acc[2][2];
    clear(acc);
    if (K > 0) it.fetch();
    const int steps = (K + KB - 1) / KB;
    Pipe<T, true, true> pipe;
    pipe.start(steps, A, B);
    pipe.run(steps, lds, am, bn, acc, A, B);

    float *part = g.chunk ? g.part + (int64_t)q * ((int64_t)N * M + N) : nullptr;
    if (sums) {                                               // the threads that hold the same features join in a fixed order
        float *red = (float *)lds;
#pragma unroll
        for (int z = 0; z < PER; ++z) red[threadIdx.x * PER + z] = B.db[z];
        __syncthreads();
        if (threadIdx.x < 128 && n0 + (int)threadIdx.x < N) {
            float v = 0.f;
            for (int i = 0; i < SM::RPP; ++i) v += red[i * 128 + threadIdx.x];
            const int n = n0 + threadIdx.x;
            if (part) part[(int64_t)N * M + n] = v;
            else ((T *)g.db)[(int64_t)e * N + n] = from_f32<T>(v);
        }
    }
    if (sums) __syncthreads();
    const int cols = M - m0 < XN ? M - m0 : XN, rows = N - n0 < XN ? N - n0 : XN;
    if (part) {
        Spill<float>::all(lds, acc, am, bn, part + (int64_t)n0 * M + m0, M, rows, cols, [](int r) { return r; });
    } else {
        Spill<T>::all(lds, acc, am, bn, (T *)g.out + ((int64_t)e * N + n0) * M + m0, M, rows, cols, [](int r) { return r; });
    }
}

// adds an expert's chunks in order: out[e][i] = sum_c part[first chunk + c][i]; the last N of a chunk's values are db's
template <typename T>
__global__ void __launch_bounds__(XT) k_grad_join(const GradArgs g)
{
    const int e = blockIdx.y;
    const int64_t NM = (int64_t)g.N * g.M, len = NM + g.N;
    int first = 0, chunks = 0;
    for (int i0 = 0; i0 <= e; i0 += 64) {
        const int lane = threadIdx.x & 63;
        int v = i0 + lane <= e ? (g.p.count[i0 + lane] + g.chunk - 1) / g.chunk : 0;
        chunks = __shfl(v, (e - i0) & 63, 64);               // (of the last round: e itself)
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
        first += v;
    }
    first -= chunks;
    const float *p = g.part + (int64_t)first * len;
    const int64_t end = g.db ? len : NM;                     // (no bias: its places were never written)
    for (int64_t i = ((int64_t)blockIdx.x * XT + threadIdx.x) * 4; i < end; i += (int64_t)gridDim.x * XT * 4) {
        // four values from `at` on: at the end they begin earlier and the first ones are a neighbour's too, who writes the same
        const int64_t at = i + 4 <= end ? i : end - 4;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int c0 = 0; c0 < chunks; c0 += 8) {             // eight in flight; behind the last: the last, not added
            Pack<float, 4> v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = *(const Pack<float, 4> *)(p + (c0 + c < chunks ? c0 + c : chunks - 1) * len + at);
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int z = 0; z < 4; ++z) s[z] = c0 + c < chunks ? s[z] + v[c].v[z] : s[z];
        }
        if (at + 4 <= NM) {
            Pack<T, 4> o;
#pragma unroll
            for (int z = 0; z < 4; ++z) o.v[z] = from_f32<T>(s[z]);
            *(Pack<T, 4> *)((T *)g.out + e * NM + at) = o;
        } else {
#pragma unroll
            for (int z = 0; z < 4; ++z)
                if (at + z < NM) ((T *)g.out)[e * NM + at + z] = from_f32<T>(s[z]);
                else ((T *)g.db)[(int64_t)e * g.N + (at + z - NM)] = from_f32<T>(s[z]);
        }
    }
}

// rows of a chunk: none cut where the experts' tiles alone are 1024 workgroups or more; else, with a last chunk for each expert, about one round: 720 in
// all, three a CU (8 experts, 1048576 pairs, 256 x 256 in bf16: 274 and 257 us for the two gradients, 1024: 294 and 284,
// 1440: 272 and 261 but 8 us more to join); in fp32, which the matrix units bound, two a CU (32768 pairs, 256 x 242 and 256 x 256: 55 and 54 us, 720:
// 65 and 65).  No chunk has fewer than 256 rows.
int escat_experts_grad_chunk(int type, int64_t P, int E, int M, int N)
{
    const int64_t tiles = (int64_t)((M + XN - 1) / XN) * ((N + XN - 1) / XN);
    if (tiles * E >= 1024 || P <= 256) return 0;
    const int64_t want = ((type == ESCAT_F32 ? 480 : 720) + tiles - 1) / tiles;
    int64_t r = (P + want - 1) / want;
    r = (r + 63) / 64 * 64;
    return (int)(r < 256 ? 256 : r);
}
int64_t escat_experts_grad_chunks(int64_t P, int E, int chunk) { return chunk ? P / chunk + (E < P ? E : P) : E; }

template <typename T, bool W2> static int launch(const GradArgs &g, hipStream_t st)
{
    const int64_t tiles = (int64_t)((g.M + XN - 1) / XN) * ((g.N + XN - 1) / XN);
    const int64_t mt = (g.M + XN - 1) / XN, stripes = (tiles / mt * g.n.E + 7) / 8 * 8;
    const int64_t wgs = g.chunk ? tiles * escat_experts_grad_chunks(g.n.rows * g.n.k, g.n.E, g.chunk) : stripes * mt;
    if (wgs > 0xffffff) return fail(ESCAT_ERANGE, "experts: %lld tiles", (long long)wgs);
    constexpr size_t lds = LDS_BYTES;
    int rc = set_lds(k_expert_grad<T, W2>, lds); if (rc) return rc;
    k_expert_grad<T, W2><<<(unsigned)wgs, XT, lds, st>>>(g);
    CHECK_LAUNCH("experts: weight gradient");
    if (g.chunk) {
        const int64_t len = (int64_t)g.N * g.M + g.N, b = (len / 4 + XT) / XT;
        k_grad_join<T><<<dim3((unsigned)(b < 4096 ? b : 4096), (unsigned)g.n.E), XT, 0, st>>>(g);
        CHECK_LAUNCH("experts: weight gradient, joined");
    }
    return ESCAT_OK;
}

int escat_experts_grad(int type, const EDims &n, const EPlan &p, const int *at, bool w2, const void *a, const void *b, const float *weights, int M, int N,
                       int chunk, float *part, void *out, void *db, hipStream_t st)
{
    const GradArgs g = {n, p, at, a, b, weights, out, db, part, M, N, chunk};
    if (w2) return type == ESCAT_F32 ? launch<float, true>(g, st) : type == ESCAT_BF16 ? launch<bf16_t, true>(g, st) : launch<f16_t, true>(g, st);
    return type == ESCAT_F32 ? launch<float, false>(g, st) : type == ESCAT_BF16 ? launch<bf16_t, false>(g, st) : launch<f16_t, false>(g, st);
}
