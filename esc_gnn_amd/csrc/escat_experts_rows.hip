// escat_experts_rows.hip -- the experts' products over rows of activations, forward and backward:
//
//   pair (t, j), e = experts[t, j]:   u = W1_e x_t + b1_e    h = silu(u)    y_t = sum_j w_tj (W2_e h + b2_e)
//   G = W2_e^T dy_t    dw_tj = h.G + b2.dy_t    du = w G silu'(u)    dx_t = sum_j W1_e^T du
//
// Rows are taken in the plan's order (sorted by expert), 128 to a tile.  The weight w goes into the hidden row before it is
// rounded to the operands' type (w h): it then serves W2's product and W2's gradient without another pass.  Nothing of the
// forward is kept for the backward: u is computed again next to G, in fp32, so that dw and silu' see no rounding of u, and the
// forward writes no u.  Results of the pairs are joined in fp32 by a pass of their own, in the order of the slots: no atomics.
#include <type_traits>
#include "escat_experts_tile.h"

struct RowArgs {
    EDims n;
    EPlan p;
    const void *x, *w1, *b1, *w2, *b2, *dy;
    const float *weights;
    void *h;                   // (P, H) sorted: w silu(u)
    void *du;                  // (P, H) sorted
    float *part;               // (P, O) or (P, D) fp32, sorted: what the joining pass reads
    float *dwp;                // (feature tiles of H, P) sorted: parts of dw
    float *ws;                 // (P) sorted: w (BWD1 leaves them for the weights' gradients)
};

enum { FWD1, FWD2, BWD1, BWD2 };

// the hardware's exponential errs by |u| 2^-24: below what 16-bit operands leave, not below what fp32 ones do
template <typename T> __device__ __forceinline__ float sigmoid_of(float u) { return 1.f / (1.f + (sizeof(T) == 4 ? expf(-u) : __expf(-u))); }

template <typename T, int MODE>
__global__ void __launch_bounds__(XT, 2) k_expert_rows(const RowArgs a)
{
    constexpr int PER = Elem<T>::PER, KB = Elem<T>::KB;
    extern __shared__ __align__(16) char lds[];
    const int D = a.n.d, H = a.n.h, O = a.n.o;
    const int M = MODE == FWD2 ? O : MODE == BWD2 ? D : H;          // features of the result
    const int mt = (M + XN - 1) / XN;
    const int live = *a.p.n_tiles * mt;                              // (the grid covers the most tiles there can be)
    if ((int)blockIdx.x >= live) return;
    const int work = xcd_swizzle(blockIdx.x, live), t = work / mt, m0 = (work - t * mt) * XN;
    const int e = a.p.tile[2 * t], r0 = a.p.tile[2 * t + 1];
    const int rows = a.p.first[e + 1] - r0 < XM ? a.p.first[e + 1] - r0 : XM;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, am = (wave & 1) * 64, bn = (wave >> 1) * 64;
    typedef Stage<T, false> SC;
    const int c = SC::chunk() * PER;
    // the thread's four rows of activations (rows behind the last of the tile repeat it: their results are not written)
    int64_t br[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = SC::row(i) < rows ? SC::row(i) : rows - 1;
        br[i] = MODE == FWD2 || MODE == BWD2 ? (int64_t)(r0 + r) : (int64_t)a.p.row[r0 + r];
    }
    float wr[2];                                                    // weights of the two rows whose results the lane holds
#pragma unroll
    for (int j = 0; j < 2; ++j) { const int r = bn + 32 * j + (lane & 31); wr[j] = MODE == BWD2 ? 1.f : a.weights[a.p.pair[r0 + (r < rows ? r : 0)]]; }
    __shared__ __align__(16) float bias[XN];
    if (MODE != BWD2 && threadIdx.x < XN) {
        const T *b = MODE == FWD2 ? (const T *)a.b2 : (const T *)a.b1;
        bias[threadIdx.x] = b && m0 + (int)threadIdx.x < M ? to_f32(b[(int64_t)e * M + m0 + threadIdx.x]) : 0.f;
    }
    acc_t acc[2][2];
    clear(acc);

    // ---- first product: W1 x (FWD1, BWD1), W2 (w h) (FWD2), W1^T du (BWD2)
    if (MODE != BWD2) {
        const int K = MODE == FWD2 ? H : D;
        const T *A = (const T *)(MODE == FWD2 ? a.w2 : a.w1) + (int64_t)e * M * K, *B = (const T *)(MODE == FWD2 ? a.h : a.x);
        RowsKC<T> la, lb;
        la.K = lb.K = K; la.c = lb.c = c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + SC::row(i) < M ? m0 + SC::row(i) : M - 1;
            la.p[i] = A + (int64_t)m * K;
            lb.p[i] = B + br[i] * K;
        }
        tile_loop<MODE == BWD1 ? 1 : 2, T, false, false>(K, lds, am, bn, acc, [&](int k0, u4 (&r)[4], int) { la.load(k0, r); }, [&](int k0, u4 (&r)[4], int) { lb.load(k0, r); },
                                   [&](int k0, u4 (&r)[4], int) { la.fix(k0, r); }, [&](int k0, u4 (&r)[4], int) { lb.fix(k0, r); });
    }
    // ---- W2^T dy (BWD1, into a second set), W1^T du (BWD2): weights with the result's features contiguous
    acc_t acc2[2][2];
    float dot[4] = {0.f, 0.f, 0.f, 0.f};                            // BWD1: the thread's share of b2 . dy of its rows
    if (MODE == BWD1 || MODE == BWD2) {
        const int K = MODE == BWD1 ? O : H;
        const T *A = (const T *)(MODE == BWD1 ? a.w2 : a.w1) + (int64_t)e * K * M, *B = (const T *)(MODE == BWD1 ? a.dy : a.du);
        typedef Stage<T, true> SM;
        const ColsKM<T> cols_a(m0, M);
        RowsKC<T> lb;
        lb.K = K; lb.c = c;
#pragma unroll
        for (int i = 0; i < 4; ++i) lb.p[i] = B + br[i] * K;
        const bool with_dot = MODE == BWD1 && m0 == 0 && a.b2 != nullptr;
        const T *b2 = MODE == BWD1 ? (const T *)a.b2 + (int64_t)e * O : nullptr;
        if (MODE == BWD1) clear(acc2);
        tile_loop<MODE == BWD1 ? 1 : 2, T, true, false>(K, lds, am, bn, MODE == BWD1 ? acc2 : acc,
            [&](int k0, u4 (&r)[4], int) {
#pragma unroll
                for (int i = 0; i < 4; ++i) { const int kk = k0 + SM::row(i); r[i] = cols_a.load(A + (int64_t)(kk < K ? kk : K - 1) * M); } },
            [&](int k0, u4 (&r)[4], int) { lb.load(k0, r); },
            [&](int k0, u4 (&r)[4], int) { cols_a.fix(r, K - k0, k0 + KB <= K); },
            [&](int k0, u4 (&r)[4], int) {
                lb.fix(k0, r);
                if (with_dot) {
                    float f[PER], g[PER];
#pragma unroll
                    for (int q = 0; q < PER; ++q) f[q] = to_f32(b2[k0 + c + q < K ? k0 + c + q : K - 1]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        to_floats<T>(r[i], g);
#pragma unroll
                        for (int q = 0; q < PER; ++q) dot[i] = fmaf(f[q], g[q], dot[i]);
                    }
                } });
    }

    // ---- epilogue.  The lane holds, for each of two rows, runs of four features; they leave through LDS
    typedef typename std::conditional<MODE == FWD1 || MODE == BWD1, T, float>::type OUT;
    const int cols = M - m0 < XN ? M - m0 : XN;
    __shared__ float red[3 * 128];                                  // BWD1: sums over the features of a half, b2 . dy
    if (MODE == BWD1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int m = 1; m < 8; m <<= 1) dot[i] += __shfl_xor(dot[i], m, 64);
            if (SC::chunk() == 0) red[256 + SC::row(i)] = dot[i];
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r = bn + 32 * j + (lane & 31);
        const float w = wr[j];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int mt_ = am + 32 * i + 8 * q + 4 * (lane >> 5), m = m0 + mt_;
                float u[4], g[4];
                f4 bv = {0.f, 0.f, 0.f, 0.f};
                if (MODE != BWD2) bv = *(const f4 *)(bias + mt_);
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    u[z] = acc[i][j][4 * q + z];
                    if (MODE == BWD1) g[z] = acc2[i][j][4 * q + z];
                    if (MODE != BWD2) u[z] += MODE == FWD2 ? w * bv[z] : bv[z];
                }
                if (MODE == FWD1) {
#pragma unroll
                    for (int z = 0; z < 4; ++z) u[z] = w * (u[z] * sigmoid_of<T>(u[z]));
                }
                if (MODE == BWD1) {
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float sg = sigmoid_of<T>(u[z]), hh = u[z] * sg;
                        if (m + z < M) sum = fmaf(hh, g[z], sum);
                        acc2[i][j][4 * q + z] = w * g[z] * (sg * (1.f + u[z] * (1.f - sg)));
                        u[z] = w * hh;
                    }
                }
                Spill<OUT>::put(lds, r, mt_, u);
            }
        if (MODE == BWD1 && m0 == 0 && am == 0 && lane < 32 && r < rows) a.ws[r0 + r] = w;
        if (MODE == BWD1) {
            sum += __shfl_xor(sum, 32, 64);
            if (lane < 32) red[(wave & 1) * 128 + r] = sum;
        }
    }
    __syncthreads();
    Spill<OUT>::write(lds, (MODE == FWD1 || MODE == BWD1 ? (OUT *)a.h : (OUT *)a.part) + (int64_t)r0 * M + m0, M, rows, cols);
    if (MODE == BWD1) {
        const int r = threadIdx.x;
        const int64_t P = a.n.rows * a.n.k;
        if (r < rows) a.dwp[(int64_t)(m0 / XN) * P + r0 + r] = red[r] + red[128 + r] + (m0 == 0 && a.b2 ? red[256 + r] : 0.f);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float g[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z) g[z] = acc2[i][j][4 * q + z];
                    Spill<OUT>::put(lds, bn + 32 * j + (lane & 31), am + 32 * i + 8 * q + 4 * (lane >> 5), g);
                }
        __syncthreads();
        Spill<OUT>::write(lds, (OUT *)a.du + (int64_t)r0 * M + m0, M, rows, cols);
    }
}

// joins the pairs of a row, in the order of its slots: out[t] = sum_j part[pos[t, j]]
template <typename T>
__global__ void __launch_bounds__(XT) k_join(const float *__restrict__ part, const int *__restrict__ pos, int64_t rows, int k, int M, T *__restrict__ out)
{
    const int per = (M + 3) / 4;
    const int64_t n = rows * per;
    for (int64_t i = (int64_t)blockIdx.x * XT + threadIdx.x; i < n; i += (int64_t)gridDim.x * XT) {
        const int64_t t = i / per;
        const int m = (int)(i - t * per) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int j = 0; j < k; ++j) {
            const int s = pos[t * k + j];
            if (s < 0) continue;
            const float *q = part + (int64_t)s * M + m;
            if (m + 4 <= M) {
                const Pack<float, 4> f = *(const Pack<float, 4> *)q;
#pragma unroll
                for (int z = 0; z < 4; ++z) v[z] += f.v[z];
            } else {
#pragma unroll
                for (int z = 0; z < 4; ++z) if (m + z < M) v[z] += q[z];
            }
        }
        T *o = out + t * M + m;
        if (m + 4 <= M) {
            Pack<T, 4> f;
#pragma unroll
            for (int z = 0; z < 4; ++z) f.v[z] = from_f32<T>(v[z]);
            *(Pack<T, 4> *)o = f;
        } else {
#pragma unroll
            for (int z = 0; z < 4; ++z) if (m + z < M) o[z] = from_f32<T>(v[z]);
        }
    }
}

__global__ void __launch_bounds__(XT) k_join_dw(const float *__restrict__ dwp, const int *__restrict__ pos, int64_t P, int parts, float *__restrict__ dw)
{
    for (int64_t i = (int64_t)blockIdx.x * XT + threadIdx.x; i < P; i += (int64_t)gridDim.x * XT) {
        const int s = pos[i];
        float v = 0.f;
        if (s >= 0) for (int q = 0; q < parts; ++q) v += dwp[(int64_t)q * P + s];
        dw[i] = v;
    }
}

// ------------------------------------------------------------------ launches (called by escat_experts.hip)
template <typename T, int MODE> static int rows_launch(const RowArgs &a, int M, hipStream_t st)
{
    const int64_t P = a.n.rows * a.n.k, wgs = plan_max_tiles(P, a.n.E) * ((M + XN - 1) / XN);
    if (wgs > 0xffffff) return fail(ESCAT_ERANGE, "experts: %lld tiles", (long long)wgs);
    const size_t lds = MODE == FWD2 || MODE == BWD2 || sizeof(T) == 4 ? LDS_ROWS : LDS_TILES;
    int rc = set_lds(k_expert_rows<T, MODE>, lds); if (rc) return rc;
    k_expert_rows<T, MODE><<<(unsigned)wgs, XT, lds, st>>>(a);
    CHECK_LAUNCH("experts: rows");
    return ESCAT_OK;
}

static unsigned grid_for(int64_t n) { const int64_t b = (n + XT - 1) / XT; return (unsigned)(b < 65536 ? b : 65536); }

template <typename T> static int join_launch(const float *part, const int *pos, int64_t rows, int k, int M, void *out, hipStream_t st)
{
    k_join<T><<<grid_for(rows * ((M + 3) / 4)), XT, 0, st>>>(part, pos, rows, k, M, (T *)out);
    CHECK_LAUNCH("experts: join");
    return ESCAT_OK;
}

template <typename T> static int fwd(const RowArgs &a, void *y, hipStream_t st)
{
    int rc = rows_launch<T, FWD1>(a, a.n.h, st); if (rc) return rc;
    rc = rows_launch<T, FWD2>(a, a.n.o, st); if (rc) return rc;
    return join_launch<T>(a.part, a.p.pos, a.n.rows, a.n.k, a.n.o, y, st);
}
template <typename T> static int bwd(const RowArgs &a, void *dx, float *dw, hipStream_t st)
{
    int rc = rows_launch<T, BWD1>(a, a.n.h, st); if (rc) return rc;
    const int64_t P = a.n.rows * a.n.k;
    if (dw) { k_join_dw<<<grid_for(P), XT, 0, st>>>(a.dwp, a.p.pos, P, (a.n.h + XN - 1) / XN, dw); CHECK_LAUNCH("experts: dw"); }
    if (!dx) return ESCAT_OK;
    rc = rows_launch<T, BWD2>(a, a.n.d, st); if (rc) return rc;
    return join_launch<T>(a.part, a.p.pos, a.n.rows, a.n.k, a.n.d, dx, st);
}

int escat_experts_rows_fwd(int type, const EDims &n, const EPlan &p, const void *x, const float *weights, const void *w1, const void *b1, const void *w2,
                           const void *b2, void *h, float *part, void *y, hipStream_t st)
{
    RowArgs a = {n, p, x, w1, b1, w2, b2, nullptr, weights, h, nullptr, part, nullptr, nullptr};
    return type == ESCAT_F32 ? fwd<float>(a, y, st) : type == ESCAT_BF16 ? fwd<bf16_t>(a, y, st) : fwd<f16_t>(a, y, st);
}
int escat_experts_rows_bwd(int type, const EDims &n, const EPlan &p, const void *x, const float *weights, const void *w1, const void *b1, const void *w2,
                           const void *b2, const void *dy, void *h, void *du, float *part, float *dwp, float *ws, void *dx, float *dw, hipStream_t st)
{
    RowArgs a = {n, p, x, w1, b1, w2, b2, dy, weights, h, du, part, dwp, ws};
    return type == ESCAT_F32 ? bwd<float>(a, dx, dw, st) : type == ESCAT_BF16 ? bwd<bf16_t>(a, dx, dw, st) : bwd<f16_t>(a, dx, dw, st);
}

