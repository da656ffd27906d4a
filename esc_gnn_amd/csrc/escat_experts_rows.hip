// escat_experts_rows.hip -- the experts' products over rows of activations, forward and backward:
//
//   pair (t, j), e = experts[t, j]:   u = W1_e x_t + b1_e    h = silu(u)    y_t = sum_j w_tj (W2_e h + b2_e)
//   G = W2_e^T dy_t    dw_tj = h.G + b2.dy_t    du = w G silu'(u)    dx_t = sum_j W1_e^T du
//
// Rows are taken in the plan's order (sorted by expert), 128 to a tile.  The weight w goes into the hidden row before it is
// rounded to the operands' type (w h): it then serves W2's product and W2's gradient without another pass.  The forward's (w h)
// may be kept for the weights' gradient.  dw and silu' see no rounding of u: it is computed again next to G in fp32, or, where
// that costs more than reading it, left in fp32 by the forward (keeps_u).  Results of the pairs are joined in fp32 by a pass of their own, in the order of the slots: no atomics.
//
// 524288 rows, k = 2 of 8 experts, 256 x 256 x 256 in bf16: 137 GFLOP a product, W1 x 276 us (0.86 GB), W2 h 230 us (0.91 GB), u, G and du 594 us
// (two products, 1.15 GB), W1^T du 221 us (0.82 GB; bytes by FETCH_SIZE, doubled, and WRITE_SIZE): neither the matrix units (a quarter of the cycles) nor memory bound; a workgroup's chain of
// tile, row, pieces and epilogue is, four steps of 64 long.  64 experts of 256 rows, 1024 x 2048 x 1024: 69 GFLOP a product (86 with the tiles' last
// rows) in 125 to 131 us, 38 % of the matrix cycles at about 1.75 GHz (W1 x 146 where it leaves u, G and du 176 with u read).  Tiles of 256 x 128 in
// eight waves, tiles in an order that shares weights, s_setprio around the products and leaving out the products of rows behind a tile's last each
// left these times as they are; zeros for data make them a tenth shorter.
#include <type_traits>
#include "escat_experts_tile.h"

struct RowArgs {
    EDims n;
    EPlan p;
    const void *x, *w1, *b1, *w2, *b2, *dy;
    const float *weights;
    void *h;                   // (P, H) by position: w silu(u); BWD1: NULL = kept by the forward, or not needed
    void *du;                  // (P, H) by position
    float *u;                  // (P, H) by position, fp32: FWD1 leaves it, BWD1U reads it
    float *part;               // by pair: (P, O) or (P, D) fp32, what the joining pass reads
    void *out;                 // by combination: y or dx
    float *dwp;                // (feature tiles of H, P) by position: parts of dw
    float *ws;                 // (P) by position: w (BWD1 leaves them for the weights' gradients)
};

enum { FWD1, FWD2, BWD1, BWD2, BWD1U };                            // BWD1U: BWD1 with u from memory
// Waves on a SIMD (workgroups of a CU) that the registers leave room for: BWD1 holds two sets of accumulators, BWD1U
// what it reads of u (with three it spills: 91 instead of 81 us in fp32, 209 instead of 177 in bf16).  Four instead of three for the
// forward's 16-bit products: 273 instead of 305 us and 230 instead of 244 (524288 rows, k = 2, 256 x 256).
template <typename T, int MODE> constexpr int waves_of() { return MODE == BWD1 || MODE == BWD1U ? 2 : MODE == BWD2 || sizeof(T) == 4 ? 3 : 4; }
// DIRECT: FWD2, BWD2: results by row; FWD1: leaves u; BWD1: writes no hidden rows

// the hardware's exponential errs by |u| 2^-24: below what 16-bit operands leave, not below what fp32 ones do
template <typename T> __device__ __forceinline__ float sigmoid_of(float u) { return __builtin_amdgcn_rcpf(1.f + (sizeof(T) == 4 ? expf(-u) : __expf(-u))); }

template <typename T, int MODE, bool DIRECT>
__global__ void __launch_bounds__(XT, (waves_of<T, MODE>())) k_expert_rows(const RowArgs a)
{
    constexpr int PER = Elem<T>::PER, KB = Elem<T>::KB;
    extern __shared__ __align__(16) char lds[];
    const int D = a.n.d, H = a.n.h, O = a.n.o;
    const int M = MODE == FWD2 ? O : MODE == BWD2 ? D : H;          // features of the result
    constexpr bool B1 = MODE == BWD1 || MODE == BWD1U;
    constexpr bool ONE = MODE == FWD1 || B1;                       // a tile's product with one of its experts, or with all
    const int mt = (M + XN - 1) / XN, per = a.p.per, of = ONE ? per * mt : mt;
    const int live = *a.p.n_tiles * of;                              // (the grid covers the most tiles there can be)
    if ((int)blockIdx.x >= live) return;
    const int work = xcd_swizzle(blockIdx.x, live), t = work / of, rest = work - t * of, dig = ONE ? rest / mt : 0, m0 = (rest - dig * mt) * XN;
    const int4 tile = *(const int4 *)(a.p.tile + 4 * t);
    const int key = tile.x, r0 = tile.y, rows = tile.z;
    const int e = key_digit(a.p, key, dig);
    if (ONE && e >= a.n.E) return;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, am = (wave & 1) * 64, bn = (wave >> 1) * 64;
    typedef Stage<T, false> SC;
    __shared__ __align__(16) float bias[XN], weight[XN];           // of the tile's features; of its rows
    acc_t acc[2][2], acc2[2][2];
    clear(acc);
    float dot[4] = {0.f, 0.f, 0.f, 0.f};                            // BWD1: the thread's share of b2 . dy of its rows

    if constexpr (ONE) {
        // ---- W1 x
        auto w1 = [&](int) { return (const char *)a.w1 + (int64_t)e * H * D * (int64_t)sizeof(T); };
        OperandKC<T, decltype(w1)> A(D, w1);
        OperandKCRows<T> B(D);
        const T *dy[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + SC::row(i) < M ? m0 + SC::row(i) : M - 1, r = SC::row(i) < rows ? SC::row(i) : rows - 1;
            const int64_t row = a.p.row[(int64_t)(r0 + r) * per + dig];
            A.off[i] = (uint32_t)m * (uint32_t)D * (uint32_t)sizeof(T);
            B.p[i] = (const T *)a.x + row * D;
            if (B1) dy[i] = (const T *)a.dy + row * O;
        }
        const int me = threadIdx.x % XN;
        const int pair = a.p.pair[(int64_t)(r0 + (me < rows ? me : 0)) * per + dig];
        Pipe<T, false, false, MODE == BWD1> pipe;
        const int steps_d = (D + KB - 1) / KB;
        if (MODE != BWD1U) pipe.start(steps_d, A, B);
        // what the epilogue needs waits in LDS
        const float w_me = a.weights[pair], b_me = a.b1 ? to_f32(((const T *)a.b1)[(int64_t)e * M + (m0 + me < M ? m0 + me : M - 1)]) : 0.f;
        if (threadIdx.x < XN) { weight[me] = w_me; bias[me] = b_me; }
        if constexpr (!B1) pipe.run(steps_d, lds, am, bn, acc, A, B);
        else {
            // ---- W2^T dy into the second set, and b2 . dy on the way (the first tile of features, for all)
            auto w2 = [&](int) { return (const char *)a.w2 + (int64_t)e * O * H * (int64_t)sizeof(T); };
            struct WithDot : OperandKCRows<T> {
                const T *b2;
                bool on;
                float (&dot)[4];
                u4 piece;
                __device__ __forceinline__ WithDot(int K, const T *b2, bool on, float (&dot)[4]) : OperandKCRows<T>(K), b2(b2), on(on), dot(dot) {}
                __device__ __forceinline__ void load(u4 (&r)[4])
                {
                    const int k0 = this->k0 + this->c, K = this->K;
                    piece = load16(b2 + (k0 < K - PER ? k0 : K - PER));
                    OperandKCRows<T>::load(r);
                }
                __device__ __forceinline__ void fix(u4 (&r)[4])
                {
                    if (on) {
                        u4 b[4] = {piece, piece, piece, piece};
                        int k0 = this->fk0;
                        fix_kc<T>(b, this->K, this->c, k0);
                        piece = b[0];
                    }
                    OperandKCRows<T>::fix(r);
                    if (!on) return;
                    float f[PER], g[PER];
                    to_floats<T>(piece, f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        to_floats<T>(r[i], g);
#pragma unroll
                        for (int q = 0; q < PER; ++q) dot[i] = fmaf(f[q], g[q], dot[i]);
                    }
                }
            };
            OperandKM<T, decltype(w2)> A2(O, m0, M, w2);
            const bool on = m0 == 0 && a.b2;
            WithDot B2(O, on ? (const T *)a.b2 + (int64_t)e * O : dy[0], on, dot);
#pragma unroll
            for (int i = 0; i < 4; ++i) B2.p[i] = dy[i];
            const int steps = (O + KB - 1) / KB;
            Pipe<T, true, false, true> pipe2;
            if constexpr (MODE == BWD1U) pipe2.start(steps, A2, B2);
            else pipe.run(steps_d, lds, am, bn, acc, A, B, [&]() { pipe2.start(steps, A2, B2); });
            clear(acc2);
            pipe2.run(steps, lds, am, bn, acc2, A2, B2);
        }
    } else {
        // ---- W2 (w h) or W1^T du of the tile's experts, one after the other into the same accumulators
        uint64_t live_at = 0; int n_live = 0;                             // the digits that name an expert, four bits each
        for (int j = per - 1; j >= 0; --j) if (key_digit(a.p, key, j) < a.n.E) { live_at = live_at << 4 | (unsigned)j; ++n_live; }
        auto weights = [&](int j) {
            const int dj = (int)(live_at >> 4 * j) & 15, q = j < n_live ? key_digit(a.p, key, dj) : 0;
            return (const char *)(MODE == FWD2 ? a.w2 : a.w1) + (int64_t)q * M * H * (int64_t)sizeof(T);
        };
        auto hidden = [&](int j) {
            const int dj = (int)(live_at >> 4 * j) & 15;
            return (const char *)(MODE == FWD2 ? a.h : a.du) + ((int64_t)r0 * per + dj) * H * (int64_t)sizeof(T);
        };
        OperandKC<T, decltype(hidden)> B(H, hidden);
#pragma unroll
        for (int i = 0; i < 4; ++i) B.off[i] = (uint32_t)((SC::row(i) < rows ? SC::row(i) : rows - 1) * per) * (uint32_t)H * (uint32_t)sizeof(T);
        const int steps = n_live * ((H + KB - 1) / KB);
        if constexpr (MODE == FWD2) {
            OperandKC<T, decltype(weights)> A(H, weights);
#pragma unroll
            for (int i = 0; i < 4; ++i) A.off[i] = (uint32_t)(m0 + SC::row(i) < M ? m0 + SC::row(i) : M - 1) * (uint32_t)H * (uint32_t)sizeof(T);
            Pipe<T, false, false> pipe;
            pipe.start(steps, A, B);
            pipe.run(steps, lds, am, bn, acc, A, B);
        } else {
            OperandKM<T, decltype(weights)> A(H, m0, M, weights);
            Pipe<T, true, false> pipe;
            pipe.start(steps, A, B);
            pipe.run(steps, lds, am, bn, acc, A, B);
        }
    }

    if (MODE == FWD2 && a.b2)                                       // + w b2 of each expert
        for (int j = 0; j < per; ++j) {
            const int ej = key_digit(a.p, key, j);
            if (ej >= a.n.E) continue;
            __syncthreads();
            if (threadIdx.x < XN) bias[threadIdx.x] = m0 + (int)threadIdx.x < M ? to_f32(((const T *)a.b2)[(int64_t)ej * M + m0 + threadIdx.x]) : 0.f;
            __syncthreads();
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                const int r = bn + 32 * jj + (lane & 31);
                const float w = a.weights[a.p.pair[(int64_t)(r0 + (r < rows ? r : 0)) * per + j]];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f4 bv = *(const f4 *)(bias + am + 32 * i + 8 * q + 4 * (lane >> 5));
#pragma unroll
                        for (int z = 0; z < 4; ++z) acc[i][jj][4 * q + z] = fmaf(w, bv[z], acc[i][jj][4 * q + z]);
                    }
            }
        }

    // ---- epilogue.  The lane holds, for each of two rows, runs of four features; they leave through LDS
    typedef typename std::conditional<ONE || DIRECT, T, float>::type OUT;
    const int cols = M - m0 < XN ? M - m0 : XN;
    __shared__ float red[3 * 128];                                  // BWD1: sums over the features of a half, b2 . dy
    if (B1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int m = 1; m < 8; m <<= 1) dot[i] += __shfl_xor(dot[i], m, 64);
            if (SC::chunk() == 0) red[256 + SC::row(i)] = dot[i];
        }
    }
    const int *row = a.p.row;
    auto by_pos = [&](int r) { return (int64_t)(r0 + r) * per + dig; };
    constexpr bool LEAVES_U = MODE == FWD1 && DIRECT;
    if constexpr (LEAVES_U) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f4 bv = *(const f4 *)(bias + am + 32 * i + 8 * q + 4 * (lane >> 5));
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int z = 0; z < 4; ++z) acc[i][j][4 * q + z] += bv[z];
            }
        Spill<float>::all(lds, acc, am, bn, a.u + m0, M, rows, cols, by_pos);
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r = bn + 32 * j + (lane & 31);
        const float w = ONE ? weight[r] : 0.f;
        const float *ur = MODE == BWD1U ? a.u + by_pos(r < rows ? r : rows - 1) * M + m0 : nullptr;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int mt_ = am + 32 * i + 8 * q + 4 * (lane >> 5);
                f4 bv = {0.f, 0.f, 0.f, 0.f};
                if (ONE && MODE != BWD1U && !LEAVES_U) bv = *(const f4 *)(bias + mt_);
                if constexpr (MODE == BWD1U) {
                    if (mt_ + 4 <= cols) bv = __builtin_bit_cast(f4, load16(ur + mt_));
                    else {
#pragma unroll
                        for (int z = 0; z < 4; ++z) if (mt_ + z < cols) bv[z] = ur[mt_ + z];
                    }
                }
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    float v = MODE == BWD1U ? bv[z] : acc[i][j][4 * q + z] + bv[z];
                    if (MODE == FWD1) v = w * (v * sigmoid_of<T>(v));
                    if (B1) {
                        const float g = acc2[i][j][4 * q + z];
                        const float sg = sigmoid_of<T>(v), hh = v * sg;
                        sum = fmaf(hh, g, sum);                     // (features behind the last: g = 0)
                        acc2[i][j][4 * q + z] = w * g * fmaf(hh, 1.f - sg, sg);          // silu' = sg (1 + v (1 - sg))
                        v = w * hh;
                    }
                    acc[i][j][4 * q + z] = v;
                }
            }
        }
        if (B1 && m0 == 0 && am == 0 && lane < 32 && r < rows) a.ws[(int64_t)(r0 + r) * per + dig] = w;
        if (B1) {
            sum += __shfl_xor(sum, 32, 64);
            if (lane < 32) red[(wave & 1) * 128 + r] = sum;
        }
    }
    if (B1 && DIRECT) { }                                 // the hidden rows are there already
    else if (ONE) Spill<OUT>::all(lds, acc, am, bn, (OUT *)a.h + m0, M, rows, cols, by_pos);
    else if (DIRECT) Spill<OUT>::all(lds, acc, am, bn, (OUT *)a.out + m0, M, rows, cols, [&](int r) { return row[(int64_t)(r0 + r) * per]; });
    else Spill<OUT>::all(lds, acc, am, bn, (OUT *)a.part + m0, M, rows, cols, [&](int r) { return r0 + r; });
    if (B1) {
        const int r = threadIdx.x;
        const int64_t P = a.n.rows * a.n.k;
        if (DIRECT) __syncthreads();
        if (r < rows) a.dwp[(int64_t)(m0 / XN) * P + by_pos(r)] = red[r] + red[128 + r] + (m0 == 0 && a.b2 ? red[256 + r] : 0.f);
        if (!DIRECT) __syncthreads();
        Spill<OUT>::all(lds, acc2, am, bn, (OUT *)a.du + m0, M, rows, cols, by_pos);
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
template <typename T, int MODE, bool DIRECT> static int rows_launch(const RowArgs &a, int M, hipStream_t st)
{
    constexpr bool ONE = MODE == FWD1 || MODE == BWD1 || MODE == BWD1U;
    const int64_t items = a.p.base ? a.n.rows : a.n.rows * a.n.k;
    const int64_t wgs = plan_max_tiles(items, a.p.keys) * ((M + XN - 1) / XN) * (ONE ? a.p.per : 1);
    if (wgs > 0xffffff) return fail(ESCAT_ERANGE, "experts: %lld tiles", (long long)wgs);
    constexpr size_t lds = LDS_BYTES;
    int rc = set_lds(k_expert_rows<T, MODE, DIRECT>, lds); if (rc) return rc;
    k_expert_rows<T, MODE, DIRECT><<<(unsigned)wgs, XT, lds, st>>>(a);
    CHECK_LAUNCH("experts: rows");
    return ESCAT_OK;
}

static unsigned grid_for(int64_t n) { const int64_t b = (n + XT - 1) / XT; return (unsigned)(b < 65536 ? b : 65536); }

// second product of a pass: results of M features to `out` by row
template <typename T, int MODE> static int second(RowArgs &a, int M, void *out, hipStream_t st)
{
    a.out = out;
    if (a.p.base) return rows_launch<T, MODE, true>(a, M, st);
    int rc = rows_launch<T, MODE, false>(a, M, st); if (rc) return rc;
    k_join<T><<<grid_for(a.n.rows * ((M + 3) / 4)), XT, 0, st>>>(a.part, a.p.pos, a.n.rows, a.n.k, M, (T *)out);
    CHECK_LAUNCH("experts: join");
    return ESCAT_OK;
}

template <typename T> static int fwd(RowArgs &a, void *y, hipStream_t st)
{
    int rc = a.u ? rows_launch<T, FWD1, true>(a, a.n.h, st) : rows_launch<T, FWD1, false>(a, a.n.h, st); if (rc) return rc;
    return second<T, FWD2>(a, a.n.o, y, st);
}
template <typename T> static int bwd(RowArgs &a, void *dx, float *dw, hipStream_t st)
{
    int rc = a.u ? rows_launch<T, BWD1U, true>(a, a.n.h, st) : a.h ? rows_launch<T, BWD1, false>(a, a.n.h, st) : rows_launch<T, BWD1, true>(a, a.n.h, st);
    if (rc) return rc;
    const int64_t P = a.n.rows * a.n.k;
    if (dw) { k_join_dw<<<grid_for(P), XT, 0, st>>>(a.dwp, a.p.pos, P, (a.n.h + XN - 1) / XN, dw); CHECK_LAUNCH("experts: dw"); }
    return dx ? second<T, BWD2>(a, a.n.d, dx, st) : ESCAT_OK;
}

int escat_experts_rows_fwd(int type, const EDims &n, const EPlan &p, const void *x, const float *weights, const void *w1, const void *b1, const void *w2,
                           const void *b2, void *h, float *u, float *part, void *y, hipStream_t st)
{
    RowArgs a = {n, p, x, w1, b1, w2, b2, nullptr, weights, h, nullptr, u, part, nullptr, nullptr, nullptr};
    return type == ESCAT_F32 ? fwd<float>(a, y, st) : type == ESCAT_BF16 ? fwd<bf16_t>(a, y, st) : fwd<f16_t>(a, y, st);
}
int escat_experts_rows_bwd(int type, const EDims &n, const EPlan &p, const void *x, const float *weights, const void *w1, const void *b1, const void *w2,
                           const void *b2, const void *dy, void *h, void *du, float *u, float *part, float *dwp, float *ws, void *dx, float *dw, hipStream_t st)
{
    RowArgs a = {n, p, x, w1, b1, w2, b2, dy, weights, h, du, u, part, nullptr, dwp, ws};
    return type == ESCAT_F32 ? bwd<float>(a, dx, dw, st) : type == ESCAT_BF16 ? bwd<bf16_t>(a, dx, dw, st) : bwd<f16_t>(a, dx, dw, st);
}
