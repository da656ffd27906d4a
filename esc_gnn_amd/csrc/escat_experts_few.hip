// escat_experts_few.hip -- the experts' forward for a few rows (one node, one small graph): matrix-vector products, one per pair.
//
//   h_p = w_p silu(W1_e x_t + b1_e) for every pair p = (t, j)          y_t = sum_j W2_e h_tj + w_tj b2_e
//
// A few rows are bound by the bytes of the weights that they touch, and by launches: no sorting, no tiles, two kernels.  A wave reads
// rows of weights, 16 bytes a lane, F of them at a time so that enough is in flight; products and sums are fp32, h stays fp32.  In the
// second product the hidden axis of all of a row's experts is split over the waves of a workgroup, which join in LDS: a row of 2048 for
// each of four experts would otherwise be 64 KB for one wave to walk alone.
#include "escat_experts_tile.h"

#define FT 256
#define FW (FT / 64)
#define OW 8                                      // waves that share a row's results
#define FEAT 4                                    // rows of weights (results) that a wave walks at once

struct FewArgs {
    EDims n;
    const int *experts;
    const void *x, *w1, *b1, *w2, *b2;
    const float *weights;
    float *h;                                     // (P, H)
    void *y;
};

template <typename T> __device__ __forceinline__ u4 piece_of(const T *row, int c, int K)          // elements c .. of a row, zeros behind K
{
    constexpr int PER = Elem<T>::PER;
    const int at = c < K - PER ? c : K - PER;
    return load16(row + at);
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(FT) k_few_hidden(const FewArgs a)
{
    constexpr int PER = Elem<T>::PER, CH = 64 * PER;
    const int D = a.n.d, H = a.n.h, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int p = blockIdx.y, f0 = (blockIdx.x * FW + wave) * FEAT;
    const int e = a.experts[p];
    if (e < 0 || e >= a.n.E || f0 >= H) return;
    const float w = a.weights[p];
    const T *x = (const T *)a.x + (int64_t)(p / a.n.k) * D, *W = (const T *)a.w1 + (int64_t)e * H * D;
    const T *row[FEAT];
    float s[FEAT], b[FEAT];
#pragma unroll
    for (int i = 0; i < FEAT; ++i) {
        const int f = f0 + i < H ? f0 + i : H - 1;
        row[i] = W + (int64_t)f * D;
        s[i] = 0.f;
        b[i] = a.b1 ? to_f32(((const T *)a.b1)[(int64_t)e * H + f]) : 0.f;
    }
    for (int c0 = lane * PER; c0 < D + lane * PER; c0 += 2 * CH) {           // (the same number of turns in every lane)
        u4 q[2][FEAT], v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            v[u] = piece_of(x, c0 + u * CH, D);
#pragma unroll
            for (int i = 0; i < FEAT; ++i) q[u][i] = piece_of(row[i], c0 + u * CH, D);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int c = c0 + u * CH, over = c > D - PER ? c - (D - PER) : 0;
            float fx[PER], fw[PER];
            to_floats<T>(moved<T>(v[u], over), fx);
#pragma unroll
            for (int i = 0; i < FEAT; ++i) {
                to_floats<T>(moved<T>(q[u][i], over), fw);
#pragma unroll
                for (int z = 0; z < PER; ++z) s[i] = fmaf(fx[z], fw[z], s[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < FEAT; ++i) {
        const float u = wave_sum(s[i]) + b[i];
        if (lane == i && f0 + i < H) a.h[(int64_t)p * H + f0 + i] = w * (u / (1.f + expf(-u)));
    }
}

template <typename T>
__global__ void __launch_bounds__(64 * OW) k_few_out(const FewArgs a)
{
    constexpr int PER = Elem<T>::PER, CH = 64 * PER;
    __shared__ float part[OW][FEAT];
    const int H = a.n.h, O = a.n.o, k = a.n.k, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.y, f0 = blockIdx.x * FEAT;
    const int chunks = (H + CH - 1) / CH, all = k * chunks;
    float s[FEAT];
#pragma unroll
    for (int i = 0; i < FEAT; ++i) s[i] = 0.f;
    for (int q0 = wave; q0 < all; q0 += 2 * OW) {            // two pieces of the (expert, hidden) axis in flight
        u4 v[2][FEAT], hv[2][PER / 4];
        bool live[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int q = q0 + u * OW < all ? q0 + u * OW : q0, j = q / chunks, c = (q - j * chunks) * CH + lane * PER;
            const int64_t p = (int64_t)t * k + j;
            const int e = a.experts[p];
            live[u] = q0 + u * OW < all && e >= 0 && e < a.n.E;
            if (!live[u]) continue;
            const T *W = (const T *)a.w2 + (int64_t)e * O * H;
            const int at = c < H - PER ? c : H - PER;
#pragma unroll
            for (int i = 0; i < FEAT; ++i) v[u][i] = load16(W + (int64_t)(f0 + i < O ? f0 + i : O - 1) * H + at);
#pragma unroll
            for (int i = 0; i < PER / 4; ++i) hv[u][i] = load16(a.h + p * H + at + 4 * i);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (!live[u]) continue;
            const int q = q0 + u * OW, c = (q % chunks) * CH + lane * PER, over = c > H - PER ? c - (H - PER) : 0;
            // weights and h were read from the same place: where that lies before c (the end of a row), the elements before c are left out
            float h[PER], fw[PER];
#pragma unroll
            for (int i = 0; i < PER / 4; ++i) {
                const f4 f = __builtin_bit_cast(f4, hv[u][i]);
#pragma unroll
                for (int z = 0; z < 4; ++z) h[4 * i + z] = 4 * i + z >= over ? f[z] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < FEAT; ++i) {
                to_floats<T>(v[u][i], fw);
#pragma unroll
                for (int z = 0; z < PER; ++z) s[i] = fmaf(h[z], z >= over ? fw[z] : 0.f, s[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < FEAT; ++i) { s[i] = wave_sum(s[i]); if (lane == 0) part[wave][i] = s[i]; }
    __syncthreads();
    if (threadIdx.x < FEAT && f0 + (int)threadIdx.x < O) {
        const int i = threadIdx.x;
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < OW; ++w) y += part[w][i];
        if (a.b2)
            for (int j = 0; j < k; ++j) {
                const int e = a.experts[(int64_t)t * k + j];
                if (e >= 0 && e < a.n.E) y = fmaf(a.weights[(int64_t)t * k + j], to_f32(((const T *)a.b2)[(int64_t)e * O + f0 + i]), y);
            }
        ((T *)a.y)[(int64_t)t * O + f0 + i] = from_f32<T>(y);
    }
}

template <typename T> static int go(const FewArgs &a, hipStream_t st)
{
    const EDims &n = a.n;
    k_few_hidden<T><<<dim3((n.h + FW * FEAT - 1) / (FW * FEAT), (unsigned)(n.rows * n.k)), FT, 0, st>>>(a);
    CHECK_LAUNCH("experts: few rows, hidden");
    k_few_out<T><<<dim3((n.o + FEAT - 1) / FEAT, (unsigned)n.rows), 64 * OW, 0, st>>>(a);
    CHECK_LAUNCH("experts: few rows, out");
    return ESCAT_OK;
}

// Taken where its estimate is below that of sorting and tiles, both in us: here every pair reads its expert's weights for itself (mostly from the
// caches, 10 TB/s) and sums its features; there the weights in use come from memory once, after a floor that the steps along a tile set.
// Forward, this form / tiles, us, k = 2, at 32, 128, 512, 2048 pairs:
//   bf16  64 wide, 8 experts 7/18  10/19  26/23  86/25      256, 8 10/22  25/23  83/28  306/30      1024, 16 28/46  83/48  318/53      2048, 64 99/145  330/268
//   fp32  64 wide, 8 experts 7/26  10/28  21/32  66/35      256, 8  9/53  21/54  65/58  245/61      1024, 16 37/158  104/160  399/165  2048, 64 177/524  586/1029
bool escat_experts_few(int type, const EDims &n)
{
    const double P = (double)n.rows * n.k, each = (double)n.h * (n.d + n.o) * escat_type_bytes(type);
    if (P > 4096) return false;
    const double here = 6 + P * (each * 1e-7 + (n.h + n.o) * 1.7e-4);
    const double tiles = 11 + (n.d + n.h) * (type == ESCAT_F32 ? 0.07 : 0.014) + (P < n.E ? P : n.E) * each * 2.2e-7;
    return here < tiles;
}

int escat_experts_few_fwd(int type, const EDims &n, const int *experts, const void *x, const float *weights, const void *w1, const void *b1, const void *w2,
                          const void *b2, float *h, void *y, hipStream_t st)
{
    const FewArgs a = {n, experts, x, w1, b1, w2, b2, weights, h, y};
    return type == ESCAT_F32 ? go<float>(a, st) : type == ESCAT_BF16 ? go<bf16_t>(a, st) : go<f16_t>(a, st);
}
