// escat_route.hip -- routing of rows (nodes) to experts, forward and backward: scores of E logits a row, k experts and weights.
//
//   s = softmax(l) or sigmoid(l)        key = s + bias  (no bias: the order of l, which is that of s)
//   group score = sum of the group's group_top largest keys; the keep best groups stay; top-k of key; ties to the lowest index
//   w_j = scale s_j / sum_chosen s  (softmax over the chosen logits; sigmoid: + 1e-20),  or scale s_j without renormalising
//   a logit or bias of -inf is never chosen; expert -1 with weight 0 where fewer than k can be; NaN counts as the largest
//
// A row belongs to LPR lanes of a wave with EPL consecutive experts each, all in registers: one read of the logits, no pass
// over memory for the selection.  k rounds of "largest key left": the lanes' maxima meet by DPP, the first lane that holds the
// maximum holds the lowest index.
//
// Which experts win is a matter of whole numbers, and s + bias in 32 bits would decide near-equal keys by the rounding of an
// exponential.  64-bit exponentials for every logit cost more than the memory traffic (E = 256: ~26 us of issue against 14 us), so
// keys are computed in 32 bits with a bound on their error, and a wave in which two keys that decide something lie within that
// bound repeats the selection with 64-bit keys (about one wave in 500 at E = 256, k = 8).
//
// 65537 rows of 256 bf16 logits, k = 8, bias and 4 of 8 groups: 71 us forward (34 MB read: 7 us; what bounds it is the instructions of the
// selection, 1200 for the two rows of a wave), 17 us backward.  524288 rows of 8 fp32 logits, k = 2: 12 us forward (25 MB, 2.1 TB/s), 9 us backward.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "escat_dev.h"
#include "escat_half.h"

#define RT 256
#define R_INF __builtin_inff()
// two 32-bit keys further apart than this (times max(1, size)) are in the order of their exact values: exp and the sum of up to
// 1024 of them err by at most 1e-6 of s <= 1, the sum with the bias by 2^-24 of its size; a place in a lane takes the last 3 bits of a key
// (E > 512: 4), 1e-6 (1.9e-6) of its size.  A group score adds two keys, whose biases may cancel: its size is that of its terms, at most
// B = max(1, the largest |bias|): 4 2^-24 (1 + B) + 2e-6 off, two of them 9e-7 + 4e-6 B at most
#define R_GAP 7.62939453125e-6f

struct RouteArgs {
    const void *logits; const float *bias; float *weights; int *experts;
    int64_t rows; int E, k, groups, keep, group_top, score, renorm; float scale;
};

// ------------------------------------------------------------------ reductions over the LPR lanes of a row
template <int CTRL> __device__ __forceinline__ float dpp(float v) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)); }
template <int CTRL> __device__ __forceinline__ double dpp(double v)
{
    const int lo = __builtin_amdgcn_mov_dpp(__double2loint(v), CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_mov_dpp(__double2hiint(v), CTRL, 0xf, 0xf, true);
    return __hiloint2double(hi, lo);
}
// all lanes of a pair of 16-lane rows (of both halves of the wave) get the first (SIDE 0) or the second (SIDE 1) one's value
template <int SIDE> __device__ __forceinline__ unsigned swap_row_u(unsigned v) { return __builtin_amdgcn_permlane16_swap(v, v, false, false)[SIDE]; }
template <int SIDE> __device__ __forceinline__ unsigned swap_half_u(unsigned v) { return __builtin_amdgcn_permlane32_swap(v, v, false, false)[SIDE]; }
template <int SIDE> __device__ __forceinline__ float swap_row(float v) { return __uint_as_float(swap_row_u<SIDE>(__float_as_uint(v))); }
template <int SIDE> __device__ __forceinline__ float swap_half(float v) { return __uint_as_float(swap_half_u<SIDE>(__float_as_uint(v))); }
template <int SIDE> __device__ __forceinline__ double swap_row(double v)
{
    return __hiloint2double((int)swap_row_u<SIDE>((unsigned)__double2hiint(v)), (int)swap_row_u<SIDE>((unsigned)__double2loint(v)));
}
template <int SIDE> __device__ __forceinline__ double swap_half(double v)
{
    return __hiloint2double((int)swap_half_u<SIDE>((unsigned)__double2hiint(v)), (int)swap_half_u<SIDE>((unsigned)__double2loint(v)));
}
template <int SIDE> __device__ __forceinline__ int swap_row(int v) { return (int)swap_row_u<SIDE>((unsigned)v); }
template <int SIDE> __device__ __forceinline__ int swap_half(int v) { return (int)swap_half_u<SIDE>((unsigned)v); }
template <int CTRL> __device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, true); }

// 32-bit keys are compared as whole numbers in the same order (one instruction a maximum, which DPP moves fold into)
__device__ __forceinline__ int sortable(float f) { const int b = __float_as_int(f); return b ^ ((b >> 31) & 0x7fffffff); }
__device__ __forceinline__ float value_of(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }
__device__ __forceinline__ double value_of(double k) { return k; }
template <typename K> struct Least;
template <> struct Least<int> { static constexpr int v = (int)0x807fffff; };                 // sortable(-inf)
template <> struct Least<double> { static constexpr double v = -__builtin_inf(); };
__device__ __forceinline__ void to_key(float f, int &k) { k = sortable(f); }
__device__ __forceinline__ void to_key(double f, double &k) { k = f; }
struct OpMax {
    template <typename K> __device__ static K f(K a, K b) { return a > b ? a : b; }
    __device__ static float f(float a, float b) { return fmaxf(a, b); }
};
struct OpSum { template <typename K> __device__ static K f(K a, K b) { return a + b; } };
template <int LPR, typename OP, typename K> __device__ __forceinline__ K row_reduce(K v)
{
    if (LPR > 1) v = OP::f(v, dpp<0xB1>(v));                // quad_perm 1,0,3,2
    if (LPR > 2) v = OP::f(v, dpp<0x4E>(v));                // quad_perm 2,3,0,1
    if (LPR > 4) v = OP::f(v, dpp<0x141>(v));               // row_half_mirror: the other four of eight
    if (LPR > 8) v = OP::f(v, dpp<0x140>(v));               // row_mirror: the other eight of sixteen
    if (LPR > 16) v = OP::f(swap_row<0>(v), swap_row<1>(v));
    if (LPR > 32) v = OP::f(swap_half<0>(v), swap_half<1>(v));
    return v;
}
// first of the row's lanes for which `has` holds (one does), counted in the row
template <int LPR> __device__ __forceinline__ int first_lane(bool has, int l0)
{
    if (LPR == 1) return 0;
    const uint64_t b = __ballot(has);
    if (LPR == 64) return __builtin_ctzll(b);
    const uint32_t half = l0 & 32 ? (uint32_t)(b >> 32) : (uint32_t)b;       // (lanes of later rows lie above the one that is found)
    return __builtin_ctz(LPR == 32 ? half : half >> (l0 & 31));
}

// lanes of one wave hand values over through LDS: order the accesses, no barrier between waves
__device__ __forceinline__ void wave_lds_sync() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier(); }

// ------------------------------------------------------------------ the selection
// key / gkey: the lane's EPL keys for experts and for group scores (Least: cannot be chosen), K = int (sortable) or double, V the
// type of their values.  sel (LDS, of the row): k results.  Returns whether two keys that decided something were closer than
// their error (CHECK only; terms: the size of what a group score adds, at least 1).
template <typename V> __device__ __forceinline__ bool too_close(V last, V now, float size = 1.f) { return !(last - now > (V)R_GAP * fmaxf(size, fabsf((float)last))); }

template <int LPR, typename K> __device__ __forceinline__ K other_lane(K v, int m)       // lane ^ m, m < LPR, inside a group of whole lanes
{
    if (m == 1) return dpp<0xB1>(v);
    if (m == 2) return dpp<0x4E>(v);
    return (K)__shfl_xor(v, m, 64);
}

// largest first (a merge-exchange network: 19 exchanges of 8)
template <int N> __device__ __forceinline__ void sort_down(int (&k)[N])
{
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const int a = k[i + j], b = k[i + j + q];
                        k[i + j] = a > b ? a : b;
                        k[i + j + q] = a > b ? b : a;
                    }
}

// The rounds where close keys are decided again anyway and a row has 16 lanes or more: the place in the lane goes into the key's last bits (2^-20
// of it: R_GAP leaves room), the lane's keys are sorted once, and a round looks at their heads alone.  Lane j keeps the j-th result.
template <int LPR, int EPL>
__device__ __forceinline__ bool pick_sorted(const RouteArgs &a, int (&key)[EPL], int lane_in_row, int l0, int *sel)
{
    constexpr int least = Least<int>::v;
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = key[i] > least ? (key[i] & -EPL) | (EPL - 1 - i) : least;
    sort_down(key);
    int my_key = least, my = -1, m = least;
    for (int j = 0; j < a.k; ++j) {
        m = row_reduce<LPR, OpMax>(key[0]);
        const int at = first_lane<LPR>(key[0] == m, l0);
        const int e = m > least ? at * EPL + (~m & (EPL - 1)) : -1;
        if (lane_in_row == j) { my_key = m; my = e; }
        const bool mine = lane_in_row == at;
#pragma unroll
        for (int i = 0; i < EPL; ++i) key[i] = mine ? (i + 1 < EPL ? key[i + 1] : least) : key[i];
    }
    if (lane_in_row < a.k) sel[lane_in_row] = my;
    // each result against the one before it, and the first that was left against the last
    const int before = __shfl_up(my_key, 1, 64), left = row_reduce<LPR, OpMax>(key[0]);
    const bool pair = lane_in_row > 0 && lane_in_row < a.k && my_key > least;
    bool close = pair && too_close(value_of(before), value_of(my_key));
    close |= left > least && too_close(value_of(m), value_of(left));
    return close;
}

template <int LPR, int EPL, typename K, typename V, bool CHECK>
__device__ bool pick(const RouteArgs &a, K (&key)[EPL], const K (&gkey)[EPL], bool key_exact, float terms, int lane_in_row, int l0, V *buf, int *sel)
{
    constexpr K least = Least<K>::v;
    const V inf = (V)R_INF;
    const int e0 = lane_in_row * EPL;
    bool close = false;
    if (a.groups > 1) {
        const int gs = a.E / a.groups, lpg = gs / EPL;
        if (lpg * EPL == gs && (lpg & (lpg - 1)) == 0) {      // a group is a power of two of whole lanes: all in registers
            K b1 = gkey[0], b2 = least;                        // the lane's two largest, then the group's
#pragma unroll
            for (int i = 1; i < EPL; ++i) { const K v = gkey[i], lo = v < b1 ? v : b1; b1 = v > b1 ? v : b1; b2 = lo > b2 ? lo : b2; }
            for (int m = 1; m < lpg; m <<= 1) {
                const K o1 = other_lane<LPR>(b1, m), o2 = other_lane<LPR>(b2, m), lo = o1 < b1 ? o1 : b1;
                b1 = o1 > b1 ? o1 : b1;
                b2 = o2 > b2 ? o2 : b2; b2 = lo > b2 ? lo : b2;
            }
            V sum = -inf;
            if (e0 < a.E && b1 > least) sum = (V)value_of(b1) + (a.group_top == 2 && b2 > least ? (V)value_of(b2) : (V)0);
            K score; to_key(sum, score);
            int ahead = 0;                                   // groups that come before the lane's
            const int mine = lane_in_row / lpg;
            for (int g = 0; g < a.groups; ++g) {
                const K o = __shfl(score, l0 + g * lpg, 64);
                ahead += o > score || (o == score && g < mine);
            }
            const bool kept = ahead < a.keep && score > least;
            if constexpr (CHECK) {                           // the least that stays against the largest that goes (~ turns the order round)
                const int stays = ~row_reduce<LPR, OpMax>(kept ? ~score : least), goes = row_reduce<LPR, OpMax>(kept ? least : score);
                close |= goes > least && too_close(value_of(stays), value_of(goes), terms);
            }
#pragma unroll
            for (int i = 0; i < EPL; ++i) if (!kept) key[i] = least;
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i) if (e0 + i < a.E) buf[e0 + i] = (V)value_of(gkey[i]);
            wave_lds_sync();
            V sum = -inf;
            if (lane_in_row < a.groups) {                    // one group a lane (LPR >= groups)
                V b1 = -inf, b2 = -inf;
                int at = lane_in_row % gs;                   // start at another place in each lane: other LDS banks
                for (int i = 0; i < gs; ++i) {
                    const V v = buf[lane_in_row * gs + at];
                    at = at + 1 == gs ? 0 : at + 1;
                    if (v > b1) { b2 = b1; b1 = v; } else if (v > b2) b2 = v;
                }
                sum = b1 == -inf ? -inf : b1 + (a.group_top == 2 && b2 > -inf ? b2 : (V)0);
            }
            wave_lds_sync();
            K score; to_key(sum, score);
            uint64_t kept = 0;
            V last = inf;
            for (int r = 0; r <= a.keep; ++r) {
                const K m = row_reduce<LPR, OpMax>(score);
                const V mv = (V)value_of(m);
                if (CHECK && r > 0 && m > least) close |= too_close(last, mv, terms);
                if (r == a.keep || m == least) break;
                const int at = first_lane<LPR>(score == m, l0);
                kept |= 1ull << at;
                if (lane_in_row == at) score = least;
                last = mv;
            }
            int g = e0 / gs, in_g = e0 - g * gs;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                if (e0 + i >= a.E || !((kept >> g) & 1)) key[i] = least;
                if (++in_g == gs) { in_g = 0; ++g; }
            }
        }
    }
    if constexpr (CHECK && LPR >= 16) { if (!key_exact) return pick_sorted<LPR, EPL>(a, key, lane_in_row, l0, sel) || close; }
    // k rounds (one more to see how far behind the next one is); no round ends early: rows of a wave would part ways
    const bool check = CHECK && !key_exact;
    V last = inf;
    for (int j = 0; ; ++j) {
        K best = key[0];
#pragma unroll
        for (int i = 1; i < EPL; ++i) best = key[i] > best ? key[i] : best;
        const K m = row_reduce<LPR, OpMax>(best);
        const bool some = m > least;
        if (check) {
            const V mv = (V)value_of(m);
            close |= j > 0 && some && too_close(last, mv);
            last = mv;
        }
        if (j == a.k) break;
        const int at = first_lane<LPR>(best == m, l0);
        const bool mine = lane_in_row == at;
        int w = EPL - 1;
#pragma unroll
        for (int i = EPL - 2; i >= 0; --i) w = key[i] == m ? i : w;
        if (mine) sel[j] = some ? e0 + w : -1;
        w = mine ? w : -1;
#pragma unroll
        for (int i = 0; i < EPL; ++i) key[i] = i == w ? least : key[i];
        if (!check && j + 1 == a.k) break;
    }
    return close;
}

__device__ __forceinline__ float sigmoid_f(float x) { return 1.f / (1.f + expf(-x)); }

// key of a score that is NaN: largest where the logit itself is the cause (NaN, or +inf under a softmax), next to it in the
// rest of such a row; a bias of -inf masks here too (its sum with a NaN does not)
__device__ __forceinline__ float spoiled(float x, float bias, float next) { return bias == -R_INF ? -R_INF : x == x && x < R_INF ? next : R_INF; }

template <typename T, int LPR, int EPL>
__global__ void __launch_bounds__(RT) k_route(const RouteArgs a)
{
    extern __shared__ __align__(8) unsigned char lds[];
    constexpr int RPB = RT / LPR;
    const int lane = threadIdx.x & 63; const int lane_in_row = threadIdx.x % LPR, l0 = lane - lane % LPR, r_in_b = threadIdx.x / LPR;
    const int e0 = lane_in_row * EPL;
    int *sel = (int *)lds + r_in_b * a.k;
    double *buf = (double *)(lds + (size_t)RPB * a.k * 8) + (size_t)r_in_b * a.E;      // groups only
    const bool fp64_keys = a.bias != nullptr || a.groups > 1;
    float bias[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) bias[i] = a.bias && e0 + i < a.E ? a.bias[e0 + i] : 0.f;
    float terms = 1.f;
    if (a.bias && a.groups > 1) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) terms = fabsf(bias[i]) < R_INF ? fmaxf(terms, fabsf(bias[i])) : terms;
        terms = row_reduce<LPR, OpMax>(terms);
    }
    // all lanes of a wave go through the same number of rows: rows behind the last are worked on as rows without an expert
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t row = r0 + r_in_b;
        const bool in = row < a.rows;
        const T *lg = (const T *)a.logits + (in ? row : 0) * a.E;
        float x[EPL];
        int key[EPL];
        if (in && e0 + EPL <= a.E) {
            const Pack<T, EPL> q = *(const Pack<T, EPL> *)(lg + e0);
#pragma unroll
            for (int i = 0; i < EPL; ++i) x[i] = to_f32(q.v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i) x[i] = in && e0 + i < a.E ? to_f32(lg[e0 + i]) : -R_INF;
        }
        float top = -R_INF, sum = 0.f;                        // softmax's statistics over the whole row
        if (a.score == 0 && (fp64_keys || !a.renorm)) {
#pragma unroll
            for (int i = 0; i < EPL; ++i) top = fmaxf(top, x[i]);           // (a NaN shows in the sum)
            top = row_reduce<LPR, OpMax>(top);
            const float base = top == -R_INF ? 0.f : top;
#pragma unroll
            for (int i = 0; i < EPL; ++i) sum += expf(x[i] - base);
            sum = row_reduce<LPR, OpSum>(sum);
            top = base;
        }
        bool again = false;
        if (!fp64_keys) {
#pragma unroll
            for (int i = 0; i < EPL; ++i) key[i] = sortable(x[i] == x[i] ? x[i] : R_INF);
            pick<LPR, EPL, int, float, false>(a, key, key, true, 1.f, lane_in_row, l0, (float *)buf, sel);
        } else {
            int gkey[EPL];
            float sc[EPL];
            bool nan = false;
            // (the form of the scores is asked for outside the loops over a lane's experts: inside it is a branch for each)
            if (a.score == 0) {
                const float inv = 1.f / sum;
#pragma unroll
                for (int i = 0; i < EPL; ++i) sc[i] = __expf(x[i] - top) * inv;
            } else {
#pragma unroll
                for (int i = 0; i < EPL; ++i) sc[i] = __builtin_amdgcn_rcpf(1.f + __expf(-x[i]));
            }
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                sc[i] += bias[i];
                nan |= sc[i] != sc[i];
                gkey[i] = sortable(x[i] == -R_INF ? -R_INF : sc[i]);
            }
            if (__any(nan)) {                                    // (rare: not a select for every logit)
#pragma unroll
                for (int i = 0; i < EPL; ++i) if (x[i] != -R_INF && sc[i] != sc[i]) gkey[i] = sortable(spoiled(x[i], bias[i], 3.4e38f));
            }
            if (a.bias) {
#pragma unroll
                for (int i = 0; i < EPL; ++i) key[i] = gkey[i];
            } else {
#pragma unroll
                for (int i = 0; i < EPL; ++i) key[i] = sortable(x[i] == x[i] ? x[i] : R_INF);
            }
            again = pick<LPR, EPL, int, float, true>(a, key, gkey, !a.bias, terms, lane_in_row, l0, (float *)buf, sel);
        }
        if (__any(again)) {
            double key2[EPL], gkey2[EPL];
            if (a.score == 0) {
                double top2 = -(double)R_INF, sum2 = 0.0;
#pragma unroll
                for (int i = 0; i < EPL; ++i) top2 = fmax(top2, (double)x[i]);
                top2 = row_reduce<LPR, OpMax>(top2);
                top2 = top2 == -(double)R_INF ? 0.0 : top2;
#pragma unroll
                for (int i = 0; i < EPL; ++i) { gkey2[i] = exp((double)x[i] - top2); sum2 += gkey2[i]; }
                sum2 = row_reduce<LPR, OpSum>(sum2);
#pragma unroll
                for (int i = 0; i < EPL; ++i) gkey2[i] /= sum2;
            } else {
#pragma unroll
                for (int i = 0; i < EPL; ++i) gkey2[i] = 1.0 / (1.0 + exp(-(double)x[i]));
            }
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                const double v = gkey2[i] + (double)bias[i];
                gkey2[i] = x[i] == -R_INF ? -(double)R_INF : v == v ? v : (double)spoiled(x[i], bias[i], 3.4e38f);
                key2[i] = a.bias ? gkey2[i] : x[i] == x[i] ? (double)x[i] : (double)R_INF;
            }
            pick<LPR, EPL, double, double, false>(a, key2, gkey2, true, 1.f, lane_in_row, l0, buf, sel);
        }
        wave_lds_sync();
        // weights: the chosen logits once more (they are in the cache), spread over the row's lanes; s_j waits in LDS next to sel
        float m = -R_INF, z = 0.f;
        if (a.score == 0 && a.renorm) {
            for (int j = lane_in_row; j < a.k; j += LPR) { const int e = sel[j]; if (in && e >= 0) { const float v = to_f32(lg[e]); m = v > m ? v : m; } }
            m = row_reduce<LPR, OpMax>(m);
        } else m = top;
        float *sj = (float *)(sel + RPB * a.k);
        for (int j = lane_in_row; j < a.k; j += LPR) {
            const int e = sel[j];
            const float v = in && e >= 0 ? to_f32(lg[e]) : 0.f;
            const float q = e < 0 ? 0.f : a.score == 0 ? expf(v - m) : sigmoid_f(v);
            sj[j] = q;
            z += q;
        }
        if (a.renorm) {
            z = row_reduce<LPR, OpSum>(z);
            z = a.score == 0 ? z : z + 1e-20f;
        } else z = a.score == 0 ? sum : 1.f;
        if (in)
            for (int j = lane_in_row; j < a.k; j += LPR) {
                const int e = sel[j];
                a.weights[row * a.k + j] = e < 0 ? 0.f : a.scale * (sj[j] / z);
                a.experts[row * a.k + j] = e;
            }
        wave_lds_sync();
    }
}

// ------------------------------------------------------------------ backward
// dl from dw: renormalised softmax  dl_j = w_j (dw_j - sum_i w_i dw_i / scale);  softmax  dl_e = scale s_e ([e chosen] dw_e - sum_j s_j dw_j);
// sigmoid  dl_j = ds_j s_j (1 - s_j) with ds = scale dw, or scale (dw_j / Z - sum_i dw_i s_i / Z^2).  The whole row of dl is written once.
struct RouteBwdArgs {
    const void *logits; const float *weights; const int *experts; const float *dw; void *dl;
    int64_t rows; int E, k, score, renorm; float scale;
};

template <typename T, int LPR, int EPL>
__global__ void __launch_bounds__(RT) k_route_bwd(const RouteBwdArgs a)
{
    constexpr int RPB = RT / LPR;
    __shared__ __align__(16) float at_expert[RPB * LPR * EPL];             // the chosen experts' gradients find their places here
    const int lane_in_row = threadIdx.x % LPR, r_in_b = threadIdx.x / LPR, e0 = lane_in_row * EPL;
    float *mine = at_expert + (size_t)threadIdx.x * EPL, *row_of = at_expert + (size_t)r_in_b * LPR * EPL;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t row = r0 + r_in_b;
        const bool in = row < a.rows;
        const int64_t rr = in ? row : 0;
        const T *lg = (const T *)a.logits + rr * a.E;
        const float *dw = a.dw + rr * a.k, *w = a.weights + rr * a.k;
        const int *ex = a.experts + rr * a.k;
        float s[EPL], z = 1.f, dot = 0.f;
        const bool all = a.score == 0 && !a.renorm;           // every expert's logit has a gradient
        if (all) {
            float top = -R_INF, sum = 0.f;
#pragma unroll
            for (int i = 0; i < EPL; ++i) { s[i] = in && e0 + i < a.E ? to_f32(lg[e0 + i]) : -R_INF; top = fmaxf(top, s[i]); }
            top = row_reduce<LPR, OpMax>(top);
            top = top == -R_INF ? 0.f : top;
#pragma unroll
            for (int i = 0; i < EPL; ++i) { s[i] = expf(s[i] - top); sum += s[i]; }
            sum = row_reduce<LPR, OpSum>(sum);
            sum = sum == 0.f ? 1.f : sum;                        // no logit above -inf: nothing was chosen
#pragma unroll
            for (int i = 0; i < EPL; ++i) s[i] /= sum;
            for (int j = lane_in_row; j < a.k; j += LPR) if (in && ex[j] >= 0) dot += w[j] * dw[j];
            dot = row_reduce<LPR, OpSum>(dot);                   // = scale sum_j s_j dw_j
        } else if (a.renorm) {
            float zz = 0.f;
            for (int j = lane_in_row; j < a.k; j += LPR)
                if (in && ex[j] >= 0) {
                    const float p = a.score == 0 ? w[j] : sigmoid_f(to_f32(lg[ex[j]]));
                    dot += p * dw[j];
                    zz += p;
                }
            dot = row_reduce<LPR, OpSum>(dot);
            if (a.score == 1) { z = row_reduce<LPR, OpSum>(zz) + 1e-20f; dot /= z; } else dot /= a.scale;
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i) mine[i] = all ? -s[i] * dot : 0.f;
        wave_lds_sync();
        for (int j = lane_in_row; j < a.k; j += LPR) {            // no expert is chosen twice
            const int e = in ? ex[j] : -1;
            if (e < 0) continue;
            float v;
            if (a.score == 0) v = a.renorm ? w[j] * (dw[j] - dot) : w[j] * dw[j];
            else {
                const float q = sigmoid_f(to_f32(lg[e]));
                v = a.scale * q * (1.f - q) * (a.renorm ? (dw[j] - dot) / z : dw[j]);
            }
            row_of[e] += v;
        }
        wave_lds_sync();
        T *out = (T *)a.dl + rr * a.E;
        if (in && e0 + EPL <= a.E) {
            Pack<T, EPL> q;
#pragma unroll
            for (int i = 0; i < EPL; ++i) q.v[i] = from_f32<T>(mine[i]);
            *(Pack<T, EPL> *)(out + e0) = q;
        } else if (in) {
#pragma unroll
            for (int i = 0; i < EPL; ++i) if (e0 + i < a.E) out[e0 + i] = from_f32<T>(mine[i]);
        }
        wave_lds_sync();
    }
}

// ------------------------------------------------------------------ entry points
// lanes of a row: enough for E experts at EPL each, and one a group
static int lanes_per_row(int E, int epl, int groups)
{
    int l = 1;
    while (l * epl < E || l < groups) l *= 2;
    return l;
}

template <template <typename, int, int> class L, typename A> static int route_dispatch(int type, int lpr, int epl, const A &a, unsigned blocks, size_t lds, hipStream_t st)
{
#define ROUTE_CASE(LPR, EPL)                                                                 \
    if (lpr == LPR && epl == EPL) {                                                          \
        if (type == ESCAT_F32) return L<float, LPR, EPL>::go(a, blocks, lds, st);            \
        if (type == ESCAT_BF16) return L<bf16_t, LPR, EPL>::go(a, blocks, lds, st);          \
        return L<f16_t, LPR, EPL>::go(a, blocks, lds, st);                                   \
    }
    ROUTE_CASE(1, 8) ROUTE_CASE(2, 8) ROUTE_CASE(4, 8) ROUTE_CASE(8, 8) ROUTE_CASE(16, 8) ROUTE_CASE(32, 8) ROUTE_CASE(64, 8) ROUTE_CASE(64, 16)
#undef ROUTE_CASE
    return fail(ESCAT_ERANGE, "route: %d lanes of %d experts", lpr, epl);
}
template <typename T, int LPR, int EPL> struct LaunchFwd {
    static int go(const RouteArgs &a, unsigned blocks, size_t lds, hipStream_t st)
    {
        int rc = set_lds(k_route<T, LPR, EPL>, lds); if (rc) return rc;
        k_route<T, LPR, EPL><<<blocks, RT, lds, st>>>(a);
        CHECK_LAUNCH("escat_route");
        return ESCAT_OK;
    }
};
template <typename T, int LPR, int EPL> struct LaunchBwd {
    static int go(const RouteBwdArgs &a, unsigned blocks, size_t, hipStream_t st)
    {
        k_route_bwd<T, LPR, EPL><<<blocks, RT, 0, st>>>(a);
        CHECK_LAUNCH("escat_route_bwd");
        return ESCAT_OK;
    }
};

static int check_route(const char *who, int type, int64_t rows, int E, int k, int score, float scale)
{
    if (!escat_type_bytes(type)) return fail(ESCAT_EINVAL, "%s: type = %d", who, type);
    if (rows < 0 || E < 1 || k < 1 || k > E) return fail(ESCAT_EINVAL, "%s: rows = %lld, E = %d, k = %d", who, (long long)rows, E, k);
    if (E > ESCAT_ROUTE_MAX_EXPERTS || k > ESCAT_ROUTE_MAX_K) return fail(ESCAT_ERANGE, "%s: E = %d (at most %d), k = %d (at most %d)", who, E, ESCAT_ROUTE_MAX_EXPERTS, k, ESCAT_ROUTE_MAX_K);
    if (score != 0 && score != 1) return fail(ESCAT_EINVAL, "%s: score = %d (0 softmax, 1 sigmoid)", who, score);
    if (!(scale > 0.f) || scale == R_INF) return fail(ESCAT_EINVAL, "%s: scale = %g", who, (double)scale);
    return ESCAT_OK;
}

extern "C" int escat_route(const void *logits, int type, int64_t rows, int E, int k, int score, const float *bias, int groups, int keep_groups,
                           int group_top, int renorm, float scale, float *weights, int32_t *experts, void *stream)
{
    int rc = check_route("escat_route", type, rows, E, k, score, scale); if (rc) return rc;
    if (groups < 1 || groups > 64 || E % groups || keep_groups < 1 || keep_groups > groups || (group_top != 1 && group_top != 2))
        return fail(ESCAT_EINVAL, "escat_route: groups = %d (1..64, dividing E = %d), keep_groups = %d, group_top = %d (1 or 2)", groups, E, keep_groups, group_top);
    if (rows == 0) return ESCAT_OK;
    if (!logits || !weights || !experts) return fail(ESCAT_EINVAL, "escat_route: null pointer");
    if (keep_groups == groups) groups = keep_groups = 1;             // every group stays: no groups
    const int epl = E > 512 ? 16 : 8, lpr = lanes_per_row(E, epl, groups), rpb = RT / lpr;
    const size_t lds = (size_t)rpb * k * 8 + (groups > 1 ? (size_t)rpb * E * 8 : 0);
    const int64_t want = (rows + rpb - 1) / rpb;
    const RouteArgs a = {logits, bias, weights, experts, rows, E, k, groups, keep_groups, group_top, score, renorm ? 1 : 0, scale};
    return route_dispatch<LaunchFwd>(type, lpr, epl, a, (unsigned)(want < 2048 ? want : 2048), lds, (hipStream_t)stream);
}

extern "C" int escat_route_bwd(const void *logits, int type, int64_t rows, int E, int k, int score, int renorm, float scale, const float *weights,
                               const int32_t *experts, const float *dweights, void *dlogits, void *stream)
{
    int rc = check_route("escat_route_bwd", type, rows, E, k, score, scale); if (rc) return rc;
    if (rows == 0) return ESCAT_OK;
    if (!logits || !weights || !experts || !dweights || !dlogits) return fail(ESCAT_EINVAL, "escat_route_bwd: null pointer");
    const int epl = E > 512 ? 16 : 8, lpr = lanes_per_row(E, epl, 1), rpb = RT / lpr;
    const int64_t want = (rows + rpb - 1) / rpb;
    const RouteBwdArgs a = {logits, weights, experts, dweights, dlogits, rows, E, k, score, renorm ? 1 : 0, scale};
    return route_dispatch<LaunchBwd>(type, lpr, epl, a, (unsigned)(want < 65536 ? want : 65536), 0, (hipStream_t)stream);
}
