// escat_adamw.hip -- one AdamW step over many tensors (the step that follows the backward of the scattering head; the
// reference takes torch's AdamW, training/prep_optimizer.py:9, and clips by the global norm, training/train.py:411-415).
//
//   c = min(1, max_norm / (sqrt(sum g^2) + 1e-6))          over all tensors, squares and sum in 64 bits
//   m = b1 m + (1-b1) c g        v = b2 v + (1-b2) (c g)^2
//   p = p (1 - lr wd) - [lr / (1-b1^t)] m / (sqrt(v) [1/sqrt(1-b2^t)] + eps)
//
// Everything between loads and stores is fp32, each operation rounded by itself (no contraction): the stored 8-bit codes are
// then a function of the inputs that elementary operations reproduce bit for bit.
//
// 8-bit states: a block of 256 consecutive elements shares a scale = (largest finite magnitude of the block) / TOP; an
// element's code is a minifloat of x = value / scale with 3 mantissa bits: 4 exponent bits and a sign for m (TOP = 15 * 2^14),
// 5 exponent bits for v, which is never negative (TOP = 14 * 2^30: squares need the wider range).  m's code 0x80 and v's 255
// stand for what is not finite, so one bad gradient spoils its own element and not the block's other 255.  Rounding is
// stochastic, by bits hashed from (seed, t, tensor, element): v moves by 1 - b2 = 1e-3 of itself a step while its codes are
// 1/8 to 1/16 apart, and rounding to nearest would never let it move.  v > 0 never becomes 0 (m / eps would follow).
//
// The tensor table travels as a kernel argument: no table in memory to keep, copy or invalidate, and a captured graph holds it.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include "escat_dev.h"
#include "escat_half.h"

#define AT 256                                   // threads: 4 waves
#define AQ 256                                   // elements of a quantisation block = one wave x 4
#define AU 4                                     // blocks of a wave: all their loads are in flight before the first is used
#define ACHUNK (AQ * AU * (AT / 64))             // elements of a workgroup
#define ATENSORS 56                              // tensors of a launch: 56 x 64 B of kernel arguments
#define NORM_WGS 2048                            // partial sums of a launch, at most
#define TOP_M 245760.0f                          // 15 * 2^14
#define TOP_V 15032385536.0f                     // 14 * 2^30
#define HDR_FLOATS 64                            // workspace header: clip, then {step size, 1/sqrt(1 - b2^t)} per group

struct ATensor { void *p; const void *g; void *m; void *v; float *ms; float *vs; int64_t n; uint32_t chunk0, ordinal; };
struct ATable { int n; uint32_t chunks; ATensor t[ATENSORS]; };
struct AGroups { int n; double lr[ESCAT_ADAMW_MAX_GROUPS], b1[ESCAT_ADAMW_MAX_GROUPS], b2[ESCAT_ADAMW_MAX_GROUPS]; };
struct AScalars { float b1, omb1, b2, omb2, eps, decay; uint32_t seed; int group; };

__device__ __forceinline__ int find_tensor(const ATable &tab, uint32_t chunk)
{
    int lo = 0, hi = tab.n - 1;                   // the last tensor whose first chunk is not behind `chunk` (chunk0 strictly increasing)
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (tab.t[mid].chunk0 <= chunk) lo = mid; else hi = mid - 1; }
    return lo;
}

// ------------------------------------------------------------------ the norm
template <typename G>
__global__ void __launch_bounds__(AT) k_grad_squares(const ATable tab, double *__restrict__ partial)
{
    __shared__ double red[AT / 64];
    const int tid = threadIdx.x;
    double acc = 0.0;
    int at = find_tensor(tab, blockIdx.x);
    for (uint32_t c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
        while (at + 1 < tab.n && tab.t[at + 1].chunk0 <= c) ++at;
        const ATensor &t = tab.t[at];
        const int64_t i0 = (int64_t)(c - t.chunk0) * ACHUNK;
        const G *g = (const G *)t.g;
        if (i0 + ACHUNK <= t.n) {
            Pack<G, 4> q[ACHUNK / AT / 4];
#pragma unroll
            for (int u = 0; u < ACHUNK / AT / 4; ++u) q[u] = *(const Pack<G, 4> *)(g + i0 + (u * AT + tid) * 4);
#pragma unroll
            for (int u = 0; u < ACHUNK / AT / 4; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) { const double x = (double)to_f32(q[u].v[k]); acc += x * x; }
        } else {
            for (int64_t i = i0 + tid; i < t.n; i += AT) { const double x = (double)to_f32(g[i]); acc += x * x; }
        }
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) acc += __shfl_xor(acc, m, 64);
    if ((tid & 63) == 0) red[tid >> 6] = acc;
    __syncthreads();
    if (tid == 0) partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ double pow_int(double b, int t)
{
    double r = 1.0;
    for (; t > 0; t >>= 1) { if (t & 1) r *= b; b *= b; }
    return r;
}

// one workgroup: joins the partial sums in a fixed order, counts the step, leaves the scalars that the update reads
__global__ void __launch_bounds__(AT) k_adamw_begin(const double *__restrict__ partial, int n_partial, int clipped, double max_norm, const AGroups gr,
                                                     int *__restrict__ step, float *__restrict__ hdr, float *__restrict__ norm_out)
{
    __shared__ double red[AT / 64];
    const int tid = threadIdx.x;
    double acc = 0.0;
    for (int i = tid; i < n_partial; i += AT) acc += partial[i];
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) acc += __shfl_xor(acc, m, 64);
    if ((tid & 63) == 0) red[tid >> 6] = acc;
    __syncthreads();
    const int t = *step + 1;
    __syncthreads();
    if (tid == 0) {
        float clip = 1.f;
        if (clipped) {
            const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
            const double c = max_norm / (norm + 1e-6);
            clip = c > 1.0 ? 1.f : (float)c;                     // a NaN norm stays NaN: every tensor shows it
            *norm_out = (float)norm;
        }
        hdr[0] = clip;
        *step = t;
    }
    if (tid < gr.n) {
        hdr[1 + 2 * tid] = (float)(gr.lr[tid] / (1.0 - pow_int(gr.b1[tid], t)));
        hdr[2 + 2 * tid] = (float)(1.0 / sqrt(1.0 - pow_int(gr.b2[tid], t)));
    }
}

// ------------------------------------------------------------------ 8-bit states
__host__ __device__ __forceinline__ uint32_t amix(uint32_t x)
{
    x = (x ^ (x >> 16)) * 0x6C8E9CF5u;
    x = (x ^ (x >> 13)) * 0x5851F42Du;
    return x ^ (x >> 16);
}

template <bool SIGNED> __device__ __forceinline__ float decode8(uint32_t c, float scale)
{
    const uint32_t a = SIGNED ? (c & 127u) : c;
    float y = a >= 8u ? __uint_as_float((a + (129u << 3)) << 20) : (float)a;
    if (SIGNED) y = c == 128u ? __uint_as_float(0x7fc00000u) : (c > 128u ? -y : y);
    else y = c == 255u ? __uint_as_float(0x7fc00000u) : y;
    return y * scale;
}

template <bool SIGNED> __device__ __forceinline__ uint32_t encode8(float x, float inv, uint32_t r16)
{
#pragma clang fp contract(off)
    const float top = SIGNED ? TOP_M : TOP_V;
    const float a = fabsf(x);
    if (!(a < __uint_as_float(0x7f800000u))) return SIGNED ? 128u : 255u;
    float y = a * inv;
    y = y < top ? y : top;
    uint32_t c;
    if (y >= 8.0f) c = ((__float_as_uint(y) + (r16 << 4)) >> 20) - (129u << 3);
    else c = (uint32_t)(y + (float)r16 * 1.52587890625e-5f);
    if (SIGNED) { c = c < 127u ? c : 127u; if (x < 0.f && c) c |= 128u; }
    else { c = c < 254u ? c : 254u; if (x > 0.f && !c) c = 1u; }
    return c;
}

// largest value of the wave's non-negative floats, in all lanes (a NaN or an infinity must not come in)
__device__ __forceinline__ float wave_max_nonneg(float v)
{
    int x = __float_as_int(v);
#define DPP_MAX(ctrl) { const int o = __builtin_amdgcn_update_dpp(0, x, ctrl, 0xf, 0xf, true); x = o > x ? o : x; }
    DPP_MAX(0x111) DPP_MAX(0x112) DPP_MAX(0x114) DPP_MAX(0x118) DPP_MAX(0x142) DPP_MAX(0x143)
#undef DPP_MAX
    return __int_as_float(__builtin_amdgcn_readlane(x, 63));
}

__device__ __forceinline__ void block_scale(float size, float top, float &scale, float &inv)
{
    // the floor keeps 1 / size finite; what lies 2^-90 and further below rounds by its share of the smallest code
    size = size > 0.f && size < 8.0779356694631609e-28f ? 8.0779356694631609e-28f : size;         // 2^-90
    scale = size * (1.0f / top);
    inv = size > 0.f ? (1.0f / size) * top : 0.f;
}

__device__ __forceinline__ float finite_size(float x) { const float a = fabsf(x); return a < __uint_as_float(0x7f800000u) ? a : 0.f; }

// ------------------------------------------------------------------ the update
// The hardware's root takes a v below 2^-126 for 0, which an eps of 1e-8 hides and one of 0 does not (m / 0): such a v goes through it multiplied by
// 2^64.  SMALL: whether that may show (root_shows)
template <bool SMALL> __device__ __forceinline__ float root_of(float v)
{
    if (!SMALL) return __builtin_amdgcn_sqrtf(v);
    const bool low = v < 1.2621774483536189e-29f;                                      // 2^-96
    const float r = __builtin_amdgcn_sqrtf(low ? v * 18446744073709551616.0f : v);
    return low ? r * 2.3283064365386963e-10f : r;                                      // 2^-32
}

struct AVals { float p, m, v; };
template <bool SMALL> __device__ __forceinline__ AVals adamw_one(float p, float g, float m, float v, const AScalars &s, float clip, float size, float isb)
{
#pragma clang fp contract(off)
    g = g * clip;
    m = m * s.b1 + g * s.omb1;
    v = v * s.b2 + (g * g) * s.omb2;
    // (hardware root and reciprocal, 1 unit in the last place of the update each: an exact root and quotient are 25 instructions more, which
    // the 8-bit form has no room for; the moments do not pass here)
    const float num = m * size, den = root_of<SMALL>(v) * isb + s.eps;
    return {p * s.decay - num * __builtin_amdgcn_rcpf(den), m, v};
}

template <typename P, typename G, int BITS, bool SMALL>
__global__ void __launch_bounds__(AT) k_adamw(const ATable tab, const AScalars s, const int *__restrict__ step, const float *__restrict__ hdr)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const ATensor &t = tab.t[find_tensor(tab, blockIdx.x)];
    const int64_t n = t.n;
    const int64_t w0 = (int64_t)(blockIdx.x - t.chunk0) * ACHUNK + (int64_t)__builtin_amdgcn_readfirstlane(wave) * (AQ * AU);
    if (w0 >= n) return;
    const float clip = hdr[0], size = hdr[1 + 2 * s.group], isb = hdr[2 + 2 * s.group];
    P *pp = (P *)t.p; const G *gp = (const G *)t.g;
    uint32_t key = 0;
    if (BITS == 8) key = amix(amix((uint32_t)*step + s.seed * 0x2545F491u) + t.ordinal * 0x632BE5ABu);
    const int64_t i0 = w0 + lane * 4;
    const int live = n - w0 >= AQ * AU ? AU : (int)((n - w0 + AQ - 1) / AQ);         // blocks of this wave (wave-uniform)

    float p[AU][4], g[AU][4], m[AU][4], v[AU][4];
    uint32_t cm[AU], cv[AU];
    const bool whole = n - w0 >= AQ * AU;
    if (whole) {
#pragma unroll
        for (int u = 0; u < AU; ++u) {
            const int64_t i = i0 + u * AQ;
            const Pack<P, 4> a = *(const Pack<P, 4> *)(pp + i);
            const Pack<G, 4> b = *(const Pack<G, 4> *)(gp + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) { p[u][k] = to_f32(a.v[k]); g[u][k] = to_f32(b.v[k]); }
            if (BITS == 32) {
                const Pack<float, 4> c = *(const Pack<float, 4> *)((const float *)t.m + i), d = *(const Pack<float, 4> *)((const float *)t.v + i);
#pragma unroll
                for (int k = 0; k < 4; ++k) { m[u][k] = c.v[k]; v[u][k] = d.v[k]; }
            } else {
                const Pack<uint8_t, 4> c = *(const Pack<uint8_t, 4> *)((const uint8_t *)t.m + i), d = *(const Pack<uint8_t, 4> *)((const uint8_t *)t.v + i);
                __builtin_memcpy(&cm[u], &c, 4); __builtin_memcpy(&cv[u], &d, 4);
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < AU; ++u) {
            cm[u] = cv[u] = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t i = i0 + u * AQ + k;
                const bool in = i < n;
                p[u][k] = in ? to_f32(pp[i]) : 0.f; g[u][k] = in ? to_f32(gp[i]) : 0.f;
                if (BITS == 32) { m[u][k] = in ? ((const float *)t.m)[i] : 0.f; v[u][k] = in ? ((const float *)t.v)[i] : 0.f; }
                else if (in) { cm[u] |= (uint32_t)((const uint8_t *)t.m)[i] << (8 * k); cv[u] |= (uint32_t)((const uint8_t *)t.v)[i] << (8 * k); }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < AU; ++u) {
        const int64_t blk = w0 / AQ + u;
        if (BITS == 8) {
            const float ms = u < live ? t.ms[blk] : 0.f, vs = u < live ? t.vs[blk] : 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) { m[u][k] = decode8<true>((cm[u] >> (8 * k)) & 255u, ms); v[u][k] = decode8<false>((cv[u] >> (8 * k)) & 255u, vs); }
        }
        float mx = 0.f, vx = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const AVals r = adamw_one<SMALL>(p[u][k], g[u][k], m[u][k], v[u][k], s, clip, size, isb);
            p[u][k] = r.p; m[u][k] = r.m; v[u][k] = r.v;
            if (BITS == 8 && (whole || i0 + u * AQ + k < n)) { mx = fmaxf(mx, finite_size(r.m)); vx = fmaxf(vx, finite_size(r.v)); }
        }
        if (BITS == 8) {
            mx = wave_max_nonneg(mx); vx = wave_max_nonneg(vx);
            float msc, minv, vsc, vinv;
            block_scale(mx, TOP_M, msc, minv); block_scale(vx, TOP_V, vsc, vinv);
            if (lane == 0 && u < live) { t.ms[blk] = msc; t.vs[blk] = vsc; }
            uint32_t om = 0, ov = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint64_t i = (uint64_t)(i0 + u * AQ + k);
                const uint32_t r = amix(amix((uint32_t)(i >> 32) + key) ^ (uint32_t)i);
                om |= encode8<true>(m[u][k], minv, r & 0xffffu) << (8 * k);
                ov |= encode8<false>(v[u][k], vinv, r >> 16) << (8 * k);
            }
            cm[u] = om; cv[u] = ov;
        }
    }
    if (whole) {
#pragma unroll
        for (int u = 0; u < AU; ++u) {
            const int64_t i = i0 + u * AQ;
            Pack<P, 4> a;
#pragma unroll
            for (int k = 0; k < 4; ++k) a.v[k] = from_f32<P>(p[u][k]);
            *(Pack<P, 4> *)(pp + i) = a;
            if (BITS == 32) {
                Pack<float, 4> c, d;
#pragma unroll
                for (int k = 0; k < 4; ++k) { c.v[k] = m[u][k]; d.v[k] = v[u][k]; }
                *(Pack<float, 4> *)((float *)t.m + i) = c; *(Pack<float, 4> *)((float *)t.v + i) = d;
            } else {
                Pack<uint8_t, 4> c, d;
                __builtin_memcpy(&c, &cm[u], 4); __builtin_memcpy(&d, &cv[u], 4);
                *(Pack<uint8_t, 4> *)((uint8_t *)t.m + i) = c; *(Pack<uint8_t, 4> *)((uint8_t *)t.v + i) = d;
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < AU; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t i = i0 + u * AQ + k;
                if (i >= n) continue;
                pp[i] = from_f32<P>(p[u][k]);
                if (BITS == 32) { ((float *)t.m)[i] = m[u][k]; ((float *)t.v)[i] = v[u][k]; }
                else { ((uint8_t *)t.m)[i] = (uint8_t)(cm[u] >> (8 * k)); ((uint8_t *)t.v)[i] = (uint8_t)(cv[u] >> (8 * k)); }
            }
    }
}

// values of an 8-bit state
template <bool SIGNED>
__global__ void __launch_bounds__(AT) k_state8_values(const uint8_t *__restrict__ code, const float *__restrict__ scale, int64_t n, float *__restrict__ out)
{
    const int64_t i0 = ((int64_t)blockIdx.x * AU * AT + threadIdx.x) * 4;
    if (i0 + (AU - 1) * AT * 4 + 4 <= n) {
        Pack<uint8_t, 4> c[AU];
        float z[AU];
#pragma unroll
        for (int u = 0; u < AU; ++u) { c[u] = *(const Pack<uint8_t, 4> *)(code + i0 + u * AT * 4); z[u] = scale[(i0 + u * AT * 4) / AQ]; }
#pragma unroll
        for (int u = 0; u < AU; ++u) {
            Pack<float, 4> o;
#pragma unroll
            for (int k = 0; k < 4; ++k) o.v[k] = decode8<SIGNED>(c[u].v[k], z[u]);
            *(Pack<float, 4> *)(out + i0 + u * AT * 4) = o;
        }
    } else {
        for (int u = 0; u < AU; ++u)
            for (int64_t j = i0 + u * AT * 4; j < i0 + u * AT * 4 + 4 && j < n; ++j) out[j] = decode8<SIGNED>(code[j], scale[j / AQ]);
    }
}

// ------------------------------------------------------------------ entry points
// walks the tensors in launches of at most ATENSORS, leaving empty ones out; f(table, launch) launches one
template <typename F> static int for_tables(const escat_adamw_tensor *ts, int n, F f)
{
    ATable tab;
    int launch = 0;
    for (int i = 0; i < n;) {
        tab.n = 0; tab.chunks = 0;
        uint64_t chunks = 0;
        for (; i < n && tab.n < ATENSORS; ++i) {
            if (ts[i].n == 0) continue;
            const uint64_t c = (uint64_t)((ts[i].n + ACHUNK - 1) / ACHUNK);
            if (chunks + c > 0xffffffull) { if (tab.n == 0) return fail(ESCAT_ERANGE, "tensor %d has %lld elements: beyond what a launch covers", i, (long long)ts[i].n); break; }
            tab.t[tab.n++] = {ts[i].param, ts[i].grad, ts[i].m, ts[i].v, ts[i].m_scale, ts[i].v_scale, ts[i].n, (uint32_t)chunks, ts[i].ordinal};
            chunks += c;
        }
        if (tab.n == 0) break;
        tab.chunks = (uint32_t)chunks;
        const int rc = f(tab, launch++); if (rc) return rc;
    }
    return ESCAT_OK;
}

static int check_tensors(const escat_adamw_tensor *ts, int n, const char *who)
{
    if (n < 0 || (n > 0 && !ts)) return fail(ESCAT_EINVAL, "%s: n_tensors = %d, tensors = %p", who, n, (const void *)ts);
    for (int i = 0; i < n; ++i)
        if (ts[i].n < 0 || (ts[i].n > 0 && !ts[i].grad)) return fail(ESCAT_EINVAL, "%s: tensor %d: n = %lld, grad = %p", who, i, (long long)ts[i].n, ts[i].grad);
    return ESCAT_OK;
}

static int max_launches(int n_tensors) { return n_tensors / 28 + 4; }        // a launch is cut at 56 tensors or 2^24 chunks, and between types

extern "C" size_t escat_adamw_workspace_bytes(int n_tensors)
{
    return n_tensors < 0 ? 0 : HDR_FLOATS * 4 + (size_t)max_launches(n_tensors) * NORM_WGS * 8;
}

extern "C" int escat_adamw_begin(const escat_adamw_tensor *tensors, int n_tensors, int grad_type, double max_norm, int partial_slot,
                                 int finish, const escat_adamw_group *groups, int n_groups, int32_t *step, float *norm_out,
                                 void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_tensors(tensors, n_tensors, "escat_adamw_begin"); if (rc) return rc;
    if (!escat_type_bytes(grad_type)) return fail(ESCAT_EINVAL, "escat_adamw_begin: grad_type = %d", grad_type);
    if (!workspace || workspace_bytes < HDR_FLOATS * 4) return fail(ESCAT_EWORKSPACE, "escat_adamw_begin: workspace of %zu bytes", workspace_bytes);
    if (((uintptr_t)workspace & 7) != 0) return fail(ESCAT_EINVAL, "escat_adamw_begin: workspace is not aligned to 8 bytes");
    if (partial_slot < 0) return fail(ESCAT_EINVAL, "escat_adamw_begin: partial_slot = %d", partial_slot);
    if (finish && (n_groups < 1 || n_groups > ESCAT_ADAMW_MAX_GROUPS || !groups || !step))
        return fail(ESCAT_EINVAL, "escat_adamw_begin: n_groups = %d (1..%d), groups = %p, step = %p", n_groups, ESCAT_ADAMW_MAX_GROUPS, (const void *)groups, (void *)step);
    const bool clip = max_norm > 0;
    if (finish && clip && !norm_out) return fail(ESCAT_EINVAL, "escat_adamw_begin: clipping needs norm_out");
    hipStream_t st = (hipStream_t)stream;
    double *partial = (double *)((char *)workspace + HDR_FLOATS * 4);
    const int64_t room = (int64_t)((workspace_bytes - HDR_FLOATS * 4) / 8);
    int slot = partial_slot;
    if (clip) {
        rc = for_tables(tensors, n_tensors, [&](const ATable &tab, int) {
            const unsigned wgs = tab.chunks < NORM_WGS ? tab.chunks : NORM_WGS;
            if (slot + (int64_t)wgs > room) return fail(ESCAT_EWORKSPACE, "escat_adamw_begin: workspace of %zu bytes holds %lld partial sums", workspace_bytes, (long long)room);
            double *out = partial + slot;
            slot += (int)wgs;
            switch (grad_type) {
            case ESCAT_F32: k_grad_squares<float><<<wgs, AT, 0, st>>>(tab, out); break;
            case ESCAT_BF16: k_grad_squares<bf16_t><<<wgs, AT, 0, st>>>(tab, out); break;
            default: k_grad_squares<f16_t><<<wgs, AT, 0, st>>>(tab, out); break;
            }
            CHECK_LAUNCH("escat_adamw_begin: squares");
            return ESCAT_OK;
        });
        if (rc) return rc;
    }
    if (!finish) return slot;
    AGroups gr;
    gr.n = n_groups;
    for (int i = 0; i < n_groups; ++i) { gr.lr[i] = groups[i].lr; gr.b1[i] = groups[i].beta1; gr.b2[i] = groups[i].beta2; }
    k_adamw_begin<<<1, AT, 0, st>>>(partial, clip ? slot : 0, clip ? 1 : 0, max_norm, gr, step, (float *)workspace, norm_out);
    CHECK_LAUNCH("escat_adamw_begin");
    return slot;
}

// A root taken for 0 is short of at most 2^-63, times its scalar 1 / sqrt(1 - b2^t) <= 1 / sqrt(1 - b2): beyond 2^-23 of eps that shows in the
// update (eps = 1e-8: not for b2 up to 1 - 8e-9).  The 8-bit form, which its instructions bound, looks after it only then: 64 Mi fp32 parameters
// 220 us without, 224 with; the 32-bit form always, 363 us either way
static bool root_shows(double eps, double b2) { return eps * sqrt(1.0 - b2) < 9.094947017729282e-13; }            // 2^-40

template <typename P, typename G>
static int launch_update(const ATable &tab, const AScalars &s, int bits, bool small, const int32_t *step, const float *hdr, hipStream_t st)
{
    if (bits == 32) k_adamw<P, G, 32, true><<<tab.chunks, AT, 0, st>>>(tab, s, step, hdr);
    else if (small) k_adamw<P, G, 8, true><<<tab.chunks, AT, 0, st>>>(tab, s, step, hdr);
    else k_adamw<P, G, 8, false><<<tab.chunks, AT, 0, st>>>(tab, s, step, hdr);
    CHECK_LAUNCH("escat_adamw_update");
    return ESCAT_OK;
}

extern "C" int escat_adamw_update(const escat_adamw_tensor *tensors, int n_tensors, int param_type, int grad_type, int state_bits,
                                  const escat_adamw_group *group, int group_index, uint32_t seed, const int32_t *step,
                                  const void *workspace, void *stream)
{
    int rc = check_tensors(tensors, n_tensors, "escat_adamw_update"); if (rc) return rc;
    if (!escat_type_bytes(param_type) || (grad_type != param_type && grad_type != ESCAT_F32))
        return fail(ESCAT_EINVAL, "escat_adamw_update: param_type = %d, grad_type = %d (the parameters' type or fp32)", param_type, grad_type);
    if (state_bits != 32 && state_bits != 8) return fail(ESCAT_EINVAL, "escat_adamw_update: state_bits = %d (32 or 8)", state_bits);
    if (!group || group_index < 0 || group_index >= ESCAT_ADAMW_MAX_GROUPS || !step || !workspace)
        return fail(ESCAT_EINVAL, "escat_adamw_update: group = %p, group_index = %d, step = %p, workspace = %p", (const void *)group, group_index, (const void *)step, workspace);
    for (int i = 0; i < n_tensors; ++i)
        if (tensors[i].n > 0 && (!tensors[i].param || !tensors[i].m || !tensors[i].v || (state_bits == 8 && (!tensors[i].m_scale || !tensors[i].v_scale))))
            return fail(ESCAT_EINVAL, "escat_adamw_update: tensor %d has a null pointer", i);
    const AScalars s = {(float)group->beta1, (float)(1.0 - group->beta1), (float)group->beta2, (float)(1.0 - group->beta2), (float)group->eps,
                        (float)(1.0 - group->lr * group->weight_decay), seed, group_index};
    hipStream_t st = (hipStream_t)stream;
    const float *hdr = (const float *)workspace;
    const bool small = root_shows(group->eps, group->beta2);
    return for_tables(tensors, n_tensors, [&](const ATable &tab, int) {
        if (param_type == ESCAT_F32) return launch_update<float, float>(tab, s, state_bits, small, step, hdr, st);
        if (param_type == ESCAT_BF16)
            return grad_type == ESCAT_BF16 ? launch_update<bf16_t, bf16_t>(tab, s, state_bits, small, step, hdr, st) : launch_update<bf16_t, float>(tab, s, state_bits, small, step, hdr, st);
        return grad_type == ESCAT_F16 ? launch_update<f16_t, f16_t>(tab, s, state_bits, small, step, hdr, st) : launch_update<f16_t, float>(tab, s, state_bits, small, step, hdr, st);
    });
}

extern "C" int escat_state8_values(const uint8_t *codes, const float *scales, int64_t n, int is_signed, float *out, void *stream)
{
    if (n < 0 || (n > 0 && (!codes || !scales || !out))) return fail(ESCAT_EINVAL, "escat_state8_values: n = %lld or a null pointer", (long long)n);
    if (n == 0) return ESCAT_OK;
    const int64_t wgs = (n + AU * AT * 4 - 1) / (AU * AT * 4);
    if (wgs > 0xffffff) return fail(ESCAT_ERANGE, "escat_state8_values: n = %lld", (long long)n);
    hipStream_t st = (hipStream_t)stream;
    if (is_signed) k_state8_values<true><<<(unsigned)wgs, AT, 0, st>>>(codes, scales, n, out);
    else k_state8_values<false><<<(unsigned)wgs, AT, 0, st>>>(codes, scales, n, out);
    CHECK_LAUNCH("escat_state8_values");
    return ESCAT_OK;
}
