// escat_experts_tile.h -- the 128 x 128 matrix tile that all products of the experts share (device code)
//
// C[m][n] += sum_k A[m][k] B[n][k], m = features (A side), n = rows of activations or features (B side).  256 threads, four
// waves of 64 x 64 each (2 x 2 MFMA blocks of 32 x 32, fp32 accumulators).  One step covers KB values of k: 64 of 16 bits or 32 of
// 32 bits, 128 bytes of a row.  Operands come from memory through registers into LDS.
//
// An operand lies in memory with k contiguous ("KC": rows of activations, W1 / W2 in the forward) or with m contiguous ("KM": the
// weights in the backward, both operands of a weight gradient).  In LDS:
//   KC  row r: 128 bytes = 8 chunks of 16, chunk c at c ^ ((r >> 1) & 7): the 16 lanes that a 16-byte read serves at once (rows 0-3, 12-15, 20-27
//       or the other half of 32) fall on the 16 slots of two rows once each, the 8 lanes of a write on 8
//   KM  row k: 16 bits: 256 bytes = 4 granules of 64, granule q at q ^ (k & 3), read by ds_read_tr16_b64, which hands each lane
//       four k of one column (4 rows x 64 bytes of a half wave on distinct banks);  32 bits: 512 bytes, read one value a lane
// MFMA operands: 16 bits 32x32x16, lane l holds k = 8 (l / 32) + 0..7 of row l % 32.  32 bits 32x32x2 (full fp32 products), lane l holds k = l / 32
// of its pair; which two k make a pair is free as long as A and B agree: KC pairs k with k + 4 so that one 16-byte read serves four.
// Result: lane l, register i: m = 8 (i / 4) + 4 (l / 32) + i % 4, n = l % 32.
#ifndef ESCAT_EXPERTS_TILE_H
#define ESCAT_EXPERTS_TILE_H
#include "escat_experts.h"

#define XT 256
#define TILE_BYTES 16384                          // one operand, one buffer

typedef float acc_t __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem;                // PER: elements of 16 bytes; KB: k of a step
template <> struct Elem<float> { static constexpr int PER = 4, KB = 32; };
template <> struct Elem<bf16_t> { static constexpr int PER = 8, KB = 64; };
template <> struct Elem<f16_t> { static constexpr int PER = 8, KB = 64; };

typedef unsigned u4 __attribute__((ext_vector_type(4)));
template <typename T> struct Vec { T v[Elem<T>::PER]; };

// Pieces at the ragged end of a row: 16 bytes are loaded so that they end with the row (one unguarded load whatever the row's length; the entry points see to it that
// it has 16 bytes) and, once they have arrived, moved down by the s elements that the piece begins behind where it was loaded, zeros behind.
template <typename T> __device__ __forceinline__ u4 load16(const T *p)
{
    const Pack<T, Elem<T>::PER> q = *(const Pack<T, Elem<T>::PER> *)p;
    u4 r; __builtin_memcpy(&r, &q, 16);
    return r;
}
// (by 32-bit selects: a 64-bit shift whose amount lies in the last VGPR of a kernel's allocation shifts by something else on this card)
template <typename T> __device__ __forceinline__ u4 moved(u4 v, int s)
{
    if (sizeof(T) == 2) {                                         // an odd number: one element first
        const unsigned by = (s & 1) * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_alignbit(i < 3 ? v[i + 1] : 0u, v[i], by);
        s >>= 1;
    }
    // words: by one or none, by two or none, all gone.  (Masks: selects became branches)
    const unsigned one = -(unsigned)(s & 1), two = -(unsigned)(s >> 1 & 1), stay = s >= 4 ? 0u : ~0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (v[i] & ~one) | (i < 3 ? v[i + 1] & one : 0u);
    return u4{((v[0] & ~two) | (v[2] & two)) & stay, ((v[1] & ~two) | (v[3] & two)) & stay, v[2] & ~two & stay, v[3] & ~two & stay};
}
template <typename T> __device__ __forceinline__ void to_floats(u4 r, float (&f)[Elem<T>::PER])
{
    Vec<T> q; __builtin_memcpy(&q, &r, 16);
#pragma unroll
    for (int i = 0; i < Elem<T>::PER; ++i) f[i] = (float)q.v[i];
}

// ---- staging: thread t's four 16-byte pieces of an operand's tile
template <typename T, bool KM> struct Stage {
    static constexpr int PER = Elem<T>::PER;
    static constexpr int CPR = KM ? 128 / PER : 8;          // chunks of an LDS row
    static constexpr int RPP = XT / CPR;                    // rows of a pass: KC 32; KM 16 (16 bits), 8 (32 bits)
    static __device__ __forceinline__ int chunk() { return threadIdx.x % CPR; }
    static __device__ __forceinline__ int row(int i) { return threadIdx.x / CPR + i * RPP; }
    static __device__ __forceinline__ void store(char *lds, const u4 (&v)[4])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row(i), c = chunk();
            const int at = !KM ? r * 128 + ((c ^ ((r >> 1) & 7)) << 4) : sizeof(T) == 4 ? r * 512 + c * 16 : r * 256 + (((c >> 2) ^ (r & 3)) << 6) + (c & 3) * 16;
            *(u4 *)(lds + at) = v[i];
        }
    }
};

// ---- one step's products of a wave: acc[i][j] += A block i x B block j
template <typename T> __device__ __forceinline__ s8 frag_kc(const char *lds, int row, int sub)
{
    const int l = threadIdx.x & 63, r = row + (l & 31), c = sub * 2 + (l >> 5);
    return *(const s8 *)(lds + r * 128 + ((c ^ ((r >> 1) & 7)) << 4));
}
__device__ __forceinline__ s8 frag_km16(const char *lds, int col, int sub)
{
    const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
    const int k = sub * 16 + (g >> 1) * 8 + (i >> 2);
    const char *p = lds + k * 256 + (((col >> 5) ^ (k & 3)) << 6) + ((g & 1) * 16 + (i & 3) * 4) * 2;
    typedef __attribute__((address_space(3))) s4 ls4;
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)p), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)(p + 4 * 256));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ acc_t mma16(bf16_t, s8 a, s8 b, acc_t c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
__device__ __forceinline__ acc_t mma16(f16_t, s8 a, s8 b, acc_t c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

template <typename T, bool AKM, bool BKM>
__device__ __forceinline__ void tile_step(const char *la, const char *lb, int am, int bn, acc_t (&acc)[2][2])
{
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            s8 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (AKM) a[i] = frag_km16(la, am + 32 * i, s); else a[i] = frag_kc<T>(la, am + 32 * i, s);
                if constexpr (BKM) b[i] = frag_km16(lb, bn + 32 * i, s); else b[i] = frag_kc<T>(lb, bn + 32 * i, s);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mma16(T{}, a[i], b[j], acc[i][j]);
        }
    } else {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int s = 0; s < 4; ++s) {                        // eight k: four pairs (k, k + 4)
            f4 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (AKM) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) a[i][q] = *(const float *)(la + (s * 8 + (l >> 5) * 4 + q) * 512 + (am + 32 * i + (l & 31)) * 4);
                } else a[i] = __builtin_bit_cast(f4, frag_kc<T>(la, am + 32 * i, s));
                if constexpr (BKM) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) b[i][q] = *(const float *)(lb + (s * 8 + (l >> 5) * 4 + q) * 512 + (bn + 32 * i + (l & 31)) * 4);
                } else b[i] = __builtin_bit_cast(f4, frag_kc<T>(lb, bn + 32 * i, s));
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i][q], b[j][q], acc[i][j], 0, 0, 0);
        }
    }
}

// ---- the loop over the steps.  a / b: operands with load(regs) -- the thread's pieces of the next step -- and fix(regs) -- the same pieces once
// they have arrived (a use inside load would wait for them there); both are called once a step, in order.  One buffer in LDS and one set of
// registers, two barriers a step: the two to four workgroups of a CU hide each other's waits.  (Measured against loads one or two steps ahead into
// a second buffer, which leaves room for two workgroups: 349 us instead of 391 for 137 GFLOP in bf16 at K = 256, the same at K = 1024; fp32
// 4 GFLOP at K = 256 62 us instead of 68.)  start() issues the first loads, so that a kernel can do other things until run(); run calls `next`
// before the last products, when no load is left to issue.  lds is free to be written on return.
struct Nothing { __device__ void operator()() const {} };
// PIN: the loads stay before the products.  The compiler likes them behind, which saves registers: with two workgroups a CU the wait is
// longer than the registers are worth (BWD1 of escat_experts_rows.hip 598 instead of 622 us), with four it is the other way (W1 x 343 instead of 288)
template <typename T, bool AKM, bool BKM, bool PIN = false> struct Pipe {
    u4 ra[4], rb[4];
    template <typename A, typename B> __device__ __forceinline__ void start(int steps, A &a, B &b)
    {
        if (steps > 0) { a.load(ra); b.load(rb); }
    }
    template <typename A, typename B> __device__ __forceinline__ void store(char *lds, A &a, B &b)
    {
        a.fix(ra); b.fix(rb);
        Stage<T, AKM>::store(lds, ra); Stage<T, BKM>::store(lds + TILE_BYTES, rb);
        __syncthreads();
    }
    // no load under a condition inside the loop: it would make the compiler wait for all of them at every turn
    template <typename A, typename B, typename N = Nothing>
    __device__ __forceinline__ void run(int steps, char *lds, int am, int bn, acc_t (&acc)[2][2], A &a, B &b, N next = N())
    {
        if (steps == 0) { next(); return; }
        for (int s = 1; s < steps; ++s) {
            store(lds, a, b);
            a.load(ra); b.load(rb);
            if (PIN) __builtin_amdgcn_sched_barrier(0);
            tile_step<T, AKM, BKM>(lds, lds + TILE_BYTES, am, bn, acc);
            __syncthreads();
        }
        store(lds, a, b);
        next();
        if (PIN) __builtin_amdgcn_sched_barrier(0);
        tile_step<T, AKM, BKM>(lds, lds + TILE_BYTES, am, bn, acc);
        __syncthreads();
    }
};

template <typename T> __device__ __forceinline__ void fix_kc(u4 (&r)[4], int K, int c, int &k0);
// ---- operands.  An operand walks through one or more segments of K values of k (by combination: one for each expert of the tile), each
// padded to whole steps; `seg(j)` says where segment j begins.
// k contiguous, rows at 32-bit offsets from a base that a segment moves
template <typename T, typename SEG> struct OperandKC {
    SEG seg;
    int K, c, k0, j, fk0;
    const char *base;
    uint32_t off[4];
    __device__ __forceinline__ OperandKC(int K, SEG seg) : seg(seg), K(K), c(Stage<T, false>::chunk() * Elem<T>::PER), k0(0), j(0), fk0(0), base(seg(0)) {}
    __device__ __forceinline__ void load(u4 (&r)[4])
    {
        constexpr int PER = Elem<T>::PER;
        const uint32_t at = (uint32_t)(k0 + c < K - PER ? k0 + c : K - PER) * (uint32_t)sizeof(T);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = load16((const T *)(base + (size_t)(off[i] + at)));
        k0 += Elem<T>::KB;
        if (k0 >= K) { k0 = 0; base = seg(++j); }
    }
    __device__ __forceinline__ void fix(u4 (&r)[4]) { fix_kc<T>(r, K, c, fk0); }
};
template <typename T> __device__ __forceinline__ void fix_kc(u4 (&r)[4], int K, int c, int &k0)
{
    constexpr int PER = Elem<T>::PER;
    if (k0 + Elem<T>::KB > K) {
        const int s = k0 + c > K - PER ? k0 + c - (K - PER) : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = moved<T>(r[i], s);
    }
    k0 += Elem<T>::KB;
    if (k0 >= K) k0 = 0;
}
// k contiguous, rows anywhere (activations by row); one segment
template <typename T> struct OperandKCRows {
    const T *p[4];
    int K, c, k0, fk0;
    __device__ __forceinline__ explicit OperandKCRows(int K) : K(K), c(Stage<T, false>::chunk() * Elem<T>::PER), k0(0), fk0(0) {}
    __device__ __forceinline__ void load(u4 (&r)[4])
    {
        constexpr int PER = Elem<T>::PER;
        const int at = k0 + c < K - PER ? k0 + c : K - PER;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = load16(p[i] + at);
        k0 += Elem<T>::KB;
    }
    __device__ __forceinline__ void fix(u4 (&r)[4]) { fix_kc<T>(r, K, c, fk0); }
};
// where the thread's pieces of a row of M features begin (KM), and how far they are to be moved
template <typename T> struct ColsKM {
    int at, s;
    bool ragged;                                        // the tile has a piece that ends behind the row
    __device__ __forceinline__ ColsKM(int m0, int M)
    {
        constexpr int PER = Elem<T>::PER;
        const int m = m0 + Stage<T, true>::chunk() * PER;
        at = m < M - PER ? m : M - PER;
        s = m - at;
        ragged = m0 + 128 > M;
    }
    __device__ __forceinline__ void fix(u4 (&r)[4], int live, bool whole) const          // live: rows of the step that exist
    {
        if (ragged) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = moved<T>(r[i], s);
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) if (Stage<T, true>::row(i) >= live) r[i] = u4{0, 0, 0, 0};
        }
    }
};
// features contiguous, rows of k one after the other from a base that a segment moves (weights in the backward)
template <typename T, typename SEG> struct OperandKM {
    SEG seg;
    ColsKM<T> cols;
    int K, k0, j, fk0;
    uint32_t row, off, last;                            // bytes: of a row, of the thread's piece in row k0 + row(0), in row K - 1
    const char *base;
    __device__ __forceinline__ OperandKM(int K, int m0, int M, SEG seg)
        : seg(seg), cols(m0, M), K(K), k0(0), j(0), fk0(0), row((uint32_t)M * (uint32_t)sizeof(T)), base(seg(0))
    {
        off = (uint32_t)Stage<T, true>::row(0) * row + (uint32_t)cols.at * (uint32_t)sizeof(T);
        last = (uint32_t)(K - 1) * row + (uint32_t)cols.at * (uint32_t)sizeof(T);
    }
    __device__ __forceinline__ void load(u4 (&r)[4])
    {
        const uint32_t o = off + (uint32_t)k0 * row;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t q = o + (uint32_t)(i * Stage<T, true>::RPP) * row;
            r[i] = load16((const T *)(base + (size_t)(q < last ? q : last)));
        }
        k0 += Elem<T>::KB;
        if (k0 >= K) { k0 = 0; base = seg(++j); }
    }
    __device__ __forceinline__ void fix(u4 (&r)[4])
    {
        cols.fix(r, K - fk0, fk0 + Elem<T>::KB <= K);
        fk0 += Elem<T>::KB;
        if (fk0 >= K) fk0 = 0;
    }
};

// ---- results through LDS, so that memory is written in whole rows of the tile: rows [0, rows), features [0, cols) to out + at(row) * ld.
// A row of 128 OUT is STRIDE bytes from the next: 16 more than its size, so that the runs of 32 rows fall on different banks.  32-bit
// results go in two halves of 64 rows: 34 KB hold either.  lds is free before (the caller's barrier) and in use on return.  The stores do not
// stay in the caches: another kernel reads what is written here, and 512 MB of it push out the weights and the rows that workgroups share
// (524288 rows, k = 2, 256 x 256 in bf16: W1 x 297 instead of 344 us, with the gradient of u 786 instead of 890).
template <typename OUT> struct Spill {
    static constexpr int STRIDE = 128 * (int)sizeof(OUT) + 16, ROWS = sizeof(OUT) == 4 ? 64 : 128, BYTES = ROWS * STRIDE;
    template <typename AT>
    static __device__ __forceinline__ void all(char *lds, const acc_t (&acc)[2][2], int am, int bn, OUT *out, int64_t ld, int rows, int cols, AT at)
    {
        constexpr int PER = 16 / (int)sizeof(OUT), CPR = 128 / PER;
        const int lane = threadIdx.x & 63, c = threadIdx.x % CPR * PER;
#pragma unroll
        for (int half = 0; half < 128 / ROWS; ++half) {
            if (half) __syncthreads();
            if (ROWS == 128 || bn == half * 64)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int n = bn - half * 64 + 32 * j + (lane & 31), m = am + 32 * i + 8 * q + 4 * (lane >> 5);
                            struct alignas(4 * sizeof(OUT)) { OUT v[4]; } p;
#pragma unroll
                            for (int z = 0; z < 4; ++z) p.v[z] = from_f32<OUT>(acc[i][j][4 * q + z]);
                            __builtin_memcpy(__builtin_assume_aligned(lds + n * STRIDE + m * (int)sizeof(OUT), 4 * sizeof(OUT)), &p, sizeof(p));
                        }
            __syncthreads();
            if (c >= cols) continue;
            for (int r = threadIdx.x / CPR; r < ROWS && r + half * 64 < rows; r += XT / CPR) {
                struct alignas(16) { OUT v[PER]; } q;
                __builtin_memcpy(&q, __builtin_assume_aligned(lds + r * STRIDE + c * (int)sizeof(OUT), 16), 16);
                OUT *o = out + (int64_t)at(r + half * 64) * ld + c;
                if (c + PER <= cols) { typedef unsigned ua __attribute__((ext_vector_type(4), aligned(2))); ua p; __builtin_memcpy(&p, &q, 16); __builtin_nontemporal_store(p, (ua *)o); }
                else {
#pragma unroll
                    for (int z = 0; z < PER; ++z) if (c + z < cols) o[z] = q.v[z];
                }
            }
        }
    }
};
#define LDS_BYTES 34816                           // of a kernel: two tiles, or results on their way out
static_assert(Spill<float>::BYTES <= LDS_BYTES && Spill<bf16_t>::BYTES <= LDS_BYTES && 2 * TILE_BYTES <= LDS_BYTES, "LDS_BYTES");

__device__ __forceinline__ void clear(acc_t (&acc)[2][2])
{
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
}
#endif
