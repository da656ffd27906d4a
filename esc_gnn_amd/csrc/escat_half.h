// escat_half.h -- element types of the head's operators (fp32 / bf16 / fp16) and loads that need no more than the element's
// own alignment; device-side only, not part of the ABI
#ifndef ESCAT_HALF_H
#define ESCAT_HALF_H
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/escat.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> __device__ __forceinline__ float to_f32(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T from_f32(float x) { return (T)x; }          // to nearest, ties to even

// N consecutive elements, aligned to one element only: gfx950 serves such vector accesses in one instruction
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[N]; };

static inline int escat_type_bytes(int t) { return t == ESCAT_F32 ? 4 : (t == ESCAT_BF16 || t == ESCAT_F16) ? 2 : 0; }
#endif
