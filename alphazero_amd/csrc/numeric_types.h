// Element types of caller-owned matrices (nnb_dtype) and their conversions to and from float32.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/nnb.h"

namespace nnb {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

// A float32 result is rounded to a 16-bit type once, to nearest even, where it is stored.
template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

// One element of an array whose type is only known at run time (bias vectors: a few loads per block).
__device__ __forceinline__ float load_as_f32(const void *p, int type, size_t i) {
    if (type == NNB_F32) return static_cast<const float *>(p)[i];
    if (type == NNB_F16) return (float)static_cast<const f16_t *>(p)[i];
    return (float)static_cast<const bf16_t *>(p)[i];
}

__host__ __device__ constexpr int dtype_bytes(int type) { return type == NNB_F32 ? 4 : 2; }

// f(T{}) for the element type `type`
template <typename F> inline void with_dtype(int type, F &&f) {
    if (type == NNB_F32) f(float{});
    else if (type == NNB_F16) f(f16_t{});
    else f(bf16_t{});
}

}  // namespace nnb
