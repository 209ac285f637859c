// What the kernels share that read fp16 or bf16 rows as pairs in 32-bit words and leave codes.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>

namespace i8tk {

__device__ __forceinline__ float2 widen(const __half*, uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float2 widen(const __nv_bfloat16*, uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// x / N correctly rounded: a quotient from the rounded reciprocal, corrected by its exact remainder (Markstein)
template <int N>
__device__ __forceinline__ float div_by(float x) {
    const float r = 1.0f / N;
    const float q = x * r;
    return fmaf(fmaf(-(float)N, q, x), r, q);
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace i8tk
