// cm_fp8.cuh -- block-scaled 8-bit floating point: the types, checks and conversions shared by
// the quantising kernels (cm_fp8.cu) and the matrix products (cm_fp8_gemm.cu).
//
// A block of 128 values x (1 x 128 for activations, 128 x 128 for weights) is held as
//   A = max(max|x|, 2^-100),  scale = A / F,  q = round(x * (F / A)) in e4m3 (F = 448) or e5m2
//   (F = 57344), to nearest even; x ~ q * scale.
// The floor of A keeps an all-zero block away from 0 / 0; at 2^-100 F / A is finite in both formats.
// The products round a_scale * b_scale to fp32 before it meets a block's sum: from 2^-126 on that is
// one rounding like the others, below it a subnormal number, a multiple of 2^-149, and up to 2^-150
// times the block's unscaled sum is lost (the sum is at most 128 F_a F_b: an error below 2^-125
// for e4m3 by e4m3, 2^-118 for the mixed formats, 2^-111 for e5m2 by e5m2).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cm_common.cuh"

namespace cm {

constexpr uint32_t kFp8Block = 128;

// bytes per element of a CM_T_* type; 0 for an unknown code
inline unsigned type_size(unsigned t) { return t == CM_T_F32 ? 4u : (t == CM_T_Q88 || t == CM_T_F16 || t == CM_T_BF16) ? 2u : 0u; }

// whether (count rows at pitch ld, last row of `cols`) stays far inside the 64-bit address range
inline bool extent_ok(uint64_t count, uint64_t ld, uint64_t cols, unsigned size) {
    return ((unsigned __int128)count * ld + cols) * size < ((unsigned __int128)1 << 60);
}

__device__ __forceinline__ float fp8_largest(uint32_t format) { return format == CM_F8_E4M3 ? 448.0f : 57344.0f; }

// Two floats -> two 8-bit values (`lo` in the low byte), to nearest even; beyond the largest
// finite value the largest finite value, NaN -> NaN.
__device__ __forceinline__ uint32_t cvt_fp8x2(uint32_t format, float lo, float hi) {
    uint16_t r;
    if (format == CM_F8_E4M3) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(int16_t v) { return (float)v * 0.00390625f; }   // Q8.8: exact

// One rounding to the output type: to nearest even, except Q8.8, which narrows as the
// framework's other kernels do (floor to 1/256, saturate; NaN -> 0).
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, int16_t& o) {
    // scaling by 256 is exact (or overflows to the infinity of v's sign, which saturates)
    o = (int16_t)max(-32768, min(32767, __float2int_rd(v * 256.0f)));
}

// Two fp32 values in one 64-bit register pair, and the instructions that work on both.
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) { return pack2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

}  // namespace cm
