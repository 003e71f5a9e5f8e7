// Shared pieces of the FP8 operators: e4m3 values with one FP32 scale per row
// and 128 columns (activations) or per 128 x 128 block (weights).
//
// A group of 128 values x_i is held as q_i = e4m3(x_i * 448 / a), s = a / 448,
// with a = max(max |x_i|, 1e-10); x_i is read back as q_i * s.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace lrb {
namespace fp8 {

constexpr int kGroup = 128;       // values that share a scale
constexpr float kTop = 448.0f;    // the largest e4m3 value
constexpr float kTiny = 1e-10f;   // a group's maximum counts as at least this

__host__ __device__ constexpr int groups(int n) { return (n + kGroup - 1) / kGroup; }

// 16 bytes that a kernel before this one may have written.  Kernels of a stream
// overlap here (programmatic dependent launch), so such data changes while this
// kernel is already running, before its griddepcontrol.wait: the read-only path
// (ld.global.nc, __ldg), which is for data that nobody writes until the kernel
// ends, is not for it.  ld_once: for what is read once.
__device__ __forceinline__ uint4 ld_once(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 ld_again(const void *p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// The larger of two magnitudes, NaN if either is: a group that holds a NaN
// must not come out as numbers.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// One group's divisor.  q = x * 448 / a is computed as (1.75 x 2^-8) / (a 2^-16):
// both factors of 1.75 = 7/4 and the powers of two are exact for a BF16 x, and
// neither side can overflow.  The quotient starts as t * (1 / d) and takes one
// residual step, q + (t - q d) / d with the residual exact in an FMA.  A value
// that lies on a border of two e4m3 values is representable, so the step makes
// it exact and the tie rounds to even as it would after an exact division; any
// other quotient of BF16 x and a is at least 2^-13 away from a border, far more
// than the last error.  Three instructions a value instead of a full division.
// A NaN maximum gives NaN; an infinite one gives 1/d = 0 and a NaN residual, so
// a group that holds an infinity is NaN throughout as well.
struct Divisor {
    float d, r;
    __device__ __forceinline__ explicit Divisor(float a) : d(a * 0x1p-16f), r(1.0f / (a * 0x1p-16f)) {}
    __device__ __forceinline__ float operator()(float x) const {
        const float t = x * (1.75f * 0x1p-8f);
        const float q = t * r;
        return fmaf(fmaf(-q, d, t), r, q);
    }
};

__device__ __forceinline__ float scale_of(float a) { return __fdiv_rn(a, kTop); }

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t pack4(const Divisor &f, float a, float b, float c, float d) {
    return pack2(f(a), f(b)) | (pack2(f(c), f(d)) << 16);
}

// Two FP32 values as packed BF16 in one conversion (two separate ones and a
// merge run at an eighth of the rate).
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Sixteen e4m3 values as FP16 (exact).
__device__ __forceinline__ void halves16(uint4 v, uint16_t (&f)[16]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] & 0xffff), __NV_E4M3);
        const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] >> 16), __NV_E4M3);
        f[4 * i] = a.x;
        f[4 * i + 1] = a.y;
        f[4 * i + 2] = b.x;
        f[4 * i + 3] = b.y;
    }
}
// acc + x * y with FP16 factors in one FP32 FMA (the product is exact).
__device__ __forceinline__ float fma_f16(uint16_t x, uint16_t y, float acc) {
    asm("fma.rn.f32.f16 %0, %1, %2, %0;" : "+f"(acc) : "h"(x), "h"(y));
    return acc;
}
// dot(16 e4m3 weights, 16 FP16 activations) in FP32.
__device__ __forceinline__ float dot16(uint4 w, const uint16_t (&x)[16]) {
    uint16_t f[16];
    halves16(w, f);
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        a = fma_f16(f[i], x[i], a);
        b = fma_f16(f[i + 1], x[i + 1], b);
    }
    return a + b;
}

}  // namespace fp8
}  // namespace lrb
