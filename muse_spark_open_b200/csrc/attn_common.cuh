// Small device functions the attention kernels share: 2^x, warp maxima and E4M3 conversions.
#pragma once

#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace msk {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// Two FP32 lanes in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 y;
    asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
        "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(y.x), "=f"(y.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 y;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(y.x), "=f"(y.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return y;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 y;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(y.x), "=f"(y.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// 2^x for two x <= 64 on the FMA pipe (the special-function unit does 4 per clock and scheduler, which bounds a softmax of
// wide tiles): x = n + f with n whole and |f| <= 1/2 (adding and subtracting 1.5 x 2^23 rounds to whole numbers), 2^f by
// a polynomial of degree 3 fitted for the smallest largest relative error (7.5e-5, a third of FP16's rounding), times 2^n
// put together from its exponent.  Below 2^-126: 2^-126 instead of less.  NaN stays NaN.
__device__ __forceinline__ float2 ex2_poly2(float2 x) {
    x.x = max_nan(x.x, -126.0f), x.y = max_nan(x.y, -126.0f);
    const float2 big = make_float2(12582912.0f, 12582912.0f);
    const float2 t = add2(x, big);
    const float2 n = add2(t, make_float2(-12582912.0f, -12582912.0f));
    const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
    float2 p = fma2(f, make_float2(0.055171702f, 0.055171702f), make_float2(0.2426112f, 0.2426112f));
    p = fma2(p, f, make_float2(0.69326097f, 0.69326097f));
    p = fma2(p, f, make_float2(0.99992806f, 0.99992806f));
    return mul2(p, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}
__device__ __forceinline__ float redux_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ uint32_t f2_to_e4m3x2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float e4m3_to_f(uint32_t byte) {
    __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
    return __half2float(*reinterpret_cast<__half*>(&h));
}
__device__ __forceinline__ float2 e4m3x2_to_f2(uint32_t two) {  // low byte -> x
    __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
    return __half22float2(*reinterpret_cast<__half2*>(&h));
}
__device__ __forceinline__ uint32_t f_to_e4m3(float a) {
    return __nv_cvt_float_to_fp8(a, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t f_to_e5m2(float a) {
    return __nv_cvt_float_to_fp8(a, __NV_SATFINITE, __NV_E5M2);
}
__device__ __forceinline__ bool has_nan(uint4 v) {  // one of 16 E4M3 values is NaN (0x7f with either sign)
    const uint32_t k = 0x7f7f7f7fu, one = 0x01010101u;
    return ((((v.x & k) + one) | ((v.y & k) + one) | ((v.z & k) + one) | ((v.w & k) + one)) & 0x80808080u) != 0;
}

}  // namespace msk
