// Rows of eight values a thread and their 8-bit form, shared by the kernels that read or write e4m3 rows (fp8_rows.cu, cache_fp8.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fp8.h"

namespace sp {

using bf16 = __nv_bfloat16;

// Eight values as they lie in memory: 16 bytes of bf16 or 32 of f32, passed by once (not kept in L1, where the weights stay).
template <typename T>
struct Raw8 {
    uint4 v[sizeof(T) / 2];
};
__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
template <typename T>
__device__ __forceinline__ Raw8<T> ld8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.v[i] = ld_stream(reinterpret_cast<const uint4*>(p) + i);
    return r;
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f[4 * i] = __uint_as_float(r.v[i].x);
        f[4 * i + 1] = __uint_as_float(r.v[i].y);
        f[4 * i + 2] = __uint_as_float(r.v[i].z);
        f[4 * i + 3] = __uint_as_float(r.v[i].w);
    }
}
__device__ __forceinline__ void unpack8(const Raw8<bf16>& r, float (&f)[8]) {
    const uint32_t u[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void st8(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void st8(bf16* p, const float (&f)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

// The greatest, or NaN where one is (fmaxf would take the others).
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two values an instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void mul2(float& a, float& b, uint64_t by) {
    asm("{\n.reg .b64 v;\nmov.b64 v, {%0, %1};\nmul.rn.f32x2 v, v, %2;\nmov.b64 {%0, %1}, v;\n}\n" : "+f"(a), "+f"(b) : "l"(by));
}
__device__ __forceinline__ void square2(uint64_t& sum, float a, float b) {
    asm("{\n.reg .b64 v;\nmov.b64 v, {%1, %2};\nfma.rn.f32x2 %0, v, v, %0;\n}\n" : "+l"(sum) : "f"(a), "f"(b));
}

__device__ __forceinline__ float rcp_approx(float v) {
    float d;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
    return d;
}

__device__ __forceinline__ float ex2_approx(float v) {
    float d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
    return d;
}
__device__ __forceinline__ float greatest8(const float (&y)[8]) {
    const float m = max_nan(max_nan(fabsf(y[0]), fabsf(y[1]), fabsf(y[2])), max_nan(fabsf(y[3]), fabsf(y[4]), fabsf(y[5])));
    return max_nan(m, fabsf(y[6]), fabsf(y[7]));
}
__device__ __forceinline__ void store8(float (&y)[8], float by, uint8_t* q) {
    const uint64_t by2 = pack2(by, by);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        mul2(y[4 * i], y[4 * i + 1], by2);
        mul2(y[4 * i + 2], y[4 * i + 3], by2);
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * i], y[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * i + 2], y[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
        w[i] = lo | hi << 16;
    }
    *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
}
__device__ __forceinline__ float scale_of(float greatest, float factor) { return max_nan(greatest * factor * (1.f / FP8_MAX), FP8_MIN_SCALE); }

}  // namespace sp
