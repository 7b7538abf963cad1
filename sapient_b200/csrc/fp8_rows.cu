// Rows to 8-bit floating point, a scale for every 128 columns, through what produces them: RMS norm with the residual's addition,
// SwiGLU, or nothing.
//
//   scale_b = max(max |y| over the block / 448, 2^-100),   q = e4m3(y / scale_b), to nearest even
//
// A thread holds eight columns, so a block of 128 is half a warp and its maximum four shuffles. A NaN or an infinity in a block makes
// its scale one too (the maximum lets NaN through), so that whatever reads the block sees it. Bytes bound both kernels: each value is
// read once and kept in registers until its row's norm is known.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "fp8.h"
#include "pdl.cuh"
#include "sp_common.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

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

// The greater of two, or NaN where one is (fmaxf would take the other).
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Columns c .. c + 7 of a row; the 16 threads of a block of 128 call together, those past the row with zeros and live false. The
// quotient is taken with the scale's reciprocal (two roundings of 2^-24 where the division has one: of a million values, one or two
// beside a border of the grid fall on its other side).
__device__ __forceinline__ void quantise8(const float (&y)[8], bool live, int c, uint8_t* q_row, float* scale_row) {
    float m = max_nan(max_nan(max_nan(fabsf(y[0]), fabsf(y[1])), max_nan(fabsf(y[2]), fabsf(y[3]))),
                      max_nan(max_nan(fabsf(y[4]), fabsf(y[5])), max_nan(fabsf(y[6]), fabsf(y[7]))));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const float scale = max_nan(__fdiv_rn(m, FP8_MAX), FP8_MIN_SCALE);
    const float inv = __frcp_rn(scale);
    if (!live) return;
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * i] * inv, y[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * i + 2] * inv, y[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
        w[i] = lo | hi << 16;
    }
    *reinterpret_cast<uint2*>(q_row + c) = make_uint2(w[0], w[1]);
    if ((c & (FP8_BLOCK - 1)) == 0) scale_row[c / FP8_BLOCK] = scale;
}

// ── RMS norm ──
// blockDim.x / tpr rows at a time, tpr threads (whole warps) a row with NC pieces of eight columns each.
template <typename T, int NC>
__global__ void __launch_bounds__(1024) fp8_norm_kernel(const Fp8NormArgs a, int tpr) {
    __shared__ float sums[2][32];
    const int tid = threadIdx.x, team = tid / tpr, t = tid - team * tpr, warp = tid >> 5, lane = tid & 31;
    const int warps = tpr >> 5, teams = blockDim.x / tpr, warp0 = team * warps;
    const T* const x = static_cast<const T*>(a.x);
    const T* const res = static_cast<const T*>(a.residual);
    T* const sum_out = static_cast<T*>(a.sum_out);
    const int64_t nb = (a.dim + FP8_BLOCK - 1) / FP8_BLOCK;
    pdl_wait();
    pdl_trigger();
    int par = 0;
    for (int64_t row0 = (int64_t)blockIdx.x * teams; row0 < a.rows; row0 += (int64_t)gridDim.x * teams, par ^= 1) {
        const int64_t row = row0 + team;
        const bool have = row < a.rows;
        float h[NC][8];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (t + i * tpr) * 8;
            if (have && c < a.dim) {
                unpack8(ld8(x + row * a.ldx + c), h[i]);
                if (res) {
                    float r[8];
                    unpack8(ld8(res + row * a.ldr + c), r);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[i][j] += r[j];
                }
                if (sum_out) st8(sum_out + row * a.lds + c, h[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(h[i][j], h[i][j], ss);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
            }
        }
        ss = warp_sum(ss);
        if (warps > 1) {
            if (lane == 0) sums[par][warp] = ss;
            __syncthreads();
            ss = 0.f;
            for (int w = 0; w < warps; ++w) ss += sums[par][warp0 + w];
        }
        const float rms = rsqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (t + i * tpr) * 8;
            const bool live = have && c < a.dim;
            float y[8];
            if (live && a.w) {
                const float4 w0 = __ldg(reinterpret_cast<const float4*>(a.w + c)), w1 = __ldg(reinterpret_cast<const float4*>(a.w + c + 4));
                const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = h[i][j] * rms * w[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = live ? h[i][j] * rms : 0.f;  // (past the row, where the norm may be infinite: zeros)
            }
            quantise8(y, live, c, a.q + row * a.dim, a.scale + row * nb);
        }
    }
}

template <typename T>
static cudaError_t norm_of(const Fp8NormArgs& a, cudaStream_t st) {
    const int nc = a.dim <= 4096 ? 1 : a.dim <= 8192 ? 2 : 4;
    const int tpr = ((a.dim + 8 * nc - 1) / (8 * nc) + 31) / 32 * 32;
    const int teams = std::max(1, 256 / tpr);
    const int64_t groups = (a.rows + teams - 1) / teams;
    const int per_sm = std::max(1, 2048 / (teams * tpr));
    const dim3 grid((unsigned)std::min<int64_t>(groups, (int64_t)device_sm_count() * per_sm)), block((unsigned)(teams * tpr));
    cudaError_t e;
    if (nc == 1) e = launch_pdl(fp8_norm_kernel<T, 1>, grid, block, 0, st, a, tpr);
    else if (nc == 2) e = launch_pdl(fp8_norm_kernel<T, 2>, grid, block, 0, st, a, tpr);
    else e = launch_pdl(fp8_norm_kernel<T, 4>, grid, block, 0, st, a, tpr);
    return e != cudaSuccess ? e : count_launch_and_check();
}

cudaError_t launch_fp8_norm(const Fp8NormArgs& a, bool bf, cudaStream_t st) {
    if (a.rows == 0) return cudaSuccess;
    if (a.dim <= 0 || a.dim % 16 != 0 || a.dim > FP8_NORM_MAX_DIM) return cudaErrorInvalidValue;
    return bf ? norm_of<bf16>(a, st) : norm_of<float>(a, st);
}

// ── SwiGLU, or rows as they are ──
template <typename T, bool GATED>
__global__ void __launch_bounds__(128) fp8_quant_kernel(const T* x, int64_t ldx, int64_t rows, int64_t dim, uint8_t* q, float* scale) {
    const int64_t c = ((int64_t)blockIdx.x * 128 + threadIdx.x) * 8, nb = (dim + FP8_BLOCK - 1) / FP8_BLOCK;
    const bool live = c < dim;
    pdl_wait();
    pdl_trigger();
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        float y[8];
        if (live) {
            const T* const p = x + row * ldx + c;
            unpack8(ld8(p), y);
            if (GATED) {
                float u[8];
                unpack8(ld8(p + dim), u);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = __fdividef(y[j], 1.f + __expf(-y[j])) * u[j];  // errors of a few 2^-22, ahead of a rounding of 2^-4
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = 0.f;
        }
        // (the offset within the block decides who stores the scale: 128 columns before c are whole blocks)
        quantise8(y, live, (int)(c & (FP8_BLOCK - 1)), q + row * dim + (c & ~(int64_t)(FP8_BLOCK - 1)), scale + row * nb + c / FP8_BLOCK);
    }
}

cudaError_t launch_fp8_quant(const void* x, int64_t ldx, int64_t rows, int64_t dim, bool gated, bool bf, uint8_t* q, float* scale, cudaStream_t st) {
    if (rows == 0) return cudaSuccess;
    const int64_t tiles = (dim + 1023) / 1024;
    if (dim <= 0 || dim % 16 != 0 || tiles > INT32_MAX) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)tiles, (unsigned)std::min<int64_t>(rows, 65535)), block(128);
    cudaError_t e;
    if (bf) e = gated ? launch_pdl(fp8_quant_kernel<bf16, true>, grid, block, 0, st, (const bf16*)x, ldx, rows, dim, q, scale)
                      : launch_pdl(fp8_quant_kernel<bf16, false>, grid, block, 0, st, (const bf16*)x, ldx, rows, dim, q, scale);
    else e = gated ? launch_pdl(fp8_quant_kernel<float, true>, grid, block, 0, st, (const float*)x, ldx, rows, dim, q, scale)
                   : launch_pdl(fp8_quant_kernel<float, false>, grid, block, 0, st, (const float*)x, ldx, rows, dim, q, scale);
    return e != cudaSuccess ? e : count_launch_and_check();
}

}  // namespace sp
