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
#include <atomic>

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

// Two values an instruction: these kernels have more instructions than bytes.
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
// Columns c .. c + 7 of a row; the 16 threads of a block of 128 call together, those past the row with zeros and live false. Multiplied
// by reciprocals where the definition divides: the scale is off by 2^-23 of itself at most, the quotient by 2^-22, so that of a million
// values one or two that lie beside a border of the grid fall on its other side; a division takes ten instructions more.
// y is `factor` times the values given: a norm's one factor for the row need not be multiplied into them.
__device__ __forceinline__ void quantise8(float (&y)[8], float factor, bool live, int c, uint8_t* q_row, float* scale_row) {
    float m = max_nan(max_nan(fabsf(y[0]), fabsf(y[1]), fabsf(y[2])), max_nan(fabsf(y[3]), fabsf(y[4]), fabsf(y[5])));
    m = max_nan(m, fabsf(y[6]), fabsf(y[7]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const float scale = max_nan(m * factor * (1.f / FP8_MAX), FP8_MIN_SCALE);
    const float by = factor * rcp_approx(scale);
    if (!live) return;
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
    *reinterpret_cast<uint2*>(q_row + c) = make_uint2(w[0], w[1]);
    if ((c & (FP8_BLOCK - 1)) == 0) scale_row[c / FP8_BLOCK] = scale;
}

// ── RMS norm ──
__host__ __device__ constexpr int fp8_norm_threads(int nc) { return nc == 1 ? 512 : 1024; }
// Blocks an SM is to hold: three of bf16 rows of up to 4096 columns (8192 x 4096 with a residual: two 44.8 us, three 40.9).
__host__ __device__ constexpr int fp8_norm_blocks(int nc, size_t size) { return nc > 1 ? 1 : size == 2 ? 3 : 2; }

// blockDim.x / tpr rows at a time, tpr threads (whole warps) a row with NC pieces of eight columns each; a row's values are on their
// way while the one before is finished.
template <typename T, int NC>
__global__ void __launch_bounds__(fp8_norm_threads(NC), fp8_norm_blocks(NC, sizeof(T))) fp8_norm_kernel(const Fp8NormArgs a, int tpr, float inv_dim) {
    __shared__ float sums[2][32];  // of the warps
    const int tid = threadIdx.x, team = tid / tpr, t = tid - team * tpr, lane = tid & 31;
    const int warps = tpr >> 5, teams = blockDim.x / tpr;
    const T* const x = static_cast<const T*>(a.x);
    const T* const res = static_cast<const T*>(a.residual);
    T* const sum_out = static_cast<T*>(a.sum_out);
    const int nb = (a.dim + FP8_BLOCK - 1) / FP8_BLOCK;
    pdl_wait();
    pdl_trigger();
    Raw8<T> xv[NC], rv[NC];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (t + i * tpr) * 8;
            if (row < a.rows && c < a.dim) {
                xv[i] = ld8(x + row * a.ldx + c);
                if (res) rv[i] = ld8(res + row * a.ldr + c);
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * teams;
    if (NC < 4) fetch((int64_t)blockIdx.x * teams + team);
    int par = 0;
    for (int64_t row0 = (int64_t)blockIdx.x * teams; row0 < a.rows; row0 += step, par ^= 1) {
        const int64_t row = row0 + team;
        const bool have = row < a.rows;
        if (NC == 4) fetch(row);  // (no registers for two rows)
        float h[NC][8];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (t + i * tpr) * 8;
            if (have && c < a.dim) {
                unpack8(xv[i], h[i]);
                if (res) {
                    float r[8];
                    unpack8(rv[i], r);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[i][j] += r[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
            }
        }
        if (NC < 4) fetch(row + step);
        uint64_t squares = 0;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (t + i * tpr) * 8;
            if (sum_out && have && c < a.dim) st8(sum_out + row * a.lds + c, h[i]);
#pragma unroll
            for (int j = 0; j < 8; j += 2) square2(squares, h[i][j], h[i][j + 1]);
        }
        float even, odd;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(even), "=f"(odd) : "l"(squares));
        float ss = warp_sum(even + odd);
        if (warps > 1) {
            if (lane == 0) sums[par][team * warps + (t >> 5)] = ss;
            __syncthreads();
            ss = warp_sum(lane < warps ? sums[par][team * warps + lane] : 0.f);
        }
        const float rms = rsqrtf(fmaf(ss, inv_dim, a.eps));
        uint8_t* const q_row = a.q + row * a.dim;
        float* const scale_row = a.scale + row * nb;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (t + i * tpr) * 8;
            const bool live = have && c < a.dim;
            if (live && a.w) {
                const ulonglong2 w0 = __ldg(reinterpret_cast<const ulonglong2*>(a.w + c)), w1 = __ldg(reinterpret_cast<const ulonglong2*>(a.w + c + 4));
                mul2(h[i][0], h[i][1], w0.x);
                mul2(h[i][2], h[i][3], w0.y);
                mul2(h[i][4], h[i][5], w1.x);
                mul2(h[i][6], h[i][7], w1.y);
            }
            // (past the row zeros, whose norm may be infinite: a factor of 1)
            quantise8(h[i], live ? rms : 1.f, live, c, q_row, scale_row);
        }
    }
}

template <typename T, int NC>
static cudaError_t norm_with(const Fp8NormArgs& a, cudaStream_t st) {
    const int tpr = ((a.dim + 8 * NC - 1) / (8 * NC) + 31) / 32 * 32;
    const int teams = std::max(1, 256 / tpr), threads = teams * tpr;
    // blocks that are there at once, by threads: each takes rows in turn
    static std::atomic<int> resident[SP_MAX_DEVICES][33];
    std::atomic<int>& known = resident[current_device_index()][threads / 32];
    int per_sm = known.load(std::memory_order_relaxed);
    if (per_sm == 0) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fp8_norm_kernel<T, NC>, threads, 0);
        if (e != cudaSuccess) return e;
        known.store(per_sm = std::max(1, per_sm), std::memory_order_relaxed);
    }
    const dim3 grid((unsigned)std::min<int64_t>((a.rows + teams - 1) / teams, (int64_t)device_sm_count() * per_sm));
    const cudaError_t e = launch_pdl(fp8_norm_kernel<T, NC>, grid, dim3((unsigned)threads), 0, st, a, tpr, 1.f / (float)a.dim);
    return e != cudaSuccess ? e : count_launch_and_check();
}

template <typename T>
static cudaError_t norm_of(const Fp8NormArgs& a, cudaStream_t st) {
    return a.dim <= 4096 ? norm_with<T, 1>(a, st) : a.dim <= 16384 ? norm_with<T, 2>(a, st) : norm_with<T, 4>(a, st);
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
    constexpr int R = 2;  // rows a thread has in flight
    for (int64_t row0 = (int64_t)blockIdx.y * R; row0 < rows; row0 += (int64_t)gridDim.y * R) {
        Raw8<T> g[R], u[R];
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (live && row0 + i < rows) {
                const T* const p = x + (row0 + i) * ldx + c;
                g[i] = ld8(p);
                if (GATED) u[i] = ld8(p + dim);
            }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (row0 + i >= rows) break;
            float y[8];
            if (live) {
                unpack8(g[i], y);
                if (GATED) {
                    float v[8];
                    unpack8(u[i], v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = y[j] * rcp_approx(1.f + ex2_approx(y[j] * -1.4426950408889634f)) * v[j];  // errors of a few 2^-22, ahead of a rounding of 2^-4
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = 0.f;
            }
            // (the offset within the block decides who stores the scale: 128 columns before c are whole blocks)
            quantise8(y, 1.f, live, (int)(c & (FP8_BLOCK - 1)), q + (row0 + i) * dim + (c & ~(int64_t)(FP8_BLOCK - 1)), scale + (row0 + i) * nb + c / FP8_BLOCK);
        }
    }
}

cudaError_t launch_fp8_quant(const void* x, int64_t ldx, int64_t rows, int64_t dim, bool gated, bool bf, uint8_t* q, float* scale, cudaStream_t st) {
    if (rows == 0) return cudaSuccess;
    const int64_t tiles = (dim + 1023) / 1024;
    if (dim <= 0 || dim % 16 != 0 || tiles > INT32_MAX) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)tiles, (unsigned)std::min<int64_t>((rows + 1) / 2, 65535)), block(128);
    cudaError_t e;
    if (bf) e = gated ? launch_pdl(fp8_quant_kernel<bf16, true>, grid, block, 0, st, (const bf16*)x, ldx, rows, dim, q, scale)
                      : launch_pdl(fp8_quant_kernel<bf16, false>, grid, block, 0, st, (const bf16*)x, ldx, rows, dim, q, scale);
    else e = gated ? launch_pdl(fp8_quant_kernel<float, true>, grid, block, 0, st, (const float*)x, ldx, rows, dim, q, scale)
                   : launch_pdl(fp8_quant_kernel<float, false>, grid, block, 0, st, (const float*)x, ldx, rows, dim, q, scale);
    return e != cudaSuccess ? e : count_launch_and_check();
}

}  // namespace sp
