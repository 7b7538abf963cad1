// Rows to 8-bit floating point, a scale for every 128 columns, through what produces them: RMS norm with the residual's addition,
// SwiGLU, or nothing.
//
//   scale_b = max(max |y| over the block / 448, 2^-100),   q = e4m3(y / scale_b), to nearest even
//
// A thread holds eight columns, so a block of 128 is half a warp and its maximum four shuffles. A NaN or an infinity in a block makes
// its scale one too (the maximum lets NaN through), so that whatever reads the block sees it. Each value is read once and kept in
// registers until its row's norm is known. Times here are of one kernel launched back to back by a small program; calls from Python on
// inputs that change, with their outputs not in L2, take what stands behind the semicolon. Bytes bound SwiGLU (4096 x 14336 bf16: 46.9 us, 45.2 at
// 6.54 TB/s; 50.8 to 53.7) and norms with a residual (8192 x 4096 bf16: 39.9 us, 36.1; 40.7 to 43.0). Norms without one (23.1 us, 15.6; 23.5)
// fill nothing: 2.5 of 4 instructions a cycle, 31 % of DRAM, 46 % of the warps, since registers leave room for two blocks an SM. A few rows
// take a launch and two latencies, 2.5 to 3.3 us.
// Rows of more than 4096 columns spill: in f32 with a residual 88 bytes a thread (4096 x 8192: 90.8 us for 66.9 of bytes, calls), of more
// than 16384 columns 404 (2048 x 16400: 143.2 us for 66.9; bf16 172 bytes, 98.6 us for 36.1).
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

// Eight columns of a row; the 16 threads of a block of 128 call together, those past the row with zeros and live false. Multiplied by
// reciprocals where the definition divides: the quotient is off by 2^-22 of itself at most, so that of a million values one or two that
// lie beside a border of the grid fall on its other side; a division takes ten instructions more. The scale has the roundings of two
// products and of 1 / 448, 3 x 2^-24 together (rows as they are: 2^-23), a norm's the error of its rsqrtf as well.
// y is `factor` (up to FACTOR_MAX) times the values given: a norm's one factor for the row need not be multiplied into them.
constexpr float FACTOR_MAX = 0x1p27f;  // times the reciprocal of the smallest scale, 2^100, it is finite
__device__ __forceinline__ void quantise8(float (&y)[8], float factor, bool live, int lane, uint8_t* q, float* scale_to) {
    float m = greatest8(y);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const float scale = scale_of(m, factor);
    if (!live) return;
    store8(y, factor * rcp_approx(scale), q);
    if ((lane & 15) == 0) *scale_to = scale;
}
// Two times eight columns, of two blocks: half of the 16 threads finish the one's maximum and scale, half the other's. The first thread
// stores the one's scale, the ninth the other's, where they are given a place.
__device__ __forceinline__ void quantise8x2(float (&y0)[8], float (&y1)[8], float factor0, float factor1, bool live0, bool live1, int lane, uint8_t* q0, uint8_t* q1,
                                            float* scale_to0, float* scale_to1) {
    const float m0 = greatest8(y0), m1 = greatest8(y1);
    const bool second = lane & 8;
    float m = max_nan(second ? m1 : m0, __shfl_xor_sync(0xFFFFFFFFu, second ? m0 : m1, 8));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const float factor = second ? factor1 : factor0, scale = scale_of(m, factor), by = factor * rcp_approx(scale), other = __shfl_xor_sync(0xFFFFFFFFu, by, 8);
    if (live0) store8(y0, second ? other : by, q0);
    if (live1) store8(y1, second ? by : other, q1);
    if ((lane & 7) == 0) {
        float* const to = second ? scale_to1 : scale_to0;
        if (to) *to = scale;
    }
}

// ── RMS norm ──
__host__ __device__ constexpr int fp8_norm_threads(int nc) { return nc == 1 ? 512 : 1024; }
// Blocks an SM is to hold: three of single bf16 rows of up to 4096 columns (8192 x 4096 with a residual: two 44.8 us, three 40.9).
__host__ __device__ constexpr int fp8_norm_blocks(int nc, int r, size_t size) { return nc > 1 ? 1 : size == 2 && r == 1 ? 3 : 2; }

// Teams of tpr threads (whole warps) take R rows at a time, NC pieces of eight columns of each a thread; the values of the next rows are
// on their way while these are finished. TINY: eps lets a row's norm fall below 1 / FACTOR_MAX.
template <typename T, int NC, int R, bool RES, bool TINY>
__global__ void __launch_bounds__(fp8_norm_threads(NC), fp8_norm_blocks(NC, R, sizeof(T))) fp8_norm_kernel(const Fp8NormArgs a, int tpr, float inv_dim) {
    static_assert(R == 1 || NC == 1, "sums of two rows: 16 warps at most");
    constexpr int P = NC * R;
    constexpr bool PAIRS = P == 2 && !RES;              // two pieces' scales together: 4096 x 8192 bf16 32.0 us, 26.5; with a residual 43.5 us, 49.5
    constexpr bool BRANCH = NC == 1 && sizeof(T) == 4;  // a branch around the residual's loads, for what the compiler then keeps in registers:
                                                        // 600 x 4096 f32 9.0 us, 8.3
    __shared__ float sums[2][32];  // of the warps
    const int tid = threadIdx.x, team = tid / tpr, t = tid - team * tpr, lane = tid & 31;
    const int warps = tpr >> 5, teams = blockDim.x / tpr;
    const T* const x = static_cast<const T*>(a.x);
    const T* const res = static_cast<const T*>(a.residual);
    T* const sum_out = static_cast<T*>(a.sum_out);
    const int nb = (a.dim + FP8_BLOCK - 1) / FP8_BLOCK;
    pdl_wait();
    pdl_trigger();
    Raw8<T> xv[P], rv[RES ? P : 1];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (t + i % NC * tpr) * 8;
            if (row + i / NC < a.rows && c < a.dim) {
                xv[i] = ld8(x + (row + i / NC) * a.ldx + c);
                if (RES && (!BRANCH || res)) rv[i] = ld8(res + (row + i / NC) * a.ldr + c);
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * teams * R;
    if (NC < 4) fetch(((int64_t)blockIdx.x * teams + team) * R);
    int par = 0;
    for (int64_t row0 = (int64_t)blockIdx.x * teams * R; row0 < a.rows; row0 += step, par ^= 1) {
        const int64_t row = row0 + team * R;
        if (NC == 4) fetch(row);  // (no registers for two rows)
        float h[P][8];
        bool live[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            live[i] = row + i / NC < a.rows && (t + i % NC * tpr) * 8 < a.dim;
            if (live[i]) {
                unpack8(xv[i], h[i]);
                if (RES && (!BRANCH || res)) {
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
        float ss[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            uint64_t squares = 0;
#pragma unroll
            for (int i = r * NC; i < (r + 1) * NC; ++i) {
                if (sum_out && live[i]) st8(sum_out + (row + r) * a.lds + (t + i % NC * tpr) * 8, h[i]);
#pragma unroll
                for (int j = 0; j < 8; j += 2) square2(squares, h[i][j], h[i][j + 1]);
            }
            float even, odd;
            asm("mov.b64 {%0, %1}, %2;" : "=f"(even), "=f"(odd) : "l"(squares));
            ss[r] = even + odd;
        }
        float rms[R];
        if constexpr (R == 1) {
            float s = warp_sum(ss[0]);
            if (warps > 1) {
                if (lane == 0) sums[par][team * warps + (t >> 5)] = s;
                __syncthreads();
                s = warp_sum(lane < warps ? sums[par][team * warps + lane] : 0.f);
            }
            rms[0] = rsqrtf(fmaf(s, inv_dim, a.eps));
        } else {  // half of a warp's threads finish the one row's sum, half the other's
            const bool second = lane & 16;
            float s = (second ? ss[1] : ss[0]) + __shfl_xor_sync(0xFFFFFFFFu, second ? ss[0] : ss[1], 16);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            if (warps > 1) {
                const int half = second ? 16 : 0;
                if ((lane & 15) == 0) sums[par][half + team * warps + (t >> 5)] = s;
                __syncthreads();
                s = (lane & 15) < warps ? sums[par][half + team * warps + (lane & 15)] : 0.f;
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            }
            const float mine = rsqrtf(fmaf(s, inv_dim, a.eps)), other = __shfl_xor_sync(0xFFFFFFFFu, mine, 16);
            rms[0] = second ? other : mine;
            rms[1] = second ? mine : other;
        }
        if constexpr (TINY) {
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (rms[r] > FACTOR_MAX) {
#pragma unroll
                    for (int i = r * NC; i < (r + 1) * NC; ++i)
#pragma unroll
                        for (int j = 0; j < 8; ++j) h[i][j] *= rms[r];
                    rms[r] = 1.f;
                }
        }
        uint8_t* q[P];
        float* scale[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (t + i % NC * tpr) * 8;
            q[i] = a.q + (row + i / NC) * a.dim + c;
            scale[i] = a.scale + (row + i / NC) * nb + c / FP8_BLOCK;
        }
        if (a.w) {
            ulonglong2 w0, w1;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int c = (t + i % NC * tpr) * 8;
                if (c < a.dim) {
                    if (i < NC) w0 = __ldg(reinterpret_cast<const ulonglong2*>(a.w + c)), w1 = __ldg(reinterpret_cast<const ulonglong2*>(a.w + c + 4));
                    mul2(h[i][0], h[i][1], w0.x);
                    mul2(h[i][2], h[i][3], w0.y);
                    mul2(h[i][4], h[i][5], w1.x);
                    mul2(h[i][6], h[i][7], w1.y);
                }
            }
        }
        if constexpr (PAIRS) {
            // the first thread of a block decides for the ninth, which stores the second scale
            const bool there = row + 1 / NC < a.rows && (t - (lane & 15) + 1 % NC * tpr) * 8 < a.dim;
            quantise8x2(h[0], h[1], rms[0], rms[R - 1], live[0], live[1], lane, q[0], q[1], live[0] ? scale[0] : nullptr, there ? scale[1] : nullptr);
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) quantise8(h[i], rms[i / NC], live[i], lane, q[i], scale[i]);
        }
    }
}

template <typename T, int NC, int R, bool RES, bool TINY>
static cudaError_t norm_kind(const Fp8NormArgs& a, cudaStream_t st) {
    const int tpr = ((a.dim + 8 * NC - 1) / (8 * NC) + 31) / 32 * 32;
    const int teams = std::max(1, 256 / tpr), threads = teams * tpr;
    // blocks that are there at once, by threads: each takes rows in turn
    static std::atomic<int> resident[SP_MAX_DEVICES][33];
    std::atomic<int>& known = resident[current_device_index()][threads / 32];
    int per_sm = known.load(std::memory_order_relaxed);
    if (per_sm == 0) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fp8_norm_kernel<T, NC, R, RES, TINY>, threads, 0);
        if (e != cudaSuccess) return e;
        known.store(per_sm = std::max(1, per_sm), std::memory_order_relaxed);
    }
    const dim3 grid((unsigned)std::min<int64_t>((a.rows + teams * R - 1) / (teams * R), (int64_t)device_sm_count() * per_sm));
    const cudaError_t e = launch_pdl(fp8_norm_kernel<T, NC, R, RES, TINY>, grid, dim3((unsigned)threads), 0, st, a, tpr, 1.f / (float)a.dim);
    return e != cudaSuccess ? e : count_launch_and_check();
}

template <typename T, int NC, int R, bool RES>
static cudaError_t norm_with(const Fp8NormArgs& a, cudaStream_t st) {
    // (by what the host knows: with the row's norm looked at in every call, 8192 x 4096 bf16 with a residual takes 43.9 us for 43.0)
    return a.eps >= 1.f / (FACTOR_MAX * FACTOR_MAX) ? norm_kind<T, NC, R, RES, false>(a, st) : norm_kind<T, NC, R, RES, true>(a, st);
}

template <typename T, bool RES>
static cudaError_t norm_of(const Fp8NormArgs& a, cudaStream_t st) {
    if (a.dim > 4096) return a.dim <= 16384 ? norm_with<T, 2, 1, RES>(a, st) : norm_with<T, 4, 1, RES>(a, st);
    return norm_with<T, 1, RES ? 1 : 2, RES>(a, st);  // two rows share their reductions where bytes leave time for those: 8192 x 4096 bf16, one row 27.9 us, two 23.1; with a residual 39.9 and 40.5
}

cudaError_t launch_fp8_norm(const Fp8NormArgs& a, bool bf, cudaStream_t st) {
    if (a.rows == 0) return cudaSuccess;
    if (a.dim <= 0 || a.dim % 16 != 0 || a.dim > FP8_NORM_MAX_DIM) return cudaErrorInvalidValue;
    if (bf) return a.residual ? norm_of<bf16, true>(a, st) : norm_of<bf16, false>(a, st);
    return a.residual ? norm_of<float, true>(a, st) : norm_of<float, false>(a, st);
}

// ── SwiGLU, or rows as they are ──
// A thread has two rows on their way and finishes one after the other (together, with their scales in one reduction: 48.1 us for 46.9).
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
                    for (int j = 0; j < 8; ++j) y[j] = y[j] * rcp_approx(1.f + ex2_approx(y[j] * -1.4426950408889634f)) * v[j];  // off by |g| 2^-23 and a few 2^-22 of itself, ahead of a rounding of 2^-4; zero where it is below 2^-126
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = 0.f;
            }
            quantise8(y, 1.f, live, threadIdx.x & 31, q + (row0 + i) * dim + c, scale + (row0 + i) * nb + c / FP8_BLOCK);
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
