// Products of fp8 rows with fp8 weights: y[m][n] = sum over blocks b of 128 columns  xs[m][b] ws[n / 128][b] sum_k xq[m][k] wq[n][k].
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "fp8.h"
#include "pdl.cuh"
#include "sp_common.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

__device__ __forceinline__ float e4m3_value(uint8_t b) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}

constexpr int FG_TILE = 64, FG_K = 32;

// A 64 x 64 tile, 4 x 4 values a thread.
__global__ void __launch_bounds__(256) fp8_tile_kernel(const Fp8MatArgs a) {
    __shared__ float xt[FG_K][FG_TILE + 1], wt[FG_K][FG_TILE + 1];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int m0 = blockIdx.y * FG_TILE, n0 = blockIdx.x * FG_TILE;
    const int nb = (a.k + FP8_BLOCK - 1) / FP8_BLOCK;
    pdl_wait();
    pdl_trigger();
    float acc[4][4] = {};
    for (int b = 0; b < nb; ++b) {
        float part[4][4] = {};
        for (int k0 = b * FP8_BLOCK; k0 < min(a.k, (b + 1) * FP8_BLOCK); k0 += FG_K) {
            for (int i = tid; i < FG_TILE * FG_K; i += 256) {
                const int row = i / FG_K, col = i % FG_K, k = k0 + col;
                xt[col][row] = m0 + row < a.m && k < a.k ? e4m3_value(a.xq[(int64_t)(m0 + row) * a.k + k]) : 0.f;
                wt[col][row] = n0 + row < a.n && k < a.k ? e4m3_value(a.wq[(int64_t)(n0 + row) * a.k + k]) : 0.f;
            }
            __syncthreads();
            for (int k = 0; k < FG_K; ++k)
                for (int i = 0; i < 4; ++i)
                    for (int j = 0; j < 4; ++j) part[i][j] = fmaf(xt[k][ty + 16 * i], wt[k][tx + 16 * j], part[i][j]);
            __syncthreads();
        }
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
                if (m < a.m && n < a.n) acc[i][j] = fmaf(part[i][j], a.xs[(int64_t)m * nb + b] * a.ws[(int64_t)(n / FP8_BLOCK) * nb + b], acc[i][j]);
            }
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m >= a.m || n >= a.n) continue;
            if (a.bf) static_cast<__nv_bfloat16*>(a.y)[(int64_t)m * a.ldy + n] = __float2bfloat16_rn(acc[i][j]);
            else static_cast<float*>(a.y)[(int64_t)m * a.ldy + n] = acc[i][j];
        }
}

cudaError_t launch_fp8_matmul(const Fp8MatArgs& a, cudaStream_t st) {
    if (a.m == 0 || a.n == 0) return cudaSuccess;
    const dim3 grid((unsigned)((a.n + FG_TILE - 1) / FG_TILE), (unsigned)((a.m + FG_TILE - 1) / FG_TILE));
    if (a.m < 0 || a.n < 0 || a.k <= 0 || a.k % 16 != 0 || grid.y > 65535) return cudaErrorInvalidValue;
    const cudaError_t e = launch_pdl(fp8_tile_kernel, grid, dim3(256), 0, st, a);
    return e != cudaSuccess ? e : count_launch_and_check();
}

// The values of an fp8 weight, as f32.
__global__ void fp8_dequant_kernel(const uint8_t* q, const float* scale, int64_t n, int64_t k, float* out) {
    const int64_t nb = (k + FP8_BLOCK - 1) / FP8_BLOCK, total = n * k;
    pdl_wait();
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / k, col = i - row * k;
        out[i] = __fmul_rn(e4m3_value(q[i]), scale[row / FP8_BLOCK * nb + col / FP8_BLOCK]);
    }
}

cudaError_t launch_fp8_dequant(const uint8_t* q, const float* scale, int64_t n, int64_t k, float* out, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    const int64_t blocks = std::min<int64_t>((n * k + 255) / 256, (int64_t)device_sm_count() * 8);
    const cudaError_t e = launch_pdl(fp8_dequant_kernel, dim3((unsigned)blocks), dim3(256), 0, st, q, scale, n, k, out);
    return e != cudaSuccess ? e : count_launch_and_check();
}

}  // namespace sp
