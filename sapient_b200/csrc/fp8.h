// Launch wrappers of the operators around 8-bit floating-point rows (fp8_rows.cu, fp8_gemm.cu) and of the token
// distributions (logprobs.cu). All pointers are device pointers; every launcher enqueues on `st`.
//
// An fp8 row of k columns (k % 16 == 0) is k e4m3 values and ceil(k / 128) f32 scales: a value stands for e4m3 x the scale of its
// block of 128 columns (the last one may be shorter). An fp8 weight [n, k] has a scale for every 128 x 128 block.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sp {

constexpr int FP8_BLOCK = 128;
constexpr float FP8_MAX = 448.f;              // largest e4m3 value
constexpr float FP8_MIN_SCALE = 0x1p-100f;    // what a block of zeros keeps; its reciprocal is finite. (Products of two scales are formed in f32: normal from 2^-126 up.)
constexpr int FP8_NORM_MAX_DIM = 32768;
inline int64_t fp8_blocks(int64_t k) { return (k + FP8_BLOCK - 1) / FP8_BLOCK; }

// Rows of x (f32, or bf16 where `bf`) through RMS norm: h = x + residual (null: h = x), sum_out = h (null: not stored; may be x or
// residual), y = h / sqrt(mean(h^2) + eps) * w (null: 1), y to q[rows][dim] and scale[rows][blocks]. The norm takes h in f32 as it is
// before it is rounded to sum_out's type. dim <= FP8_NORM_MAX_DIM.
struct Fp8NormArgs {
    const void* x;
    const void* residual;
    void* sum_out;
    const float* w;
    int64_t ldx, ldr, lds;
    int64_t rows;
    int dim;
    float eps;
    uint8_t* q;
    float* scale;
};
cudaError_t launch_fp8_norm(const Fp8NormArgs& a, bool bf, cudaStream_t st);
// Rows as they are (gated false), or silu(x[0 .. dim)) * x[dim .. 2 dim).
cudaError_t launch_fp8_quant(const void* x, int64_t ldx, int64_t rows, int64_t dim, bool gated, bool bf, uint8_t* q, float* scale, cudaStream_t st);

// Y[m][n] (row stride ldy, f32 or bf16) = X W^T of fp8 rows and an fp8 weight, k % 16 == 0, xq and wq on 16-byte boundaries.
struct Fp8MatArgs {
    const uint8_t* xq;
    const float* xs;   // [m][blocks]
    const uint8_t* wq;
    const float* ws;   // [ceil(n / 128)][blocks]
    void* y;
    int64_t ldy;
    int m, n, k;
    bool bf;
    int* waits;        // WaitFlags of the launch's owner
};
cudaError_t launch_fp8_matmul(const Fp8MatArgs& a, cudaStream_t st);
cudaError_t launch_fp8_dequant(const uint8_t* q, const float* scale, int64_t n, int64_t k, float* out, cudaStream_t st);

// Of each row of logits (f32, or bf16 where `bf`; row stride ld): the log probability of ids[row], the entropy, and the `top` largest
// logits' ids (largest first, the lowest id among equal ones) with their log probabilities. Every output may be null.
constexpr int LOGPROBS_MAX_TOP = 32;
struct LogprobsArgs {
    const void* z;
    int64_t ld, rows;
    int n, top;
    const uint32_t* ids;
    float* logprob;
    float* entropy;
    uint32_t* top_ids;
    float* top_logprobs;
};
cudaError_t launch_logprobs(const LogprobsArgs& a, bool bf, cudaStream_t st);

}  // namespace sp
