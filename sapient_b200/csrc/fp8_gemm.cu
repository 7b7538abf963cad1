// Products of fp8 rows with fp8 weights: y[m][n] = sum over blocks b of 128 columns  xs[m][b] ws[n / 128][b] sum_k xq[m][k] wq[n][k].
//
// The tensor cores add up a block's 128 columns (products of e4m3 values are exact in f32); what they have is scaled and added in f32
// registers, since no two blocks of a row need have the same scale. That is 1 multiplication of a thread for 128 of the tensor cores,
// and each block's sums pass through registers: the accumulators in tensor memory are a ring, not a result.
//   up to 16 rows, but for large     fp8_gemv_kernel    mma.sync, 16 weight rows a block
//   up to 128 rows, or long K        fp8_stream_kernel  tcgen05, 128 weight rows are the lanes, K shared by a cluster
//   few tiles                        fp8_lone_kernel    tcgen05, 128 activation rows are the lanes, one tile a block
//   many                             fp8_wide_kernel    the same, tiles of 256 weight rows in rounds, by one SM or a pair
// Every sum has one order, which depends on the sizes, on whether the operands start on 32 bytes (up to 16 rows) and on the number of SMs.
// gemv_takes and way_of choose, with the times of both sides. Times are of kernels launched back to back, where nothing else is said.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "fp8.h"
#include "kernels.h"
#include "pdl.cuh"
#include "plan_common.cuh"
#include "sp_common.cuh"
#include "tc5_ptx.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

__device__ __forceinline__ float e4m3_value(uint8_t b) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}

__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(tc5_smem_u32(bar)), "r"(arrivals) : "memory");
}

// Arrives on a barrier of the cluster without waiting for the thread's own loads and stores: what is handed over is tensor memory, which
// fences of its own order. With the default, a release, an arrival waits for the scales on their way (4096 x 14336 x 4096: 358 us for 217).
__device__ __forceinline__ void arrive_relaxed(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}

// e4m3 x e4m3 -> f32, both operands K-major.
__host__ __device__ constexpr uint32_t fp8_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void fp8_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void store(const Fp8MatArgs& p, int m, int n, float f) {
    if (p.bf) static_cast<bf16*>(p.y)[(int64_t)m * p.ldy + n] = __float2bfloat16_rn(f);
    else static_cast<float*>(p.y)[(int64_t)m * p.ldy + n] = f;
}

// ── Up to 16 rows ──
// A block owns 16 weight rows; its warps take blocks of 128 columns in turn and add up in shared memory. Columns may be multiplied in
// any order: a lane's 32 bytes of a row are eight 4-byte operands of mma.sync, and the activations are read alike, so that nothing is
// rearranged. No tensor memory, barriers or descriptors to set up, which is most of a small product's time: 1 x 4096 x 4096 takes 5.3 us
// from cold weights, of which their bytes are 2.6 (3.7 from L2); the rest is the launch, the first loads' latency and the warps' sum.
// Four lanes load 128 bytes of a row at once: with 64 the L1's tags bound it (6.2 us, from L2 too). Few registers, so that blocks of the
// next product start beside the last ones of this: four blocks of columns ahead instead of two took 6.5 us.
constexpr int FV_ROWS = 16;

// 32 bytes, in one load where they start on 32; weights are not kept in L1.
template <bool ALIGNED>
__device__ __forceinline__ void fv_weights(const uint8_t* p, uint4 (&v)[2]) {
    if constexpr (ALIGNED)
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                     : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z), "=r"(v[1].w) : "l"(p) : "memory");
    else
#pragma unroll
        for (int i = 0; i < 2; ++i)
            asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v[i].x), "=r"(v[i].y), "=r"(v[i].z), "=r"(v[i].w) : "l"(p + 16 * i) : "memory");
}
template <bool ALIGNED>
__device__ __forceinline__ void fv_rows(const uint8_t* p, uint4 (&v)[2]) {
    if constexpr (ALIGNED)
        asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                     : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z), "=r"(v[1].w) : "l"(p) : "memory");
    else
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = *reinterpret_cast<const uint4*>(p + 16 * i);
}
__device__ __forceinline__ void fv_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: activation rows / 8. AHEAD: blocks of 128 columns that a warp has on their way. ALIGNED: rows start on 32 bytes.
template <int NT, int FV_WARPS, int AHEAD, bool ALIGNED>
__global__ void __launch_bounds__(32 * FV_WARPS, 16 / FV_WARPS) fp8_gemv_kernel(const Fp8MatArgs p) {
    __shared__ float part[FV_WARPS][8 * NT][FV_ROWS + 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * FV_ROWS, blocks = (p.k + FP8_BLOCK - 1) / FP8_BLOCK;
    const uint8_t* const w0 = p.wq + (int64_t)min(n0 + g, p.n - 1) * p.k + 32 * t;
    const uint8_t* const w1 = p.wq + (int64_t)min(n0 + 8 + g, p.n - 1) * p.k + 32 * t;
    const float* const ws = p.ws + (int64_t)(n0 / FP8_BLOCK) * blocks;
    struct Stage {
        uint4 w[2][2], x[NT][2];  // [rows 0 to 7, 8 to 15][16 columns]
        float xs[NT][2], ws;
    } stage[AHEAD];
    auto load = [&](Stage& s, int b) {
        const int c = b * FP8_BLOCK;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const int left = p.k - c - 32 * t;  // columns from the lane's first on: 32, or of the last block 16 or fewer
        if (left >= 32) {
            fv_weights<ALIGNED>(w0 + c, s.w[0]);
            fv_weights<ALIGNED>(w1 + c, s.w[1]);
        } else {
            const bool half = !ALIGNED && left > 0;
            s.w[0][0] = half ? *reinterpret_cast<const uint4*>(w0 + c) : zero;
            s.w[1][0] = half ? *reinterpret_cast<const uint4*>(w1 + c) : zero;
            s.w[0][1] = s.w[1][1] = zero;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint8_t* const x = p.xq + (int64_t)(8 * j + g) * p.k + c + 32 * t;
            s.x[j][0] = s.x[j][1] = zero;
            if (8 * j + g < p.m) {
                if (left >= 32) fv_rows<ALIGNED>(x, s.x[j]);
                else if (!ALIGNED && left > 0) s.x[j][0] = *reinterpret_cast<const uint4*>(x);
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int m = 8 * j + 2 * t + i;
                s.xs[j][i] = m < p.m ? __ldg(p.xs + (int64_t)m * blocks + b) : 0.f;
            }
        s.ws = __ldg(ws + b);
    };
    pdl_wait();
    pdl_trigger();
    float acc[NT][4] = {};
#pragma unroll
    for (int d = 0; d < AHEAD; ++d)
        if (warp + FV_WARPS * d < blocks) load(stage[d], warp + FV_WARPS * d);
    for (int b0 = warp; b0 < blocks; b0 += FV_WARPS * AHEAD) {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
            const int b = b0 + FV_WARPS * d;
            if (b >= blocks) break;
            Stage& s = stage[d];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    fv_mma(c, s.w[0][h].x, s.w[1][h].x, s.w[0][h].y, s.w[1][h].y, s.x[j][h].x, s.x[j][h].y);
                    fv_mma(c, s.w[0][h].z, s.w[1][h].z, s.w[0][h].w, s.w[1][h].w, s.x[j][h].z, s.x[j][h].w);
                }
                const float s0 = s.xs[j][0] * s.ws, s1 = s.xs[j][1] * s.ws;
                acc[j][0] = fmaf(c[0], s0, acc[j][0]);
                acc[j][1] = fmaf(c[1], s1, acc[j][1]);
                acc[j][2] = fmaf(c[2], s0, acc[j][2]);
                acc[j][3] = fmaf(c[3], s1, acc[j][3]);
            }
            if (b + FV_WARPS * AHEAD < blocks) load(s, b + FV_WARPS * AHEAD);
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[warp][8 * j + 2 * t + (i & 1)][g + 8 * (i >> 1)] = acc[j][i];
    __syncthreads();
    const int row = tid & (FV_ROWS - 1);
    for (int m = tid / FV_ROWS; m < p.m; m += 32 * FV_WARPS / FV_ROWS)
        if (n0 + row < p.n) {
            float f = 0.f;
#pragma unroll
            for (int w = 0; w < FV_WARPS; ++w) f += part[w][m][row];
            store(p, m, n0 + row, f);
        }
}

// ── Few rows: a stream of weights ──
// The weights' bytes bound it (13 x 28672 x 4096: 22.7 us, 5.2 TB/s): they fill the tile's 128 lanes whatever the number of activation
// rows, which are the products' N of 16 to 128. Two blocks an SM keep 200 KB on their way. Where tiles are fewer than SMs, the blocks of a
// cluster take parts of K and add them up through distributed shared memory in the parts' order (32 x 1024 x 8192: 8 parts 8.6 us).
constexpr int FS_BM = 128;                     // weight rows of a tile
constexpr int FS_THREADS = 192;                // MMA warp, TMA warp, four drain warps
constexpr int FS_W_BYTES = FS_BM * FP8_BLOCK;  // of a stage
constexpr int FS_SMEM = 108 * 1024;            // per block, two of which share an SM
constexpr int FS_MAX_STAGES = 6, FS_MAX_PARTS = 8;

struct Fp8StreamArgs {
    Fp8MatArgs p;
    int parts, stages, x_rows;  // x_rows: of activations that a copy brings
};

// BN: activation rows of a tile.
template <int BN>
__global__ void __launch_bounds__(FS_THREADS, 2) fp8_stream_kernel(const Fp8StreamArgs a, const __grid_constant__ CUtensorMap map_w,
                                                               const __grid_constant__ CUtensorMap map_x) {
    constexpr int BUFS = BN >= 128 ? 2 : 4, COLS = BUFS * BN, STAGE = FS_W_BYTES + BN * FP8_BLOCK;
    extern __shared__ uint8_t fs_smem_raw[];
    __shared__ __align__(8) uint64_t full[FS_MAX_STAGES], empty[FS_MAX_STAGES], sum_full[BUFS], sum_empty[BUFS];
    __shared__ __align__(16) float scales[2][BN];
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const Fp8MatArgs& p = a.p;
    const int n0 = blockIdx.x * FS_BM, r0 = blockIdx.y * BN, rows = min(BN, p.m - r0);
    const int blocks = (p.k + FP8_BLOCK - 1) / FP8_BLOCK, part = blockIdx.z;
    const int b0 = (int)((int64_t)part * blocks / a.parts), count = (int)((int64_t)(part + 1) * blocks / a.parts) - b0;
    uint8_t* const smem = fs_smem_raw + ((1024u - (tc5_smem_u32(fs_smem_raw) & 1023u)) & 1023u);
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc5_smem_u32(&tmem_slot)), "n"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (tid == 32) {
        tc5_prefetch_map(&map_w);
        tc5_prefetch_map(&map_x);
        for (int i = 0; i < a.stages; ++i) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], 1);
        }
        for (int i = 0; i < BUFS; ++i) {
            bar_init(&sum_full[i], 1);
            bar_init(&sum_empty[i], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    pdl_trigger();
    bool ok = true;
    float* const partial = reinterpret_cast<float*>(smem);  // [BN][128], once the ring has drained
    if (warp == 0) {
        const bool leader = tc5_elect();
        const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        const uint32_t idesc = fp8_idesc(FS_BM, BN);
        const uint64_t ad0 = tc5_desc(tc5_smem_u32(smem));
        for (int c = 0, st = 0, u = 0; c < count; ++c) {
            const int buf = c % BUFS, turn = c / BUFS;
            if (turn > 0) ok = tc5_wait(&sum_empty[buf], (uint32_t)((turn - 1) & 1));
            ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&full[st], (uint32_t)(u & 1)));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const uint64_t ad = ad0 + (uint64_t)((uint32_t)(st * STAGE) >> 4), bd = ad + (FS_W_BYTES >> 4);
            if (leader) {
#pragma unroll
                for (int i = 0; i < FP8_BLOCK / 32; ++i) fp8_mma(tm + (uint32_t)(buf * BN), ad + 2u * i, bd + 2u * i, idesc, i > 0);
                tc5_commit(&empty[st]);
                tc5_commit(&sum_full[buf]);
            }
            __syncwarp();
            if (++st == a.stages) { st = 0; ++u; }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int issued = 0;
            for (int c = 0, st = 0, u = 0; c < count; ++c, ++st) {
                if (st == a.stages) { st = 0; ++u; }
                if (u > 0) ok = tc5_wait(&empty[st], (uint32_t)((u - 1) & 1));
                if (!ok) break;
                const uint32_t bar = tc5_smem_u32(&full[st]), dst = tc5_smem_u32(smem + st * STAGE);
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(FS_W_BYTES + a.x_rows * FP8_BLOCK) : "memory");
                tc5_tma_2d(dst, &map_w, (b0 + c) * FP8_BLOCK, n0, bar);
                tc5_tma_2d(dst + FS_W_BYTES, &map_x, (b0 + c) * FP8_BLOCK, r0, bar);
                issued = c + 1;
            }
            // nothing is in flight towards this block when it goes on to the end: copies, or the arrivals that follow the last products
            for (int c = max(0, issued - a.stages); c < issued; ++c) {
                uint64_t* const bars = ok ? empty : full;
                ok = tc5_wait(&bars[c % a.stages], (uint32_t)((c / a.stages) & 1)) && ok;
            }
        }
        __syncwarp();
    } else {
        const int q4 = warp & 3, n = n0 + 32 * q4 + lane, t = tid - 64;
        const uint32_t lanes = tmem + ((uint32_t)(32 * q4) << 16);
        // the thread whose number is an activation row's brings that row's scale times the weights', a block ahead of its use
        const bool brings = t < BN && t < rows;
        const float* const xs = p.xs + (int64_t)(r0 + (brings ? t : 0)) * blocks + b0;
        const float* const ws = p.ws + (int64_t)(n0 / FP8_BLOCK) * blocks + b0;
        float acc[BN];
#pragma unroll
        for (int j = 0; j < BN; ++j) acc[j] = 0.f;
        float xv = brings && count > 0 ? xs[0] : 0.f, wv = count > 0 ? ws[0] : 0.f;
        for (int c = 0; c < count; ++c) {
            const int buf = c % BUFS;
            if (t < BN) scales[c & 1][t] = xv * wv;
            if (c + 1 < count) {
                if (brings) xv = xs[c + 1];
                wv = ws[c + 1];
            }
            ok = __all_sync(0xFFFFFFFFu, tc5_wait(&sum_full[buf], (uint32_t)((c / BUFS) & 1)));
            // (the one barrier a block of 128 columns: its scales are there, and those of the one before have been read)
            int all_ok;
            asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %1, 0;\nbarrier.cta.red.and.pred q, 1, 128, p;\nselp.b32 %0, 1, 0, q;\n}\n" : "=r"(all_ok) : "r"((int)ok) : "memory");
            ok = all_ok != 0;
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll
            for (int j0 = 0; j0 < BN; j0 += 16) {
                uint32_t v[16];
                tc5_ld16(lanes + (uint32_t)(buf * BN + j0), v);
                asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                if (j0 + 16 == BN) {
                    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                    if (lane == 0) arrive_relaxed(tc5_smem_u32(&sum_empty[buf]));
                }
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 s = *reinterpret_cast<const float4*>(&scales[c & 1][j0 + j]);
                    acc[j0 + j] = fmaf(__uint_as_float(v[j]), s.x, acc[j0 + j]);
                    acc[j0 + j + 1] = fmaf(__uint_as_float(v[j + 1]), s.y, acc[j0 + j + 1]);
                    acc[j0 + j + 2] = fmaf(__uint_as_float(v[j + 2]), s.z, acc[j0 + j + 2]);
                    acc[j0 + j + 3] = fmaf(__uint_as_float(v[j + 3]), s.w, acc[j0 + j + 3]);
                }
            }
        }
        if (a.parts == 1) {
            if (ok && n < p.n) {
#pragma unroll
                for (int j = 0; j < BN; ++j)
                    if (j < rows) store(p, r0 + j, n, acc[j]);
            }
        } else {
            if (ok) {
#pragma unroll
                for (int j = 0; j < BN; ++j) partial[j * FS_BM + 32 * q4 + lane] = acc[j];
            }
            cluster_sync();
            // the cluster's blocks share out the rows, eight on their way at a time; each adds its rows' parts in order
            const uint32_t mine = tc5_smem_u32(partial + 32 * q4 + lane);
            constexpr int NR = 8;
            for (int j0 = part; j0 < rows && n < p.n; j0 += NR * a.parts) {
                float f[NR] = {};
                for (int o = 0; o < a.parts; ++o) {
                    const uint32_t peer = peer_smem(mine, o);
                    float v[NR];
#pragma unroll
                    for (int i = 0; i < NR; ++i) v[i] = ld_peer(peer + (uint32_t)(min(j0 + i * a.parts, rows - 1) * FS_BM * 4));
#pragma unroll
                    for (int i = 0; i < NR; ++i) f[i] += v[i];
                }
#pragma unroll
                for (int i = 0; i < NR; ++i)
                    if (ok && j0 + i * a.parts < rows) store(p, r0 + j0 + i * a.parts, n, f[i]);
            }
        }
    }
    if (a.parts > 1) {
        if (warp < 2) { __syncwarp(); cluster_sync(); }  // the service warps' share of the first barrier
        cluster_sync();                                  // nobody leaves while its parts are being read
    }
    if (!ok) report_wait(p.waits, WAIT_FP8);
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "n"(COLS) : "memory");
}

// Two values a step.
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t v0, uint32_t v1, uint64_t s) {
    asm("{\n.reg .b64 v;\nmov.b64 v, {%1, %2};\nfma.rn.f32x2 %0, v, %3, %0;\n}\n" : "+l"(acc) : "r"(v0), "r"(v1), "l"(s));
}
__device__ __forceinline__ uint64_t pair2(float2 f) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(f.x), "f"(f.y));
    return v;
}
__device__ __forceinline__ float2 both(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}

constexpr int FP_DRAINS = 8;
constexpr int FP_OUT = 2 * 32 * 128;  // of a drain warp's part of the result on its way out

// 64 columns of bf16 or 32 of f32, 128 bytes of a lane's row, to shared memory: 16-byte pieces lie at piece ^ (row & 7), as TMA's 128-byte
// swizzle has them, which keeps both directions free of bank conflicts.
template <typename T>
__device__ __forceinline__ void put_line(uint8_t* out, const uint64_t* acc, int lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t u[4];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 f = both(acc[2 * i + j]);
                u[2 * j] = __float_as_uint(f.x);
                u[2 * j + 1] = __float_as_uint(f.y);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = both(acc[4 * i + j]);
                const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
                u[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        *reinterpret_cast<uint4*>(out + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}
// What put_line left of 32 rows, to rows of y that start anywhere: a row an instruction, so that what it writes lies together, in words of
// the alignment that the row has. Out: T's columns of y, or 32 of f32 that become bf16.
template <typename T, typename Out>
__device__ __forceinline__ void store_rows(void* y, int64_t ldy, int rows, int columns, const uint8_t* out, int lane) {
    auto word = [&](int row) { return *reinterpret_cast<const uint32_t*>(out + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4); };
    Out* at = static_cast<Out*>(y);
    if constexpr (sizeof(T) == 4) {
#pragma unroll 8
        for (int row = 0; row < 32; ++row, at += ldy) {
            const float f = __uint_as_float(word(row));
            if (row < rows && lane < columns) at[lane] = (Out)f;
        }
    } else {
        const int last = min(columns, 64);
        const bool odd0 = (reinterpret_cast<uintptr_t>(y) & 2) != 0, odd1 = odd0 != ((ldy & 1) != 0);  // whether rows 0, 2, ... and 1, 3, ... start between words
        uint16_t* to = static_cast<uint16_t*>(y) + 2 * lane;
        if (!odd0 && !odd1) {
#pragma unroll 8
            for (int row = 0; row < 32; ++row, to += ldy) {
                const uint32_t v = word(row);
                if (row < rows && 2 * lane + 1 < last) *reinterpret_cast<uint32_t*>(to) = v;
            }
        } else {
#pragma unroll 8
            for (int row = 0; row < 32; ++row, to += ldy) {
                const int odd = (row & 1) ? odd1 : odd0;
                const uint32_t v = word(row), next = __shfl_down_sync(0xFFFFFFFFu, v, 1);
                if (row < rows && 2 * lane + odd + 1 < last) *reinterpret_cast<uint32_t*>(to + odd) = __funnelshift_r(v, next, 16 * odd);
            }
        }
        // a row a lane: the first column of rows that start between words, the last one that is half a word
        const int odd = (lane & 1) ? odd1 : odd0;
        auto one = [&](int c) { static_cast<uint16_t*>(y)[lane * ldy + c] = *reinterpret_cast<const uint16_t*>(out + lane * 128 + (((c >> 3) ^ (lane & 7)) << 4) + (c & 7) * 2); };
        if (lane < rows && odd && last > 0) one(0);
        if (lane < rows && last > odd && ((last - odd) & 1)) one(last - 1);
    }
}
// The same where rows start on 16 bytes (ALIGNED): four rows an instruction. Kernels have either as a parameter: the two together cost
// the aligned way 2 %. (755 x 30158 x 1728 bf16 with the aligned way's pieces stored an element at a time: 87 us for 45.)
template <typename T, bool ALIGNED, typename Out = T>
__device__ __forceinline__ void store_lines(const Fp8MatArgs& p, const uint8_t* out, int r0, int n0, int lane) {
    constexpr int PER = 16 / sizeof(T);
    if constexpr (!ALIGNED) {
        store_rows<T, Out>(static_cast<Out*>(p.y) + (int64_t)r0 * p.ldy + n0, p.ldy, p.m - r0, p.n - n0, out, lane);
        return;
    }
    const int piece = lane & 7, n = n0 + piece * PER;
    Out* at = static_cast<Out*>(p.y) + (int64_t)(r0 + (lane >> 3)) * p.ldy + n;
#pragma unroll
    for (int i = 0; i < 8; ++i, at += 4 * p.ldy) {
        const int row = 4 * i + (lane >> 3);
        const uint4 v = *reinterpret_cast<const uint4*>(out + row * 128 + ((piece ^ (row & 7)) << 4));
        if (r0 + row >= p.m) continue;
        const T* const e = reinterpret_cast<const T*>(&v);
        if (n + PER <= p.n) {
            if constexpr (sizeof(Out) < sizeof(T)) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(e[0], e[1]), hi = __floats2bfloat162_rn(e[2], e[3]);
                *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            } else {
                *reinterpret_cast<uint4*>(at) = v;
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (n + j < p.n) at[j] = (Out)e[j];
        }
    }
}
// 32 columns that put_line left in f32, to y of either type.
template <bool ALIGNED>
__device__ __forceinline__ void store_f32_lines(const Fp8MatArgs& p, const uint8_t* out, int r0, int n0, int lane) {
    if (p.bf) store_lines<float, ALIGNED, bf16>(p, out, r0, n0, lane);
    else store_lines<float, ALIGNED>(p, out, r0, n0, lane);
}

// Whether all drain warps' waits were in time; a barrier between them.
__device__ __forceinline__ bool drains_agree(bool ok) {
    int all;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %1, 0;\nbarrier.cta.red.and.pred q, 1, %2, p;\nselp.b32 %0, 1, 0, q;\n}\n" : "=r"(all) : "r"((int)ok), "n"(32 * FP_DRAINS) : "memory");
    return all != 0;
}

// ── Many rows: activation rows are the lanes ──
// A tile of 128 G activation rows x 256 weight rows, by one block or by a pair (G = 2: each block has 128 activation rows in its tensor
// memory and half of the weight rows in its shared memory), or by one block 128 x 128 or 128 x 64 of a product that does not fill the SMs.
//
// The wide kernel's two halves of 128 weight rows have sums and drain warps of their own, two of each: while one is drained three are
// with the tensor cores. 4096 x 14336 x 4096: 205 to 209 us in a burst, 2.3 PFLOP/s, at the 1.5 GHz to which the power limit takes the
// clock (168 without drains); calls without a pause on inputs that change 237 to 244, 2.0 PFLOP/s. The tensor cores always have products to do, but a half takes 417 cycles for 256 of products (335 without drains):
// drains read the tensor memory that products add into. Slower: products of 256 columns with two sums (220 us), 16 drain warps (238),
// results by TMA (232), columns of tiles first (221). No effect: more stages, a second warp that issues products.
constexpr int FP_BN = 256;
constexpr int FP_FIRST_DRAIN = 4;               // warp 0 issues products, warp 1 copies, warps 2 and 3 store results of drains
constexpr int FP_THREADS = 32 * (FP_FIRST_DRAIN + FP_DRAINS);
constexpr int FP_COLS = 2 * FP_BN;
__host__ __device__ constexpr int fp_stage(int g) { return (128 + FP_BN / g) * FP8_BLOCK; }  // a block's share of a stage
__host__ __device__ constexpr int fp_stages(int g) { return g == 2 ? 4 : 3; }
__host__ __device__ constexpr int fp_smem(int g) { return fp_stages(g) * fp_stage(g) + FP_DRAINS * FP_OUT; }
template <int G>
__device__ __forceinline__ void wide_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t accumulate) {
    constexpr uint32_t idesc = fp8_idesc(128 * G, FP_BN / 2);
    if constexpr (G == 1) {
        fp8_mma(d_tmem, adesc, bdesc, idesc, accumulate);
    } else {
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
            "}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}
// Arrives on the barrier at this place in the tile's blocks once the products issued so far are done.
template <int G>
__device__ __forceinline__ void wide_commit(uint64_t* bar) {
    if constexpr (G == 1) tc5_commit(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(tc5_smem_u32(bar)), "h"((uint16_t)3)
                     : "memory");
}
template <int G>
__device__ __forceinline__ void wide_tma(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (G == 1) tc5_tma_2d(dst, map, x, y, bar);
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst), "l"(map),
            "r"(x), "r"(y), "r"(bar)
            : "memory");
}
// 32 consecutive tensor-memory columns of the warp's 32 lanes.
__device__ __forceinline__ void wide_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

// Adds 32 P columns of a sum, scaled, to the lane's; `freed` hears when they have been read.
template <int P>
__device__ __forceinline__ void drain_add(uint32_t taddr, float f, uint64_t (&acc)[16 * P], uint32_t freed, int lane) {
    const uint64_t scale = pair2(make_float2(f, f));
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    // (a piece is on its way while the one before is added)
    uint32_t v[2][32];
    wide_ld32(taddr, v[0]);
#pragma unroll
    for (int i = 0; i < P; ++i) {
        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
        if (i + 1 < P) {
            wide_ld32(taddr + (uint32_t)(32 * (i + 1)), v[(i + 1) & 1]);
        } else {
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            if (lane == 0) arrive_relaxed(freed);
        }
#pragma unroll
        for (int j = 0; j < 32; j += 2) fma2(acc[16 * i + j / 2], v[i & 1][j], v[i & 1][j + 1], scale);
    }
}

struct Fp8WideArgs {
    Fp8MatArgs p;
    int row_tiles, x_rows;        // x_rows: of activations that a copy brings
    int whole, items;             // items: tiles up to `whole`, halves of the following tiles (128 of their weight rows) after them
    bool handed;                  // results leave by warps of their own while the drains go on with the next tile
};
template <int G>
struct Fp8Item {
    int r0, n0, first, last;  // activation and weight rows of the tile, halves
    __device__ __forceinline__ Fp8Item(const Fp8WideArgs& a, int i) {
        const int over = i - a.whole, tile = over < 0 ? i : a.whole + (over >> 1);
        first = over < 0 ? 0 : over & 1;
        last = over < 0 ? 1 : first;
        r0 = tile % a.row_tiles * (128 * G);
        n0 = tile / a.row_tiles * FP_BN;
    }
};

// ALIGNED: rows of y start on 16 bytes.
template <int G, bool ALIGNED>
__global__ void __launch_bounds__(FP_THREADS, 1) fp8_wide_kernel(const Fp8WideArgs a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
    constexpr int STAGES = fp_stages(G), STAGE = fp_stage(G), HALF = FP_BN / 2 / G;  // HALF: weight rows of half a tile in this block
    extern __shared__ uint8_t fp_smem_raw[];
    __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], sum_full[4], sum_empty[4], out_full[FP_DRAINS], out_empty[FP_DRAINS];
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const Fp8MatArgs& p = a.p;
    const int rank = G == 2 ? blockIdx.x & 1 : 0, team = blockIdx.x / G, teams = gridDim.x / G;
    const int blocks = (p.k + FP8_BLOCK - 1) / FP8_BLOCK;
    uint8_t* const smem = fp_smem_raw + ((1024u - (tc5_smem_u32(fp_smem_raw) & 1023u)) & 1023u);
    if (warp == 0) {
        if constexpr (G == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc5_smem_u32(&tmem_slot)), "n"(FP_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc5_smem_u32(&tmem_slot)), "n"(FP_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
        }
    }
    if (tid == 32) {
        tc5_prefetch_map(&map_w);
        tc5_prefetch_map(&map_x);
        for (int i = 0; i < STAGES; ++i) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            bar_init(&sum_full[i], 1);
            bar_init(&sum_empty[i], G * FP_DRAINS / 2);
        }
        for (int i = 0; i < FP_DRAINS; ++i) {
            bar_init(&out_full[i], 32);
            bar_init(&out_empty[i], 32);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (G == 2) cluster_sync();  // both blocks' barriers are there
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    pdl_trigger();
    bool ok = true;
    if (warp < FP_FIRST_DRAIN) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");  // 128 x 56 + 256 x 224 = 384 x 168
        if (warp == 0) {
            if (rank == 0) {
                const bool leader = tc5_elect();
                const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
                const uint64_t ad0 = tc5_desc(tc5_smem_u32(smem));
                int st = 0, u = 0, c = 0, item = team;  // stage and its turn; blocks of 128 columns so far, over all items
                for (; ok && item < a.whole; item += teams)
                    for (int b = 0; b < blocks; ++b, ++c) {
                        const int buf = c & 1, turn = c >> 1;
                        ok = __all_sync(0xFFFFFFFFu, tc5_wait(&full[st], (uint32_t)(u & 1)));
                        const uint64_t ad = ad0 + (uint64_t)((uint32_t)(st * STAGE) >> 4), bd = ad + ((128 * FP8_BLOCK) >> 4);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (turn > 0) ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&sum_empty[2 * buf + h], (uint32_t)((turn - 1) & 1)));
                            if (!ok) break;
                            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                            if (leader) {
#pragma unroll
                                for (int i = 0; i < FP8_BLOCK / 32; ++i)
                                    wide_mma<G>(tm + (uint32_t)(buf * FP_BN + 128 * h), ad + 2u * i, bd + (uint32_t)(h * ((HALF * FP8_BLOCK) >> 4)) + 2u * i, i > 0);
                                if (h) wide_commit<G>(&empty[st]);
                                wide_commit<G>(&sum_full[2 * buf + h]);
                            }
                        }
                        if (!ok) break;
                        __syncwarp();
                        if (++st == STAGES) { st = 0; ++u; }
                    }
                for (; ok && item < a.items; item += teams) {
                    const int h = (item - a.whole) & 1;
                    for (int b = 0; b < blocks; ++b, ++c) {
                        const int buf = c & 1, turn = c >> 1;
                        ok = __all_sync(0xFFFFFFFFu, tc5_wait(&full[st], (uint32_t)(u & 1)));
                        if (turn > 0) ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&sum_empty[2 * buf + h], (uint32_t)((turn - 1) & 1)));
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                        const uint64_t ad = ad0 + (uint64_t)((uint32_t)(st * STAGE) >> 4), bd = ad + (uint32_t)(((128 + HALF * h) * FP8_BLOCK) >> 4);
                        if (leader) {
#pragma unroll
                            for (int i = 0; i < FP8_BLOCK / 32; ++i) wide_mma<G>(tm + (uint32_t)(buf * FP_BN + 128 * h), ad + 2u * i, bd + 2u * i, i > 0);
                            wide_commit<G>(&empty[st]);
                            wide_commit<G>(&sum_full[2 * buf + h]);
                        }
                        __syncwarp();
                        if (++st == STAGES) { st = 0; ++u; }
                    }
                }
            }
        } else if (warp == 1) {
            if (lane == 0) {
                int st = 0, u = 0, issued = 0;
                for (int item = team; ok && item < a.items; item += teams) {
                    const Fp8Item<G> it(a, item);
                    const int r0 = it.r0 + 128 * rank, n0 = it.n0 + HALF * rank, bytes = a.x_rows * FP8_BLOCK + (it.last - it.first + 1) * HALF * FP8_BLOCK;
                    for (int b = 0; b < blocks; ++b) {
                        if (u > 0) ok = tc5_wait(&empty[st], (uint32_t)((u - 1) & 1));
                        if (!ok) break;
                        const uint32_t here = tc5_smem_u32(&full[st]), bar = G == 1 ? here : peer_smem(here, 0), dst = tc5_smem_u32(smem + st * STAGE);
                        // (the other block's bytes may be there before they are expected: the phase waits for this arrival)
                        if (rank == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(here), "r"(G * bytes) : "memory");
                        wide_tma<G>(dst, &map_x, b * FP8_BLOCK, r0, bar);
                        if (it.first == 0) wide_tma<G>(dst + 128 * FP8_BLOCK, &map_w, b * FP8_BLOCK, n0, bar);
                        if (it.last == 1) wide_tma<G>(dst + (128 + HALF) * FP8_BLOCK, &map_w, b * FP8_BLOCK, n0 + 128, bar);
                        ++issued;
                        if (++st == STAGES) { st = 0; ++u; }
                    }
                }
                // nothing is in flight towards this block when it goes on to the end: copies, or the arrivals that follow the last products
                for (int c = max(0, issued - STAGES); c < issued; ++c)
                    if (ok) ok = tc5_wait(&empty[c % STAGES], (uint32_t)((c / STAGES) & 1));
                    else if (rank == 0) tc5_wait(&full[c % STAGES], (uint32_t)((c / STAGES) & 1));
            }
            __syncwarp();
        } else {
            // stores: warp 2 for the drains of one half, warp 3 for the other's; a team's last item is its drains' own
            const int half = warp - 2;
            int turn = 0;
            for (int item = team; ok && a.handed && item + teams < a.items; item += teams) {
                const Fp8Item<G> it(a, item);
                for (int q = 0; ok && q < 4; ++q) {
                    const int d = 4 * half + q, q4 = (FP_FIRST_DRAIN + d) & 3, r0 = it.r0 + 128 * rank + 32 * q4, n0 = it.n0 + 128 * half;
                    const uint8_t* const out = smem + STAGES * STAGE + d * FP_OUT;
                    ok = __all_sync(0xFFFFFFFFu, tc5_wait(&out_full[d], (uint32_t)(turn & 1)));
                    if (!ok) break;
                    for (int i = 0; i < 2; ++i) {
                        if (p.bf) store_lines<bf16, ALIGNED>(p, out + 4096 * i, r0, n0 + 64 * i, lane);
                        else store_lines<float, ALIGNED>(p, out + 4096 * i, r0, n0 + 64 + 32 * i, lane);
                    }
                    tc5_arrive(&out_empty[d]);
                }
                ++turn;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;\n");
        const int q4 = warp & 3, drain = warp - FP_FIRST_DRAIN, half = drain >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(32 * q4) << 16) + (uint32_t)(128 * half);
        uint8_t* const out = smem + STAGES * STAGE + drain * FP_OUT;
        const uint32_t freed[2] = {peer_smem(tc5_smem_u32(&sum_empty[half]), 0), peer_smem(tc5_smem_u32(&sum_empty[2 + half]), 0)};
        // 64 columns of the warp's rows that are in `out` (f32: in both its lines), to y
        auto store_out = [&](int r0, int n0) {
            __syncwarp();
            if (p.bf) {
                store_lines<bf16, ALIGNED>(p, out, r0, n0, lane);
            } else {
                store_lines<float, ALIGNED>(p, out, r0, n0, lane);
                store_lines<float, ALIGNED>(p, out + 4096, r0, n0 + 32, lane);
            }
        };
        int c = 0, turns = 0;
        for (int item = team; ok && item < a.items; item += teams) {
            const Fp8Item<G> it(a, item);
            if (half < it.first || half > it.last) continue;
            const int r0 = it.r0 + 128 * rank + 32 * q4, n0 = it.n0 + 128 * half;
            const float* const xs = p.xs + (int64_t)min(r0 + lane, p.m - 1) * blocks;
            const float* const ws = p.ws + (int64_t)(min(n0, p.n - 1) / FP8_BLOCK) * blocks;
            uint64_t acc[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) acc[j] = 0;
            float xv = xs[0], wv = ws[0];
            for (int b = 0; b < blocks; ++b, ++c) {
                const int buf = c & 1;
                const float f = xv * wv;
                uint64_t scale;
                asm("mov.b64 %0, {%1, %1};" : "=l"(scale) : "f"(f));
                if (b + 1 < blocks) { xv = xs[b + 1]; wv = ws[b + 1]; }
                ok = __all_sync(0xFFFFFFFFu, tc5_wait(&sum_full[2 * buf + half], (uint32_t)((c >> 1) & 1)));
                if (!ok) break;
                // (as drain_add, which costs this loop spills and a tenth of its time)
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                uint32_t v[2][32];
                wide_ld32(lanes + (uint32_t)(buf * FP_BN), v[0]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                    if (i < 3) {
                        wide_ld32(lanes + (uint32_t)(buf * FP_BN + 32 * (i + 1)), v[(i + 1) & 1]);
                    } else {
                        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                        if (lane == 0) arrive_relaxed(freed[buf]);
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 2) fma2(acc[16 * i + j / 2], v[i & 1][j], v[i & 1][j + 1], scale);
                }
            }
            if (!ok) break;
            // of long products bf16 results leave by the storing warp, of f32 ones, twice the bytes, half
            const bool handed = a.handed && item + teams < a.items;
            if (turns > 0) ok = __all_sync(0xFFFFFFFFu, tc5_wait(&out_empty[drain], (uint32_t)((turns - 1) & 1)));
            if (!ok) break;
            __syncwarp();
            if (p.bf) {
                put_line<bf16>(out, acc, lane);
                put_line<bf16>(out + 4096, acc + 32, lane);
            } else {
                put_line<float>(out, acc, lane);
                put_line<float>(out + 4096, acc + 16, lane);
                store_out(r0, n0);
                __syncwarp();
                put_line<float>(out, acc + 32, lane);
                put_line<float>(out + 4096, acc + 48, lane);
            }
            if (handed) {
                tc5_arrive(&out_full[drain]);
                ++turns;
            } else if (p.bf) {
                __syncwarp();
                store_lines<bf16, ALIGNED>(p, out, r0, n0, lane);
                store_lines<bf16, ALIGNED>(p, out + 4096, r0, n0 + 64, lane);
            } else {
                store_out(r0, n0 + 64);
            }
        }
    }
    if (!ok) report_wait(p.waits, WAIT_FP8);
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (G == 2) cluster_sync();  // neither block leaves before the other's products, copies and arrivals are through
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    if (warp == 0) {
        if constexpr (G == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "n"(FP_COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "n"(FP_COLS) : "memory");
    }
}

// A tile of 128 activation rows x W weight rows a block, no more tiles than SMs: what counts is how many bytes are on their way and how
// soon the tensor cores go on. All of shared memory is stages; there are four accumulators, and the two groups of drain warps take
// blocks of 128 columns in turn and add up at the end (W = 128 spills 80 bytes a thread). An SM takes in about 60 bytes a cycle, which bounds it: 128 x 4096 x 4096 10.6 us
// with tiles of 64 weight rows (13.2 with one warp that issues products and one that copies, 12.1 with two and one, two and two here).
// Of tiles of 64 two or four blocks of a cluster may share K; they add up through distributed shared memory, each its share of the rows.
__host__ __device__ constexpr int lone_stage(int w) { return (128 + w) * FP8_BLOCK; }
__host__ __device__ constexpr int lone_stages(int w) { return 210 * 1024 / lone_stage(w); }

// A cluster's blocks share out the rows that put_line left in each, in f32: of a warp's 32 each block adds up its own, the parts in order,
// eight values of a lane on their way at a time, and stores them.
template <int LINES>
__device__ __forceinline__ void add_parts(const Fp8MatArgs& p, const uint8_t* out, int parts, int part, int r0, int c0, int lane) {
    const uint32_t at = tc5_smem_u32(out);
    const int rows = 32 / parts;
    for (int i0 = 0; i0 < rows * LINES; i0 += 8) {
        float f[8] = {};
        for (int o = 0; o < parts; ++o) {
            const uint32_t peer = peer_smem(at, o);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int u = min(i0 + i, rows * LINES - 1), line = u / rows, row = part * rows + u - line * rows;
                v[i] = ld_peer(peer + (uint32_t)(4096 * line + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] += v[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int u = i0 + i, line = u / rows, row = r0 + part * rows + u - line * rows, n = c0 + 32 * line + lane;
            if (u < rows * LINES && row < p.m && n < p.n) store(p, row, n, f[i]);
        }
    }
}

template <int W, bool ALIGNED>
__global__ void __launch_bounds__(FP_THREADS, 1) fp8_lone_kernel(const Fp8MatArgs p, int k_parts, int x_rows, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
    constexpr int STAGES = lone_stages(W), STAGE = lone_stage(W), COLS = 4 * W;
    extern __shared__ uint8_t fp_smem_raw[];
    __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], sum_full[4], sum_empty[4];
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const int n0 = blockIdx.x * W, m0 = blockIdx.y * 128;
    const int all = (p.k + FP8_BLOCK - 1) / FP8_BLOCK, parts = W == 64 ? k_parts : 1, part = W == 64 ? blockIdx.z : 0;
    const int first = (int)((int64_t)part * all / parts), blocks = (int)((int64_t)(part + 1) * all / parts) - first;
    uint8_t* const smem = fp_smem_raw + ((1024u - (tc5_smem_u32(fp_smem_raw) & 1023u)) & 1023u);
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc5_smem_u32(&tmem_slot)), "n"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (tid == 32) {
        tc5_prefetch_map(&map_w);
        tc5_prefetch_map(&map_x);
        for (int i = 0; i < STAGES; ++i) {
            bar_init(&full[i], 2);
            bar_init(&empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            bar_init(&sum_full[i], 1);
            bar_init(&sum_empty[i], FP_DRAINS / 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    pdl_trigger();
    bool ok = true;
    if (warp < FP_FIRST_DRAIN) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");  // 128 x 56 + 256 x 224 = 384 x 168
        if (warp == 0 || warp == 2) {
            // blocks of 128 columns in turn: of a warp that issues them all, waits and instructions take 540 cycles a block, its products 192
            const bool leader = tc5_elect();
            const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
            const uint64_t ad0 = tc5_desc(tc5_smem_u32(smem));
            int st = warp >> 1, u = 0;
            for (int b = warp >> 1; b < blocks; b += 2) {
                const int q = b & 3, turn = b >> 2;
                ok = __all_sync(0xFFFFFFFFu, tc5_wait(&full[st], (uint32_t)(u & 1)));
                if (turn > 0) ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&sum_empty[q], (uint32_t)((turn - 1) & 1)));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const uint64_t ad = ad0 + (uint64_t)((uint32_t)(st * STAGE) >> 4), bd = ad + ((128 * FP8_BLOCK) >> 4);
                if (leader) {
#pragma unroll
                    for (int i = 0; i < FP8_BLOCK / 32; ++i) fp8_mma(tm + (uint32_t)(q * W), ad + 2u * i, bd + 2u * i, fp8_idesc(128, W), i > 0);
                    tc5_commit(&empty[st]);
                    tc5_commit(&sum_full[q]);
                }
                __syncwarp();
                if ((st += 2) >= STAGES) { st -= STAGES; ++u; }
            }
        } else {
            // warp 1 copies activations, warp 3 weights
            if (lane == 0) {
                const bool x = warp == 1;
                const CUtensorMap* const map = x ? &map_x : &map_w;
                const int row = x ? m0 : n0, bytes = (x ? x_rows : W) * FP8_BLOCK, place = x ? 0 : 128 * FP8_BLOCK;
                int issued = 0;
                for (int st = 0, u = 0; issued < blocks; ++issued) {
                    if (u > 0) ok = tc5_wait(&empty[st], (uint32_t)((u - 1) & 1));
                    if (!ok) break;
                    const uint32_t bar = tc5_smem_u32(&full[st]);
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
                    tc5_tma_2d(tc5_smem_u32(smem + st * STAGE + place), map, (first + issued) * FP8_BLOCK, row, bar);
                    if (++st == STAGES) { st = 0; ++u; }
                }
                // nothing is in flight towards this block when it goes on to the end: copies, or the arrivals that follow the last products
                for (int c = max(0, issued - STAGES); c < issued; ++c) {
                    uint64_t* const bars = ok ? empty : full;
                    ok = tc5_wait(&bars[c % STAGES], (uint32_t)((c / STAGES) & 1)) && ok;
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;\n");
        const int q4 = warp & 3, group = (warp - FP_FIRST_DRAIN) >> 2, r0 = m0 + 32 * q4;
        const uint32_t lanes = tmem + ((uint32_t)(32 * q4) << 16);
        const float* const xs = p.xs + (int64_t)min(r0 + lane, p.m - 1) * all + first;
        const float* const ws = p.ws + (int64_t)(n0 / FP8_BLOCK) * all + first;
        uint64_t acc[W / 2];
#pragma unroll
        for (int j = 0; j < W / 2; ++j) acc[j] = 0;
        float xv = group < blocks ? xs[group] : 0.f, wv = group < blocks ? ws[group] : 0.f;
        for (int b = group; b < blocks; b += 2) {
            const float f = xv * wv;
            if (b + 2 < blocks) { xv = xs[b + 2]; wv = ws[b + 2]; }
            const int q = b & 3;
            ok = __all_sync(0xFFFFFFFFu, tc5_wait(&sum_full[q], (uint32_t)((b >> 2) & 1)));
            if (!ok) break;
            drain_add<W / 32>(lanes + (uint32_t)(q * W), f, acc, tc5_smem_u32(&sum_empty[q]), lane);
        }
        // Once all drains are here the products are done and nothing reads the stages any more: in their place the groups exchange half
        // of their sums, and the results take their way to y. The first group keeps the lower columns.
        ok = drains_agree(ok);
        constexpr int LINES = W / 64;  // of 32 f32 columns, that a group keeps
        uint8_t* const mine = smem + 4096 * LINES * (4 * group + q4);
        const uint8_t* const others = smem + 4096 * LINES * (4 * (group ^ 1) + q4);
        // (what a warp gave has its own place: its result goes behind all of those)
        uint8_t* const out = smem + 4096 * LINES * FP_DRAINS + 4096 * LINES * (4 * group + q4);
        const int c0 = n0 + W / 2 * group;
        auto finish = [&](uint64_t* keep, const uint64_t* give) {
            if (ok) {
#pragma unroll
                for (int i = 0; i < LINES; ++i) put_line<float>(mine + 4096 * i, give + 16 * i, lane);
            }
            ok = drains_agree(ok);
            if (!ok) return;
#pragma unroll
            for (int j = 0; j < W / 8; ++j) {
                const float4 f = *reinterpret_cast<const float4*>(others + 4096 * (j >> 3) + lane * 128 + (((j & 7) ^ (lane & 7)) << 4));
                const float2 lo = both(keep[2 * j]), hi = both(keep[2 * j + 1]);
                keep[2 * j] = pair2(make_float2(lo.x + f.x, lo.y + f.y));
                keep[2 * j + 1] = pair2(make_float2(hi.x + f.z, hi.y + f.w));
            }
            if (p.bf && LINES == 2 && parts == 1) {
                put_line<bf16>(out, keep, lane);
                __syncwarp();
                store_lines<bf16, ALIGNED>(p, out, r0, c0, lane);
            } else {
#pragma unroll
                for (int i = 0; i < LINES; ++i) put_line<float>(out + 4096 * i, keep + 16 * i, lane);
                __syncwarp();
                if (parts == 1)
                    for (int i = 0; i < LINES; ++i) store_f32_lines<ALIGNED>(p, out + 4096 * i, r0, c0 + 32 * i, lane);
            }
        };
        if (group == 0) finish(acc, acc + W / 4);
        else finish(acc + W / 4, acc);
        if (parts > 1) {
            cluster_sync();
            if (ok) add_parts<LINES>(p, out, parts, part, r0, c0, lane);
        }
    }
    if (parts > 1) {
        if (warp < FP_FIRST_DRAIN) { __syncwarp(); cluster_sync(); }  // the service warps' share of the first barrier
        cluster_sync();                                               // nobody leaves while its parts are being read
    }
    if (!ok) report_wait(p.waits, WAIT_FP8);
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "n"(COLS) : "memory");
}

// [rows][k] bytes, boxes of 128 columns x box_rows, zeros past the matrix.
static bool fp8_map(CUtensorMap* map, const uint8_t* q, int64_t k, int64_t rows, int box_rows) {
    const PFN_encodeTiled encode = tensor_map_encoder();
    const cuuint64_t dim[2] = {(cuuint64_t)k, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)k};
    const cuuint32_t box[2] = {FP8_BLOCK, (cuuint32_t)box_rows}, estr[2] = {1u, 1u};
    return encode && encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(q), dim, stride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows past the last that a copy would fill with zeros cost more than those that are there (17 x 14336 x 4096 with boxes of 128 rows:
// 24.5 us, of 24 rows 15.0), so where there is one tile of rows it copies those, in eights; sums of what lies behind them are not stored.
static int copied_rows(int m, int tile) { return std::min(tile, (m + 7) / 8 * 8); }

template <int BN>
static cudaError_t stream_of(const Fp8MatArgs& a, int parts, cudaStream_t st) {
    const int x_rows = copied_rows(a.m, BN);
    CUtensorMap mw, mx;
    if (!fp8_map(&mw, a.wq, a.k, a.n, FS_BM) || !fp8_map(&mx, a.xq, a.k, a.m, x_rows)) return cudaErrorInvalidValue;
    static PerDeviceOnce once;
    cudaError_t e = once.run([] { return cudaFuncSetAttribute(fp8_stream_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, FS_SMEM + 1024); });
    if (e != cudaSuccess) return e;
    constexpr int STAGE = FS_W_BYTES + BN * FP8_BLOCK;
    const Fp8StreamArgs k{a, parts, std::min(FS_MAX_STAGES, FS_SMEM / STAGE), x_rows};
    const dim3 grid((unsigned)((a.n + FS_BM - 1) / FS_BM), (unsigned)((a.m + BN - 1) / BN), (unsigned)parts);
    e = launch_pdl_cluster(fp8_stream_kernel<BN>, grid, dim3(FS_THREADS), (size_t)(k.stages * STAGE + 1024), st, parts, k, mw, mx);
    return e != cudaSuccess ? e : count_launch_and_check();
}

template <int G, bool ALIGNED>
static cudaError_t wide_with(const Fp8MatArgs& a, cudaStream_t st) {
    const int x_rows = G == 1 ? copied_rows(a.m, 128) : 128;
    CUtensorMap mw, mx;
    if (!fp8_map(&mw, a.wq, a.k, a.n, FP_BN / 2 / G) || !fp8_map(&mx, a.xq, a.k, a.m, x_rows)) return cudaErrorInvalidValue;
    static PerDeviceOnce once;
    cudaError_t e = once.run([] { return cudaFuncSetAttribute(fp8_wide_kernel<G, ALIGNED>, cudaFuncAttributeMaxDynamicSharedMemorySize, fp_smem(G) + 1024); });
    if (e != cudaSuccess) return e;
    const int64_t row_tiles = (a.m + 128 * G - 1) / (128 * G), tiles = row_tiles * ((a.n + FP_BN - 1) / FP_BN);
    const int most = device_sm_count() / G;
    if (tiles > INT32_MAX / 4) return cudaErrorInvalidValue;
    // the last round's tiles are halved where all halves find a place
    const int left = (int)(tiles % most), halved = 2 * left <= most ? left : 0;
    const Fp8WideArgs k{a, (int)row_tiles, x_rows, (int)tiles - halved, (int)tiles + halved, a.k > 1024};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(std::min(k.items, most) * G));
    cfg.blockDim = dim3(FP_THREADS);
    cfg.dynamicSmemBytes = (size_t)(fp_smem(G) + 1024);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)G;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = G;
    e = cudaLaunchKernelEx(&cfg, fp8_wide_kernel<G, ALIGNED>, k, mw, mx);
    return e != cudaSuccess ? e : count_launch_and_check();
}

static bool y_aligned(const Fp8MatArgs& a) { return ((reinterpret_cast<uintptr_t>(a.y) | (uintptr_t)(a.ldy * (a.bf ? 2 : 4))) & 15) == 0; }
template <int G>
static cudaError_t wide_of(const Fp8MatArgs& a, cudaStream_t st) { return y_aligned(a) ? wide_with<G, true>(a, st) : wide_with<G, false>(a, st); }

template <int W, bool ALIGNED>
static cudaError_t lone_with(const Fp8MatArgs& a, int parts, cudaStream_t st) {
    const int x_rows = copied_rows(a.m, 128);
    CUtensorMap mw, mx;
    if (!fp8_map(&mw, a.wq, a.k, a.n, W) || !fp8_map(&mx, a.xq, a.k, a.m, x_rows)) return cudaErrorInvalidValue;
    constexpr int SMEM = lone_stages(W) * lone_stage(W) + 1024;
    static_assert(SMEM - 1024 >= 2 * FP_DRAINS * 4096 * (W / 64), "sums and results take the stages' place");
    static PerDeviceOnce once;
    cudaError_t e = once.run([] { return cudaFuncSetAttribute(fp8_lone_kernel<W, ALIGNED>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); });
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)((a.n + W - 1) / W), (unsigned)((a.m + 127) / 128), (unsigned)parts), block(FP_THREADS);
    static_assert(W == 64 || W == 128, "clusters share K of the lower tiles only");
    e = parts == 1 ? launch_pdl(fp8_lone_kernel<W, ALIGNED>, grid, block, (size_t)SMEM, st, a, parts, x_rows, mw, mx)
                   : launch_pdl_cluster(fp8_lone_kernel<W, ALIGNED>, grid, block, (size_t)SMEM, st, parts, a, parts, x_rows, mw, mx);
    return e != cudaSuccess ? e : count_launch_and_check();
}

template <int W>
static cudaError_t lone_of(const Fp8MatArgs& a, int parts, cudaStream_t st) { return y_aligned(a) ? lone_with<W, true>(a, parts, st) : lone_with<W, false>(a, parts, st); }

// Where the kernel of 16 weight rows a block is the faster one (it / the stream of weights, us, weights from memory). Up to 8 rows until
// the bytes of 100 MB and more count for all (1 row: 2048 x 2048 2.8 / 5.7, 4096 x 4096 5.3 / 8.2, 14336 x 4096 13.6 / 14.2, 28672 x 4096
// 22.6 / 22.5); from 9 rows on each block also reads as much of the activations as of the weights (12 rows: 2048 x 2048 3.3 / 7.4,
// 4096 x 4096 7.2 / 10.6, 6144 x 4096 10.7 / 9.7). Where rows do not start on 32 bytes it loads 16 at a time (4096 x 4096 5.8, 14336 x 4096 14.6).
static bool gemv_aligned(const Fp8MatArgs& a) { return ((reinterpret_cast<uintptr_t>(a.wq) | reinterpret_cast<uintptr_t>(a.xq) | (uintptr_t)a.k) & 31) == 0; }
static bool gemv_takes(const Fp8MatArgs& a) {
    return a.m <= 16 && (int64_t)a.n * a.k <= (a.m > 8 ? 1 << 24 : gemv_aligned(a) ? 96 << 20 : 32 << 20);
}
static cudaError_t gemv_of(const Fp8MatArgs& a, cudaStream_t st) {
    const int sms = device_sm_count(), blocks = (int)fp8_blocks(a.k);
    const dim3 grid((unsigned)((a.n + FV_ROWS - 1) / FV_ROWS));
    auto with = [&](void (*kernel)(Fp8MatArgs), int warps) {
        const cudaError_t e = launch_pdl(kernel, grid, dim3(32 * warps), 0, st, a);
        return e != cudaSuccess ? e : count_launch_and_check();
    };
    if (!gemv_aligned(a)) return a.m <= 8 ? with(fp8_gemv_kernel<1, 8, 2, false>, 8) : with(fp8_gemv_kernel<2, 8, 1, false>, 8);
    // 16 warps where a block has its SM for itself, 4 where there are more than two an SM (1 row: 2048 x 8192 5.7, 8 warps 6.8, 4 10.1;
    // 4096 x 4096 6.7, 5.3, 6.7; 9400 x 1024 7.2, 4.6, 3.7); a third block of columns on its way where a warp has more than six
    // (4096 x 14336 12.7 for 13.4; 9400 x 1024 4.7 for 4.6). Of 16 rows one block of columns is ahead (4096 x 4096 7.2, two 8.2).
    if ((int)grid.x <= sms) return a.m <= 8 ? with(fp8_gemv_kernel<1, 16, 3, true>, 16) : with(fp8_gemv_kernel<2, 16, 1, true>, 16);
    if ((int)grid.x <= 2 * sms) {
        if (a.m > 8) return with(fp8_gemv_kernel<2, 8, 1, true>, 8);
        return blocks > 6 * 8 ? with(fp8_gemv_kernel<1, 8, 3, true>, 8) : with(fp8_gemv_kernel<1, 8, 2, true>, 8);
    }
    if (a.m > 8) return with(fp8_gemv_kernel<2, 4, 1, true>, 4);
    return blocks > 6 * 4 ? with(fp8_gemv_kernel<1, 4, 3, true>, 4) : with(fp8_gemv_kernel<1, 4, 2, true>, 4);
}

// More than 16 rows, and what the kernel above leaves: the way that takes least time in a model of each, us on 148 SMs, fitted to 2500
// times of 580 sizes (17 to 2048 rows, 40 matrices of 300 x 512 to 28672 x 4096); what it takes is 1 % over the best way on average.
// Some of them, bf16 results, us (stream; tiles of 128 x 64, one a block, K whole or shared by 2 or 4; 128 x 128; 128 x 256; 256 x 256 by
// two SMs):
//    32 x  1024 x  8192    8.5   10.1 (4)   19.5   29.0   25.8         256 x  4096 x 4096    -    10.9   12.5   17.2   16.0
//    64 x  4096 x 14336   17.2   19.4 (2)   32.0   48.7   42.8         512 x  4096 x 4096    -      -    13.1   17.4   16.3
//   128 x  2048 x   512    9.1    3.9        4.9    5.4    5.7         256 x 14336 x 4096    -      -      -    22.6   20.1
//   128 x  4096 x  8192   18.2   14.6 (2)   20.3   29.5   26.4         384 x  1536 x 8960    -  14.6 (2) 20.9   31.4   27.9
//   128 x 14336 x  4096   24.7     -        15.2   18.9   19.9        2048 x  8192 x 4096    -      -      -    70.1   62.4
//   128 x 28672 x  4096   37.5     -          -    27.3   36.3
// A cluster of the tiles' blocks starts 3 us later than as many blocks.
enum Fp8Way { WAY_STREAM, WAY_LONE64, WAY_LONE64_2, WAY_LONE64_4, WAY_LONE128, WAY_WIDE1, WAY_WIDE2 };
static int stream_rows(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128; }
static int stream_parts(const Fp8MatArgs& a) {
    const int64_t tiles = (int64_t)((a.n + FS_BM - 1) / FS_BM) * ((a.m + stream_rows(a.m) - 1) / stream_rows(a.m));
    const int blocks = (int)fp8_blocks(a.k);
    int parts = 1;
    while (parts < FS_MAX_PARTS && tiles * parts < device_sm_count() && blocks >= 4 * parts) parts *= 2;
    return parts;
}
static Fp8Way way_of(const Fp8MatArgs& a) {
    if (a.m <= 16) return WAY_STREAM;
    auto over = [](int64_t v, int by) { return (double)((v + by - 1) / by); };
    const double sms = device_sm_count(), blocks = (double)fp8_blocks(a.k), weights = (double)a.n * a.k / 6.2e6;
    // Rows that do not start on 128 bytes, or not on the 32 of a sector: an SM takes in more lines for the same columns (325 x 4266, tiles of
    // 128 x 128: K of 7040 21.0 us, 7008 26.1, 7024 32.6; 256 x 256 by two SMs 24.9, 25.3, 25.9).
    const double skew = a.k % 128 == 0 ? 0.0 : a.k % 32 == 0 ? 0.4 : 1.0;
    Fp8Way best = WAY_WIDE2;
    double least = 1e30;
    auto offer = [&](Fp8Way way, double us) {
        if (us < least) { least = us; best = way; }
    };
    for (int g = 1; g <= 2; ++g) {
        const double teams = floor(sms / g), tiles = over(a.m, 128 * g) * over(a.n, FP_BN), left = fmod(tiles, teams), half = g == 1 ? 0.685 : 0.762;
        const double rounds = floor(tiles / teams) + (left == 0 ? 0.0 : 2 * left <= teams ? half : 1.0);
        offer(g == 1 ? WAY_WIDE1 : WAY_WIDE2, g == 1 ? 3.62 + rounds * ((0.557 + 0.06 * skew) * blocks + 1.47) : 3.77 + rounds * (0.425 * blocks + 1.95));
    }
    const double low = over(a.m, 128) * over(a.n, 64), high = over(a.m, 128) * over(a.n, 128);
    if (low <= sms) offer(WAY_LONE64, std::max(2.68 + (0.216 + 0.03 * skew) * blocks + 2.2 * low / sms, 3.9 + weights));
    if (2 * low <= sms && blocks >= 16) offer(WAY_LONE64_2, std::max(6.1 + (0.22 + 0.03 * skew) * ceil(blocks / 2) + 1.7 * 2 * low / sms, 6.9 + weights));
    if (4 * low <= 0.87 * sms && blocks >= 32) offer(WAY_LONE64_4, std::max(6.1 + (0.225 + 0.03 * skew) * ceil(blocks / 4) + 0.7 * 4 * low / sms, 6.5 + weights));
    if (high <= sms) offer(WAY_LONE128, std::max(3.3 + (0.25 + 0.17 * skew) * blocks + 3.2 * high / sms, 4.9 + weights));
    // (several tiles of 128 rows only where K is long and they still fit side by side: 384 x 512 x 14336 16.4 us, tiles of 128 x 64 26.7)
    const int rows = stream_rows(a.m), parts = stream_parts(a);
    const double teams = over(a.n, FS_BM) * over(a.m, rows) * parts;
    if (a.m <= 128 || teams <= sms) {
        const double each = rows == 32 ? 0.442 : rows == 64 ? 0.368 : 0.79;
        const double load = std::min(std::max(teams / sms, 1.0), 2.0), rounds = over((int64_t)teams, (int)(2 * sms));
        offer(WAY_STREAM, std::max(3.2 + (parts > 1 ? 0.47 : 0.0) + rounds * (ceil(blocks / parts) * each * (1 + 0.3 * (load - 1)) + 0.038 * rows), 6.4 + weights));
    }
    return best;
}

cudaError_t launch_fp8_matmul(const Fp8MatArgs& a, cudaStream_t st) {
    if (a.m == 0 || a.n == 0) return cudaSuccess;
    if (a.m < 0 || a.n < 0 || a.k <= 0 || a.k % 16 != 0) return cudaErrorInvalidValue;
    if (gemv_takes(a)) return gemv_of(a, st);
    switch (way_of(a)) {
        case WAY_LONE64: return lone_of<64>(a, 1, st);
        case WAY_LONE64_2: return lone_of<64>(a, 2, st);
        case WAY_LONE64_4: return lone_of<64>(a, 4, st);
        case WAY_LONE128: return lone_of<128>(a, 1, st);
        case WAY_WIDE1: return wide_of<1>(a, st);
        case WAY_WIDE2: return wide_of<2>(a, st);
        case WAY_STREAM: break;
    }
    const int parts = stream_parts(a);
    switch (stream_rows(a.m)) {
        case 16: return stream_of<16>(a, parts, st);
        case 32: return stream_of<32>(a, parts, st);
        case 64: return stream_of<64>(a, parts, st);
        default: return stream_of<128>(a, parts, st);
    }
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
