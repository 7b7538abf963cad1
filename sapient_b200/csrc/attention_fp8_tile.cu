// Attention of many rows over a cache of 8-bit rows on the 5th-generation tensor cores (formulas and precision: attention_fp8.cu).
//
// A block has two groups of four warps, each with 128 rows whose scores S = Q K^T [128 x 128 keys] and sums O [128 x head_dim] lie in
// tensor memory, a row a lane. While one group turns scores into weights, the tensor cores work for the other:
//   warps 0-3, 4-7   weights: a thread has a row; S is read twice, for its maximum and for the exponentials, which go back over it as fp16
//                    and are the first operand of the second product from there. O is rescaled only when a row's reference moves.
//   warps 8-11       keys: e4m3 rows to fp16 in shared memory (128-byte swizzle, K-major), and the scales of keys and values
//   warps 12-15      values, as they lie (MN-major)
//   warp 16          issues the products
// ROWS: the groups have 128 rows each of 256, and keys in common. KEYS (up to 128 rows): the same rows, key tiles by turns; their sums
// are added up at the end. Keys may be shared out to the blocks of a cluster as well, which add up through shared memory.
//
// A row's weights are e^(z - M) s' with one M for the lift of the header and the scales' size: with u the power of two not below the tile's largest
// finite scale, M is moved when z + u passes M + 15 (log2), to z + u - 9; sum of e^(z - M) and O move along.
#include <algorithm>
#include <type_traits>

#include "attention_fp8.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tc5_ptx.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

constexpr int AT_KEYS = 128, AT_PAGES = AT_KEYS / KV_PAGE, AT_THREADS = 640, AT_RING = 4, AT_MAX_PARTS = 8;
constexpr float AT_MOST = 15.f, AT_SET = 9.f;  // log2 of the largest weight, and of it when M is set

template <typename T, int DP, bool KEYS>
struct AtShape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PLANES = F32 ? 2 : 1, TILES = KEYS ? 1 : 2;      // of Q
    static constexpr int STAGES = F32 && !KEYS && DP == 128 ? 1 : 2;      // of keys and of values
    static constexpr int TILE = 128 * DP * 2;                             // bytes of 128 rows in fp16
    static constexpr int Q = PLANES * TILES * TILE, SMEM = Q + 2 * STAGES * TILE + 1024;
    static constexpr int LDO = DP + 4, SUMS = 2 * 128 * LDO * 4;          // takes the operands' place
    static constexpr int WEIGHTS = KEYS ? 128 * 2 * 4 : 256 * 4;           // of the sums of a block's share of rows, behind them (parts x rows of a share is at most that)
    static_assert(SUMS + WEIGHTS <= SMEM - 1024, "sums of both groups");
};

__device__ __forceinline__ void at_init(uint64_t* bar, uint32_t arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(tc5_smem_u32(bar)), "r"(arrivals) : "memory");
}
__device__ __forceinline__ uint32_t at_idesc(int n, bool b_mn) { return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }
// Values as they lie: rows of 64 coordinates (128 bytes, swizzled) a token, 8 tokens 1024 bytes apart; the next 64 coordinates 128 tokens on.
__device__ __forceinline__ uint64_t at_desc_values(uint32_t saddr) {
    return (tc5_desc(saddr) & ~((uint64_t)0x3FFF << 16)) | (uint64_t)(128 * 128 >> 4) << 16;
}
__device__ __forceinline__ void at_mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void at_ld32(uint32_t taddr, float* f) {
    uint32_t* const r = reinterpret_cast<uint32_t*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void at_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
                 "r"(r[15]), "r"(taddr)
                 : "memory");
}
// The values that the wait is for go through it, so that nothing looks at them before.
__device__ __forceinline__ void at_wait_for(float (&f)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3]), "+f"(f[4]), "+f"(f[5]), "+f"(f[6]), "+f"(f[7]), "+f"(f[8]), "+f"(f[9]), "+f"(f[10]), "+f"(f[11]),
                   "+f"(f[12]), "+f"(f[13]), "+f"(f[14]), "+f"(f[15]), "+f"(f[16]), "+f"(f[17]), "+f"(f[18]), "+f"(f[19]), "+f"(f[20]), "+f"(f[21]), "+f"(f[22]),
                   "+f"(f[23]), "+f"(f[24]), "+f"(f[25]), "+f"(f[26]), "+f"(f[27]), "+f"(f[28]), "+f"(f[29])
                 :
                 : "memory");
    asm volatile("" : "+f"(f[30]), "+f"(f[31]) : : "memory");
}
__device__ __forceinline__ void at_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void at_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void at_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void at_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void at_fence_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Two values an instruction.
__device__ __forceinline__ void at_mul2(float& a, float& b, float u, float v) {
    asm("{\n.reg .b64 x, y;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n" : "+f"(a), "+f"(b) : "f"(u), "f"(v));
}
__device__ __forceinline__ void at_fma2(float& a, float& b, float u, float v) {  // a u + v, b u + v
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %2};\nmov.b64 z, {%3, %3};\nfma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}\n"
        : "+f"(a), "+f"(b) : "f"(u), "f"(v));
}
__device__ __forceinline__ void at_add2(float& a, float& b, float u, float v) {
    asm("{\n.reg .b64 x, y;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n" : "+f"(a), "+f"(b) : "f"(u), "f"(v));
}
__device__ __forceinline__ float4 at_peer4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float at_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <typename T, int DP, bool KEYS>
__global__ void __launch_bounds__(AT_THREADS, 1) attention_tile_kernel(const AttentionFp8Args a, int parts, int tiles) {
    using Sh = AtShape<T, DP, KEYS>;
    constexpr bool F32 = Sh::F32;
    constexpr int STAGES = Sh::STAGES, ROWS = 128 * Sh::TILES;
    extern __shared__ uint8_t at_smem_raw[];
    __shared__ __align__(8) uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2], p_full[2], o_full;
    __shared__ __align__(16) float k_scale[AT_RING][AT_KEYS], v_scale[AT_RING][AT_KEYS];
    __shared__ uint32_t gone_s[AT_RING];  // pages of the tile that are not there
    __shared__ float row_factor[ROWS];
    __shared__ float part_m[2][128], part_l[2][128];
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const int head = blockIdx.x % a.c.n_kv, part = blockIdx.z, group = a.n_heads / a.c.n_kv, dim = a.c.dim;
    pdl_wait();
    pdl_trigger();
    // (the tiles with the most keys first)
    const AfTile tile = af_tile(a, blockIdx.y, tiles - 1 - blockIdx.x / a.c.n_kv, ROWS);
    if (tile.n <= 0) return;  // (the whole cluster)
    uint8_t* const smem = at_smem_raw + ((1024u - (tc5_smem_u32(at_smem_raw) & 1023u)) & 1023u);
    uint8_t *const ks_ = smem + Sh::Q, *const vs_ = ks_ + STAGES * Sh::TILE;
    // ── the block's keys ──
    const int last_row = tile.row0 + tile.n - 1;
    const int pos_first = tile.len - tile.rows + tile.row0 / group, pos_last = tile.len - tile.rows + last_row / group;
    const int held = (int)min((int64_t)tile.len, (int64_t)a.c.max_pages * KV_PAGE);
    const int k_end = min(pos_last + 1, held), k_begin = a.window > 0 ? max(0, pos_first - a.window + 1) : 0;
    const int t_begin = k_begin / AT_KEYS, t_end = k_end > k_begin ? (k_end + AT_KEYS - 1) / AT_KEYS : t_begin;
    const int per = (t_end - t_begin + parts - 1) / parts;
    const int b_begin = min(t_end, t_begin + part * per), n_kv = min(t_end, b_begin + per) - b_begin;  // key tiles of the block
    const int groups = KEYS || tile.n > 128 ? 2 : 1, jobs = KEYS ? n_kv : groups * n_kv;  // job j is group j % groups'
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(tc5_smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (tid == 32) {
        for (int i = 0; i < STAGES; ++i) {
            at_init(&k_full[i], 4);
            at_init(&v_full[i], 4);
            at_init(&k_empty[i], 1);
            at_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            at_init(&s_full[i], 1);
            at_init(&p_full[i], 4);
        }
        at_init(&o_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    // ── queries: fp16 operands, eight values a thread ──
    if (warp < 16) {
        constexpr int PER = DP / 8, AT_ONCE = 512 / PER;  // threads of a row, rows at once
        const int u = tid % PER;
        constexpr int BATCH = 4;
        for (int r0 = tid / PER; r0 < ROWS; r0 += BATCH * AT_ONCE) {
            float x[BATCH][8];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int r = r0 + i * AT_ONCE, row = tile.row0 + min(r, tile.n - 1);
                const T* const src = static_cast<const T*>(a.q) + (int64_t)(tile.first + row / group) * a.ldq + (int64_t)(head * group + row % group) * dim + 8 * u;
                if (r < tile.n && 8 * u < dim) {
                    if constexpr (F32) {
                        const float4 v = reinterpret_cast<const float4*>(src)[0], w = reinterpret_cast<const float4*>(src)[1];
                        x[i][0] = v.x; x[i][1] = v.y; x[i][2] = v.z; x[i][3] = v.w;
                        x[i][4] = w.x; x[i][5] = w.y; x[i][6] = w.z; x[i][7] = w.w;
                    } else {
                        const uint4 v = *reinterpret_cast<const uint4*>(src);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            x[i][2 * j] = __uint_as_float(w[j] << 16);
                            x[i][2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[i][j] = 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int r = r0 + i * AT_ONCE;
                float most = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[i][j]));
#pragma unroll
                for (int o = PER / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
                float by, back;
                af_row_scale(most, by, back);
                if (a.scale < 0.f) by = -by;
                if (r < ROWS) {
                    if (u == 0) row_factor[r] = back * fabsf(a.scale) * AF_LOG2E;
                    uint4 hi, lo;
                    uint32_t *const h = &hi.x, *const l = &lo.x;
#pragma unroll
                    for (int j = 0; j < 4; ++j) af_split(x[i][2 * j] * by, x[i][2 * j + 1] * by, h[j], l[j]);
                    uint8_t* const to = smem + r / 128 * Sh::TILE + u / 8 * (128 * 128) + r % 128 * 128 + ((u % 8) ^ (r & 7)) * 16;
                    *reinterpret_cast<uint4*>(to) = hi;
                    if constexpr (F32) *reinterpret_cast<uint4*>(to + Sh::TILES * Sh::TILE) = lo;
                }
            }
        }
    }
    at_fence_smem();
    at_before();
    __syncthreads();
    at_after();
    const uint32_t tmem = tmem_slot;  // S of the groups at columns 0 and 128, O at 256 and 256 + DP
    bool ok = true;
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;\n");  // 128 x 48 + 256 x 80 + 256 x 136 = 640 x 96
        if (warp == 16) {
        const bool leader = tc5_elect();
        const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        const uint32_t id_s = at_idesc(AT_KEYS, false), id_o = at_idesc(dim, true);
        const uint64_t qd = tc5_desc(tc5_smem_u32(smem)), kd = tc5_desc(tc5_smem_u32(ks_)), vd = at_desc_values(tc5_smem_u32(vs_));
        const int steps = dim / 16;
        auto scores = [&](int j) {
            const int t = groups == 2 ? j & 1 : 0, kv = KEYS || groups == 1 ? j : j >> 1, st = kv % STAGES;
            if (KEYS || t == 0) ok = __all_sync(0xFFFFFFFFu, tc5_wait(&k_full[st], (uint32_t)((kv / STAGES) & 1)));
            if (!ok) return;
            at_after();
            if (leader) {
                const uint64_t q = qd + (uint64_t)((KEYS ? 0 : t) * (Sh::TILE >> 4)), k = kd + (uint64_t)(st * (Sh::TILE >> 4));
#pragma unroll
                for (int p = Sh::PLANES - 1; p >= 0; --p)
                    for (int s = 0; s < steps; ++s) {
                        const uint64_t at = (uint64_t)((s >> 2) * (128 * 128 >> 4) + (s & 3) * 2);
                        tc5_mma(tm + 128u * t, q + at + (uint64_t)(p * Sh::TILES * (Sh::TILE >> 4)), k + at, id_s, p != Sh::PLANES - 1 || s > 0);
                    }
                tc5_commit(&s_full[t]);
                if (KEYS || t == groups - 1) tc5_commit(&k_empty[st]);
            }
            __syncwarp();
        };
        for (int j = 0; j < groups && j < jobs && ok; ++j) scores(j);
        for (int j = 0; j < jobs && ok; ++j) {
            const int t = groups == 2 ? j & 1 : 0, i = groups == 2 ? j >> 1 : j, kv = KEYS ? j : i, st = kv % STAGES;
            bool here = tc5_wait(&p_full[t], (uint32_t)(i & 1));
            if (KEYS || t == 0) here = here && tc5_wait(&v_full[st], (uint32_t)((kv / STAGES) & 1));
            ok = __all_sync(0xFFFFFFFFu, here);
            if (!ok) break;
            at_after();
            if (leader) {
                const uint64_t v = vd + (uint64_t)(st * (Sh::TILE >> 4));
#pragma unroll
                for (int s = 0; s < AT_KEYS / 16; ++s)
#pragma unroll
                    for (int p = Sh::PLANES - 1; p >= 0; --p)
                        at_mma_tmem(tm + 256u + (uint32_t)(DP * t), tm + 128u * t + (uint32_t)(F32 ? 32 * (s / 2) + 16 * p + 8 * (s % 2) : 8 * s), v + (uint64_t)(s * (2048 >> 4)), id_o,
                                    i > 0 || s > 0 || p != Sh::PLANES - 1);
                if (KEYS || t == groups - 1) tc5_commit(&v_empty[st]);
            }
            __syncwarp();
            if (j + groups < jobs) scores(j + groups);
        }
        if (jobs > 0) {
            if (ok && leader) tc5_commit(&o_full);
            __syncwarp();
            // no arrival is on its way to this block when it goes on to the end
            for (int kv = max(0, n_kv - STAGES); kv < n_kv; ++kv) {
                const uint32_t parity = (uint32_t)((kv / STAGES) & 1);
                ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&k_empty[kv % STAGES], parity) && tc5_wait(&v_empty[kv % STAGES], parity));
            }
            ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&o_full, 0));
        }
        }
        if (parts > 1) {
            cluster_sync();
            cluster_sync();
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;\n");
        // Sixteen bytes of a row a copy, 64 coordinates of eight tokens a warp at once: stores of eight threads fall on 32 different banks.
        const bool values = warp >= 12;
        constexpr int HALVES = DP / 64, N = 4 * HALVES;  // copies of a thread: tokens tok0 + 32 i, coordinates 16 ch and 64 + 16 ch
        const int p = tid - (values ? 384 : 256), ch = p % 4, tok0 = p / 4;
        const int32_t* const table = a.c.page_table + (int64_t)max(0, min(tile.slot, a.c.n_slots - 1)) * a.c.max_pages;
        auto page_of = [&](int kv) {  // lanes 0 to 7: the tile's pages
            const int index = (b_begin + kv) * AT_PAGES + (lane & 7);
            const int page = kv < n_kv && index < a.c.max_pages && index * KV_PAGE < k_end ? table[index] : -1;
            return page < a.c.n_pages ? max(page, -1) : -1;
        };
        const int64_t page_rows = (int64_t)2 * a.c.n_kv * KV_PAGE;
        const uint8_t* const from = a.c.values + (a.c.row(0, values ? 1 : 0, head) + tok0 % KV_PAGE) * dim + 16 * ch;
        uint4 raw[N];
        auto load = [&](int pages) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int page = __shfl_sync(0xFFFFFFFFu, pages, tok0 / KV_PAGE + 2 * i);
                const uint8_t* const row = from + (int64_t)max(page, 0) * page_rows * dim;
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    raw[HALVES * i + h] = make_uint4(0, 0, 0, 0);
                    if (page >= 0 && 64 * h + 16 * ch < dim) raw[HALVES * i + h] = __ldg(reinterpret_cast<const uint4*>(row + 64 * h));
                }
            }
        };
        uint8_t* const to0 = (values ? vs_ : ks_) + tok0 * 128;
        const int u0 = ((2 * ch) ^ (tok0 & 7)) * 16, u1 = ((2 * ch + 1) ^ (tok0 & 7)) * 16;
        uint64_t *const full = values ? v_full : k_full, *const empty = values ? v_empty : k_empty;
        int pages = page_of(0);
        load(pages);
        for (int kv = 0; kv < n_kv; ++kv) {
            const int st = kv % STAGES, use = kv / STAGES;
            float sk = 0.f, sv = 0.f;
            if (!values) {  // of token p
                const int page = __shfl_sync(0xFFFFFFFFu, pages, p / KV_PAGE);
                if (page >= 0) {
                    const int64_t at = a.c.row(page, 0, head) + p % KV_PAGE;
                    sk = __ldg(a.c.scales + at);
                    sv = __ldg(a.c.scales + at + (int64_t)a.c.n_kv * KV_PAGE);
                }
            }
            const uint32_t gone = __ballot_sync(0xFFFFFFFFu, pages < 0) & 0xFFu;
            pages = page_of(kv + 1);
            if (use > 0) ok = __all_sync(0xFFFFFFFFu, tc5_wait(&empty[st], (uint32_t)((use - 1) & 1)));
            if (!ok) break;
            uint8_t* const to = to0 + st * Sh::TILE;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                uint32_t h[8];
                af_halves(raw[i].x, h[0], h[1]);
                af_halves(raw[i].y, h[2], h[3]);
                af_halves(raw[i].z, h[4], h[5]);
                af_halves(raw[i].w, h[6], h[7]);
                if (values) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[j] = af_finite(h[j]);
                }
                uint8_t* const row = to + i / HALVES * (32 * 128) + i % HALVES * (128 * 128);
                *reinterpret_cast<uint4*>(row + u0) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4*>(row + u1) = make_uint4(h[4], h[5], h[6], h[7]);
            }
            if (!values) {
                k_scale[kv % AT_RING][p] = sk;
                v_scale[kv % AT_RING][p] = sv;
                if (p == 0) gone_s[kv % AT_RING] = gone;
            }
            at_fence_smem();
            __syncwarp();
            if (lane == 0) tc5_arrive(&full[st]);
            if (kv + 1 < n_kv) load(pages);
        }
        if (parts > 1) {
            cluster_sync();
            cluster_sync();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 136;\n");
        const int t = warp >> 2, r = 32 * (warp & 3) + lane, row = (KEYS ? 0 : 128 * t) + r;  // of the block's rows
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16), S = lanes + 128u * t, O = lanes + 256u + (uint32_t)(DP * t);
        const int at = tile.row0 + row, pos = tile.len - tile.rows + at / group;
        const int limit = row < tile.n ? min(pos, held - 1) : -1, low = a.window > 0 ? pos - a.window + 1 : 0;
        // keys that all rows of the group see
        const int row_a = KEYS ? 0 : 128 * t, row_b = min(row_a + 127, tile.n - 1);
        const int whole_to = min(tile.len - tile.rows + (tile.row0 + row_a) / group, held - 1), whole_from = a.window > 0 ? tile.len - tile.rows + (tile.row0 + row_b) / group - a.window + 1 : 0;
        const float c = row_factor[row];
        const int mine = t >= groups ? 0 : (jobs - t + groups - 1) / groups;  // jobs of the group
        float m = -INFINITY, l0 = 0.f, l1 = 0.f;
        for (int i = 0; i < mine; ++i) {
            const int kv = KEYS ? 2 * i + t : i, key0 = (b_begin + kv) * AT_KEYS, slot = kv % AT_RING;
            ok = __all_sync(0xFFFFFFFFu, tc5_wait(&s_full[t], (uint32_t)(i & 1)));
            if (!ok) break;
            at_after();
            float s0[32], s1[32];
            at_ld32(S, s0);
            const uint32_t gone = gone_s[slot];
            const bool masked = gone != 0 || key0 < whole_from || key0 + AT_KEYS - 1 > whole_to;
            const int hi = limit - key0, lo = low - key0;
            // the power of two not below the largest finite scale of values that the block may see
            uint32_t big = 0;
            {
                const float4 v = *reinterpret_cast<const float4*>(&v_scale[slot][4 * lane]);
                const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = key0 + 4 * lane + j;
                    if (f[j] > 0.f && f[j] < INFINITY && (!masked || (k >= k_begin && k < k_end))) big = max(big, __float_as_uint(f[j]));
                }
                big = __reduce_max_sync(0xFFFFFFFFu, big);
            }
            const float up = (float)(min(max((int)((big + 0x7FFFFFu) >> 23), 27), 253) - 127);
            // One job, with and without keys that a row does not see: both as code of its own, since decided at each value it is 6 instructions more.
            auto job = [&](auto with_mask) {
                constexpr bool MASK = decltype(with_mask)::value;
                // bits of the keys k0 .. k0 + 31 that the row sees
                auto seen = [&](int k0) {
                    const int from = lo - k0, to = hi - k0;
                    uint32_t bits = to >= 31 ? 0xFFFFFFFFu : to < 0 ? 0u : (2u << to) - 1u;
                    bits = from <= 0 ? bits : from > 31 ? 0u : bits & (0xFFFFFFFFu << from);
                    const uint32_t no = gone >> (k0 / KV_PAGE);
                    return bits & ~((no & 1 ? 0xFFFFu : 0u) | (no & 2 ? 0xFFFF0000u : 0u));
                };
                // keys k0 .. k0 + 31: scores times their scale; what a row does not see is -inf
                auto scaled = [&](float (&s)[32], int k0, uint32_t bits) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&k_scale[slot][k0 + k]);
                        at_mul2(s[k], s[k + 1], f.x, f.y);
                        at_mul2(s[k + 2], s[k + 3], f.z, f.w);
                    }
                    if constexpr (MASK) {
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(bits >> k & 1)) s[k] = -INFINITY;
                    }
                };
                float b0 = -INFINITY, b1 = -INFINITY, b2 = -INFINITY, b3 = -INFINITY;
                auto largest = [&](const float (&s)[32]) {
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        b0 = at_max3(b0, s[k], s[k + 1]);
                        b1 = at_max3(b1, s[k + 2], s[k + 3]);
                        b2 = at_max3(b2, s[k + 4], s[k + 5]);
                        b3 = at_max3(b3, s[k + 6], s[k + 7]);
                    }
                };
#pragma unroll 1
                for (int k0 = 0; k0 < AT_KEYS; k0 += 64) {  // the next 32 are on their way while these are looked at
                    at_wait_for(s0);
                    at_ld32(S + k0 + 32, s1);
                    scaled(s0, k0, MASK ? seen(k0) : 0u);
                    largest(s0);
                    at_wait_for(s1);
                    at_ld32(S + (k0 + 64) % AT_KEYS, s0);  // at the end: the first again
                    scaled(s1, k0 + 32, MASK ? seen(k0 + 32) : 0u);
                    largest(s1);
                }
                const float best = fmaxf(fmaxf(b0, b1), fmaxf(b2, b3));
                // (nothing seen: best is -inf, which a factor of 0 would turn into NaN)
                const float x = best == -INFINITY ? -INFINITY : fmaf(best, c, up);
                const bool moves = x > m + AT_MOST;
                if (__any_sync(0xFFFFFFFFu, moves)) {
                    const float to = moves ? x - AT_SET : m, by = moves ? af_ex2(m - to) : 1.f;  // (m = -inf: 0)
                    m = to;
                    l0 *= by;
                    l1 *= by;
                    if (i > 0) {
#pragma unroll 1
                        for (int d = 0; d < dim; d += 16) {
                            uint32_t o[16];
                            tc5_ld16(O + d, o);
                            at_wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * by);
                            at_st16(O + d, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : -m;
                auto weights = [&](float (&s)[32], int k0) {
                    uint32_t w_hi[16], w_lo[16];
                    const uint32_t bits = MASK ? seen(k0) : 0u;
                    scaled(s, k0, bits);
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&v_scale[slot][k0 + k]);
                        const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                        for (int j = 0; j < 4; j += 2) {
                            float p0 = s[k + j], p1 = s[k + j + 1];
                            at_fma2(p0, p1, c, base);
                            p0 = af_ex2(p0);
                            p1 = af_ex2(p1);
                            if constexpr (MASK) {  // (-inf times a factor of 0 is NaN)
                                if (!(bits >> (k + j) & 1)) p0 = 0.f;
                                if (!(bits >> (k + j + 1) & 1)) p1 = 0.f;
                            }
                            at_add2(l0, l1, p0, p1);
                            at_mul2(p0, p1, v[j], v[j + 1]);
                            if constexpr (MASK) {  // (what is masked may have any scale)
                                if (!(bits >> (k + j) & 1)) p0 = 0.f;
                                if (!(bits >> (k + j + 1) & 1)) p1 = 0.f;
                            }
                            const int w = (k + j) / 2;
                            if constexpr (F32) af_split(p0, p1, w_hi[w], w_lo[w]);
                            else w_hi[w] = af_pack(p0, p1);
                        }
                    }
                    if constexpr (F32) {  // over the scores that they come from
                        at_st16(S + k0, w_hi);
                        at_st16(S + k0 + 16, w_lo);
                    } else {
                        at_st16(S + k0 / 2, w_hi);
                    }
                };
#pragma unroll 1
                for (int k0 = 0; k0 < AT_KEYS; k0 += 64) {
                    at_wait_for(s0);
                    at_ld32(S + k0 + 32, s1);
                    weights(s0, k0);
                    at_wait_for(s1);
                    if (k0 + 64 < AT_KEYS) at_ld32(S + k0 + 64, s0);
                    weights(s1, k0 + 32);
                }
            };
            if (masked) job(std::true_type{});
            else job(std::false_type{});
            at_wait_st();
            at_before();
            __syncwarp();
            if (lane == 0) tc5_arrive(&p_full[t]);
        }
        const float l = l0 + l1;
        if (jobs > 0) ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&o_full, 0));
        at_after();
        T* const out = static_cast<T*>(a.out) + (int64_t)head * group * dim;
        if (!KEYS && parts == 1) {
            const float by = l == 0.f || mine == 0 ? 0.f : 1.f / l;
            T* const to = out + (int64_t)(tile.first + at / group) * a.ldo + (int64_t)(at % group) * dim;
#pragma unroll 1
            for (int d = 0; ok && d < dim; d += 32) {
                float o[32];
                at_ld32(O + d, o);
                at_wait_for(o);
                if (row < tile.n) {
                    constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
                    for (int j = 0; j < 32; j += PER) {
                        uint4 w;
                        uint32_t* const u = &w.x;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            if constexpr (F32) u[q] = mine > 0 ? __float_as_uint(o[j + q] * by) : 0u;
                            else u[q] = mine > 0 ? pack_bf16(o[j + 2 * q] * by, o[j + 2 * q + 1] * by) : 0u;
                        }
                        if (d + j < dim) *reinterpret_cast<uint4*>(to + d + j) = w;
                    }
                }
            }
        } else {
            float* const sums = reinterpret_cast<float*>(smem);  // [group][row][LDO], over the operands, which have been read
            float* const weights = sums + Sh::SUMS / 4;          // [row of the block's share][sum]
#pragma unroll 1
            for (int d = 0; d < dim; d += 32) {
                float o[32];
                if (mine > 0 && ok) {
                    at_ld32(O + d, o);
                    at_wait_for(o);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < 32; j += 4)
                    if (d + j < dim) *reinterpret_cast<float4*>(&sums[(128 * t + r) * Sh::LDO + d + j]) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
            }
            part_m[t][r] = m;
            part_l[t][r] = l;
            asm volatile("barrier.cta.sync 1, 256;\n" ::: "memory");
            if (parts > 1) cluster_sync();
            // The blocks share the rows out: row q of the block's is part + parts q of the tile. Sum s of a row is part s / SETS's, group s % SETS's
            // (KEYS) or its own group's.
            constexpr int SETS = KEYS ? 2 : 1;
            const int sets = parts * SETS, rows_here = (tile.n - part + parts - 1) / parts;
            for (int e = tid; e < rows_here * sets; e += 256) {
                const int q = e / sets, s = e - q * sets, of = part + parts * q;
                float pm = 0.f, top = -INFINITY, total = 0.f;
                for (int x = 0; x < sets; ++x) {
                    const int g = KEYS ? x % SETS : of / 128;
                    const uint32_t at_m = smem_addr(&part_m[g][of % 128]), at_l = smem_addr(&part_l[g][of % 128]);
                    const float xm = parts > 1 ? ld_peer(peer_smem(at_m, x / SETS)) : part_m[g][of % 128], xl = parts > 1 ? ld_peer(peer_smem(at_l, x / SETS)) : part_l[g][of % 128];
                    const float to = fmaxf(top, xm);
                    total = total * (top == to ? 1.f : af_ex2(top - to)) + (xm == to ? xl : xl * af_ex2(xm - to));
                    top = to;
                    if (x == s) pm = xm;
                }
                weights[e] = total == 0.f || pm == -INFINITY ? 0.f : af_ex2(pm - top) / total;
            }
            asm volatile("barrier.cta.sync 1, 256;\n" ::: "memory");
            const int quads = dim / 4;
            for (int e = tid; e < rows_here * quads; e += 256) {
                const int q = e / quads, d = 4 * (e - q * quads), of = part + parts * q;
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int x0 = 0; x0 < sets; x0 += 4) {
                    float4 v[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        if (x0 + x >= sets) break;
                        const float* const src = sums + ((KEYS ? (x0 + x) % SETS : of / 128) * 128 + of % 128) * Sh::LDO + d;
                        v[x] = parts > 1 ? at_peer4(peer_smem(smem_addr(src), (x0 + x) / SETS)) : *reinterpret_cast<const float4*>(src);
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        if (x0 + x >= sets) break;
                        const float w = weights[q * sets + x0 + x];
                        y.x = fmaf(v[x].x, w, y.x);
                        y.y = fmaf(v[x].y, w, y.y);
                        y.z = fmaf(v[x].z, w, y.z);
                        y.w = fmaf(v[x].w, w, y.w);
                    }
                }
                const int where = tile.row0 + of;
                T* const to = out + (int64_t)(tile.first + where / group) * a.ldo + (int64_t)(where % group) * dim + d;
                if (!ok) continue;
                if constexpr (F32) *reinterpret_cast<float4*>(to) = y;
                else *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
            }
            if (parts > 1) cluster_sync();  // nobody leaves while its sums are being read
        }
    }
    if (!ok) report_wait(a.waits, WAIT_ATTENTION);
    at_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

template <typename T, int DP, bool KEYS>
static cudaError_t launch_tiles(const AttentionFp8Args& a, cudaStream_t st) {
    using Sh = AtShape<T, DP, KEYS>;
    static PerDeviceOnce once;
    cudaError_t e = once.run([] { return cudaFuncSetAttribute(attention_tile_kernel<T, DP, KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM); });
    if (e != cudaSuccess) return e;
    const int64_t rows = (int64_t)a.max_rows * (a.n_heads / a.c.n_kv), height = 128 * Sh::TILES, tiles = (rows + height - 1) / height, clusters = tiles * a.c.n_kv * a.n_seqs;
    // an SM a block, each with four tiles of keys at least
    int parts = 1;
    while (parts < AT_MAX_PARTS && clusters * parts * 2 <= device_sm_count() && (int64_t)a.max_len >= 4 * AT_KEYS * 2 * parts) parts *= 2;
    e = launch_pdl_cluster(attention_tile_kernel<T, DP, KEYS>, dim3((unsigned)(tiles * a.c.n_kv), (unsigned)a.n_seqs, (unsigned)parts), dim3(AT_THREADS), Sh::SMEM, st, parts, a,
                           parts, (int)tiles);
    return e != cudaSuccess ? e : count_launch_and_check();
}

template <typename T, int DP>
static cudaError_t tiles_as(const AttentionFp8Args& a, cudaStream_t st) {
    return (int64_t)a.max_rows * (a.n_heads / a.c.n_kv) <= 128 ? launch_tiles<T, DP, true>(a, st) : launch_tiles<T, DP, false>(a, st);
}
cudaError_t launch_attention_fp8_tiles(const AttentionFp8Args& a, bool bf, cudaStream_t st) {
    if (a.c.dim <= 64) return bf ? tiles_as<bf16, 64>(a, st) : tiles_as<float, 64>(a, st);
    return bf ? tiles_as<bf16, 128>(a, st) : tiles_as<float, 128>(a, st);
}

}  // namespace sp
