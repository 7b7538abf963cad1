// Attention of many rows over a cache of 8-bit rows on the 5th-generation tensor cores (formulas and precision: attention_fp8.cu).
//
// A block has two groups of four warps, each with 128 rows whose scores S = Q K^T [128 x 128 keys] and sums O [128 x head_dim] lie in
// tensor memory, a row a lane. While one group turns scores into weights, the tensor cores work for the other:
//   warps 0-3, 4-7   weights: a thread has a row of S in registers; its maximum, exponentials, which go back over S as fp16 (handed over in two parts),
//                    and are the first operand of the second product from there. O is rescaled only when a row's reference moves.
//   warps 8-11       values: e4m3 rows to fp16 in shared memory, as they lie (MN-major, 128-byte swizzle); f32: keys as well (K-major)
//   warp 12          issues the products
//   warp 13          keys of bf16 rows, as they are, a page a TMA copy, and the scales
// bf16 rows are multiplied with the keys' own bytes: q is two e4m3 digits, whose products run at twice fp16's rate. A row scaled so that its largest
// value lies in [128, 256) is its digits' sum exactly, but for values below 2^-9 of the largest, which are off by up to 2^-17 of that. What
// bounds the tiles is the shared memory's bandwidth (operands, their conversion, scales), so that keys that need no conversion count for more
// than the instructions: 8192 x 8192, 8B shape, 690 us with keys converted to fp16, 620 so on the same day (640 to 680 from call to call since:
// the power limit, 0.81 to 0.86 PFLOP/s); 2.1 us a tile of 256 rows by 128 keys. Short prompts are bound by a block's start (5 us until its queries are
// operands) and end (2 us): 9 x 1500 rows, 2.7B shape, 244 to 249 us. Values' bytes that are NaN are looked for as they are converted (af_finite).
// ROWS: the groups have 128 rows each of 256, and keys in common. KEYS (up to 128 rows): the same rows, key tiles by turns; their sums
// are added up at the end. f32: one group with two tiles of scores; the tensor cores cut off what falls below a sum's last bits, always towards
// zero (2^-26 of it an addition: 1.8e-5 after 8192 keys), so that O is added to a sum of its own by the vector units every AT_FLUSH tiles (64 rows at
// 131072 keys: 1.7e-6 off with four, 1.2e-6 with two, which take 2 % longer). Keys may be shared out to the blocks of a cluster as well, which add
// up through shared memory.
//
// A tile's values have a power of two 2^u, not below the largest of their scales. For bf16 rows they are multiplied by s' 2^(7 - u) as they become
// fp16 (off by 2^-11 of themselves), so that a weight is one exponential, 2^(z - M + u - 7); for f32 rows values stay exact and weights
// are 2^(z - M) s', as fp16 plus the fp16 of the remainder. Either way they must stay below 2^16: the row's reference M is moved when
// z + u - 7 (f32: z + u) passes M + 15, to 9 below it, and the sums move along. A scale that is NaN or infinite counts as 0 and makes the token's scores NaN.
#include <cuda_fp8.h>

#include <algorithm>

#include "attention_fp8.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tc5_ptx.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

constexpr int AT_KEYS = 128, AT_PAGES = AT_KEYS / KV_PAGE, AT_THREADS = 512, AT_RING = 8;
constexpr int AT_FLUSH = 2, AT_NONE = INT32_MAX;
constexpr float AT_MOST = 15.f, AT_SET = 9.f;  // log2 of the largest weight, and of it when M is set
constexpr int AT_UP = 7, AT_LEAST = -80;       // values times 2^7 are below 2^16; smaller u would let a sum of 2^(z - M) pass 2^127

template <typename T, int DP, bool KEYS>
struct AtShape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PLANES = 2, TILES = KEYS ? 1 : 2;                      // of Q: digits, or fp16 and remainders
    static constexpr int K_STAGES = F32 ? 2 : 3, V_STAGES = 2, SETS = KEYS && !F32 ? 2 : 1;  // SETS: sums of a row
    static_assert(KEYS || !F32, "f32: tiles of 128 rows");
    static constexpr int TILE = 128 * DP * 2, K_TILE = F32 ? TILE : 128 * 128;  // bytes of 128 rows in fp16; of keys and of a plane of Q
    static constexpr int Q = PLANES * TILES * K_TILE, SMEM = Q + K_STAGES * K_TILE + V_STAGES * TILE + 1024;
    static constexpr int LDO = DP + 4, SUMS = 2 * 128 * LDO * 4;                // takes the operands' place
    static constexpr int WEIGHTS = (128 * TILES + AF_MAX_PARTS) * SETS * 4;              // of the sums of a block's share of rows, behind them
    static_assert(SUMS + WEIGHTS <= SMEM - 1024, "sums of both groups");
};

// log2 of the power of two not below a scale, given by its bits (positive and finite, or 0).
__device__ __forceinline__ int at_power(uint32_t bits) { return max((int)((bits + 0x7FFFFFu) >> 23) - 127, AT_LEAST); }

// Four values as e4m3, to nearest even.
__device__ __forceinline__ uint32_t at_digits(const float* x) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// tc5_wait for warps that are ahead of the others: it looks now and then, so that the others have the issue slots.
__device__ __forceinline__ bool at_wait_idle(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < 64; ++i) {
        if (tc5_peek(bar, parity)) return true;
        __nanosleep(100);
    }
    return tc5_wait(bar, parity);
}

__device__ __forceinline__ void at_init(uint64_t* bar, uint32_t arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(tc5_smem_u32(bar)), "r"(arrivals) : "memory");
}
__device__ __forceinline__ uint32_t at_idesc(int n, bool b_mn) { return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }
// Values as they lie: rows of 64 coordinates (128 bytes, swizzled) a token, 8 tokens 1024 bytes apart; the next 64 coordinates 128 tokens on.
__device__ __forceinline__ uint64_t at_desc_values(uint32_t saddr) {
    return (tc5_desc(saddr) & ~((uint64_t)0x3FFF << 16)) | (uint64_t)(128 * 128 >> 4) << 16;
}
__device__ __forceinline__ void at_mma_digits(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {  // e4m3 x e4m3, 32 columns
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
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
// 32 columns of the warp's lanes, two in a register pair.
__device__ __forceinline__ void at_ld32(uint32_t taddr, uint64_t (&v)[16]) {
    asm volatile(
        "{\n.reg .b32 r<32>;\n"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {r0, r1, r2, r3, r4, r5, r6, r7, r8, r9, r10, r11, r12, r13, r14, r15, r16, r17, r18, r19, r20, r21, r22, r23, r24, r25, r26, r27, r28, r29, r30, r31}, [%16];\n"
        "mov.b64 %0, {r0, r1};\n"
        "mov.b64 %1, {r2, r3};\n"
        "mov.b64 %2, {r4, r5};\n"
        "mov.b64 %3, {r6, r7};\n"
        "mov.b64 %4, {r8, r9};\n"
        "mov.b64 %5, {r10, r11};\n"
        "mov.b64 %6, {r12, r13};\n"
        "mov.b64 %7, {r14, r15};\n"
        "mov.b64 %8, {r16, r17};\n"
        "mov.b64 %9, {r18, r19};\n"
        "mov.b64 %10, {r20, r21};\n"
        "mov.b64 %11, {r22, r23};\n"
        "mov.b64 %12, {r24, r25};\n"
        "mov.b64 %13, {r26, r27};\n"
        "mov.b64 %14, {r28, r29};\n"
        "mov.b64 %15, {r30, r31};\n"
        "}\n"
        : "=l"(v[0]), "=l"(v[1]), "=l"(v[2]), "=l"(v[3]), "=l"(v[4]), "=l"(v[5]), "=l"(v[6]), "=l"(v[7]), "=l"(v[8]), "=l"(v[9]), "=l"(v[10]), "=l"(v[11]), "=l"(v[12]), "=l"(v[13]), "=l"(v[14]), "=l"(v[15])
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
__device__ __forceinline__ void at_wait_for(uint64_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+l"(v[0]), "+l"(v[1]), "+l"(v[2]), "+l"(v[3]), "+l"(v[4]), "+l"(v[5]), "+l"(v[6]), "+l"(v[7]), "+l"(v[8]), "+l"(v[9]), "+l"(v[10]), "+l"(v[11]), "+l"(v[12]), "+l"(v[13]), "+l"(v[14]), "+l"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void at_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void at_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void at_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void at_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void at_fence_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Two values an instruction, kept in register pairs.
__device__ __forceinline__ float2 at_two(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t at_mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t at_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t at_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float4 at_peer4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float at_max3(float a, uint64_t two) {
    const float2 f = at_two(two);
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(f.x), "f"(f.y));
    return d;
}

// 16 bytes of N tokens, PER apart, as fp16 to `to` (of the first) and u0, u1. Keys as they are; values without NaN and, for bf16 rows, times `by`. The second
// half of a row's threads (odd) swap the halves of their 16 bytes: eight threads' stores fall on 32 different banks. Back: whether values had NaN,
// of tokens less than `live` behind the first: past a sequence's end bytes may be anything, and to look for rows that see them would take 5 us.
template <bool F32, bool VALUES, int PER, int N>
__device__ __forceinline__ uint32_t at_convert(const uint4 (&raw)[N], const uint32_t (&by)[N], uint8_t* to, int u0, int u1, bool odd, int live) {
    uint32_t dropped = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        uint32_t h[8];
        af_halves(odd ? raw[i].z : raw[i].x, h[0], h[1]);
        af_halves(odd ? raw[i].w : raw[i].y, h[2], h[3]);
        af_halves(odd ? raw[i].x : raw[i].z, h[4], h[5]);
        af_halves(odd ? raw[i].y : raw[i].w, h[6], h[7]);
        if constexpr (VALUES) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[j] = af_finite(h[j], dropped, PER * i < live);
                if constexpr (!F32) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(h[j]) : "r"(by[i]));
            }
        }
        *reinterpret_cast<uint4*>(to + PER * i * 128 + u0) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(to + PER * i * 128 + u1) = make_uint4(h[4], h[5], h[6], h[7]);
    }
    return dropped;
}

template <typename T, int DP, bool KEYS>
__global__ void __launch_bounds__(AT_THREADS, 1) attention_tile_kernel(const AttentionFp8Args a, int parts, int tiles, const __grid_constant__ CUtensorMap map) {
    using Sh = AtShape<T, DP, KEYS>;
    constexpr bool F32 = Sh::F32;
    constexpr int K_STAGES = Sh::K_STAGES, V_STAGES = Sh::V_STAGES, ROWS = 128 * Sh::TILES;
    extern __shared__ uint8_t at_smem_raw[];
    __shared__ __align__(8) uint64_t k_full[K_STAGES], k_empty[K_STAGES], v_full[V_STAGES], v_empty[V_STAGES], s_full[2], p_full[2][2], o_done, o_full, q_full;
    __shared__ __align__(16) float k_scale[AT_RING][AT_KEYS], v_scale[AT_RING][F32 ? AT_KEYS : 4];
    __shared__ uint32_t gone_s[AT_RING];     // pages of the tile that are not there
    __shared__ int nan_from;                 // the first tile with value bytes that are NaN (AT_NONE: none)
    __shared__ __align__(16) uint32_t largest_s[AT_RING][4];  // scales of values that count, of 32 tokens each
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
    uint8_t *const ks_ = smem + Sh::Q, *const vs_ = ks_ + K_STAGES * Sh::K_TILE;
    // ── the block's keys ──
    const int last_row = tile.row0 + tile.n - 1;
    // Token and head of the block's row q: with rem = row0 % group, (rem + q) / group by a reciprocal is exact, since (rem + q + 1/2) / group is at
    // least 1 / (2 group) from a whole number and rem + q < 2^21
    const int tok_base = tile.row0 / group, rem = tile.row0 - tok_base * group;
    const float per_group = 1.f / (float)group;
    auto token_of = [&](int q) { return (int)(((float)(rem + q) + 0.5f) * per_group); };
    const int64_t q_first = (int64_t)(tile.first + tok_base);
    // offset of row q's head in a matrix of row stride ld
    auto offset_of = [&](int q, int64_t ld) {
        const int tok = token_of(q);
        return (q_first + tok) * ld + (int64_t)(head * group + rem + q - tok * group) * dim;
    };
    // ── queries: the first are on their way while the block sets itself up (8 prompts of 512 rows, 8B shape, 65.1 us, 62.1 so) ──
    constexpr int PER = DP / 8, AT_ONCE = 32 / PER, ROWS_OF = KEYS ? 16 : 32;  // threads of a row, rows at once, rows of a warp (KEYS: the groups share them out)
    constexpr int COUNT = ROWS_OF / AT_ONCE, BATCH = COUNT < 8 ? COUNT : 8;    // rows of a thread, and at a time, so that one's latencies hide the others'
    static_assert(!F32 || COUNT == BATCH, "f32: one batch");
    const int q_part = lane % PER, q_row = ROWS_OF * (warp & 7);
    const int64_t q_at = offset_of(q_row + lane % ROWS_OF, a.ldq);
    uint4 q_raw[BATCH][F32 ? 2 : 1], q_next[COUNT > BATCH ? BATCH : 1][F32 ? 2 : 1];
    auto load_q = [&](auto& to, int i0) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int r = (i0 + i) * AT_ONCE + lane / PER;
            const int64_t from = __shfl_sync(0xFFFFFFFFu, q_at, r);
#pragma unroll
            for (int e = 0; e < (F32 ? 2 : 1); ++e) {
                to[i][e] = make_uint4(0, 0, 0, 0);
                if (q_row + r < tile.n && 8 * q_part < dim) to[i][e] = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + from + 8 * q_part)[e];
            }
        }
    };
    if (warp < 8) load_q(q_raw, 0);
    const int pos_first = tile.len - tile.rows + tok_base, pos_last = tile.len - tile.rows + last_row / group;
    const int held = (int)min((int64_t)tile.len, (int64_t)a.c.max_pages * KV_PAGE);
    const int k_end = min(pos_last + 1, held), k_begin = a.window > 0 ? max(0, max(pos_first, 0) - a.window + 1) : 0;
    const int t_begin = k_begin / AT_KEYS, t_end = k_end > k_begin ? (k_end - 1) / AT_KEYS + 1 : t_begin;  // (k_end may be near 2^31)
    const int per = (t_end - t_begin + parts - 1) / parts;
    const int b_begin = min(t_end, t_begin + part * per), n_kv = min(t_end, b_begin + per) - b_begin;  // key tiles of the block
    const int groups = KEYS || tile.n > 128 ? 2 : 1, jobs = KEYS ? n_kv : groups * n_kv;  // job j is group j % groups'
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(tc5_smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (tid == 32) {
        nan_from = AT_NONE;
        for (int i = 0; i < K_STAGES; ++i) {
            at_init(&k_full[i], F32 ? 4 : 1);
            at_init(&k_empty[i], 1);
        }
        for (int i = 0; i < V_STAGES; ++i) {
            at_init(&v_full[i], 4);
            at_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            at_init(&s_full[i], 1);
            at_init(&p_full[i][0], 4);
            at_init(&p_full[i][1], 4);
        }
        at_init(&o_full, 1);
        at_init(&o_done, 1);
        at_init(&q_full, 8);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    at_before();
    __syncthreads();
    at_after();
    const uint32_t tmem = tmem_slot;  // S of the groups at columns 0 and 128, O at 256 and 256 + DP
    bool ok = true;
    // ── where the keys and values are ──
    const int32_t* const table = a.c.page_table + (int64_t)max(0, min(tile.slot, a.c.n_slots - 1)) * a.c.max_pages;
    auto page_of = [&](int kv) {  // lanes 0 to 7 (and so on): the tile's pages; -1: none
        const int index = (b_begin + kv) * AT_PAGES + (lane & 7);
        const int page = kv < n_kv && index < a.c.max_pages && index * KV_PAGE < k_end ? table[index] : -1;
        return page < a.c.n_pages ? max(page, -1) : -1;
    };
    const int page_rows = 2 * a.c.n_kv * KV_PAGE, page_bytes = page_rows * dim, to_values = a.c.n_kv * KV_PAGE;
    const float* const s_from = a.c.scales + head * KV_PAGE;
    // A value's scale as it counts: none of what no row of the block sees, nor of what is NaN or infinite
    auto counts = [&](float s, int token) { return s > 0.f && s < INFINITY && token >= k_begin && token < k_end; };
    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");  // 128 x 56 + 128 x 88 + 256 x 184 = 512 x 128 (f32: 56, 104, 176)
        if (!F32 && warp == 13) {
            // a lane looks after tokens 4 lane .. 4 lane + 3 of a tile, lanes 0 to 7 after a page
            int pages = page_of(0), next = page_of(1);
            float4 sk, sv;
            auto load = [&]() {
                const int page = __shfl_sync(0xFFFFFFFFu, pages, lane / 4);
                const float4* const at = reinterpret_cast<const float4*>(s_from + (int64_t)max(page, 0) * page_rows + 4 * lane % KV_PAGE);
                sk = __ldg(at);
                sv = page >= 0 ? __ldg(at + to_values / 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            };
            if (n_kv > 0) load();
            int issued = 0;
            for (int kv = 0; kv < n_kv; ++kv) {
                const int st = kv % K_STAGES, use = kv / K_STAGES, slot = kv % AT_RING, token = (b_begin + kv) * AT_KEYS + 4 * lane;
                if (use > 0) ok = __all_sync(0xFFFFFFFFu, at_wait_idle(&k_empty[st], (uint32_t)((use - 1) & 1)));
                if (!ok) break;
                const uint32_t gone = __ballot_sync(0xFFFFFFFFu, pages < 0) & 0xFFu;
                const float v[4] = {sv.x, sv.y, sv.z, sv.w}, k[4] = {sk.x, sk.y, sk.z, sk.w};
                float4 to;
                float* const f = &to.x;
                uint32_t big = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f[j] = v[j] < INFINITY && v[j] > -INFINITY ? af_number(k[j]) : __uint_as_float(0x7FC00000u);
                    if (counts(v[j], token + j)) big = max(big, __float_as_uint(v[j]));
                }
                *reinterpret_cast<float4*>(&k_scale[slot][4 * lane]) = to;
                big = __reduce_max_sync(0xFFFFFFFFu, big);
                if (lane == 0) {
                    *reinterpret_cast<uint4*>(largest_s[slot]) = make_uint4(big, big, big, big);
                    gone_s[slot] = gone;
                }
                __syncwarp();
                const uint32_t bar = tc5_smem_u32(&k_full[st]);
                if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"((uint32_t)(AT_PAGES - __popc(gone)) * KV_PAGE * 128u) : "memory");
                __syncwarp();
                if (lane < AT_PAGES && pages >= 0) tc5_tma_2d(tc5_smem_u32(ks_ + st * Sh::K_TILE) + lane * (KV_PAGE * 128), &map, 0, (pages * 2 * a.c.n_kv + head) * KV_PAGE, bar);
                issued = kv + 1;
                pages = next;
                next = page_of(kv + 2);
                if (kv + 1 < n_kv) load();
            }
            // no copy is on its way to this block when it goes on to the end
            for (int kv = max(0, issued - K_STAGES); kv < issued; ++kv) ok = tc5_wait(&k_full[kv % K_STAGES], (uint32_t)((kv / K_STAGES) & 1)) && ok;
        }
        if (warp == 12) {
        const bool leader = tc5_elect();
        const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        const uint32_t id_s = at_idesc(AT_KEYS, false), id_o = at_idesc(dim, true);
        const uint64_t qd = tc5_desc(tc5_smem_u32(smem)), kd = tc5_desc(tc5_smem_u32(ks_)), vd = at_desc_values(tc5_smem_u32(vs_));
        const int steps = F32 ? dim / 16 : (dim + 31) / 32;  // of 32 bytes
        if (jobs > 0) ok = __all_sync(0xFFFFFFFFu, tc5_wait(&q_full, 0));
        auto scores = [&](int j) {
            const int t = groups == 2 ? j & 1 : 0, kv = KEYS || groups == 1 ? j : j >> 1, st = kv % K_STAGES;
            if (KEYS || t == 0) ok = __all_sync(0xFFFFFFFFu, tc5_wait(&k_full[st], (uint32_t)((kv / K_STAGES) & 1)));
            if (!ok) return;
            at_after();
            if (leader) {
                const uint64_t q = qd + (uint64_t)((KEYS ? 0 : t) * (Sh::K_TILE >> 4)), k = kd + (uint64_t)(st * (Sh::K_TILE >> 4));
#pragma unroll
                for (int p = Sh::PLANES - 1; p >= 0; --p)
                    for (int s = 0; s < steps; ++s) {
                        const uint64_t at = (uint64_t)((s >> 2) * (128 * 128 >> 4) + (s & 3) * 2), from = q + at + (uint64_t)(p * Sh::TILES * (Sh::K_TILE >> 4));
                        const uint32_t more = p != Sh::PLANES - 1 || s > 0;
                        if constexpr (F32) tc5_mma(tm + 128u * t, from, k + at, id_s, more);
                        else at_mma_digits(tm + 128u * t, from, k + at, id_s, more);
                    }
                tc5_commit(&s_full[t]);
                if (KEYS || t == groups - 1) tc5_commit(&k_empty[st]);
            }
            __syncwarp();
        };
        for (int j = 0; j < (F32 ? 1 : groups) && j < jobs && ok; ++j) scores(j);
        for (int j = 0; j < jobs && ok; ++j) {
            if (F32 && j + 1 < jobs) scores(j + 1);  // into the other tile of scores
            if (!ok) break;
            const int t = groups == 2 ? j & 1 : 0, i = groups == 2 ? j >> 1 : j, kv = KEYS ? j : i, st = kv % V_STAGES;
            if (KEYS || t == 0) ok = __all_sync(0xFFFFFFFFu, tc5_wait(&v_full[st], (uint32_t)((kv / V_STAGES) & 1)));
#pragma unroll 1
            for (int half = 0; half < 2 && ok; ++half) {  // three quarters of the tile's keys, the last
                ok = __all_sync(0xFFFFFFFFu, tc5_wait(&p_full[t][half], (uint32_t)(i & 1)));
                if (!ok) break;
                at_after();
                if (leader) {
                    const uint64_t v = vd + (uint64_t)(st * (Sh::TILE >> 4) + half * (6 * 2048 >> 4));
                    const uint32_t w = tm + 128u * t + (F32 ? 96u : 48u) * half;
#pragma unroll 2
                    for (int s = 0; s < (half ? 2 : 6); ++s)
#pragma unroll
                        for (int p = F32 ? 1 : 0; p >= 0; --p)
                            at_mma_tmem(tm + 256u + (uint32_t)(F32 ? 0 : DP * t), w + (uint32_t)(F32 ? 32 * (s / 2) + 16 * p + 8 * (s % 2) : 8 * s), v + (uint64_t)(s * (2048 >> 4)), id_o,
                                        (F32 ? j % AT_FLUSH > 0 : i > 0) || half > 0 || s > 0 || (F32 && p == 0));
                    if (half == 1 && (KEYS || t == groups - 1)) tc5_commit(&v_empty[st]);
                    if (F32 && half == 1) tc5_commit(&o_done);
                }
                __syncwarp();
            }
            if (!ok) break;
            if (!F32 && j + groups < jobs) scores(j + groups);
        }
        if (jobs > 0) {
            if (leader) tc5_commit(&o_full);  // (after a wait that ran out too: no product is under way when its tensor memory is given back)
            __syncwarp();
            // no arrival is on its way to this block when it goes on to the end
            for (int kv = max(0, n_kv - K_STAGES); kv < n_kv; ++kv) ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&k_empty[kv % K_STAGES], (uint32_t)((kv / K_STAGES) & 1)));
            for (int kv = max(0, n_kv - V_STAGES); kv < n_kv; ++kv) ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&v_empty[kv % V_STAGES], (uint32_t)((kv / V_STAGES) & 1)));
            ok = __all_sync(0xFFFFFFFFu, tc5_wait(&o_full, 0) && ok);
        }
        }
        if (parts > 1) {
            cluster_sync();
            cluster_sync();
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(F32 ? 104 : 88));
        // of a tile: 16 bytes of tokens tok0 + PER i a copy; a warp's threads have whole rows, so that a request is few lines
        constexpr int CH = DP / 16, N = CH, PER = 128 / CH;
        const int p = tid - 256, ch = p % CH, tok0 = p / CH;
        const uint8_t* const k_from = a.c.values + ((int64_t)head * KV_PAGE + tok0 % KV_PAGE) * dim + 16 * ch;
        const uint8_t* const v_from = k_from + (int64_t)to_values * dim;
        // (of a page that is not there the first one's rows are taken: nobody sees them)
        auto load = [&](uint4 (&raw)[N], const uint8_t* from, int pages) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int page = __shfl_sync(0xFFFFFFFFu, pages, (tok0 + PER * i) / KV_PAGE);
                if (16 * ch < dim) raw[i] = __ldg(reinterpret_cast<const uint4*>(from + (int64_t)max(page, 0) * page_bytes));
            }
        };
        const bool odd = ch / 4;
        const int x = tok0 & 7, u0 = ((2 * (ch % 4) + odd) ^ x) * 16, u1 = ((2 * (ch % 4) + 1 - odd) ^ x) * 16, row0 = ch / 4 * (128 * 128) + tok0 * 128;
        auto hand_over = [&](uint64_t* bar) {
            at_fence_smem();
            __syncwarp();
            if (lane == 0) tc5_arrive(bar);
        };
        [[maybe_unused]] uint4 raw_k[N];
        uint4 raw_v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) raw_k[i] = raw_v[i] = make_uint4(0, 0, 0, 0);
        [[maybe_unused]] float sk = 0.f, sv = 0.f;  // f32: of token p
        float four[4] = {};                         // bf16: of the values of tokens 4 lane .. 4 lane + 3
        auto load_scales = [&](int pages) {
            const int page = __shfl_sync(0xFFFFFFFFu, pages, F32 ? p / KV_PAGE : lane / 4);
            const float* const at = s_from + (int64_t)max(page, 0) * page_rows;
            if constexpr (F32) {
                sk = __ldg(at + p % KV_PAGE);
                sv = page >= 0 ? __ldg(at + to_values + p % KV_PAGE) : 0.f;
            } else {
                const float4 f = __ldg(reinterpret_cast<const float4*>(at + to_values + 4 * lane % KV_PAGE));
                four[0] = f.x; four[1] = f.y; four[2] = f.z; four[3] = f.w;
            }
        };
        int pages = page_of(0), next = page_of(1);  // (looked up a tile ahead of the rows, which are requested a tile ahead of their use)
        if (n_kv > 0) {
            if constexpr (F32) load(raw_k, k_from, pages);
            load_scales(pages);
            load(raw_v, v_from, pages);
        }
        for (int kv = 0; kv < n_kv; ++kv) {
            const int key0 = (b_begin + kv) * AT_KEYS;
            uint32_t by[N] = {};  // what values are multiplied by, as pairs of fp16
            if constexpr (F32) {
                const int st = kv % K_STAGES, use = kv / K_STAGES, slot = kv % AT_RING;
                const uint32_t gone = __ballot_sync(0xFFFFFFFFu, pages < 0) & 0xFFu;
                if (use > 0) ok = __all_sync(0xFFFFFFFFu, at_wait_idle(&k_empty[st], (uint32_t)((use - 1) & 1)));
                if (!ok) break;
                at_convert<F32, false, PER>(raw_k, by, ks_ + st * Sh::K_TILE + row0, u0, u1, odd, 0);
                const float v = counts(sv, key0 + p) ? sv : 0.f;
                k_scale[slot][p] = sv < INFINITY && sv > -INFINITY ? af_number(sk) : __uint_as_float(0x7FC00000u);
                v_scale[slot][p] = v;
                const uint32_t big = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v));
                if (lane == 0) largest_s[slot][warp - 8] = big;
                if (p == 0) gone_s[slot] = gone;
                hand_over(&k_full[st]);
                if (kv + 1 < n_kv) load(raw_k, k_from, next);
            } else {
                const int mine = __shfl_sync(0xFFFFFFFFu, pages, lane / 4), token = key0 + 4 * lane;
                uint32_t big = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (mine < 0 || !counts(four[j], token + j)) four[j] = 0.f;
                    big = max(big, __float_as_uint(four[j]));
                }
                const float lift = __uint_as_float((uint32_t)(127 + AT_UP - at_power(__reduce_max_sync(0xFFFFFFFFu, big))) << 23);
                const uint32_t two0 = af_pack(four[0] * lift, four[1] * lift), two1 = af_pack(four[2] * lift, four[3] * lift);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int tok = tok0 + PER * i;
                    const uint32_t a0 = __shfl_sync(0xFFFFFFFFu, two0, tok / 4), a1 = __shfl_sync(0xFFFFFFFFu, two1, tok / 4);
                    by[i] = __byte_perm(tok & 2 ? a1 : a0, 0, tok & 1 ? 0x3232 : 0x1010);
                }
            }
            if (kv + 1 < n_kv) load_scales(next);
            const int st = kv % V_STAGES, use = kv / V_STAGES;
            if (use > 0) ok = __all_sync(0xFFFFFFFFu, at_wait_idle(&v_empty[st], (uint32_t)((use - 1) & 1)));
            if (!ok) break;
            if (at_convert<F32, true, PER>(raw_v, by, vs_ + st * Sh::TILE + row0, u0, u1, odd, k_end - key0 - tok0) != 0) atomicMin(&nan_from, kv);
            hand_over(&v_full[st]);
            pages = next;
            next = page_of(kv + 2);
            if (kv + 1 < n_kv) load(raw_v, v_from, pages);
        }
        if (parts > 1) {
            cluster_sync();
            cluster_sync();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(F32 ? 176 : 184));
        const int t = warp >> 2, r = 32 * (warp & 3) + lane, row = (KEYS ? 0 : 128 * t) + r;  // of the block's rows
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16), O = lanes + 256u + (uint32_t)(F32 ? 0 : DP * t);
        [[maybe_unused]] const uint32_t O_sum = O + DP;  // f32: what O has been added to
        const int pos = pos_first + token_of(row);
        const int limit = row < tile.n ? min(pos, held - 1) : -1, low = a.window > 0 ? max(pos, 0) - a.window + 1 : 0;
        // keys that all rows of the group see
        const int row_a = KEYS ? 0 : 128 * t, row_b = min(row_a + 127, tile.n - 1);
        const int whole_to = min(pos_first + token_of(row_a), held - 1), whole_from = a.window > 0 ? max(pos_first + token_of(row_b), 0) - a.window + 1 : 0;
        const int mine = F32 ? (t == 0 ? jobs : 0) : t >= groups ? 0 : (jobs - t + groups - 1) / groups;  // jobs of the group
        // ── queries as operands, eight values a thread and row ──
        float c;  // scale log2(e) / what the row is multiplied by; never 0, since scores of -inf are multiplied by it
        {
#pragma unroll 1
            for (int i0 = 0; i0 < COUNT; i0 += BATCH) {
                if constexpr (COUNT > BATCH)
                    if (i0 + BATCH < COUNT) load_q(q_next, i0 + BATCH);
                uint32_t most[BATCH];  // absolute values as whole numbers: NaN is the largest
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    if constexpr (F32) {
                        const uint4 v = q_raw[i][0], w = q_raw[i][1];
                        most[i] = max(max(max(v.x & 0x7FFFFFFFu, v.y & 0x7FFFFFFFu), max(v.z & 0x7FFFFFFFu, v.w & 0x7FFFFFFFu)),
                                      max(max(w.x & 0x7FFFFFFFu, w.y & 0x7FFFFFFFu), max(w.z & 0x7FFFFFFFu, w.w & 0x7FFFFFFFu)));
                    } else {
                        const uint4 v = q_raw[i][0];
                        most[i] = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
                        most[i] = max(most[i] & 0xFFFF0000u, most[i] << 16);  // as f32
                    }
                }
#pragma unroll
                for (int o = PER / 2; o > 0; o >>= 1)
#pragma unroll
                    for (int i = 0; i < BATCH; ++i) most[i] = max(most[i], __shfl_xor_sync(0xFFFFFFFFu, most[i], o));
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int q = q_row + (i0 + i) * AT_ONCE + lane / PER;
                    float by, back;
                    af_row_scale(__uint_as_float(most[i]), F32 ? 12 : 7, by, back);
                    if (a.scale < 0.f) by = -by;
                    if (q_part == 0) row_factor[q] = fmaxf(back * fabsf(a.scale) * AF_LOG2E, 0x1p-149f);
                    float x[8];
                    if constexpr (F32) {
                        const uint32_t w[8] = {q_raw[i][0].x, q_raw[i][0].y, q_raw[i][0].z, q_raw[i][0].w, q_raw[i][1].x, q_raw[i][1].y, q_raw[i][1].z, q_raw[i][1].w};
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(w[j]) * by;
                        uint4 hi, lo;
                        uint32_t *const h = &hi.x, *const l = &lo.x;
#pragma unroll
                        for (int j = 0; j < 4; ++j) af_split(x[2 * j], x[2 * j + 1], h[j], l[j]);
                        uint8_t* const to = smem + q / 128 * Sh::K_TILE + q_part / 8 * (128 * 128) + q % 128 * 128 + ((q_part % 8) ^ (q & 7)) * 16;
                        *reinterpret_cast<uint4*>(to) = hi;
                        *reinterpret_cast<uint4*>(to + Sh::TILES * Sh::K_TILE) = lo;
                    } else {
                        const uint32_t w[4] = {q_raw[i][0].x, q_raw[i][0].y, q_raw[i][0].z, q_raw[i][0].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            x[2 * j] = __uint_as_float(w[j] << 16) * by;
                            x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u) * by;
                        }
                        uint32_t hi[2], lo[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            hi[j] = at_digits(x + 4 * j);
                            uint32_t h0, h1;
                            af_halves(hi[j], h0, h1);
                            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                            const float d[4] = {x[4 * j] - f0.x, x[4 * j + 1] - f0.y, x[4 * j + 2] - f1.x, x[4 * j + 3] - f1.y};
                            lo[j] = at_digits(d);
                        }
                        uint8_t* const to = smem + q / 128 * Sh::K_TILE + q % 128 * 128 + ((q_part / 2) ^ (q & 7)) * 16 + q_part % 2 * 8;
                        *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
                        *reinterpret_cast<uint2*>(to + Sh::TILES * Sh::K_TILE) = make_uint2(lo[0], lo[1]);
                    }
                }
                if constexpr (COUNT > BATCH) {
#pragma unroll
                    for (int i = 0; i < BATCH; ++i) q_raw[i][0] = q_next[i][0];
                }
            }
            at_fence_smem();
            if constexpr (KEYS) asm volatile("barrier.cta.sync 1, 256;\n" ::: "memory");  // (the factors of rows that other warps have done)
            else __syncwarp();
            if (lane == 0) tc5_arrive(&q_full);
            c = row_factor[row];
        }
        float m = -INFINITY, l = 0.f;
        for (int job = 0; job < mine; ++job) {
            const int of = F32 ? job & 1 : t, i = F32 ? job >> 1 : job;  // the tile of scores, its how manieth use
            const int kv = KEYS && !F32 ? 2 * i + t : job, key0 = (b_begin + kv) * AT_KEYS, slot = kv % AT_RING;
            const uint32_t S = lanes + 128u * of;
            ok = __all_sync(0xFFFFFFFFu, tc5_wait(&s_full[of], (uint32_t)(i & 1)));
            if (!ok) break;
            at_after();
            const bool flush = F32 && job > 0 && job % AT_FLUSH == 0;
            if (flush) {
                ok = __all_sync(0xFFFFFFFFu, tc5_wait(&o_done, (uint32_t)((job - 1) & 1)));
                if (!ok) break;
                at_after();
#pragma unroll 1
                for (int d = 0; d < dim; d += 16) {
                    uint32_t o[16], sum[16];
                    tc5_ld16(O + d, o);
                    if (job > AT_FLUSH) tc5_ld16(O_sum + d, sum);
                    at_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) + (job > AT_FLUSH ? __uint_as_float(sum[j]) : 0.f));
                    at_st16(O_sum + d, o);
                }
                at_wait_st();
            }
            uint64_t s[4][16];  // 32 scores each, two a register pair
#pragma unroll
            for (int q = 0; q < 4; ++q) at_ld32(S + 32 * q, s[q]);
            const uint4 big = *reinterpret_cast<const uint4*>(largest_s[slot]);
            const int power = at_power(max(max(big.x, big.y), max(big.z, big.w))) - (F32 ? 0 : AT_UP);
            const uint32_t gone = gone_s[slot];
            const bool masked = gone != 0 || key0 < whole_from || key0 + AT_KEYS - 1 > whole_to;
            float b0 = -INFINITY, b1 = -INFINITY, b2 = -INFINITY, b3 = -INFINITY;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                at_wait_for(s[q]);
                const ulonglong2* const f = reinterpret_cast<const ulonglong2*>(&k_scale[slot][32 * q]);
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    const ulonglong2 w = f[k / 2];
                    s[q][k] = at_mul2(s[q][k], w.x);
                    s[q][k + 1] = at_mul2(s[q][k + 1], w.y);
                }
            }
            if (masked) {  // (a branch around it: selected at each value it would be three instructions more for every tile)
                const int hi = limit - key0, lo = low - key0;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int from = lo - 32 * q, to = hi - 32 * q;
                    uint32_t bits = to >= 31 ? 0xFFFFFFFFu : to < 0 ? 0u : (2u << to) - 1u;  // of the keys that the row sees
                    bits = from <= 0 ? bits : from > 31 ? 0u : bits & (0xFFFFFFFFu << from);
                    const uint32_t no = gone >> (2 * q);
                    bits &= ~((no & 1 ? 0xFFFFu : 0u) | (no & 2 ? 0xFFFF0000u : 0u));
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float2 f = at_two(s[q][k]);
                        s[q][k] = pack2(bits >> (2 * k) & 1 ? f.x : -INFINITY, bits >> (2 * k + 1) & 1 ? f.y : -INFINITY);
                    }
                    asm volatile("" ::: "memory");
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    b0 = at_max3(b0, s[q][k]);
                    b1 = at_max3(b1, s[q][k + 1]);
                    b2 = at_max3(b2, s[q][k + 2]);
                    b3 = at_max3(b3, s[q][k + 3]);
                }
            const float x = fmaf(fmaxf(fmaxf(b0, b1), fmaxf(b2, b3)), c, (float)power);
            const bool moves = x > m + AT_MOST;
            if (__any_sync(0xFFFFFFFFu, moves)) {
                const float to = moves ? x - AT_SET : m, by = moves ? ex2_approx(m - to) : 1.f;  // (m = -inf: 0)
                m = to;
                l *= by;
                auto scale = [&](uint32_t at) {
#pragma unroll 1
                    for (int d = 0; d < dim; d += 16) {
                        uint32_t o[16];
                        tc5_ld16(at + d, o);
                        at_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * by);
                        at_st16(at + d, o);
                    }
                };
                if constexpr (F32) {
                    if (job % AT_FLUSH > 0) {
                        ok = __all_sync(0xFFFFFFFFu, tc5_wait(&o_done, (uint32_t)((job - 1) & 1)));
                        if (!ok) break;
                        at_after();
                        scale(O);
                    }
                    if (job >= AT_FLUSH) scale(O_sum);
                } else if (i > 0) {
                    scale(O);
                }
            }
            const float base = (m == -INFINITY ? 0.f : -m) + (F32 ? 0.f : (float)power);
            const uint64_t c2 = pack2(c, c), base2 = pack2(base, base);
            uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t w_hi[16];
                [[maybe_unused]] uint32_t w_lo[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    float2 p = at_two(at_fma2(s[q][k], c2, base2));
                    p.x = ex2_approx(p.x);
                    p.y = ex2_approx(p.y);
                    const uint64_t pair = pack2(p.x, p.y);
                    if (k % 2) sum1 = at_add2(sum1, pair);
                    else sum0 = at_add2(sum0, pair);
                    if constexpr (F32) {
                        const float2 w = at_two(at_mul2(pair, *reinterpret_cast<const uint64_t*>(&v_scale[slot][32 * q + 2 * k])));
                        af_split(w.x, w.y, w_hi[k], w_lo[k]);
                    } else {
                        w_hi[k] = af_pack(p.x, p.y);
                    }
                }
                if constexpr (F32) {
                    at_st16(S + 32 * q, w_hi);
                    at_st16(S + 32 * q + 16, w_lo);
                } else {
                    at_st16(S + 16 * q, w_hi);
                }
                if (q >= 2) {
                    at_wait_st();
                    at_before();
                    __syncwarp();
                    if (lane == 0) tc5_arrive(&p_full[of][q - 2]);
                }
            }
            const float2 sum = at_two(at_add2(sum0, sum1));
            l = fmaf(sum.x + sum.y, F32 ? 1.f : __uint_as_float((uint32_t)(127 - power) << 23), l);
        }
        // what comes now takes the operands' place: the products have been made, or there are none and the queries have been written
        if (jobs > 0) ok = __all_sync(0xFFFFFFFFu, ok && tc5_wait(&o_full, 0));
        else asm volatile("barrier.cta.sync 1, 256;\n" ::: "memory");
        at_after();
        if (jobs > 0 && ok && nan_from != AT_NONE) {  // (written before the products whose end has been waited for; bytes that nobody sees may be among them)
#pragma unroll 1
            for (int kv = nan_from; kv < n_kv; ++kv) {
                const int key0 = (b_begin + kv) * AT_KEYS;
                uint32_t tokens[AT_KEYS / 32];
                af_nan_tokens(a.c, table, head, key0, k_end, tokens);
#pragma unroll
                for (int q = 0; q < AT_KEYS / 32; ++q)
                    if (af_sees(tokens[q], key0 + 32 * q, low, limit)) l = __uint_as_float(0x7FC00000u);
            }
        }
        T* const out = static_cast<T*>(a.out);
        if (!KEYS && parts == 1) {  // (bf16 rows, 256 of them)
            const float by = l == 0.f || mine == 0 ? 0.f : 1.f / l;
            // A warp's 32 rows through its part of shared memory (the operands have been read), so that stores write whole lines
            constexpr int UNITS = DP / 8, AT_ONCE = 32 / UNITS;  // pieces of a row, rows a store
            uint8_t* const mem = smem + warp * (32 * DP * 2);
#pragma unroll 1
            for (int d = 0; d < DP; d += 32) {
                uint64_t o[16];
                if (mine > 0 && ok) {
                    at_ld32(O + d, o);
                    at_wait_for(o);
                }
                const uint64_t by2 = pack2(by, by);
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    uint4 w;
                    uint32_t* const u = &w.x;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float2 f = at_two(mine > 0 ? at_mul2(o[j + q], by2) : 0);
                        u[q] = pack_bf16(f.x, f.y);
                    }
                    const int unit = (d + 2 * j) / 8;
                    *reinterpret_cast<uint4*>(mem + lane * (16 * UNITS) + ((unit & ~7) | ((unit ^ lane) & 7)) * 16) = w;
                }
            }
            __syncwarp();
            const int row_w = 128 * t + 32 * (warp & 3), unit = lane % UNITS;
            const int64_t mine_to = offset_of(row_w + lane, a.ldo);
#pragma unroll 4
            for (int q0 = 0; ok && q0 < 32; q0 += AT_ONCE) {
                const int q = q0 + lane / UNITS;
                const int64_t to = __shfl_sync(0xFFFFFFFFu, mine_to, q);
                const uint4 w = *reinterpret_cast<const uint4*>(mem + q * (16 * UNITS) + ((unit & ~7) | ((unit ^ q) & 7)) * 16);
                if (row_w + q < tile.n && unit * 8 < dim) *reinterpret_cast<uint4*>(out + to + unit * 8) = w;
            }
        } else {
            float* const sums = reinterpret_cast<float*>(smem);  // [group][row][LDO], over the operands, which have been read
            float* const weights = sums + Sh::SUMS / 4;          // [row of the block's share][sum]
#pragma unroll 1
            for (int d = 0; d < dim; d += 32) {
                uint64_t o[16];
                if (mine > 0 && ok) {
                    at_ld32(O + d, o);
                    at_wait_for(o);
                    if (F32 && mine > AT_FLUSH) {
                        uint64_t sum[16];
                        at_ld32(O_sum + d, sum);
                        at_wait_for(sum);
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = at_add2(o[j], sum[j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = 0;
                }
                if (t >= Sh::SETS && KEYS) break;  // (f32: the second group has no sum)
#pragma unroll
                for (int j = 0; j < 16; j += 2)
                    if (d + 2 * j < dim) *reinterpret_cast<ulonglong2*>(&sums[(128 * t + r) * Sh::LDO + d + 2 * j]) = make_ulonglong2(o[j], o[j + 1]);
            }
            part_m[t][r] = m;
            part_l[t][r] = l;
            asm volatile("barrier.cta.sync 1, 256;\n" ::: "memory");
            if (parts > 1) cluster_sync();
            // The blocks share the rows out: row q of the block's is part + parts q of the tile. Sum s of a row is part s / SETS's, group s % SETS's
            // (KEYS) or its own group's.
            constexpr int SETS = Sh::SETS;
            const int sets = parts * SETS, rows_here = (tile.n - part + parts - 1) / parts;
            const int width = sets > 1 ? 1 << (32 - __clz(sets - 1)) : 1, x = lane & (width - 1);  // lanes of a row
#pragma unroll 1
            for (int q0 = tid / 32 * (32 / width); q0 < rows_here; q0 += 256 / width) {
                const int q = q0 + lane / width;
                float m = -INFINITY, l = 0.f;
                if (q < rows_here && x < sets) {
                    const int of = part + parts * q, g = KEYS ? x % SETS : of / 128;
                    const uint32_t at_m = smem_addr(&part_m[g][of % 128]), at_l = smem_addr(&part_l[g][of % 128]);
                    m = parts > 1 ? ld_peer(peer_smem(at_m, x / SETS)) : part_m[g][of % 128];
                    l = parts > 1 ? ld_peer(peer_smem(at_l, x / SETS)) : part_l[g][of % 128];
                }
                float top = m;
                for (int o = width / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                const float w = m == -INFINITY ? 0.f : ex2_approx(m - top);
                float total = l * w;
                for (int o = width / 2; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
                if (q < rows_here && x < sets) weights[q * sets + x] = w == 0.f || total == 0.f ? 0.f : w / total;
            }
            asm volatile("barrier.cta.sync 1, 256;\n" ::: "memory");
            const int quads = dim / 4;
            constexpr int SUMS = 8;  // on their way at a time: a load from another block takes half a microsecond
#pragma unroll 1
            for (int e = tid; e < rows_here * quads; e += 256) {
                const int q = e / quads, d = 4 * (e - q * quads), of = part + parts * q;
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                for (int x0 = 0; x0 < sets; x0 += SUMS) {
                    float4 v[SUMS];
#pragma unroll
                    for (int i = 0; i < SUMS; ++i) {
                        if (x0 + i >= sets) break;
                        const int x = x0 + i;
                        const float* const src = sums + ((KEYS ? x % SETS : of / 128) * 128 + of % 128) * Sh::LDO + d;
                        v[i] = parts > 1 ? at_peer4(peer_smem(smem_addr(src), x / SETS)) : *reinterpret_cast<const float4*>(src);
                    }
#pragma unroll
                    for (int i = 0; i < SUMS; ++i) {
                        if (x0 + i >= sets) break;
                        const float w = weights[q * sets + x0 + i];
                        y.x = fmaf(v[i].x, w, y.x);
                        y.y = fmaf(v[i].y, w, y.y);
                        y.z = fmaf(v[i].z, w, y.z);
                        y.w = fmaf(v[i].w, w, y.w);
                    }
                }
                T* const to = out + offset_of(of, a.ldo) + d;
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
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

// Microseconds of a tile of keys, of a block's start and end, and of adding parts up. KEYS: fitted to 64 calls (3 to 35 rows a head, 240 to 32768 keys,
// 1 to 32 sequences, 8B, 1.5B and 0.5B shapes), from which they are 3 to 8 % off; ROWS: 512 rows at 8704 of the 8B shape, taken for all head sizes. Other
// calls are not checked against them; head sizes between 64 and 128 take 128's.
template <typename T, int DP, bool KEYS>
struct AtTimes {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr double PIECE = !KEYS ? 2.2 : F32 ? (DP == 128 ? 3.4 : 2.5) : DP == 128 ? 1.7 : 1.2;
    static constexpr double FIXED = !KEYS ? 9. : F32 ? (DP == 128 ? 6.5 : 5.5) : DP == 128 ? 7. : 6.5, JOINED = !KEYS ? 5. : F32 ? 2.5 : DP == 128 ? 3.5 : 3.;
};

template <typename T, int DP, bool KEYS>
static cudaError_t launch_tiles(const AttentionFp8Args& a, cudaStream_t st, AfShare* plan) {
    using Sh = AtShape<T, DP, KEYS>;
    static PerDeviceOnce once;
    static ClusterFits fits[SP_MAX_DEVICES];
    const auto kernel = attention_tile_kernel<T, DP, KEYS>;
    ClusterFits& mine = fits[current_device_index()];
    cudaError_t e = once.run([&] { return af_fits(reinterpret_cast<const void*>(kernel), AT_THREADS, Sh::SMEM, &mine); });
    if (e != cudaSuccess) return e;
    const int64_t rows = (int64_t)a.max_rows * (a.n_heads / a.c.n_kv), height = 128 * Sh::TILES, tiles = (rows + height - 1) / height, clusters = tiles * a.c.n_kv * a.n_seqs;
    using At = AtTimes<T, DP, KEYS>;
    const AfShare share = af_share(mine, clusters, (af_keys(a) + AT_KEYS - 1) / AT_KEYS, At::PIECE, At::FIXED, At::JOINED);
    const int parts = share.parts;
    if (plan) {
        *plan = share;
        return cudaSuccess;
    }
    CUtensorMap map{};
    if (!Sh::F32 && (e = af_page_map(a.c, &map)) != cudaSuccess) return e;
    e = launch_pdl_cluster(kernel, dim3((unsigned)(tiles * a.c.n_kv), (unsigned)a.n_seqs, (unsigned)parts), dim3(AT_THREADS), Sh::SMEM, st, parts, a, parts, (int)tiles, map);
    return e != cudaSuccess ? e : count_launch_and_check();
}

template <typename T, int DP>
static cudaError_t tiles_as(const AttentionFp8Args& a, cudaStream_t st, AfShare* plan) {
    if constexpr (sizeof(T) == 4) return launch_tiles<T, DP, true>(a, st, plan);
    else return (int64_t)a.max_rows * (a.n_heads / a.c.n_kv) <= 128 ? launch_tiles<T, DP, true>(a, st, plan) : launch_tiles<T, DP, false>(a, st, plan);
}
cudaError_t launch_attention_fp8_tiles(const AttentionFp8Args& a, bool bf, cudaStream_t st, AfShare* plan) {
    if (a.c.dim <= 64) return bf ? tiles_as<bf16, 64>(a, st, plan) : tiles_as<float, 64>(a, st, plan);
    return bf ? tiles_as<bf16, 128>(a, st, plan) : tiles_as<float, 128>(a, st, plan);
}

}  // namespace sp
