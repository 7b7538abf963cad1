// Attention of the newest tokens of sequences over a paged cache of 8-bit rows (cache_fp8.h).
//
//   z_k = scale (q . K_k) s_k,   o = sum_k e^(z_k - m) s'_k V_k / sum_k e^(z_k - m)
//
// with e4m3 rows K_k, V_k and their scales s_k, s'_k; a row sees keys k <= its position, of which the newest `window`; one that sees none
// gives zeros. The queries of a key head are rows of one product (row = token x heads per key head + head), so that its keys are read
// once for all of them.
//
// Precision. e4m3 values are exact in fp16, the scales are applied in f32. Here (few rows; attention_fp8_tile.cu has its own) a row of q is
// multiplied by a power of two so that its largest value lies in [2^12, 2^13): bf16 values are then exact in fp16 (down to 2^-30 of the largest),
// f32 values are taken as fp16 plus the fp16 of the remainder. The weights e^(z - m) s' enter the second product as fp16 (11 bits, where the result
// has bf16's 8) or, for f32, as fp16 plus remainder, multiplied by a power of two that keeps them out of fp16's subnormals: with the largest scale
// so far, R, rounded up to a power of two and e^(z - m) <= 2^LAZY, the weights are e^(z - m) s' 2^(15 - LAZY) / R <= 2^15. Sums, maxima and the
// output are f32.
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_fp8.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "ring.h"
#include "tc5_ptx.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

// ── Few rows: mma.sync, a warp takes 32 keys at a time ──
// The cache is read once, which is what bounds it: every warp keeps asynchronous copies in flight. Keys and values are the first operands of
// K q^T and V^T P^T, 16 keys or coordinates high, so that eight rows are a product's width. A thread's part of a product of 16 columns is four
// neighbouring bytes of a key's row (the order of columns does not matter where q has the same), and of values it has four tokens'
// 16 neighbouring coordinates, two a product. So nothing is rearranged but pairs of tokens' bytes, and the weights, which two 8 x 8
// transpositions make the second product's operand. (e4m3 operands of mma.sync are converted to fp16 at every use on this GPU: two digits
// of q against the keys' own bytes took 982 instructions for 32 keys.) A page's keys or values of a head are one TMA copy, whose 128-byte
// swizzle lets eight threads' reads fall on 32 different banks; copied by threads, 16 bytes each, every one was a request of its own to L2:
// 131072 keys of the 8B shape 106 us, 74 so (61 with blocks of 12 warps).
// Keys are shared out to the warps of a block and the blocks of a cluster, which add up their parts through shared memory: no workspace.
constexpr int AR_KEYS = 32, AR_PAGES = AR_KEYS / KV_PAGE, AR_FLUSH = 8;

template <typename T, int DP, int NT, int W>
struct ArShape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PLANES = F32 ? 2 : 1, STEPS = DP / 16, CHUNKS = DP / 64;       // of q: products of 16 columns
    static constexpr int STAGES = 2;
    static constexpr int PAGE = KV_PAGE * 128, STAGE = 2 * AR_PAGES * PAGE, SCALES = 2 * AR_KEYS * 4;  // [page][keys, values], their scales
    static constexpr int Q = NT * PLANES * STEPS * 256, RING = W * STAGES * (STAGE + SCALES);
    static constexpr int ROWS = 8 * NT, LDO = DP + 4;
    static constexpr int SUMS = W * ROWS * LDO * 4;  // takes the ring's place
    static constexpr int SMEM = Q + (RING > SUMS ? RING : SUMS) + 1024;
};

__device__ __forceinline__ uint32_t af_transpose(uint32_t v) {  // of an 8 x 8 matrix of 16-bit values, a row of pairs four threads
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(v));
    return d;
}

template <typename T, int DP, int NT, int W>
__global__ void __launch_bounds__(32 * W, W == 4 ? 3 : 1) attention_rows_kernel(const AttentionFp8Args a, int parts, const __grid_constant__ CUtensorMap map) {
    using Sh = ArShape<T, DP, NT, W>;
    constexpr bool F32 = Sh::F32, HELD = NT == 1 && !F32;  // q stays in registers
    constexpr int STAGES = Sh::STAGES;
    extern __shared__ uint8_t ar_smem_raw[];
    __shared__ __align__(8) uint64_t full[W][STAGES];
    __shared__ float row_factor[Sh::ROWS];  // scale log2(e) / what the row was multiplied by
    __shared__ float warp_m[W][Sh::ROWS], warp_l[W][Sh::ROWS];
    __shared__ float part_m[Sh::ROWS], part_l[Sh::ROWS];
    __shared__ uint32_t nan_dropped[W];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int head = blockIdx.x % a.c.n_kv, part = blockIdx.z, group = a.n_heads / a.c.n_kv, dim = a.c.dim;
    pdl_wait();
    pdl_trigger();
    const AfTile tile = af_tile(a, blockIdx.y, blockIdx.x / a.c.n_kv, Sh::ROWS);
    if (tile.n <= 0) return;  // (the whole cluster)
    // ── this warp's keys ──
    const int pos_base = tile.len - tile.rows;
    const int pos_first = pos_base + tile.row0 / group, pos_last = pos_base + (tile.row0 + tile.n - 1) / group;  // of the tile's rows
    const int held = (int)min((int64_t)tile.len, (int64_t)a.c.max_pages * KV_PAGE);
    const int k_end = min(pos_last + 1, held), k_begin = a.window > 0 ? max(0, max(pos_first, 0) - a.window + 1) : 0;
    const int s_begin = k_begin / AR_KEYS, s_end = k_end > k_begin ? (k_end - 1) / AR_KEYS + 1 : s_begin;  // (k_end may be near 2^31)
    const int per = (s_end - s_begin + parts - 1) / parts;
    const int b_begin = min(s_end, s_begin + part * per), b_end = min(s_end, b_begin + per);
    const int steps = max(0, (b_end - b_begin - warp + W - 1) / W);  // of this warp: b_begin + warp + i W
    const int32_t* const table = a.c.page_table + (int64_t)max(0, min(tile.slot, a.c.n_slots - 1)) * a.c.max_pages;
    uint8_t* const ar_smem = ar_smem_raw + ((1024u - (smem_addr(ar_smem_raw) & 1023u)) & 1023u);
    uint8_t *const ring = ar_smem + warp * STAGES * Sh::STAGE, *const scale_ring = ar_smem + W * STAGES * Sh::STAGE + warp * STAGES * Sh::SCALES;
    uint8_t* const qs = ar_smem + (Sh::SMEM - 1024 - Sh::Q);
    if (lane == 0) {
        if (F32) nan_dropped[warp] = 0;
#pragma unroll
        for (int i = 0; i < STAGES; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(tc5_smem_u32(&full[warp][i])) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncwarp();
    // pages of the warp's steps: a group of 16 steps in the lanes, the next one on its way
    constexpr int GROUP = 32 / AR_PAGES;
    auto look_up = [&](int i0) {
        const int i = i0 + lane / AR_PAGES, index = (b_begin + warp + i * W) * AR_PAGES + lane % AR_PAGES;
        const int page = i < steps && index < a.c.max_pages && index * KV_PAGE < k_end ? table[index] : -1;
        return page < a.c.n_pages ? page : -1;
    };
    int pages = look_up(0), pages_next = -1;
    uint32_t present = 0;  // a bit for each page of the ring's steps: it is one
    // lanes 0 to 3 copy a page's keys or values each, lanes 4 to 7 their scales
    const int pg_of = lane / 2 % AR_PAGES, row_of = (lane % 2 * a.c.n_kv + head) * KV_PAGE, page_rows = 2 * a.c.n_kv * KV_PAGE;
    auto copy_step = [&](int i, int stage) {
        const int page = __shfl_sync(0xFFFFFFFFu, pages, i % GROUP * AR_PAGES + pg_of);
        const uint32_t here = __ballot_sync(0xFFFFFFFFu, page >= 0), bits = (here & 1) | (here >> 1 & 2);  // of lanes 0 and 2: the step's pages
        present = (present & ~(3u << (2 * stage))) | bits << (2 * stage);
        const uint32_t bar = tc5_smem_u32(&full[warp][stage]);
        if (lane == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"((uint32_t)__popc(bits) * (2u * Sh::PAGE + 2u * KV_PAGE * 4u)) : "memory");
        __syncwarp();
        if (page >= 0) {
            const int row = page * page_rows + row_of;
            if (lane < 4) tc5_tma_2d(tc5_smem_u32(ring + stage * Sh::STAGE) + lane * Sh::PAGE, &map, 0, row, bar);
            else if (lane < 8)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                                 tc5_smem_u32(scale_ring + stage * Sh::SCALES) + (uint32_t)((lane % 2 * AR_KEYS + pg_of * KV_PAGE) * 4)),
                             "l"(a.c.scales + row), "r"(KV_PAGE * 4), "r"(bar)
                             : "memory");
        }
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        if (i < steps) copy_step(i, i);
    // ── queries: operands in the order in which they are used ──
    for (int r = warp; r < Sh::ROWS; r += W) {
        const int row = tile.row0 + min(r, tile.n - 1);
        const T* const src = static_cast<const T*>(a.q) + (int64_t)(tile.first + row / group) * a.ldq + (int64_t)(head * group + row % group) * dim;
        float x[DP / 32];
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
            const int e = 32 * i + lane;
            x[i] = r < tile.n && e < dim ? to_f32(src[e]) : 0.f;
            most = fmaxf(most, fabsf(x[i]));
        }
        most = warp_max(most);
        float by, back;
        af_row_scale(most, 12, by, back);
        if (lane == 0) row_factor[r] = back * a.scale * AF_LOG2E;
        // element e: 16 of them (c = e / 16) are thread t's, its chunk h; four make a product's part, the first two in the first register
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
            const int e = 32 * i + lane, c = e / 16, step = 4 * (c % Sh::CHUNKS) + e % 16 / 4, of = 4 * (r % 8) + c / Sh::CHUNKS;
            const float v = x[i] * by;
            const __half hi = __float2half_rn(v);
            uint8_t* const to = qs + (size_t)(r / 8 * Sh::PLANES * Sh::STEPS + step) * 256 + of * 8 + e % 4 * 2;
            *reinterpret_cast<__half*>(to) = hi;
            if constexpr (F32) *reinterpret_cast<__half*>(to + Sh::STEPS * 256) = __float2half_rn(v - __half2float(hi));
        }
    }
    __syncthreads();
    auto query = [&](int n, int p, int step) { return *reinterpret_cast<const uint2*>(qs + ((n * Sh::PLANES + p) * Sh::STEPS + step) * 256 + lane * 8); };
    uint2 q_held[HELD ? Sh::PLANES : 1][HELD ? Sh::STEPS : 1];
    if constexpr (HELD) {
#pragma unroll
        for (int p = 0; p < Sh::PLANES; ++p)
#pragma unroll
            for (int i = 0; i < Sh::STEPS; ++i) q_held[p][i] = query(0, p, i);
    }
    // ── scores, weights, sums: of rows 8 n + 2 t and + 1 ──
    float o[NT][DP / 16][4], m[NT][2], l[NT][2], factor[NT][2];
    float o_sum[F32 ? NT : 1][F32 ? DP / 16 : 1][4] = {};  // f32: what o has been added to
    float ref = 0x1p-100f;         // R of the header: o is the sum times AF_LIFT / ref
    int limit[NT][2], low[NT][2];  // a row sees keys low .. limit
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < DP / 16; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = 8 * n + 2 * t + e, pos = pos_base + (tile.row0 + row) / group;
            m[n][e] = -INFINITY;
            l[n][e] = 0.f;
            limit[n][e] = row < tile.n ? min(pos, held - 1) : -1;
            low[n][e] = a.window > 0 ? max(pos, 0) - a.window + 1 : 0;
            factor[n][e] = row_factor[row];
        }
    }
    const int whole_from = a.window > 0 ? max(pos_last, 0) - a.window + 1 : 0, whole_to = min(pos_first, held - 1);  // keys that all rows see
    [[maybe_unused]] uint32_t dropped = 0;  // values' bytes that are NaN, where MASK (f32: nan_dropped, one register less: 8 x 8 rows at 4096 57.3 us, 56.1 so)
    // MASK: some row does not see some key. Only then can a byte that is NaN belong to a key that a row does not see; else the product makes its
    // coordinate NaN.
    auto work = [&](auto with_mask, const uint8_t* at, const float* scales, int key0, uint32_t gone) {
        constexpr bool MASK = decltype(with_mask)::value;
        float s[NT][2][4];  // keys 16 pg + g and + 8
        // The tensor cores cut off what falls below an accumulator's last bits, always towards zero. f32 rows therefore have three short sums, of the
        // remainders and of each 64 columns, instead of one (518 keys: 1.3e-6 off in all, 3.8e-7 so), and o is added up apart every AR_FLUSH steps.
        constexpr int SUMS = F32 ? 1 + Sh::CHUNKS : 1;
        float sums[SUMS][NT][2][4];
#pragma unroll
        for (int c = 0; c < SUMS; ++c)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int pg = 0; pg < 2; ++pg) sums[c][n][pg][0] = sums[c][n][pg][1] = sums[c][n][pg][2] = sums[c][n][pg][3] = 0.f;
#pragma unroll
        for (int h = 0; h < Sh::CHUNKS; ++h)
#pragma unroll
            for (int pg = 0; pg < 2; ++pg) {
                const uint8_t* const from = at + 2 * pg * Sh::PAGE + g * 128 + ((Sh::CHUNKS * t + h) ^ g) * 16;
                const uint4 k0 = *reinterpret_cast<const uint4*>(from), k1 = *reinterpret_cast<const uint4*>(from + 8 * 128);
                const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint4 k;
                    af_halves(w0[w], k.x, k.z);
                    af_halves(w1[w], k.y, k.w);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int p = Sh::PLANES - 1; p >= 0; --p) {
                            uint2 q;
                            if constexpr (HELD) q = q_held[p][4 * h + w];
                            else q = query(n, p, 4 * h + w);
                            af_mma(sums[!F32 || p == 1 ? 0 : 1 + h][n][pg], k, q.x, q.y);
                        }
                }
            }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int pg = 0; pg < 2; ++pg)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if constexpr (!F32) s[n][pg][c] = sums[0][n][pg][c];
                    else if constexpr (Sh::CHUNKS == 1) s[n][pg][c] = sums[1][n][pg][c] + sums[0][n][pg][c];
                    else s[n][pg][c] = sums[1][n][pg][c] + sums[2][n][pg][c] + sums[0][n][pg][c];
                }
        float ks[4], vs[4];  // of keys g + 8 j
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ks[j] = af_number(scales[8 * j]);
            vs[j] = af_number(scales[AR_KEYS + 8 * j]);
        }
        float big = 0.f;  // the largest finite scale of values that a row of the tile may see
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = key0 + 8 * j + g;
            if (vs[j] < INFINITY && (!MASK || (k >= k_begin && k < k_end && !(gone >> (j / 2) & 1)))) big = fmaxf(big, vs[j]);
        }
        bool move = big > ref;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float best = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float& z = s[n][j / 2][2 * (j % 2) + e];
                    z = z * ks[j] * factor[n][e];
                    if (MASK) {
                        const int k = key0 + 8 * j + g;
                        if (k > limit[n][e] || k < low[n][e] || (gone >> (j / 2) & 1)) z = -INFINITY;
                    }
                    best = fmaxf(best, z);
                }
                move |= best > m[n][e] + AF_LAZY;  // (of -inf: as soon as there is a score)
            }
        if (__any_sync(0xFFFFFFFFu, move)) {  // the rows' largest scores and the largest scale, over the threads that share them
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, x));
            const float up = fmaxf(ref, af_power(big)), shrink = ref / up;  // (powers of two)
            ref = up;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float best = fmaxf(fmaxf(s[n][0][e], s[n][0][2 + e]), fmaxf(s[n][1][e], s[n][1][2 + e]));
#pragma unroll
                    for (int x = 4; x <= 16; x <<= 1) best = fmaxf(best, __shfl_xor_sync(0xFFFFFFFFu, best, x));
                    const float to = fmaxf(m[n][e], best), by = m[n][e] == to ? 1.f : ex2_approx(m[n][e] - to);
                    m[n][e] = to;
                    l[n][e] *= by;
#pragma unroll
                    for (int j = 0; j < DP / 16; ++j) {
                        o[n][j][e] *= by * shrink;
                        o[n][j][2 + e] *= by * shrink;
                        if constexpr (F32) {
                            o_sum[n][j][e] *= by * shrink;
                            o_sum[n][j][2 + e] *= by * shrink;
                        }
                    }
                }
        }
        const float lift = AF_LIFT / ref;
#pragma unroll
        for (int j = 0; j < 4; ++j) vs[j] *= lift;
        uint2 pb[NT][F32 ? 2 : 1][2];  // weights as the second product's operand, of 16 keys each
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float from0 = m[n][0] == -INFINITY ? 0.f : m[n][0], from1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
            uint32_t hi[4];
            [[maybe_unused]] uint32_t lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float z0 = s[n][j / 2][2 * (j % 2)], z1 = s[n][j / 2][2 * (j % 2) + 1];
                float w0 = ex2_approx(z0 - from0), w1 = ex2_approx(z1 - from1);
                l[n][0] += w0;
                l[n][1] += w1;
                w0 = MASK && z0 == -INFINITY ? 0.f : w0 * vs[j];  // (what is masked may have any scale)
                w1 = MASK && z1 == -INFINITY ? 0.f : w1 * vs[j];
                if constexpr (F32) af_split(w0, w1, hi[j], lo[j]);
                else hi[j] = af_pack(w0, w1);
            }
#pragma unroll
            for (int pg = 0; pg < 2; ++pg) {
                pb[n][0][pg] = make_uint2(af_transpose(hi[2 * pg]), af_transpose(hi[2 * pg + 1]));
                if constexpr (F32) pb[n][1][pg] = make_uint2(af_transpose(lo[2 * pg]), af_transpose(lo[2 * pg + 1]));
            }
        }
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
            constexpr int WORDS = DP / 32;  // of a thread's part of a token's values
            uint32_t vw[4][WORDS];
            [[maybe_unused]] uint32_t near = 0, far = 0;  // tokens 2 t, 2 t + 1 and tokens 2 t + 8, 2 t + 9 with such bytes
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = 2 * t + (j & 1) + 8 * (j >> 1);
                const uint8_t* const from = at + (2 * pg + 1) * Sh::PAGE + key * 128 + ((DP / 8 * g / 16) ^ (key & 7)) * 16 + DP / 8 * g % 16;
                if constexpr (DP == 128) {
                    const uint4 v = *reinterpret_cast<const uint4*>(from);
                    vw[j][0] = v.x; vw[j][1] = v.y; vw[j][2] = v.z; vw[j][3] = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(from);
                    vw[j][0] = v.x; vw[j][1] = v.y;
                }
            }
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                uint4 v[2];  // of two coordinates each: tokens 2 t, 2 t + 1 of the one and the other, tokens 2 t + 8, 2 t + 9
                af_halves(__byte_perm(vw[0][w], vw[1][w], 0x5140), v[0].x, v[0].y);
                af_halves(__byte_perm(vw[2][w], vw[3][w], 0x5140), v[0].z, v[0].w);
                af_halves(__byte_perm(vw[0][w], vw[1][w], 0x7362), v[1].x, v[1].y);
                af_halves(__byte_perm(vw[2][w], vw[3][w], 0x7362), v[1].z, v[1].w);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if (MASK) v[q] = make_uint4(af_finite(v[q].x, near), af_finite(v[q].y, near), af_finite(v[q].z, far), af_finite(v[q].w, far));
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int p = F32 ? 1 : 0; p >= 0; --p) af_mma(o[n][2 * w + q], v[q], pb[n][p][pg].x, pb[n][p][pg].y);
                }
            }
            if (MASK && !(gone >> pg & 1)) {  // (bytes that nobody sees may be anything)
                auto counts = [&](int token) { return key0 + token >= k_begin && key0 + token < k_end; };
                const int k = KV_PAGE * pg + 2 * t;
                const uint32_t here = (near & ((counts(k) ? 0xFFFFu : 0u) | (counts(k + 1) ? 0xFFFF0000u : 0u))) |
                                      (far & ((counts(k + 8) ? 0xFFFFu : 0u) | (counts(k + 9) ? 0xFFFF0000u : 0u)));
                if constexpr (!F32) dropped |= here;
                else if (here != 0) nan_dropped[warp] = 1;
            }
        }
    };
    bool ok = true;
    uint32_t parity = 0;
    int i = 0;
    for (int stage = 0; i < steps; ++i) {
        const int ahead = i + STAGES - 1;
        if (ahead % GROUP == 0) pages = pages_next;
        if (ahead % GROUP == GROUP / 2) pages_next = look_up(ahead / GROUP * GROUP + GROUP);
        __syncwarp();  // the stage that the next copies go to has been read
        if (ahead < steps) copy_step(ahead, stage == 0 ? STAGES - 1 : stage - 1);
        ok = __all_sync(0xFFFFFFFFu, tc5_wait(&full[warp][stage], parity));
        if (!ok) break;
        const uint32_t gone = ~present >> (stage * AR_PAGES) & ((1u << AR_PAGES) - 1);
        const uint8_t* const at = ring + stage * Sh::STAGE;
        const float* const scales = reinterpret_cast<const float*>(scale_ring + stage * Sh::SCALES) + g;
        const int key0 = (b_begin + warp + i * W) * AR_KEYS;
        if (gone != 0 || key0 < whole_from || key0 + AR_KEYS - 1 > whole_to) work(std::true_type{}, at, scales, key0, gone);
        else work(std::false_type{}, at, scales, key0, 0u);
        if constexpr (F32) {
            if (i % AR_FLUSH == AR_FLUSH - 1) {
#pragma unroll
                for (int j = 0; j < NT * DP / 16 * 4; ++j) {
                    (&o_sum[0][0][0])[j] += (&o[0][0][0])[j];
                    (&o[0][0][0])[j] = 0.f;
                }
            }
        }
        if (++stage == STAGES) {
            stage = 0;
            parity ^= 1;
        }
    }
    if (!ok && lane == 0) {  // copies on their way to this block are waited for, for as long again each
        report_wait(a.waits, WAIT_ATTENTION);
        for (int k = i; k < ring_requested(i, STAGES, steps); ++k) tc5_wait(&full[warp][ring_at(k, STAGES).stage], ring_at(k, STAGES).parity);
    }
    __syncwarp();
    if (F32 ? nan_dropped[warp] != 0 : __any_sync(0xFFFFFFFFu, dropped != 0)) {
#pragma unroll 1
        for (int i = 0; i < steps; ++i) {
            const int key0 = (b_begin + warp + i * W) * AR_KEYS;
            uint32_t tokens[1];
            af_nan_tokens(a.c, table, head, key0, k_end, tokens);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (af_sees(tokens[0], key0, low[n][e], limit[n][e])) l[n][e] = __uint_as_float(0x7FC00000u);
        }
    }
    // ── the warps' sums into one, then the blocks' ──
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) l[n][e] += __shfl_xor_sync(0xFFFFFFFFu, l[n][e], x);
            if (g == 0) {
                warp_m[warp][8 * n + 2 * t + e] = m[n][e];
                warp_l[warp][8 * n + 2 * t + e] = l[n][e];
            }
        }
    __syncthreads();  // the rings have been read
    float* const sums = reinterpret_cast<float*>(ar_smem);  // [warp][row][LDO]
    const float back = ref * (1.f / AF_LIFT);
    if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < NT * DP / 16 * 4; ++j) (&o[0][0][0])[j] += (&o_sum[0][0][0])[j];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)  // coordinates DP / 8 g + 2 j and + 1
                *reinterpret_cast<float2*>(&sums[(warp * Sh::ROWS + 8 * n + 2 * t + e) * Sh::LDO + DP / 8 * g + 2 * j]) = make_float2(o[n][j][e] * back, o[n][j][2 + e] * back);
    __syncthreads();
    auto store = [&](int row, int col, float y) {
        const int at = tile.row0 + row;
        static_cast<T*>(a.out)[(int64_t)(tile.first + at / group) * a.ldo + (int64_t)(head * group + at % group) * dim + col] = from_f32<T>(y);
    };
    for (int row = warp; row < tile.n; row += W) {
        float top = -INFINITY, total = 0.f, w[W], y[DP / 32];
#pragma unroll
        for (int i = 0; i < W; ++i) top = fmaxf(top, warp_m[i][row]);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            w[i] = warp_m[i][row] == -INFINITY ? 0.f : ex2_approx(warp_m[i][row] - top);
            total += warp_l[i][row] * w[i];
        }
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            y[c] = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) y[c] = fmaf(sums[(i * Sh::ROWS + row) * Sh::LDO + 32 * c + lane], w[i], y[c]);
        }
        if (parts == 1) {
            const float by = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
            for (int c = 0; c < DP / 32; ++c)
                if (32 * c + lane < dim) store(row, 32 * c + lane, y[c] * by);
        } else {
            if (lane == 0) {
                part_m[row] = top;
                part_l[row] = total;
            }
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) sums[row * Sh::LDO + 32 * c + lane] = y[c];
        }
    }
    if (parts == 1) return;
    cluster_sync();
    for (int row = part + parts * warp; row < tile.n; row += parts * W) {  // the cluster's warps share the rows out
        // lane i looks at part i
        const float pm = lane < parts ? ld_peer(peer_smem(smem_addr(&part_m[row]), lane)) : -INFINITY;
        const float pl = lane < parts ? ld_peer(peer_smem(smem_addr(&part_l[row]), lane)) : 0.f;
        const float top = warp_max(pm), w = pm == -INFINITY ? 0.f : ex2_approx(pm - top), total = warp_sum(pl * w);
        float y[DP / 32] = {};
        for (int i = 0; i < parts; ++i) {
            const float wi = __shfl_sync(0xFFFFFFFFu, w, i);
            const uint32_t from = peer_smem(smem_addr(sums + row * Sh::LDO + lane), i);
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) y[c] = fmaf(ld_peer(from + 128u * c), wi, y[c]);
        }
        const float by = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c)
            if (32 * c + lane < dim) store(row, 32 * c + lane, y[c] * by);
    }
    cluster_sync();  // nobody leaves while its parts are being read
}

// The pool's rows, 16 of them (a page's keys or values of a head) a copy, filled up to 128 bytes with zeros, 128-byte swizzle.
cudaError_t af_page_map(const CacheFp8& c, CUtensorMap* map) {
    const PFN_encodeTiled encode = tensor_map_encoder();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)c.dim, (cuuint64_t)c.n_pages * 2 * c.n_kv * KV_PAGE}, strides[1] = {(cuuint64_t)c.dim};
    const cuuint32_t box[2] = {128, KV_PAGE}, each[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, c.values, dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

cudaError_t af_fits(const void* kernel, int threads, int smem, ClusterFits* out) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);  // (more than eight blocks)
    for (int p = 1; p <= AF_MAX_PARTS && e == cudaSuccess; ++p) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(1, 1, (unsigned)(64 * p));
        cfg.blockDim = dim3((unsigned)threads);
        cfg.dynamicSmemBytes = (size_t)smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = at[0].val.clusterDim.y = 1;
        at[0].val.clusterDim.z = (unsigned)p;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int found = 0;
        e = cudaOccupancyMaxActiveClusters(&found, kernel, &cfg);
        out->at_once[p].store(found, std::memory_order_relaxed);
    }
    return e;
}

AfShare af_share(const ClusterFits& fits, int64_t clusters, int64_t pieces, double piece, double fixed, double joined) {
    AfShare best{1, 1e30};
    for (int p = 1; p <= AF_MAX_PARTS; ++p) {
        const int at_once = fits.at_once[p].load(std::memory_order_relaxed);
        if (at_once < 1) continue;
        const double rounds = (double)clusters / at_once, waves = rounds <= 1. ? 1. : (rounds + std::ceil(rounds)) / 2;
        const double time = waves * ((double)((pieces + p - 1) / p) * piece + fixed + (p > 1 ? joined : 0.));
        if (time < best.time) best = AfShare{p, time};
    }
    return best;
}

// Microseconds of a warp's step with twelve warps on an SM, of a block's start and end, and of adding parts up. Few bf16 rows: measured, 131072 keys of
// the 8B shape in one to 16 parts, 518 keys; the others are fitted to 64 calls (3 to 35 rows a head, 240 to 32768 keys, 1 to 32 sequences, 8B, 1.5B and
// 0.5B shapes), from which they are 3 to 8 % off. Other calls are not checked against them; head sizes between 64 and 128 take 128's.
template <typename T, int DP, int NT>
struct ArTimes {
    static constexpr bool F32 = sizeof(T) == 4, FEW = NT == 1 && !F32;
    static constexpr double STEP = FEW ? 1.4 : F32 ? (DP == 128 ? 2.2 : 1.8) : DP == 128 ? 2.4 : 2.1;
    static constexpr double FIXED = FEW ? 4. : F32 ? (DP == 128 ? 5. : 4.) : DP == 128 ? 6.5 : 5., JOINED = FEW ? 0.5 : F32 && DP == 128 ? 1.5 : 2.;
};

template <typename T, int DP, int NT, int W>
struct RowsLaunch {
    using Sh = ArShape<T, DP, NT, W>;
    using At = ArTimes<T, DP, NT>;
    static constexpr auto kernel = attention_rows_kernel<T, DP, NT, W>;
    static cudaError_t share(int64_t clusters, int64_t len, AfShare* out) {
        static PerDeviceOnce once;
        static ClusterFits fits[SP_MAX_DEVICES];
        ClusterFits& mine = fits[current_device_index()];
        const cudaError_t e = once.run([&] { return af_fits(reinterpret_cast<const void*>(kernel), 32 * W, Sh::SMEM, &mine); });
        if (e == cudaSuccess) *out = af_share(mine, clusters, (len + AR_KEYS * W - 1) / (AR_KEYS * W), At::STEP, At::FIXED, At::JOINED);
        return e;
    }
    static cudaError_t go(const AttentionFp8Args& a, const CUtensorMap& map, int tiles, int parts, cudaStream_t st) {
        return launch_pdl_cluster(kernel, dim3((unsigned)(a.c.n_kv * tiles), (unsigned)a.n_seqs, (unsigned)parts), dim3(32 * W), Sh::SMEM, st, parts, a, parts, map);
    }
};

// Blocks of 12 warps fill an SM, and the longest sequences are fastest with them (64 x 1024 keys of the 1.5B shape 10.8 us, 10.9 if four were taken); of
// four, three share one, which many short sequences want (1000 x 90 keys 36.3 us, with 12 warps 72.2; 300 x 200 17.8, 26.9). More rows than one
// block has are shared out to several, which read the same keys, or go to the tiles, whichever takes less by the times above (f32, 24 rows at 4096
// keys of the 8B shape 12 us, tiles 20.5; 8 x 32 rows 56, 65; 32 x 56 rows at 1024 of the 0.5B shape 28, 18; bf16, 4 x 30 at 32768 of
// the 1.5B shape 42, 56; 8 x 64 at 4096 of the 8B shape 65, 38; 16 rows, one block's: 8 x 4096 keys 24, 36).
template <typename T, int DP, int NT>
static cudaError_t launch_rows(const AttentionFp8Args& a, cudaStream_t st) {
    const int tiles = (int)(((int64_t)a.max_rows * (a.n_heads / a.c.n_kv) + 8 * NT - 1) / (8 * NT));
    const int64_t clusters = (int64_t)a.c.n_kv * tiles * a.n_seqs, len = af_keys(a);
    AfShare wide, narrow;
    CUtensorMap map{};
    cudaError_t e = RowsLaunch<T, DP, NT, 12>::share(clusters, len, &wide);
    if (e == cudaSuccess) e = RowsLaunch<T, DP, NT, 4>::share(clusters, len, &narrow);
    if (e == cudaSuccess && tiles > 1) {
        AfShare other;
        e = launch_attention_fp8_tiles(a, sizeof(T) == 2, st, &other);
        if (e == cudaSuccess && other.time < std::min(wide.time, narrow.time)) return launch_attention_fp8_tiles(a, sizeof(T) == 2, st, nullptr);
    }
    if (e == cudaSuccess) e = af_page_map(a.c, &map);
    if (e == cudaSuccess)
        e = wide.time <= narrow.time ? RowsLaunch<T, DP, NT, 12>::go(a, map, tiles, wide.parts, st) : RowsLaunch<T, DP, NT, 4>::go(a, map, tiles, narrow.parts, st);
    return e != cudaSuccess ? e : count_launch_and_check();
}

template <typename T, int DP>
static cudaError_t attention_as(const AttentionFp8Args& a, cudaStream_t st) {
    if constexpr (sizeof(T) == 2)  // (f32: two sets of sums of 16 rows do not fit the registers)
        if ((int64_t)a.max_rows * (a.n_heads / a.c.n_kv) > 8) return launch_rows<T, DP, 2>(a, st);
    return launch_rows<T, DP, 1>(a, st);
}
cudaError_t launch_attention_fp8(const AttentionFp8Args& a, bool bf, cudaStream_t st) {
    if (a.c.dim <= 64) return bf ? attention_as<bf16, 64>(a, st) : attention_as<float, 64>(a, st);
    return bf ? attention_as<bf16, 128>(a, st) : attention_as<float, 128>(a, st);
}

}  // namespace sp
