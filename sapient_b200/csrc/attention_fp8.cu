// Attention of the newest tokens of sequences over a paged cache of 8-bit rows (cache_fp8.h).
//
//   z_k = scale (q . K_k) s_k,   o = sum_k e^(z_k - m) s'_k V_k / sum_k e^(z_k - m)
//
// with e4m3 rows K_k, V_k and their scales s_k, s'_k; a row sees keys k <= its position, of which the newest `window`; one that sees none
// gives zeros. The queries of a key head are rows of one product (row = token x heads per key head + head), so that its keys are read
// once for all of them.
//
// Precision. e4m3 values are exact in fp16, the scales are applied in f32. A row of q is multiplied by a power of two so that its
// largest value lies in [2^12, 2^13): bf16 values are then exact in fp16 (down to 2^-30 of the largest), f32 values are taken as fp16
// plus the fp16 of the remainder. The weights e^(z - m) s' enter the second product as fp16 (11 bits, where the result has bf16's 8) or,
// for f32, as fp16 plus remainder, multiplied by a power of two that keeps them out of fp16's subnormals: with the largest scale so far, R,
// rounded up to a power of two and e^(z - m) <= 2^LAZY, the weights are e^(z - m) s' 2^(15 - LAZY) / R <= 2^15. Sums, maxima and the output are f32.
#include <algorithm>

#include "attention_fp8.cuh"
#include "kernels.h"
#include "pdl.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

// ── Few rows: mma.sync, a warp takes 32 keys at a time ──
// The cache is read once, which is what bounds it: every warp keeps a ring of asynchronous copies in flight. A thread copies just the
// bytes that it multiplies itself: keys as the second operand of q K^T, four consecutive bytes of a row being one thread's part of a
// product of 16 columns (the order of columns does not matter where q has the same), values of four tokens as the second operand
// of P V, 16 neighbouring columns each, so that a column of the product is a coordinate of each sixteen. So nothing is rearranged but pairs of
// tokens' bytes, and the accumulators of the first product are the first operand of the second.
// Keys are shared out to the warps of a block and the blocks of a cluster, which add up their parts through shared memory: no workspace.
constexpr int AR_WARPS = 4, AR_THREADS = 32 * AR_WARPS, AR_KEYS = 32, AR_PAGES = AR_KEYS / KV_PAGE, AR_STAGES = 3, AR_MAX_PARTS = 16;

template <typename T, int DP, int R>
struct ArShape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PLANES = F32 ? 2 : 1, STEPS = DP / 16, CHUNKS = DP / 64;
    static constexpr int KBYTES = AR_KEYS * DP, STAGE = 2 * KBYTES + 2 * AR_KEYS * 4;  // keys, values, their scales
    static constexpr int Q = R * PLANES * STEPS * 512, RING = AR_WARPS * AR_STAGES * STAGE;
    static constexpr int ROWS = 16 * R, LDO = DP + 4;
    static constexpr int SUMS = AR_WARPS * ROWS * LDO * 4;  // takes the ring's place
    static constexpr int SMEM = Q + (RING > SUMS ? RING : SUMS);
};

template <typename T, int DP, int R>
__global__ void __launch_bounds__(AR_THREADS) attention_rows_kernel(const AttentionFp8Args a, int parts) {
    using Sh = ArShape<T, DP, R>;
    constexpr bool F32 = Sh::F32;
    extern __shared__ __align__(16) uint8_t ar_smem[];
    __shared__ float row_factor[Sh::ROWS];              // scale log2(e) / what the row was multiplied by
    __shared__ float warp_m[AR_WARPS][Sh::ROWS], warp_l[AR_WARPS][Sh::ROWS];
    __shared__ float part_m[Sh::ROWS], part_l[Sh::ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int head = blockIdx.x % a.c.n_kv, part = blockIdx.z, group = a.n_heads / a.c.n_kv, dim = a.c.dim;
    pdl_wait();
    pdl_trigger();
    const AfTile tile = af_tile(a, blockIdx.y, blockIdx.x / a.c.n_kv, Sh::ROWS);
    if (tile.n <= 0) return;  // (the whole cluster)
    // ── queries: fp16 operands in the order in which they are used ──
    uint8_t* const qs = ar_smem;
    {
        for (int r = warp; r < Sh::ROWS; r += AR_WARPS) {
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
            // element e: chunk c = e / 16 is thread t = c % 4's, h = c / 4; step 4 h + (e % 16) / 4; of its four bytes the first two in
            // the registers of columns 2 t, the others in those of columns 2 t + 8
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const int e = 32 * i + lane, c = e / 16, step = 4 * (c / 4) + e % 16 / 4, of = 4 * (r % 8) + c % 4, reg = (e & 2) + (r % 16 >= 8);
                const float v = x[i] * by;
                const __half hi = __float2half_rn(v);
                uint8_t* const to = qs + (size_t)(r / 16 * Sh::PLANES * Sh::STEPS + step) * 512 + of * 16 + reg * 4 + (e & 1) * 2;
                *reinterpret_cast<__half*>(to) = hi;
                if constexpr (F32) *reinterpret_cast<__half*>(to + Sh::STEPS * 512) = __float2half_rn(v - __half2float(hi));
            }
        }
    }
    __syncthreads();
    // ── this warp's keys ──
    const int last_row = tile.row0 + tile.n - 1;
    const int pos_first = tile.len - tile.rows + tile.row0 / group, pos_last = tile.len - tile.rows + last_row / group;  // of the tile's rows
    const int held = (int)min((int64_t)tile.len, (int64_t)a.c.max_pages * KV_PAGE);
    const int k_end = min(pos_last + 1, held), k_begin = a.window > 0 ? max(0, pos_first - a.window + 1) : 0;
    const int s_begin = k_begin / AR_KEYS, s_end = k_end > k_begin ? (k_end + AR_KEYS - 1) / AR_KEYS : s_begin;
    const int per = (s_end - s_begin + parts - 1) / parts;
    const int b_begin = min(s_end, s_begin + part * per), b_end = min(s_end, b_begin + per);
    const int steps = max(0, (b_end - b_begin - warp + AR_WARPS - 1) / AR_WARPS);  // of this warp: b_begin + warp + i AR_WARPS
    const int32_t* const table = a.c.page_table + (int64_t)max(0, min(tile.slot, a.c.n_slots - 1)) * a.c.max_pages;
    uint8_t* const ring = ar_smem + Sh::Q + warp * AR_STAGES * Sh::STAGE;
    const uint32_t ring_at = smem_addr(ring);
    // pages of the warp's steps: a group of 16 steps in the lanes, the next one on its way
    constexpr int GROUP = 32 / AR_PAGES;
    auto look_up = [&](int i0) {
        const int i = i0 + lane / AR_PAGES, index = (b_begin + warp + i * AR_WARPS) * AR_PAGES + lane % AR_PAGES;
        const int page = i < steps && index < a.c.max_pages && index * KV_PAGE < k_end ? table[index] : -1;
        return page < a.c.n_pages ? page : -1;
    };
    int pages = look_up(0), pages_next = -1;
    uint32_t present = 0;  // a bit for each page of the ring's steps: it is one
    auto copy_step = [&](int i) {
        const int stage = i % AR_STAGES;
        const uint32_t at = ring_at + (uint32_t)(stage * Sh::STAGE);
#pragma unroll
        for (int pg = 0; pg < AR_PAGES; ++pg) {
            const int page = __shfl_sync(0xFFFFFFFFu, pages, i % GROUP * AR_PAGES + pg);
            const bool there = page >= 0;
            const uint32_t bit = 1u << (stage * AR_PAGES + pg);
            present = there ? present | bit : present & ~bit;
            const int64_t krow = a.c.row(max(page, 0), 0, head), vrow = krow + (int64_t)a.c.n_kv * KV_PAGE;
            const uint8_t *const k = a.c.values + krow * dim, *const v = a.c.values + vrow * dim;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < Sh::CHUNKS; ++h) {
                    const int c = 16 * (t + 4 * h);
                    const bool in = there && c < dim;
                    af_copy16(at + (uint32_t)((((pg * 2 + j) * Sh::CHUNKS + h) * 32 + lane) * 16), in ? k + (8 * j + g) * dim + c : k, in);
                }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = 2 * t + (j & 1) + 8 * (j >> 1), c = DP / 8 * g;
                const bool in = there && c < dim;
                const uint8_t* const src = in ? v + key * dim + c : v;
                if constexpr (DP == 128) af_copy16(at + (uint32_t)(Sh::KBYTES + ((pg * 4 + j) * 32 + lane) * 16), src, in);
                else af_copy8(at + (uint32_t)(Sh::KBYTES + ((pg * 4 + j) * 32 + lane) * 8), src, in);
            }
            if (lane / 8 == pg) {  // scales: 64 bytes of the keys, then of the values
                const int q = lane % 8;
                af_copy16(at + (uint32_t)(2 * Sh::KBYTES + (q / 4 * AR_KEYS + pg * KV_PAGE + q % 4 * 4) * 4), a.c.scales + (q < 4 ? krow : vrow) + q % 4 * 4, there);
            }
        }
    };
    // ── scores, weights, sums ──
    float o[R][DP / 8][4], m[R][2], l[R][2], factor[R][2];
    float ref = 0x1p-100f;     // R of the header: o is the sum times AF_LIFT / ref
    int limit[R][2], low[R][2];  // a row sees keys low .. limit
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) o[r][j][0] = o[r][j][1] = o[r][j][2] = o[r][j][3] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = 16 * r + g + 8 * e, pos = tile.len - tile.rows + (tile.row0 + row) / group;
            m[r][e] = -INFINITY;
            l[r][e] = 0.f;
            limit[r][e] = row < tile.n ? min(pos, held - 1) : -1;
            low[r][e] = a.window > 0 ? pos - a.window + 1 : 0;
            factor[r][e] = row_factor[row];
        }
    }
    const int whole_from = a.window > 0 ? pos_last - a.window + 1 : 0, whole_to = min(pos_first, held - 1);  // keys that all rows see
#pragma unroll
    for (int i = 0; i < AR_STAGES - 1; ++i) {
        if (i < steps) copy_step(i);
        cp_async_commit();
    }
    for (int i = 0; i < steps; ++i) {
        const int ahead = i + AR_STAGES - 1, stage = i % AR_STAGES;
        if (ahead % GROUP == 0) pages = pages_next;
        if (ahead % GROUP == GROUP / 2) pages_next = look_up(ahead / GROUP * GROUP + GROUP);
        cp_async_wait<AR_STAGES - 2>();
        __syncwarp();  // every lane's copies of this step have come, and the stage that the next copies go to has been read
        const uint32_t gone = ~present >> (stage * AR_PAGES) & ((1u << AR_PAGES) - 1);
        if (ahead < steps) copy_step(ahead);
        cp_async_commit();
        const uint8_t* const at = ring + stage * Sh::STAGE;
        const int key0 = (b_begin + warp + i * AR_WARPS) * AR_KEYS;
        float s[R][4][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[r][j][0] = s[r][j][1] = s[r][j][2] = s[r][j][3] = 0.f;
#pragma unroll
        for (int h = 0; h < Sh::CHUNKS; ++h)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint4 qv[R][Sh::PLANES];
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int p = 0; p < Sh::PLANES; ++p)
                        qv[r][p] = *reinterpret_cast<const uint4*>(qs + ((r * Sh::PLANES + p) * Sh::STEPS + 4 * h + w) * 512 + lane * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t k = *reinterpret_cast<const uint32_t*>(at + ((j * Sh::CHUNKS + h) * 32 + lane) * 16 + 4 * w);
                    uint32_t b0, b1;
                    af_halves(k, b0, b1);
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int p = Sh::PLANES - 1; p >= 0; --p) af_mma(s[r][j], qv[r][p], b0, b1);
                }
            }
        const float* const scales = reinterpret_cast<const float*>(at + 2 * Sh::KBYTES);
        float2 ks[4], vs[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ks[j] = *reinterpret_cast<const float2*>(scales + 8 * j + 2 * t);
            vs[j] = *reinterpret_cast<const float2*>(scales + AR_KEYS + 8 * j + 2 * t);
        }
        const bool masked = gone != 0 || key0 < whole_from || key0 + AR_KEYS - 1 > whole_to;
        float big = 0.f;  // the largest finite scale of values that a row of the tile may see
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = key0 + 8 * j + 2 * t;
            if (vs[j].x < INFINITY && (!masked || (k >= k_begin && k < k_end))) big = fmaxf(big, vs[j].x);
            if (vs[j].y < INFINITY && (!masked || (k + 1 >= k_begin && k + 1 < k_end))) big = fmaxf(big, vs[j].y);
        }
        float best[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                best[r][e] = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float& z = s[r][j][2 * e + c];
                        z = z * (c ? ks[j].y : ks[j].x) * factor[r][e];
                        if (masked) {
                            const int k = key0 + 8 * j + 2 * t + c;
                            if (k > limit[r][e] || k < low[r][e] || (gone >> (j / 2) & 1)) z = -INFINITY;
                        }
                        best[r][e] = fmaxf(best[r][e], z);
                    }
            }
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
            big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, x));
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < 2; ++e) best[r][e] = fmaxf(best[r][e], __shfl_xor_sync(0xFFFFFFFFu, best[r][e], x));
        }
        bool move = big > ref;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) move |= best[r][e] > m[r][e] + AF_LAZY;  // (of -inf: as soon as there is a score)
        if (__any_sync(0xFFFFFFFFu, move)) {
            const float up = fmaxf(ref, af_power(big)), shrink = ref / up;  // (powers of two)
            ref = up;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float to = fmaxf(m[r][e], best[r][e]), by = m[r][e] == to ? 1.f : af_ex2(m[r][e] - to);
                    m[r][e] = to;
                    l[r][e] *= by;
#pragma unroll
                    for (int j = 0; j < DP / 8; ++j) {
                        o[r][j][2 * e] *= by * shrink;
                        o[r][j][2 * e + 1] *= by * shrink;
                    }
                }
        }
        const float lift = AF_LIFT / ref;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float from = m[r][e] == -INFINITY ? 0.f : m[r][e];
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float& z = s[r][j][2 * e + c];
                        const float w = af_ex2(z - from);
                        l[r][e] += w;
                        z = masked && z == -INFINITY ? 0.f : w * ((c ? vs[j].y : vs[j].x) * lift);  // (what is masked may have any scale)
                    }
            }
#pragma unroll
        for (int pg = 0; pg < AR_PAGES; ++pg) {
            uint4 pa[R][Sh::PLANES];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float (&u)[4] = s[r][2 * pg], (&v)[4] = s[r][2 * pg + 1];
                if constexpr (F32) {
                    af_split(u[0], u[1], pa[r][0].x, pa[r][1].x);
                    af_split(u[2], u[3], pa[r][0].y, pa[r][1].y);
                    af_split(v[0], v[1], pa[r][0].z, pa[r][1].z);
                    af_split(v[2], v[3], pa[r][0].w, pa[r][1].w);
                } else {
                    pa[r][0] = make_uint4(af_pack(u[0], u[1]), af_pack(u[2], u[3]), af_pack(v[0], v[1]), af_pack(v[2], v[3]));
                }
            }
            constexpr int WORDS = DP / 32;  // of a thread's part of a token's values
            uint32_t vw[4][WORDS];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint8_t* const from = at + Sh::KBYTES + ((pg * 4 + j) * 32 + lane) * (DP / 8);
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
                uint32_t b0[4], b1[4];  // of four coordinates: tokens 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
                af_halves(__byte_perm(vw[0][w], vw[1][w], 0x5140), b0[0], b0[1]);
                af_halves(__byte_perm(vw[0][w], vw[1][w], 0x7362), b0[2], b0[3]);
                af_halves(__byte_perm(vw[2][w], vw[3][w], 0x5140), b1[0], b1[1]);
                af_halves(__byte_perm(vw[2][w], vw[3][w], 0x7362), b1[2], b1[3]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    b0[q] = af_finite(b0[q]);
                    b1[q] = af_finite(b1[q]);
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int p = Sh::PLANES - 1; p >= 0; --p) af_mma(o[r][4 * w + q], pa[r][p], b0[q], b1[q]);
                }
            }
        }
    }
    cp_async_wait<0>();
    // ── the warps' sums into one, then the blocks' ──
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[r][e] += __shfl_xor_sync(0xFFFFFFFFu, l[r][e], 1);
            l[r][e] += __shfl_xor_sync(0xFFFFFFFFu, l[r][e], 2);
            if (t == 0) {
                warp_m[warp][16 * r + g + 8 * e] = m[r][e];
                warp_l[warp][16 * r + g + 8 * e] = l[r][e];
            }
        }
    __syncthreads();  // the rings have been read
    float* const sums = reinterpret_cast<float*>(ar_smem + Sh::Q);  // [warp][row][LDO]
    const float back = ref * (1.f / AF_LIFT);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < DP / 8; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)  // column c of product j is coordinate DP / 8 c + j
                sums[(warp * Sh::ROWS + 16 * r + g + 8 * (q / 2)) * Sh::LDO + DP / 8 * (2 * t + q % 2) + j] = o[r][j][q] * back;
    __syncthreads();
    auto store = [&](int row, int col, float y) {
        const int at = tile.row0 + row;
        static_cast<T*>(a.out)[(int64_t)(tile.first + at / group) * a.ldo + (int64_t)(head * group + at % group) * dim + col] = from_f32<T>(y);
    };
    for (int row = warp; row < tile.n; row += AR_WARPS) {
        float top = -INFINITY, total = 0.f, w[AR_WARPS], y[DP / 32];
#pragma unroll
        for (int i = 0; i < AR_WARPS; ++i) top = fmaxf(top, warp_m[i][row]);
#pragma unroll
        for (int i = 0; i < AR_WARPS; ++i) {
            w[i] = warp_m[i][row] == -INFINITY ? 0.f : af_ex2(warp_m[i][row] - top);
            total += warp_l[i][row] * w[i];
        }
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            y[c] = 0.f;
#pragma unroll
            for (int i = 0; i < AR_WARPS; ++i) y[c] = fmaf(sums[(i * Sh::ROWS + row) * Sh::LDO + 32 * c + lane], w[i], y[c]);
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
    for (int row = part + parts * warp; row < tile.n; row += parts * AR_WARPS) {  // the cluster's warps share the rows out
        // lane i looks at part i
        const float pm = lane < parts ? ld_peer(peer_smem(smem_addr(&part_m[row]), lane)) : -INFINITY;
        const float pl = lane < parts ? ld_peer(peer_smem(smem_addr(&part_l[row]), lane)) : 0.f;
        const float top = warp_max(pm), w = pm == -INFINITY ? 0.f : af_ex2(pm - top), total = warp_sum(pl * w);
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

template <typename T, int DP, int R>
static cudaError_t launch_rows(const AttentionFp8Args& a, cudaStream_t st) {
    using Sh = ArShape<T, DP, R>;
    static PerDeviceOnce once;
    cudaError_t e = once.run([] {
        const cudaError_t f = cudaFuncSetAttribute(attention_rows_kernel<T, DP, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM);
        return f != cudaSuccess ? f : cudaFuncSetAttribute(attention_rows_kernel<T, DP, R>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);  // (more than eight blocks)
    });
    if (e != cudaSuccess) return e;
    const int64_t rows = (int64_t)a.max_rows * (a.n_heads / a.c.n_kv), tiles = (rows + Sh::ROWS - 1) / Sh::ROWS, clusters = tiles * a.c.n_kv * a.n_seqs;
    // two blocks an SM, each with 256 keys at least
    int parts = 1;
    while (parts < AR_MAX_PARTS && clusters * parts * 2 <= 2 * device_sm_count() && (int64_t)a.max_len >= 256 * 2 * parts) parts *= 2;
    e = launch_pdl_cluster(attention_rows_kernel<T, DP, R>, dim3((unsigned)(tiles * a.c.n_kv), (unsigned)a.n_seqs, (unsigned)parts), dim3(AR_THREADS), Sh::SMEM, st, parts, a, parts);
    return e != cudaSuccess ? e : count_launch_and_check();
}

template <typename T>
static cudaError_t attention_as(const AttentionFp8Args& a, cudaStream_t st) {
    const int64_t rows = (int64_t)a.max_rows * (a.n_heads / a.c.n_kv);
    const bool tiles = (int64_t)a.c.n_pages * 2 * a.c.n_kv * KV_PAGE <= INT32_MAX;  // (a copy's row is counted in 32 bits)
    if (rows > 32 && tiles) return launch_attention_fp8_tiles(a, sizeof(T) == 2, st);
    const bool few = rows <= 16;
    if (a.c.dim <= 64) return few ? launch_rows<T, 64, 1>(a, st) : launch_rows<T, 64, 2>(a, st);
    return few ? launch_rows<T, 128, 1>(a, st) : launch_rows<T, 128, 2>(a, st);
}
cudaError_t launch_attention_fp8(const AttentionFp8Args& a, bool bf, cudaStream_t st) { return bf ? attention_as<bf16>(a, st) : attention_as<float>(a, st); }

}  // namespace sp
