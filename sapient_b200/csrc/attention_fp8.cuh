// What the kernels of attention over a cache of 8-bit rows share (attention_fp8.cu, attention_fp8_tile.cu).
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "cache_fp8.h"
#include "fp8_rows.cuh"
#include "plan_common.cuh"

namespace sp {

constexpr float AF_LOG2E = 1.4426950408889634f;
// A row's reference m is the largest score when it was last moved; it is moved when a score passes it by more than this (log2).
constexpr float AF_LAZY = 6.f;
constexpr float AF_LIFT = 512.f;  // 2^(15 - LAZY)

// Four e4m3 values of a word as two pairs of fp16.
__device__ __forceinline__ void af_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}\n" : "=r"(lo), "=r"(hi) : "r"(w));
}
// NaN bytes of values become 448: they must not reach rows that do not see them through 0 x NaN. `dropped`, else 0, is NaN from the first on
// (a sum of zeros, on the pipe that has the least to do here; collected by the vector units' logic it took 3 to 5 % of the f32 tiles); then the rows that do
// see one are looked for at the end (af_nan_tokens, af_sees) and get NaN as their sum of weights.
__device__ __forceinline__ uint32_t af_finite(uint32_t two, uint32_t& dropped, bool live = true) {
    uint32_t d;
    asm("min.f16x2 %0, %1, %2;" : "=r"(d) : "r"(two), "r"(0x5F005F00u));
    if (live) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(dropped) : "r"(two), "r"(0u));
    return d;
}
__device__ __forceinline__ bool af_has_nan(const uint4& v) {
    auto of = [](uint32_t four) { return (four & 0x7F7F7F7Fu) + 0x01010101u; };  // a byte of 0x7F or 0xFF carries into its sign
    return ((of(v.x) | of(v.y) | of(v.z) | of(v.w)) & 0x80808080u) != 0;
}
// Of the 32 N tokens from key0 (a multiple of 32) to k_end, a bit for each that has a NaN among its values' bytes.
template <int N>
__device__ __forceinline__ void af_nan_tokens(const CacheFp8& c, const int32_t* table, int head, int key0, int k_end, uint32_t (&tokens)[N]) {
    const uint4* row[N];
    bool nan[N] = {};
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int key = key0 + 32 * n + (int)(threadIdx.x & 31), page = key < k_end ? table[key / KV_PAGE] : -1;
        row[n] = page >= 0 && page < c.n_pages ? reinterpret_cast<const uint4*>(c.values + (c.row(page, 1, head) + key % KV_PAGE) * c.dim) : nullptr;
    }
#pragma unroll 4
    for (int i = 0; i < c.dim / 16; ++i)
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (row[n]) nan[n] |= af_has_nan(row[n][i]);
#pragma unroll
    for (int n = 0; n < N; ++n) tokens[n] = __ballot_sync(0xFFFFFFFFu, nan[n]);
}
// Whether a row that sees keys low .. limit sees one of those tokens.
__device__ __forceinline__ bool af_sees(uint32_t tokens, int key0, int low, int limit) {
    const int from = max(low, key0) - key0, to = min(limit - key0, 31);
    return to >= from && (tokens >> from << (31 - to + from)) != 0;
}
// A scale; NaN for one that is infinite, with which a score of the wrong sign would be the weight 0.
__device__ __forceinline__ float af_number(float s) { return fmaf(s, 0.f, s); }
__device__ __forceinline__ uint32_t af_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// fp16 of two values, and of what that rounding dropped.
__device__ __forceinline__ void af_split(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = af_pack(a - f.x, b - f.y);
}
__device__ __forceinline__ void af_mma(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// A power of two by which a row is multiplied so that its largest value lies in [2^to, 2^(to + 1)), and its reciprocal. Rows of zeros: 1. Rows with
// infinities or NaN are multiplied by NaN: their scores are infinite or NaN, and so softmax has no value, but an infinity that is converted to e4m3
// would be a large number there.
__device__ __forceinline__ void af_row_scale(float most, int to, float& by, float& back) {
    const int e = (int)(__float_as_uint(most) >> 23);  // (most >= 0)
    const int up = e == 0 || e == 255 ? 0 : min(max(127 + to - e, -126), 126);
    by = __uint_as_float(e == 255 ? 0x7FC00000u : (uint32_t)(127 + up) << 23);
    back = __uint_as_float((uint32_t)(127 - up) << 23);
}
// The smallest power of two that is not below a scale (positive and finite), within what has a reciprocal.
__device__ __forceinline__ float af_power(float s) {
    const uint32_t u = (__float_as_uint(s) + 0x7FFFFFu) & 0x7F800000u;
    return __uint_as_float(min(max(u, 1u << 23), 253u << 23));
}

// ── attention_fp8.cu ──
cudaError_t af_page_map(const CacheFp8& c, CUtensorMap* map);
// How keys are shared out to the blocks of a cluster. What fits on the GPU at once depends on where its SMs are: of 148, clusters of 16 blocks that
// fill an SM each hold 112, of 10 or 8 110 and 120, of 6 132; eight clusters of 16 are two rounds.
constexpr int AF_MAX_PARTS = 16;
struct ClusterFits {
    std::atomic<int> at_once[AF_MAX_PARTS + 1];  // clusters of that many blocks (threads whose first calls coincide all write them)
};
cudaError_t af_fits(const void* kernel, int threads, int smem, ClusterFits* out);  // and the kernel's attributes for it
struct AfShare {
    int parts;
    double time;  // us
};
// The number of parts for which `clusters` of them take least, a block for `piece` of each of its share of `pieces`, and `fixed` and `joined` (where
// there are parts to add up) besides. Rounds that do not fill the GPU count half: blocks are of unequal length. `pieces` are the longest sequence's for every
// block: prompts and ragged batches have about half of that, so that their times come out too long.
AfShare af_share(const ClusterFits& fits, int64_t clusters, int64_t pieces, double piece, double fixed, double joined);
// attention_fp8_tile.cu; plan: nothing is launched, only how it would be, and how long it would take, is said
cudaError_t launch_attention_fp8_tiles(const AttentionFp8Args& a, bool bf, cudaStream_t st, AfShare* plan);
// Keys that a row can see, of the longest sequence.
inline int64_t af_keys(const AttentionFp8Args& a) { return a.window > 0 ? std::min<int64_t>(a.max_len, (int64_t)a.window + a.max_rows) : a.max_len; }

// What a block works on: rows of one key head of one sequence.
struct AfTile {
    int slot, len, rows, first;  // of the sequence; first: its first row in q
    int row0, n;                 // of the tile, in (token, head) rows of the sequence's key head
};
__device__ __forceinline__ AfTile af_tile(const AttentionFp8Args& a, int seq, int tile, int height) {
    AfTile t;
    const int len = a.seq_len[seq], end = a.row_start[seq + 1];  // (all on their way at once)
    t.first = a.row_start[seq];
    t.slot = a.seq_slot ? a.seq_slot[seq] : seq;
    t.rows = end - t.first;
    t.len = t.slot >= 0 && t.slot < a.c.n_slots ? max(len, 0) : 0;  // (a slot that is not there holds nothing)
    t.row0 = tile * height;
    t.n = min(height, min(t.rows, a.max_rows) * (a.n_heads / a.c.n_kv) - t.row0);
    return t;
}

}  // namespace sp
