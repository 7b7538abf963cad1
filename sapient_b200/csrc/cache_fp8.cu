// Writing keys and values into a paged cache of 8-bit rows, with the norms and the rotation that precede it, and reading them back.
//
//   head h of a token:  y = x                                   or  x / sqrt(mean(x^2) + eps) * w   (w of queries, of keys)
//                       (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin)   for the pairs of the first `rotary` coordinates
//   queries leave as they are, keys and values as  scale = max(max |y| / 448, 2^-100),  q = e4m3(y / scale)
//
// Everything is f32 between the one read and the one write.
#include "cache_fp8.h"

#include <algorithm>

#include "fp8_rows.cuh"
#include "pdl.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

// ── append ──
// A head is 4 or 8 threads of 16 coordinates each: eight pairs that are rotated together, so that nothing is exchanged but a sum and a
// maximum. The teams of a token take its heads in turn, the next one on its way; place and angles are loaded once. Few tokens are spread over
// as many threads as they have heads for (1 token of the 8B shape 2.2 us, with two warps 3.3), of many a token is two warps' (8192 tokens 39.2
// us, with a team for each head 57.6; two or three heads at a time 46 and 49: registers). What is left above the bytes' 28.4 us (1024 tokens 8.9 of 3.6,
// 4096 23.2 of 14.5) is a start in which SMs wait for their first rows, and too few of them on their way: 80 registers leave a third of an SM's warps.
constexpr int CA_THREADS = 256;

template <typename T, int TEAM>
__global__ void __launch_bounds__(CA_THREADS) cache_append_kernel(const CacheAppendArgs a, int per_token) {  // threads of a token, whole warps
    pdl_wait();
    pdl_trigger();
    const int64_t tok = (int64_t)blockIdx.x * (blockDim.x / per_token) + threadIdx.x / per_token;
    if (tok >= a.n_tok) return;
    const int slot = a.slots[tok], pos = a.positions[tok];
    const int mine = threadIdx.x % per_token, part = mine % TEAM, team = mine / TEAM, teams = per_token / TEAM, dim = a.c.dim, half = a.rotary / 2;
    const bool live = 16 * part < dim, turns = 16 * part < a.rotary;
    // coordinates of the thread: two runs of eight
    int e0 = 16 * part, e1 = e0 + 8;
    if (turns && !a.pairs) { e0 = 8 * part; e1 = half + 8 * part; }
    const int queries = a.q ? a.n_heads : 0, heads = queries + 2 * a.c.n_kv;
    const T *const q0 = static_cast<const T*>(a.q) + tok * a.ldq, *const k0 = static_cast<const T*>(a.k) + tok * a.ldk - (int64_t)queries * dim,
            *const v0 = static_cast<const T*>(a.v) + tok * a.ldv - (int64_t)(queries + a.c.n_kv) * dim;
    Raw8<T> next[2];
    auto load = [&](int h) {
        if (live && h < heads) {
            const T* const from = (h < queries ? q0 : h < queries + a.c.n_kv ? k0 : v0) + h * dim;
            next[0] = ld8(from + e0);
            next[1] = ld8(from + e1);
        }
    };
    load(team);  // (before the place is known, which takes two loads one after the other)
    if (!a.c.has(slot, pos) || (a.rotary > 0 && pos >= a.n_angles)) return;
    const int page = a.c.page_of(slot, pos), row = pos % KV_PAGE;
    float cosine[8], sine[8];
    if (turns) {
        const float4* const at = reinterpret_cast<const float4*>(a.angles + (int64_t)pos * half + 8 * part);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 w = at[i];
            cosine[2 * i] = w.x; sine[2 * i] = w.y;
            cosine[2 * i + 1] = w.z; sine[2 * i + 1] = w.w;
        }
    }
    for (int h = team; __any_sync(0xFFFFFFFFu, h < heads); h += teams) {  // (a warp's threads go round together: they exchange values)
        const Raw8<T> raw[2] = {next[0], next[1]};
        load(h + teams);
        const int kind = h < queries ? 0 : h < queries + a.c.n_kv ? 1 : 2;  // query, key, value
        const bool here = live && h < heads;
        float x[8], y[8];
        if (here) {
            unpack8(raw[0], x);
            unpack8(raw[1], y);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
        }
        const float* const w = kind == 0 ? a.q_w : kind == 1 ? a.k_w : nullptr;
        if (__any_sync(0xFFFFFFFFu, w != nullptr)) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], fmaf(y[i], y[i], sum));
#pragma unroll
            for (int o = TEAM / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (w && here) {
                const float factor = rsqrtf(sum / (float)dim + a.eps);
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 u = *reinterpret_cast<const float4*>(w + e0 + i), v = *reinterpret_cast<const float4*>(w + e1 + i);
                    x[i] *= factor * u.x; x[i + 1] *= factor * u.y; x[i + 2] *= factor * u.z; x[i + 3] *= factor * u.w;
                    y[i] *= factor * v.x; y[i + 1] *= factor * v.y; y[i + 2] *= factor * v.z; y[i + 3] *= factor * v.w;
                }
            }
        }
        if (turns && kind < 2) {
            if (a.pairs) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = x[2 * i], v = x[2 * i + 1], s = y[2 * i], t = y[2 * i + 1];
                    x[2 * i] = u * cosine[i] - v * sine[i];
                    x[2 * i + 1] = v * cosine[i] + u * sine[i];
                    y[2 * i] = s * cosine[4 + i] - t * sine[4 + i];
                    y[2 * i + 1] = t * cosine[4 + i] + s * sine[4 + i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float u = x[i], v = y[i];
                    x[i] = u * cosine[i] - v * sine[i];
                    y[i] = v * cosine[i] + u * sine[i];
                }
            }
        }
        if (here && kind == 0) {
            T* const to = static_cast<T*>(a.q_out) + tok * a.ldqo + (int64_t)h * dim;
            st8(to + e0, x);
            st8(to + e1, y);
        }
        if (__any_sync(0xFFFFFFFFu, kind != 0)) {
            float most = max_nan(greatest8(x), greatest8(y));
#pragma unroll
            for (int o = TEAM / 2; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
            if (here && kind != 0 && page >= 0) {
                const int64_t at = a.c.row(page, kind - 1, h - queries - (kind - 1) * a.c.n_kv) + row;
                const float scale = scale_of(most, 1.f), by = rcp_approx(scale);
                store8(x, by, a.c.values + at * dim + e0);
                store8(y, by, a.c.values + at * dim + e1);
                if (part == 0) a.c.scales[at] = scale;
            }
        }
    }
}

template <typename T>
static cudaError_t append_as(const CacheAppendArgs& a, cudaStream_t st) {
    const int team = a.c.dim <= 64 ? 4 : 8, heads = (a.q ? a.n_heads : 0) + 2 * a.c.n_kv;
    // fewer threads a token as soon as eleven warps an SM are left (8B shape, bf16, 256 and 64 threads: 128 tokens 2.8 and 4.3 us, 512 6.0 and 5.2, 1024 9.6
    // and 8.8, 4096 31.3 and 22.8; 0.5B shape, 96 and 64: 1024 2.8 and 3.5, 4096 8.2 and 7.8)
    int per_token = std::min(CA_THREADS, (heads * team + 31) / 32 * 32);
    while (per_token > 64 && a.n_tok * (per_token / 2) >= (int64_t)device_sm_count() * 352) per_token = (per_token / 2 + 31) / 32 * 32;
    const int tokens = std::max(1, 64 / per_token), threads = tokens * per_token;
    const cudaError_t e = launch_pdl(team == 4 ? cache_append_kernel<T, 4> : cache_append_kernel<T, 8>, dim3((unsigned)((a.n_tok + tokens - 1) / tokens)), dim3(threads), 0, st, a, per_token);
    return e != cudaSuccess ? e : count_launch_and_check();
}
cudaError_t launch_cache_append(const CacheAppendArgs& a, bool bf, cudaStream_t st) { return bf ? append_as<bf16>(a, st) : append_as<float>(a, st); }

// ── read ──
// A thread takes eight coordinates at a time. Few tokens: a block has one. Many: a warp has four, whose pages are looked up at once, and eight
// requests on their way where a token's pieces are that many (from memory, bf16, four tokens a warp and a token a block; 8B shape, 256 pieces: 65536 tokens
// 76.9 us and 90.7, 20000 28.1 and 29.4, 8192 13.9 and 13.8, 2048 7.3 and 4.1; 0.5B shape, 32 pieces: 65536 31.8 and 68.6, 20000 11.8 and 21.4,
// 8192 6.3 and 9.3, 2048 5.0 and 3.8). The border is set for wide tokens: narrow ones would cross over near 4000.
constexpr int CR_THREADS = 128, CR_TOKENS = 4, CR_MANY = 10000;

template <typename T, int TOKENS>
__global__ void __launch_bounds__(CR_THREADS) cache_read_kernel(const CacheReadArgs a) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, per = a.c.dim / 8, pieces = a.c.n_kv * per;
    const int64_t first = TOKENS == 1 ? blockIdx.x : ((int64_t)blockIdx.x * (CR_THREADS / 32) + threadIdx.x / 32) * TOKENS;
    int page = -1, pos = 0;
    if (lane < TOKENS && first + lane < a.n_tok) {
        const int slot = a.slots[first + lane];
        pos = a.positions[first + lane];
        if (a.c.has(slot, pos)) page = a.c.page_of(slot, pos);
    }
#pragma unroll 1
    for (int i = 0; i < TOKENS; ++i) {
        const int64_t tok = first + i;
        const int pg = __shfl_sync(0xFFFFFFFFu, page, i), row = __shfl_sync(0xFFFFFFFFu, pos, i) % KV_PAGE;
        if (pg < 0) continue;
        constexpr int STEP = TOKENS == 1 ? CR_THREADS : 32, N = TOKENS == 1 ? 2 : 8;
#pragma unroll 1
        for (int p0 = TOKENS == 1 ? threadIdx.x : lane; p0 < 2 * pieces; p0 += N * STEP) {
            uint2 raw[N];
            float scale[N];
            T* to[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int i0 = p0 + n * STEP, which = i0 >= pieces, p = i0 - which * pieces, h = p / per, c = 8 * (p - h * per);
                T* const base = static_cast<T*>(which ? a.v : a.k);
                to[n] = nullptr;
                if (i0 < 2 * pieces && base) {
                    const int64_t at = a.c.row(pg, which, h) + row;
                    raw[n] = *reinterpret_cast<const uint2*>(a.c.values + at * a.c.dim + c);
                    scale[n] = a.c.scales[at];
                    to[n] = base + tok * (which ? a.ldv : a.ldk) + 8 * p;
                }
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (!to[n]) continue;
                float y[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t two = (j < 2 ? raw[n].x : raw[n].y) >> (16 * (j & 1)) & 0xFFFFu;
                    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3)));
                    y[2 * j] = f.x * scale[n];
                    y[2 * j + 1] = f.y * scale[n];
                }
                st8(to[n], y);
            }
        }
    }
}

template <typename T>
static cudaError_t read_as(const CacheReadArgs& a, cudaStream_t st) {
    const bool many = a.n_tok >= CR_MANY;
    const int64_t per_block = many ? CR_THREADS / 32 * CR_TOKENS : 1;
    const cudaError_t e = launch_pdl(many ? cache_read_kernel<T, CR_TOKENS> : cache_read_kernel<T, 1>, dim3((unsigned)((a.n_tok + per_block - 1) / per_block)), dim3(CR_THREADS), 0, st, a);
    return e != cudaSuccess ? e : count_launch_and_check();
}
cudaError_t launch_cache_read(const CacheReadArgs& a, bool bf, cudaStream_t st) { return bf ? read_as<bf16>(a, st) : read_as<float>(a, st); }

}  // namespace sp
