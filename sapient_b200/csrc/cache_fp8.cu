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
// maximum. A block is a token; its teams take heads in turn, two on their way at a time, and the angles are loaded once.
constexpr int CA_THREADS = 256;

template <typename T, int TEAM>
__global__ void __launch_bounds__(CA_THREADS) cache_append_kernel(const CacheAppendArgs a) {
    pdl_wait();
    pdl_trigger();
    const int64_t tok = blockIdx.x;
    const int slot = a.slots[tok], pos = a.positions[tok];
    if (!a.c.has(slot, pos) || (a.rotary > 0 && pos >= a.n_angles)) return;
    const int part = threadIdx.x % TEAM, team = threadIdx.x / TEAM, teams = blockDim.x / TEAM, dim = a.c.dim, half = a.rotary / 2;
    const bool live = 16 * part < dim, turns = 16 * part < a.rotary;
    // coordinates of the thread: two runs of eight
    int e0 = 16 * part, e1 = e0 + 8;
    if (turns && !a.pairs) { e0 = 8 * part; e1 = half + 8 * part; }
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
    const int queries = a.q ? a.n_heads : 0, heads = queries + 2 * a.c.n_kv;
    auto source = [&](int h) -> const T* {
        if (h < queries) return static_cast<const T*>(a.q) + tok * a.ldq + (int64_t)h * dim;
        h -= queries;
        if (h < a.c.n_kv) return static_cast<const T*>(a.k) + tok * a.ldk + (int64_t)h * dim;
        return static_cast<const T*>(a.v) + tok * a.ldv + (int64_t)(h - a.c.n_kv) * dim;
    };
    constexpr int R = 2;
    for (int h0 = team; __any_sync(0xFFFFFFFFu, h0 < heads); h0 += R * teams) {  // (a warp's threads go round together: they exchange values)
        Raw8<T> raw[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int h = h0 + r * teams;
            if (live && h < heads) {
                raw[r][0] = ld8(source(h) + e0);
                raw[r][1] = ld8(source(h) + e1);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int h = h0 + r * teams, kind = h < queries ? 0 : h < queries + a.c.n_kv ? 1 : 2;  // query, key, value
            const bool here = live && h < heads;
            float x[8], y[8];
            if (here) {
                unpack8(raw[r][0], x);
                unpack8(raw[r][1], y);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
            }
            const float* const w = kind == 0 ? a.q_w : kind == 1 ? a.k_w : nullptr;
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
            float most = max_nan(greatest8(x), greatest8(y));
#pragma unroll
            for (int o = TEAM / 2; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
            if (!here) continue;
            if (kind == 0) {
                T* const to = static_cast<T*>(a.q_out) + tok * a.ldqo + (int64_t)h * dim;
                st8(to + e0, x);
                st8(to + e1, y);
            } else if (page >= 0) {
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
    // two heads a team, where that fits the block
    const int threads = std::min(CA_THREADS, ((heads + 1) / 2 * team + 31) / 32 * 32);
    const cudaError_t e = launch_pdl(team == 4 ? cache_append_kernel<T, 4> : cache_append_kernel<T, 8>, dim3((unsigned)a.n_tok), dim3(threads), 0, st, a);
    return e != cudaSuccess ? e : count_launch_and_check();
}
cudaError_t launch_cache_append(const CacheAppendArgs& a, bool bf, cudaStream_t st) { return bf ? append_as<bf16>(a, st) : append_as<float>(a, st); }

// ── read ──
// A thread takes eight coordinates; a block the rows of one token, so that its page is looked up once.
constexpr int CR_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(CR_THREADS) cache_read_kernel(const CacheReadArgs a) {
    pdl_wait();
    pdl_trigger();
    const int64_t tok = blockIdx.x;
    const int slot = a.slots[tok], pos = a.positions[tok];
    if (!a.c.has(slot, pos)) return;
    const int page = a.c.page_of(slot, pos);
    if (page < 0) return;
    const int per = a.c.dim / 8, pieces = a.c.n_kv * per;
    for (int i = threadIdx.x; i < 2 * pieces; i += CR_THREADS) {
        const int which = i >= pieces, p = i - which * pieces, h = p / per, c = 8 * (p - h * per);
        T* const to = static_cast<T*>(which ? a.v : a.k);
        if (!to) continue;
        const int64_t at = a.c.row(page, which, h) + pos % KV_PAGE;
        const uint2 raw = *reinterpret_cast<const uint2*>(a.c.values + at * a.c.dim + c);
        const float scale = a.c.scales[at];
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t two = (j < 2 ? raw.x : raw.y) >> (16 * (j & 1)) & 0xFFFFu;
            const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3)));
            y[2 * j] = f.x * scale;
            y[2 * j + 1] = f.y * scale;
        }
        st8(to + tok * (which ? a.ldv : a.ldk) + (int64_t)h * a.c.dim + c, y);
    }
}

template <typename T>
static cudaError_t read_as(const CacheReadArgs& a, cudaStream_t st) {
    const cudaError_t e = launch_pdl(cache_read_kernel<T>, dim3((unsigned)a.n_tok), dim3(CR_THREADS), 0, st, a);
    return e != cudaSuccess ? e : count_launch_and_check();
}
cudaError_t launch_cache_read(const CacheReadArgs& a, bool bf, cudaStream_t st) { return bf ? read_as<bf16>(a, st) : read_as<float>(a, st); }

}  // namespace sp
