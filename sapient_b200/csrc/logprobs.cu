// Token distributions from logits: log probability of a given token, entropy, and the most likely tokens, in one pass.
//
//   M = max x,  R = sum exp(x - M) over all but one maximum,  T = sum (x - M) exp(x - M)
//   log p(i) = x_i - M - log1p(R),   entropy = log1p(R) - T / (1 + R)
//
// The maximum's own 1 is kept out of R: where one token has nearly all of the mass, R and T are small numbers of full precision, and
// so are the two results. Sums are f32 per thread (a few hundred terms) and joined in a fixed order.
//
// A row is read by one block, or by a cluster of up to 16 where rows are few; bytes bound it from some hundred rows on, latency below.
// The largest ones are found on the way: a value that does not exceed the block's threshold, a lower bound of the `top`-th largest
// that rises as the row goes by, costs one comparison of a thread's 16 values' maximum; the others go to a buffer in shared memory,
// which is cut to the `top` largest when it fills. Keys (value, then lower index) are distinct, so that the order in which threads push
// changes nothing. The first threshold is the least of the maxima of 8 or 32 groups of threads: at least that many values reach it.
#include <cuda_bf16.h>

#include <algorithm>

#include "fp8.h"
#include "pdl.cuh"
#include "sp_common.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

using bf16 = __nv_bfloat16;

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_VALUES = 16;         // a thread's share of a chunk
constexpr int LP_CHUNK = LP_THREADS * LP_VALUES;
constexpr int LP_BUF = 1024;          // candidates
constexpr int LP_CUT = 512;           // cut back from here on
constexpr float LP_LOW = -200.f;      // exp is zero from here down in f32; keeps 0 x infinity out of T
constexpr unsigned LP_ALL = 0xFFFFFFFFu;

// Order-preserving bits: -0 counts as 0, any NaN as the largest.
__device__ __forceinline__ uint32_t lp_mono(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(v + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t m) { return __uint_as_float(m >> 31 ? m & 0x7FFFFFFFu : ~m); }
__device__ __forceinline__ uint64_t lp_key(float v, int index) { return (uint64_t)lp_mono(v) << 32 | (LP_ALL - (uint32_t)index); }

__device__ __forceinline__ float lp_max(float a, float b) {  // NaN where one is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Running sums of a part of a row. m: its maximum (-inf: nothing but masked values so far); bad: it holds a NaN or +inf.
struct LpSums {
    float m, r, t;
    int bad;
};
__device__ __forceinline__ LpSums lp_join(const LpSums& a, const LpSums& b) {
    const bool first = a.m >= b.m;
    const LpSums &u = first ? a : b, &v = first ? b : a;  // u: the greater maximum
    LpSums o = u;
    o.bad = a.bad | b.bad;
    if (v.m > -INFINITY && !o.bad) {
        const float d = fmaxf(v.m - u.m, LP_LOW), f = __expf(d), s = v.r + 1.f;
        o.r = fmaf(f, s, u.r);
        o.t = fmaf(f, fmaf(d, s, v.t), u.t);
    }
    return o;
}
__device__ __forceinline__ LpSums lp_shfl(const LpSums& a, int o) {
    return LpSums{__shfl_xor_sync(LP_ALL, a.m, o), __shfl_xor_sync(LP_ALL, a.r, o), __shfl_xor_sync(LP_ALL, a.t, o), __shfl_xor_sync(LP_ALL, a.bad, o)};
}

// 32 keys of a warp in descending order, and the 32 largest of two such lists.
__device__ __forceinline__ uint64_t lp_step(uint64_t k, int o, bool keep_max) {
    const uint64_t p = __shfl_xor_sync(LP_ALL, k, o);
    return (k > p) == keep_max ? k : p;
}
__device__ __forceinline__ uint64_t lp_merge_bitonic(uint64_t k, int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) k = lp_step(k, o, (lane & o) == 0);
    return k;
}
__device__ __forceinline__ uint64_t lp_sort(uint64_t k, int lane) {
#pragma unroll
    for (int w = 2; w <= 32; w *= 2)
#pragma unroll
        for (int o = w / 2; o > 0; o >>= 1) k = lp_step(k, o, ((lane & o) == 0) == ((lane & w) == 0 || w == 32));
    return k;
}
__device__ __forceinline__ uint64_t lp_merge(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = __shfl_sync(LP_ALL, b, 31 - lane);
    return lp_merge_bitonic(a > r ? a : r, lane);
}

struct LpShared {
    uint64_t buf[LP_BUF];
    uint64_t list[LP_WARPS][32];  // [0]: a part's result
    uint64_t threshold;
    LpSums sums[LP_WARPS];
    LpSums part;
    uint32_t first[LP_THREADS];
    int count;
};

// The lists of the block's warps to list[0]; every thread calls.
__device__ __forceinline__ void lp_join_lists(LpShared& sh, uint64_t mine, int warp, int lane) {
    sh.list[warp][lane] = mine;
#pragma unroll
    for (int half = LP_WARPS / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (warp < half) {
            mine = lp_merge(mine, sh.list[warp + half][lane], lane);
            sh.list[warp][lane] = mine;
        }
    }
    __syncthreads();
}
// The 32 largest candidates, sorted, to list[0].
__device__ __forceinline__ void lp_cut(LpShared& sh, int warp, int lane) {
    const int n = min(sh.count, LP_BUF);
    uint64_t best = 0;
    for (int g = warp * 32; g < n; g += LP_THREADS) {
        const uint64_t k = lp_sort(g + lane < n ? sh.buf[g + lane] : 0ull, lane);
        best = g < LP_THREADS ? k : lp_merge(best, k, lane);
    }
    lp_join_lists(sh, best, warp, lane);
}

__device__ __forceinline__ void lp_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t lp_peer(const void* p, int rank) {
    uint32_t d;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return d;
}
__device__ __forceinline__ uint64_t lp_ld_peer64(uint32_t a) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lp_ld_peer32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// One 16-byte piece of a row to values; e0: index of its first one, which the row need not have. Only whole pieces are read as such.
__device__ __forceinline__ void lp_load(const float* row, int64_t e0, int n, float* v) {
    if (e0 >= 0 && e0 + 4 <= n) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(row + e0));
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = e0 + i >= 0 && e0 + i < n ? row[e0 + i] : -INFINITY;
    }
}
__device__ __forceinline__ void lp_load(const bf16* row, int64_t e0, int n, float* v) {
    if (e0 >= 0 && e0 + 8 <= n) {
        const uint4 f = __ldcs(reinterpret_cast<const uint4*>(row + e0));
        const uint32_t u[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = e0 + i >= 0 && e0 + i < n ? __bfloat162float(row[e0 + i]) : -INFINITY;
    }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const LogprobsArgs a, int parts) {
    __shared__ LpShared sh;
    constexpr int VEC = 16 / sizeof(T), PIECES = LP_VALUES / VEC;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t r = blockIdx.x / parts;
    const int part = blockIdx.x - (int)r * parts;
    const T* const row = static_cast<const T*>(a.z) + r * a.ld;
    // pieces start on 16-byte boundaries: the first and the last may hang over the row's ends
    const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int pieces = (int)(((int64_t)skew + a.n + VEC - 1) / VEC), per = (pieces + parts - 1) / parts;
    const int begin = min(part * per, pieces), end = min(begin + per, pieces);
    if (TOP && tid == 0) sh.count = 0;
    pdl_wait();
    pdl_trigger();
    float given = 0.f;
    uint32_t id = 0;
    if (part == 0 && tid == 0 && a.ids) {
        id = a.ids[r];
        given = id < (uint32_t)a.n ? (float)row[id] : 0.f;
    }
    LpSums s{-INFINITY, 0.f, 0.f, 0};
    uint64_t threshold = 0;
    float low = -INFINITY;  // of the threshold

    float next[LP_VALUES];
    auto fetch = [&](int p0) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int p = p0 + j * LP_THREADS + tid;
            // (a piece past the part reads nothing: as if the row had ended)
            lp_load(row, (int64_t)p * VEC - skew, p < end ? a.n : -VEC, next + j * VEC);
        }
    };
    if (begin < end) fetch(begin);
    for (int p0 = begin; p0 < end; p0 += LP_THREADS * PIECES) {
        float x[LP_VALUES];
#pragma unroll
        for (int i = 0; i < LP_VALUES; ++i) x[i] = next[i];
        if (p0 + LP_THREADS * PIECES < end) fetch(p0 + LP_THREADS * PIECES);
        float c = x[0];
#pragma unroll
        for (int i = 1; i < LP_VALUES; ++i) c = lp_max(c, x[i]);

        if (!(c <= s.m)) {  // a new maximum, or a NaN
            if (!(c < INFINITY)) s.bad = 1;
            else {
                if (s.m > -INFINITY) {
                    const float d = fmaxf(s.m - c, LP_LOW), f = __expf(d);
                    s.t = f * fmaf(d, s.r + 1.f, s.t);
                    s.r = f * (s.r + 1.f);
                }
                s.m = c;
                bool seen = false;
#pragma unroll
                for (int i = 0; i < LP_VALUES; ++i) {
                    if (x[i] == c && !seen) { seen = true; continue; }
                    const float d = fmaxf(x[i] - c, LP_LOW), e = __expf(d);
                    s.r += e;
                    s.t = fmaf(d, e, s.t);
                }
            }
        } else if (c > -INFINITY) {
            float r0 = 0.f, r1 = 0.f, t0 = 0.f, t1 = 0.f;
#pragma unroll
            for (int i = 0; i < LP_VALUES; i += 2) {
                const float d0 = fmaxf(x[i] - s.m, LP_LOW), d1 = fmaxf(x[i + 1] - s.m, LP_LOW), e0 = __expf(d0), e1 = __expf(d1);
                r0 += e0;
                r1 += e1;
                t0 = fmaf(d0, e0, t0);
                t1 = fmaf(d1, e1, t1);
            }
            s.r += r0 + r1;
            s.t += t0 + t1;
        }

        if (TOP) {
            auto index = [&](int i) { return (p0 + (i / VEC) * LP_THREADS + tid) * VEC - skew + i % VEC; };
            auto there = [&](int i) { return p0 + (i / VEC) * LP_THREADS + tid < end && index(i) >= 0 && index(i) < a.n; };
            if (p0 == begin) {
                uint32_t m = 0;  // (a thread without values of its own: 0, below every key)
#pragma unroll
                for (int i = 0; i < LP_VALUES; ++i)
                    if (there(i)) m = max(m, lp_mono(x[i]));
                if (a.top <= LP_WARPS) {
                    m = __reduce_max_sync(LP_ALL, m);
                    if (lane == 0) sh.first[warp] = m;
                    __syncthreads();
                    m = sh.first[lane & (LP_WARPS - 1)];
                } else {
                    sh.first[tid] = m;
                    __syncthreads();
                    m = sh.first[lane];
#pragma unroll
                    for (int w = 1; w < LP_WARPS; ++w) m = max(m, sh.first[w * 32 + lane]);
                }
                threshold = (uint64_t)__reduce_min_sync(LP_ALL, m) << 32;
                low = lp_value((uint32_t)(threshold >> 32));
            }
            uint32_t pending = 0;
            if (!(c < low)) {
#pragma unroll
                for (int i = 0; i < LP_VALUES; ++i)
                    if (!(x[i] < low) && there(i)) pending |= 1u << i;
            }
            for (;;) {
                bool full = false;
                if (pending) {
#pragma unroll
                    for (int i = 0; i < LP_VALUES; ++i) {
                        if (!(pending >> i & 1)) continue;
                        const uint64_t k = lp_key(x[i], index(i));
                        if (k <= threshold) { pending &= ~(1u << i); continue; }
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < LP_BUF) {
                            sh.buf[at] = k;
                            pending &= ~(1u << i);
                        }
                        full |= at >= LP_CUT;
                    }
                }
                if (!__syncthreads_or(full)) break;
                lp_cut(sh, warp, lane);
                if (warp == 0) {
                    sh.buf[lane] = sh.list[0][lane];
                    if (lane == 0) {
                        // (a full buffer holds more than 32)
                        sh.count = 32;
                        sh.threshold = sh.list[0][a.top - 1];
                    }
                }
                __syncthreads();
                threshold = sh.threshold;
                low = lp_value((uint32_t)(threshold >> 32));
            }
        }
    }

    // the block's sums
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s = lp_join(s, lp_shfl(s, o));
    if (lane == 0) sh.sums[warp] = s;
    __syncthreads();
    if (TOP) lp_cut(sh, warp, lane);
    if (warp == 0) {
        s = sh.sums[lane & (LP_WARPS - 1)];
#pragma unroll
        for (int o = LP_WARPS / 2; o > 0; o >>= 1) s = lp_join(s, lp_shfl(s, o));
        if (parts > 1 && lane == 0) sh.part = s;
    }
    uint64_t best = TOP && warp == 0 ? sh.list[0][lane] : 0ull;
    if (parts > 1) {
        lp_cluster_sync();
        if (part == 0) {
            if (warp == 0) {
                const uint32_t p = lp_peer(&sh.part, lane < parts ? lane : 0);
                s = LpSums{__uint_as_float(lp_ld_peer32(p)), __uint_as_float(lp_ld_peer32(p + 4)), __uint_as_float(lp_ld_peer32(p + 8)), (int)lp_ld_peer32(p + 12)};
                if (lane >= parts) s = LpSums{-INFINITY, 0.f, 0.f, 0};
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) s = lp_join(s, lp_shfl(s, o));
            }
            if (TOP) {
                uint64_t mine = 0;
                for (int q = warp; q < parts; q += LP_WARPS) {
                    const uint64_t k = lp_ld_peer64(lp_peer(&sh.list[0][lane], q));
                    mine = q < LP_WARPS ? k : lp_merge(mine, k, lane);
                }
                __syncthreads();  // every warp has read this block's own list
                lp_join_lists(sh, mine, warp, lane);
                best = sh.list[0][lane];
            }
        }
        lp_cluster_sync();  // nobody leaves while its part is being read
        if (part != 0) return;
    }
    if (warp != 0) return;
    const bool empty = !(s.m > -INFINITY);  // nothing but masked values
    const float lse1 = log1pf(s.r), nan = __uint_as_float(0x7FC00000u);
    auto logprob = [&](float x) { return s.bad ? nan : empty ? -INFINITY : x - s.m - lse1; };
    if (lane == 0) {
        if (a.logprob && a.ids) a.logprob[r] = id < (uint32_t)a.n ? logprob(given) : nan;
        if (a.entropy) a.entropy[r] = s.bad ? nan : empty ? 0.f : lse1 - s.t / (1.f + s.r);
    }
    if (TOP && lane < a.top) {
        if (a.top_ids) a.top_ids[r * a.top + lane] = LP_ALL - (uint32_t)best;
        if (a.top_logprobs) a.top_logprobs[r * a.top + lane] = logprob(lp_value((uint32_t)(best >> 32)));
    }
}

template <typename T>
static cudaError_t logprobs_of(const LogprobsArgs& a, cudaStream_t st) {
    const int sms = device_sm_count();
    int parts = 1;
    while (parts < 8 && a.rows * parts * 2 <= 2 * sms && a.n / (parts * 2) >= LP_CHUNK) parts *= 2;
    if (a.rows * parts > INT32_MAX) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * parts));
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    const cudaError_t e = a.top > 0 ? cudaLaunchKernelEx(&cfg, logprobs_kernel<T, true>, a, parts) : cudaLaunchKernelEx(&cfg, logprobs_kernel<T, false>, a, parts);
    return e != cudaSuccess ? e : count_launch_and_check();
}

cudaError_t launch_logprobs(const LogprobsArgs& a, bool bf, cudaStream_t st) {
    if (a.rows == 0) return cudaSuccess;
    if (a.n < 1 || a.top < 0 || a.top > LOGPROBS_MAX_TOP || a.top > a.n) return cudaErrorInvalidValue;
    return bf ? logprobs_of<bf16>(a, st) : logprobs_of<float>(a, st);
}

}  // namespace sp
