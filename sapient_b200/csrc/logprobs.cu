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
constexpr int LP_STAGES = 3;          // chunks of a block on their way or in use
constexpr int LP_BUF = 256;           // candidates for the largest
constexpr int LP_CELLS = 4;           // maxima a thread keeps
constexpr int LP_QUEUE = 512;         // of them that can be read again
constexpr int LP_MAX_PARTS = 8;       // blocks of a row
constexpr float LP_LOW = -200.f;      // lp_exp is zero from here down; keeps 0 x infinity out of T
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
__device__ __forceinline__ float lp_max(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// exp without the handling of results below 2^-126, which are zero here.
__device__ __forceinline__ float lp_exp(float v) {
    float d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v * 1.4426950408889634f));
    return d;
}

// Running sums of a part of a row. m: its maximum (-inf: nothing but masked values so far); bad: it holds a NaN or +inf.
struct __align__(16) LpSums {
    float m, r, t;
    int bad;
};
__device__ __forceinline__ LpSums lp_join(const LpSums& a, const LpSums& b) {
    const bool first = a.m >= b.m;
    const LpSums &u = first ? a : b, &v = first ? b : a;  // u: the greater maximum
    LpSums o = u;
    o.bad = a.bad | b.bad;
    if (v.m > -INFINITY && !o.bad) {
        const float d = fmaxf(v.m - u.m, LP_LOW), f = lp_exp(d), s = v.r + 1.f;
        o.r = fmaf(f, s, u.r);
        o.t = fmaf(f, fmaf(d, s, v.t), u.t);
    }
    return o;
}
__device__ __forceinline__ LpSums lp_shfl(const LpSums& a, int o) {
    return LpSums{__shfl_xor_sync(LP_ALL, a.m, o), __shfl_xor_sync(LP_ALL, a.r, o), __shfl_xor_sync(LP_ALL, a.t, o), __shfl_xor_sync(LP_ALL, a.bad, o)};
}

// The nth largest (from 0) of a warp's values.
__device__ __forceinline__ uint32_t lp_nth(uint32_t v, int nth, int lane) {
    int rank = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const uint32_t o = __shfl_sync(LP_ALL, v, i);
        rank += o > v || (o == v && i < lane);
    }
    return __shfl_sync(LP_ALL, v, __ffs(__ballot_sync(LP_ALL, rank == nth)) - 1);
}

struct LpShared {
    float cells[LP_CELLS][LP_THREADS];
    uint64_t inbox[LP_MAX_PARTS * LOGPROBS_MAX_TOP];  // of a cluster's first block: every part's largest
    LpSums parts[LP_MAX_PARTS];                       // and sums
    LpSums sums[LP_WARPS];
    int count, queued;
};
// In the ring's place once the row has been read.
struct LpTail {
    uint64_t buf[LP_BUF];
    uint64_t list[LOGPROBS_MAX_TOP];  // the result
    union {
        uint32_t first[LP_THREADS];
        uint16_t queue[LP_QUEUE];
    };
};

// The largest of n keys (0: none), sorted, to list: a key's place is the number of greater ones. Every thread calls.
__device__ __forceinline__ void lp_largest(const uint64_t* keys, int n, uint64_t* list, int tid) {
    const uint64_t mine = tid < n ? keys[tid] : 0;
    if (tid < LOGPROBS_MAX_TOP) list[tid] = 0;
    __syncthreads();
    int rank = 0;
    if (tid / 32 * 32 < n)
        for (int i = 0; i < n; ++i) rank += keys[i] > mine;
    if (mine && rank < LOGPROBS_MAX_TOP) list[rank] = mine;
    __syncthreads();
}

__device__ __forceinline__ void lp_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void lp_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
// The same place in the cluster's first block.
__device__ __forceinline__ uint32_t lp_first(const void* p) {
    uint32_t d;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(d) : "r"((uint32_t)__cvta_generic_to_shared(p)));
    return d;
}

// Copies a whole 16-byte piece of a row to shared memory, without waiting.
__device__ __forceinline__ void lp_copy(uint4* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
// A 16-byte piece of a row whose first value has index e0: nothing outside the row's n values is read.
template <typename T>
__device__ __forceinline__ uint4 lp_piece(const T* row, int64_t e0, int n) {
    constexpr int VEC = 16 / sizeof(T);
    if (e0 >= 0 && e0 + VEC <= n) return *reinterpret_cast<const uint4*>(row + e0);
    union {
        uint4 all;
        uint16_t half[8];
        uint32_t word[4];
    } v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const T x = e0 + i >= 0 && e0 + i < n ? row[e0 + i] : (T)-INFINITY;
        if constexpr (sizeof(T) == 2) v.half[i] = *reinterpret_cast<const uint16_t*>(&x);
        else v.word[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
    return v.all;
}
__device__ __forceinline__ void lp_unpack(const uint4& f, float* v, float) {
    v[0] = __uint_as_float(f.x); v[1] = __uint_as_float(f.y); v[2] = __uint_as_float(f.z); v[3] = __uint_as_float(f.w);
}
__device__ __forceinline__ void lp_unpack(const uint4& f, float* v, bf16) {
    const uint32_t u[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 4) logprobs_kernel(const LogprobsArgs a, int parts) {
    __shared__ LpShared sh;
    extern __shared__ uint4 lp_ring[];  // [stage][piece][thread]: a thread reads what it has copied, so that no barrier stands between
    constexpr int VEC = 16 / sizeof(T), PIECES = LP_VALUES / VEC, STEP = LP_THREADS * PIECES;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t r = blockIdx.x / parts;
    const int part = blockIdx.x - (int)r * parts;
    const T* const row = static_cast<const T*>(a.z) + r * a.ld;
    // pieces start on 16-byte boundaries: the first and the last may hang over the row's ends
    const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int pieces = (int)(((int64_t)skew + a.n + VEC - 1) / VEC), per = (pieces + parts - 1) / parts;
    const int begin = min(part * per, pieces), end = min(begin + per, pieces);
    LpTail& tail = *reinterpret_cast<LpTail*>(lp_ring);
    if (TOP && tid == 0) sh.count = sh.queued = 0;
    if (parts > 1) lp_cluster_arrive();  // (waited for before a peer's memory is written: all blocks run by then)
    pdl_wait();
    pdl_trigger();
    float given = 0.f;
    uint32_t id = 0;
    if (part == 0 && tid == 0 && a.ids) {
        id = a.ids[r];
        given = id < (uint32_t)a.n ? (float)row[id] : 0.f;
    }
    LpSums s{-INFINITY, 0.f, 0.f, 0};  // m and bad: of the warp
    bool holds = false;
    const int chunks = (end - begin + STEP - 1) / STEP;
    // A thread's maxima over runs of `cell` chunks stay in shared memory: where the largest values are looked for afterwards.
    const int cell = (chunks + LP_CELLS - 1) / LP_CELLS;
    int n_cells = 0, in_cell = 0;
    float peak = -INFINITY;
    auto fetch = [&](int k) {
        if (k < chunks) {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                uint4* const to = lp_ring + (k % LP_STAGES * PIECES + j) * LP_THREADS + tid;
                const int p = begin + k * STEP + j * LP_THREADS + tid, e0 = p * VEC - skew;
                if (p < end && e0 >= 0 && e0 + VEC <= a.n) {
                    lp_copy(to, row + e0);
                } else {  // past the part, or a piece that hangs over an end of the row: masked values in the others' places
                    *to = lp_piece(row, e0, p < end ? a.n : 0);
                }
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < LP_STAGES - 1; ++k) fetch(k);
    for (int k = 0; k < chunks; ++k) {
        fetch(k + LP_STAGES - 1);
        asm volatile("cp.async.wait_group %0;\n" ::"n"(LP_STAGES - 1) : "memory");
        const uint4* const mine = lp_ring + k % LP_STAGES * PIECES * LP_THREADS + tid;
        float x[LP_VALUES];
#pragma unroll
        for (int j = 0; j < PIECES; ++j) lp_unpack(mine[j * LP_THREADS], x + j * VEC, T());
        float c = lp_max(x[0], x[1]);
#pragma unroll
        for (int i = 2; i < LP_VALUES; i += 2) c = lp_max(c, x[i], x[i + 1]);

        if (TOP) {
            peak = lp_max(peak, c);
            if (++in_cell == cell || k + 1 == chunks) {
                sh.cells[n_cells++][tid] = peak;
                peak = -INFINITY;
                in_cell = 0;
            }
        }
        // The maximum is the warp's: lanes would have new ones of their own in nearly every chunk, and the warp would walk both ways. One
        // lane holds it, and leaves that one value out of its sums.
        if (__any_sync(LP_ALL, !(c <= s.m))) {
            float m = c;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = lp_max(m, __shfl_xor_sync(LP_ALL, m, o));
            if (!(m < INFINITY)) s.bad = 1;  // (the sums mean nothing from here on)
            else {
                if (s.m > -INFINITY) {
                    if (holds) s.r += 1.f;
                    const float d = fmaxf(s.m - m, LP_LOW), f = lp_exp(d);
                    s.t = f * fmaf(d, s.r, s.t);
                    s.r *= f;
                }
                s.m = m;
                const uint32_t who = __ballot_sync(LP_ALL, c == m);
                holds = lane == __ffs(who) - 1;
                if (holds) {
                    int skip = 0;
#pragma unroll
                    for (int i = LP_VALUES - 1; i >= 0; --i)
                        if (x[i] == m) skip = i;
#pragma unroll
                    for (int i = 0; i < LP_VALUES; ++i)
                        if (i == skip) x[i] = -INFINITY;
                }
            }
        }
        if (s.m > -INFINITY) {
            float r0 = 0.f, r1 = 0.f, t0 = 0.f, t1 = 0.f;
#pragma unroll
            for (int i = 0; i < LP_VALUES; i += 2) {
                const float d0 = fmaxf(x[i] - s.m, LP_LOW), d1 = fmaxf(x[i + 1] - s.m, LP_LOW), e0 = lp_exp(d0), e1 = lp_exp(d1);
                r0 += e0;
                r1 += e1;
                t0 = fmaf(d0, e0, t0);
                t1 = fmaf(d1, e1, t1);
            }
            s.r += r0 + r1;
            s.t += t0 + t1;
        }
    }

    // the block's sums
    s.r = warp_sum(s.r);
    s.t = warp_sum(s.t);
    if (lane == 0) sh.sums[warp] = s;
    __syncthreads();
    if (TOP) {
        // a first threshold: the `top`-th largest of the maxima of 32 groups of eight threads, which that many values reach
        peak = -INFINITY;
        for (int j = 0; j < n_cells; ++j) peak = lp_max(peak, sh.cells[j][tid]);
        tail.first[tid] = lp_mono(peak);
        __syncthreads();
        uint32_t m = tail.first[lane];
#pragma unroll
        for (int w = 1; w < LP_WARPS; ++w) m = max(m, tail.first[w * 32 + lane]);
        __syncthreads();  // (the maxima's place is the queue's)
        uint64_t threshold = (uint64_t)lp_nth(m, a.top - 1, lane) << 32;
        float low = lp_value((uint32_t)(threshold >> 32));
        // A value to the buffer, if it is a candidate: 0, there was room; 1, the buffer fills; 2, it is full.
        auto push = [&](float v, int id) {
            if (v < low || id < 0 || id >= a.n) return 0;
            const uint64_t key = lp_key(v, id);
            if (key <= threshold) return 0;
            const int at = atomicAdd(&sh.count, 1);
            if (at < LP_BUF) tail.buf[at] = key;
            return at < LP_BUF / 2 ? 0 : at < LP_BUF ? 1 : 2;
        };
        // the cells whose maximum is not below the threshold are read again, each by a warp, a piece a lane
        for (int j = 0; j < n_cells; ++j)
            if (!(sh.cells[j][tid] < low)) {
                const int at = atomicAdd(&sh.queued, 1);
                if (at < LP_QUEUE) tail.queue[at] = (uint16_t)(j * LP_THREADS + tid);
            }
        __syncthreads();
        const int queued = sh.queued, cell_pieces = cell * PIECES;
        bool over = queued > LP_QUEUE;
        constexpr int AHEAD = 4;  // cells of a warp on their way
        for (int q0 = warp; !over && q0 < queued; q0 += AHEAD * LP_WARPS)
            for (int u = lane; u < cell_pieces; u += 32) {
                uint4 got[AHEAD];
                int piece[AHEAD];
#pragma unroll
                for (int e = 0; e < AHEAD; ++e) {
                    const int q = q0 + e * LP_WARPS;
                    piece[e] = end;
                    if (q >= queued) continue;
                    const int from = tail.queue[q], k = from / LP_THREADS * cell + u / PIECES;
                    piece[e] = k < chunks ? begin + k * STEP + u % PIECES * LP_THREADS + from % LP_THREADS : end;
                    got[e] = lp_piece(row, (int64_t)piece[e] * VEC - skew, piece[e] < end ? a.n : 0);
                }
#pragma unroll
                for (int e = 0; e < AHEAD; ++e) {
                    if (piece[e] >= end) continue;
                    float v[VEC];
                    lp_unpack(got[e], v, T());
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (!(v[i] < low)) over |= push(v[i], piece[e] * VEC - skew + i) == 2;
                }
            }
        if (__syncthreads_or(over)) {
            // More candidates than places (many equal logits at the top): once more, a chunk at a time, cut back to the largest between.
            if (tid == 0) sh.count = 0;
            __syncthreads();
            for (int k = 0; k < chunks; ++k) {
                uint32_t pending = sh.cells[k / cell][tid] < low ? 0 : (1u << LP_VALUES) - 1;
                for (;;) {
                    int said = 0;
                    for (uint32_t left = pending; left; left &= left - 1) {
                        const int i = __ffs(left) - 1, p = begin + k * STEP + i / VEC * LP_THREADS + tid, id = p * VEC - skew + i % VEC;
                        const int got = p < end && id >= 0 && id < a.n ? push((float)row[id], id) : 0;
                        if (got < 2) pending &= ~(1u << i);
                        said = max(said, got);
                    }
                    if (!__syncthreads_or(said)) break;
                    lp_largest(tail.buf, min(sh.count, LP_BUF), tail.list, tid);
                    const uint64_t key = tail.list[lane];
                    const int kept = __popc(__ballot_sync(LP_ALL, key != 0));
                    if (warp == 0) tail.buf[lane] = key;
                    if (tid == 0) sh.count = kept;
                    threshold = max(threshold, tail.list[a.top - 1]);
                    low = lp_value((uint32_t)(threshold >> 32));
                    __syncthreads();
                }
            }
        }
        lp_largest(tail.buf, sh.count, tail.list, tid);
    }
    if (warp == 0) {
        s = sh.sums[lane & (LP_WARPS - 1)];
#pragma unroll
        for (int o = LP_WARPS / 2; o > 0; o >>= 1) s = lp_join(s, lp_shfl(s, o));
    }
    if (parts > 1) {
        // every block writes its part into the first one's memory, which goes on alone
        lp_cluster_wait();
        if (warp == 0) {
            if (lane == 0) {
                const uint32_t to = lp_first(&sh.parts[part]);
                asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(to), "r"(__float_as_uint(s.m)), "r"(__float_as_uint(s.r)), "r"(__float_as_uint(s.t)), "r"(s.bad) : "memory");
            }
            if (TOP && lane < a.top) asm volatile("st.shared::cluster.u64 [%0], %1;\n" ::"r"(lp_first(&sh.inbox[part * a.top + lane])), "l"(tail.list[lane]) : "memory");
        }
        __syncwarp();
        lp_cluster_arrive();
        lp_cluster_wait();
        if (part != 0) return;
        if (warp == 0) {
            s = (lane & (LP_MAX_PARTS - 1)) < parts ? sh.parts[lane & (LP_MAX_PARTS - 1)] : LpSums{-INFINITY, 0.f, 0.f, 0};
#pragma unroll
            for (int o = LP_MAX_PARTS / 2; o > 0; o >>= 1) s = lp_join(s, lp_shfl(s, o));
        }
        if (TOP) lp_largest(sh.inbox, parts * a.top, tail.list, tid);
    }
    const uint64_t best = TOP && warp == 0 ? tail.list[lane] : 0;
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
    while (parts < LP_MAX_PARTS && a.rows * parts * 2 <= 2 * sms && a.n / (parts * 2) >= LP_CHUNK) parts *= 2;
    if (a.rows * parts > INT32_MAX) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * parts));
    cfg.blockDim = dim3(LP_THREADS);
    cfg.dynamicSmemBytes = LP_STAGES * LP_CHUNK * sizeof(T);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    static PerDeviceOnce once;
    cudaError_t e = once.run([] {
        const cudaError_t f = cudaFuncSetAttribute(logprobs_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, LP_STAGES * LP_CHUNK * sizeof(T));
        return f != cudaSuccess ? f : cudaFuncSetAttribute(logprobs_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, LP_STAGES * LP_CHUNK * sizeof(T));
    });
    if (e != cudaSuccess) return e;
    e = a.top > 0 ? cudaLaunchKernelEx(&cfg, logprobs_kernel<T, true>, a, parts) : cudaLaunchKernelEx(&cfg, logprobs_kernel<T, false>, a, parts);
    return e != cudaSuccess ? e : count_launch_and_check();
}

cudaError_t launch_logprobs(const LogprobsArgs& a, bool bf, cudaStream_t st) {
    if (a.rows == 0) return cudaSuccess;
    if (a.n < 1 || a.top < 0 || a.top > LOGPROBS_MAX_TOP || a.top > a.n) return cudaErrorInvalidValue;
    return bf ? logprobs_of<bf16>(a, st) : logprobs_of<float>(a, st);
}

}  // namespace sp
