// Token distributions from logits: log probability of a given token, entropy, and the most likely tokens, in one pass.
//
//   M = max x,  R = sum exp(x - M) over all but one maximum,  T = sum (x - M) exp(x - M)
//   log p(i) = x_i - M - log1p(R),   entropy = log1p(R) - T / (1 + R)
//
// The maximum's own 1 is kept out of R: where one token has nearly all of the mass, R and T are small numbers of full precision, and
// so are the two results. Sums are f32 per thread (a few hundred terms) and joined in a fixed order.
//
// A row is read by one block, or shared by a cluster of up to 16 where rows are few; its values pass through a ring of asynchronous
// copies in shared memory, 16 a thread at a time. The maximum is a warp's: of a row of random values a thread would find a new one of
// its own in most of its steps, and all of the warp would rescale. The `top` largest cost the reading pass a comparison a value: a
// thread keeps the maxima of a quarter each of what it reads (cells); afterwards the `top`-th largest of the maxima of groups of threads
// is a bound which that many values reach, the few cells that reach it are read again, from L2 or, of short rows, from the ring, and the
// values above it are ranked.
// Keys (value, then lower index) are distinct, so that no order of threads changes the result.
//
// Bytes bound it from some hundred rows on, with the exponentials close behind (16 a cycle and SM); below that the chain of steps does,
// a good part of it instructions that are fetched for the first time, so that what runs once is kept short. us, launched back
// to back by a small program (floor at 6.54 TB/s); calls on logits that change take 94.8 to 101.8 us for the first, 65 for the second:
//   1024 x 128256 f32 top 1      91.7 (80.3)     32 x 128256 bf16 top 20   10.8 (1.3)      1 x 151936 f32 top 5    7.1 (0.1)
//   1024 x 128256 bf16 top 1     59.9 (40.2)     64 x 128256 bf16 top 1    10.9 (2.5)      1 x 151936 f32 top 0    4.5 (0.1)
//   53 x 1913 bf16 top 12         4.7 (0.0; 7.0 with cells from L2)
// Two values an instruction wherever there is one (1024 x 128256 bf16 top 1: 64.5 us without).
#include <cuda_bf16.h>

#include <algorithm>

#include "fp8.h"
#include "pdl.cuh"
#include "sp_common.cuh"

namespace sp {

cudaError_t count_launch_and_check();  // kernels.cu

using bf16 = __nv_bfloat16;

constexpr int LP_VALUES = 16;         // a thread's share of a chunk
constexpr int LP_STAGES = 3;          // chunks of a block on their way or in use
constexpr int LP_CELLS = 4;           // maxima a thread keeps
constexpr int LP_QUEUE = 512;         // of the cells that can be read again
constexpr int LP_MAX_PARTS = 16;      // blocks of a row
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
// 2^v without the handling of results below 2^-126, which are zero here.
__device__ __forceinline__ float lp_ex2(float v) {
    float d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
    return d;
}
__device__ __forceinline__ float lp_exp(float v) { return lp_ex2(v * 1.4426950408889634f); }
// Two values an instruction.
__device__ __forceinline__ uint64_t lp_pair(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void lp_split(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t lp_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t lp_mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t lp_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
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

template <int THREADS>
struct __align__(16) LpShared {
    LpSums parts[LP_MAX_PARTS];  // of a cluster's first block
    LpSums sums[THREADS / 32];
    float cells[LP_CELLS][THREADS];
    uint32_t low;
    int count, queued;
};
// In the ring's place once the row has been read.
template <int THREADS>
struct __align__(16) LpTail {
    uint64_t buf[THREADS + 4];  // candidates for the largest
    uint64_t list[LOGPROBS_MAX_TOP];  // the result
    union {
        uint32_t first[THREADS];
        uint16_t queue[LP_QUEUE];
    };
};

// The largest of n keys, sorted, to list: a key's place is the number of greater ones. Every thread calls; room for four more keys.
__device__ __forceinline__ void lp_largest(uint64_t* keys, int n, uint64_t* list, int tid) {
    const uint64_t mine = tid < n ? keys[tid] : 0;
    if (tid < LOGPROBS_MAX_TOP) list[tid] = 0;
    if (tid < 4) keys[n + tid] = 0;
    __syncthreads();
    if (tid / 32 * 32 < n) {
        int rank = 0;
        const ulonglong2* const pairs = reinterpret_cast<const ulonglong2*>(keys);
        for (int i = 0; i < n; i += 4) {
            const ulonglong2 u = pairs[i / 2], v = pairs[i / 2 + 1];
            rank += (u.x > mine) + (u.y > mine) + (v.x > mine) + (v.y > mine);
        }
        if (mine && rank < LOGPROBS_MAX_TOP) list[rank] = mine;
    }
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

template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprobs_kernel(const LogprobsArgs a, int parts) {
    __shared__ LpShared<THREADS> sh;
    extern __shared__ uint4 lp_ring[];  // [stage][piece][thread]: a thread reads what it has copied, so that no barrier stands between
    constexpr int VEC = 16 / sizeof(T), PIECES = LP_VALUES / VEC, STEP = THREADS * PIECES;
    static_assert(sizeof(LpTail<THREADS>) <= STEP * sizeof(uint4) && LP_STAGES - 1 <= LP_CELLS, "the tail fits one stage, a cell a chunk of those that stay");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t r = blockIdx.x / parts;
    const int part = blockIdx.x - (int)r * parts;
    const T* const row = static_cast<const T*>(a.z) + r * a.ld;
    // pieces start on 16-byte boundaries: the first and the last may hang over the row's ends
    const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int pieces = (int)(((int64_t)skew + a.n + VEC - 1) / VEC), per = (pieces + parts - 1) / parts;
    const int begin = min(part * per, pieces), end = min(begin + per, pieces);
    uint64_t* const inbox = reinterpret_cast<uint64_t*>(lp_ring + LP_STAGES * PIECES * THREADS);  // of a cluster's first block: every part's largest
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
    // few chunks stay in the ring, whose last stage they do not use: there the largest are looked for where they are
    const bool stays = chunks < LP_STAGES;
    LpTail<THREADS>& tail = *reinterpret_cast<LpTail<THREADS>*>(lp_ring + (stays ? (LP_STAGES - 1) * STEP : 0));
    // A thread's maxima over runs of `cell` chunks stay in shared memory: where the largest values are looked for afterwards.
    const int cell = (chunks + LP_CELLS - 1) / LP_CELLS;
    int n_cells = 0, in_cell = 0;
    float peak = -INFINITY;
    auto fetch = [&](int k) {
        if (k < chunks) {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                uint4* const to = lp_ring + (k % LP_STAGES * PIECES + j) * THREADS + tid;
                const int p = begin + k * STEP + j * THREADS + tid, e0 = p * VEC - skew;
                if (p < end && e0 >= 0 && e0 + VEC <= a.n) {
                    lp_copy(to, row + e0);
                } else {  // past the part, or a piece that hangs over an end of the row: masked values in the others' places
                    constexpr uint32_t MASKED = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
                    *to = make_uint4(MASKED, MASKED, MASKED, MASKED);
                    if (p < end) {
#pragma unroll 1
                        for (int i = 0; i < VEC; ++i)
                            if (e0 + i >= 0 && e0 + i < a.n) reinterpret_cast<T*>(to)[i] = row[e0 + i];
                    }
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
        const uint4* const mine = lp_ring + k % LP_STAGES * PIECES * THREADS + tid;
        float x[LP_VALUES];
#pragma unroll
        for (int j = 0; j < PIECES; ++j) lp_unpack(mine[j * THREADS], x + j * VEC, T());
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
            uint64_t r2 = 0, t2 = 0;  // of even and odd values
            const uint64_t minus = lp_pair(-s.m, -s.m), log2e = lp_pair(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
            for (int i = 0; i < LP_VALUES; i += 2) {
                float d0, d1, e0, e1;
                lp_split(lp_add2(lp_pair(x[i], x[i + 1]), minus), d0, d1);
                const uint64_t d = lp_pair(fmaxf(d0, LP_LOW), fmaxf(d1, LP_LOW));
                lp_split(lp_mul2(d, log2e), e0, e1);
                const uint64_t e = lp_pair(lp_ex2(e0), lp_ex2(e1));
                r2 = lp_add2(r2, e);
                t2 = lp_fma2(d, e, t2);
            }
            float r0, r1, t0, t1;
            lp_split(r2, r0, r1);
            lp_split(t2, t0, t1);
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
        // a first threshold: the `top`-th largest of the maxima of 32 groups of eight threads, which that many values reach; of 64
        // where that would be about the least of them (64 rows of 128256 bf16, top 32: 41.8 us, 13.6; they cost others 0.4 us)
        float cells[LP_CELLS];
        peak = -INFINITY;
#pragma unroll
        for (int j = 0; j < LP_CELLS; ++j) {
            cells[j] = j < n_cells ? sh.cells[j][tid] : -INFINITY;
            peak = lp_max(peak, cells[j]);
        }
        tail.first[tid] = lp_mono(peak);
        __syncthreads();
        auto rank_groups = [&](uint32_t m0, uint32_t m1, int groups) {  // (each warp looks at its share of the groups)
#pragma unroll 4
            for (int i = 0; i < groups / (THREADS / 32); ++i) {
                const int c = warp * (groups / (THREADS / 32)) + i;
                const uint32_t v = __shfl_sync(LP_ALL, c < 32 ? m0 : m1, c & 31);
                int greater = __popc(__ballot_sync(LP_ALL, m0 > v || (m0 == v && lane < c)));
                if (groups > 32) greater += __popc(__ballot_sync(LP_ALL, m1 > v || (m1 == v && lane + 32 < c)));
                if (greater == a.top - 1 && lane == 0) sh.low = v;
            }
        };
        uint32_t m[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            m[h] = tail.first[h * (THREADS / 2) + lane];
#pragma unroll
            for (int w = 1; w < THREADS / 64; ++w) m[h] = max(m[h], tail.first[h * (THREADS / 2) + w * 32 + lane]);
        }
        if (a.top <= 24) rank_groups(max(m[0], m[1]), 0, 32);
        else rank_groups(m[0], m[1], 64);
        __syncthreads();  // (the maxima's place is the queue's)
        uint64_t threshold = (uint64_t)sh.low << 32;
        float low = lp_value((uint32_t)(threshold >> 32));
        // A value to the buffer, if it is a candidate: 0, there was room; 1, the buffer fills; 2, it is full.
        auto push = [&](float v, int id) {
            if (v < low || id < 0 || id >= a.n) return 0;
            const uint64_t key = lp_key(v, id);
            if (key <= threshold) return 0;
            const int at = atomicAdd(&sh.count, 1);
            if (at < THREADS) tail.buf[at] = key;
            return at < THREADS / 2 ? 0 : at < THREADS ? 1 : 2;
        };
        // the cells whose maximum is not below the threshold are read again, a piece a thread
        bool over = false;
        if (stays) {  // (a cell is a chunk)
            for (int k = 0; k < chunks; ++k) {
                if (sh.cells[k][tid] < low) continue;
                const uint4* const mine = lp_ring + k * STEP + tid;
                uint32_t reach = 0;
#pragma unroll
                for (int j = 0; j < PIECES; ++j) {
                    float v[VEC];
                    lp_unpack(mine[j * THREADS], v, T());
#pragma unroll
                    for (int i = 0; i < VEC; ++i) reach |= (uint32_t)!(v[i] < low) << (j * VEC + i);
                }
                for (; reach; reach &= reach - 1) {
                    const int at = __ffs(reach) - 1, j = at / VEC, p = begin + k * STEP + j * THREADS + tid, id = p * VEC - skew + at % VEC;
                    if (p < end) over |= push((float)reinterpret_cast<const T*>(mine + j * THREADS)[at % VEC], id) == 2;
                }
            }
            __syncthreads();
        } else {
#pragma unroll
        for (int j = 0; j < LP_CELLS; ++j)
            if (j < n_cells && !(cells[j] < low)) {
                const int at = atomicAdd(&sh.queued, 1);
                if (at < LP_QUEUE) tail.queue[at] = (uint16_t)(j * THREADS + tid);
            }
        __syncthreads();
        const int queued = sh.queued, cell_pieces = cell * PIECES, items = min(queued, LP_QUEUE) * cell_pieces;
        over = queued > LP_QUEUE;
        constexpr int AHEAD = 4;  // pieces of a thread on their way
        for (int i0 = tid; !over && i0 < items; i0 += AHEAD * THREADS) {
            // (one copy of what follows a candidate, not one for each value: it runs once, and its instructions have to be fetched)
            auto piece_of = [&](int e) {
                const int i = i0 + e * THREADS, q = i / cell_pieces, u = i - q * cell_pieces;
                if (i >= items) return end;
                const int from = tail.queue[q], k = from / THREADS * cell + u / PIECES;
                return k < chunks ? begin + k * STEP + u % PIECES * THREADS + from % THREADS : end;
            };
            uint4 got[AHEAD];
            uint32_t edge = 0, reach = 0;
#pragma unroll
            for (int e = 0; e < AHEAD; ++e) {
                const int p = piece_of(e), e0 = p * VEC - skew;
                if (p < end && e0 >= 0 && e0 + VEC <= a.n) got[e] = *reinterpret_cast<const uint4*>(row + e0);
                else edge |= (p < end) << e;
            }
#pragma unroll
            for (int e = 0; e < AHEAD; ++e) {
                float v[VEC];
                lp_unpack(got[e], v, T());
                uint32_t mask = 0;
#pragma unroll
                for (int i = 0; i < VEC; ++i) mask |= !(v[i] < low) << i;
                if (i0 + e * THREADS >= items) mask = 0;
                if (edge >> e & 1) mask = (1u << VEC) - 1;
                reach |= mask << e * VEC;
            }
            for (; reach; reach &= reach - 1) {
                const int at = __ffs(reach) - 1, p = piece_of(at / VEC), id = p * VEC - skew + at % VEC;
                if (p < end && id >= 0 && id < a.n) over |= push((float)row[id], id) == 2;
            }
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
                        const int i = __ffs(left) - 1, p = begin + k * STEP + i / VEC * THREADS + tid, id = p * VEC - skew + i % VEC;
                        const int got = p < end && id >= 0 && id < a.n ? push((float)row[id], id) : 0;
                        if (got < 2) pending &= ~(1u << i);
                        said = max(said, got);
                    }
                    if (!__syncthreads_or(said)) break;
                    lp_largest(tail.buf, min(sh.count, THREADS), tail.list, tid);
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
        s = sh.sums[lane & (THREADS / 32 - 1)];
#pragma unroll 1
        for (int o = THREADS / 64; o > 0; o >>= 1) s = lp_join(s, lp_shfl(s, o));
    }
    if (parts > 1) {
        // every block writes its part into the first one's memory, which goes on alone
        lp_cluster_wait();
        if (warp == 0) {
            if (lane == 0) {
                const uint32_t to = lp_first(&sh.parts[part]);
                asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(to), "r"(__float_as_uint(s.m)), "r"(__float_as_uint(s.r)), "r"(__float_as_uint(s.t)), "r"(s.bad) : "memory");
            }
            if (TOP && lane < a.top) asm volatile("st.shared::cluster.u64 [%0], %1;\n" ::"r"(lp_first(&inbox[part * a.top + lane])), "l"(tail.list[lane]) : "memory");
        }
        __syncwarp();
        lp_cluster_arrive();
        lp_cluster_wait();
        if (part != 0) return;
        if (warp == 0) {
            s = (lane & (LP_MAX_PARTS - 1)) < parts ? sh.parts[lane & (LP_MAX_PARTS - 1)] : LpSums{-INFINITY, 0.f, 0.f, 0};
#pragma unroll 1
            for (int o = LP_MAX_PARTS / 2; o > 0; o >>= 1) s = lp_join(s, lp_shfl(s, o));
        }
        if (TOP) lp_largest(inbox, parts * a.top, tail.list, tid);
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

template <typename T, int THREADS>
static cudaError_t logprobs_with(const LogprobsArgs& a, int parts, cudaStream_t st) {
    if (a.rows * parts > INT32_MAX) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * parts));
    cfg.blockDim = dim3(THREADS);
    constexpr size_t ring = LP_STAGES * (THREADS * LP_VALUES) * sizeof(T), most = ring + (THREADS + 4) * sizeof(uint64_t);
    cfg.dynamicSmemBytes = parts > 1 ? ring + (parts * a.top + 4) * sizeof(uint64_t) : ring;
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
        for (const auto kernel : {logprobs_kernel<T, true, THREADS>, logprobs_kernel<T, false, THREADS>}) {
            cudaError_t f = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
            if (f == cudaSuccess) f = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);  // (more than eight blocks)
            if (f != cudaSuccess) return f;
        }
        return cudaSuccess;
    });
    if (e != cudaSuccess) return e;
    e = a.top > 0 ? cudaLaunchKernelEx(&cfg, logprobs_kernel<T, true, THREADS>, a, parts) : cudaLaunchKernelEx(&cfg, logprobs_kernel<T, false, THREADS>, a, parts);
    return e != cudaSuccess ? e : count_launch_and_check();
}

template <typename T>
static cudaError_t logprobs_of(const LogprobsArgs& a, cudaStream_t st) {
    const int sms = device_sm_count();
    // up to two blocks an SM; 16 where rows are few and there are few keys to rank (8 x 128256 f32, 8 parts and 16: top 5 7.9 us, 7.7;
    // top 16 8.6 us, 10.3; 1 x 151936 top 0 5.9 us, 4.6)
    int parts = 1;
    while (parts < 8 && a.rows * parts * 2 <= 2 * sms && a.n / (parts * 2) >= 256 * LP_VALUES) parts *= 2;
    if (parts == 8 && a.rows * 16 <= sms && a.n / 16 >= 256 * LP_VALUES && a.top <= 8) parts = 16;
    // Many short rows: twice as many of half as many threads, for more of the chains that follow the reading (4000 x 1500 f32 top 5 30.3 us,
    // 18.0; 2561 x 10581 bf16 top 20 40.0, 32.8; not 894 x 28496 f32 27.2, 28.9, and a few rows 1 x 5000 4.2, 5.1).
    if (a.rows > 2 * sms && (int64_t)a.n * sizeof(T) <= 65536) return logprobs_with<T, 128>(a, 1, st);
    return logprobs_with<T, 256>(a, parts, st);
}

cudaError_t launch_logprobs(const LogprobsArgs& a, bool bf, cudaStream_t st) {
    if (a.rows == 0) return cudaSuccess;
    if (a.n < 1 || a.top < 0 || a.top > LOGPROBS_MAX_TOP || a.top > a.n) return cudaErrorInvalidValue;
    return bf ? logprobs_of<bf16>(a, st) : logprobs_of<float>(a, st);
}

}  // namespace sp
