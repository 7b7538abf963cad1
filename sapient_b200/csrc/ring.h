// A ring of stages that asynchronous copies fill by turns: which stage a step's copies go to, and the parity of its barrier's phase that they complete.
// Plain arithmetic, shared by device code and its test.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define SP_RING_FN __host__ __device__ constexpr
#else
#define SP_RING_FN constexpr
#endif

namespace sp {

struct RingAt {
    int stage;
    uint32_t parity;
};
SP_RING_FN RingAt ring_at(int step, int stages) { return RingAt{step % stages, (uint32_t)(step / stages) & 1u}; }
// One past the last step whose copies may be on their way while step i is waited for: each step requests the one `stages - 1` on before it waits.
SP_RING_FN int ring_requested(int i, int stages, int steps) { return i + stages < steps ? i + stages : steps; }

}  // namespace sp
