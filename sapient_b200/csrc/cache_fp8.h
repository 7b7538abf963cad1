// Launch wrappers of the operators around a paged cache of 8-bit rows (cache_fp8.cu, attention_fp8.cu). All pointers are device
// pointers; every launcher enqueues on `st`.
//
// The cache: pages of 16 tokens, values[page][key | value][kv head][token][head_dim] in e4m3, scales[page][key | value][kv head][token]
// in f32. A token's head is an fp8 row (fp8.h) of head_dim <= 128 columns: one scale. page_table[slot][i] is the page of a slot's tokens
// 16 i .. 16 i + 15; one that is not a page's number is not followed.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "sp_common.cuh"

namespace sp {

constexpr int CACHE_MAX_DIM = 128;

struct CacheFp8 {
    uint8_t* values;
    float* scales;
    const int32_t* page_table;
    int n_pages, n_slots, max_pages, n_kv, dim;
    // of (page, keys or values, head, first token): the scale's index, which times dim is the values'
    __host__ __device__ __forceinline__ int64_t row(int page, int which, int head) const { return ((int64_t)(2 * (int64_t)page + which) * n_kv + head) * KV_PAGE; }
    // The page of a slot's token, or -1.
    __device__ __forceinline__ int page_of(int slot, int pos) const {
        const int page = page_table[(int64_t)slot * max_pages + pos / KV_PAGE];
        return page >= 0 && page < n_pages ? page : -1;
    }
    __device__ __forceinline__ bool has(int slot, int pos) const { return slot >= 0 && slot < n_slots && pos >= 0 && pos / KV_PAGE < max_pages; }
};

struct CacheAppendArgs {
    CacheFp8 c;
    const int32_t *slots, *positions;
    int64_t n_tok;
    const void *q, *k, *v;  // q null: keys and values alone
    void* q_out;            // may be q
    int64_t ldq, ldk, ldv, ldqo;
    int n_heads;
    const float *q_w, *k_w;  // null: those heads are not normed
    float eps;
    const float2* angles;    // [n_angles][rotary / 2]
    int64_t n_angles;
    int rotary;
    bool pairs;              // neighbours are rotated together; else coordinates rotary / 2 apart
};
cudaError_t launch_cache_append(const CacheAppendArgs& a, bool bf, cudaStream_t st);

struct CacheReadArgs {
    CacheFp8 c;
    const int32_t *slots, *positions;
    int64_t n_tok;
    void *k, *v;  // either may be null
    int64_t ldk, ldv;
};
cudaError_t launch_cache_read(const CacheReadArgs& a, bool bf, cudaStream_t st);

// Rows row_start[i] .. row_start[i + 1] - 1 are the newest of sequence i, whose tokens with them are seq_len[i]: the last row sees them all,
// each row before it one less. They lie in slot seq_slot[i] (null: i).
struct AttentionFp8Args {
    CacheFp8 c;
    const void* q;
    void* out;
    int64_t ldq, ldo;
    int n_heads, n_seqs;
    const int32_t *seq_slot, *row_start, *seq_len;
    int max_rows, max_len;  // of any sequence; max_len only decides how the work is shared out
    float scale;
    int window;             // 0: none; else a row sees its newest `window` tokens
    int* waits;             // WaitFlags of the launch's owner
};
cudaError_t launch_attention_fp8(const AttentionFp8Args& a, bool bf, cudaStream_t st);

}  // namespace sp
