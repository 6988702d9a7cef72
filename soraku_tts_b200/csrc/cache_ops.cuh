// Shared pieces of the cache operators: chunk attention (chunk_attn.cu),
// windowed decode attention (window_decode.cu) and eviction (evict.cu), all
// over the paged FP32 pool [n_pages][K, V][KVH][page][128] that decode
// attention reads.
//
// A row's slots 0 .. cached-1 are filled; new tokens take the next ones.  A
// slot is where a token lies, its RoPE position is apart from it (after an
// eviction positions run ahead of slots).  The query at slot i sees slot
// j <= i if there is no window (window == 0), or i - j < window, or j < sinks.
#pragma once

#include <atomic>

#include "ops.cuh"
#include "trunk.cuh"

namespace skb {

constexpr int CO_MAX_REP = 4;  // query heads per kv head
// 32-bit units of rows that are not in the pool: none is meant (zeros), or its
// page is outside (not a number).
constexpr uint32_t UT_NONE = 0xffffffffu, UT_BAD = 0xfffffffeu;

struct CacheView {
    float* pool;
    const int* page_table;  // [rows][max_pages]
    int max_pages;
    int page_log2;
    int KVH;
    int n_pages;
    // Index in units of 128 floats of slot `slot` of (row, head g): its key;
    // the value lies KVH << page_log2 units further.  -1 for a table entry
    // that names no page of the pool.
    __device__ __forceinline__ long long key_unit(int row, int slot, int g) const {
        const int page = __ldg(page_table + (long long)row * max_pages + (slot >> page_log2));
        if ((unsigned)page >= (unsigned)n_pages) return -1;
        return ((((long long)page * 2) * KVH + g) << page_log2) + (slot & ((1 << page_log2) - 1));
    }
    __device__ __forceinline__ long long value_step() const { return (long long)KVH << page_log2; }
};

// The inputs both attention operators share.
struct CacheAttnArgs {
    const float* qkv;  // [tokens][(H + 2 KVH) * 128]
    const float* qn;   // q_norm weight [128]
    const float* kn;   // k_norm weight [128]
    float eps;
    const float* rope_cos;  // [max_pos][64]
    const float* rope_sin;
    int max_pos;
    const int* cached;  // [rows] filled slots; negative: the row is idle
    const int* pos;     // [rows] RoPE position of the row's first new token
    CacheView kv;
    int H, rows;
    int window, sinks;
    float* mass;  // [rows][KVH][max_pages << page_log2] or null
    float* out;   // [tokens][H * 128]
};

// Checks of the arguments that both attention operators take; SKB_OK or the
// status of a refusal.
int cache_attn_check(const char* what, const void* qkv, int rows, int H, int KVH, int hd, const void* qn,
                     const void* kn, const void* rc, const void* rs, int max_pos, const void* cached, const void* pos,
                     const void* kv_pool, const void* page_table, int max_pages, int page_size, int n_pages,
                     int window, int sinks, const void* out);

inline int log2_of(int v) {
    int lg = 0;
    while ((1 << lg) < v) ++lg;
    return lg;
}

// set_smem_attrs once per kernel and device: the call costs as much as a third
// of a launch.  Like every address cached per device, what it set is gone after
// cudaDeviceReset.
template <typename K>
inline cudaError_t smem_attrs_once(K* kernel, size_t bytes, std::atomic<unsigned long long>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = set_smem_attrs(kernel, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// exp2 in one instruction (relative error 2^-22); the argument of a softmax
// weight is at most a few units above 0.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A score below every real one: softmax statistics start from it instead of
// -inf, so that -inf - -inf never arises.
constexpr float CO_LOW = -3e38f;
constexpr float CO_LOG2E = 1.4426950408889634f;

}  // namespace skb
