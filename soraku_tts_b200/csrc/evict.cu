// Eviction from the paged cache by accumulated attention weight.  Of a row
// with more than `budget` filled slots each kv head keeps the first `sinks`,
// the last `recent`, and of the slots between them the heaviest (equal
// weights: the lower slot), in slot order; keys, values and weights move
// together to the front.  Keys keep the RoPE rotation of the position
// they were written with.
//
// Two launches:
//   evict_select  one CTA per (row, kv head): the weight at the border by a
//                 radix search over order-preserving integer keys (8 bits a
//                 pass), then a scan that writes the kept slots and weights;
//   evict_move    the copy, in place.  A kept slot never moves up, so a CTA
//                 that goes through the kept slots in order reads each round
//                 before it writes it and never overwrites what it still has
//                 to read.  Columns are independent, so the 512-byte rows are
//                 cut into parts of 128 bytes that separate CTAs move: 8 CTAs
//                 per (row, kv head), enough loads in flight without any
//                 order between CTAs.
// Bound by memory: each kept slot that moves is 1 KB in and 1 KB out.
#include "cache_ops.cuh"

namespace skb {

constexpr int EV_THREADS = 1024;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_MOVE_THREADS = 256;
constexpr int EV_PARTS = 4;                                   // 128-byte column parts of a row
constexpr int EV_LANES = 32 / EV_PARTS;                       // 16-byte words of a part
constexpr int EV_ROWS = EV_MOVE_THREADS / EV_LANES;           // rows side by side
constexpr int EV_UNROLL = 8;                                  // rows per thread and round

struct EvictArgs {
    const float* mass;  // [rows][KVH][slots]
    const int* cached;  // [rows]
    CacheView kv;
    int rows, slots, budget, sinks, recent;
    int* kept;         // [rows][KVH][budget]
    float* mass_out;   // [rows][KVH][slots]
    int* cached_out;   // [rows]
    int* first_moved;  // [rows][KVH]: kept slots before it stay where they are; -1: nothing moves
};

// Filled slots of a row: the count, with numbers outside the cache taken as none.
__device__ __forceinline__ int evict_filled(const EvictArgs& a, int r) {
    const int c = a.cached[r];
    return c < 0 || c > a.slots ? 0 : c;
}

// Unsigned keys in the order of the floats; NaN of either sign above all.
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);  // -0 ranks with +0
    if (x != x) return 0xffffffffu;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const EvictArgs a) {
    __shared__ int hist[256];
    __shared__ int wcount[EV_WARPS][2];
    __shared__ unsigned border;
    __shared__ int left;
    __shared__ int first;
    const int g = blockIdx.x, r = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long rg = (long long)r * a.kv.KVH + g;
    const float* mass = a.mass + rg * a.slots;
    float* mass_out = a.mass_out + rg * a.slots;
    int* kept = a.kept + rg * a.budget;
    const int n = evict_filled(a, r);
    const int keep = min(n, a.budget);
    if (g == 0 && tid == 0) a.cached_out[r] = a.cached[r] < 0 || a.cached[r] > a.slots ? a.cached[r] : keep;
    for (int i = keep + tid; i < a.slots; i += EV_THREADS) mass_out[i] = 0.f;
    for (int i = keep + tid; i < a.budget; i += EV_THREADS) kept[i] = -1;
    if (n <= a.budget) {
        for (int i = tid; i < n; i += EV_THREADS) {
            kept[i] = i;
            mass_out[i] = mass[i];
        }
        if (tid == 0) a.first_moved[rg] = -1;
        return;
    }
    // candidates [lo, hi); `want` of them stay
    const int lo = a.sinks, hi = n - a.recent;
    const int want = a.budget - a.sinks - a.recent;
    unsigned prefix = 0;
    int need = want;  // of the candidates that share `prefix`, how many stay
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
            for (int i0 = lo; i0 < hi; i0 += EV_THREADS) {
                const int i = i0 + tid;
                const unsigned k = i < hi ? order_key(mass[i]) : 0u;
                const bool in = i < hi && (k & mask) == prefix;
                // one addition per distinct bin of the warp: weights crowd into few bins
                const unsigned bin = in ? (k >> shift) & 255u : 256u;
                const unsigned peers = __match_any_sync(FULL, bin);
                if (in && lane == __ffs(peers) - 1) atomicAdd(&hist[bin], __popc(peers));
            }
            __syncthreads();
            if (warp == 0) {
                // bins from the top: lane l holds bins 255 - 8 l .. 248 - 8 l
                int c[8], sum = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    c[j] = hist[255 - 8 * lane - j];
                    sum += c[j];
                }
                int before = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(FULL, before, o);
                    if (lane >= o) before += v;
                }
                before -= sum;
                if (before < need && before + sum >= need) {
                    int acc = before;
                    for (int j = 0; j < 8; ++j) {
                        if (acc + c[j] >= need) {
                            border = prefix | ((unsigned)(255 - 8 * lane - j) << shift);
                            left = need - acc;
                            break;
                        }
                        acc += c[j];
                    }
                }
            }
            __syncthreads();
            prefix = border;
            need = left;
        }
    } else {
        prefix = 0xffffffffu;  // nothing lies above it
        need = 0;
    }
    // ---- scan: kept are the sinks, the recent ones, candidates above the
    // border, and the first `need` that equal it.  Warp w takes the w-th
    // stretch of slots, so positions need one exchange between warps.
    if (tid == 0) first = a.slots;
    const int per = ((n + EV_WARPS - 1) / EV_WARPS + 31) & ~31;
    const int b = min(n, warp * per), e = min(n, b + per);
    int n_sure = 0, n_tie = 0;
    for (int i0 = b; i0 < e; i0 += 32) {
        const int i = i0 + lane;
        const bool here = i < e, mid = here && i >= lo && i < hi;
        const unsigned k = mid ? order_key(mass[i]) : 0u;
        n_sure += __popc(__ballot_sync(FULL, here && (!mid || k > prefix)));
        n_tie += __popc(__ballot_sync(FULL, mid && k == prefix));
    }
    if (lane == 0) {
        wcount[warp][0] = n_sure;
        wcount[warp][1] = n_tie;
    }
    __syncthreads();
    int sure = 0, tie = 0;
    for (int x = 0; x < warp; ++x) {
        sure += wcount[x][0];
        tie += wcount[x][1];
    }
    int my_first = a.slots;
    const unsigned below = (1u << lane) - 1u;
    for (int i0 = b; i0 < e; i0 += 32) {
        const int i = i0 + lane;
        const bool here = i < e, mid = here && i >= lo && i < hi;
        const float x = here ? mass[i] : 0.f;
        const unsigned k = mid ? order_key(x) : 0u;
        const bool is_sure = here && (!mid || k > prefix), is_tie = mid && k == prefix;
        const unsigned bs = __ballot_sync(FULL, is_sure), bt = __ballot_sync(FULL, is_tie);
        const int t = tie + __popc(bt & below);  // equal ones before this slot
        const int at = sure + __popc(bs & below) + min(t, need);
        if (is_sure || (is_tie && t < need)) {
            kept[at] = i;
            mass_out[at] = x;
            if (at != i) my_first = min(my_first, at);
        }
        sure += __popc(bs);
        tie += __popc(bt);
    }
    if (my_first < a.slots) atomicMin(&first, my_first);
    __syncthreads();
    if (tid == 0) a.first_moved[rg] = first < a.slots ? first : -1;
}

__global__ void __launch_bounds__(EV_MOVE_THREADS) evict_move_kernel(const EvictArgs a) {
    const int part = blockIdx.x % EV_PARTS, value = blockIdx.x / EV_PARTS, g = blockIdx.y, r = blockIdx.z;
    const long long rg = (long long)r * a.kv.KVH + g;
    const int from = a.first_moved[rg];
    if (from < 0) return;
    const int* kept = a.kept + rg * a.budget;
    const int tr = threadIdx.x / EV_LANES, tc = threadIdx.x % EV_LANES;
    float4* pool4 = reinterpret_cast<float4*>(a.kv.pool);
    const long long off = (value ? a.kv.value_step() * 32 : 0) + part * EV_LANES + tc;
    constexpr int ROUND = EV_ROWS * EV_UNROLL;
    for (int i0 = from; i0 < a.budget; i0 += ROUND) {
        float4 x[EV_UNROLL];
        bool ok[EV_UNROLL];
#pragma unroll
        for (int j = 0; j < EV_UNROLL; ++j) {
            const int i = i0 + j * EV_ROWS + tr;
            ok[j] = false;
            if (i < a.budget) {
                const long long u = a.kv.key_unit(r, kept[i], g);
                ok[j] = u >= 0;
                if (ok[j]) x[j] = __ldcg(pool4 + u * 32 + off);
            }
        }
        __syncthreads();  // the round is read before any of it is written
#pragma unroll
        for (int j = 0; j < EV_UNROLL; ++j) {
            const int i = i0 + j * EV_ROWS + tr;
            if (ok[j]) {
                const long long u = a.kv.key_unit(r, i, g);
                if (u >= 0) pool4[u * 32 + off] = x[j];
            }
        }
    }
}

}  // namespace skb

using namespace skb;

extern "C" int64_t skb_evict_workspace(int rows, int n_kv_heads) {
    return rows < 0 || n_kv_heads < 1 ? -1 : (int64_t)rows * n_kv_heads * 4;
}

extern "C" int skb_evict_cache(const float* mass, const int32_t* cached, int rows, int n_kv_heads, int head_dim,
                               float* kv_pool, const int32_t* page_table, int max_pages, int page_size, int n_pages,
                               int budget, int sinks, int recent, int32_t* kept, float* mass_out,
                               int32_t* cached_out, void* work, int64_t work_bytes, cudaStream_t stream) {
    if (!mass || !cached || !kv_pool || !page_table || !kept || !mass_out || !cached_out)
        return fail(SKB_ERR_ARG, "evict_cache: null pointer");
    if (head_dim != 128 || rows < 0 || rows > 65535 || n_kv_heads < 1 || n_kv_heads > 65535 || max_pages < 1 ||
        n_pages < 1)
        return fail(SKB_ERR_ARG, "evict_cache: bad sizes (head_dim must be 128)");
    if (page_size < 1 || (page_size & (page_size - 1)) != 0 || (long long)max_pages * page_size > (1ll << 30))
        return fail(SKB_ERR_ARG, "evict_cache: page_size must be a power of two, and a row at most 2^30 slots");
    if (budget < 1 || sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
        return fail(SKB_ERR_ARG, "evict_cache: budget must be at least 1 and hold the sinks and the recent slots");
    if (mass_out == mass || cached_out == cached)
        return fail(SKB_ERR_ARG, "evict_cache: the new weights and counts need memory of their own");
    if ((uintptr_t)kv_pool & 15u) return fail(SKB_ERR_ARG, "evict_cache: kv_pool must be 16-byte aligned");
    if (!work || work_bytes < skb_evict_workspace(rows, n_kv_heads))
        return fail(SKB_ERR_ARG, "evict_cache: needs a workspace of skb_evict_workspace bytes");
    if (rows == 0) return SKB_OK;
    EvictArgs a = {};
    a.mass = mass;
    a.cached = cached;
    a.kv = {kv_pool, page_table, max_pages, log2_of(page_size), n_kv_heads, n_pages};
    a.rows = rows;
    a.slots = max_pages * page_size;
    a.budget = budget;
    a.sinks = sinks;
    a.recent = recent;
    a.kept = kept;
    a.mass_out = mass_out;
    a.cached_out = cached_out;
    a.first_moved = static_cast<int*>(work);
    cudaError_t e = launch(evict_select_kernel, dim3(n_kv_heads, rows), dim3(EV_THREADS), 0, stream, false, a);
    if (e == cudaSuccess && budget < a.slots)
        e = launch(evict_move_kernel, dim3(2 * EV_PARTS, n_kv_heads, rows), dim3(EV_MOVE_THREADS), 0, stream, false, a);
    return e == cudaSuccess ? SKB_OK : fail(SKB_ERR_CUDA, "evict_cache: %s", cudaGetErrorString(e));
}
