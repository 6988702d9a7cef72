// Eviction from the paged cache by accumulated attention weight.  Of a row
// with more than `budget` filled slots each kv head keeps the first `sinks`,
// the last `recent`, and of the slots between them the heaviest (equal
// weights: the lower slot), in slot order; keys, values and weights move
// together to the front.  Keys keep the RoPE rotation of the position
// they were written with.
//
// One launch, a thread-block cluster of 8 (or 2) CTAs per (row, kv head):
//   select  the weight at the border by a radix search over order-preserving
//           integer keys (8 bits a pass), then a scan that writes the kept slots
//           and weights.  Up to EV_LOCAL slots every CTA does all of it for
//           itself, the keys in registers: no CTA waits for another.  Beyond,
//           each counts its share, and the counts are added through distributed
//           shared memory, which costs two cluster barriers a pass.
//   move    the copy, in place.  A kept slot never moves up, so a CTA that goes
//           through the kept slots in order reads a round before it writes it
//           and never overwrites what it still has to read.  Columns are
//           independent, so the 512-byte rows may be cut into parts of 128
//           bytes: the cluster's CTAs move keys or values, a part each,
//           without any order between them.  Where rows come from and go to is looked up
//           for EV_BLOCK rows at once, so that a round waits for its data alone,
//           and two rounds are on their way at a time.
// Each kept slot that moves is 1 KB in and 1 KB out.  128 groups of 5k to 8k slots
// to 2k take 121 us, 69 % of a plain copy's rate; with weights that keep the
// first slots, so that only the 256 recent ones move, 34.  So about a quarter is
// the search, which all groups do at the same time while memory is idle, and the move
// runs near a copy's rate (a longer ring in shared memory, with fewer CTAs an
// SM, took 122 us, and 142 instead of 120 at 32k slots).
#include "cache_ops.cuh"

namespace skb {

constexpr int EV_THREADS = 512;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_UNROLL = 4;     // rows per thread and round
constexpr int EV_KEYS = 16;      // keys a thread can hold
constexpr int EV_LOCAL = 2048;   // slots up to which every CTA searches for itself

// CTAS per (row, kv head): rows are moved in CTAS / 2 parts.
template <int CTAS>
struct EvictShape {
    static constexpr int PARTS = CTAS / 2;
    static constexpr int LANES = 32 / PARTS;            // 16-byte words of a part
    static constexpr int ROWS = EV_THREADS / LANES;     // rows side by side
    static constexpr int ROUND = ROWS * EV_UNROLL;
};
constexpr int EV_BLOCK = 2048;   // rows whose places are looked up at once
static_assert(EV_BLOCK % (2 * EvictShape<8>::ROUND) == 0 && EV_BLOCK % (2 * EvictShape<2>::ROUND) == 0, "whole rounds");

struct EvictArgs {
    const float* mass;  // [rows][KVH][slots]
    const int* cached;  // [rows]
    CacheView kv;
    int rows, slots, budget, sinks, recent;
    int* kept;        // [rows][KVH][budget]
    float* mass_out;  // [rows][KVH][slots]
    int* cached_out;  // [rows]
};

struct EvictSmem {
    int hist[2][256];   // this CTA's counts, read by the cluster; passes alternate
    int total[256];
    int sure, tie;      // this CTA's kept for certain, and equal to the border
    int first;          // its first kept slot that moves
    int wcount[EV_WARPS][2];
    unsigned border;
    int left;
    uint32_t src[EV_BLOCK], dst[EV_BLOCK];  // units in the pool; src UT_NONE: nothing to move, UT_BAD: no page
};

// Unsigned keys in the order of the floats; NaN of either sign above all.
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);  // -0 ranks with +0
    if (x != x) return 0xffffffffu;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ int ld_peer_int(const int* p, uint32_t rank) {
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(p)), "r"(rank));
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(ra) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// What the scan and the search ask of a warp's stretch of slots [wb, we), 32 at
// a time: the key of slot i if it is a candidate.  HELD: in registers.
template <bool HELD>
struct Stretch {
    const float* mass;
    int wb, we, lo, hi, lane;
    unsigned key[HELD ? EV_KEYS : 1];
    __device__ __forceinline__ bool mid(int i) const { return i < we && i >= lo && i < hi; }
    __device__ __forceinline__ void load() {
        if constexpr (HELD) {
#pragma unroll
            for (int j = 0; j < EV_KEYS; ++j) {
                const int i = wb + 32 * j + lane;
                key[j] = mid(i) ? order_key(mass[i]) : 0u;
            }
        }
    }
    // f(slot, candidate, its key), by whole warps
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        if constexpr (HELD) {
#pragma unroll
            for (int j = 0; j < EV_KEYS; ++j) {
                const int i = wb + 32 * j + lane;
                if (wb + 32 * j < we) f(i, mid(i), key[j]);
            }
        } else {
            for (int i0 = wb; i0 < we; i0 += 32 * 8) {
                unsigned k[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = i0 + 32 * j + lane;
                    k[j] = mid(i) ? order_key(mass[i]) : 0u;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = i0 + 32 * j + lane;
                    if (i0 + 32 * j < we) f(i, mid(i), k[j]);
                }
            }
        }
    }
};

// Writes the kept slots and their weights; returns the first that moves.
// `part` of `parts` CTAs go through an equal share of the slots each.
template <bool HELD, int CTAS>
__device__ int evict_select(const EvictArgs& a, EvictSmem& sm, const float* mass, int* kept, float* mass_out, int n, int part,
                            int parts) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = ((n + parts * EV_WARPS - 1) / (parts * EV_WARPS) + 31) & ~31;
    Stretch<HELD> t;
    t.mass = mass;
    t.wb = min(n, (part * EV_WARPS + warp) * per);
    t.we = min(n, t.wb + per);
    t.lo = a.sinks;  // candidates [lo, hi); `want` of them stay
    t.hi = n - a.recent;
    t.lane = lane;
    t.load();
    const int want = a.budget - a.sinks - a.recent;
    unsigned prefix = 0xffffffffu;  // the border: nothing lies above this one
    int need = 0;                   // of the candidates at the border, how many stay
    if (want > 0) {
        prefix = 0;
        need = want;
        for (int pass = 0; pass < 4; ++pass) {
            const int shift = 24 - 8 * pass, b = pass & 1;
            if (tid < 256) sm.hist[b][tid] = 0;
            __syncthreads();
            const unsigned mask = pass == 0 ? 0u : ~0u << (shift + 8);
            t.each([&](int, bool mid, unsigned k) {
                const bool in = mid && (k & mask) == prefix;
                // one addition per distinct bin of the warp: weights crowd into few bins
                const unsigned bin = in ? (k >> shift) & 255u : 256u;
                const unsigned peers = __match_any_sync(FULL, bin);
                if (in && lane == __ffs(peers) - 1) atomicAdd(&sm.hist[b][bin], __popc(peers));
            });
            const int* total = sm.hist[b];
            if (parts > 1) {
                cluster_sync_all();
                if (tid < 256) {
                    int c = 0;
#pragma unroll
                    for (int p = 0; p < CTAS; ++p) c += ld_peer_int(&sm.hist[b][tid], p);
                    sm.total[tid] = c;
                }
                total = sm.total;
            }
            __syncthreads();
            if (warp == 0) {
                // bins from the top: lane l holds bins 255 - 8 l .. 248 - 8 l
                int c[8], sum = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    c[j] = total[255 - 8 * lane - j];
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
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (acc < need && acc + c[j] >= need) {
                            sm.border = prefix | ((unsigned)(255 - 8 * lane - j) << shift);
                            sm.left = need - acc;
                        }
                        acc += c[j];
                    }
                }
            }
            __syncthreads();
            prefix = sm.border;
            need = sm.left;
        }
    }
    // ---- scan: kept are the sinks, the recent ones, candidates above the
    // border, and the first `need` that equal it
    int n_sure = 0, n_tie = 0;
    t.each([&](int i, bool mid, unsigned k) {
        n_sure += __popc(__ballot_sync(FULL, i < t.we && (!mid || k > prefix)));
        n_tie += __popc(__ballot_sync(FULL, mid && k == prefix));
    });
    if (lane == 0) {
        sm.wcount[warp][0] = n_sure;
        sm.wcount[warp][1] = n_tie;
    }
    if (tid == 0) sm.first = a.budget;
    __syncthreads();
    int sure = 0, tie = 0;  // before this warp
    for (int w = 0; w < warp; ++w) {
        sure += sm.wcount[w][0];
        tie += sm.wcount[w][1];
    }
    if (parts > 1) {
        if (tid == EV_THREADS - 1) {  // the CTA's own
            sm.sure = sure + n_sure;
            sm.tie = tie + n_tie;
        }
        cluster_sync_all();
        for (int p = 0; p < part; ++p) {
            sure += ld_peer_int(&sm.sure, p);
            tie += ld_peer_int(&sm.tie, p);
        }
    }
    int my_first = a.budget;
    const unsigned below = (1u << lane) - 1u;
    t.each([&](int i, bool mid, unsigned k) {
        const bool is_sure = i < t.we && (!mid || k > prefix), is_tie = mid && k == prefix;
        const unsigned bs = __ballot_sync(FULL, is_sure), bt = __ballot_sync(FULL, is_tie);
        const int before = tie + __popc(bt & below);  // equal ones before this slot
        // kept before it: the certain ones, and of the equal ones the first `need`
        const int at = sure + __popc(bs & below) + min(before, need);
        if (is_sure || (is_tie && before < need)) {
            kept[at] = i;
            mass_out[at] = mass[i];
            if (at != i) my_first = min(my_first, at);
        }
        sure += __popc(bs);
        tie += __popc(bt);
    });
    my_first = __reduce_min_sync(FULL, my_first);
    if (lane == 0 && my_first < a.budget) atomicMin(&sm.first, my_first);
    if (parts > 1) cluster_sync_all();
    else __syncthreads();  // every kept slot is written
    int from = sm.first;
    if (parts > 1)
        for (int p = 0; p < CTAS; ++p) from = min(from, ld_peer_int(&sm.first, p));
    return from;
}

template <int CTAS>
__global__ void __launch_bounds__(EV_THREADS, 2) evict_kernel(const EvictArgs a) {
    using Shape = EvictShape<CTAS>;
    __shared__ EvictSmem sm;
    const int s = blockIdx.x, g = blockIdx.y, r = blockIdx.z, tid = threadIdx.x;
    const long long rg = (long long)r * a.kv.KVH + g;
    const float* mass = a.mass + rg * a.slots;
    float* mass_out = a.mass_out + rg * a.slots;
    int* kept = a.kept + rg * a.budget;
    const int count = a.cached[r];
    const int n = count < 0 || count > a.slots ? 0 : count;  // numbers outside the cache: nothing filled
    const int keep = min(n, a.budget);
    if (s == 0 && g == 0 && tid == 0) a.cached_out[r] = n == count ? keep : count;
    const int ct = s * EV_THREADS + tid;  // thread of the cluster
    for (int i = keep + ct; i < a.slots; i += CTAS * EV_THREADS) mass_out[i] = 0.f;
    for (int i = keep + ct; i < a.budget; i += CTAS * EV_THREADS) kept[i] = -1;
    if (n <= a.budget) {  // the whole cluster leaves
        for (int i = ct; i < n; i += CTAS * EV_THREADS) {
            kept[i] = i;
            mass_out[i] = mass[i];
        }
        return;
    }
    const bool local = n <= EV_LOCAL;
    int from;
    if (local) from = evict_select<true, CTAS>(a, sm, mass, kept, mass_out, n, 0, 1);  // all CTAs write the same
    else if (n <= CTAS * EV_KEYS * EV_THREADS) from = evict_select<true, CTAS>(a, sm, mass, kept, mass_out, n, s, CTAS);
    else from = evict_select<false, CTAS>(a, sm, mass, kept, mass_out, n, s, CTAS);

    // ---- move: this CTA's part of keys or values
    const int tr = tid / Shape::LANES;
    float4* pool4 = reinterpret_cast<float4*>(a.kv.pool) + (s >= Shape::PARTS ? a.kv.value_step() * 32 : 0) +
                    (s % Shape::PARTS) * Shape::LANES + tid % Shape::LANES;
    for (int b0 = from; b0 < a.budget; b0 += EV_BLOCK) {
        const int m = min(EV_BLOCK, a.budget - b0);
        __syncthreads();  // the last block's places are read
        for (int i = tid; i < EV_BLOCK; i += EV_THREADS) {
            long long u = -1, d = -1;
            if (i < m) {
                u = a.kv.key_unit(r, __ldcg(kept + b0 + i), g);
                d = a.kv.key_unit(r, b0 + i, g);
            }
            // a kept slot without a page: its new place must not go on holding another's row
            sm.src[i] = d < 0 ? UT_NONE : u < 0 ? UT_BAD : (uint32_t)u;
            sm.dst[i] = (uint32_t)d;
        }
        __syncthreads();
        auto fetch = [&](float4 (&x)[EV_UNROLL], int i0) {
#pragma unroll
            for (int j = 0; j < EV_UNROLL; ++j) {
                const uint32_t u = sm.src[i0 + j * Shape::ROWS + tr];
                if (u < UT_BAD) x[j] = __ldcg(pool4 + (long long)u * 32);
                else x[j].x = x[j].y = x[j].z = x[j].w = __int_as_float(0x7fffffff);
            }
        };
        auto store = [&](const float4 (&x)[EV_UNROLL], int i0) {
#pragma unroll
            for (int j = 0; j < EV_UNROLL; ++j) {
                const int i = i0 + j * Shape::ROWS + tr;
                if (sm.src[i] != UT_NONE) pool4[(long long)sm.dst[i] * 32] = x[j];
            }
        };
        // Rounds k and k + 1 are read before round k is written, and round k
        // lies below every slot that later rounds read.
        float4 d0[EV_UNROLL], d1[EV_UNROLL];
        fetch(d0, 0);
        for (int i0 = 0; i0 < m; i0 += 2 * Shape::ROUND) {
            fetch(d1, i0 + Shape::ROUND);
            __syncthreads();
            store(d0, i0);
            if (i0 + 2 * Shape::ROUND < EV_BLOCK) fetch(d0, i0 + 2 * Shape::ROUND);
            __syncthreads();
            store(d1, i0 + Shape::ROUND);
        }
    }
    if (!local) cluster_sync_all();  // peers have read this CTA's shared memory
}

}  // namespace skb

using namespace skb;

extern "C" int skb_evict_cache(const float* mass, const int32_t* cached, int rows, int n_kv_heads, int head_dim,
                               float* kv_pool, const int32_t* page_table, int max_pages, int page_size, int n_pages,
                               int budget, int sinks, int recent, int32_t* kept, float* mass_out,
                               int32_t* cached_out, cudaStream_t stream) {
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
    if ((long long)n_pages * 2 * n_kv_heads * page_size >= 0xfffffffell)
        return fail(SKB_ERR_ARG, "evict_cache: the pool must hold fewer than 2^32 - 2 key and value rows");
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
    // 8 CTAs a group while all of them fit the card at once (two on each of
    // 148 SMs); more groups take whole rows.  Measured, us a call in eights, fours
    // (no variant here) and twos, rows of up to 8k slots to 2k: 32 groups 41, 43, 57;
    // 40 groups 71, 51, 61; 64 groups 86, 68, 72; 96 groups 124, 106, 100; 128 groups
    // 161, 129, 121; rows of up to 842 slots to 512: 40 groups 27, 20, 18.  40 and 64
    // groups of 20k slots to 5k: 133, 105, 154 and 157, 147, 174: there eights would
    // be the better of the two that there are.
    const int ctas = (long long)rows * n_kv_heads * 8 <= 296 ? 8 : 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, n_kv_heads, rows);
    cfg.blockDim = dim3(EV_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, ctas == 8 ? evict_kernel<8> : evict_kernel<2>, a);
    return e == cudaSuccess ? SKB_OK : fail(SKB_ERR_CUDA, "evict_cache: %s", cudaGetErrorString(e));
}
