// Drawing a token from each row of logits by a given uniform number, after
// temperature, top-k, top-p and min-p.
//
// Definition, in the order (logit descending, index ascending) with weights
// e_j = exp((l_j - max) / T): the first k stay; of those the shortest prefix
// whose mass is at least p times theirs; of those the ones with e_j >= min_p.
// Every filter keeps a prefix, so the kept mass S is the least of three prefix
// masses, and the token is the first whose running sum passes u S.  Each of
// these is one question: where does a running sum (of ones, or of weights)
// along the order reach a target?
//
// It is answered without sorting.  Weights are whole multiples of 2^-44 from a
// 64-bit exponential, so sums are exact in any order and a draw does not depend
// on the order of atomics; what weighs less than 2^-45 of the largest weighs
// nothing, and all of it together (2^18 logits at most) is less than the last
// step 2^-24 of a uniform number.  A cluster of CTAs holds the row in shared
// memory, read once.  One pass counts and weighs the logits in 2048 bins along
// the order; the bin where a sum reaches its target is then gathered in one CTA,
// which adds up, for each of its few logits, what stands before it.  A bin too
// full for that is binned again by (logit, index), as often as it takes.
#include <cooperative_groups.h>

#include "int8_ops.cuh"

namespace skb {
namespace cg = cooperative_groups;

constexpr int ST_THREADS = 512, ST_WARPS = ST_THREADS / 32;
constexpr int ST_BINS = 2048;
constexpr int ST_LIST = 512;        // logits of one gathered bin
constexpr int ST_QUICK_K = 128;     // top-k up to here: the first k and their bin are gathered at once
constexpr int ST_MAX_V = 1 << 18;
constexpr double ST_ONE = 17592186044416.0;  // 2^44: the largest logit's weight

typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    long long ld;
    int rows, V, slice;  // slice: logits of one CTA
    const float* uniform;
    const float *temperature, *top_p, *min_p;  // of each row, or null: the numbers below
    const int* top_k;
    float temperature0, top_p0, min_p0;
    int top_k0;
    int64_t* tokens;
    float* logprob;
};

// Where a running sum reached its target.
struct Found {
    u64 mass;  // of the prefix that ends here
    float logit;
    int index;
};
struct Bin {
    u64 mass_before, mass;
    unsigned count_before, count;
    int bin;
};

struct SampleShared {
    float top, low;            // this CTA's
    u64 mass, mass_min_p;      // this CTA's totals
    unsigned count;
    u64 lo, hi;                // smallest and largest key of a bin, this CTA's
    Bin bin;                   // written by the CTA that found it, to all
    Found found;
    unsigned listed;           // the first CTA's: logits gathered
    u64 warp_mass[ST_WARPS];
    unsigned warp_count[ST_WARPS];
    u64 prefix[3];
    u64 key[ST_LIST], weight[ST_LIST];
};

// (logit descending, index ascending) as ascending whole numbers.
__device__ __forceinline__ u64 st_key(float l, int index) {
    const unsigned u = __float_as_uint(l + 0.0f);  // -0 is 0
    const unsigned up = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
    return (u64)(~up) << 18 | (u64)index;
}
__device__ __forceinline__ float st_logit(u64 key) {
    const unsigned up = ~(unsigned)(key >> 18);
    return __uint_as_float(up ^ ((up >> 31) ? 0x80000000u : 0xffffffffu));
}

template <class TX>
struct Row {
    const TX* data;  // this CTA's slice in shared memory
    int n, first;    // logits, and the first one's index
    float top, cut, inv_width;
    double inv_t;
    // how far below the largest; beyond `cut`: without weight
    __device__ __forceinline__ float gap(float l) const { return l == top ? 0.f : top - l; }
    __device__ __forceinline__ bool counts(float l) const { return gap(l) <= cut && l > -INFINITY; }
    __device__ __forceinline__ int bin(float l) const { return min((int)fminf(gap(l) * inv_width, 3e4f), ST_BINS - 1); }
    __device__ __forceinline__ double score(float l) const { return l == top ? 0.0 : ((double)l - (double)top) * inv_t; }
    __device__ __forceinline__ double e(float l) const { return exp(score(l)); }
    __device__ __forceinline__ static u64 mass(double e) { return __double2ull_rn(e * ST_ONE); }
};

template <class TX, int C>
struct Sampler {
    SampleShared& sm;
    unsigned *count, *low, *high;  // bins of this CTA's logits: number, and mass in two words
    unsigned* pre_count;           // of this CTA's share of the bins, cluster-wide: what stands before each
    u64* pre_mass;
    const Row<TX>& row;
    cg::cluster_group cl;
    int tid, rank;
    u64 all_mass;
    unsigned all_count;
    bool fresh;  // the bins hold the whole row

    template <class T>
    __device__ __forceinline__ T* at(T* p, int r) { return C == 1 ? p : cl.map_shared_rank(p, r); }
    __device__ __forceinline__ void sync() {
        if (C == 1) __syncthreads();
        else cl.sync();
    }

    __device__ __forceinline__ void add(int b, u64 m) {
        atomicAdd(&count[b], 1u);
        if (m == 0) return;
        const unsigned lo = (unsigned)m, old = atomicAdd(&low[b], lo);
        const unsigned hi = (unsigned)(m >> 32) + (old + lo < old ? 1u : 0u);
        if (hi) atomicAdd(&high[b], hi);
    }

    // Bins of what `bin_of` puts into one (-1: none), and the sums before each.
    template <class F>
    __device__ void fill(bool with_mass, F bin_of) {
        for (int i = tid; i < ST_BINS; i += ST_THREADS) count[i] = low[i] = high[i] = 0;
        __syncthreads();
        for (int i = tid; i < row.n; i += ST_THREADS) {
            const float l = to_float(row.data[i]);
            const int b = row.counts(l) ? bin_of(l, row.first + i) : -1;
            if (b >= 0) add(b, with_mass ? row.mass(row.e(l)) : 0);
        }
        sync();
        constexpr int SHARE = ST_BINS / C, PER = SHARE > ST_THREADS ? SHARE / ST_THREADS : 1;
        const int b0 = tid * PER;
        unsigned n = 0, cn[PER];
        u64 m = 0, cm[PER];
        if (b0 < SHARE) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                cn[j] = n, cm[j] = m;
                const int b = rank * SHARE + b0 + j;
#pragma unroll
                for (int r = 0; r < C; ++r) {
                    n += *at(&count[b], r);
                    m += (u64)*at(&high[b], r) << 32;
                    m += *at(&low[b], r);
                }
            }
        }
        // running sums over the CTA's threads
        unsigned in = n;
        u64 im = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned a = __shfl_up_sync(FULL, in, o);
            const u64 b = __shfl_up_sync(FULL, im, o);
            if ((tid & 31) >= o) in += a, im += b;
        }
        if ((tid & 31) == 31) sm.warp_count[tid >> 5] = in, sm.warp_mass[tid >> 5] = im;
        __syncthreads();
        unsigned wn = 0;
        u64 wm = 0;
        for (int w = 0; w < (tid >> 5); ++w) wn += sm.warp_count[w], wm += sm.warp_mass[w];
        in += wn, im += wm;
        if (tid == ST_THREADS - 1) sm.count = in, sm.mass = im;
        sync();
        unsigned before = 0;
        u64 before_mass = 0;
        all_count = 0, all_mass = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) {
            const unsigned a = *at(&sm.count, r);
            const u64 b = *at(&sm.mass, r);
            if (r < rank) before += a, before_mass += b;
            all_count += a, all_mass += b;
        }
        if (b0 < SHARE) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                pre_count[b0 + j] = before + in - n + cn[j];
                pre_mass[b0 + j] = before_mass + im - m + cm[j];
            }
            if (b0 + PER == SHARE) {
                pre_count[SHARE] = before + in;
                pre_mass[SHARE] = before_mass + im;
            }
        }
        __syncthreads();
    }

    // The bin in which the count or the mass reaches `target` (1 to the whole).
    __device__ Bin find(bool by_count, u64 target, u64 mass_before, unsigned count_before) {
        constexpr int SHARE = ST_BINS / C;
        for (int i = tid; i < SHARE; i += ST_THREADS) {
            const u64 m0 = mass_before + pre_mass[i], m1 = mass_before + pre_mass[i + 1];
            const unsigned n0 = count_before + pre_count[i], n1 = count_before + pre_count[i + 1];
            if (by_count ? n0 < target && target <= n1 : m0 < target && target <= m1) {
                const Bin b = {m0, m1 - m0, n0, n1 - n0, rank * SHARE + i};
                for (int r = 0; r < C; ++r) *at(&sm.bin, r) = b;
            }
        }
        sync();
        const Bin b = sm.bin;
        __syncthreads();
        return b;
    }

    // What `wanted` says, into the first CTA's list.
    template <class F>
    __device__ int gather(F wanted) {
        if (tid == 0) sm.listed = 0;
        sync();
        SampleShared* first = at(&sm, 0);
        for (int i = tid; i < row.n; i += ST_THREADS) {
            const float l = to_float(row.data[i]);
            if (row.counts(l) && wanted(l, row.first + i)) {
                const unsigned p = atomicAdd(&first->listed, 1u);
                if (p < ST_LIST) {
                    first->key[p] = st_key(l, row.first + i);
                    first->weight[p] = row.mass(row.e(l));
                }
            }
        }
        sync();
        return min((int)first->listed, ST_LIST);
    }

    // Number and mass of the listed ones before listed one `i`, by two threads each.
    __device__ __forceinline__ void before_in_list(int n, int i, unsigned& cnt, u64& mass) {
        cnt = 0, mass = 0;
        if (i < n) {
            const u64 mine = sm.key[i];
            for (int j = tid & 1; j < n; j += 2)
                if (sm.key[j] < mine) cnt += 1, mass += sm.weight[j];
        }
        cnt += __shfl_xor_sync(FULL, cnt, 1);
        mass += __shfl_xor_sync(FULL, mass, 1);
    }

    // The logit at which the count or the mass reaches `target`.
    __device__ Found select(bool by_count, u64 target) {
        if (!fresh) {
            fill(true, [&](float l, int) { return row.bin(l); });
            fresh = true;
        }
        Bin b = find(by_count, target, 0, 0);
        const int bin0 = b.bin;
        u64 lo = 0, hi = ~0ull;
        auto inside = [&](float l, int i) {
            if (row.bin(l) != bin0) return false;
            const u64 k = st_key(l, i);
            return lo <= k && k <= hi;
        };
        while (b.count > ST_LIST) {
            // the smallest and largest key there is between lo and hi
            u64 a = ~0ull, z = 0;
            for (int i = tid; i < row.n; i += ST_THREADS) {
                const float l = to_float(row.data[i]);
                if (row.counts(l) && inside(l, row.first + i)) {
                    const u64 k = st_key(l, row.first + i);
                    a = min(a, k), z = max(z, k);
                }
            }
            if (tid == 0) sm.lo = ~0ull, sm.hi = 0;
            __syncthreads();
            atomicMin(&sm.lo, a);
            atomicMax(&sm.hi, z);
            sync();
            a = ~0ull, z = 0;
#pragma unroll
            for (int r = 0; r < C; ++r) a = min(a, *at(&sm.lo, r)), z = max(z, *at(&sm.hi, r));
            const int width = 64 - __clzll((long long)(z - a)), shift = max(0, width - 11);
            fill(true, [&](float l, int i) { return inside(l, i) ? (int)((st_key(l, i) - a) >> shift) : -1; });
            fresh = false;
            b = find(by_count, target, b.mass_before, b.count_before);
            lo = a + ((u64)b.bin << shift);
            hi = lo + ((1ull << shift) - 1);
        }
        const int n = gather(inside);
        if (rank == 0) {
            for (int i0 = 0; i0 < n; i0 += ST_THREADS / 2) {
                const int i = i0 + (tid >> 1);
                unsigned cnt;
                u64 mass;
                before_in_list(n, i, cnt, mass);
                if (i < n && (tid & 1) == 0) {
                    cnt += b.count_before, mass += b.mass_before;
                    const u64 w = sm.weight[i];
                    if (by_count ? cnt + 1 == target : mass < target && target <= mass + w) {
                        const Found f = {mass + w, st_logit(sm.key[i]), (int)(sm.key[i] & (ST_MAX_V - 1))};
                        for (int r = 0; r < C; ++r) *at(&sm.found, r) = f;
                    }
                }
            }
        }
        sync();
        const Found f = sm.found;
        __syncthreads();
        return f;
    }
};

// Least whole target of p times a mass, and the first number above u times one.
__device__ __forceinline__ u64 share_of(float p, u64 mass) {
    const double t = ceil((double)p * (double)mass);
    return t >= (double)mass ? mass : t < 1.0 ? 1ull : (u64)t;
}
__device__ __forceinline__ u64 drawn_at(float u, u64 mass) {
    const double t = floor((double)u * (double)mass);
    return t >= (double)mass ? mass : t < 1.0 ? 1ull : (u64)t + 1;  // + 1 in whole numbers: past 2^53 a double has none
}

template <class TX, int C>
__global__ void __launch_bounds__(ST_THREADS, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char st_raw[];
    __shared__ SampleShared sm;
    __shared__ float red[2 * ST_WARPS];
    __shared__ u64 red_mass[ST_WARPS];
    u64* pre_mass = reinterpret_cast<u64*>(st_raw);
    unsigned* pre_count = reinterpret_cast<unsigned*>(pre_mass + ST_BINS / C + 2);
    unsigned* count = pre_count + ST_BINS / C + 4;
    TX* data = reinterpret_cast<TX*>(count + 3 * ST_BINS);
    const int tid = threadIdx.x;
    const int r = blockIdx.x / C;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = C == 1 ? 0 : (int)cl.block_rank();

    pdl_wait();
    pdl_trigger();
    const float temperature = a.temperature ? __ldcg(a.temperature + r) : a.temperature0;
    float top_p = a.top_p ? __ldcg(a.top_p + r) : a.top_p0;
    float min_p = a.min_p ? __ldcg(a.min_p + r) : a.min_p0;
    int top_k = a.top_k ? __ldcg(a.top_k + r) : a.top_k0;
    const float u = __ldcg(a.uniform + r);

    // the slice, in the places mod 16 bytes that it has in memory
    Row<TX> row;
    row.first = rank * a.slice;
    row.n = max(0, min(a.slice, a.V - row.first));
    {
        constexpr int VN = Vec<TX>::N;
        const TX* src = static_cast<const TX*>(a.logits) + (long long)r * a.ld + row.first;
        const int off = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(TX));
        row.data = data + off;
        float hi = -INFINITY, lo = INFINITY;
        for (int i = tid * VN; i < row.n + off; i += ST_THREADS * VN) {
            if (i >= off && i + VN <= row.n + off) {
                const uint4 v = __ldcs(reinterpret_cast<const uint4*>(src + (i - off)));
                *reinterpret_cast<uint4*>(data + i) = v;
                const TX* e = reinterpret_cast<const TX*>(&v);
#pragma unroll
                for (int j = 0; j < VN; ++j) {
                    const float l = to_float(e[j]);
                    asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(l));
                    if (l > -INFINITY) lo = fminf(lo, l);
                }
            } else {
                for (int j = max(i, off); j < min(i + VN, row.n + off); ++j) {
                    const TX e = __ldcs(src + (j - off));
                    data[j] = e;
                    const float l = to_float(e);
                    asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(l));
                    if (l > -INFINITY) lo = fminf(lo, l);
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float h = __shfl_xor_sync(FULL, hi, o);
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(h));
            lo = fminf(lo, __shfl_xor_sync(FULL, lo, o));
        }
        if ((tid & 31) == 0) red[tid >> 5] = hi, red[ST_WARPS + (tid >> 5)] = lo;
        __syncthreads();
        if (tid < 32) {
            hi = tid < ST_WARPS ? red[tid] : -INFINITY;
            lo = tid < ST_WARPS ? red[ST_WARPS + tid] : INFINITY;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float h = __shfl_xor_sync(FULL, hi, o);
                asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(h));
                lo = fminf(lo, __shfl_xor_sync(FULL, lo, o));
            }
            if (tid == 0) sm.top = hi, sm.low = lo;
        }
    }
    Sampler<TX, C> s = {sm, count, count + ST_BINS, count + 2 * ST_BINS, pre_count, pre_mass, row, cl, tid, rank, 0, 0, false};
    s.sync();
    float top = -INFINITY, low = INFINITY;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const float h = s.at(&sm, c)->top;
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(h));
        low = fminf(low, s.at(&sm, c)->low);
    }
    if (!(top > -INFINITY)) {  // nothing to draw from, or not a number
        if (rank == 0 && tid == 0) {
            a.tokens[r] = -1;
            a.logprob[r] = __int_as_float(0x7fffffff);
        }
        s.sync();  // peers have read this CTA's shared memory
        return;
    }
    double t = (double)temperature;
    if (!(temperature > 0.f)) t = 1.0, top_k = 1, top_p = 1.f, min_p = 0.f;  // the largest logit, the first of equal ones
    row.top = top;
    row.inv_t = 1.0 / t;
    row.cut = (float)fmin(32.0 * t, 3e38);
    row.inv_width = (float)ST_BINS / fmaxf(fminf(row.cut, top == low ? 1.f : top - low), 1e-30f);
    min_p = fminf(min_p, 1.f);

    u64 kept;
    Found f;
    if (top_k > 0 && top_k <= ST_QUICK_K) {
        // numbers alone, then the first k with what shares their last bin
        s.fill(false, [&](float l, int) { return row.bin(l); });
        const unsigned want = min((unsigned)top_k, s.all_count);
        const Bin b = s.find(true, want, 0, 0);
        if (b.count_before + b.count <= ST_LIST) {
            const int n = s.gather([&](float l, int) { return row.bin(l) <= b.bin; });
            if (rank == 0) {
                if (tid < 3) sm.prefix[tid] = ~0ull;
                __syncthreads();
                constexpr int ROUNDS = ST_LIST / (ST_THREADS / 2);
                unsigned cnt[ROUNDS];
                u64 before[ROUNDS];
#pragma unroll
                for (int q = 0; q < ROUNDS; ++q) {
                    const int i = q * (ST_THREADS / 2) + (tid >> 1);
                    s.before_in_list(n, i, cnt[q], before[q]);
                    if (i < n && (tid & 1) == 0 && cnt[q] + 1 == want) sm.prefix[0] = before[q] + sm.weight[i];
                }
                __syncthreads();
                const u64 mass_k = sm.prefix[0], target = share_of(top_p, mass_k);
                u64 passing = 0;
#pragma unroll
                for (int q = 0; q < ROUNDS; ++q) {
                    const int i = q * (ST_THREADS / 2) + (tid >> 1);
                    if (i >= n || (tid & 1) != 0) continue;
                    const u64 end = before[q] + sm.weight[i];
                    if (top_p < 1.f && before[q] < target && target <= end) sm.prefix[1] = end;
                    if (!(row.e(st_logit(sm.key[i])) < (double)min_p)) passing = max(passing, end);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) passing = max(passing, __shfl_xor_sync(FULL, passing, o));
                if ((tid & 31) == 0) red_mass[tid >> 5] = passing;
                __syncthreads();
                for (int w = 0; w < ST_WARPS; ++w) passing = max(passing, red_mass[w]);
                kept = min(min(mass_k, sm.prefix[1]), passing);
                const u64 drawn = drawn_at(u, kept);
#pragma unroll
                for (int q = 0; q < ROUNDS; ++q) {
                    const int i = q * (ST_THREADS / 2) + (tid >> 1);
                    if (i >= n || (tid & 1) != 0) continue;
                    if (before[q] < drawn && drawn <= before[q] + sm.weight[i]) {
                        a.tokens[r] = (int64_t)(sm.key[i] & (ST_MAX_V - 1));
                        a.logprob[r] = (float)(row.score(st_logit(sm.key[i])) - log((double)kept / ST_ONE));
                    }
                }
            }
            s.sync();  // no CTA leaves while another may read its shared memory
            return;
        }
    }
    s.fill(true, [&](float l, int) { return row.bin(l); });
    s.fresh = true;
    const u64 all_mass = s.all_mass;
    kept = all_mass;
    if (top_k > 0 && (unsigned)top_k < s.all_count) kept = s.select(true, (u64)top_k).mass;
    if (top_p < 1.f) kept = s.select(false, share_of(top_p, kept)).mass;
    if (min_p > 0.f) {
        u64 m = 0;
        for (int i = tid; i < row.n; i += ST_THREADS) {
            const float l = to_float(row.data[i]);
            if (row.counts(l)) {
                const double e = row.e(l);
                if (!(e < (double)min_p)) m += row.mass(e);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(FULL, m, o);
        if ((tid & 31) == 0) red_mass[tid >> 5] = m;
        __syncthreads();
        if (tid == 0) {
            m = 0;
            for (int w = 0; w < ST_WARPS; ++w) m += red_mass[w];
            sm.mass_min_p = m;
        }
        s.sync();
        m = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) m += s.at(&sm, c)->mass_min_p;
        kept = min(kept, m);
    }
    f = s.select(false, drawn_at(u, kept));
    if (rank == 0 && tid == 0) {
        a.tokens[r] = f.index;
        a.logprob[r] = (float)(row.score(f.logit) - log((double)kept / ST_ONE));
    }
    s.sync();
}

template <class TX, int C>
static cudaError_t sample_launch(SampleArgs a, cudaStream_t s) {
    a.slice = ((a.V + C - 1) / C + 7) & ~7;
    const size_t smem = (ST_BINS / C + 2) * 8 + (ST_BINS / C + 4) * 4 + 3 * ST_BINS * 4 + (size_t)a.slice * sizeof(TX) + 16;
    cudaError_t e = prepare_kernel<sample_kernel<TX, C>>(200 * 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * C);
    cfg.blockDim = dim3(ST_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, sample_kernel<TX, C>, a);
}

template <class TX>
static cudaError_t sample_typed(const SampleArgs& a, cudaStream_t s) {
    if (a.V <= 8192) return sample_launch<TX, 1>(a, s);
    return sample_launch<TX, 8>(a, s);
}

}  // namespace skb

using namespace skb;

extern "C" int skb_sample_tokens(const void* logits, int type, int64_t ld, int rows, int V, const float* uniform,
                                 const float* temperatures, float temperature, const int32_t* top_ks, int top_k,
                                 const float* top_ps, float top_p, const float* min_ps, float min_p, int64_t* tokens,
                                 float* logprob, cudaStream_t stream) {
    if (!logits || !uniform || !tokens || !logprob) return fail(SKB_ERR_ARG, "sample_tokens: null pointer");
    if (rows < 0 || rows > (1 << 27) || V < 1 || V > ST_MAX_V || ld < V)
        return fail(SKB_ERR_ARG, "sample_tokens: bad sizes (%d rows of %d logits, 1 to %d)", rows, V, ST_MAX_V);
    if (type < SKB_F32 || type > SKB_F16) return fail(SKB_ERR_ARG, "sample_tokens: unknown type %d", type);
    if (reinterpret_cast<uintptr_t>(logits) % type_size(type) != 0 || reinterpret_cast<uintptr_t>(tokens) % 8 != 0 ||
        (reinterpret_cast<uintptr_t>(uniform) | reinterpret_cast<uintptr_t>(temperatures) |
         reinterpret_cast<uintptr_t>(top_ks) | reinterpret_cast<uintptr_t>(top_ps) | reinterpret_cast<uintptr_t>(min_ps) |
         reinterpret_cast<uintptr_t>(logprob)) % 4 != 0)
        return fail(SKB_ERR_ARG, "sample_tokens: misaligned pointer");
    if (rows == 0) return SKB_OK;
    const SampleArgs a = {logits, ld, rows, V, 0, uniform, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p,
                          top_k, tokens, logprob};
    const cudaError_t e = type == SKB_F32    ? sample_typed<float>(a, stream)
                          : type == SKB_BF16 ? sample_typed<__nv_bfloat16>(a, stream)
                                             : sample_typed<__half>(a, stream);
    return e == cudaSuccess ? SKB_OK : fail(SKB_ERR_CUDA, "sample_tokens: %s", cudaGetErrorString(e));
}
