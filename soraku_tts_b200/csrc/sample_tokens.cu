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
// Weights are whole multiples of 2^-44, formed in 64 bits, so sums are exact in
// any order and a draw does not depend on the order of atomics; what weighs less than
// 2^-45 of the largest weighs nothing, and all of it together (2^18 logits at most)
// is less than the last step 2^-24 of a uniform number.  A cluster of CTAs holds
// the row in shared memory, read once from the device's.
//
// With a top-k of up to 1536: the k-th largest of the threads' own largest logits
// bounds the k-th logit from below, and hardly more than k logits are above it
// (k = 1000 of 151,936: about 1150).  Those alone are gathered in one CTA, put in
// order and weighed.
//
// Else one pass counts the logits in 2048 bins along the order.  Counts times the
// weight at a bin's middle say to a few places where each sum will reach its
// target; a second pass weighs every logit, adds up what stands before windows of
// a few hundred logits about those places, and lists what is in them.  The list is
// put in order in one CTA, and the answers read off exactly.
//
// Where the windows miss, or more equal logits share a bin than a list holds, the
// bins are weighed too and the bin of each answer is binned again by (logit,
// index), as often as it takes (st_general).
#include <cooperative_groups.h>

#include "int8_ops.cuh"

namespace skb {
namespace cg = cooperative_groups;

constexpr int ST_THREADS = 512, ST_WARPS = ST_THREADS / 32;
constexpr int ST_BINS = 2048;
constexpr int ST_LIST = 512;        // logits of one gathered bin
constexpr int ST_SORT = 2048;       // logits that are gathered to be put in order
constexpr int ST_QUICK_K = 1536;
constexpr int ST_FOUR = ST_SORT / ST_THREADS;  // listed logits a thread holds, and bins
static_assert(ST_BINS == ST_SORT, "as many bins as listed logits");
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

// Bins [b0, b1] about an answer.
struct Window {
    int b0, b1;
};

struct SampleShared {
    Window window[3];          // apart and in order; written by the first CTA, to all
    int windows;               // -1: no list can hold them
    u64 part[5];               // this CTA's masses: before each window, all, passing min-p
    unsigned before[3];        // logits before each window
    float approx[4];
    int answer[3];
    u64 delta[3];
    int starts[3];
    float top, low;            // this CTA's
    u64 mass, mass_min_p;      // this CTA's totals
    unsigned count;
    u64 lo, hi;                // smallest and largest key of a bin, this CTA's
    Bin bin;                   // written by the CTA that found it, to all
    Found found;
    unsigned listed;           // logits that this CTA has listed
    u64 warp_mass[ST_WARPS];
    unsigned warp_count[ST_WARPS];
    float red[2 * ST_WARPS];
    u64 prefix[3];
    double power[32];          // 2^(i / 32)
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

// Least whole target of p times a mass, and the first number above u times one.
__device__ __forceinline__ u64 share_of(float p, u64 mass) {
    const double t = ceil((double)p * (double)mass);
    return t >= (double)mass ? mass : !(t >= 1.0) ? 1ull : (u64)t;
}
__device__ __forceinline__ u64 drawn_at(float u, u64 mass) {
    const double t = floor((double)u * (double)mass);
    return t >= (double)mass ? mass : !(t >= 1.0) ? 1ull : (u64)t + 1;  // + 1 in whole numbers: past 2^53 a double has none
}

template <class TX>
struct Row {
    const TX* data;  // this CTA's slice in shared memory
    const double* power;
    int n, first;    // logits, and the first one's index
    float top, cut, inv_width;
    double inv_t, scale;  // 1 / T, and 32 log2(e) / T
    // how far below the largest; beyond `cut`: without weight
    __device__ __forceinline__ float gap(float l) const { return l == top ? 0.f : top - l; }
    __device__ __forceinline__ bool counts(float l) const { return gap(l) <= cut && l > -INFINITY; }
    __device__ __forceinline__ int bin(float l) const { return min((int)fminf(gap(l) * inv_width, 3e4f), ST_BINS - 1); }
    __device__ __forceinline__ double score(float l) const { return l == top ? 0.0 : ((double)l - (double)top) * inv_t; }
    // exp((l - top) / T) 2^44 for a logit that counts: 2^(n / 32) from a table and the
    // power series of what is left, |x| <= log(2) / 64, to its fifth power (the sixth is
    // 2^-48).  The exponent is at least 44 - 48: no underflow.
    __device__ __forceinline__ double weight(float l) const {
        if (l == top) return ST_ONE;
        constexpr double MAGIC = 6755399441055744.0, LN2_32 = 0.021660849392498290;
        const double y = ((double)l - (double)top) * scale;
        const double m = y + MAGIC;
        const int n = __double2loint(m);
        const double x = (y - (m - MAGIC)) * LN2_32;
        double p = fma(x, 1.0 / 120, 1.0 / 24);
        p = fma(p, x, 1.0 / 6);
        p = fma(p, x, 0.5);
        p = fma(p, x, 1.0);
        p = fma(p, x, 1.0) * power[n & 31];
        return __hiloint2double(__double2hiint(p) + (((n >> 5) + 44) << 20), __double2loint(p));
    }
    __device__ __forceinline__ static u64 mass(double weight) {
        // up to 2^44, rounded by adding 2^52
        return (u64)__double_as_longlong(weight + 4503599627370496.0) & 0xfffffffffffffull;
    }
};

template <class TX, int C>
struct Sampler {
    SampleShared& sm;
    u64 *key, *weight;             // the list
    unsigned *count, *low, *high;  // bins of this CTA's logits: number, and mass in two words
    unsigned* pre_count;           // of this CTA's share of the bins, cluster-wide: what stands before each
    u64* pre_mass;
    const Row<TX>& row;
    cg::cluster_group cl;
    int tid, rank;
    u64 all_mass, mass_min_p;
    unsigned all_count;
    bool fresh;  // the bins hold the whole row

    template <class T>
    __device__ __forceinline__ T* at(T* p, int r) { return C == 1 ? p : cl.map_shared_rank(p, r); }
    __device__ __forceinline__ void sync() {
        if (C == 1) __syncthreads();
        else cl.sync();
    }

    __device__ __forceinline__ void clear() {
        for (int i = tid; i < ST_BINS; i += ST_THREADS) count[i] = low[i] = high[i] = 0;
        __syncthreads();
    }
    __device__ __forceinline__ void add(int b, u64 m) {
        atomicAdd(&count[b], 1u);
        if (m == 0) return;
        const unsigned lo = (unsigned)m, old = atomicAdd(&low[b], lo);
        const unsigned hi = (unsigned)(m >> 32) + (old + lo < old ? 1u : 0u);
        if (hi) atomicAdd(&high[b], hi);
    }

    // Every CTA's bins into running sums over the cluster's, each CTA a share of the bins.
    // passing: this thread's mass of what min-p lets stay.
    __device__ __forceinline__ void total(u64 passing) {
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
        unsigned in = n;
        u64 im = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned a = __shfl_up_sync(FULL, in, o);
            const u64 b = __shfl_up_sync(FULL, im, o);
            if ((tid & 31) >= o) in += a, im += b;
            passing += __shfl_xor_sync(FULL, passing, o);
        }
        if ((tid & 31) == 31) sm.warp_count[tid >> 5] = in, sm.warp_mass[tid >> 5] = im;
        if ((tid & 31) == 0 && passing) atomicAdd(&sm.mass_min_p, passing);
        __syncthreads();
        unsigned wn = 0;
        u64 wm = 0;
        for (int w = 0; w < (tid >> 5); ++w) wn += sm.warp_count[w], wm += sm.warp_mass[w];
        in += wn, im += wm;
        if (tid == ST_THREADS - 1) sm.count = in, sm.mass = im;
        sync();
        unsigned before = 0;
        u64 before_mass = 0;
        all_count = 0, all_mass = 0, mass_min_p = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) {
            const unsigned a = *at(&sm.count, r);
            const u64 b = *at(&sm.mass, r);
            if (r < rank) before += a, before_mass += b;
            all_count += a, all_mass += b;
            mass_min_p += *at(&sm.mass_min_p, r);
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
    // The whole row's bins.
    __device__ __forceinline__ void fill(double min_weight) {
        clear();
        u64 passing = 0;
        for (int i = tid; i < row.n; i += ST_THREADS) {
            const float l = to_float(row.data[i]);
            if (row.counts(l)) {
                const double w = row.weight(l);
                const u64 m = row.mass(w);
                add(row.bin(l), m);
                if (!(w < min_weight)) passing += m;
            }
        }
        total(passing);
        fresh = true;
    }

    // The bin in which the count or the mass reaches `target` (1 to the whole).
    // Nothing is listed any more.
    __device__ __forceinline__ Bin find(bool by_count, u64 target, u64 mass_before, unsigned count_before) {
        constexpr int SHARE = ST_BINS / C;
        if (tid == 0) sm.listed = 0;
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

    // What `wanted` says, into this CTA's list.
    template <class F>
    __device__ __forceinline__ void list(F wanted) {
        for (int i = tid; i < row.n; i += ST_THREADS) {
            const float l = to_float(row.data[i]);
            if (wanted(l)) {
                const unsigned p = atomicAdd(&sm.listed, 1u);
                if (p < ST_SORT) key[p] = st_key(l, row.first + i);
            }
        }
    }
    // The first CTA: everybody's lists, in order, to its own.  `fine`: bins [0, ST_BINS)
    // along the order, the finer the better.  The number of logits; more than
    // ST_SORT: nothing was done.
    template <class F>
    __device__ __forceinline__ int collect(F fine) {
        unsigned from[C + 1];
        from[0] = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) from[r + 1] = from[r] + *at(&sm.listed, r);
        const int n = (int)min(from[C], (unsigned)ST_SORT + 1);
        if (n > ST_SORT) return n;
        u64 k[ST_FOUR];
        unsigned slot[ST_FOUR];
        int bin[ST_FOUR];
#pragma unroll
        for (int j = 0; j < ST_FOUR; ++j) {
            const int i = j * ST_THREADS + tid;
            k[j] = ~0ull;
            if (i < n) {
                int r = 0;
                while (from[r + 1] <= (unsigned)i) ++r;
                k[j] = at(key, r)[i - from[r]];
            }
        }
        for (int i = tid; i < ST_BINS; i += ST_THREADS) count[i] = 0;
        if (tid == 0) sm.answer[0] = 0;
        __syncthreads();
        if (n <= 128) {
            // few: each counts those before it
            if (tid < n) key[tid] = k[0];
            __syncthreads();
            const int i = tid >> 2;  // four threads each
            unsigned before = 0;
            u64 mine = 0;
            if (i < n) {
                mine = key[i];
                for (int j = tid & 3; j < n; j += 4) before += key[j] < mine;
            }
            before += __shfl_xor_sync(FULL, before, 1);
            before += __shfl_xor_sync(FULL, before, 2);
            __syncthreads();
            if (i < n && (tid & 3) == 0) key[before] = mine;
            __syncthreads();
            return n;
        }
        int crowd = 0;
#pragma unroll
        for (int j = 0; j < ST_FOUR; ++j)
            if (j * ST_THREADS + tid < n) {
                bin[j] = fine(st_logit(k[j]));
                slot[j] = atomicAdd(&count[bin[j]], 1u);
                crowd = max(crowd, (int)slot[j]);
            }
        crowd = __reduce_max_sync(FULL, crowd);
        if ((tid & 31) == 0 && crowd > 32) sm.answer[0] = 1;
        __syncthreads();
        if (sm.answer[0]) {  // many equal ones
#pragma unroll
            for (int j = 0; j < ST_FOUR; ++j)
                if (j * ST_THREADS + tid < n) key[j * ST_THREADS + tid] = k[j];
            __syncthreads();
            sort(n);
            return n;
        }
        // bins' counts to where they begin; then each place within a bin
        const uint4 c = reinterpret_cast<const uint4*>(count)[tid];
        unsigned sum = c.x + c.y + c.z + c.w, upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(FULL, upto, o);
            if ((tid & 31) >= o) upto += x;
        }
        if ((tid & 31) == 31) sm.warp_count[tid >> 5] = upto;
        __syncthreads();
        unsigned at0 = upto - sum;
        for (int w = 0; w < (tid >> 5); ++w) at0 += sm.warp_count[w];
        reinterpret_cast<uint4*>(count)[tid] = make_uint4(at0, at0 + c.x, at0 + c.x + c.y, at0 + c.x + c.y + c.z);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ST_FOUR; ++j)
            if (j * ST_THREADS + tid < n) key[count[bin[j]] + slot[j]] = k[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ST_FOUR; ++j)
            if (j * ST_THREADS + tid < n) {
                const unsigned b0 = count[bin[j]], b1 = bin[j] + 1 < ST_BINS ? count[bin[j] + 1] : (unsigned)n;
                slot[j] = b0;
                for (unsigned i = b0; i < b1; ++i) slot[j] += key[i] < k[j];
            }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ST_FOUR; ++j)
            if (j * ST_THREADS + tid < n) key[slot[j]] = k[j];
        __syncthreads();
        return n;
    }

    // What `wanted` says, into the first CTA's list; how many there are, listed or not.
    template <class F>
    __device__ __forceinline__ unsigned gather(int room, F wanted) {
        unsigned* listed = at(&sm.listed, 0);
        u64* keys = at(key, 0);
        for (int i = tid; i < row.n; i += ST_THREADS) {
            const float l = to_float(row.data[i]);
            if (wanted(l, row.first + i)) {
                const unsigned p = atomicAdd(listed, 1u);
                if (p < room) keys[p] = st_key(l, row.first + i);
            }
        }
        sync();
        return *listed;
    }
    __device__ __forceinline__ u64 weigh(u64 k) { return row.mass(row.weight(st_logit(k))); }

    // The logit at which the count or the mass reaches `target`.
    __device__ __forceinline__ Found select(bool by_count, u64 target) {
        if (!fresh) fill(INFINITY);
        Bin b = find(by_count, target, 0, 0);
        const int bin0 = b.bin;
        u64 lo = 0, hi = ~0ull;
        auto inside = [&](float l, int i) {
            if (!row.counts(l) || row.bin(l) != bin0) return false;
            const u64 k = st_key(l, i);
            return lo <= k && k <= hi;
        };
        while (b.count > ST_LIST) {
            // the smallest and largest key there is between lo and hi
            u64 a = ~0ull, z = 0;
            for (int i = tid; i < row.n; i += ST_THREADS) {
                const float l = to_float(row.data[i]);
                if (inside(l, row.first + i)) {
                    const u64 k = st_key(l, row.first + i);
                    a = min(a, k), z = max(z, k);
                }
            }
            if (tid == 0) sm.lo = ~0ull, sm.hi = 0;
            clear();
            if (a <= z) {
                atomicMin(&sm.lo, a);
                atomicMax(&sm.hi, z);
            }
            sync();
            a = ~0ull, z = 0;
#pragma unroll
            for (int r = 0; r < C; ++r) a = min(a, *at(&sm.lo, r)), z = max(z, *at(&sm.hi, r));
            const int width = 64 - __clzll((long long)(z - a)), shift = max(0, width - 11);
            for (int i = tid; i < row.n; i += ST_THREADS) {
                const float l = to_float(row.data[i]);
                if (inside(l, row.first + i)) add((int)((st_key(l, row.first + i) - a) >> shift), row.mass(row.weight(l)));
            }
            total(0);
            fresh = false;
            b = find(by_count, target, b.mass_before, b.count_before);
            lo = a + ((u64)b.bin << shift);
            hi = lo + ((1ull << shift) - 1);
        }
        const int n = min(gather(ST_LIST, inside), (unsigned)ST_LIST);
        if (rank == 0) {
            for (int i = tid; i < n; i += ST_THREADS) weight[i] = weigh(key[i]);
            __syncthreads();
            // two threads each add up what stands before one
            for (int i0 = 0; i0 < n; i0 += ST_THREADS / 2) {
                const int i = i0 + (tid >> 1);
                unsigned cnt = 0;
                u64 mass = 0;
                if (i < n) {
                    const u64 mine = key[i];
                    for (int j = tid & 1; j < n; j += 2)
                        if (key[j] < mine) cnt += 1, mass += weight[j];
                }
                cnt += __shfl_xor_sync(FULL, cnt, 1);
                mass += __shfl_xor_sync(FULL, mass, 1);
                if (i < n && (tid & 1) == 0) {
                    cnt += b.count_before, mass += b.mass_before;
                    const u64 w = weight[i];
                    if (by_count ? cnt + 1 == target : mass < target && target <= mass + w) {
                        const Found f = {mass + w, st_logit(key[i]), (int)(key[i] & (ST_MAX_V - 1))};
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

    // The first CTA: windows about where the answers will be, to all.  total: its bins'
    // counts; span: the logits they cover.
    __device__ __forceinline__ void choose_windows(const unsigned* total, float span, double t, int top_k, float top_p, float min_p,
                                                   float u) {
        const int lane = tid & 31, warp = tid >> 5;
        const uint4 c4 = reinterpret_cast<const uint4*>(total)[tid];
        const unsigned c[ST_FOUR] = {c4.x, c4.y, c4.z, c4.w};
        // mass by the weight at the middle of each bin (nothing of the first is above its beginning)
        const float step = (float)(span / ST_BINS / t);
        float m[ST_FOUR], mass = 0.f;
        unsigned cnt = 0;
#pragma unroll
        for (int j = 0; j < ST_FOUR; ++j) {
            const int b = tid * ST_FOUR + j;
            m[j] = c[j] == 0 ? 0.f : b == 0 ? 1.f + (float)(c[j] - 1) * __expf(-0.5f * step) : (float)c[j] * __expf(-((float)b + 0.5f) * step);
            mass += m[j], cnt += c[j];
        }
        float mass_at = mass;
        unsigned cnt_at = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float x = __shfl_up_sync(FULL, mass_at, o);
            const unsigned y = __shfl_up_sync(FULL, cnt_at, o);
            if (lane >= o) mass_at += x, cnt_at += y;
        }
        float* warp_mass = sm.red;
        if (lane == 31) warp_mass[warp] = mass_at, sm.warp_count[warp] = cnt_at;
        if (tid < 3) sm.answer[tid] = -1, sm.approx[tid] = -1.f;
        __syncthreads();
        mass_at -= mass, cnt_at -= cnt;
        float all = 0.f;
        unsigned everyone = 0;
        for (int w = 0; w < ST_WARPS; ++w) {
            if (w < warp) mass_at += warp_mass[w], cnt_at += sm.warp_count[w];
            all += warp_mass[w], everyone += sm.warp_count[w];
        }
        // what stands up to each of this thread's bins
        float mb[ST_FOUR + 1];
        unsigned cb[ST_FOUR + 1];
        mb[0] = mass_at, cb[0] = cnt_at;
#pragma unroll
        for (int j = 0; j < ST_FOUR; ++j) mb[j + 1] = mb[j] + m[j], cb[j + 1] = cb[j] + c[j];
        const bool with_k = top_k > 0 && (unsigned)top_k < everyone;
        // the last bin that min-p lets stay
        const float edge = min_p > 0.f ? fminf(-__logf(fminf(min_p, 1.f)) / step, 3e4f) : 3e4f;
#pragma unroll
        for (int j = 0; j < ST_FOUR; ++j) {
            const int b = tid * ST_FOUR + j;
            if (with_k && cb[j] < (unsigned)top_k && (unsigned)top_k <= cb[j + 1]) sm.answer[0] = b, sm.approx[0] = 0.5f * (mb[j] + mb[j + 1]);
            if ((int)edge == b) sm.approx[1] = mb[j + 1];
        }
        __syncthreads();
        float kept = with_k ? sm.approx[0] : all;
        auto locate = [&](int which, float target) {
#pragma unroll
            for (int j = 0; j < ST_FOUR; ++j)
                if (c[j] > 0 && mb[j] <= target && target < mb[j + 1]) sm.answer[which] = tid * ST_FOUR + j;
        };
        if (top_p < 1.f) {
            kept *= fmaxf(top_p, 0.f);
            locate(1, kept);
        }
        if (sm.approx[1] >= 0.f) kept = fminf(kept, sm.approx[1]);
        locate(2, kept * fminf(fmaxf(u, 0.f), 1.f));
        __syncthreads();
        // as many logits to each side as the list has room for
        int at[3] = {sm.answer[0], sm.answer[1], sm.answer[2]};
        if (at[1] < 0 && top_p < 1.f) at[1] = ST_BINS - 1;  // rounding of the sums
        if (at[2] < 0) at[2] = at[1] >= 0 ? at[1] : ST_BINS - 1;
        int n = 0;
        for (unsigned room = 384;; room = room > 100 ? room / 4 : 0) {
            __syncthreads();
            if (tid < 3) sm.window[tid] = {at[tid], at[tid]};
#pragma unroll
            for (int q = 0; q < 3; ++q)
                if (at[q] >= 0 && at[q] / ST_FOUR == tid) {
#pragma unroll
                    for (int j = 0; j < ST_FOUR; ++j)
                        if (at[q] % ST_FOUR == j) sm.before[q] = cb[j], sm.starts[q] = (int)cb[j + 1];
                }
            __syncthreads();
#pragma unroll
            for (int q = 1; q < 3; ++q)
                if (at[q] >= 0) {
#pragma unroll
                    for (int j = 0; j < ST_FOUR; ++j) {
                        const int b = tid * ST_FOUR + j;
                        if (b < at[q] && sm.before[q] - cb[j] <= room) atomicMin(&sm.window[q].b0, b);
                        if (b > at[q] && cb[j + 1] - (unsigned)sm.starts[q] <= room) atomicMax(&sm.window[q].b1, b);
                    }
                }
            __syncthreads();
            // in order, and those that touch as one
            Window w[3];
            n = 0;
            int order[3] = {2, 1, 0};  // what is drawn comes first, top-k's end last
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                if (at[order[q]] < 0) continue;
                const Window x = sm.window[order[q]];
                int i = n;
                while (i > 0 && w[i - 1].b0 > x.b0) w[i] = w[i - 1], --i;
                w[i] = x;
                ++n;
            }
            int k = 0;
            for (int q = 1; q < n; ++q) {
                if (w[q].b0 <= w[k].b1 + 1) w[k].b1 = max(w[k].b1, w[q].b1);
                else w[++k] = w[q];
            }
            n = k + 1;
            // how many logits there are in them, and before them
            __syncthreads();
            if (tid == 0) sm.listed = 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < ST_FOUR; ++j) {
                const int b = tid * ST_FOUR + j;
                for (int q = 0; q < n; ++q) {
                    if (w[q].b0 == b) sm.before[q] = cb[j], atomicSub(&sm.listed, cb[j]);
                    if (w[q].b1 == b) atomicAdd(&sm.listed, cb[j + 1]);
                }
            }
            __syncthreads();
            const unsigned listed = sm.listed;
            if (listed <= ST_SORT || room == 0) {
                if (listed > ST_SORT) n = -1;
                if (tid < C) {
                    SampleShared* peer = at_rank(tid);
                    peer->windows = n;
                    for (int q = 0; q < 3; ++q) peer->window[q] = q < n ? w[q] : Window{-1, -1};
                    for (int q = 0; q < 5; ++q) peer->part[q] = 0;
                }
                __syncthreads();
                if (tid == 0) sm.listed = 0;
                return;
            }
        }
    }
    __device__ __forceinline__ SampleShared* at_rank(int r) { return at(&sm, r); }

    // The n listed keys in ascending order, the first CTA's threads all.
    __device__ __forceinline__ void sort(int n) {
        int size = 32;
        while (size < n) size <<= 1;
        for (int i = n + tid; i < size; i += ST_THREADS) key[i] = ~0ull;
        __syncthreads();
        for (int k = 2; k <= size; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int p = tid; p < size / 2; p += ST_THREADS) {
                    const int i = 2 * p - (p & (j - 1)), o = i + j;
                    const u64 x = key[i], y = key[o];
                    if ((x > y) == ((i & k) == 0)) key[i] = y, key[o] = x;
                }
                __syncthreads();
            }
        __syncthreads();
    }
};

// The row by bins with their masses, binned again as often as it takes.
template <class TX, int C>
__device__ __noinline__ void st_general(const SampleArgs& a, Row<TX> row, SampleShared& sm, unsigned* count, int r, int rank,
                                        int top_k, float top_p, double min_weight, float u) {
    u64* pre_mass = reinterpret_cast<u64*>(count) - (ST_BINS / C + 2) - (ST_BINS / C + 4) / 2;
    unsigned* pre_count = reinterpret_cast<unsigned*>(pre_mass + ST_BINS / C + 2);
    u64* key = reinterpret_cast<u64*>(count + ST_BINS);
    Sampler<TX, C> s = {sm, key, key + ST_LIST, count, count + ST_BINS, count + 2 * ST_BINS, pre_count, pre_mass, row,
                        cg::this_cluster(), (int)threadIdx.x, rank, 0, 0, 0, false};
    s.sync();  // whatever was being read in this CTA's shared memory has been
    s.fill(min_weight);
    u64 kept = s.all_mass;
    const u64 passing = min_weight > 0 ? s.mass_min_p : kept;
    Found f;
    // where top-k ends, where top-p does, and what is drawn
#pragma unroll 1
    for (int question = 0; question < 3; ++question) {
        u64 target;
        if (question == 0) {
            if (top_k <= 0 || (unsigned)top_k >= s.all_count) continue;
            target = (u64)top_k;
        } else if (question == 1) {
            if (!(top_p < 1.f)) continue;
            target = share_of(top_p, kept);
        } else {
            kept = min(kept, passing);
            target = drawn_at(u, kept);
        }
        f = s.select(question == 0, target);
        if (question < 2) kept = f.mass;
    }
    if (rank == 0 && threadIdx.x == 0) {
        a.tokens[r] = f.index;
        a.logprob[r] = (float)(row.score(f.logit) - log((double)kept / ST_ONE));
    }
    s.sync();
}

template <class TX, int C>
__global__ void __launch_bounds__(ST_THREADS, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char st_raw[];
    __shared__ SampleShared sm;
    u64* pre_mass = reinterpret_cast<u64*>(st_raw);
    unsigned* pre_count = reinterpret_cast<unsigned*>(pre_mass + ST_BINS / C + 2);
    unsigned* count = pre_count + ST_BINS / C + 4;
    // the list lies over the bins' masses: those are summed up before anything is listed
    u64* key = reinterpret_cast<u64*>(count + ST_BINS);
    static_assert(ST_SORT * 8 <= 2 * ST_BINS * 4, "the list fits");
    TX* data = reinterpret_cast<TX*>(count + 3 * ST_BINS);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / C;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = C == 1 ? 0 : (int)cl.block_rank();
    if (tid < 32) sm.power[tid] = exp2(tid / 32.0);
    for (int i = tid; i < ST_BINS; i += ST_THREADS) count[i] = 0;
    if (tid == 0) sm.listed = 0;

    pdl_wait();
    pdl_trigger();
    const float temperature = a.temperature ? __ldcg(a.temperature + r) : a.temperature0;
    float top_p = a.top_p ? __ldcg(a.top_p + r) : a.top_p0;
    float min_p = a.min_p ? __ldcg(a.min_p + r) : a.min_p0;
    int top_k = a.top_k ? __ldcg(a.top_k + r) : a.top_k0;
    const float u = __ldcg(a.uniform + r);

    // the slice, in the places mod 16 bytes that it has in memory
    Row<TX> row;
    row.power = sm.power;
    row.first = rank * a.slice;
    row.n = max(0, min(a.slice, a.V - row.first));
    float mine = -INFINITY;  // this thread's largest
    {
        constexpr int VN = Vec<TX>::N;
        const TX* src = static_cast<const TX*>(a.logits) + (long long)r * a.ld + row.first;
        const int off = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(TX));
        row.data = data + off;
        float lo = INFINITY;
        auto see = [&](float l) {
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(mine) : "f"(l));
            if (l > -INFINITY) lo = fminf(lo, l);
        };
#pragma unroll 4
        for (int i = tid * VN; i < row.n + off; i += ST_THREADS * VN) {
            Vec<TX> v;
            if (i >= off && i + VN <= row.n + off) {
                v.raw = __ldcs(reinterpret_cast<const uint4*>(src + (i - off)));
                *reinterpret_cast<uint4*>(data + i) = v.raw;
                float f[VN];
                v.get(f);
#pragma unroll
                for (int j = 0; j < VN; ++j) see(f[j]);
            } else {
                for (int j = max(i, off); j < min(i + VN, row.n + off); ++j) {
                    const TX e = __ldcs(src + (j - off));
                    data[j] = e;
                    see(to_float(e));
                }
            }
        }
        float hi = mine;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float h = __shfl_xor_sync(FULL, hi, o);
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(h));
            lo = fminf(lo, __shfl_xor_sync(FULL, lo, o));
        }
        if (lane == 0) sm.red[warp] = hi, sm.red[ST_WARPS + warp] = lo;
        __syncthreads();
        if (warp == 0) {
            hi = lane < ST_WARPS ? sm.red[lane] : -INFINITY;
            lo = lane < ST_WARPS ? sm.red[ST_WARPS + lane] : INFINITY;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float h = __shfl_xor_sync(FULL, hi, o);
                asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(h));
                lo = fminf(lo, __shfl_xor_sync(FULL, lo, o));
            }
            if (lane == 0) sm.top = hi, sm.low = lo, sm.mass_min_p = 0, sm.windows = 0;
        }
    }
    Sampler<TX, C> s = {sm, key, key + ST_LIST, count, count + ST_BINS, count + 2 * ST_BINS, pre_count, pre_mass, row, cl,
                        tid, rank, 0, 0, 0, false};
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
    row.scale = 46.166241308446828 / t;
    row.cut = (float)fmin(32.0 * t, 3e38);
    const float span = fmaxf(fminf(row.cut, top == low ? 1.f : top - low), 1e-30f);
    row.inv_width = (float)ST_BINS / span;
    const double min_weight = min_p > 0.f ? (double)fminf(min_p, 1.f) * ST_ONE : 0.0;
    const bool quick = top_k > 0 && top_k <= ST_QUICK_K;

    u64 part[5] = {};  // masses before each window, of all, and of what min-p lets stay
    if (quick) {
        // the bin of the k-th of the threads' largest: all that is in later bins
        // comes behind the first k.  (Not in a bin: weighs nothing.)
        if (row.counts(mine)) atomicAdd(s.at(&count[row.bin(mine)], 0), 1u);
        s.sync();
        if (rank == 0) {
            const uint4 c4 = reinterpret_cast<const uint4*>(count)[tid];
            const unsigned c[ST_FOUR] = {c4.x, c4.y, c4.z, c4.w}, sum = c4.x + c4.y + c4.z + c4.w;
            unsigned at = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned x = __shfl_up_sync(FULL, at, o);
                if (lane >= o) at += x;
            }
            if (lane == 31) sm.warp_count[warp] = at;
            if (tid == 0) sm.answer[0] = ST_BINS - 1;
            __syncthreads();
            at -= sum;
            for (int w = 0; w < warp; ++w) at += sm.warp_count[w];
#pragma unroll
            for (int j = 0; j < ST_FOUR; ++j) {
                if (at < (unsigned)top_k && (unsigned)top_k <= at + c[j]) sm.answer[0] = tid * ST_FOUR + j;
                at += c[j];
            }
            __syncthreads();
            if (tid < C) *s.at(&sm.window[0], tid) = {0, sm.answer[0]};
        }
        s.sync();
        const int last = sm.window[0].b1;
        s.list([&](float l) { return row.counts(l) && row.bin(l) <= last; });
        s.sync();
    } else {
        for (int i = tid; i < row.n; i += ST_THREADS) {
            const float l = to_float(row.data[i]);
            if (row.counts(l)) atomicAdd(&count[row.bin(l)], 1u);
        }
        s.sync();
        // each CTA adds up a share of the bins, into the first one's list
        constexpr int SHARE = ST_BINS / C;
        unsigned* total = reinterpret_cast<unsigned*>(key);
        for (int i = tid; i < SHARE; i += ST_THREADS) {
            unsigned n = 0;
#pragma unroll
            for (int c = 0; c < C; ++c) n += *s.at(&count[rank * SHARE + i], c);
            s.at(total, 0)[rank * SHARE + i] = n;
        }
        s.sync();
        if (rank == 0) s.choose_windows(total, span, t, top_k, top_p, min_p, u);
        s.sync();
        const int windows = sm.windows;
        if (windows < 0) {
            st_general<TX, C>(a, row, sm, count, r, rank, top_k, top_p, min_weight, u);
            return;
        }
        const Window w0 = sm.window[0], w1 = sm.window[1], w2 = sm.window[2];
        for (int i = tid; i < row.n; i += ST_THREADS) {
            const float l = to_float(row.data[i]);
            if (!row.counts(l)) continue;
            const double w = row.weight(l);
            const u64 m = row.mass(w);
            const int b = row.bin(l);
            part[3] += m;
            if (!(w < min_weight)) part[4] += m;
            if (b < w0.b0) part[0] += m;
            if (b < w1.b0) part[1] += m;
            if (b < w2.b0) part[2] += m;
            if ((w0.b0 <= b && b <= w0.b1) || (w1.b0 <= b && b <= w1.b1) || (w2.b0 <= b && b <= w2.b1)) {
                const unsigned p = atomicAdd(&sm.listed, 1u);
                if (p < ST_SORT) key[p] = st_key(l, row.first + i);
            }
        }
#pragma unroll
        for (int j = 0; j < 5; ++j) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) part[j] += __shfl_xor_sync(FULL, part[j], o);
            if (lane == 0) atomicAdd(&sm.part[j], part[j]);
        }
        s.sync();
    }
    // the first CTA reads the answers off the list
    if (rank == 0) {
        float lo[3], per[3];  // where each window begins, and its fine bins' width
        const int windows = quick ? 1 : sm.windows, each = ST_BINS / windows;
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            lo[j] = (float)sm.window[j].b0;
            per[j] = (float)each / (float)(sm.window[j].b1 - sm.window[j].b0 + 1);
        }
        auto window_of = [&](int b) {
            return (windows > 1 && b >= sm.window[1].b0 ? 1 : 0) + (windows > 2 && b >= sm.window[2].b0 ? 1 : 0);
        };
        const int n = s.collect([&](float l) {
            const int w = window_of(row.bin(l));
            const float at = (fminf(row.gap(l) * row.inv_width, (float)ST_BINS) - (w == 0 ? lo[0] : w == 1 ? lo[1] : lo[2])) *
                             (w == 0 ? per[0] : w == 1 ? per[1] : per[2]);
            return w * each + max(0, min((int)at, each - 1));
        });
        bool found = n <= ST_SORT;
        if (found) {
            if (tid < 3) sm.prefix[tid] = ~0ull, sm.starts[tid] = 0;
            if (!quick && tid < 5) {
                u64 m = 0;
                for (int c = 0; c < C; ++c) m += s.at(&sm, c)->part[tid];
                sm.delta[tid < 3 ? tid : 0] = 0;
                sm.warp_mass[tid] = m;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 5; ++j) part[j] = quick ? 0 : sm.warp_mass[j];
            __syncthreads();
            // `run` in a row to a thread
            const int run = (n + ST_THREADS - 1) / ST_THREADS;
            u64 w[ST_FOUR], sum = 0;
            int passing = 0, in[ST_FOUR];
#pragma unroll
            for (int j = 0; j < ST_FOUR; ++j) {
                const int i = tid * run + j;
                w[j] = 0, in[j] = 0;
                if (j < run && i < n) {
                    const float l = st_logit(key[i]);
                    const double x = row.weight(l);
                    w[j] = row.mass(x);
                    if (!(x < min_weight) && (!quick || i < top_k)) passing = i + 1;
                    in[j] = window_of(row.bin(l));
                }
                sum += w[j];
            }
            u64 upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 x = __shfl_up_sync(FULL, upto, o);
                if (lane >= o) upto += x;
            }
            passing = __reduce_max_sync(FULL, passing);
            if (lane == 31) sm.warp_mass[warp] = upto;
            if (lane == 0) sm.warp_count[warp] = passing;
            __syncthreads();
            u64 all = 0, at = upto - sum;
            for (int q = 0; q < ST_WARPS; ++q) {
                if (q < warp) at += sm.warp_mass[q];
                all += sm.warp_mass[q];
                passing = max(passing, (int)sm.warp_count[q]);
            }
            // sums in the list to sums in the row: windows begin with what stands before them
            u64 ends[ST_FOUR];
            u64 before = at;
#pragma unroll
            for (int j = 0; j < ST_FOUR; ++j) {
                const int i = tid * run + j;
                if (j < run && i < n && (i == 0 || in[j] != window_of(row.bin(st_logit(key[i - 1])))))
                    sm.delta[in[j]] = (quick ? 0 : part[in[j] == 0 ? 0 : in[j] == 1 ? 1 : 2]) - before, sm.starts[in[j]] = i;
                before += w[j];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < ST_FOUR; ++j) {
                const int i = tid * run + j;
                at += w[j];
                ends[j] = at + sm.delta[in[j]];
                if (j >= run || i >= n) ends[j] = 0, w[j] = 0;
                else {
                    const unsigned nth = (quick ? 0u : sm.before[in[j]]) + (unsigned)(i - sm.starts[in[j]]) + 1;
                    if (top_k > 0 && nth == (unsigned)top_k) sm.prefix[0] = ends[j];
                    if (quick && i + 1 == passing) sm.prefix[2] = ends[j];
                }
            }
            __syncthreads();
            u64 kept = sm.prefix[0];  // of the first k, if there are as many
            if (kept == ~0ull) kept = quick ? all : part[3];
            const u64 target = share_of(top_p, kept);
#pragma unroll
            for (int j = 0; j < ST_FOUR; ++j)
                if (top_p < 1.f && ends[j] - w[j] < target && target <= ends[j]) sm.prefix[1] = ends[j];
            __syncthreads();
            if (top_p < 1.f) {
                if (sm.prefix[1] == ~0ull) found = false;  // the window missed
                kept = min(kept, sm.prefix[1]);
            }
            kept = min(kept, quick ? sm.prefix[2] : min_weight > 0 ? part[4] : ~0ull);
            const u64 drawn = drawn_at(u, kept);
            int here = 0;
#pragma unroll
            for (int j = 0; j < ST_FOUR; ++j) {
                if (found && ends[j] - w[j] < drawn && drawn <= ends[j]) {
                    const u64 k = key[tid * run + j];
                    a.tokens[r] = (int64_t)(k & (ST_MAX_V - 1));
                    a.logprob[r] = (float)(row.score(st_logit(k)) - log((double)kept / ST_ONE));
                    here = 1;
                }
            }
            if (!quick) found = __syncthreads_or(here) != 0;
        }
        __syncthreads();
        if (tid < C) s.at(&sm, tid)->windows = found ? 0 : -1;
    }
    s.sync();  // no CTA leaves while another may read its shared memory
    if (sm.windows < 0) st_general<TX, C>(a, row, sm, count, r, rank, top_k, top_p, min_weight, u);
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
