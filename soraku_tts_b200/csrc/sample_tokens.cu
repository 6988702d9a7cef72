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
// Weights are whole multiples of 2^-44 of the largest, so sums are exact in any order and a
// draw does not depend on the order of atomics.  Each is within 2^-38 of its value (a table
// and a series in 64 bits, cut off behind its third power): borders of top-p and min-p
// are where they are to that.  What weighs less than 2^-45 of the largest weighs nothing,
// and all of it together (2^18 logits at most) is less than the last step 2^-24 of a
// uniform number.  A cluster of CTAs holds
// the row in shared memory, read once from the device's.
//
// With a top-k of up to 1280: the k-th largest of the threads' own largest logits (four each)
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
//
// Times: 64 rows of 2051 by top-k 50, top-p and min-p 7.4 us; one row of 151,936 by top-p
// and min-p 26; 128 rows of those by top-k 1000, top-p and min-p 36 (78 MB, 11.9 us at a
// copy's rate).  A small batch is bound by latency: code that runs once, barriers over
// the cluster, and the first CTA putting its list in order, where phases by half of
// its threads were no faster.  A large one by instructions a logit beside the stream.
// All are at 64 registers a thread: those for clusters keep 632 bytes of arrays in local
// memory and spill 176 to 260, those of short rows 132 to 156, streamed ones 72 at most.
#include <cooperative_groups.h>

#include <type_traits>

#include "int8_ops.cuh"

namespace skb {
namespace cg = cooperative_groups;

constexpr int ST_WARPS = 32;        // most of a CTA
constexpr int ST_BINS = 2048;
constexpr int ST_LIST = 512;        // logits of one gathered bin
constexpr int ST_SORT = 2048;       // logits that are gathered to be put in order
constexpr int ST_QUICK_K = 1280;
constexpr int ST_TURN = 16;         // logits that a thread reads at a time
constexpr int ST_OWN = 4;           // parts of a thread's logits that have a largest of their own
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

// Bins [b0, b1] about an answer; none: {-1, -1}.
struct Window {
    int b0, b1;
};

struct SampleShared {
    float top, low;            // this CTA's
    Window window[3];          // apart and in order; written by the first CTA, to all
    int go_on;                 // 1: the list has the answer, 0: st_general has to
    u64 part[5];               // this CTA's masses: before each window, all, passing min-p
    unsigned before[3];        // logits before each window
    unsigned listed;           // logits that this CTA has listed
    int few[3];                // logits of one fine bin, for each question
    int answer[3];
    int hit[3];                // the fine bin that a sum reaches its target in
    u64 hit_mass[3];
    unsigned hit_count[3];
    Found reached[3];
    float approx[2];
    u64 mass, mass_min_p;      // this CTA's totals
    unsigned count;
    u64 lo, hi;                // smallest and largest key of a bin, this CTA's
    Bin bin;                   // written by the CTA that found it, to all
    Found found;
    u64 warp_mass[ST_WARPS];
    unsigned warp_count[ST_WARPS];
    unsigned red[2][ST_WARPS];
    u64 warp_part[5][ST_WARPS];
    double power[128];         // 2^(i / 128)
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

// This CTA's part of a row: 16-byte vectors, in shared memory (HELD) or the
// device's; what lies before the first logit or behind the last reads as -infinity.
template <class TX, int NT, bool HELD>
struct Row {
    static constexpr int VN = Vec<TX>::N;
    const TX* data;  // on 16 bytes
    const double* power;
    int off, n, first;  // the first logit's place, how many there are, and its index in the row
    float top, cut, inv_width;
    double inv_t, scale;  // 1 / T, and 128 log2(e) / T
    // how far below the largest; beyond `cut`: without weight
    __device__ __forceinline__ float gap(float l) const { return l == top ? 0.f : top - l; }
    __device__ __forceinline__ bool counts(float l) const { return gap(l) <= cut; }
    // along the bins, [0, ST_BINS - 1], of what counts; and the nearest one, by an
    // addition that leaves it in the low bits
    __device__ __forceinline__ float place(float g) const { return g * inv_width; }
    __device__ __forceinline__ int bin_at(float g) const { return __float_as_int(fmaf(g, inv_width, 8388608.f)) & 4095; }
    __device__ __forceinline__ int bin(float l) const { return bin_at(gap(l)); }
    __device__ __forceinline__ double score(float l) const { return l == top ? 0.0 : ((double)l - (double)top) * inv_t; }
    // exp((l - top) / T) 2^44 for a logit that counts: 2^(n / 128) from a table and the
    // power series of what is left, |x| <= log(2) / 256, to its third power (the fourth
    // is 2^-38).  The exponent is at least 44 - 48: no underflow.  top is finite.
    __device__ __forceinline__ double weight(float l) const {
        constexpr double MAGIC = 6755399441055744.0, LN = 0.69314718055994531 / 128;
        const double y = ((double)l - (double)top) * scale;
        const double m = y + MAGIC;
        const int n = __double2loint(m);
        const double x = y - (m - MAGIC);
        const double p = fma(fma(fma(LN * LN * LN / 6, x, LN * LN / 2), x, LN), x, 1.0) * power[n & 127];
        return __hiloint2double(__double2hiint(p) + (((n >> 7) + 44) << 20), __double2loint(p));
    }
    // rounded by adding 2^52: weights are up to 2^44
    __device__ __forceinline__ static double whole(double weight) { return __dadd_rn(__dadd_rn(weight, 4503599627370496.0), -4503599627370496.0); }
    __device__ __forceinline__ u64 mass(float l) const {
        return l == top ? (u64)ST_ONE : (u64)__double_as_longlong(weight(l) + 4503599627370496.0) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ double safe_weight(float l) const { return l == top ? ST_ONE : weight(l); }
    // f(logits, index of the first) for B vectors from this thread's one at i on.
    template <int B, class F>
    __device__ __forceinline__ void turn(int i, F f) const {
        const int end = off + n;
        Vec<TX> v[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int at = i + b * NT * VN;
            if (HELD ? at < end : at >= off && at + VN <= end) {
                if (HELD) v[b].raw = *reinterpret_cast<const uint4*>(data + at);
                else v[b].raw = __ldcg(reinterpret_cast<const uint4*>(data + at));
            } else {
#pragma unroll
                for (int j = 0; j < VN; ++j)
                    v[b].e[j] = !HELD && at + j >= off && at + j < end ? read(data + at + j) : from_float<TX>(-INFINITY);
            }
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            float l[VN];
            v[b].get(l);
            f(l, first + i + b * NT * VN - off);
        }
    }
    // f for every vector, B of them read at a time.
    template <int B, class F>
    __device__ __forceinline__ void each(F f) const {
        for (int i = threadIdx.x * VN; i < off + n; i += B * NT * VN) turn<B>(i, f);
    }
};

template <class TX, int C, int NT, bool HELD>
struct Sampler {
    static constexpr int VN = Vec<TX>::N, WARPS = NT / 32;
    static constexpr int PER = ST_BINS / NT;   // bins of a thread, and listed logits
    static constexpr int SHARE = ST_BINS / C;  // bins that a CTA adds up for the cluster
    using R = Row<TX, NT, HELD>;

    SampleShared& sm;
    unsigned* count;               // bins of this CTA's logits
    unsigned *low, *high;          // their masses, in two words
    u64* key;                      // this CTA's list, in the place of the masses
    unsigned* pre_count;           // of this CTA's share of the bins, cluster-wide: what stands before each
    u64* pre_mass;
    const R& row;
    int tid, rank;
    u64 all_mass, mass_min_p;
    unsigned all_count;
    bool fresh;  // the bins hold the whole row

    __device__ __forceinline__ Sampler(SampleShared& sm, unsigned char* raw, const R& row, int rank)
        : sm(sm), row(row), tid(threadIdx.x), rank(rank), all_mass(0), mass_min_p(0), all_count(0), fresh(false) {
        count = reinterpret_cast<unsigned*>(raw);
        low = count + ST_BINS, high = low + ST_BINS;
        key = reinterpret_cast<u64*>(low);
        pre_mass = reinterpret_cast<u64*>(high + ST_BINS);
        pre_count = reinterpret_cast<unsigned*>(pre_mass + SHARE + 2);
    }
    static constexpr int BYTES = 3 * ST_BINS * 4 + (SHARE + 2) * 8 + (SHARE + 4) * 4;  // a multiple of 16

    template <class T>
    __device__ __forceinline__ T* at(T* p, int r) const { return C == 1 ? p : cg::this_cluster().map_shared_rank(p, r); }
    __device__ __forceinline__ void sync() const {
        if (C == 1) __syncthreads();
        else cg::this_cluster().sync();
    }
    __device__ __forceinline__ void clear() {
        for (int i = tid; i < 3 * ST_BINS / 4; i += NT) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void add(int b, u64 m) {
        atomicAdd(&count[b], 1u);
        if (m == 0) return;
        const unsigned lo = (unsigned)m, old = atomicAdd(&low[b], lo);
        const unsigned hi = (unsigned)(m >> 32) + (old + lo < old ? 1u : 0u);
        if (hi) atomicAdd(&high[b], hi);
    }
    __device__ __forceinline__ u64 bin_mass(int b) const { return ((u64)high[b] << 32) + low[b]; }
    // What stands before this thread in the CTA, and all of it.
    template <class A, class B>
    __device__ __forceinline__ void scan(A& n, B& m, A& all_n, B& all_m, A* warp_n, B* warp_m) const {
        const int lane = tid & 31, warp = tid >> 5;
        auto in_warp = [&](A& x, B& y) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const A p = __shfl_up_sync(FULL, x, o);
                const B q = __shfl_up_sync(FULL, y, o);
                if (lane >= o) x += p, y += q;
            }
        };
        const A own_n = n;
        const B own_m = m;
        in_warp(n, m);
        if (lane == 31) warp_n[warp] = n, warp_m[warp] = m;
        __syncthreads();
        A wn = lane < WARPS ? warp_n[lane] : A(0);
        B wm = lane < WARPS ? warp_m[lane] : B(0);
        in_warp(wn, wm);
        all_n = __shfl_sync(FULL, wn, 31), all_m = __shfl_sync(FULL, wm, 31);
        const A pn = __shfl_sync(FULL, wn, (warp + 31) & 31);
        const B pm = __shfl_sync(FULL, wm, (warp + 31) & 31);
        n = n - own_n + (warp > 0 ? pn : A(0)), m = m - own_m + (warp > 0 ? pm : B(0));
        __syncthreads();  // the arrays may be used again
    }

    // ---- the list ------------------------------------------------------
    __device__ __forceinline__ void list(float l, int index) {
        const unsigned p = atomicAdd(&sm.listed, 1u);
        if (p < ST_SORT) key[p] = st_key(l, index);
    }

    // The first CTA: the answers from everybody's lists.  The listed logits are
    // those of `windows` windows of bins; part: the masses before them, of all, and of
    // what min-p lets stay (known, but for a list that has the first k).
    // False if the list does not have them.
    __device__ __forceinline__ bool answer(int windows, bool first_k, int top_k, float top_p, double min_weight, float u, u64 (&part)[5],
                                           int64_t* token, float* logprob) {
        unsigned from[C], n = 0;
        const unsigned theirs = (tid & 31) < C ? *at(&sm.listed, tid & 31) : 0;
#pragma unroll
        for (int r = 0; r < C; ++r) from[r] = __shfl_sync(FULL, theirs, r);
#pragma unroll
        for (int r = 0; r < C; ++r) {
            const unsigned x = from[r];
            from[r] = n, n += x;
        }
        if (n > ST_SORT) return false;
        const Window w0 = sm.window[0], w1 = sm.window[1], w2 = sm.window[2];
        const int each = windows == 1 ? ST_BINS : windows == 2 ? ST_BINS / 2 : ST_BINS / 3;
        const float per0 = (float)each / (float)(w0.b1 - w0.b0 + 1), per1 = (float)each / (float)(w1.b1 - w1.b0 + 1),
                    per2 = (float)each / (float)(w2.b1 - w2.b0 + 1);
        u64 k[PER], m[PER], passing = 0;
        int fine[PER], in[PER];
        if (tid < 3) sm.few[tid] = 0, sm.hit[tid] = -1, sm.reached[tid].index = -1;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const unsigned i = j * NT + tid;
            k[j] = ~0ull, m[j] = 0, fine[j] = -1, in[j] = 0;
            if (i < n) {
                u64* list = at(key, 0);
                unsigned base = 0;
#pragma unroll
                for (int r = 1; r < C; ++r)
                    if (i >= from[r]) list = at(key, r), base = from[r];
                k[j] = list[i - base];
                const float l = st_logit(k[j]), g = top_gap(l), x = row.place(g);
                const double w = row.safe_weight(l);
                m[j] = (u64)R::whole(w);
                if (!(w < min_weight)) passing += m[j];
                const int b = row.bin_at(g);
                in[j] = (windows > 1 && b >= w1.b0 ? 1 : 0) + (windows > 2 && b >= w2.b0 ? 1 : 0);
                const float f = (x + 0.5f - (float)(in[j] == 0 ? w0.b0 : in[j] == 1 ? w1.b0 : w2.b0)) * (in[j] == 0 ? per0 : in[j] == 1 ? per1 : per2);
                fine[j] = in[j] * each + max(0, min((int)f, each - 1));
            }
        }
        const bool small = n <= NT / 4;
        u64 all = 0;
        unsigned all_n = n;
        // small: of this thread's logit, else of its fine bins: what stands before, and how much it is
        u64 before[PER], size[PER];
        unsigned count_before[PER], number[PER];
        __syncthreads();
        if (small) {
            // four threads a logit add up what stands before it in its window
            if (tid < (int)n) key[tid] = k[0], key[NT / 4 + tid] = m[0], count[tid] = in[0];
            __syncthreads();
            const int i = tid >> 2;
            u64 mass = 0, mine = 0;
            unsigned cnt = 0;
            int q = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) k[j] = ~0ull, m[j] = 0, fine[j] = -1, before[j] = 0, size[j] = 0, count_before[j] = 0, number[j] = 0;
            if (i < (int)n) {
                mine = key[i], q = count[i];
                for (int j = tid & 3; j < (int)n; j += 4) {
                    const u64 w = key[NT / 4 + j];
                    all += w;
                    if (key[j] < mine && (int)count[j] == q) mass += w, cnt += 1;
                }
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                mass += __shfl_xor_sync(FULL, mass, o), cnt += __shfl_xor_sync(FULL, cnt, o);
                all += __shfl_xor_sync(FULL, all, o);
            }
            if (i < (int)n && (tid & 3) == 0) {
                k[0] = mine, m[0] = key[NT / 4 + i], fine[0] = i;
                before[0] = mass, size[0] = m[0], count_before[0] = cnt, number[0] = 1;
                if (!first_k) before[0] += q == 0 ? part[0] : q == 1 ? part[1] : part[2], count_before[0] += sm.before[q];
            }
            // the sum of all is known where there is a logit: in the first warp
            if (tid == 0) sm.warp_mass[0] = all;
            __syncthreads();
            all = sm.warp_mass[0];
            __syncthreads();
        } else {
            clear();
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (fine[j] >= 0) add(fine[j], m[j]);
            __syncthreads();
            // sums along the fine bins; each window begins with what stands before it
            unsigned cnt = 0;
            u64 mass = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                number[j] = count[tid * PER + j], size[j] = bin_mass(tid * PER + j);
                cnt += number[j], mass += size[j];
            }
            scan(cnt, mass, all_n, all, sm.warp_count, sm.warp_mass);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                before[j] = mass, count_before[j] = cnt;
                mass += size[j], cnt += number[j];
            }
            if (!first_k) {
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int b = tid * PER + j;
                    if (b % each == 0 && b / each < 3) sm.part[b / each] = before[j], sm.answer[b / each] = (int)count_before[j];
                }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int q = min((tid * PER + j) / each, windows - 1);
                    before[j] += (q == 0 ? part[0] : q == 1 ? part[1] : part[2]) - sm.part[q];
                    count_before[j] += sm.before[q] - (unsigned)sm.answer[q];
                }
            }
        }
        if (first_k && min_weight > 0) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) passing += __shfl_xor_sync(FULL, passing, o);
            if ((tid & 31) == 0) sm.warp_part[0][tid >> 5] = passing;
            __syncthreads();
            passing = (tid & 31) < WARPS ? sm.warp_part[0][tid & 31] : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) passing += __shfl_xor_sync(FULL, passing, o);
        }
        u64 kept = first_k ? all : part[3];
        const u64 allowed = first_k ? passing : part[4];
        // where top-k ends, where top-p does, and what is drawn
#pragma unroll 1
        for (int question = 0; question < 3; ++question) {
            u64 target;
            if (question == 0) {
                if (top_k <= 0 || (unsigned)top_k >= (first_k ? all_n : all_count)) continue;
                target = (u64)top_k;
            } else if (question == 1) {
                if (!(top_p < 1.f)) continue;
                target = share_of(top_p, kept);
            } else {
                if (min_weight > 0) kept = min(kept, allowed);
                target = drawn_at(u, kept);
            }
            const bool by_count = question == 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const u64 start = by_count ? (u64)count_before[j] : before[j], extent = by_count ? (u64)number[j] : size[j];
                if (start < target && target <= start + extent) {
                    if (small) sm.reached[question] = {before[j] + size[j], st_logit(k[j]), (int)(k[j] & (ST_MAX_V - 1))};
                    else sm.hit[question] = tid * PER + j, sm.hit_mass[question] = before[j], sm.hit_count[question] = count_before[j];
                }
            }
            __syncthreads();
            if (!small) {
                const int b = sm.hit[question];
                if (b < 0) return false;  // the windows missed
#pragma unroll
                for (int j = 0; j < PER; ++j)
                    if (fine[j] == b) {
                        const int i = atomicAdd(&sm.few[question], 1);
                        if (i < ST_SORT / 2) key[i] = k[j], key[ST_SORT / 2 + i] = m[j];
                    }
                __syncthreads();
                const int few = sm.few[question];
                if (few > ST_SORT / 2) return false;
                for (int i = tid; i < few; i += NT) {
                    const u64 mine = key[i], w = key[ST_SORT / 2 + i];
                    u64 mass = sm.hit_mass[question], cnt = sm.hit_count[question];
                    for (int j = 0; j < few; ++j)
                        if (key[j] < mine) cnt += 1, mass += key[ST_SORT / 2 + j];
                    if (by_count ? cnt + 1 == target : mass < target && target <= mass + w)
                        sm.reached[question] = {mass + w, st_logit(mine), (int)(mine & (ST_MAX_V - 1))};
                }
                __syncthreads();
            }
            if (sm.reached[question].index < 0) return false;
            if (question < 2) kept = sm.reached[question].mass;
        }
        if (tid == 0) {
            *token = sm.reached[2].index;
            *logprob = (float)(row.score(sm.reached[2].logit) - log((double)kept / ST_ONE));
        }
        return true;
    }
    __device__ __forceinline__ float top_gap(float l) const { return row.gap(l); }

    // The first CTA: windows about where the answers will be, to all.  total: its bins'
    // counts; step: a bin's width by T.  How many windows, 0: no list can hold them.
    __device__ __forceinline__ int choose_windows(const unsigned* total, float step, int top_k, float top_p, float min_p, float u) {
        // mass by the weight at the middle of each bin
        unsigned c[PER], cnt = 0, everyone;
        float m[PER], mass = 0.f, all;
        float* warp_mass = reinterpret_cast<float*>(sm.red[0]);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int b = tid * PER + j;
            c[j] = total[b];
            m[j] = b == 0 ? (float)c[j] : (float)c[j] * __expf(-(float)b * step);
            cnt += c[j], mass += m[j];
        }
        if (tid < 3) sm.answer[tid] = -1;
        if (tid == 3) sm.approx[0] = sm.approx[1] = -1.f;
        scan(cnt, mass, everyone, all, sm.warp_count, warp_mass);
        all_count = everyone;
        unsigned cb[PER + 1];
        float mb[PER + 1];
        cb[0] = cnt, mb[0] = mass;
#pragma unroll
        for (int j = 0; j < PER; ++j) cb[j + 1] = cb[j] + c[j], mb[j + 1] = mb[j] + m[j];
        const bool with_k = top_k > 0 && (unsigned)top_k < everyone;
        // the last bin that min-p lets stay
        const float edge = min_p > 0.f ? fminf(-__logf(fminf(min_p, 1.f)) / step + 0.5f, 3e4f) : 3e4f;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int b = tid * PER + j;
            if (with_k && cb[j] < (unsigned)top_k && (unsigned)top_k <= cb[j + 1]) sm.answer[2] = b, sm.approx[0] = 0.5f * (mb[j] + mb[j + 1]);
            if ((int)edge == b) sm.approx[1] = mb[j + 1];
        }
        __syncthreads();
        float kept = with_k ? sm.approx[0] : all;
        auto locate = [&](int which, float target) {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (c[j] > 0 && mb[j] <= target && target < mb[j + 1]) sm.answer[which] = tid * PER + j;
        };
        const bool with_p = top_p < 1.f;
        if (with_p) {
            kept *= fmaxf(top_p, 0.f);
            locate(1, kept);
        }
        if (sm.approx[1] >= 0.f) kept = fminf(kept, sm.approx[1]);
        locate(0, kept * fminf(fmaxf(u, 0.f), 1.f));
        __syncthreads();
        // in order: what is drawn, top-p's end, top-k's
        const int at_k = sm.answer[2];
        int at_p = sm.answer[1], at_d = sm.answer[0];
        if (with_p && at_p < 0) at_p = at_k >= 0 ? at_k : ST_BINS - 1;  // rounding of the sums
        if (at_d < 0) at_d = at_p >= 0 ? at_p : at_k >= 0 ? at_k : ST_BINS - 1;
        // 384 logits to each side, or as many as the list has room for
#pragma unroll 1
        for (unsigned room = 384;; room = room > 100 ? room / 4 : 0) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int b = tid * PER + j;
                if (b == at_d) sm.window[0] = {b, b}, sm.before[0] = cb[j], sm.part[0] = cb[j + 1];
                if (b == at_p) sm.window[1] = {b, b}, sm.before[1] = cb[j], sm.part[1] = cb[j + 1];
            }
            if (tid == 0) sm.listed = 0;
            __syncthreads();
            const unsigned d0 = sm.before[0], d1 = (unsigned)sm.part[0], p0 = sm.before[1], p1 = (unsigned)sm.part[1];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int b = tid * PER + j;
                if (b < at_d && d0 - cb[j] <= room) atomicMin(&sm.window[0].b0, b);
                if (b > at_d && cb[j + 1] - d1 <= room) atomicMax(&sm.window[0].b1, b);
                if (with_p && b < at_p && p0 - cb[j] <= room) atomicMin(&sm.window[1].b0, b);
                if (with_p && b > at_p && cb[j + 1] - p1 <= room) atomicMax(&sm.window[1].b1, b);
            }
            __syncthreads();
            // those that touch become one
            const Window none = {-1, -1};
            Window w0 = sm.window[0], w1 = none, w2 = none;
            if (with_p) {
                const Window p = sm.window[1];
                if (p.b0 <= w0.b1 + 1) w0.b0 = min(w0.b0, p.b0), w0.b1 = max(w0.b1, p.b1);
                else w1 = p;
            }
            if (at_k >= 0) {
                const Window k = {at_k, at_k};
                Window& last = w1.b0 >= 0 ? w1 : w0;
                if (k.b0 <= last.b1 + 1) last.b0 = min(last.b0, k.b0), last.b1 = max(last.b1, k.b1);
                else if (w1.b0 >= 0) w2 = k;
                else w1 = k;
            }
            __syncthreads();
            // logits in them, and before them
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int b = tid * PER + j;
                if (b == w0.b0) sm.before[0] = cb[j], atomicSub(&sm.listed, cb[j]);
                if (b == w1.b0) sm.before[1] = cb[j], atomicSub(&sm.listed, cb[j]);
                if (b == w2.b0) sm.before[2] = cb[j], atomicSub(&sm.listed, cb[j]);
                if (b == w0.b1) atomicAdd(&sm.listed, cb[j + 1]);
                if (b == w1.b1) atomicAdd(&sm.listed, cb[j + 1]);
                if (b == w2.b1) atomicAdd(&sm.listed, cb[j + 1]);
            }
            __syncthreads();
            const unsigned listed = sm.listed;
            if (listed > ST_SORT && room > 0) continue;
            const int windows = listed > ST_SORT ? 0 : 1 + (w1.b0 >= 0) + (w2.b0 >= 0);
            if (tid < C) {
                SampleShared* peer = at(&sm, tid);
                peer->window[0] = w0, peer->window[1] = w1, peer->window[2] = w2;
                peer->go_on = windows > 0;
            }
            __syncthreads();
            if (tid == 0) sm.listed = 0;
            return windows;
        }
    }

    // ---- bins with masses, again and again -----------------------------
    // Every CTA's bins into running sums over the cluster's, each CTA a share of the bins.
    // passing: this thread's mass of what min-p lets stay.
    __device__ __forceinline__ void total(u64 passing) {
        sync();
        constexpr int EACH = SHARE > NT ? SHARE / NT : 1;
        const int b0 = tid * EACH;
        unsigned n = 0, cn[EACH];
        u64 m = 0, cm[EACH];
        if (b0 < SHARE) {
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
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
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) passing += __shfl_xor_sync(FULL, passing, o);
        if ((tid & 31) == 0 && passing) atomicAdd(&sm.mass_min_p, passing);
        unsigned all_n;
        u64 all_m;
        scan(n, m, all_n, all_m, sm.warp_count, sm.warp_mass);
        if (tid == 0) sm.count = all_n, sm.mass = all_m;
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
            for (int j = 0; j < EACH; ++j) {
                pre_count[b0 + j] = before + n + cn[j];
                pre_mass[b0 + j] = before_mass + m + cm[j];
            }
        }
        if (tid == 0) pre_count[SHARE] = before + all_n, pre_mass[SHARE] = before_mass + all_m;
        __syncthreads();
    }
    // The whole row's bins.
    __device__ __forceinline__ void fill(double min_weight) {
        __syncthreads();
        clear();
        __syncthreads();
        u64 passing = 0;
        row.template each<1>([&](const float (&l)[VN], int) {
#pragma unroll
            for (int j = 0; j < VN; ++j)
                if (row.counts(l[j])) {
                    const u64 m = row.mass(l[j]);
                    add(row.bin(l[j]), m);
                    if (!(row.safe_weight(l[j]) < min_weight)) passing += m;
                }
        });
        total(passing);
        fresh = true;
    }

    // The bin in which the count or the mass reaches `target` (1 to the whole).
    // Nothing is listed any more.
    __device__ __forceinline__ Bin find(bool by_count, u64 target, u64 mass_before, unsigned count_before) {
        if (tid == 0) sm.listed = 0;
        for (int i = tid; i < SHARE; i += NT) {
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
            row.template each<1>([&](const float (&l)[VN], int i) {
#pragma unroll
                for (int j = 0; j < VN; ++j)
                    if (inside(l[j], i + j)) a = min(a, st_key(l[j], i + j)), z = max(z, st_key(l[j], i + j));
            });
            if (tid == 0) sm.lo = ~0ull, sm.hi = 0;
            clear();
            __syncthreads();
            if (a <= z) {
                atomicMin(&sm.lo, a);
                atomicMax(&sm.hi, z);
            }
            sync();
            a = ~0ull, z = 0;
#pragma unroll
            for (int r = 0; r < C; ++r) a = min(a, *at(&sm.lo, r)), z = max(z, *at(&sm.hi, r));
            const int width = 64 - __clzll((long long)(z - a)), shift = max(0, width - 11);
            row.template each<1>([&](const float (&l)[VN], int i) {
#pragma unroll
                for (int j = 0; j < VN; ++j)
                    if (inside(l[j], i + j)) add((int)((st_key(l[j], i + j) - a) >> shift), row.mass(l[j]));
            });
            total(0);
            fresh = false;
            b = find(by_count, target, b.mass_before, b.count_before);
            lo = a + ((u64)b.bin << shift);
            hi = lo + ((1ull << shift) - 1);
        }
        // into the first CTA's list
        unsigned* listed = at(&sm.listed, 0);
        u64* keys = at(key, 0);
        row.template each<1>([&](const float (&l)[VN], int i) {
#pragma unroll
            for (int j = 0; j < VN; ++j)
                if (inside(l[j], i + j)) {
                    const unsigned p = atomicAdd(listed, 1u);
                    if (p < ST_LIST) keys[p] = st_key(l[j], i + j);
                }
        });
        sync();
        if (rank == 0) {
            const int n = min((int)sm.listed, ST_LIST);
            u64* weight = key + ST_LIST;
            for (int i = tid; i < n; i += NT) weight[i] = row.mass(st_logit(key[i]));
            __syncthreads();
            for (int i = tid; i < n; i += NT) {
                const u64 mine = key[i], w = weight[i];
                u64 mass = b.mass_before, cnt = b.count_before;
                for (int j = 0; j < n; ++j)
                    if (key[j] < mine) cnt += 1, mass += weight[j];
                if (by_count ? cnt + 1 == target : mass < target && target <= mass + w) {
                    const Found f = {mass + w, st_logit(mine), (int)(mine & (ST_MAX_V - 1))};
                    for (int r = 0; r < C; ++r) *at(&sm.found, r) = f;
                }
            }
        }
        sync();
        const Found f = sm.found;
        __syncthreads();
        return f;
    }
};

// The row by bins with their masses, binned again as often as it takes.
template <class TX, int C, int NT, bool HELD>
__device__ __noinline__ void st_general(Row<TX, NT, HELD> row, SampleShared& sm, unsigned char* raw, int rank, int top_k, float top_p,
                                        double min_weight, float u, int64_t* token, float* logprob) {
    Sampler<TX, C, NT, HELD> s(sm, raw, row, rank);
    s.sync();  // whatever was being read in this CTA's shared memory has been
    s.fill(min_weight);
    u64 kept = s.all_mass;
    const u64 passing = min_weight > 0 ? s.mass_min_p : kept;
    Found f;
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
        *token = f.index;
        *logprob = (float)(row.score(f.logit) - log((double)kept / ST_ONE));
    }
    s.sync();
}

template <class TX, int C, int NT, bool HELD>
__global__ void __launch_bounds__(NT, 1024 / NT) sample_kernel(const SampleArgs a) {
    using S = Sampler<TX, C, NT, HELD>;
    constexpr int VN = Vec<TX>::N, WARPS = NT / 32;
    extern __shared__ __align__(16) unsigned char st_raw[];
    __shared__ SampleShared sm;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / C;
    const int rank = C == 1 ? 0 : (int)cg::this_cluster().block_rank();
    Row<TX, NT, HELD> row;
    S s(sm, st_raw, row, rank);
    if (tid < 128) sm.power[tid] = exp2(tid / 128.0);
    if (tid == 128) sm.listed = 0, sm.mass_min_p = 0, sm.go_on = 1;
    s.clear();

    pdl_wait();
    pdl_trigger();
    const float temperature = a.temperature ? __ldcg(a.temperature + r) : a.temperature0;
    float top_p = a.top_p ? __ldcg(a.top_p + r) : a.top_p0;
    float min_p = a.min_p ? __ldcg(a.min_p + r) : a.min_p0;
    int top_k = a.top_k ? __ldcg(a.top_k + r) : a.top_k0;
    const float u = __ldcg(a.uniform + r);

    row.power = sm.power;
    row.first = rank * a.slice;
    row.n = max(0, min(a.slice, a.V - row.first));
    float mine[ST_OWN], low = INFINITY;  // largest of this thread's parts, and its smallest that is finite
#pragma unroll
    for (int q = 0; q < ST_OWN; ++q) mine[q] = -INFINITY;
    {
        const TX* src = static_cast<const TX*>(a.logits) + (long long)r * a.ld + row.first;
        row.off = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(TX));
        src -= row.off;
        TX* held = reinterpret_cast<TX*>(st_raw + S::BYTES);
        float* largest = reinterpret_cast<float*>(st_raw + S::BYTES);  // of each thread's turns, where the row is not held
        row.data = HELD ? held : src;
        constexpr int B = ST_TURN / VN;
        const int end = row.off + row.n;
        for (int i = tid * VN, turn = 0; i < end; i += B * NT * VN, ++turn) {
            float most = -INFINITY;
            Vec<TX> v[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int at = i + b * NT * VN;
                if (at >= row.off && at + VN <= end) {
                    v[b].raw = HELD ? __ldcs(reinterpret_cast<const uint4*>(src + at)) : __ldcg(reinterpret_cast<const uint4*>(src + at));
                } else {
#pragma unroll
                    for (int j = 0; j < VN; ++j)
                        v[b].e[j] = at + j >= row.off && at + j < end ? read(src + at + j) : from_float<TX>(-INFINITY);
                }
            }
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int at = i + b * NT * VN;
                if (HELD && at < end) *reinterpret_cast<uint4*>(held + at) = v[b].raw;
                float l[VN];
                v[b].get(l);
#pragma unroll
                for (int j = 0; j < VN; ++j) {
                    asm("max.NaN.f32 %0, %0, %1;" : "+f"(mine[(b * VN + j) * ST_OWN / (B * VN)]) : "f"(l[j]));
                    low = fminf(low, l[j] > -INFINITY ? l[j] : INFINITY);
                    most = fmaxf(most, l[j]);
                }
            }
            if (!HELD) largest[turn * NT + tid] = most;
        }
    }
    // the order of numbers as that of whole ones, NaN (max.NaN gives the positive one) on top
    auto up = [](float x) {
        const unsigned b = __float_as_uint(x);
        return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    };
    auto down = [](unsigned b) { return __uint_as_float(b ^ ((b >> 31) ? 0x80000000u : 0xffffffffu)); };
    {
        float most = mine[0];
#pragma unroll
        for (int q = 1; q < ST_OWN; ++q) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(mine[q]));
        const unsigned h = __reduce_max_sync(FULL, up(most)), l = __reduce_min_sync(FULL, up(low));
        if (lane == 0) sm.red[0][warp] = h, sm.red[1][warp] = l;
    }
    __syncthreads();
    float top = down(__reduce_max_sync(FULL, lane < WARPS ? sm.red[0][lane] : 0u));
    low = down(__reduce_min_sync(FULL, lane < WARPS ? sm.red[1][lane] : 0xffffffffu));
    if (C > 1) {
        if (tid == 0) sm.top = top, sm.low = low;
        s.sync();
        // a lane for each CTA: a peer's memory is asked once a warp
        top = down(__reduce_max_sync(FULL, lane < C ? up(s.at(&sm, lane)->top) : 0u));
        low = down(__reduce_min_sync(FULL, lane < C ? up(s.at(&sm, lane)->low) : 0xffffffffu));
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
    row.scale = 184.66496523378731 * row.inv_t;
    row.cut = (float)fmin(32.0 * t, 3e38);
    const float span = fmaxf(fminf(row.cut, top == low ? 1.f : top - low), 1e-30f);
    row.inv_width = (float)(ST_BINS - 1) / span;
    const double min_weight = min_p > 0.f ? (double)fminf(min_p, 1.f) * ST_ONE : 0.0;
    const bool quick = top_k > 0 && top_k <= ST_QUICK_K;

    if (top == INFINITY) {  // which cannot be subtracted
        st_general<TX, C, NT, HELD>(row, sm, st_raw, rank, top_k, top_p, min_weight, u, a.tokens + r, a.logprob + r);
        return;
    }
    u64 part[5] = {};  // masses before each window, of all, and of what min-p lets stay
    int windows = 1;
    if (quick) {
        // the bin of the k-th of the threads' largest: all that is in later bins
        // comes behind the first k
#pragma unroll
        for (int q = 0; q < ST_OWN; ++q)
            if (top - mine[q] <= row.cut) atomicAdd(s.at(&s.count[row.bin_at(top - mine[q])], 0), 1u);
        s.sync();
        if (rank == 0) {
            unsigned c[S::PER], at = 0, zero = 0, all, none;
#pragma unroll
            for (int j = 0; j < S::PER; ++j) c[j] = s.count[tid * S::PER + j], at += c[j];
            if (tid == 0) sm.answer[0] = ST_BINS - 1;
            s.scan(at, zero, all, none, sm.warp_count, sm.red[0]);
#pragma unroll
            for (int j = 0; j < S::PER; ++j) {
                if (at < (unsigned)top_k && (unsigned)top_k <= at + c[j]) sm.answer[0] = tid * S::PER + j;
                at += c[j];
            }
            __syncthreads();
            if (tid < C) s.at(&sm, tid)->window[0] = {0, sm.answer[0]};
        }
        s.sync();
        const int last = sm.window[0].b1;
        // bins up to `last` reach half a bin behind it; with room for rounding, that is as
        // far as a vector's largest has to be looked at
        const float reach = last == ST_BINS - 1 ? -INFINITY : top - ((float)last + 1.f) * (span / (ST_BINS - 1)) - fabsf(top) * 1e-6f;
        auto see = [&](const float (&l)[VN], int i) {
            float most = l[0];
#pragma unroll
            for (int j = 1; j < VN; ++j) most = fmaxf(most, l[j]);
            if (most < reach) return;
#pragma unroll
            for (int j = 0; j < VN; ++j)
                if (top - l[j] <= row.cut && row.bin_at(top - l[j]) <= last) s.list(l[j], i + j);
        };
        if constexpr (HELD) {
            row.template each<4>(see);
        } else {
            // a thread reads again only the turns that reach so far: one in eight for the
            // first 1000 of 151,936
            const float* largest = reinterpret_cast<const float*>(st_raw + S::BYTES);
            constexpr int STEP = ST_TURN * NT;
            static_assert((ST_MAX_V + 8) / STEP + 1 <= 32, "a thread's turns as bits");
            unsigned far = 0;
            for (int i = tid * VN, turn = 0; i < row.off + row.n; i += STEP, ++turn)
                if (!(largest[turn * NT + tid] < reach)) far |= 1u << turn;
            // each lane its next one: a warp goes round as often as its busiest lane has any
            for (; far != 0; far &= far - 1) row.template turn<ST_TURN / VN>(tid * VN + (__ffs(far) - 1) * STEP, see);
        }
        s.sync();
    } else {
        row.template each<4>([&](const float (&l)[VN], int) {
#pragma unroll
            for (int j = 0; j < VN; ++j)
                if (top - l[j] <= row.cut) atomicAdd(&s.count[row.bin_at(top - l[j])], 1u);
        });
        s.sync();
        // each CTA adds up a share of the bins, into the first one's list
        unsigned* total = reinterpret_cast<unsigned*>(s.key);
        for (int i = tid; i < S::SHARE; i += NT) {
            unsigned n = 0;
#pragma unroll
            for (int c = 0; c < C; ++c) n += *s.at(&s.count[rank * S::SHARE + i], c);
            s.at(total, 0)[rank * S::SHARE + i] = n;
        }
        s.sync();
        if (rank == 0) {
            windows = s.choose_windows(total, (float)((double)(span / (ST_BINS - 1)) * row.inv_t), top_k, top_p, min_p, u);
        }
        s.sync();
        if (!sm.go_on) {
            st_general<TX, C, NT, HELD>(row, sm, st_raw, rank, top_k, top_p, min_weight, u, a.tokens + r, a.logprob + r);
            return;
        }
        const Window w0 = sm.window[0], w1 = sm.window[1], w2 = sm.window[2];
        // a thread's masses add up to 2^52 at most, whole numbers, as doubles
        double sum[5] = {};
        auto weigh = [&](auto three) {
            row.template each<1>([&](const float (&l)[VN], int i) {
                double m[VN], w[VN];
                int b[VN];
#pragma unroll
                for (int j = 0; j < VN; ++j) {
                    const float g = top - l[j];
                    const bool in = g <= row.cut;
                    w[j] = row.weight(in ? l[j] : top);
                    m[j] = in ? row.whole(w[j]) : 0.0;
                    b[j] = in ? row.bin_at(g) : ST_BINS;
                }
#pragma unroll
                for (int j = 0; j < VN; ++j) {
                    sum[3] += m[j];
                    if (!(w[j] < min_weight)) sum[4] += m[j];
                    if (b[j] < w0.b0) sum[0] += m[j];
                    if (b[j] < w1.b0) sum[1] += m[j];
                    bool listed = (w0.b0 <= b[j] && b[j] <= w0.b1) || (w1.b0 <= b[j] && b[j] <= w1.b1);
                    if (decltype(three)::value) {
                        if (b[j] < w2.b0) sum[2] += m[j];
                        listed |= w2.b0 <= b[j] && b[j] <= w2.b1;
                    }
                    if (listed) s.list(l[j], i + j);
                }
            });
        };
        if (w2.b0 < 0) weigh(std::false_type());
        else weigh(std::true_type());
#pragma unroll
        for (int j = 0; j < 5; ++j) {
            // in two halves of 26 bits, which a warp's sum keeps within 32
            const u64 x = (u64)sum[j];
            const unsigned lo = __reduce_add_sync(FULL, (unsigned)x & 0x3ffffffu), hi = __reduce_add_sync(FULL, (unsigned)(x >> 26));
            if (lane == 0) sm.warp_part[j][warp] = ((u64)hi << 26) + lo;
        }
        __syncthreads();
        if (warp < 5) {
            u64 x = lane < WARPS ? sm.warp_part[warp][lane] : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(FULL, x, o);
            if (lane == 0) sm.part[warp] = x;
        }
        s.sync();
        if (rank == 0) {
            if (warp < 5) {
                u64 x = lane < C ? s.at(&sm, lane)->part[warp] : 0;
#pragma unroll
                for (int o = 1; o < C; o <<= 1) x += __shfl_xor_sync(FULL, x, o);
                if (lane == 0) sm.warp_part[0][warp] = x;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 5; ++j) part[j] = sm.warp_part[0][j];
            __syncthreads();
        }
    }
    // the first CTA reads the answers off the list
    if (rank == 0) {
        const bool found = s.answer(windows, quick, top_k, top_p, min_weight, u, part, a.tokens + r, a.logprob + r);
        __syncthreads();
        if (tid < C) s.at(&sm, tid)->go_on = found;
    }
    s.sync();  // and no CTA leaves while another may read its shared memory
    if (!sm.go_on) st_general<TX, C, NT, HELD>(row, sm, st_raw, rank, top_k, top_p, min_weight, u, a.tokens + r, a.logprob + r);
}

template <class TX, int C, int NT, bool HELD>
static size_t sample_smem(int slice) {
    constexpr int TURN = NT * ST_TURN;
    return Sampler<TX, C, NT, HELD>::BYTES + (HELD ? (size_t)slice * sizeof(TX) + 32 : (size_t)((slice + 8 + TURN - 1) / TURN) * NT * 4);
}

template <class TX, int C, int NT, bool HELD>
static cudaError_t sample_launch(SampleArgs a, cudaStream_t s) {
    a.slice = ((a.V + C - 1) / C + 7) & ~7;
    cudaError_t e = prepare_kernel<sample_kernel<TX, C, NT, HELD>>(200 * 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * C);
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = sample_smem<TX, C, NT, HELD>(a.slice);
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
    return cudaLaunchKernelEx(&cfg, sample_kernel<TX, C, NT, HELD>, a);
}

// Clusters of 8 that run at once on the current device: a CTA of theirs takes an SM, so
// that the length of a row is of no account.
template <class TX>
static int sample_clusters() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    int n = known[dev].load(std::memory_order_relaxed);
    if (n > 0) return n;
    if (prepare_kernel<sample_kernel<TX, 8, 1024, true>>(200 * 1024) != cudaSuccess) return 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(8);
    cfg.blockDim = dim3(1024);
    cfg.dynamicSmemBytes = sample_smem<TX, 8, 1024, true>(ST_MAX_V / 8);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 8;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, sample_kernel<TX, 8, 1024, true>, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        return 1;
    }
    known[dev].store(n, std::memory_order_relaxed);
    return n;
}

// Up to 8192 logits by half as many threads, held in one CTA's shared memory (8192 by
// top-k 50 7.6 us, streamed 8.5).  More by a top-k that all rows share: a row
// streams through one CTA, which has little to do but read it (one row of 16,000 8.5 us and
// of 151,936 15.1; by a cluster 13.2 and 31.2).  By windows each logit costs more, and
// a cluster shares that: 1 row of 32,000 20 us, of 151,936 26, streamed 27 and 75.  But
// few clusters run at once: 16 rows 41 and 52 us, streamed 27 and 76, 32 rows of 151,936 79
// and 75.  A top-k of each row's own is on the device, so that the call goes by the
// windows' rule, also where the rows' are small and streaming would be faster (16 rows of
// 151,936 by their own top-k 50 64 us, by one number 20; 32 rows 20 and 20).
template <class TX>
static cudaError_t sample_typed(const SampleArgs& a, cudaStream_t s) {
    if (a.V <= 8192) return sample_launch<TX, 1, 512, true>(a, s);
    if (a.top_k == nullptr && a.top_k0 > 0 && a.top_k0 <= ST_QUICK_K) return sample_launch<TX, 1, 1024, false>(a, s);
    const int turns = (a.rows - 1) / sample_clusters<TX>() + 1;
    if ((float)turns * (18.f + (float)a.V / 18000.f) < 14.f + (float)a.V / 2500.f) return sample_launch<TX, 8, 1024, true>(a, s);
    return sample_launch<TX, 1, 1024, false>(a, s);
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
