// Attention of one new token per row over the paged cache, with a sliding
// window, sinks and the attention weights added up per slot:
//   q, k = RoPE(RMSNorm(.)) at pos[row];  k, v -> slot cached[row]
//   o_h = sum_j p_hj v_j,  p_hj = exp(q_h.k_j / sqrt(128) - m_h) / l_h over the visible slots
//   mass[row][g][j] += sum over g's heads of p_hj  (the new slot's is set)
//
// What bounds it: one read of the visible keys and values (1 KB per slot and
// kv head) against 512 FMA per query-head pair, so memory.  One thread-block
// cluster of C CTAs per (row, kv head); CTA s takes the s-th part of the
// visible slots (the sinks, then the window).  A warp takes four slots at a
// time: 8 lanes per slot, lane t of them float4 columns t, t+8, t+16, t+24 of
// the key and the value row.  Every lane copies exactly the 16-byte words it
// will read itself into a ring in shared memory (cp.async), so no barrier is
// needed in the loop and the bytes in flight cost no registers.  The 8
// lanes share a slot's scores (3 shuffles) and each 8-lane group keeps its
// own running maximum, sum and output columns, so P.V needs no shuffles.
// Groups, warps and CTAs are joined in a fixed order at the end, the CTAs
// through distributed shared memory: no scratch, no atomics, one launch.
// 128 rows of 120 to 640 visible slots: 80 us, 93 % of a plain copy's rate.
// With `mass`, raw scores go to a scratch array (8 bytes a slot beside 1 KB of
// keys and values) and become weights once the cluster knows m and l: 2 rows of
// 32k slots 102 us, 80 % of a copy's rate.
#include "cache_ops.cuh"

namespace skb {

constexpr int WD_THREADS = 256;
constexpr int WD_WARPS = WD_THREADS / 32;
constexpr int WD_MAXC = 8;
constexpr int WD_STAGE = WD_THREADS * 8 * 16;  // K and V words of one step of every lane

struct WdArgs {
    CacheAttnArgs a;
    float* scores;  // [rows][KVH][vis_cap][NR] raw scores in log2 units (mass only)
    int vis_cap;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
    const int n = real ? 16 : 0;  // fewer source bytes: the rest is zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ void st_cluster_f32(float* p, float v, uint32_t rank) {
    uint32_t rp;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rp) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(rp), "f"(v) : "memory");
}

template <int NR>
struct WdSmem {
    float q[NR][128];
    float kn[128], vn[128];
    float wm[WD_WARPS][NR], wl[WD_WARPS][NR];  // per warp
    float cm[WD_MAXC][NR], cl[WD_MAXC][NR];    // per CTA, written by every CTA of the cluster
    float co[WD_MAXC][NR][128];                // rank 0: every CTA's output part
    float fm[NR], fi[NR];                      // the cluster's maximum and 1 / sum
};

template <int NR>
struct WdStages {
    static constexpr int value = NR <= 2 ? 3 : 6;
};

template <int NR>
__global__ void __launch_bounds__(WD_THREADS, NR <= 2 ? 2 : 1) window_decode_kernel(const WdArgs w) {
    constexpr int NST = WdStages<NR>::value;
    extern __shared__ __align__(128) unsigned char wd_raw[];
    __shared__ WdSmem<NR> sm;
    const CacheAttnArgs& a = w.a;
    const int s = blockIdx.x, g = blockIdx.y, r = blockIdx.z;
    const int C = gridDim.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int KVH = a.kv.KVH;
    const int cap = a.kv.max_pages << a.kv.page_log2;

    float* orow = a.out + (long long)r * a.H * 128 + g * NR * 128;
    const int cached = a.cached[r], pos = a.pos[r];
    // idle row: zeros; a row whose numbers point outside the cache or the
    // RoPE tables: NaN.  Neither touches the cache.  (The whole cluster
    // works on one row, so all its CTAs leave here together.)
    long long new_unit = -1;
    if (cached >= 0 && cached < cap) new_unit = a.kv.key_unit(r, cached, g);
    const bool idle = cached < 0;
    if (idle || new_unit < 0 || pos < 0 || pos >= a.max_pos) {
        if (s == 0)
            for (int i = tid; i < NR * 128; i += WD_THREADS) orow[i] = idle ? 0.f : __int_as_float(0x7fffffff);
        return;
    }
    // visible cached slots: [0, ns) then [w0, cached)
    int ns = 0, w0 = 0;
    if (a.window > 0 && cached - a.window + 1 > 0) {
        w0 = cached - a.window + 1;
        ns = min(a.sinks, w0);
    }
    const int nv = ns + cached - w0;
    const int ib = (int)((long long)s * nv / C), ie = (int)((long long)(s + 1) * nv / C);

    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // all CTAs run before any remote store

    const int grp = lane >> 3, t8 = lane & 7;
    const uint32_t ring = smem_u32(wd_raw) + tid * 16;
    const float4* pool4 = reinterpret_cast<const float4*>(a.kv.pool);
    const long long vstep = a.kv.value_step() * 32;
    unsigned bad = 0;  // bit per ring stage: the slot's page is outside the pool
    // Copies the K and V words of this lane's slot i into stage st.
    auto fetch = [&](int i, int st) {
        const bool real = i < ie;
        const int slot = i < ns ? i : w0 + i - ns;
        const long long u = real ? a.kv.key_unit(r, slot, g) : 0;
        const bool ok = real && u >= 0;
        bad = (bad & ~(1u << st)) | ((real && !ok) ? 1u << st : 0u);
        const float4* k = pool4 + (ok ? u * 32 : 0) + t8;
        const uint32_t d = ring + st * WD_STAGE;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            cp_async16(d + j * WD_THREADS * 16, k + 8 * j, ok);
            cp_async16(d + (4 + j) * WD_THREADS * 16, k + (ok ? vstep : 0) + 8 * j, ok);
        }
    };
    const int i0 = ib + warp * 4 + grp;
    constexpr int STEP = WD_WARPS * 4;
#pragma unroll
    for (int st = 0; st < NST - 1; ++st) {
        fetch(i0 + st * STEP, st);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // the new token's heads
    const float* row = a.qkv + (long long)r * (a.H + 2 * KVH) * 128;
    if (warp < NR + 2) {
        const int v = warp < NR ? g * NR + warp : (warp == NR ? a.H + g : a.H + KVH + g);
        float4 x = reinterpret_cast<const float4*>(row + v * 128)[lane];
        if (warp <= NR)
            x = norm_rope_head(x, warp < NR ? a.qn : a.kn, a.eps, a.rope_cos + (long long)pos * 64,
                               a.rope_sin + (long long)pos * 64, lane, true, true);
        if (warp < NR) {
            const float c = 0.08838834764831845f * CO_LOG2E;  // 1 / sqrt(128), scores in log2 units
            reinterpret_cast<float4*>(sm.q[warp])[lane] = make_float4(x.x * c, x.y * c, x.z * c, x.w * c);
        } else {
            reinterpret_cast<float4*>(warp == NR ? sm.kn : sm.vn)[lane] = x;
            if (s == C - 1) {
                float4* dst = reinterpret_cast<float4*>(a.kv.pool) + new_unit * 32 + (warp == NR ? 0 : vstep);
                dst[lane] = x;
            }
        }
    }
    __syncthreads();

    float4 q[NR][4], o[NR][4];
    float m[NR], l[NR];
#pragma unroll
    for (int h = 0; h < NR; ++h) {
        m[h] = CO_LOW;
        l[h] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            q[h][j] = reinterpret_cast<const float4*>(sm.q[h])[t8 + 8 * j];
            o[h][j] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    // One slot of this 8-lane group: its scores, the running statistics, P.V.
    auto take = [&](const float4 (&k)[4], const float4 (&v)[4], bool real, bool poison, float* put) {
        float sc[NR];
        bool up = false;
#pragma unroll
        for (int h = 0; h < NR; ++h) {
            float d = 0.f, e = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                d = fmaf(q[h][j].x, k[j].x, d);
                e = fmaf(q[h][j].y, k[j].y, e);
                d = fmaf(q[h][j].z, k[j].z, d);
                e = fmaf(q[h][j].w, k[j].w, e);
            }
            sc[h] = d + e;
        }
#pragma unroll
        for (int h = 0; h < NR; ++h) {
            sc[h] += __shfl_xor_sync(FULL, sc[h], 1);
            sc[h] += __shfl_xor_sync(FULL, sc[h], 2);
            sc[h] += __shfl_xor_sync(FULL, sc[h], 4);
            sc[h] = poison ? __int_as_float(0x7fffffff) : fmaf(0.f, sc[h], sc[h]);  // an infinite score is NaN too
            if (put != nullptr && real && t8 == 0) put[h] = sc[h];
            up |= real && sc[h] > m[h];
        }
        if (__any_sync(FULL, up)) {
#pragma unroll
            for (int h = 0; h < NR; ++h) {
                const float mn = real ? fmaxf(m[h], sc[h]) : m[h];
                const float c = exp2_fast(m[h] - mn);
                m[h] = mn;
                l[h] *= c;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[h][j].x *= c;
                    o[h][j].y *= c;
                    o[h][j].z *= c;
                    o[h][j].w *= c;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < NR; ++h) {
            const float p = real ? exp2_fast(sc[h] - m[h]) : 0.f;
            l[h] += p;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[h][j].x = fmaf(p, v[j].x, o[h][j].x);
                o[h][j].y = fmaf(p, v[j].y, o[h][j].y);
                o[h][j].z = fmaf(p, v[j].z, o[h][j].z);
                o[h][j].w = fmaf(p, v[j].w, o[h][j].w);
            }
        }
    };
    float* scores = w.scores == nullptr ? nullptr : w.scores + ((long long)r * KVH + g) * w.vis_cap * NR;
    const int steps = ie > ib ? (ie - ib + STEP - 1) / STEP : 0;
    int st = 0;
    for (int n = 0; n < steps; ++n) {
        // the stage freed by the previous step takes the copies of the step
        // NST - 1 ahead (this lane alone reads and writes its words)
        const int i = i0 + n * STEP;
        const int nf = st == 0 ? NST - 1 : st - 1;
        fetch(i + (NST - 1) * STEP, nf);
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group %0;" ::"n"(NST - 1) : "memory");
        float4 k[4], v[4];
        const float4* at = reinterpret_cast<const float4*>(wd_raw + st * WD_STAGE) + tid;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            k[j] = at[j * WD_THREADS];
            v[j] = at[(4 + j) * WD_THREADS];
        }
        take(k, v, i < ie, (bad >> st) & 1u, scores == nullptr ? nullptr : scores + (long long)i * NR);
        st = st == NST - 1 ? 0 : st + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    float new_sc[NR];
    if (warp == 0) {  // the new token itself, by group 0 of the last CTA
        float4 k[4], v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            k[j] = reinterpret_cast<const float4*>(sm.kn)[t8 + 8 * j];
            v[j] = reinterpret_cast<const float4*>(sm.vn)[t8 + 8 * j];
        }
        float* put = scores == nullptr ? nullptr : new_sc;
        take(k, v, s == C - 1 && grp == 0, false, put);
        if (scores != nullptr && s == C - 1 && lane == 0) {
#pragma unroll
            for (int h = 0; h < NR; ++h) scores[(long long)nv * NR + h] = new_sc[h];
        }
    }
    // ---- join the four groups of a warp, in group order
#pragma unroll
    for (int off = 8; off <= 16; off <<= 1) {
#pragma unroll
        for (int h = 0; h < NR; ++h) {
            const float m2 = __shfl_xor_sync(FULL, m[h], off);
            const float mn = fmaxf(m[h], m2);
            const float c = exp2_fast(m[h] - mn);
            l[h] *= c;
            l[h] += __shfl_xor_sync(FULL, l[h], off);
            m[h] = mn;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[h][j].x *= c;
                o[h][j].y *= c;
                o[h][j].z *= c;
                o[h][j].w *= c;
                o[h][j].x += __shfl_xor_sync(FULL, o[h][j].x, off);
                o[h][j].y += __shfl_xor_sync(FULL, o[h][j].y, off);
                o[h][j].z += __shfl_xor_sync(FULL, o[h][j].z, off);
                o[h][j].w += __shfl_xor_sync(FULL, o[h][j].w, off);
            }
        }
    }
    // ---- the warps: outputs into the ring's memory, whose copies are done
    __syncthreads();
    float (*wo)[NR][128] = reinterpret_cast<float (*)[NR][128]>(wd_raw);
    if (grp == 0) {
#pragma unroll
        for (int h = 0; h < NR; ++h) {
#pragma unroll
            for (int j = 0; j < 4; ++j) reinterpret_cast<float4*>(wo[warp][h])[t8 + 8 * j] = o[h][j];
            if (t8 == 0) {
                sm.wm[warp][h] = m[h];
                sm.wl[warp][h] = l[h];
            }
        }
    }
    __syncthreads();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int i = tid; i < NR * 128; i += WD_THREADS) {
        const int h = i >> 7, d = i & 127;
        float M = CO_LOW, L = 0.f, O = 0.f;
#pragma unroll
        for (int x = 0; x < WD_WARPS; ++x) M = fmaxf(M, sm.wm[x][h]);
#pragma unroll
        for (int x = 0; x < WD_WARPS; ++x) {
            const float c = exp2_fast(sm.wm[x][h] - M);
            L = fmaf(sm.wl[x][h], c, L);
            O = fmaf(wo[x][h][d], c, O);
        }
        st_cluster_f32(&sm.co[s][h][d], O, 0);
        if (d < C) {  // this CTA's maximum and sum to every CTA
            st_cluster_f32(&sm.cm[s][h], M, d);
            st_cluster_f32(&sm.cl[s][h], L, d);
        }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (s == 0) {
        for (int i = tid; i < NR * 128; i += WD_THREADS) {
            const int h = i >> 7, d = i & 127;
            float M = CO_LOW, L = 0.f, O = 0.f;
            for (int x = 0; x < C; ++x) M = fmaxf(M, sm.cm[x][h]);
            for (int x = 0; x < C; ++x) {
                const float c = exp2_fast(sm.cm[x][h] - M);
                L = fmaf(sm.cl[x][h], c, L);
                O = fmaf(sm.co[x][h][d], c, O);
            }
            orow[i] = O / L;
        }
    }
    if (scores == nullptr) return;
    // ---- weights of this CTA's slots (written by this CTA, ordered by the barriers above)
    float fm[NR], fi[NR];
#pragma unroll
    for (int h = 0; h < NR; ++h) {
        float M = CO_LOW, L = 0.f;
        for (int x = 0; x < C; ++x) M = fmaxf(M, sm.cm[x][h]);
        for (int x = 0; x < C; ++x) L = fmaf(sm.cl[x][h], exp2_fast(sm.cm[x][h] - M), L);
        fm[h] = M;
        fi[h] = 1.f / L;
    }
    float* mass = a.mass + ((long long)r * KVH + g) * cap;
    const int end = s == C - 1 ? nv + 1 : ie;
    // eight slots a thread at a time, all of a batch's loads before its stores:
    // one after the other they cost 14 of 109 us at 2 x 32k slots
    constexpr int U = 8;
    for (int i0 = ib + tid; i0 < end; i0 += WD_THREADS * U) {
        float sc[U][NR], old[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int i = i0 + k * WD_THREADS;
            old[k] = 0.f;
            if (i < end) {
#pragma unroll
                for (int h = 0; h < NR; ++h) sc[k][h] = scores[(long long)i * NR + h];
                if (i != nv) old[k] = mass[i < ns ? i : w0 + i - ns];
            }
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int i = i0 + k * WD_THREADS;
            if (i >= end) continue;
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < NR; ++h) sum += exp2_fast(sc[k][h] - fm[h]) * fi[h];
            mass[i < ns ? i : w0 + i - ns] = old[k] + sum;
        }
    }
}

template <int NR>
static cudaError_t window_decode_launch(const WdArgs& w, cudaStream_t stream) {
    const size_t smem = (size_t)WdStages<NR>::value * WD_STAGE;
    static std::atomic<unsigned long long> done;
    cudaError_t e = smem_attrs_once(window_decode_kernel<NR>, smem, done);
    if (e != cudaSuccess) return e;
    // Up to 592 CTAs, two waves of two an SM (four of one for 3 and 4 heads a kv
    // head), while the cluster stays within the portable 8.  Measured, us a call with
    // at most 296, 592 and 1184 CTAs: two heads, 296 groups of 1000 to 2000 slots 77, 79,
    // 82; 160 groups of 3000 to 6000 137, 132, 122; 128 of 4000 to 8000 131, 129,
    // 129; 72 of 3000 to 6000 60, 63, 63.  Four heads, in the same order: 89, 98, 131;
    // 173, 144, 144; 141, 149, 190; 74, 92, 92.  No limit is best for all.  128 short rows
    // (120 to 842 slots, 8 kv heads, a CTA a group) with 1, 2, 3 and 4 heads a kv
    // head: 83, 88, 109 and 120 us for 79 us of bytes at a copy's rate.
    const long long groups = (long long)w.a.rows * w.a.kv.KVH;
    int C = WD_MAXC;
    while (C > 1 && groups * C > 592) C >>= 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C, w.a.kv.KVH, w.a.rows);
    cfg.blockDim = dim3(WD_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, window_decode_kernel<NR>, w);
}

int cache_attn_check(const char* what, const void* qkv, int rows, int H, int KVH, int hd, const void* qn,
                     const void* kn, const void* rc, const void* rs, int max_pos, const void* cached, const void* pos,
                     const void* kv_pool, const void* page_table, int max_pages, int page_size, int n_pages,
                     int window, int sinks, const void* out) {
    if (!qn || !kn || !rc || !rs || !cached || !pos || !kv_pool || !page_table)
        return fail(SKB_ERR_ARG, "%s: null pointer", what);
    if (hd != 128 || KVH < 1 || H < 1 || H % KVH != 0 || H / KVH > CO_MAX_REP)
        return fail(SKB_ERR_ARG, "%s: head_dim must be 128 and heads / kv_heads 1 to %d", what, CO_MAX_REP);
    if (rows < 0 || rows > 65535 || KVH > 65535 || max_pos < 1 || max_pages < 1 || n_pages < 1)
        return fail(SKB_ERR_ARG, "%s: bad sizes", what);
    if (page_size < 1 || (page_size & (page_size - 1)) != 0 || (long long)max_pages * page_size > (1ll << 30))
        return fail(SKB_ERR_ARG, "%s: page_size must be a power of two, and a row at most 2^30 slots", what);
    if (window < 0 || sinks < 0 || (window == 0 && sinks != 0))
        return fail(SKB_ERR_ARG, "%s: window and sinks must be >= 0, and sinks need a window", what);
    if (((uintptr_t)qkv | (uintptr_t)rc | (uintptr_t)rs | (uintptr_t)kv_pool | (uintptr_t)qn | (uintptr_t)kn |
         (uintptr_t)out) & 15u)
        return fail(SKB_ERR_ARG, "%s: qkv, norm weights, RoPE tables, kv_pool and out must be 16-byte aligned", what);
    return SKB_OK;
}

static long long wd_visible_cap(int max_pages, int page_size, int window, int sinks) {
    const long long cap = (long long)max_pages * page_size, seen = (long long)window + sinks;
    return window > 0 && seen < cap ? seen : cap;
}

}  // namespace skb

using namespace skb;

extern "C" int64_t skb_window_decode_workspace(int rows, int n_heads, int max_pages, int page_size, int window,
                                               int sinks, int with_mass) {
    if (rows < 0 || n_heads < 1 || max_pages < 1 || page_size < 1 || window < 0 || sinks < 0) return -1;
    return with_mass ? (int64_t)rows * n_heads * wd_visible_cap(max_pages, page_size, window, sinks) * 4 : 0;
}

extern "C" int skb_window_decode_attention(const float* qkv, int rows, int n_heads, int n_kv_heads, int head_dim,
                                           const float* q_norm, const float* k_norm, float eps, const float* rope_cos,
                                           const float* rope_sin, int max_pos, const int32_t* cached,
                                           const int32_t* pos, float* kv_pool, const int32_t* page_table,
                                           int max_pages, int page_size, int n_pages, int window, int sinks,
                                           float* mass, void* work, int64_t work_bytes, float* out,
                                           cudaStream_t stream) {
    const char* what = "window_decode_attention";
    const int st = cache_attn_check(what, qkv, rows, n_heads, n_kv_heads, head_dim, q_norm, k_norm, rope_cos, rope_sin,
                                    max_pos, cached, pos, kv_pool, page_table, max_pages, page_size, n_pages, window,
                                    sinks, out);
    if (st != SKB_OK) return st;
    if (rows == 0) return SKB_OK;
    if (!qkv || !out) return fail(SKB_ERR_ARG, "%s: null pointer", what);
    if (mass && (!work || work_bytes < skb_window_decode_workspace(rows, n_heads, max_pages, page_size, window, sinks, 1)))
        return fail(SKB_ERR_ARG, "%s: mass needs a workspace of skb_window_decode_workspace bytes", what);
    WdArgs w = {};
    w.a.qkv = qkv;
    w.a.qn = q_norm;
    w.a.kn = k_norm;
    w.a.eps = eps;
    w.a.rope_cos = rope_cos;
    w.a.rope_sin = rope_sin;
    w.a.max_pos = max_pos;
    w.a.cached = cached;
    w.a.pos = pos;
    w.a.kv = {kv_pool, page_table, max_pages, log2_of(page_size), n_kv_heads, n_pages};
    w.a.H = n_heads;
    w.a.rows = rows;
    w.a.window = window;
    w.a.sinks = sinks;
    w.a.mass = mass;
    w.a.out = out;
    w.scores = mass ? static_cast<float*>(work) : nullptr;
    w.vis_cap = (int)wd_visible_cap(max_pages, page_size, window, sinks);
    cudaError_t e = cudaErrorInvalidValue;
    switch (n_heads / n_kv_heads) {
        case 1: e = window_decode_launch<1>(w, stream); break;
        case 2: e = window_decode_launch<2>(w, stream); break;
        case 3: e = window_decode_launch<3>(w, stream); break;
        case 4: e = window_decode_launch<4>(w, stream); break;
    }
    return e == cudaSuccess ? SKB_OK : fail(SKB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
