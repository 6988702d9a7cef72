// Attention of a chunk of new tokens per row over the paged cache: ragged
// chunks behind each row's cached slots, causal, with an optional sliding
// window and sinks, and optionally the attention weights added up per slot.
//   q_i, k_i = RoPE(RMSNorm(.)) at pos[row] + i;  k_i, v_i -> slot cached[row] + i
//   o_ih = sum_j p_ihj v_j,  p_ihj = exp(q_ih.k_j / sqrt(128) - lse_ih) over the slots i sees
//   mass[row][g][j] += sum_i sum over g's heads of p_ihj  (new slots begin at zero)
//
// Three launches: chunk_prep norms, rotates, appends k and v and writes the
// queries as split fp16 tiles; chunk_attn; and, with `mass`, chunk_mass.
// A query tile is 128 (token, head) pairs of one kv head, P = 128 / n_rep
// tokens, so a key or value tile that was loaded once serves all of them.
#include "umma.cuh"

namespace skb {

struct ChunkArgs {
    CacheAttnArgs a;
    const int* chunk_start;  // [rows + 1]
    int tokens, max_chunk;
    int n_rep, P;           // heads per kv head, tokens per query tile
    unsigned char* qtiles;  // workspace [tiles][KVH][2 UT_BYTES]: queries in log2 units, hi | lo
    float* lse;             // workspace [tiles][KVH][128] (mass only), log2 units
};

// What a row asks for: its tokens [b, b + n) and whether its numbers lie
// inside the inputs, the cache and the RoPE tables.
struct ChunkRow {
    int b, n, cached;
    bool idle, bad;
};
__device__ __forceinline__ ChunkRow chunk_row(const ChunkArgs& c, int r) {
    ChunkRow x;
    const int b = c.chunk_start[r], e = c.chunk_start[r + 1], pos = c.a.pos[r];
    x.b = max(0, min(b, c.tokens));
    x.n = max(0, min(e, c.tokens) - x.b);
    x.cached = c.a.cached[r];
    x.idle = x.cached < 0;
    const long long cap = (long long)c.a.kv.max_pages << c.a.kv.page_log2;
    x.bad = b < 0 || e < b || e > c.tokens || x.n > c.max_chunk || (long long)x.cached + x.n > cap || pos < 0 ||
            (long long)pos + x.n > c.a.max_pos;
    return x;
}
// Index of a row's query tile t in the workspace: rows' stretches do not
// overlap, since (b + n) / P + 1 >= b / P + ceil(n / P), and none passes
// tokens / P + rows.
__device__ __forceinline__ long long chunk_tile(const ChunkArgs& c, const ChunkRow& x, int r, int t) {
    return x.b / c.P + r + t;
}

// A whole number e with |q| < 2^e for every query in log2 units: a normed head
// is at most sqrt(128) max|w| long per element, its rotation sqrt(2) times that.
__device__ __forceinline__ float query_exponent(const float* qn, int lane) {
    const float4 w = __ldg(reinterpret_cast<const float4*>(qn) + lane);
    const float m = warp_max(fmaxf(fmaxf(fabsf(w.x), fabsf(w.y)), fmaxf(fabsf(w.z), fabsf(w.w))));
    const int e = (int)(__float_as_uint(m * 2.0405f) >> 23) - 126;
    return (float)max(-100, min(100, e));
}

constexpr float CH_QSCALE = 0.08838834764831845f * CO_LOG2E;  // 1 / sqrt(128), scores in log2 units

// grid (min(max_chunk, 4096), rows, ceil((H + 2 KVH) / 8)), 256 threads: a warp per head vector
__global__ void __launch_bounds__(256) chunk_prep_kernel(const ChunkArgs c) {
    const CacheAttnArgs& a = c.a;
    const int r = blockIdx.y, lane = threadIdx.x & 31, v = blockIdx.z * 8 + (threadIdx.x >> 5);
    const ChunkRow x = chunk_row(c, r);
    const int H = a.H, KVH = a.kv.KVH;
    pdl_trigger();
    if (v >= H + 2 * KVH) return;
    const float eq = query_exponent(a.qn, lane);
    for (int i = blockIdx.x; i < x.n; i += gridDim.x) {
        const long long t = x.b + i;
        if (x.idle || x.bad) {
            const float o = x.idle ? 0.f : __int_as_float(0x7fffffff);
            if (v < H) reinterpret_cast<float4*>(a.out)[(t * H + v) * 32 + lane] = make_float4(o, o, o, o);
            continue;
        }
        const int pos = a.pos[r] + i, slot = x.cached + i;
        float4 y = reinterpret_cast<const float4*>(a.qkv)[(t * (H + 2 * KVH) + v) * 32 + lane];
        if (v < H + KVH)
            y = norm_rope_head(y, v < H ? a.qn : a.kn, a.eps, a.rope_cos + (long long)pos * 64,
                               a.rope_sin + (long long)pos * 64, lane, true, true);
        if (v < H) {
            const int g = v / c.n_rep, m = (i % c.P) * c.n_rep + v % c.n_rep;
            unsigned char* tile = c.qtiles + (chunk_tile(c, x, r, i / c.P) * KVH + g) * (2 * UT_BYTES);
            put_row(tile, m, lane, make_float4(y.x * CH_QSCALE, y.y * CH_QSCALE, y.z * CH_QSCALE, y.w * CH_QSCALE), eq);
        } else {
            const bool value = v >= H + KVH;
            const long long u = a.kv.key_unit(r, slot, v - H - (value ? KVH : 0));
            if (u >= 0) reinterpret_cast<float4*>(a.kv.pool)[(u + (value ? a.kv.value_step() : 0)) * 32 + lane] = y;
        }
    }
}

// ------------------------------------------------------------ the key tiles
// The tiles of 128 slots that a query tile (slots own_lo .. own_hi) sees, as
// a list: first those that all its queries see whole, then the others (the
// sinks, the window's edge, the diagonal).
struct TileList {
    int n, full, full0;      // tiles; how many are whole; the first whole one
    int a1, b0, head;        // sink tiles [0, a1); window tiles from b0; of them `head` before the whole ones
    __device__ __forceinline__ TileList(int own_lo, int own_hi, int window, int sinks) {
        const int w0 = window > 0 ? max(0, own_lo - window + 1) : 0;  // first slot of any query's window
        a1 = (min(sinks, w0) + 127) >> 7;
        b0 = max(w0 >> 7, a1);
        const int end = (own_hi >> 7) + 1;  // every tile before it holds a visible slot
        const int whole0 = window > 0 && own_hi - window + 1 > 0 ? (own_hi - window + 1 + 127) >> 7 : 0;
        full0 = max(b0, whole0);
        const int whole1 = (own_lo + 1) >> 7;
        full = max(0, min(whole1, end) - full0);
        if (b0 > end) b0 = end;
        if (full == 0) full0 = end;  // then every window tile counts as head
        head = full0 - b0;
        n = a1 + (end - b0);
    }
    __device__ __forceinline__ int tile(int k) const {
        if (k < full) return full0 + k;
        k -= full;
        if (k < a1) return k;
        k -= a1;
        return k < head ? b0 + k : full0 + full + (k - head);
    }
};

// -------------------------------------------------------------- chunk_attn
constexpr int CA_SOFTMAX_WARPS = 4, CA_CONV_WARPS = 8;
constexpr int CA_MMA_WARP = CA_SOFTMAX_WARPS + CA_CONV_WARPS;
constexpr int CA_THREADS = 512;  // whole warpgroups: softmax, two of converters, one whose first warp issues products
// Registers a thread: all are launched with 128.  The softmax threads hold a
// whole output row, so they take from the others meanwhile; every sum over the
// four warpgroups stays within the launch's 4 x 128.  Nobody takes registers
// back before the softmax threads have given theirs up (a CTA-wide barrier
// lies between): a warpgroup that is done early, or has nothing to do, would
// otherwise take what they still wait for.
constexpr int CA_REGS = 65536 / CA_THREADS, CA_REGS_SOFTMAX = 240, CA_REGS_CONV = 104, CA_REGS_MMA = 64;
static_assert(CA_REGS_SOFTMAX + 2 * CA_REGS_CONV + CA_REGS_MMA <= 4 * CA_REGS, "register split");
template <int N>
__device__ __forceinline__ void regs_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
constexpr int CA_ROWS_PER_WARP = UT_ROWS / CA_CONV_WARPS;  // 16
constexpr uint32_t CA_TM_O = 256, CA_TM_P = 384;           // TMEM columns: scores [0, 256), output, weights
constexpr int CA_OUT_LD = 132;                              // floats of a staged output row
constexpr int CA_MAX_SPLITS = 8;

struct CaSmem {
    unsigned char q[2 * UT_BYTES];
    unsigned char k[2 * UT_BYTES];
    unsigned char v[2 * UT_BYTES];
    float kc[3][128];                // factor of a key's scores: its scale undone
    float ve[2][128];                // exponent of a value row
    float vg[2][128];                // factor of its weights: 2^(exponent - the tile's running one + 6)
    float vmax[2][CA_CONV_WARPS];    // largest exponent of a warp's rows
    float m[128], l[128];            // this split's statistics
    uint64_t q_full, k_full, k_empty, v_full, v_empty, p_full, s_full[2], ve_full[2], o_full;
    uint32_t tmem;
    int abort;
};
constexpr size_t CA_SMEM = sizeof(CaSmem) + 1024;
static_assert(CA_SMEM <= 227 * 1024, "shared memory of one CTA");
static_assert(128 * CA_OUT_LD * 4 <= 2 * 2 * UT_BYTES, "the staged output lies over the query and key tiles");

// The four softmax warps.
__device__ __forceinline__ void warpgroup_sync() { asm volatile("bar.sync 2, 128;" ::: "memory"); }

__device__ __forceinline__ float4 ld_peer4(uint32_t local, uint32_t rank) {
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(local), "r"(rank));
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(ra)
                 : "memory");
    return v;
}
__device__ __forceinline__ float ld_peer(const float* p, uint32_t rank) {
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(p)), "r"(rank));
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ra) : "memory");
    return v;
}

// Converter warps: where rows w*16 .. w*16+15 of a key tile lie.  Lane i < 16
// holds row i's unit in the pool; CA_NONE: no query sees the slot (zeros),
// CA_BAD: its page is outside the pool.
constexpr uint32_t CA_NONE = 0xffffffffu, CA_BAD = 0xfffffffeu;

// grid (splits * query tiles, KVH, rows), clusters of `splits` CTAs
__global__ void __launch_bounds__(CA_THREADS, 1) chunk_attn_kernel(const ChunkArgs c, int splits) {
    extern __shared__ unsigned char ca_raw[];
    CaSmem& sm = *reinterpret_cast<CaSmem*>(ca_raw + ((1024u - (smem_u32(ca_raw) & 1023u)) & 1023u));
    const CacheAttnArgs& a = c.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = blockIdx.y, r = blockIdx.z, z = blockIdx.x % splits;
    const int tiles_x = gridDim.x / splits;
    const int t = tiles_x - 1 - blockIdx.x / splits;  // the last query tile sees the most: first
    const ChunkRow x = chunk_row(c, r);
    const int i0 = t * c.P;
    if (x.idle || x.bad || i0 >= x.n) {  // the same for a whole cluster
        pdl_wait();
        return;
    }
    const int nq = min(c.P, x.n - i0);
    const int own_lo = x.cached + i0, own_hi = own_lo + nq - 1;
    const TileList list(own_lo, own_hi, a.window, a.sinks);
    const int k0 = (int)((long long)z * list.n / splits), k1 = (int)((long long)(z + 1) * list.n / splits);
    const int nt = k1 - k0;
    const long long tile_at = chunk_tile(c, x, r, t) * a.kv.KVH + g;

    if (tid == 0) {
        mbar_init(&sm.q_full, 1);
        mbar_init(&sm.k_full, CA_CONV_WARPS);
        mbar_init(&sm.k_empty, 1);
        mbar_init(&sm.v_full, CA_CONV_WARPS);
        mbar_init(&sm.v_empty, 1);
        mbar_init(&sm.p_full, CA_SOFTMAX_WARPS);
        mbar_init(&sm.o_full, 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sm.s_full[b], 1);
            mbar_init(&sm.ve_full[b], CA_CONV_WARPS);
        }
        mbar_fence_init();
        sm.abort = 0;
    }
    if (warp == CA_MMA_WARP) ut_alloc(&sm.tmem);
    ut_fence_before();
    __syncthreads();
    ut_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* abort = &sm.abort;
    pdl_wait();
    if (c.lse) pdl_trigger();  // chunk_mass follows

    if (warp >= CA_MMA_WARP) {
        regs_down<CA_REGS_MMA>();
        if (warp == CA_MMA_WARP && lane == 0 && nt > 0) {
            mbar_expect_tx(&sm.q_full, 2 * UT_BYTES);
            bulk_g2s(sm.q, c.qtiles + tile_at * (2 * UT_BYTES), 2 * UT_BYTES, &sm.q_full);
            const uint32_t q = smem_u32(sm.q), k = smem_u32(sm.k), v = smem_u32(sm.v);
            bool go = ut_wait(&sm.q_full, 0, abort);
            auto weigh = [&](int i) {  // O = P_i V_i
                go = ut_wait(&sm.v_full, i & 1, abort) && ut_wait(&sm.p_full, i & 1, abort);
                if (!go) return;
                ut_fence_after();
                ut_mma_pv(tmem + CA_TM_O, tmem + CA_TM_P, v);
                ut_commit(&sm.v_empty);
            };
            for (int i = 0; i < nt && go; ++i) {
                go = ut_wait(&sm.k_full, i & 1, abort);
                if (!go) break;
                ut_fence_after();
                ut_mma_qk(tmem + (i & 1) * 128, q, k);
                ut_commit(&sm.k_empty);
                ut_commit(&sm.s_full[i & 1]);
                if (i > 0) weigh(i - 1);
            }
            if (go) weigh(nt - 1);
            ut_commit(&sm.o_full);  // every product issued so far
            ut_wait(&sm.o_full, 0, abort);
        }
        __syncwarp();
    } else if (warp >= CA_SOFTMAX_WARPS) {
        // ---- converters: FP32 rows of the pool -> split tiles
        regs_down<CA_REGS_CONV>();
        const int cw = warp - CA_SOFTMAX_WARPS, row0 = cw * CA_ROWS_PER_WARP;
        const float4* pool4 = reinterpret_cast<const float4*>(a.kv.pool) + lane;
        const uint32_t vstep = (uint32_t)a.kv.value_step();
        const float qfac = pow2_whole(query_exponent(a.qn, lane) - 13.f);
        const int w_lo = a.window > 0 ? max(0, own_lo - a.window + 1) : 0;
        auto units = [&](int i) -> uint32_t {
            const int slot = list.tile(k0 + i) * 128 + row0 + (lane & 15);
            if (i >= nt || slot > own_hi || (slot < w_lo && slot >= a.sinks)) return CA_NONE;
            const long long u = a.kv.key_unit(r, slot, g);
            return u < 0 ? CA_BAD : (uint32_t)u;
        };
        float4 d[CA_ROWS_PER_WARP];
        auto load = [&](int j, uint32_t us, uint32_t step) {
            const uint32_t u = __shfl_sync(FULL, us, j);
            d[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (u == CA_BAD) d[j].x = __int_as_float(0x7fffffff);
            else if (u != CA_NONE) d[j] = __ldcg(pool4 + (long long)(u + step) * 32);
        };
        auto exponents = [&]() {  // lane j < 16: row j's
            float e = UT_POISON_E;
#pragma unroll
            for (int j = 0; j < CA_ROWS_PER_WARP; ++j) {
                const float x = row_exponent(d[j]);
                if (lane == j) e = x;
            }
            return e;
        };
        // Writes the 16 rows and, behind each, asks for the row that takes
        // its place in the registers.
        auto put = [&](unsigned char* tile, float e, uint32_t us, uint32_t step) {
#pragma unroll
            for (int j = 0; j < CA_ROWS_PER_WARP; ++j) {
                put_row(tile, row0 + j, lane, d[j], __shfl_sync(FULL, e, j));
                load(j, us, step);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        uint32_t u_cur = units(0), u_next = CA_NONE;
        bool go = nt > 0;
        if (go) {
#pragma unroll
            for (int j = 0; j < CA_ROWS_PER_WARP; ++j) load(j, u_cur, 0);
        }
        auto key_tile = [&](int i, uint32_t us, uint32_t step) {
            const float e = exponents();
            if (lane < 16) sm.kc[i % 3][row0 + lane] = e == e ? pow2_whole(fmaxf(e, -100.f) - 13.f) * qfac : e;
            if (i > 0) go = ut_wait(&sm.k_empty, (i - 1) & 1, abort);
            if (!go) return;
            put(sm.k, e, us, step);
            if (lane == 0) ut_arrive(&sm.k_full);
        };
        // order: K0, K1, V0, K2, V1, ...; d always holds the next one
        if (go) {
            u_next = units(1);
            key_tile(0, nt > 1 ? u_next : u_cur, nt > 1 ? 0 : vstep);
        }
        for (int i = 0; i < nt && go; ++i) {
            if (i + 1 < nt) {
                key_tile(i + 1, u_cur, vstep);
                if (!go) break;
            }
            const float e = exponents();
            if (lane < 16) sm.ve[i & 1][row0 + lane] = e;
            const float top = warp_max(e);
            if (lane == 0) sm.vmax[i & 1][cw] = top;
            __syncwarp();
            if (lane == 0) ut_arrive(&sm.ve_full[i & 1]);
            if (i > 0) go = ut_wait(&sm.v_empty, (i - 1) & 1, abort);
            if (!go) break;
            // behind V_i comes K_{i+2}, or V_{i+1} if there is none
            const uint32_t u2 = units(i + 2);
            const bool more = i + 2 < nt;
            put(sm.v, e, more ? u2 : u_next, more ? 0 : vstep);
            if (lane == 0) ut_arrive(&sm.v_full);
            u_cur = u_next;
            u_next = u2;
        }
        __syncwarp();
    } else {
        // ---- softmax: thread = query row
        regs_up<CA_REGS_SOFTMAX>();
        const int row = tid, own = own_lo + row / c.n_rep;
        const bool live = row < nq * c.n_rep;
        const int hi = live ? own : -1;                                       // sees slots <= hi
        const int lo = a.window > 0 ? own - a.window : -1;                    // and > lo, or < sinks
        const uint32_t lane_tm = tmem + ((uint32_t)(32 * warp) << 16);
        float m = CO_LOW, l = 0.f, E = UT_POISON_E;
        // The output row, over the tiles before the newest, in units
        // 2^(E - 13 - 6) of that tile's E and m; f_o takes it there.
        uint64_t acc[64];
#pragma unroll
        for (int q = 0; q < 64; ++q) acc[q] = 0;
        float f_o = 1.f;
        auto gather = [&]() {  // acc = acc f_o + the newest tile's product
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
                uint32_t o[32];
                ut_ld32(lane_tm + CA_TM_O + ch * 32, o);
                ut_wait_ld();
#pragma unroll
                for (int q = 0; q < 16; ++q)
                    acc[ch * 16 + q] = fma2p(acc[ch * 16 + q], pack2(f_o, f_o),
                                             pack2(__uint_as_float(o[2 * q]), __uint_as_float(o[2 * q + 1])));
            }
        };
        // A wait that ran out ends every later one at once; the loop still runs
        // through, because its barrier needs all four warps.
        for (int i = 0; i < nt; ++i) {
            const int b = i & 1, base = list.tile(k0 + i) * 128;
            const bool whole = k0 + i < list.full;
            const uint32_t st = lane_tm + b * 128;
            const float4* kc = reinterpret_cast<const float4*>(sm.kc[i % 3]);
            ut_wait(&sm.s_full[b], (i >> 1) & 1, abort);
            ut_fence_after();
            // largest score (and, where queries differ in what they see, the
            // largest exponent among the values this query sees)
            float mx = CO_LOW, ex = UT_POISON_E;
            if (!whole) ut_wait(&sm.ve_full[b], (i >> 1) & 1, abort);
#pragma unroll 1
            for (int ch = 0; ch < 4; ++ch) {
                uint32_t s[32];
                ut_ld32(st + ch * 32, s);
                ut_wait_ld();
                if (whole) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const float4 f = kc[ch * 8 + q];
                        const float2 u = mul2(make_float2(__uint_as_float(s[4 * q]), __uint_as_float(s[4 * q + 1])),
                                              make_float2(f.x, f.y));
                        const float2 v = mul2(make_float2(__uint_as_float(s[4 * q + 2]), __uint_as_float(s[4 * q + 3])),
                                              make_float2(f.z, f.w));
                        mx = fmaxf(fmaxf(mx, u.x), u.y);
                        mx = fmaxf(fmaxf(mx, v.x), v.y);
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 32; ++q) {
                        const int j = base + ch * 32 + q;
                        if (j <= hi && (j > lo || j < a.sinks)) {
                            mx = fmaxf(mx, __uint_as_float(s[q]) * sm.kc[i % 3][ch * 32 + q]);
                            ex = fmaxf(ex, sm.ve[b][ch * 32 + q]);
                        }
                    }
                }
            }
            if (whole) {
                ut_wait(&sm.ve_full[b], (i >> 1) & 1, abort);
                const float4 e0 = reinterpret_cast<const float4*>(sm.vmax[b])[0];
                const float4 e1 = reinterpret_cast<const float4*>(sm.vmax[b])[1];
                ex = fmaxf(fmaxf(fmaxf(e0.x, e0.y), fmaxf(e0.z, e0.w)), fmaxf(fmaxf(e1.x, e1.y), fmaxf(e1.z, e1.w)));
            }
            if (!live) mx = CO_LOW;
            // The running maximum follows only when it is passed by 2^8, the
            // running exponent with 3 bits to spare: weights stay below 2^8,
            // scaled ones below 2^14.
            const float m_new = mx > m + 8.f ? mx : m;
            const float E_new = ex > E ? ex + 3.f : E;
            const float f_l = exp2_fast(m - m_new), f_new = f_l * exp2_fast(E - E_new);
            m = m_new;
            E = E_new;
            l *= f_l;
            if (whole) {  // E is the same for every row of the tile here
                sm.vg[b][row] = exp2_fast(sm.ve[b][row] - E + 6.f);
                warpgroup_sync();
            }
            if (i > 0) {  // P is free, and the product there, once P_{i-1} V_{i-1} is done
                ut_wait(&sm.v_empty, (i - 1) & 1, abort);
                ut_fence_after();
                gather();
            }
            f_o = i == 0 ? 0.f : f_new;
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
            for (int ch = 0; ch < 8; ++ch) {
                uint32_t s[16], ph[8], pl[8];
                ut_ld16(st + ch * 16, s);
                ut_wait_ld();
                const float4* vg = reinterpret_cast<const float4*>(sm.vg[b]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 f = kc[ch * 4 + q];
                    float2 u = fma2(make_float2(__uint_as_float(s[4 * q]), __uint_as_float(s[4 * q + 1])),
                                    make_float2(f.x, f.y), make_float2(-m, -m));
                    float2 v = fma2(make_float2(__uint_as_float(s[4 * q + 2]), __uint_as_float(s[4 * q + 3])),
                                    make_float2(f.z, f.w), make_float2(-m, -m));
                    u = make_float2(exp2_fast(u.x), exp2_fast(u.y));
                    v = make_float2(exp2_fast(v.x), exp2_fast(v.y));
                    if (whole) {
                        sum = add2(sum, add2(u, v));
                        const float4 w = vg[ch * 4 + q];
                        u = mul2(u, make_float2(w.x, w.y));
                        v = mul2(v, make_float2(w.z, w.w));
                    } else {
                        float p[4] = {u.x, u.y, v.x, v.y};
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const int j = base + ch * 16 + 4 * q + y;
                            const bool see = j <= hi && (j > lo || j < a.sinks);
                            sum.x += see ? p[y] : 0.f;
                            p[y] = see ? p[y] * exp2_fast(sm.ve[b][ch * 16 + 4 * q + y] - E + 6.f) : 0.f;
                        }
                        u = make_float2(p[0], p[1]);
                        v = make_float2(p[2], p[3]);
                    }
                    split2(u, ph[2 * q], pl[2 * q]);
                    split2(v, ph[2 * q + 1], pl[2 * q + 1]);
                }
                ut_st8(lane_tm + CA_TM_P + ch * 8, ph);
                ut_st8(lane_tm + CA_TM_P + 64 + ch * 8, pl);
            }
            l += sum.x + sum.y;
            ut_wait_st();
            ut_fence_before();
            __syncwarp();
            if (lane == 0) ut_arrive(&sm.p_full);
        }
        // ---- this split's output over its own sum, staged in shared memory
        if (nt > 0) {
            ut_wait(&sm.o_full, 0, abort);
            ut_fence_after();
            gather();
        }
        float* stage = reinterpret_cast<float*>(sm.q) + row * CA_OUT_LD;
        // rows that saw nothing, and dead ones, give zeros
        const float f = l == 0.f || !live ? 0.f : exp2_fast(E - 19.f) / l;
#pragma unroll
        for (int q = 0; q < 32; ++q) {
            float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
            const float2 u = unpack2(acc[2 * q]), v = unpack2(acc[2 * q + 1]);
            if (f != 0.f) w = make_float4(u.x * f, u.y * f, v.x * f, v.y * f);
            *reinterpret_cast<float4*>(stage + 4 * q) = w;
        }
        sm.m[row] = m;
        sm.l[row] = *abort ? __int_as_float(0x7fffffff) : l;  // a wait that ran out shows as NaN
        ut_fence_before();
        warpgroup_sync();
        regs_down<CA_REGS>();
    }
    __syncthreads();
    if (warp >= CA_SOFTMAX_WARPS) regs_up<CA_REGS>();  // what the softmax threads gave back
    if (warp == CA_MMA_WARP) {
        ut_fence_after();
        ut_free(tmem);
    }
    // ---- join the splits: CTA z of the cluster takes a part of the rows
    if (splits > 1)
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int rows_used = nq * c.n_rep;
    const int ra = z * rows_used / splits, rb = (z + 1) * rows_used / splits;
    const uint32_t stage = smem_u32(sm.q);
    for (int q = warp; q < rb - ra; q += CA_THREADS / 32) {  // a warp per row
        const int row = ra + q;
        float4 o;
        float M = CO_LOW, L = 0.f;
        const uint32_t at = stage + (uint32_t)(row * CA_OUT_LD + 4 * lane) * 4u;
        if (splits == 1) {
            o = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm.q) + row * CA_OUT_LD + 4 * lane);
            M = sm.m[row];
            L = sm.l[row];
            if (L != L) o.x = o.y = o.z = o.w = L;
        } else {
            o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int p = 0; p < splits; ++p) M = fmaxf(M, ld_peer(&sm.m[row], p));
            for (int p = 0; p < splits; ++p) {
                const float w = ld_peer(&sm.l[row], p) * exp2_fast(ld_peer(&sm.m[row], p) - M);
                const float4 y = ld_peer4(at, p);
                L += w;
                o.x = fmaf(w, y.x, o.x);
                o.y = fmaf(w, y.y, o.y);
                o.z = fmaf(w, y.z, o.z);
                o.w = fmaf(w, y.w, o.w);
            }
            const float inv = 1.f / L;
            o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        }
        const long long tok = x.b + i0 + row / c.n_rep;
        reinterpret_cast<float4*>(a.out)[(tok * a.H + g * c.n_rep + row % c.n_rep) * 32 + lane] = o;
        if (c.lse && lane == 0) c.lse[tile_at * 128 + row] = M + log2f(L);
    }
    if (splits > 1)  // peers still read this CTA's shared memory
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// -------------------------------------------------------------- chunk_mass
// One CTA per (128 slots, kv head, row): its keys become one split tile, the
// rows of the products; the query tiles that see any of them pass through
// as columns.  A thread owns a slot and half of the columns, so weights are added in
// a fixed order without atomics:
//   sum over columns of exp2(s - lse)
constexpr int CM_SUM_WARPS = 8;                             // two per TMEM quadrant
constexpr int CM_THREADS = 32 * (CM_SUM_WARPS + 1);
constexpr int CM_MMA_WARP = CM_SUM_WARPS;

struct CmSmem {
    unsigned char k[2 * UT_BYTES];
    unsigned char q[2][2 * UT_BYTES];
    float lse[2][128];
    float kc[128];
    float part[2][128];
    uint64_t k_full, q_full[2], q_empty[2], s_full[2], s_empty[2];
    uint32_t tmem;
    int abort;
};
constexpr size_t CM_SMEM = sizeof(CmSmem) + 1024;
static_assert(CM_SMEM <= 227 * 1024, "shared memory of one CTA");

__global__ void __launch_bounds__(CM_THREADS, 1) chunk_mass_kernel(const ChunkArgs c) {
    extern __shared__ unsigned char cm_raw[];
    CmSmem& sm = *reinterpret_cast<CmSmem*>(cm_raw + ((1024u - (smem_u32(cm_raw) & 1023u)) & 1023u));
    const CacheAttnArgs& a = c.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = blockIdx.y, r = blockIdx.z;
    const ChunkRow x = chunk_row(c, r);
    pdl_wait();
    if (x.idle || x.bad || x.n == 0) return;
    const int last = x.cached + x.n - 1;
    // the blockIdx.x-th tile that any query sees
    int tile;
    {
        const int w0 = a.window > 0 ? max(0, x.cached - a.window + 1) : 0;
        const int a1 = (min(a.sinks, w0) + 127) >> 7, b0 = max(w0 >> 7, a1);
        tile = (int)blockIdx.x < a1 ? blockIdx.x : b0 + (blockIdx.x - a1);
    }
    const int base = tile * 128;
    if (base > last) return;
    // queries (slots) that may see a slot of the tile: from `from` to `to`
    const int from = max(base, x.cached);
    int to = last;
    if (a.window > 0 && base >= a.sinks) to = (int)min((long long)to, (long long)base + 127 + a.window - 1);
    if (from > to) return;
    const int t0 = (from - x.cached) / c.P, nt = (to - x.cached) / c.P - t0 + 1;

    if (tid == 0) {
        mbar_init(&sm.k_full, CM_SUM_WARPS);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sm.q_full[b], 1);
            mbar_init(&sm.q_empty[b], 1);
            mbar_init(&sm.s_full[b], 1);
            mbar_init(&sm.s_empty[b], CM_SUM_WARPS);
        }
        mbar_fence_init();
        sm.abort = 0;
    }
    if (warp == CM_MMA_WARP) ut_alloc(&sm.tmem);
    ut_fence_before();
    __syncthreads();
    ut_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* abort = &sm.abort;

    if (warp == CM_MMA_WARP) {
        if (lane == 0) {
            const long long at0 = chunk_tile(c, x, r, t0) * a.kv.KVH + g;
            auto fetch = [&](int i) {
                const long long at = at0 + (long long)i * a.kv.KVH;
                mbar_expect_tx(&sm.q_full[i & 1], 2 * UT_BYTES + 512);
                bulk_g2s(sm.q[i & 1], c.qtiles + at * (2 * UT_BYTES), 2 * UT_BYTES, &sm.q_full[i & 1]);
                bulk_g2s(sm.lse[i & 1], c.lse + at * 128, 512, &sm.q_full[i & 1]);
            };
            int fetched = 0;
            for (; fetched < 2 && fetched < nt; ++fetched) fetch(fetched);
            bool go = ut_wait(&sm.k_full, 0, abort);
            int i = 0;
            for (; i < nt && go; ++i) {
                go = ut_wait(&sm.q_full[i & 1], (i >> 1) & 1, abort);
                if (go && i >= 2) go = ut_wait(&sm.s_empty[i & 1], ((i - 2) >> 1) & 1, abort);
                if (!go) break;
                ut_fence_after();
                ut_mma_qk(tmem + (i & 1) * 128, smem_u32(sm.k), smem_u32(sm.q[i & 1]));
                ut_commit(&sm.q_empty[i & 1]);
                ut_commit(&sm.s_full[i & 1]);
                // the other buffer's tile: its products are done and its
                // sums read (they use the tile's lse) before it is refilled
                if (i >= 1 && i + 1 < nt) {
                    go = ut_wait(&sm.q_empty[(i - 1) & 1], ((i - 1) >> 1) & 1, abort) &&
                         ut_wait(&sm.s_empty[(i - 1) & 1], ((i - 1) >> 1) & 1, abort);
                    if (go) {
                        fetch(i + 1);
                        ++fetched;
                    }
                }
            }
            // leave nothing in flight: the copies asked for, the products issued
            if (i < nt)
                for (int f = max(0, fetched - 2); f < fetched; ++f) mbar_wait(&sm.q_full[f & 1], (f >> 1) & 1, nullptr);
        }
        __syncwarp();
    } else {
        {  // the keys, 16 rows a warp
            const float4* pool4 = reinterpret_cast<const float4*>(a.kv.pool) + lane;
            const float qfac = pow2_whole(query_exponent(a.qn, lane) - 13.f);
            float4 d[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int slot = base + warp * 16 + j;
                d[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (slot <= last) {
                    const long long u = a.kv.key_unit(r, slot, g);
                    if (u >= 0) d[j] = __ldcg(pool4 + u * 32);
                    else d[j].x = __int_as_float(0x7fffffff);
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float e = row_exponent(d[j]);
                put_row(sm.k, warp * 16 + j, lane, d[j], e);
                if (lane == 0) sm.kc[warp * 16 + j] = e == e ? pow2_whole(fmaxf(e, -100.f) - 13.f) * qfac : e;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) ut_arrive(&sm.k_full);
            asm volatile("bar.sync 2, 256;" ::: "memory");
        }
        const int key = 32 * (warp & 3) + lane, half = warp >> 2, slot = base + key;
        const float kc = sm.kc[key];
        const uint32_t lane_tm = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + half * 64;
        const bool sink = slot < a.sinks;
        float2 sum = make_float2(0.f, 0.f);
        for (int i = 0; i < nt; ++i) {
            const int b = i & 1;
            const int first = x.cached + (t0 + i) * c.P;            // slot of the tile's first query
            const int nq = min(c.P, last + 1 - first);
            // seen whole: every column is a query, behind every slot, inside the window
            const bool whole = nq * c.n_rep == 128 && first >= base + 127 &&
                               (a.window == 0 || first + nq - 1 - base < a.window || base + 128 <= a.sinks);
            if (!ut_wait(&sm.s_full[b], (i >> 1) & 1, abort)) break;
            // also waited for: the lse that came with the tile
            if (!ut_wait(&sm.q_full[b], (i >> 1) & 1, abort)) break;
            ut_fence_after();
#pragma unroll 1
            for (int ch = 0; ch < 2; ++ch) {
                uint32_t s[32];
                ut_ld32(lane_tm + b * 128 + ch * 32, s);
                ut_wait_ld();
                const float4* lse = reinterpret_cast<const float4*>(sm.lse[b] + half * 64 + ch * 32);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float4 f = lse[q];
                    const float2 k2 = make_float2(kc, kc);
                    float2 u = fma2(make_float2(__uint_as_float(s[4 * q]), __uint_as_float(s[4 * q + 1])), k2,
                                    make_float2(-f.x, -f.y));
                    float2 v = fma2(make_float2(__uint_as_float(s[4 * q + 2]), __uint_as_float(s[4 * q + 3])), k2,
                                    make_float2(-f.z, -f.w));
                    float p[4] = {exp2_fast(u.x), exp2_fast(u.y), exp2_fast(v.x), exp2_fast(v.y)};
                    if (!whole) {
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const int col = half * 64 + ch * 32 + 4 * q + y, qi = col / c.n_rep, own = first + qi;
                            const bool see = qi < nq && slot <= own && (a.window == 0 || own - slot < a.window || sink);
                            if (!see) p[y] = 0.f;
                        }
                    }
                    sum = add2(sum, add2(make_float2(p[0], p[1]), make_float2(p[2], p[3])));
                }
            }
            ut_fence_before();
            __syncwarp();
            if (lane == 0) ut_arrive(&sm.s_empty[b]);
        }
        sm.part[half][key] = sum.x + sum.y;
    }
    __syncthreads();
    if (warp == CM_MMA_WARP) {
        ut_fence_after();
        ut_free(tmem);
    }
    const int slot = base + tid;
    if (tid < 128 && slot <= last) {
        float s = sm.part[0][tid] + sm.part[1][tid];
        if (*abort) s = __int_as_float(0x7fffffff);
        float* mass = a.mass + (((long long)r * a.kv.KVH + g) * a.kv.max_pages << a.kv.page_log2) + slot;
        *mass = slot >= x.cached ? s : *mass + s;
    }
}

static int64_t align256(int64_t n) { return (n + 255) & ~255ll; }
static int64_t chunk_tiles(int tokens, int rows, int n_rep) { return tokens / (128 / n_rep) + rows + 1; }

}  // namespace skb

using namespace skb;

extern "C" int64_t skb_chunk_attention_workspace(int tokens, int rows, int max_chunk, int n_heads, int n_kv_heads,
                                                 int max_pages, int page_size, int with_mass) {
    if (tokens < 0 || rows < 0 || max_chunk < 0 || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads != 0 ||
        n_heads / n_kv_heads > CO_MAX_REP || max_pages < 1 || page_size < 1)
        return -1;
    const int64_t tiles = chunk_tiles(tokens, rows, n_heads / n_kv_heads) * n_kv_heads;
    return tiles * (2 * (int64_t)UT_BYTES) + (with_mass ? align256(tiles * 512) : 0);
}

extern "C" int skb_chunk_attention(const float* qkv, int tokens, int rows, int n_heads, int n_kv_heads, int head_dim,
                                   const float* q_norm, const float* k_norm, float eps, const float* rope_cos,
                                   const float* rope_sin, int max_pos, const int32_t* chunk_start, int max_chunk,
                                   const int32_t* cached, const int32_t* pos, float* kv_pool,
                                   const int32_t* page_table, int max_pages, int page_size, int n_pages, int window,
                                   int sinks, float* mass, void* work, int64_t work_bytes, float* out,
                                   cudaStream_t stream) {
    const char* what = "chunk_attention";
    const int st = cache_attn_check(what, qkv, rows, n_heads, n_kv_heads, head_dim, q_norm, k_norm, rope_cos, rope_sin,
                                    max_pos, cached, pos, kv_pool, page_table, max_pages, page_size, n_pages, window,
                                    sinks, out);
    if (st != SKB_OK) return st;
    if (!chunk_start) return fail(SKB_ERR_ARG, "%s: null pointer", what);
    if (tokens < 0 || max_chunk < 0) return fail(SKB_ERR_ARG, "%s: bad sizes", what);
    if ((long long)n_pages * 2 * n_kv_heads * page_size >= 0xfffffffell)
        return fail(SKB_ERR_ARG, "%s: the pool must hold fewer than 2^32 - 2 key and value rows", what);
    if (rows == 0 || tokens == 0) return SKB_OK;
    if (!qkv || !out) return fail(SKB_ERR_ARG, "%s: null pointer", what);
    if (!work || ((uintptr_t)work & 255u) ||
        work_bytes < skb_chunk_attention_workspace(tokens, rows, max_chunk, n_heads, n_kv_heads, max_pages, page_size, mass != nullptr))
        return fail(SKB_ERR_ARG, "%s: needs a workspace of skb_chunk_attention_workspace bytes, 256-byte aligned", what);
    ChunkArgs c = {};
    c.a.qkv = qkv;
    c.a.qn = q_norm;
    c.a.kn = k_norm;
    c.a.eps = eps;
    c.a.rope_cos = rope_cos;
    c.a.rope_sin = rope_sin;
    c.a.max_pos = max_pos;
    c.a.cached = cached;
    c.a.pos = pos;
    c.a.kv = {kv_pool, page_table, max_pages, log2_of(page_size), n_kv_heads, n_pages};
    c.a.H = n_heads;
    c.a.rows = rows;
    c.a.window = window;
    c.a.sinks = sinks;
    c.a.mass = mass;
    c.a.out = out;
    c.chunk_start = chunk_start;
    c.tokens = tokens;
    c.max_chunk = max_chunk;
    c.n_rep = n_heads / n_kv_heads;
    c.P = 128 / c.n_rep;
    c.qtiles = static_cast<unsigned char*>(work);
    const long long tiles = chunk_tiles(tokens, rows, c.n_rep);
    c.lse = mass ? reinterpret_cast<float*>(c.qtiles + tiles * n_kv_heads * (2 * (long long)UT_BYTES)) : nullptr;

    // no more tokens than there are, whatever max_chunk says
    const int most = max_chunk < 1 ? 1 : (max_chunk < tokens ? max_chunk : tokens);
    const int tiles_x = (most + c.P - 1) / c.P;
    const long long cap = (long long)max_pages * page_size;
    // CTAs that have work, at most; while they leave SMs idle, up to 8 share a
    // query tile's key tiles.  A row's keys are not known here; the cache, or
    // the window, bounds them.
    long long ctas = (long long)rows * tiles_x;
    if (ctas > tiles) ctas = tiles;
    ctas *= n_kv_heads;
    long long seen = cap;
    if (window > 0 && (long long)window + sinks + c.P < cap) seen = (long long)window + sinks + c.P;
    const long long key_tiles = seen / 128 + 1;
    int splits = 1;
    while (splits < CA_MAX_SPLITS && ctas * splits * 2 <= 148 && splits * 2 <= key_tiles) splits *= 2;

    cudaError_t e = set_smem_attrs(chunk_attn_kernel, CA_SMEM);
    if (e == cudaSuccess && mass) e = set_smem_attrs(chunk_mass_kernel, CM_SMEM);
    if (e == cudaSuccess)
        e = launch(chunk_prep_kernel, dim3(most < 4096 ? most : 4096, rows, (n_heads + 2 * n_kv_heads + 7) / 8), dim3(256),
                   0, stream, false, c);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(splits * tiles_x, n_kv_heads, rows);
        cfg.blockDim = dim3(CA_THREADS);
        cfg.dynamicSmemBytes = CA_SMEM;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = splits;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, chunk_attn_kernel, c, splits);
    }
    if (e == cudaSuccess && mass) {
        // tiles that the row's queries see: the sinks' and the window's, or all
        long long n = (cap + 127) / 128;
        if (window > 0) {
            const long long w = ((long long)sinks + 127) / 128 + ((long long)window + most + 127) / 128 + 1;
            if (w < n) n = w;
        }
        e = launch(chunk_mass_kernel, dim3((unsigned)n, n_kv_heads, rows), dim3(CM_THREADS), CM_SMEM, stream, true, c);
    }
    return e == cudaSuccess ? SKB_OK : fail(SKB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
