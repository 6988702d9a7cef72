// Attention of a chunk of new tokens per row over the paged cache: ragged
// chunks behind each row's cached slots, causal, with an optional sliding
// window and sinks, and optionally the attention weights added up per slot.
//   q_i, k_i = RoPE(RMSNorm(.)) at pos[row] + i;  k_i, v_i -> slot cached[row] + i
//   o_ih = sum_j p_ihj v_j,  p_ihj = exp(q_ih.k_j / sqrt(128) - lse_ih) over the slots i sees
//   mass[row][g][j] += sum_i sum over g's heads of p_ihj  (new slots begin at zero)
//
//   chunk_prep  norms, rotates and appends; queries to the workspace
//   chunk_attn  one warp per (token, kv head)
//   chunk_mass  one warp per (slot, kv head)
#include "cache_ops.cuh"

namespace skb {

struct ChunkArgs {
    CacheAttnArgs a;
    const int* chunk_start;  // [rows + 1]
    int tokens, max_chunk;
    float* q;    // workspace [tokens][H][128]: queries, scaled to log2 units
    float* lse;  // workspace [tokens][H] (mass only), log2 units
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

// grid (min(max_chunk, 1024), rows), 256 threads: warp w takes head vectors w, w + 8, ...
__global__ void __launch_bounds__(256) chunk_prep_kernel(const ChunkArgs c) {
    const CacheAttnArgs& a = c.a;
    const int r = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const ChunkRow x = chunk_row(c, r);
    const int H = a.H, KVH = a.kv.KVH;
    for (int i = blockIdx.x; i < x.n; i += gridDim.x) {
        const long long t = x.b + i;
        if (x.idle || x.bad) {
            const float v = x.idle ? 0.f : __int_as_float(0x7fffffff);
            for (int d = threadIdx.x; d < H * 128; d += 256) a.out[t * H * 128 + d] = v;
            continue;
        }
        const int pos = a.pos[r] + i, slot = x.cached + i;
        const float4* row = reinterpret_cast<const float4*>(a.qkv + t * (H + 2 * KVH) * 128);
        const float* cosr = a.rope_cos + (long long)pos * 64;
        const float* sinr = a.rope_sin + (long long)pos * 64;
        for (int v = warp; v < H + 2 * KVH; v += 8) {
            float4 y = row[v * 32 + lane];
            if (v < H) {
                y = norm_rope_head(y, a.qn, a.eps, cosr, sinr, lane, true, true);
                const float s = 0.08838834764831845f * CO_LOG2E;  // 1 / sqrt(128), scores in log2 units
                reinterpret_cast<float4*>(c.q)[(t * H + v) * 32 + lane] = make_float4(y.x * s, y.y * s, y.z * s, y.w * s);
                continue;
            }
            const bool value = v >= H + KVH;
            const int g = v - H - (value ? KVH : 0);
            if (!value) y = norm_rope_head(y, a.kn, a.eps, cosr, sinr, lane, true, true);
            const long long u = a.kv.key_unit(r, slot, g);
            if (u >= 0) reinterpret_cast<float4*>(a.kv.pool)[(u + (value ? a.kv.value_step() : 0)) * 32 + lane] = y;
        }
    }
}

// grid (ceil(max_chunk / 8), KVH, rows), 256 threads: warp w takes token 8 blockIdx.x + w
__global__ void __launch_bounds__(256) chunk_attn_kernel(const ChunkArgs c) {
    const CacheAttnArgs& a = c.a;
    const int g = blockIdx.y, r = blockIdx.z, lane = threadIdx.x & 31;
    const ChunkRow x = chunk_row(c, r);
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (x.idle || x.bad || i >= x.n) return;
    const int NR = a.H / a.kv.KVH, own = x.cached + i;
    const int w0 = a.window > 0 ? max(0, own - a.window + 1) : 0, ns = min(a.sinks, w0);
    const float4* pool4 = reinterpret_cast<const float4*>(a.kv.pool);
    for (int h = g * NR; h < (g + 1) * NR; ++h) {
        const long long th = (long long)(x.b + i) * a.H + h;
        const float4 q = reinterpret_cast<const float4*>(c.q)[th * 32 + lane];
        float m = CO_LOW, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int n = 0; n < ns + own + 1 - w0; ++n) {
            const long long u = a.kv.key_unit(r, n < ns ? n : w0 + n - ns, g);
            float s = __int_as_float(0x7fffffff);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (u >= 0) {
                const float4 k = __ldcg(pool4 + u * 32 + lane);
                v = __ldcg(pool4 + (u + a.kv.value_step()) * 32 + lane);
                s = warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w);
            }
            const float mn = fmaxf(m, s), f = exp2_fast(m - mn), p = exp2_fast(s - mn);
            m = mn;
            l = fmaf(l, f, p);
            o = make_float4(fmaf(o.x, f, p * v.x), fmaf(o.y, f, p * v.y), fmaf(o.z, f, p * v.z), fmaf(o.w, f, p * v.w));
        }
        const float inv = 1.f / l;
        reinterpret_cast<float4*>(a.out)[th * 32 + lane] = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        if (c.lse && lane == 0) c.lse[th] = m + log2f(l);
    }
}

// grid (ceil(slots / 8), KVH, rows), 256 threads: warp w takes slot 8 blockIdx.x + w
__global__ void __launch_bounds__(256) chunk_mass_kernel(const ChunkArgs c) {
    const CacheAttnArgs& a = c.a;
    const int g = blockIdx.y, r = blockIdx.z, lane = threadIdx.x & 31;
    const ChunkRow x = chunk_row(c, r);
    const int j = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (x.idle || x.bad || j >= x.cached + x.n) return;
    const int NR = a.H / a.kv.KVH;
    const long long u = a.kv.key_unit(r, j, g);
    const float4 k = u >= 0 ? __ldcg(reinterpret_cast<const float4*>(a.kv.pool) + u * 32 + lane)
                            : make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    for (int i = max(0, j - x.cached); i < x.n; ++i) {
        if (a.window > 0 && x.cached + i - j >= a.window && j >= a.sinks) break;
        for (int h = g * NR; h < (g + 1) * NR; ++h) {
            const long long th = (long long)(x.b + i) * a.H + h;
            const float4 q = reinterpret_cast<const float4*>(c.q)[th * 32 + lane];
            const float s = warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w);
            sum += u >= 0 ? exp2_fast(s - c.lse[th]) : __int_as_float(0x7fffffff);
        }
    }
    float* mass = a.mass + (((long long)r * a.kv.KVH + g) * a.kv.max_pages << a.kv.page_log2) + j;
    if (lane == 0) *mass = j >= x.cached ? sum : *mass + sum;
}

static int64_t align256(int64_t n) { return (n + 255) & ~255ll; }

}  // namespace skb

using namespace skb;

extern "C" int64_t skb_chunk_attention_workspace(int tokens, int rows, int max_chunk, int n_heads, int n_kv_heads,
                                                 int max_pages, int page_size, int with_mass) {
    if (tokens < 0 || rows < 0 || max_chunk < 0 || n_heads < 1 || n_kv_heads < 1 || max_pages < 1 || page_size < 1)
        return -1;
    return align256((int64_t)tokens * n_heads * 512) + (with_mass ? align256((int64_t)tokens * n_heads * 4) : 0);
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
    c.q = static_cast<float*>(work);
    c.lse = mass ? reinterpret_cast<float*>(static_cast<char*>(work) + align256((int64_t)tokens * n_heads * 512)) : nullptr;
    const int most = max_chunk < 1 ? 1 : max_chunk;
    cudaError_t e = launch(chunk_prep_kernel, dim3(most < 1024 ? most : 1024, rows), dim3(256), 0, stream, false, c);
    if (e == cudaSuccess)
        e = launch(chunk_attn_kernel, dim3((most + 7) / 8, n_kv_heads, rows), dim3(256), 0, stream, false, c);
    if (e == cudaSuccess && mass)
        e = launch(chunk_mass_kernel, dim3((unsigned)(((long long)max_pages * page_size + 7) / 8), n_kv_heads, rows),
                   dim3(256), 0, stream, false, c);
    return e == cudaSuccess ? SKB_OK : fail(SKB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
