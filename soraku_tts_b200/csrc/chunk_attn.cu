// Attention of a chunk of new tokens per row over the paged cache: ragged
// chunks behind each row's cached slots, causal, with an optional sliding
// window and sinks, and optionally the attention weights added up per slot.
//   q_i, k_i = RoPE(RMSNorm(.)) at pos[row] + i;  k_i, v_i -> slot cached[row] + i
//   o_ih = sum_j p_ihj v_j,  p_ihj = exp(q_ih.k_j / sqrt(128) - lse_ih) over the slots i sees
//   mass[row][g][j] += sum_i sum over g's heads of p_ihj  (new slots begin at zero)
//
// Three launches.  chunk_prep norms, rotates and appends the new keys and
// values, and writes queries, and all keys and values that are seen, as split
// fp16 tiles (umma.cuh) in the order in which the tensor cores read them;
// chunk_attn; and, with `mass`, chunk_mass.  The tiles are written once for
// all query tiles of a row: splitting them inside chunk_attn, per query tile,
// took its warps 7 to 11 thousand cycles a key tile, against 4 thousand now.
// chunk_prep is bound by memory (8 prompts of 611 to 1024 tokens: 270 MB in 55
// us, 4.9 TB/s), chunk_attn by the softmax of a tile (4 thousand cycles, beside
// 3.1 thousand of products) and, in short rows, by the 9 thousand cycles in which a
// CTA fills and drains its pipeline (the 8 prompts: 108 us; 512 tokens behind
// 8192 slots: 90 us, 1.2 PFLOP/s of fp16 products, 70 % of what a library's
// bf16 product reaches).
// A query tile is 128 (token, head) pairs of one kv head, P = 128 / n_rep
// tokens, so a key or value tile that was loaded once serves all of them.
#include <type_traits>

#include "umma.cuh"

namespace skb {

struct ChunkArgs {
    CacheAttnArgs a;
    const int* chunk_start;  // [rows + 1]
    int tokens, max_chunk;
    int n_rep, P;           // heads per kv head, tokens per query tile
    unsigned rep_inv;       // for over_rep
    // workspace
    unsigned char* qtiles;  // [query tiles][KVH][2 UT_BYTES]: queries in log2 units, hi | lo
    unsigned char* kvtiles; // [key tiles][KVH][2][2 UT_BYTES]: keys, values, hi | lo
    float* meta;            // [key tiles][KVH][2][128]: factor of a key's scores; exponent of a value row
    float* lse;             // [query tiles][KVH][128] (mass only), log2 units
    struct RowJob* jobs;    // [rows]: by the tiles they see, most first; null: rows as they are
    int key_tiles;
    bool roomy;             // they are enough for any rows, even ones that claim more than the pool has
};

// x / n_rep without a division; right for x below 2^22 at least.
__device__ __forceinline__ int over_rep(const ChunkArgs& c, int x) {
    return (int)((unsigned long long)(unsigned)x * c.rep_inv >> 24);
}

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

// A row as chunk_attn takes it: one read in place of a chain of three.
struct __align__(32) RowJob {
    int row, b, n, cached;
    int first, tiles;  // its query tiles among those of all rows, in the order of the jobs
    long long base;    // where its key tiles begin in the workspace
};

// The tiles of 128 slots that any query of a row sees: [0, a1) for the sinks,
// [b0, end) for the windows.
struct RowTiles {
    int a1, b0, n, w0;
    __device__ __forceinline__ RowTiles(const ChunkArgs& c, const ChunkRow& x) {
        w0 = c.a.window > 0 ? max(0, x.cached - c.a.window + 1) : 0;  // first slot of the first query's window
        a1 = (min(c.a.sinks, w0) + 127) >> 7;
        b0 = max(w0 >> 7, a1);
        n = x.idle || x.bad || x.n == 0 ? 0 : a1 + ((x.cached + x.n - 1) >> 7) + 1 - b0;
    }
    __device__ __forceinline__ int index(int tile) const { return tile < a1 ? tile : a1 + tile - b0; }
    __device__ __forceinline__ int tile(int k) const { return k < a1 ? k : b0 + k - a1; }
};
// Whether every slot in sight of a row has a page.  By a whole warp.
__device__ __forceinline__ bool row_mapped(const ChunkArgs& c, int r, const ChunkRow& x, const RowTiles& rt) {
    const int lane = threadIdx.x & 31, lg = c.a.kv.page_log2;
    const int* table = c.a.kv.page_table + (long long)r * c.a.kv.max_pages;
    bool all = true;
    auto look = [&](int p0, int p1) {
        for (; all && p0 <= p1; p0 += 128) {
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int p = p0 + 32 * j + lane;
                if (p <= p1) bad |= (unsigned)__ldg(table + p) >= (unsigned)c.a.kv.n_pages;
            }
            all = !__any_sync(FULL, bad);
        }
    };
    const int sinks = min(c.a.sinks, rt.w0);
    if (sinks > 0) look(0, (sinks - 1) >> lg);
    look(rt.w0 >> lg, (x.cached + x.n - 1) >> lg);
    return all;
}
// row_base where the rows see more than the pool can hold, so that some see
// slots without a page: room for the others alone.  Every warp goes through the
// rows one by one, 1 us each, so only for up to CP_SORTED of them; of more, those
// before the first that finds no room have theirs, in the plain order.
constexpr int CP_SORTED = 512;   // more rows than that are taken as they come
__device__ __forceinline__ int row_base_mapped(const ChunkArgs& c, int r, int before) {
    if (c.a.rows > CP_SORTED)
        return before + RowTiles(c, chunk_row(c, r)).n <= c.key_tiles ? before : -1;
    int base = 0;
    for (int p = 0; p <= r; ++p) {
        const ChunkRow x = chunk_row(c, p);
        const RowTiles rt(c, x);
        // the count first: a row that is longer than the pool is not looked through
        const bool place = rt.n > 0 && base + rt.n <= c.key_tiles && row_mapped(c, p, x, rt);
        if (p == r) return place ? base : -1;
        if (place) base += rt.n;
    }
    return -1;
}
// Where a row's key tiles begin in the workspace: behind those of the rows
// before it; -1 if there is no room for them.  By a whole warp.  Rows may claim
// 2^23 tiles each, so a lane's sum stops at CHUNK_TILES, which is more than any
// workspace holds (and 32 such sums are less than 2^31).
constexpr int CHUNK_TILES = 1 << 25;
__device__ __forceinline__ int row_base(const ChunkArgs& c, int r) {
    int before = 0, all = 0;
    const int rows = c.roomy ? r : c.a.rows;
    for (int p = threadIdx.x & 31; p < rows; p += 32) {
        all = min(all + RowTiles(c, chunk_row(c, p)).n, CHUNK_TILES);
        if (p < r) before = all;
    }
    before = __reduce_add_sync(FULL, before);
    if (!c.roomy && __reduce_add_sync(FULL, all) > c.key_tiles) return row_base_mapped(c, r, before);
    return before;
}

// A whole number e with |q| < 2^e for every query in log2 units: a normed head
// is at most sqrt(128) max|w| long per element, its rotation sqrt(2) times that.
__device__ __forceinline__ float query_exponent(const float* qn, int lane) {
    const float4 w = __ldg(reinterpret_cast<const float4*>(qn) + lane);
    const float m = warp_max(fmaxf(fmaxf(fabsf(w.x), fabsf(w.y)), fmaxf(fabsf(w.z), fabsf(w.w))));
    const int e = (int)(__float_as_uint(m * 2.0405f) >> 23) - 126;
    return (float)max(-100, min(127, e));
}

// A head vector, a float4 per lane: RMSNorm with weight w, then rotated.
__device__ __forceinline__ float4 norm_rope(float4 x, float4 w, float eps, float4 c, float4 s, int lane) {
    const float inv = rsqrtf(warp_sum(x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w) / 128.0f + eps);
    x = make_float4(w.x * (x.x * inv), w.y * (x.y * inv), w.z * (x.z * inv), w.w * (x.w * inv));
    float4 o;  // the other half's: 64 elements away
    o.x = __shfl_xor_sync(FULL, x.x, 16);
    o.y = __shfl_xor_sync(FULL, x.y, 16);
    o.z = __shfl_xor_sync(FULL, x.z, 16);
    o.w = __shfl_xor_sync(FULL, x.w, 16);
    const float t = lane < 16 ? -1.f : 1.f;
    return make_float4(x.x * c.x + t * (o.x * s.x), x.y * c.y + t * (o.y * s.y), x.z * c.z + t * (o.z * s.z),
                       x.w * c.w + t * (o.w * s.w));
}

constexpr float CH_QSCALE = 0.08838834764831845f * CO_LOG2E;  // 1 / sqrt(128), scores in log2 units

constexpr int CP_TILES = 64;     // blocks side by side over a row's key tiles
constexpr int CP_NQ = 2;         // groups of four rows a warp holds at once

// The first `token_blocks` blocks: `per_block` new tokens each (1, 2 or 4), 8 /
// per_block warps to a token, which take its head vectors in turn.  Few tokens
// are spread over many warps, many share a warp's look at their row's numbers.
// The next block puts the rows in order.  The others: cached slots, a block per
// (key tile, keys or values, kv head, row).
__global__ void __launch_bounds__(256, 4) chunk_prep_kernel(const __grid_constant__ ChunkArgs c, int token_blocks, int per_block, int tiles_x) {
    const CacheAttnArgs& a = c.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int H = a.H, KVH = a.kv.KVH, nv = H + 2 * KVH;
    pdl_trigger();
    const float eq = query_exponent(a.qn, lane);
    const float qfac = pow2_whole(eq - 13.f);
    if ((int)blockIdx.x < token_blocks) {
        const int wpt = 8 / per_block, w = warp % wpt;
        const int t = blockIdx.x * per_block + warp / wpt;
        if (t >= c.tokens) return;
        // r: rows that end at or before the token; with them row_base, in one
        // look at the rows' numbers
        int r = 0, before = 0, all = 0;
        for (int p = lane; p - lane < a.rows; p += 32) {
            bool ends = false;
            if (p < a.rows) {
                const int n = RowTiles(c, chunk_row(c, p)).n;
                ends = c.chunk_start[p + 1] <= t;
                all = min(all + n, CHUNK_TILES);
                if (ends) before = all;
            }
            r += __popc(__ballot_sync(FULL, ends));
        }
        if (r >= a.rows) return;
        ChunkRow x = chunk_row(c, r);
        const int i = t - x.b;
        if (i < 0 || i >= x.n) return;
        const RowTiles rt(c, x);
        int base = __reduce_add_sync(FULL, before);
        if (!c.roomy && __reduce_add_sync(FULL, all) > c.key_tiles) base = row_base_mapped(c, r, base);
        // (rows that begin before the one ahead ends are counted otherwise elsewhere)
        if (base < 0 || base + rt.n > c.key_tiles) x.bad = true;
        if (x.idle || x.bad) {
            const float o = x.idle ? 0.f : __int_as_float(0x7fffffff);
            for (int v = w; v < H; v += wpt)
                reinterpret_cast<float4*>(a.out)[((long long)t * H + v) * 32 + lane] = make_float4(o, o, o, o);
            return;
        }
        const int pos = a.pos[r] + i, slot = x.cached + i;
        const float4* row = reinterpret_cast<const float4*>(a.qkv) + (long long)t * nv * 32 + lane;
        // what all vectors of the token share, in registers
        const float4 cs = reinterpret_cast<const float4*>(a.rope_cos + (long long)pos * 64)[lane & 15];
        const float4 sn = reinterpret_cast<const float4*>(a.rope_sin + (long long)pos * 64)[lane & 15];
        const float4 qw = __ldg(reinterpret_cast<const float4*>(a.qn) + lane);
        const float4 kw = __ldg(reinterpret_cast<const float4*>(a.kn) + lane);
        const long long tile = base + rt.index(slot >> 7), unit0 = a.kv.key_unit(r, slot, 0);
        const int qrow = i % c.P * c.n_rep;
        unsigned char* qtile = c.qtiles + chunk_tile(c, x, r, i / c.P) * KVH * (2 * UT_BYTES);
        for (int v0 = w; v0 < nv; v0 += 4 * wpt) {
            float4 y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v0 + wpt * j < nv) y[j] = row[(v0 + wpt * j) * 32];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int v = v0 + wpt * j;
                if (v >= nv) break;
                if (v < H + KVH) y[j] = norm_rope(y[j], v < H ? qw : kw, a.eps, cs, sn, lane);
                if (v < H) {
                    const int g = over_rep(c, v), m = qrow + v - g * c.n_rep;
                    put4(qtile + (long long)g * (2 * UT_BYTES) + ut_at(m, lane), y[j], CH_QSCALE * pow2_whole(13.f - eq));
                    continue;
                }
                const int value = v >= H + KVH, g = v - H - (value ? KVH : 0);
                const long long u = unit0 < 0 ? -1 : unit0 + ((long long)g << a.kv.page_log2);
                if (u >= 0) reinterpret_cast<float4*>(a.kv.pool)[(u + (value ? a.kv.value_step() : 0)) * 32 + lane] = y[j];
                float top = max3_abs(max3_abs(y[j].x, y[j].y, y[j].z), y[j].w, 0.f);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = max3_abs(top, __shfl_xor_sync(FULL, top, o), 0.f);
                const float e = u >= 0 ? top_exponent(top) : __int_as_float(0x7fffffff);
                if (!(e >= -100.f)) y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                put4(c.kvtiles + ((tile * KVH + g) * 2 + value) * (2 * UT_BYTES) + ut_at(slot & 127, lane), y[j], row_scale(e));
                if (lane == 0)
                    c.meta[((tile * KVH + g) * 2 + value) * 128 + (slot & 127)] =
                        value ? e : e == e ? pow2_whole(fmaxf(e, -100.f) - 13.f) * qfac : e;
            }
        }
        return;
    }
    int b = blockIdx.x - token_blocks;
    if (b == 0 && c.jobs) {  // the order in which chunk_attn takes the rows
        __shared__ int seen[CP_SORTED], tiles[CP_SORTED];
        __shared__ unsigned long long all;  // 512 rows of up to 2^23 tiles
        if (threadIdx.x == 0) all = 0;
        __syncthreads();
        for (int p = threadIdx.x; p < a.rows; p += 256) {
            const ChunkRow x = chunk_row(c, p);
            seen[p] = RowTiles(c, x).n;
            tiles[p] = seen[p] == 0 ? 0 : (x.n + c.P - 1) / c.P;
            atomicAdd(&all, (unsigned long long)seen[p]);
        }
        __syncthreads();
        if (all > (unsigned long long)c.key_tiles) {  // rows without room are left out
            for (int p = warp; p < a.rows; p += 8)
                if (row_base_mapped(c, p, 0) < 0 && lane == 0) seen[p] = tiles[p] = 0;
            __syncthreads();
        }
        for (int p = threadIdx.x; p < a.rows; p += 256) {
            int rank = 0, first = 0;
            long long base = 0;
            for (int q = 0; q < a.rows; ++q) {
                const bool ahead = seen[q] > seen[p] || (seen[q] == seen[p] && q < p);
                rank += ahead;
                first += ahead ? tiles[q] : 0;
                base += q < p ? seen[q] : 0;
            }
            const ChunkRow x = chunk_row(c, p);
            c.jobs[rank] = RowJob{p, x.b, x.n, x.cached, first, tiles[p], base};
        }
        return;
    }
    if (c.jobs) --b;
    const int k0 = b % tiles_x;
    b /= tiles_x;
    const int value = b & 1, g = (b >> 1) % KVH, r = (b >> 1) / KVH;
    const ChunkRow x = chunk_row(c, r);
    const int base = row_base(c, r);  // asked for beside the row's own numbers
    const RowTiles rt(c, x);
    if (k0 >= rt.n || base < 0) return;
    const float* pool = a.kv.pool + (value ? a.kv.value_step() * 128 : 0);
    const int row0 = warp * 16, i4 = lane >> 3, last = x.cached + x.n - 1;
    for (int k = k0; k < rt.n; k += tiles_x) {
        const int first = rt.tile(k) * 128 + row0;
        if (first >= x.cached && first + 15 <= last) continue;  // new tokens only: theirs are written above
        const long long at = ((long long)(base + k) * KVH + g) * 2 + value;
        uint32_t units[4];  // of this lane's rows i4, 4 + i4, ...: one look at the page table
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int slot = first + 4 * q + i4;
            units[q] = UT_NONE;
            if (slot < x.cached && (slot >= rt.w0 || slot < a.sinks)) {
                const long long u = a.kv.key_unit(r, slot, g);
                units[q] = u < 0 ? UT_BAD : (uint32_t)u;
            }
        }
#pragma unroll
        for (int part = 0; part < 16; part += 4 * CP_NQ) {
            RowSet<CP_NQ> d;
            uint32_t unit[CP_NQ];
#pragma unroll
            for (int q = 0; q < CP_NQ; ++q) unit[q] = units[part / 4 + q];
#pragma unroll
            for (int q = 0; q < CP_NQ; ++q) d.load(q, pool, unit[q], lane);
#pragma unroll
            for (int q = 0; q < CP_NQ; ++q) {
                const float e = d.exponent(q, unit[q]);
                const int row = row0 + part + 4 * q + i4, slot = first - row0 + row;
                if (slot >= x.cached && slot <= last) continue;
                d.put(q, c.kvtiles + at * (2 * UT_BYTES), row0 + part, row_scale(e), lane);
                if ((lane & 7) == 0)  // (a value that is not there counts among no exponents)
                    c.meta[at * 128 + row] = value ? (unit[q] == UT_NONE ? __int_as_float(0x7fffffff) : e)
                                             : e == e ? pow2_whole(fmaxf(e, -100.f) - 13.f) * qfac
                                                      : e;
            }
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
    int w0, last;            // first slot of any query's window; the last slot seen
    __device__ __forceinline__ TileList(int own_lo, int own_hi, int window, int sinks) {
        w0 = window > 0 ? max(0, own_lo - window + 1) : 0;
        last = own_hi;
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
// A CTA takes one query tile and a part of the key tiles it sees:
//   warp P     asks for key and value tiles, 64 KB bulk copies into three
//              stages, in the order K0 K1 V0 K2 V1 ...
//   warp M, O  issue the products: S_i = Q K_i, a tile ahead, and O = P_i V_i.
//              Two warps, so that neither product stands behind the other's waits
//   warp E     a tile's factors and exponents from the workspace, and the
//              running exponent of the values
//   softmax    CA_PARTS threads per query row, each with a part of a tile's
//              keys and of the output's columns
// Queries stay in tensor memory; weights overwrite their scores there; each
// tile's output is added up in registers.
constexpr int CA_PARTS = 4;
constexpr int CA_W = 128 / CA_PARTS;  // a thread's keys, and its output columns
static_assert(CA_W == 32, "a part is a warp's width");
constexpr int CA_SOFTMAX_WARPS = 4 * CA_PARTS, CA_WARP_M = CA_SOFTMAX_WARPS, CA_WARP_P = CA_WARP_M + 1,
              CA_WARP_E = CA_WARP_M + 2, CA_WARP_O = CA_WARP_M + 3;
constexpr int CA_THREADS = 32 * (CA_SOFTMAX_WARPS + 4);
constexpr int CA_STAGES = 3;
// TMEM columns: two score tiles, a tile's output, the queries
constexpr uint32_t CA_TM_O = 256, CA_TM_Q = 384;
constexpr int CA_OUT_LD = 132;  // floats of a staged output row
constexpr int CA_MAX_SPLITS = 8;
// Weights are held as p 2^(e - E + CA_UP) in fp16 pairs, e the exponent of the
// value row, whose own numbers are below 2^14.  A pair resolves 2^-25 whatever it
// holds, so what counts is where a query's largest contribution p 2^e lies.
//   Values of like sizes: E is set by the first tile, CA_ABOVE above its largest e
//   (or, where queries see different parts of it, above one e that they share),
//   and serves as long as every e in sight lies in [E - CA_SPREAD, E].  The factors
//   2^(e - E + CA_UP) are then the same for all queries, and the key with the largest
//   weight, 1/2 at least, gives 2^(CA_UP - CA_SPREAD - 1) = 4, or 2^27 times the resolution.
//   Else (one large value that hardly anybody looks at, a zero one that all look
//   at) E follows the query's largest contribution from that tile on, and each weight
//   is formed by an exponential of its own beside the one that goes into the sum
//   (8 prompts: 194 us a call instead of 166).
// Which of them holds goes by the values that the query sees, and no other.
constexpr float CA_UP = 12.f, CA_ABOVE = 3.f, CA_SPREAD = 9.f;
constexpr float CA_SLACK = 3.f;  // how far a score, or a contribution, may pass its reference: 2^(12 + 3) fits fp16

struct CaSmem {
    unsigned char stage[CA_STAGES][2 * UT_BYTES];
    float kc[2][128];                    // factor of a key's scores: its scale undone
    float ve[2][128];                    // exponent of a value row
    float vg[2][128];                    // factor of its weights: 2^(exponent - E + CA_UP)
    float mx[2][CA_PARTS][128];          // a row part's largest score,
    float ex[2][CA_PARTS][128], lo[2][CA_PARTS][128];  // its largest and smallest value exponent,
    float cx[CA_PARTS][128];             // its largest contribution
    float m[128], l[CA_PARTS][128];      // this split's statistics (sums of row parts)
    float E[2];                          // E of the tiles that all queries see whole; inf: it follows the contributions
    float top[2], low[2];                // largest and smallest exponent of a tile's values
    float own_vg[CA_SOFTMAX_WARPS][CA_W];  // a warp's factors in a tile that is not whole
    uint64_t q_landed, q_full, full[CA_STAGES], empty[CA_STAGES], s_full[2], p_full[2], pv_done[2], o_free, meta_full[2];
    uint64_t s_end, o_full;  // every product of warp M, of warp O
    // what the CTA works on
    TileList list;
    int k0, nt;          // its key tiles: list entries [k0, k0 + nt)
    int live;            // rows that are queries
    int own[128];        // a row's slot; -1: no query
    int token0;          // token of the first query
    long long tile_at;   // query tile in the workspace
    uint32_t tmem;
    int abort;
};
constexpr size_t CA_SMEM = sizeof(CaSmem) + 1024;
static_assert(CA_SMEM <= 227 * 1024, "shared memory of one CTA");
static_assert(128 * CA_OUT_LD * 4 <= CA_STAGES * 2 * UT_BYTES, "the staged output lies over the tiles");

// The warps that share a quadrant's 32 rows.
__device__ __forceinline__ void softmax_sync() {
    asm volatile("bar.sync %0, %1;" ::"r"(2 + ((threadIdx.x >> 5) & 3)), "n"(32 * CA_PARTS) : "memory");
}

// The same; whether any of their threads says so.
__device__ __forceinline__ bool softmax_any(bool mine) {
    uint32_t any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.or.pred p, %2, %3, q;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(any)
        : "r"((uint32_t)mine), "r"(2 + ((threadIdx.x >> 5) & 3)), "n"(32 * CA_PARTS)
        : "memory");
    return any != 0;
}

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

// Clusters of `splits` CTAs, one per (query tile, kv head): with jobs in their
// order, a row's last query tile, which sees the most, first; without, in a grid
// (splits * query tiles, KVH, rows) in which rows may have fewer.
__global__ void __launch_bounds__(CA_THREADS, 1) chunk_attn_kernel(const __grid_constant__ ChunkArgs c, int splits) {
    extern __shared__ unsigned char ca_raw[];
    CaSmem& sm = *reinterpret_cast<CaSmem*>(ca_raw + ((1024u - (smem_u32(ca_raw) & 1023u)) & 1023u));
    const CacheAttnArgs& a = c.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int z = blockIdx.x % splits;
    int g, t, r;
    ChunkRow x;
    long long base;
    if (c.jobs) {
        const int unit = blockIdx.x / splits, tile = unit / a.kv.KVH;
        g = unit % a.kv.KVH;
        pdl_wait();
        t = -1;
        for (int p = lane; p - lane < a.rows && t < 0; p += 32) {  // the job that has this tile
            int4 j = make_int4(0, 0, 0, 0), k = j;
            if (p < a.rows) {
                j = reinterpret_cast<const int4*>(c.jobs)[2 * p];
                k = reinterpret_cast<const int4*>(c.jobs)[2 * p + 1];
            }
            const unsigned has = __ballot_sync(FULL, tile >= k.x && tile - k.x < k.y);
            if (has == 0) continue;
            const int src = __ffs(has) - 1;
            r = __shfl_sync(FULL, j.x, src);
            x.b = __shfl_sync(FULL, j.y, src);
            x.n = __shfl_sync(FULL, j.z, src);
            x.cached = __shfl_sync(FULL, j.w, src);
            t = __shfl_sync(FULL, k.y - 1 - (tile - k.x), src);
            base = (long long)(((unsigned long long)(unsigned)__shfl_sync(FULL, k.w, src) << 32) |
                               (unsigned)__shfl_sync(FULL, k.z, src));
        }
        if (t < 0) return;  // the grid holds the most tiles that there could be
        x.idle = x.bad = false;
    } else {
        g = blockIdx.y;
        r = blockIdx.z;
        t = gridDim.x / splits - 1 - blockIdx.x / splits;
        x = chunk_row(c, r);
        base = row_base(c, r);
    }
    const int i0 = t * c.P;
    const RowTiles rt(c, x);
    if (x.idle || x.bad || i0 >= x.n || base < 0) {  // the same for a whole cluster
        pdl_wait();
        return;
    }
    // where a tile of the row's keys lies in the workspace
    auto place = [&](int tile) { return (long long)(base + rt.index(tile)) * a.kv.KVH + g; };
    auto ask = [&](int n, int tile, int value) {  // copy n
        const int s = n % CA_STAGES;
        mbar_expect_tx(&sm.full[s], 2 * UT_BYTES);
        bulk_g2s(sm.stage[s], c.kvtiles + (place(tile) * 2 + value) * (2 * UT_BYTES), 2 * UT_BYTES, &sm.full[s]);
    };
    if (tid == 32 * CA_WARP_P) {
        // the first copies are on their way while the CTA gets ready; the
        // queries by way of the last stage
        mbar_init(&sm.q_landed, 1);
        for (int b = 0; b < CA_STAGES; ++b) mbar_init(&sm.full[b], 1);
        mbar_fence_init();
        const int nq = min(c.P, x.n - i0);
        const TileList list(x.cached + i0, x.cached + i0 + nq - 1, a.window, a.sinks);
        const int k0 = (int)((unsigned)z * (unsigned)list.n / (unsigned)splits);  // z < 8, fewer than 2^23 tiles
        const int k1 = (int)((unsigned)(z + 1) * (unsigned)list.n / (unsigned)splits);
        const long long tile_at = chunk_tile(c, x, r, t) * a.kv.KVH + g;
        pdl_wait();
        if (k0 < k1) {
            mbar_expect_tx(&sm.q_landed, 2 * UT_BYTES);
            bulk_g2s(sm.stage[CA_STAGES - 1], c.qtiles + tile_at * (2 * UT_BYTES), 2 * UT_BYTES, &sm.q_landed);
            ask(0, list.tile(k0), 0);
            if (k0 + 1 < k1) ask(1, list.tile(k0 + 1), 0);
        }
        sm.list = list;
        sm.k0 = k0;
        sm.nt = k1 - k0;
        sm.live = nq * c.n_rep;
        sm.token0 = x.b + i0;
        sm.tile_at = tile_at;
    } else if (tid == 0) {
        mbar_init(&sm.q_full, CA_SOFTMAX_WARPS);
        mbar_init(&sm.o_free, CA_SOFTMAX_WARPS);
        mbar_init(&sm.s_end, 1);
        mbar_init(&sm.o_full, 1);
        for (int b = 0; b < CA_STAGES; ++b) mbar_init(&sm.empty[b], 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sm.s_full[b], 1);
            mbar_init(&sm.p_full[b], CA_SOFTMAX_WARPS);
            mbar_init(&sm.pv_done[b], 1);
            mbar_init(&sm.meta_full[b], 1);
        }
        mbar_fence_init();
        sm.abort = 0;
    }
    if (tid < 128) {
        const int q = over_rep(c, tid);
        sm.own[tid] = q < min(c.P, x.n - i0) ? x.cached + i0 + q : -1;
    }
    if (warp == CA_WARP_M) ut_alloc<512>(&sm.tmem);
    ut_fence_before();
    __syncthreads();
    ut_fence_after();
    const uint32_t tmem = sm.tmem;
    const int nt = sm.nt;
    volatile int* abort = &sm.abort;
    pdl_wait();
    if (c.lse) pdl_trigger();  // chunk_mass follows

    if (warp == CA_WARP_P) {
        if (lane == 0) {
            int n = min(nt, 2);  // copies asked for
            auto fetch = [&](int i, int value) {
                if (n == CA_STAGES - 1 && !ut_wait(&sm.q_full, 0, abort)) return false;  // the queries were there
                if (n >= CA_STAGES && !ut_wait(&sm.empty[n % CA_STAGES], ((n - CA_STAGES) / CA_STAGES) & 1, abort))
                    return false;
                ask(n, sm.list.tile(sm.k0 + i), value);
                ++n;
                return true;
            };
            bool go = true;
            for (int i = 0; i < nt && go; ++i) {
                if (i > 0 && i + 1 < nt) go = fetch(i + 1, 0);
                if (go) go = fetch(i, 1);
            }
            // no copy may be in flight when the CTA ends early
            if (!go && nt > 0) mbar_wait(&sm.q_landed, 0, nullptr);
            if (!go)
                for (int landed = max(0, n - CA_STAGES); landed < n; ++landed)
                    mbar_wait(&sm.full[landed % CA_STAGES], (landed / CA_STAGES) & 1, nullptr);
        }
        __syncwarp();
    } else if (warp == CA_WARP_M) {
        if (lane == 0 && nt > 0) {
            bool go = ut_wait(&sm.q_full, 0, abort);
            for (int i = 0; i < nt && go; ++i) {  // S_i = Q K_i, over the weights of tile i - 2
                const int n = i == 0 ? 0 : 2 * i - 1, s = n % CA_STAGES;
                go = ut_wait(&sm.full[s], (n / CA_STAGES) & 1, abort) &&
                     (i < 2 || ut_wait(&sm.pv_done[i & 1], ((i - 2) >> 1) & 1, abort));
                if (!go) break;
                ut_fence_after();
                ut_mma_qk<128>(tmem + (i & 1) * 128, tmem + CA_TM_Q, smem_u32(sm.stage[s]));
                ut_commit(&sm.empty[s]);
                ut_commit(&sm.s_full[i & 1]);
            }
            ut_commit(&sm.s_end);
            mbar_wait(&sm.s_end, 0, nullptr);
        }
        __syncwarp();
    } else if (warp == CA_WARP_O) {
        if (lane == 0 && nt > 0) {
            bool go = true;
            for (int i = 0; i < nt && go; ++i) {  // O = P_i V_i
                const int n = i + 1 < nt ? 2 * i + 2 : 2 * nt - 1, s = n % CA_STAGES;
                // the weights first: with them the stage's copy before, K_i, is
                // known to be over, so that `full` cannot be taken a phase early
                go = ut_wait(&sm.p_full[i & 1], (i >> 1) & 1, abort) &&
                     (i == 0 || ut_wait(&sm.o_free, (i - 1) & 1, abort)) &&
                     ut_wait(&sm.full[s], (n / CA_STAGES) & 1, abort);
                if (!go) break;
                ut_fence_after();
                ut_mma_pv(tmem + CA_TM_O, tmem + (i & 1) * 128, smem_u32(sm.stage[s]));
                ut_commit(&sm.empty[s]);
                ut_commit(&sm.pv_done[i & 1]);
            }
            ut_commit(&sm.o_full);
            mbar_wait(&sm.o_full, 0, nullptr);  // tensor memory is not given back under a product
        }
        __syncwarp();
    } else if (warp == CA_WARP_E) {
        float E = UT_POISON_E;
        for (int i = 0; i < nt; ++i) {
            const int b = i & 1;
            const float* at = c.meta + place(sm.list.tile(sm.k0 + i)) * 256;
            const float4 k = reinterpret_cast<const float4*>(at)[lane], v = reinterpret_cast<const float4*>(at)[32 + lane];
            // exponents, NaN aside
            const float top = warp_max(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
            const float low = -warp_max(-fminf(fminf(v.x, v.y), fminf(v.z, v.w)));
            // the softmax of tile i - 2 is done with the buffers
            if (i >= 2 && !ut_wait(&sm.pv_done[b], ((i - 2) >> 1) & 1, abort)) break;
            if (sm.k0 + i < sm.list.full) {
                if (i == 0) E = top + CA_ABOVE;
                if (top > E || low < E - CA_SPREAD || low == UT_POISON_E) E = INFINITY;
            }
            reinterpret_cast<float4*>(sm.kc[b])[lane] = k;
            reinterpret_cast<float4*>(sm.ve[b])[lane] = v;
            reinterpret_cast<float4*>(sm.vg[b])[lane] = make_float4(exp2_fast(v.x - E + CA_UP), exp2_fast(v.y - E + CA_UP),
                                                                    exp2_fast(v.z - E + CA_UP), exp2_fast(v.w - E + CA_UP));
            if (lane == 0) {
                sm.E[b] = E;
                sm.top[b] = top;
                sm.low[b] = low;
            }
            __syncwarp();
            if (lane == 0) ut_arrive(&sm.meta_full[b]);
        }
        __syncwarp();
    } else if (warp < CA_SOFTMAX_WARPS) {
        const int part = warp >> 2, row = tid & 127;
        const uint32_t lane_tm = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        // m is a whole number, so that moving it and E multiplies by powers of two
        float m = CO_LOW, l = 0.f, E = UT_POISON_E;
        bool own = false;  // E follows this query's contributions
        // A part of the output row, over the tiles before the newest, in
        // units 2^(E - 13 - CA_UP) of that tile's E and m; f_o takes it there.
        uint64_t acc[CA_W / 2];
#pragma unroll
        for (int q = 0; q < CA_W / 2; ++q) acc[q] = 0;
        float f_o = 1.f;
        auto gather = [&]() {  // acc = acc f_o + the newest tile's product
#pragma unroll
            for (int ch = 0; ch < CA_W / 32; ++ch) {
                uint32_t o[32];
                ut_ld32(lane_tm + CA_TM_O + part * CA_W + ch * 32, o);
                ut_wait_ld();
#pragma unroll
                for (int q = 0; q < 16; ++q)
                    acc[ch * 16 + q] = fma2p(acc[ch * 16 + q], pack2(f_o, f_o),
                                             pack2(__uint_as_float(o[2 * q]), __uint_as_float(o[2 * q + 1])));
            }
        };
        if (nt > 0 && part < 2) {  // the queries into tensor memory: this row of hi, or of lo
            ut_wait(&sm.q_landed, 0, abort);
            ut_row_to_tmem(sm.stage[CA_STAGES - 1] + part * UT_BYTES, row, lane_tm + CA_TM_Q + part * 64);
            ut_fence_before();
        }
        __syncwarp();
        if (lane == 0) ut_arrive(&sm.q_full);
        // A wait that ran out ends every later one at once; the loop still runs
        // through, because its barriers need all softmax warps.
        for (int i = 0; i < nt; ++i) {
            const int b = i & 1, base_slot = sm.list.tile(sm.k0 + i) * 128 + part * CA_W;
            const bool whole = sm.k0 + i < sm.list.full;
            const uint32_t st = lane_tm + b * 128 + part * CA_W;
            const float4* kc = reinterpret_cast<const float4*>(sm.kc[b] + part * CA_W);
            const float* ve = sm.ve[b] + part * CA_W;
            // a row sees slots <= hi that are > lo, or < sinks
            const int hi = sm.own[row], lo = a.window > 0 ? max(-1, hi - a.window) : -1;
            ut_wait(&sm.meta_full[b], (i >> 1) & 1, abort);
            ut_wait(&sm.s_full[b], (i >> 1) & 1, abort);
            ut_fence_after();
            // scores and the largest
            float2 s[CA_W / 2];
            float mx = CO_LOW;
            uint32_t seen = FULL;  // bit per key of the part
            if (!whole) {
                const auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? FULL : (1u << n) - 1u; };
                const int at = base_slot - 1;  // keys base_slot .. hi, less those <= lo that are no sinks
                seen = below(hi - at) & (~below(lo - at) | below(a.sinks - base_slot));
            }
            {
                uint32_t w[32];
                ut_ld32(st, w);
                ut_wait_ld();
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float4 f = kc[q];
                    s[2 * q] = mul2(make_float2(__uint_as_float(w[4 * q]), __uint_as_float(w[4 * q + 1])),
                                    make_float2(f.x, f.y));
                    s[2 * q + 1] = mul2(make_float2(__uint_as_float(w[4 * q + 2]), __uint_as_float(w[4 * q + 3])),
                                        make_float2(f.z, f.w));
                }
            }
            if (__all_sync(FULL, seen == FULL)) {
#pragma unroll
                for (int q = 0; q < 16; ++q) mx = fmaxf(fmaxf(mx, s[q].x), s[q].y);
            } else {
#pragma unroll
                for (int q = 0; q < 16; ++q) {  // what is not seen weighs nothing from here on
                    if (!(seen >> (2 * q) & 1u)) s[q].x = -INFINITY;
                    if (!(seen >> (2 * q + 1) & 1u)) s[q].y = -INFINITY;
                    mx = fmaxf(fmaxf(mx, s[q].x), s[q].y);
                }
            }
            float E_new = E;
            float2 sum;
            // Scores -> weights, scaled by their values' exponents, as hi | lo
            // over the scores.  `vg`: the factors 2^(exponent - E + CA_UP), if one
            // set holds for the warp; else (EACH) every thread forms its own.
            // MASKED: some keys are not seen, whatever their factors are.
            auto weigh = [&](const float2* vg, auto masked, auto each) {
                sum = make_float2(0.f, 0.f);
                const float2 mm = make_float2(-m, -m);
#pragma unroll
                for (int ch = 0; ch < CA_W / 16; ++ch) {
                    uint32_t ph[8], pl[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        float2 p = add2(s[ch * 8 + q], mm);
                        p = make_float2(exp2_fast(p.x), exp2_fast(p.y));
                        sum = add2(sum, p);
                        float2 f = vg[ch * 8 + q];
                        if (decltype(each)::value)
                            f = make_float2(exp2_fast(f.x - E + CA_UP), exp2_fast(f.y - E + CA_UP));
                        p = mul2(p, f);
                        if (decltype(masked)::value) {
                            if (!(seen >> (ch * 16 + 2 * q) & 1u)) p.x = 0.f;
                            if (!(seen >> (ch * 16 + 2 * q + 1) & 1u)) p.y = 0.f;
                        }
                        split2(p, ph[q], pl[q]);
                    }
                    ut_st8(st + ch * 16, ph);
                    ut_st8(st + ch * 16 + 8, pl);
                }
            };
            // The same where some of the warp's rows have an E that follows their
            // contributions: factors are part of those rows' weights.  16 scores at a
            // time, read again, so that the 32 held above are not held here as well.
            auto weigh_mixed = [&]() {
                sum = make_float2(0.f, 0.f);
#pragma unroll 1
                for (int k = 0; k < CA_W; k += 16) {
                    uint32_t w[16], ph[8], pl[8];
                    ut_ld16(st + k, w);
                    ut_wait_ld();
                    const float2* kf = reinterpret_cast<const float2*>(sm.kc[b] + part * CA_W + k);
                    const float2* vf = reinterpret_cast<const float2*>(ve + k);
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const bool sx = seen >> (k + 2 * q) & 1u, sy = seen >> (k + 2 * q + 1) & 1u;
                        float2 x = mul2(make_float2(__uint_as_float(w[2 * q]), __uint_as_float(w[2 * q + 1])), kf[q]);
                        x = make_float2(sx ? x.x - m : -INFINITY, sy ? x.y - m : -INFINITY);
                        const float2 p = make_float2(exp2_fast(x.x), exp2_fast(x.y));
                        sum = add2(sum, p);
                        float2 f = make_float2(vf[q].x - E + CA_UP, vf[q].y - E + CA_UP);
                        f = make_float2(exp2_fast(own ? x.x + f.x : f.x), exp2_fast(own ? x.y + f.y : f.y));
                        f = make_float2(own ? f.x : p.x * f.x, own ? f.y : p.y * f.y);
                        split2(make_float2(sx ? f.x : 0.f, sy ? f.y : 0.f), ph[q], pl[q]);
                    }
                    ut_st8(st + k, ph);
                    ut_st8(st + k + 8, pl);
                }
            };
            // The running maximum follows only when it is passed by 2^CA_SLACK.  In
            // a whole tile the exponents are every row's, and where no thread passed
            // its maximum the row's parts need not tell one another theirs.
            // (Barriers are taken or not by what a barrier said, so that the warps agree
            // also when a wait ran out and they read what is still being written.)
            float d_m = 0.f;
            bool mixed = false;
            if (whole) E_new = sm.E[b];
            if (!whole || i == 0 || softmax_any((mx > m + CA_SLACK && hi >= 0) || E_new == INFINITY)) {
                // A row without E takes it from one value that it sees, the same
                // for as many rows as can be.  The exponents that a row sees are looked
                // through only where those of the tile do not all fit.
                const float top = sm.top[b], low = sm.low[b];
                const bool ask = !whole && hi >= 0 && !own;
                if (ask && E == UT_POISON_E) {
                    const int first = base_slot - part * CA_W;
                    const int one = first < a.sinks ? first : min(max(sm.own[0], first), first + 127);
                    const float e = sm.ve[b][one - first];
                    if (one <= hi && (one > lo || one < a.sinks) && e > UT_POISON_E) E_new = e + CA_ABOVE;
                }
                const bool look = __any_sync(FULL, ask && (E_new == UT_POISON_E || top > E_new || low < E_new - CA_SPREAD));
                float ex = UT_POISON_E, bot = INFINITY;
                if (look) {
#pragma unroll 1
                    for (int q = 0; q < CA_W; ++q) {
                        if (!(seen >> q & 1u)) continue;
                        ex = fmaxf(ex, ve[q]);
                        bot = fminf(bot, ve[q]);
                    }
                    sm.ex[b][part][row] = ex;
                    sm.lo[b][part][row] = bot;
                }
                sm.mx[b][part][row] = mx;
                // some row's E follows its contributions, or may have to
                mixed = softmax_any(whole ? E_new == INFINITY
                                          : hi >= 0 && (own || (E_new == UT_POISON_E ? bot < INFINITY : ex > E_new || bot < E_new - CA_SPREAD)));
#pragma unroll
                for (int q = 0; q < CA_PARTS; ++q) mx = fmaxf(mx, sm.mx[b][q][row]);
                const float m_new = mx > m + CA_SLACK && hi >= 0 ? ceilf(mx) : m;
                d_m = m - m_new;
                m = m_new;
                l *= exp2_fast(d_m);
                if (look) {
#pragma unroll
                    for (int q = 0; q < CA_PARTS; ++q) {
                        ex = fmaxf(ex, sm.ex[b][q][row]);
                        bot = fminf(bot, sm.lo[b][q][row]);
                    }
                    if (ask && E_new == UT_POISON_E && ex > UT_POISON_E) E_new = ex + CA_ABOVE;
                    own = own || (ask && (ex > E_new || bot < E_new - CA_SPREAD || bot == UT_POISON_E));
                }
            }
            if (whole) own = E_new == INFINITY;
            if (mixed) {
                float cx = CO_LOW;
#pragma unroll
                for (int q = 0; q < 16; ++q) cx = fmaxf(fmaxf(cx, s[q].x - m + ve[2 * q]), s[q].y - m + ve[2 * q + 1]);
                sm.cx[part][row] = cx;
                softmax_sync();
#pragma unroll
                for (int q = 0; q < CA_PARTS; ++q) cx = fmaxf(cx, sm.cx[q][row]);
                if (own) E_new = cx > E + d_m + CA_SLACK ? ceilf(cx) : E + d_m;  // else where it was
            }
            const float f_new = i == 0 ? 0.f : exp2_fast(d_m + (E - E_new));
            E = E_new;
            if (mixed) {
                weigh_mixed();
            } else if (whole) {
                weigh(reinterpret_cast<const float2*>(sm.vg[b] + part * CA_W), std::false_type{}, std::false_type{});
            } else if (const float E_0 = __shfl_sync(FULL, E, 0); __all_sync(FULL, hi < 0 || E == E_0)) {
                sm.own_vg[warp][lane] = exp2_fast(ve[lane] - E_0 + CA_UP);
                __syncwarp();
                weigh(reinterpret_cast<const float2*>(sm.own_vg[warp]), std::true_type{}, std::false_type{});
            } else {
                weigh(reinterpret_cast<const float2*>(ve), std::true_type{}, std::true_type{});
            }
            l += sum.x + sum.y;
            ut_wait_st();
            ut_fence_before();
            __syncwarp();
            if (lane == 0) ut_arrive(&sm.p_full[b]);
            if (i > 0) {  // the last tile's product, before this one's takes its place
                ut_wait(&sm.pv_done[b ^ 1], ((i - 1) >> 1) & 1, abort);
                ut_fence_after();
                gather();
                ut_fence_before();
                __syncwarp();
                if (lane == 0) ut_arrive(&sm.o_free);
            }
            f_o = f_new;
        }
        // ---- this split's output over its own sum, staged in shared memory
        if (nt > 0) {
            ut_wait(&sm.o_full, 0, abort);
            ut_fence_after();
            gather();
        }
        sm.l[part][row] = l;
        softmax_sync();
        l = 0.f;
#pragma unroll
        for (int q = 0; q < CA_PARTS; ++q) l += sm.l[q][row];
        if (*abort) l = __int_as_float(0x7fffffff);  // a wait that ran out shows as NaN
        float* stage = reinterpret_cast<float*>(sm.stage) + row * CA_OUT_LD + part * CA_W;
        // rows that saw nothing, and dead ones, give zeros.  2^E in two steps: E
        // itself may lie below what a normal number holds
        const bool none = l == 0.f || row >= sm.live;
        const float half = rintf(0.5f * E), f = exp2_fast(half - 13.f - CA_UP) / l, g = exp2_fast(E - half);
        if (splits == 1 && c.lse && part == 0 && row < sm.live) c.lse[sm.tile_at * 128 + row] = m + log2f(l);
#pragma unroll
        for (int q = 0; q < CA_W / 4; ++q) {
            float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
            const float2 u = unpack2(acc[2 * q]), v = unpack2(acc[2 * q + 1]);
            if (!none) w = make_float4(u.x * f * g, u.y * f * g, v.x * f * g, v.y * f * g);
            *reinterpret_cast<float4*>(stage + 4 * q) = w;
        }
        if (part == 0) sm.m[row] = m;
        softmax_sync();  // all parts have read the sums
        if (part == 0) sm.l[0][row] = l;
        ut_fence_before();
    }
    __syncthreads();
    if (warp == CA_WARP_M) {
        ut_fence_after();
        ut_free<512>(tmem);
    }
    auto place_out = [&](int row) {  // a row's output, in float4
        const int q = over_rep(c, row);
        return reinterpret_cast<float4*>(a.out) + ((long long)(sm.token0 + q) * a.H + g * c.n_rep + row - q * c.n_rep) * 32;
    };
    if (splits == 1) {  // a CTA alone: its rows leave as they are, in whole lines
        for (int row = warp; row < sm.live; row += CA_THREADS / 32)
            place_out(row)[lane] = reinterpret_cast<const float4*>(sm.stage)[row * (CA_OUT_LD / 4) + lane];
        return;
    }
    // ---- join the splits: CTA z of the cluster takes a part of the rows.  The
    // weights of all rows first, then all outputs: two trips to the peers' memory
    // in all, where a warp that took row after row made two for each.
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int part = blockIdx.x % splits;
    const int ra = part * sm.live / splits, rb = (part + 1) * sm.live / splits;
    float (*weight)[128] = sm.mx[0];  // [split][row]; the maxima are done with
    static_assert(2 * CA_PARTS >= CA_MAX_SPLITS, "weights fit the maxima's place");
    for (int i = tid; i < (rb - ra) * splits; i += CA_THREADS) {
        const int row = ra + i / splits, p = i % splits;
        float M = CO_LOW, L = 0.f, mine = 0.f;
#pragma unroll 4
        for (int q = 0; q < splits; ++q) {
            const float m = ld_peer(&sm.m[row], q), l = ld_peer(&sm.l[0][row], q);
            const float up = fmaxf(M, m), f = exp2_fast(M - up), w = l * exp2_fast(m - up);
            mine = q == p ? w : mine * f;
            L = fmaf(L, f, w);
            M = up;
        }
        weight[p][row] = mine / L;
        if (c.lse && p == 0) c.lse[sm.tile_at * 128 + row] = M + log2f(L);
    }
    __syncthreads();
    const uint32_t stage = smem_u32(sm.stage);
    for (int i = tid; i < (rb - ra) * 32; i += CA_THREADS) {
        const int row = ra + (i >> 5), col = i & 31;
        const int at = row * CA_OUT_LD + 4 * col;
        float4 o = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm.stage) + at);
        const float own = weight[part][row];
        o = make_float4(o.x * own, o.y * own, o.z * own, o.w * own);
#pragma unroll 2
        for (int q = 1; q < splits; ++q) {
            const int p = part + q < splits ? part + q : part + q - splits;
            const float4 y = ld_peer4(stage + (uint32_t)at * 4u, p);
            const float w = weight[p][row];
            o = make_float4(fmaf(w, y.x, o.x), fmaf(w, y.y, o.y), fmaf(w, y.z, o.z), fmaf(w, y.w, o.w));
        }
        place_out(row)[col] = o;
    }
    // peers still read this CTA's shared memory
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// -------------------------------------------------------------- chunk_mass
// One CTA per (key tile, kv head, row): its keys, in tensor memory, are the rows
// of the products; the queries that see any of them pass through as columns, half
// a query tile a step.  A thread owns a slot and half of a step's columns, so weights
// are added in a fixed order without atomics:
//   sum over columns of exp2(s - lse)
// Steps of half a tile let two CTAs share an SM: a CTA has few steps between its
// start and its end, which then lie beside the other's work (4 windowed pieces of
// 130 to 256 tokens with their weights: 88 us in whole tiles, one CTA an SM; 84 so).
constexpr int CM_N = 64;                                    // columns of a step
constexpr int CM_PARTS = 2;                                 // threads per slot
constexpr int CM_SUM_WARPS = 4 * CM_PARTS;
constexpr int CM_W = CM_N / CM_PARTS;                       // a thread's columns
constexpr int CM_STAGES = 3;
constexpr int CM_LSE = 4;                                   // steps' lse held
constexpr int CM_THREADS = 32 * (CM_SUM_WARPS + 1);
constexpr int CM_MMA_WARP = CM_SUM_WARPS;
constexpr uint32_t CM_TM_K = 2 * CM_N;                      // TMEM columns: two products, then the keys
constexpr int CM_TM = 256;
static_assert(CM_TM_K + 128 <= CM_TM && 2 * CM_TM <= 512, "tensor memory of two CTAs");

struct CmSmem {
    unsigned char stage[CM_STAGES][UT_BYTES];  // at first the keys in 0 and 1; step i's queries, hi | lo, in (i + 2) % 3
    float lse[CM_LSE][CM_N];
    float kc[128];
    float part[CM_PARTS][128];
    int own[CM_SUM_WARPS][CM_W];  // slots of the queries in a warp's columns; -1: none
    uint64_t k_full, k_copied, q_full[CM_STAGES], q_empty[CM_STAGES], s_full[2], s_empty[2], lse_full[CM_LSE], end;
    uint32_t tmem;
    int abort;
};
constexpr size_t CM_SMEM = sizeof(CmSmem) + 1024;
static_assert(CM_W == 32, "a part is a warp's width");
static_assert(4 * CM_N * 128 == UT_BYTES, "a step's queries fill a stage");
static_assert(2 * (CM_SMEM + 1024) <= 227 * 1024, "shared memory of two CTAs");

__global__ void __launch_bounds__(CM_THREADS, 2) chunk_mass_kernel(const __grid_constant__ ChunkArgs c) {
    extern __shared__ unsigned char cm_raw[];
    CmSmem& sm = *reinterpret_cast<CmSmem*>(cm_raw + ((1024u - (smem_u32(cm_raw) & 1023u)) & 1023u));
    const CacheAttnArgs& a = c.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = blockIdx.y, r = blockIdx.z;
    const ChunkRow x = chunk_row(c, r);
    pdl_wait();
    if (x.idle || x.bad || x.n == 0) return;
    const int last = x.cached + x.n - 1;
    const RowTiles rt(c, x);
    if ((int)blockIdx.x >= rt.n) return;
    const int row_at = row_base(c, r);
    if (row_at < 0) return;
    const int tile = rt.tile(blockIdx.x);
    const int base = tile * 128;
    if (base > last) return;
    // queries (slots) that may see a slot of the tile: from `from` to `to`
    const int from = max(base, x.cached);
    int to = last;
    if (a.window > 0 && base >= a.sinks) to = (int)min((long long)to, (long long)base + 127 + a.window - 1);
    if (from > to) return;
    // steps: halves of query tiles, numbered through the row
    auto step_of = [&](int own, int head) {
        const int t = (own - x.cached) / c.P, column = (own - x.cached - t * c.P) * c.n_rep + head;
        return 2 * t + column / CM_N;
    };
    const int s0 = step_of(from, 0), ns = step_of(to, c.n_rep - 1) - s0 + 1;

    if (tid == 0) {
        mbar_init(&sm.k_full, 1);
        mbar_init(&sm.k_copied, CM_SUM_WARPS);
        mbar_init(&sm.end, 1);
        for (int b = 0; b < CM_STAGES; ++b) {
            mbar_init(&sm.q_full[b], 1);
            mbar_init(&sm.q_empty[b], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sm.s_full[b], 1);
            mbar_init(&sm.s_empty[b], CM_SUM_WARPS);
        }
        for (int b = 0; b < CM_LSE; ++b) mbar_init(&sm.lse_full[b], 1);
        mbar_fence_init();
        sm.abort = 0;
    }
    if (warp == CM_MMA_WARP) ut_alloc<CM_TM>(&sm.tmem);
    ut_fence_before();
    __syncthreads();
    ut_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* abort = &sm.abort;

    if (warp == CM_MMA_WARP) {
        if (lane == 0) {
            auto fetch = [&](int i) {
                const int s = s0 + i, b = (i + 2) % CM_STAGES;
                const long long at = chunk_tile(c, x, r, s >> 1) * a.kv.KVH + g;
                const unsigned char* q = c.qtiles + at * (2 * UT_BYTES) + (s & 1) * (CM_N * 128);
                mbar_expect_tx(&sm.q_full[b], UT_BYTES);
#pragma unroll
                for (int k = 0; k < 4; ++k)  // hi and lo, two halves of 64 columns each
                    bulk_g2s(sm.stage[b] + k * (CM_N * 128), q + k * UT_HALF, CM_N * 128, &sm.q_full[b]);
                mbar_expect_tx(&sm.lse_full[i % CM_LSE], CM_N * 4);
                bulk_g2s(sm.lse[i % CM_LSE], c.lse + at * 128 + (s & 1) * CM_N, CM_N * 4, &sm.lse_full[i % CM_LSE]);
            };
            const long long kat = ((long long)(row_at + blockIdx.x) * a.kv.KVH + g) * 2;
            mbar_expect_tx(&sm.k_full, 2 * UT_BYTES + 512);
            bulk_g2s(sm.stage[0], c.kvtiles + kat * (2 * UT_BYTES), 2 * UT_BYTES, &sm.k_full);
            bulk_g2s(sm.kc, c.meta + kat * 128, 512, &sm.k_full);
            fetch(0);
            int fetched = 1;
            bool go = ut_wait(&sm.k_copied, 0, abort);
            for (; go && fetched < CM_STAGES && fetched < ns; ++fetched) fetch(fetched);
            for (int i = 0; i < ns && go; ++i) {
                const int b = (i + 2) % CM_STAGES;
                go = ut_wait(&sm.q_full[b], (i / CM_STAGES) & 1, abort) &&
                     (i < 2 || ut_wait(&sm.s_empty[i & 1], ((i - 2) >> 1) & 1, abort));
                if (!go) break;
                ut_fence_after();
                ut_mma_qk<CM_N>(tmem + (i & 1) * CM_N, tmem + CM_TM_K, smem_u32(sm.stage[b]));
                ut_commit(&sm.q_empty[b]);
                ut_commit(&sm.s_full[i & 1]);
                // into the stage of step i - 1, when its products are done; the lse
                // that step i - 2 left is read, since its sums were waited for above
                if (i >= 1 && i + 2 < ns) {
                    go = ut_wait(&sm.q_empty[(i + 1) % CM_STAGES], ((i - 1) / CM_STAGES) & 1, abort);
                    if (go) {
                        fetch(i + 2);
                        ++fetched;
                    }
                }
            }
            // leave nothing in flight: the copies asked for, the products issued
            if (!go) {
                mbar_wait(&sm.k_full, 0, nullptr);
                for (int f = max(0, fetched - CM_STAGES); f < fetched; ++f) {
                    mbar_wait(&sm.q_full[(f + 2) % CM_STAGES], (f / CM_STAGES) & 1, nullptr);
                    mbar_wait(&sm.lse_full[f % CM_LSE], (f / CM_LSE) & 1, nullptr);
                }
            }
            ut_commit(&sm.end);
            mbar_wait(&sm.end, 0, nullptr);
        }
        __syncwarp();
    } else {
        const int key = 32 * (warp & 3) + lane, part = warp >> 2, slot = base + key;
        const uint32_t lane_tm = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        ut_wait(&sm.k_full, 0, abort);
        ut_row_to_tmem(sm.stage[part], key, lane_tm + CM_TM_K + part * 64);  // hi, or lo
        ut_fence_before();
        __syncwarp();
        if (lane == 0) ut_arrive(&sm.k_copied);
        const float kc = sm.kc[key];
        // queries at slots >= this do not see the slot
        const unsigned upto = a.window == 0 || slot < a.sinks ? 0x7fffffffu : (unsigned)slot + (unsigned)a.window;
        float2 sum = make_float2(0.f, 0.f);
        for (int i = 0; i < ns; ++i) {
            const int b = i & 1, t = (s0 + i) >> 1, column = ((s0 + i) & 1) * CM_N;
            const int first = x.cached + t * c.P;            // slot of the tile's first query
            const int nq = min(c.P, last + 1 - first);
            // seen whole: every column is a query, behind every slot, inside the window
            const bool whole = nq * c.n_rep >= column + CM_N && first >= base + 127 &&
                               (a.window == 0 || first + nq - 1 - base < a.window || base + 128 <= a.sinks);
            if (!whole) {  // once a column, not once a weight
                const int qi = over_rep(c, column + part * CM_W + lane);
                sm.own[warp][lane] = qi < nq ? first + qi : -1;
                __syncwarp();
            }
            if (!ut_wait(&sm.s_full[b], (i >> 1) & 1, abort)) break;
            if (!ut_wait(&sm.lse_full[i % CM_LSE], (i / CM_LSE) & 1, abort)) break;
            ut_fence_after();
            {
                uint32_t s[32];
                ut_ld32(lane_tm + b * CM_N + part * CM_W, s);
                ut_wait_ld();
                const float4* lse = reinterpret_cast<const float4*>(sm.lse[i % CM_LSE] + part * CM_W);
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
                        const int4 own = reinterpret_cast<const int4*>(sm.own[warp])[q];
                        const int w[4] = {own.x, own.y, own.z, own.w};
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            if (w[y] < slot || (unsigned)w[y] >= upto) p[y] = 0.f;
                    }
                    sum = add2(sum, add2(make_float2(p[0], p[1]), make_float2(p[2], p[3])));
                }
            }
            ut_fence_before();
            __syncwarp();  // also: the slots in sm.own are read
            if (lane == 0) ut_arrive(&sm.s_empty[b]);
        }
        sm.part[part][key] = sum.x + sum.y;
    }
    __syncthreads();
    if (warp == CM_MMA_WARP) {
        ut_fence_after();
        ut_free<CM_TM>(tmem);
    }
    const int slot = base + tid;
    if (tid < 128 && slot <= last) {
        float s = 0.f;
#pragma unroll
        for (int p = 0; p < CM_PARTS; ++p) s += sm.part[p][tid];
        if (*abort) s = __int_as_float(0x7fffffff);
        float* mass = a.mass + (((long long)r * a.kv.KVH + g) * a.kv.max_pages << a.kv.page_log2) + slot;
        *mass = slot >= x.cached ? s : *mass + s;
    }
}

static long long chunk_query_tiles(int tokens, int rows, int n_rep) { return tokens / (128 / n_rep) + rows + 1; }

// Key tiles of one row, at most: by the cache's width and by its window.
static long long chunk_row_tiles(int max_chunk, int max_pages, int page_size, int window, int sinks) {
    const long long n = ((long long)max_pages * page_size + 127) / 128;
    const long long w = ((long long)sinks + 127) / 128 + ((long long)window + max_chunk + 127) / 128 + 1;
    return window > 0 && w < n ? w : n;
}
// Key tiles of all rows together, at most: each row's; all of them by the pool, whose pages belong to one row each.
// Slots out of sight may have no page, so a row's tiles are counted against the
// slots it sees: up to one tile more for its end, for the window's beginning and
// for the sinks' end (a stretch of L slots lies in at most (L + 254) / 128
// tiles, one that begins with a tile in (L + 127) / 128).
static long long chunk_key_tiles(int rows, int max_chunk, int max_pages, int page_size, long long n_pages, int window, int sinks) {
    const long long n = chunk_row_tiles(max_chunk, max_pages, page_size, window, sinks) * rows;
    const long long all = n_pages * page_size / 128 + (window > 0 && sinks > 0 ? 3ll : 2ll) * rows;
    return all < n ? all : n;
}

struct ChunkWork {
    long long q, kv, meta, jobs, lse, total;  // byte offsets
    ChunkWork(long long qtiles, long long ktiles, int KVH, int rows, bool with_mass) {
        q = 0;
        kv = qtiles * KVH * (2 * (long long)UT_BYTES);
        meta = kv + ktiles * KVH * (4 * (long long)UT_BYTES);
        jobs = meta + ktiles * KVH * 1024;
        lse = jobs + (rows * (long long)sizeof(RowJob) + 255) / 256 * 256;
        total = lse + (with_mass ? (qtiles * KVH * 512 + 255) / 256 * 256 : 0);
    }
};

}  // namespace skb

using namespace skb;

extern "C" int64_t skb_chunk_attention_workspace(int tokens, int rows, int max_chunk, int n_heads, int n_kv_heads,
                                                 int max_pages, int page_size, int n_pages, int window, int sinks,
                                                 int with_mass) {
    if (tokens < 0 || rows < 0 || max_chunk < 0 || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads != 0 ||
        n_heads / n_kv_heads > CO_MAX_REP || max_pages < 1 || page_size < 1 || n_pages < 1 || window < 0 || sinks < 0)
        return -1;
    return ChunkWork(chunk_query_tiles(tokens, rows, n_heads / n_kv_heads),
                     chunk_key_tiles(rows, max_chunk, max_pages, page_size, n_pages, window, sinks), n_kv_heads, rows,
                     with_mass)
        .total;
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
    if ((uintptr_t)kv_pool & 31u)  // chunk_prep reads cached rows 32 bytes a lane
        return fail(SKB_ERR_ARG, "%s: kv_pool must be 32-byte aligned", what);
    if ((long long)n_pages * 2 * n_kv_heads * page_size >= 0xfffffffell)
        return fail(SKB_ERR_ARG, "%s: the pool must hold fewer than 2^32 - 2 key and value rows", what);
    if (rows == 0 || tokens == 0) return SKB_OK;
    if (!qkv || !out) return fail(SKB_ERR_ARG, "%s: null pointer", what);
    if (!work || ((uintptr_t)work & 255u) ||
        work_bytes < skb_chunk_attention_workspace(tokens, rows, max_chunk, n_heads, n_kv_heads, max_pages, page_size, n_pages,
                                                   window, sinks, mass != nullptr))
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
    c.rep_inv = ((1u << 24) + c.n_rep - 1) / c.n_rep;
    const long long tiles = chunk_query_tiles(tokens, rows, c.n_rep);
    const long long key_tiles = chunk_key_tiles(rows, max_chunk, max_pages, page_size, n_pages, window, sinks);
    if (key_tiles >= CHUNK_TILES) return fail(SKB_ERR_ARG, "%s: too many slots", what);  // 4 TB of workspace
    c.key_tiles = (int)key_tiles;
    c.roomy = key_tiles == chunk_row_tiles(max_chunk, max_pages, page_size, window, sinks) * rows;
    const ChunkWork at(tiles, c.key_tiles, n_kv_heads, rows, mass != nullptr);
    unsigned char* w = static_cast<unsigned char*>(work);
    c.qtiles = w + at.q;
    c.kvtiles = w + at.kv;
    c.meta = reinterpret_cast<float*>(w + at.meta);
    c.lse = mass ? reinterpret_cast<float*>(w + at.lse) : nullptr;

    // no more tokens than there are, whatever max_chunk says
    const int most = max_chunk < 1 ? 1 : (max_chunk < tokens ? max_chunk : tokens);
    const int tiles_x = (most + c.P - 1) / c.P;
    // key tiles of one row, at most
    long long row_tiles = chunk_row_tiles(most, max_pages, page_size, window, sinks);
    if (row_tiles > c.key_tiles) row_tiles = c.key_tiles;
    // CTAs that have work, at most; while they leave SMs idle, up to 8 share a
    // query tile's key tiles, as long as no SM gets two.  (Sharing where they fill
    // the card already makes clusters wait for SMs and adds the join: 8 prompts 199 us
    // in pairs, 117 alone.  Calls alone, in pairs, in threes: 512 tokens behind 8192
    // slots, 64 CTAs, 193, 112 with the two that this rule gives, 149; 640, 80 CTAs,
    // 174 alone as it gives, 190, 151; 1152, 144 CTAs, 232, 251, 300.  Two rows of
    // five tokens 18.5 alone, 17.3 in threes, one for each of their key tiles.)
    long long ctas = (long long)rows * tiles_x;
    if (ctas > tiles) ctas = tiles;
    ctas *= n_kv_heads;
    long long splits = 148 / ctas;
    if (splits > row_tiles) splits = row_tiles;
    if (splits > CA_MAX_SPLITS) splits = CA_MAX_SPLITS;
    if (splits < 1) splits = 1;
    // A grid over rows of unequal length starts CTAs that have nothing to do; where
    // it is more than one wave, the CTAs go by a list of the rows, the longest
    // first.  (One wave does without: a row's numbers are then read before
    // chunk_prep is over.)
    const long long grid = splits * tiles_x * n_kv_heads * rows;
    c.jobs = grid > 148 && rows <= CP_SORTED ? reinterpret_cast<RowJob*>(w + at.jobs) : nullptr;
    if (c.jobs && ctas * splits > 0x7fffffffll) return fail(SKB_ERR_ARG, "%s: too many tokens and rows", what);
    const int prep_x = row_tiles < CP_TILES ? (int)row_tiles : CP_TILES;
    const int per_block = tokens <= 1024 ? 1 : 4;
    const int token_blocks = (tokens + per_block - 1) / per_block;
    const long long prep_blocks = token_blocks + (c.jobs ? 1 : 0) + (long long)prep_x * 2 * n_kv_heads * rows;
    if (prep_blocks > 0x7fffffffll) return fail(SKB_ERR_ARG, "%s: too many tokens and rows", what);

    static std::atomic<unsigned long long> attn_done, mass_done;
    cudaError_t e = smem_attrs_once(chunk_attn_kernel, CA_SMEM, attn_done);
    if (e == cudaSuccess && mass) e = smem_attrs_once(chunk_mass_kernel, CM_SMEM, mass_done);
    if (e == cudaSuccess)
        e = launch(chunk_prep_kernel, dim3((unsigned)prep_blocks), dim3(256), 0, stream, false, c, token_blocks, per_block,
                   prep_x);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = c.jobs ? dim3((unsigned)(ctas * splits)) : dim3((unsigned)splits * tiles_x, n_kv_heads, rows);
        cfg.blockDim = dim3(CA_THREADS);
        cfg.dynamicSmemBytes = CA_SMEM;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)splits;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, chunk_attn_kernel, c, (int)splits);
    }
    if (e == cudaSuccess && mass)
        e = launch(chunk_mass_kernel, dim3((unsigned)row_tiles, n_kv_heads, rows), dim3(CM_THREADS), CM_SMEM, stream, true, c);
    return e == cudaSuccess ? SKB_OK : fail(SKB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
