// Products of a few tokens' codes with 8-bit weights, bound by the weights'
// bytes: the tokens' rows become codes in every CTA's shared memory (one launch
// for norm, codes and product), each warp streams whole weight rows, four a
// step, and adds up products of four bytes an instruction.
//
// 2 tokens of 1024 FP32 values with a norm to 4096 channels 4.6 us (weights in L2 3.4), to
// 32816 11 (33.6 MB from device memory; 9.7 from codes, in L2 7.7): about 1.5 us to the
// first codes, the stream, and sums across a warp for every row.  Rows announced to L2
// four groups ahead (bulk prefetch) took 2 us more.
#include "int8_ops.cuh"

namespace skb {

constexpr int GV_THREADS = 256, GV_WARPS = 8;
constexpr int GV_CHUNK = 512;   // bytes of a row that a warp reads at once
constexpr int GV_MAX_K = 8192;        // values of a row; of two tokens' twice, of one's three times as many
constexpr int GV_MAX_X = 8 * GV_MAX_K;  // bytes of codes in shared memory
constexpr int GV_FUSED_T = 2, GV_FUSED = 4096;  // tokens, and values in all, up to which each CTA makes the codes itself
constexpr long long GV_READS = 6 << 20;         // bytes of weights, read once for every 8 tokens

// TT: tokens a CTA holds (the last ones may be missing); R: weight rows a warp
// takes at a time (with SwiGLU R / 2 gate rows and their up rows).  8 / R chunks of
// each are on their way: 4 KB a warp.
template <class TX, int TT, int R, bool GLU>
__global__ void __launch_bounds__(GV_THREADS, 2) int8_gemv_kernel(const Int8Args a, bool early) {
    extern __shared__ __align__(16) int8_t gv_x[];  // [TT][kp]
    __shared__ alignas(16) float red[TT * ROW_RED];
    __shared__ float sx[TT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int K = a.in.K, kp = ceil16(K);
    const int t0 = blockIdx.y * TT, nt = min(TT, a.in.T - t0);
    constexpr int D = 8 / R;
    constexpr int PER = GLU ? R / 2 : R;  // output columns a step
    const int groups = (a.N + PER - 1) / PER;
    const int chunks = (kp + GV_CHUNK - 1) / GV_CHUNK;
    const int stride = gridDim.x * GV_WARPS;
    int group = blockIdx.x * GV_WARPS + warp;

    // the next chunk to fetch, of this group or the next
    int f_group = group, f_chunk = 0;
    auto fetch = [&](uint4 (&w)[R]) {
        const int k = f_chunk * GV_CHUNK + lane * 16;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int m = GLU ? r / PER : 0, n = f_group * PER + (GLU ? r % PER : r);
            w[r] = make_uint4(0, 0, 0, 0);
            if (f_group < groups && n < a.N && k < kp)
                w[r] = __ldcg(reinterpret_cast<const uint4*>(a.w[m] + n * a.ldw[m] + k));
        }
        if (++f_chunk == chunks) f_chunk = 0, f_group += stride;
    };
    uint4 w[D][R];
    if (!early) pdl_wait();
#pragma unroll
    for (int d = 0; d < D; ++d) fetch(w[d]);
    if (early) pdl_wait();
    pdl_trigger();

    // the tokens' codes
    if constexpr (sizeof(TX) == 1) {
        for (int i = tid; i < TT * (kp / 16); i += GV_THREADS) {
            const int t = i / (kp / 16), k = i % (kp / 16) * 16;
            uint4 c = make_uint4(0, 0, 0, 0);
            if (t < nt) c = __ldcg(reinterpret_cast<const uint4*>(static_cast<const int8_t*>(a.in.x) + (t0 + t) * a.in.ld + k));
            // whatever lies behind K counts for nothing, here and in the weights
            uint32_t b[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int left = K - k - 4 * j;
                if (left < 4) b[j] = left <= 0 ? 0u : b[j] & (0xffffffffu >> (32 - 8 * left));
            }
            *reinterpret_cast<uint4*>(gv_x + t * kp + k) = make_uint4(b[0], b[1], b[2], b[3]);
        }
        if (tid < TT) sx[tid] = tid < nt ? __ldcg(a.in.scale + t0 + tid) : 0.f;
    } else {
        constexpr int G = GV_THREADS / TT;
        const int t = tid / G;
        // a missing token repeats the last one, so that all threads take the same way
        const TX* x = static_cast<const TX*>(a.in.x) + (long long)(t0 + min(t, nt - 1)) * a.in.ld;
        const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
        const float s = quantize_row<TX, G, 16 / Vec<TX>::N>(x, a.in.nw, a.in.eps, K, aligned, gv_x + t * kp, tid % G,
                                                             red + t * ROW_RED);
        if (tid % G == 0) sx[t] = s;
    }
    __syncthreads();

    auto finish_group = [&](int group, int (&acc)[R][TT]) {
        // lane (t, column) takes its sum
        int v = 0, u = 0;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const int sum = __reduce_add_sync(FULL, acc[r][t]);
                acc[r][t] = 0;
                if (lane == t * PER + (GLU ? r % PER : r)) {
                    if (GLU && r >= PER) u = sum;
                    else v = sum;
                }
            }
        const int t = lane / PER, n = group * PER + lane % PER;
        if (t < nt && lane < TT * PER && n < a.N) {
            float y;
            if constexpr (GLU) {
                y = finish_glu(v, u, sx[t], __ldcg(a.ws[0] + n), __ldcg(a.ws[1] + n));
            } else {
                y = finish(v, sx[t], __ldcg(a.ws[0] + n), a.bias ? __ldcg(a.bias + n) : 0.f);
                if (a.residual) y += load_as(a.residual, a.out_type, (t0 + t) * a.ldr + n);
            }
            store_as(a.out, a.out_type, (t0 + t) * a.ldo + n, y);
        }
    };
    int acc[R][TT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[r][t] = 0;
    int c = 0;
    while (group < groups) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (group < groups) {
                const int k = c * GV_CHUNK + lane * 16;
                if (k < kp) {
#pragma unroll
                    for (int t = 0; t < TT; ++t) {
                        const int4 x = *reinterpret_cast<const int4*>(gv_x + t * kp + k);
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            acc[r][t] = __dp4a((int)w[d][r].x, x.x, acc[r][t]);
                            acc[r][t] = __dp4a((int)w[d][r].y, x.y, acc[r][t]);
                            acc[r][t] = __dp4a((int)w[d][r].z, x.z, acc[r][t]);
                            acc[r][t] = __dp4a((int)w[d][r].w, x.w, acc[r][t]);
                        }
                    }
                }
                fetch(w[d]);
                if (++c == chunks) {
                    c = 0;
                    finish_group(group, acc);
                    group += stride;
                }
            }
        }
    }
}

// Codes made by every CTA save a launch and cost what their values take: with a norm, 1
// token of 1024 FP32 values to 4096 channels 3.9 us, in two launches 4.3, 2 tokens 4.2 and
// 4.4, 1 of 4096 to 1024 5.2 and 5.4; 2 of 4096 to 4096 9.9 and 7.6.  Beside many
// channels it no longer shows (2 tokens to 32816 10.6 and 10.3).
bool int8_gemv_fuses(int T, int K) { return T <= GV_FUSED_T && T * ceil16(K) <= GV_FUSED; }

// Here, or on the tensor cores; from codes, us.  Up to 4 tokens weights come in about as
// fast either way and there is less around them (4 tokens of 1024 to 4096 channels 3.5 and
// 6.5, to 32816 11.6 and 17; of 8192 to 4096 13.3 and 11.8).  With more, four-byte products
// take longer than the bytes, once for every 8 tokens: 16 of 2048 to 1024 4.9 here and
// 6.6 there, 5 of 1024 to 4096 4.6 and 6.5, 16 of these 7.5 and 6.5, 8 of 4096 to 4096
// 9.6 and 8.7.  A warp takes a whole row by itself, so that long ones are slow:
// 4 tokens of 16384 to 4096 22.5 and 16.7, one of 131071 to 1024 91 and 40.  To few channels
// one or two tokens are faster a little further (2 of 16384 to 64 9.0 and 9.4, of 24000
// 12.4 and 11.4; 1 of 20000 9.4 and 10.6, of 33000 14.2 and 13.8).
bool int8_gemv_serves(const Int8Args& a, bool glu) {
    const int T = a.in.T;
    const long long bytes = (long long)a.N * max(a.in.K, GV_CHUNK) * (glu ? 2 : 1);
    if (a.in.K > GV_MAX_K) return T <= 2 && a.in.K <= (4 - T) * GV_MAX_K && bytes <= GV_READS;
    return T <= 4 || (T <= 16 && (T + 7) / 8 * bytes <= GV_READS);
}

template <auto Kernel>
static cudaError_t gemv_go(const Int8Args& a, int R, int tt, bool glu, bool early, cudaStream_t s) {
    const cudaError_t e = prepare_kernel<Kernel>(GV_MAX_X);
    if (e != cudaSuccess) return e;
    const int per = glu ? R / 2 : R, blocks = ((a.N + per - 1) / per + GV_WARPS - 1) / GV_WARPS;
    const dim3 grid(blocks < 296 ? blocks : 296, (a.in.T + tt - 1) / tt);
    return launch(Kernel, grid, dim3(GV_THREADS), (size_t)tt * ceil16(a.in.K), s, true, a, early);
}

// As many rows a warp at a time as gives every warp of 296 CTAs, two an SM, rows to take.
// Two tokens of 1024 values by one, two and four, us: to 2048 channels 2.7, 2.8, 3.0, to
// 4096 4.3, 3.6, 3.9, to 8192 6.3, 5.4, 5.0, to 32816 14.9, 10.8, 9.9; SwiGLU by a pair and
// two pairs: to 2048 3.6 and 3.8, to 4096 5.2 and 4.8.
template <class TX, int TT, bool GLU>
static cudaError_t gemv_rows(const Int8Args& a, bool early, cudaStream_t s) {
    const long long rows = (long long)a.N * (GLU ? 2 : 1);
    if (rows > 2 * GV_WARPS * 296) return gemv_go<int8_gemv_kernel<TX, TT, 4, GLU>>(a, 4, TT, GLU, early, s);
    if constexpr (!GLU) {
        if (rows <= GV_WARPS * 296) return gemv_go<int8_gemv_kernel<TX, TT, 1, GLU>>(a, 1, TT, GLU, early, s);
    }
    return gemv_go<int8_gemv_kernel<TX, TT, 2, GLU>>(a, 2, TT, GLU, early, s);
}

template <class TX, bool GLU>
static cudaError_t gemv_typed(const Int8Args& a, bool early, cudaStream_t s) {
    const int T = a.in.T;
    const int tt = T == 1 ? 1 : T == 2 ? 2 : T <= 4 ? 4 : 8;
    if (tt == 1) return gemv_rows<TX, 1, GLU>(a, early, s);
    if (tt == 2) return gemv_rows<TX, 2, GLU>(a, early, s);
    if constexpr (sizeof(TX) == 1) {
        if (tt == 4) return gemv_rows<TX, 4, GLU>(a, early, s);
        return gemv_rows<TX, 8, GLU>(a, early, s);
    }
    return cudaErrorInvalidValue;
}

// early: the kernel before this one in the stream is quantize_launch's of the same
// call, which has waited for all before it when it lets this one begin; so the
// weights are there, and only the codes are waited for.
cudaError_t int8_gemv_launch(const Int8Args& a, bool glu, bool early, cudaStream_t s) {
    auto go = [&](auto x) { return glu ? gemv_typed<decltype(x), true>(a, early, s) : gemv_typed<decltype(x), false>(a, early, s); };
    return a.in.type == SKB_I8 ? go(int8_t()) : with_type(a.in.type, go);
}

}  // namespace skb
