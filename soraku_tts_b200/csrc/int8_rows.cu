// Rows of values to rows of 8-bit codes, each with its scale (int8_ops.cuh has
// the definition).  Activations before a product, weights once.
//
// One pass over memory: a row stays in registers between the search for its largest
// and its codes.  From device memory: 6541 rows of 1024 FP32 values with a norm 7.8 us,
// 4.3 TB/s; 20000 without 18.9, 5.4.  16-bit rows are bound by instructions, 12 a value
// (4096 of 4096 BF16 12.1 us, 4.2 TB/s, FP16 10.1; four vectors a thread need more
// registers than two CTAs' worth); a few rows by latency, 1.0 to 2 us.  Rows brought to
// shared memory by bulk copies, a warp to each, were no faster: 5.4 us for the 6541 without
// a norm where this took 6.2, 8.2 with one (7.3), 18.9 for the BF16 rows (12.0).
// The order of a row's squares (Squares) costs rows of 64 and 128 threads up to 0.3 us
// (6541 of 1024 FP32 values 7.0 -> 7.3 in L2), others nothing.
#include "int8_ops.cuh"

namespace skb {

// G threads a row, which hold it in registers, CH vectors each, between the
// search for the largest and the codes.  A CTA takes rows one after the other:
// the norm's weights stay in registers, and the next row is on its way while this
// one is finished.
template <class TX, int G, int CH, bool NORM>
__global__ void __launch_bounds__(256, CH * Vec<TX>::N <= 8 ? 4 : CH * Vec<TX>::N > 16 ? 2 : NORM ? 3 : 4)
    quantize_kernel(const RowsIn in, int8_t* __restrict__ q, long long ldq, float* __restrict__ scale) {
    using SQ = Squares<G, CH>;
    constexpr int V = Vec<TX>::N, ROWS = 256 / G, WARPS = G / 32;
    __shared__ alignas(16) float red[2][2][ROWS][SQ::CHAINS];  // warps' largest; chains
    const int slot = threadIdx.x / G, t = threadIdx.x % G;
    const int K = in.K, kp = ceil16(K);
    pdl_wait();
    pdl_trigger();
    float w[NORM ? CH : 1][V];
    if constexpr (NORM) {
        const bool aligned = (reinterpret_cast<uintptr_t>(in.nw) & 15) == 0;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                const int k = (c * G + t) * V + 4 * h;
                Vec<float> raw;
                raw.template load<true>(in.nw + k, K - k, aligned);
                float f[4];
                raw.get(f);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[c][4 * h + i] = f[i];
            }
    }
    Vec<TX> next[CH];
    const bool all_aligned = ((reinterpret_cast<uintptr_t>(in.x) | (uintptr_t)(in.ld * (long long)sizeof(TX))) & 15) == 0;
    auto load = [&](long long row) {
        const TX* x = static_cast<const TX*>(in.x) + row * in.ld;
        const bool aligned = all_aligned || (reinterpret_cast<uintptr_t>(x) & 15) == 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = (c * G + t) * V;
            next[c].load(x + k, row < in.T ? K - k : 0, aligned);
        }
    };
    const long long step = (long long)gridDim.x * ROWS;
    long long row = (long long)blockIdx.x * ROWS + slot;
    load(row);
    for (int turn = 0; row - slot < in.T; row += step, turn ^= 1) {
        float v[CH][V], top = 0.f, ss = 0.f;
        SQ squares;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            next[c].get(v[c]);
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                if constexpr (NORM) {
                    const float2 x = make_float2(v[c][i], v[c][i + 1]), y = mul2(x, make_float2(w[c][i], w[c][i + 1]));
                    squares.add(c, x);
                    v[c][i] = y.x, v[c][i + 1] = y.y;
                }
                top = max3_abs(top, v[c][i], v[c][i + 1]);
            }
        }
        float2 ends;
        if constexpr (NORM) ends = squares.ends();
        if (row - slot + step < in.T) load(row + step);
        top = warp_top(top);
        if (NORM) ss = SQ::over_lanes(ends, t & 31);
        if constexpr (G > 32) {
            // two places in turn, so that one barrier a row is enough
            if constexpr (NORM && SQ::N == 2) {
                if ((t & 15) == 0) red[1][turn][slot][SQ::place(t)] = ss;
                if ((t & 31) == 0) red[0][turn][slot][t >> 5] = top;
            } else {
                if ((t & 31) == 0) red[0][turn][slot][t >> 5] = top, red[1][turn][slot][t >> 5] = ss;
            }
            __syncthreads();
            top = warp_top(red[0][turn][slot][t % WARPS]);
        } else if constexpr (NORM && SQ::N == 2) {
            ss += __shfl_sync(FULL, ss, 16);  // of use to lane 0: its chain, then the other
        }
        if (row >= in.T) continue;
        const float r = codes_per(top);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = (c * G + t) * V;
            if (k < kp) {
                uint32_t word[V / 4];
                encode<V>(v[c], top, r, word);
                put_codes<V>(q + row * ldq + k, word);
            }
        }
        if (t == 0) {
            if constexpr (NORM && G > 32) ss = SQ::total(red[1][turn][slot]);
            const float s = step_of(top);
            scale[row] = NORM ? s * rsqrtf(ss / (float)K + in.eps) : s;
        }
    }
}

// Rows of more than 8192 values: a CTA each, all but the last piece read again.
template <class TX>
__global__ void __launch_bounds__(256) quantize_long_kernel(const RowsIn in, int8_t* __restrict__ q, long long ldq,
                                                            float* __restrict__ scale) {
    __shared__ alignas(16) float red[ROW_RED];
    pdl_wait();
    pdl_trigger();
    const long long row = blockIdx.x;
    const TX* x = static_cast<const TX*>(in.x) + row * in.ld;
    const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    const float s = quantize_row<TX, 256, 32 / Vec<TX>::N>(x, in.nw, in.eps, in.K, aligned, q + row * ldq, threadIdx.x, red);
    if (threadIdx.x == 0) scale[row] = s;
}

// CTAs that are resident at once: rows are dealt out to just as many.
template <auto Kernel>
static int resident() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, 256, 0) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = 1;
        }
        n *= 148;
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

template <class TX, int G, int CH, bool NORM>
static cudaError_t rows_go(const RowsIn& in, int8_t* q, long long ldq, float* scale, cudaStream_t s) {
    constexpr int ROWS = 256 / G;
    const int need = (in.T + ROWS - 1) / ROWS, most = resident<quantize_kernel<TX, G, CH, NORM>>();
    return launch(quantize_kernel<TX, G, CH, NORM>, dim3(need < most ? need : most), dim3(256), 0, s, true, in, q, ldq, scale);
}
template <class TX, int G, int CH>
static cudaError_t rows_launch(const RowsIn& in, int8_t* q, long long ldq, float* scale, cudaStream_t s) {
    return in.nw ? rows_go<TX, G, CH, true>(in, q, ldq, scale, s) : rows_go<TX, G, CH, false>(in, q, ldq, scale, s);
}

template <class TX>
static cudaError_t quantize_typed(const RowsIn& in, int8_t* q, long long ldq, float* scale, cudaStream_t s) {
    constexpr int V = Vec<TX>::N;
    const int vectors = (in.K + V - 1) / V;
    // a warp's one vector a lane (33000 rows of 256 BF16 values 8.5 us, by two a lane 10.8)
    if (vectors <= 32) return rows_launch<TX, 32, 1>(in, q, ldq, scale, s);
    // rows that are few: as many threads as a row has vectors (128 rows of 1024 values with
    // a norm, FP32 1.5 us, by two vectors a thread 1.7, BF16 1.6 and 2.0; 300 rows, FP32, 1.9
    // and 1.75)
    if (in.T <= 296) {
        if (vectors <= 256) return rows_launch<TX, 256, 1>(in, q, ldq, scale, s);
        if (vectors <= 512) return rows_launch<TX, 256, 2>(in, q, ldq, scale, s);
    }
    // many: two vectors a thread, which leaves room for four CTAs an SM (6541 rows of 1024
    // FP32 values 6.8 us, by four vectors 6.7, by one 8.5; 5003 of 2048 BF16 8.6, 10.2
    // and 9.3)
    if (vectors <= 64) return rows_launch<TX, 32, 2>(in, q, ldq, scale, s);
    if (vectors <= 128) return rows_launch<TX, 64, 2>(in, q, ldq, scale, s);
    if (vectors <= 256) return rows_launch<TX, 128, 2>(in, q, ldq, scale, s);
    if (vectors <= 512) return rows_launch<TX, 256, 2>(in, q, ldq, scale, s);
    if (vectors <= 1024) return rows_launch<TX, 256, 4>(in, q, ldq, scale, s);
    if constexpr (V == 4) {
        if (vectors <= 2048) return rows_launch<TX, 256, 8>(in, q, ldq, scale, s);
    }
    return launch(quantize_long_kernel<TX>, dim3(in.T), dim3(256), 0, s, true, in, q, ldq, scale);
}

cudaError_t quantize_launch(const RowsIn& in, int8_t* q, long long ldq, float* scale, cudaStream_t s) {
    return with_type(in.type, [&](auto x) { return quantize_typed<decltype(x)>(in, q, ldq, scale, s); });
}

}  // namespace skb
