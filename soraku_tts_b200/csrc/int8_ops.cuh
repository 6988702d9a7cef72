// Shared pieces of the products in 8-bit integers (int8_rows.cu, int8_gemv.cu,
// int8_gemm.cu).
//
// A row y of K values becomes codes q_k = round(y_k / s), s = max |y| (1 / 127),
// so that y is about q s.  The quotient is the FP32 one, rounded to even: a
// code is a definite number, the same from every kernel.  With a norm,
// y_k = x_k w_k and the row's scale is s / sqrt(mean x^2 + eps): the root mean
// square divides a whole row, so it moves the scale and no code.  Squares are added
// up in one order (Squares below), so that neither codes nor scale depend on the
// rows beside it or on the kernel.
//
// A product's sum over K is exact in 32 bits (K <= 131071), in any order;
//   out = (sum_k q_x q_w) s_x s_w + bias + residual
// is FP32 from there, rounded once to the output's type.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "ops.cuh"
#include "umma.cuh"

namespace skb {

constexpr int I8_MAX_K = 131071;  // 128 * 128 * K < 2^31

__host__ __device__ inline int ceil16(int k) { return (k + 15) & ~15; }
inline int type_size(int t) { return t == SKB_F32 ? 4 : t == SKB_I8 ? 1 : 2; }

// Activations: values with an optional norm, or codes with their scales.
struct RowsIn {
    const void* x;
    int type;
    long long ld;        // elements
    const float* scale;  // of codes
    const float* nw;     // norm weight [K] or null
    float eps;
    int T, K;
};

struct Int8Args {
    RowsIn in;
    const int8_t* w[2];     // weights (or gate, up) [N][ldw]
    long long ldw[2];       // bytes
    const float* ws[2];     // [N]
    int N;                  // output columns
    const float* bias;      // [N] or null
    const void* residual;   // of the output's type, or null
    long long ldr;
    void* out;
    int out_type;
    long long ldo;
};

// Shared-memory attributes of a kernel, once on each device.
template <auto Kernel>
cudaError_t prepare_kernel(size_t dyn_bytes) {
    static std::atomic<bool> done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool known = dev >= 0 && dev < 64;
    if (known && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    e = set_smem_attrs(Kernel, dyn_bytes);
    if (e == cudaSuccess && known) done[dev].store(true, std::memory_order_release);
    return e;
}

cudaError_t quantize_launch(const RowsIn& in, int8_t* q, long long ldq, float* scale, cudaStream_t s);
// Tensor maps: rows of K bytes in boxes of 128 bytes x `box` rows, 128-byte swizzle,
// zeros outside; an output in boxes of 32 columns x `tokens` rows.
bool int8_map(CUtensorMap* m, const void* p, int K, int rows, long long ld, int box);
bool out_map(CUtensorMap* m, void* p, int type, int N, int T, long long ld, int tokens);
bool int8_wide_serves(const Int8Args& a);
cudaError_t int8_wide_launch(const Int8Args& a, bool glu, bool early, cudaStream_t s);
bool int8_gemv_serves(const Int8Args& a, bool glu);
bool int8_gemv_fuses(int T, int K);
cudaError_t int8_gemv_launch(const Int8Args& a, bool glu, bool early, cudaStream_t s);
cudaError_t int8_gemm_launch(const Int8Args& a, bool glu, bool early, cudaStream_t s);

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// A value by way of L2, or of L1 (NEAR).  CUDA's own __ldcg and __ldca of 16-bit types
// are not volatile: the compiler may take them out of the condition that guards them (a
// residual that is not there was read, an illegal address) or past a wait.  Those of
// whole numbers are.
template <bool NEAR = false, class T>
__device__ __forceinline__ T read(const T* p) {
    if constexpr (sizeof(T) == 2) {
        const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
        const unsigned short bits = NEAR ? __ldca(u) : __ldcg(u);
        if constexpr (std::is_same<T, __half>::value) return __ushort_as_half(bits);
        else return __ushort_as_bfloat16(bits);
    } else {
        return NEAR ? __ldca(p) : __ldcg(p);
    }
}

// The place of this CTA's shared memory in that of a CTA of its cluster; all of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Of numbers that are not negative, a warp's largest, NaN above all: in the order
// of their bits.
__device__ __forceinline__ float warp_top(float a) {
    return __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(a) & 0x7fffffffu));
}
// s = max times FP32's 1 / 127, as elementary operations on the device form max / 127 (a
// true division gave another s in some rows, and there another code where y / s was
// next to a half: one of 6.7 million); no smaller than the smallest normal number, where the
// quotient by it stays finite.  NaN for a row that holds something not finite.
__device__ __forceinline__ float step_of(float top) {
    return top <= 3.402823466e38f ? fmaxf(__fmul_rn(top, 1.f / 127.f), 1.17549435e-38f) : __int_as_float(0x7fffffff);
}
// About 1 / s, which is enough to find codes by (encode).
__device__ __forceinline__ float codes_per(float top) {
    return top > 1e-30f && top < 1e30f ? __fdividef(127.f, top) : __fdiv_rn(1.f, step_of(top));
}

// 16 bytes of a row's values.
template <class TX>
struct Vec {
    static constexpr int N = 16 / sizeof(TX);
    union {
        uint4 raw;
        TX e[N];
    };
    __device__ __forceinline__ Vec() {}
    // The `left` values at p, zeros behind them.  NEAR: by way of L1, for what many warps
    // of an SM read; all of them at L2, the few lines that a norm's weights are serve one
    // after the other (2368 rows of 512 BF16 values 8.0 us with a norm, 2.4 without).
    template <bool NEAR = false>
    __device__ __forceinline__ void load(const TX* p, int left, bool aligned) {
        if (aligned && left >= N) {
            const uint4* v = reinterpret_cast<const uint4*>(p);
            raw = NEAR ? __ldca(v) : __ldcg(v);
        } else {
            raw = make_uint4(0, 0, 0, 0);
            if (left > 0) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i < left) e[i] = read<NEAR>(p + i);
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[N]) const {
        if constexpr (sizeof(TX) == 4) {
            v[0] = __uint_as_float(raw.x), v[1] = __uint_as_float(raw.y);
            v[2] = __uint_as_float(raw.z), v[3] = __uint_as_float(raw.w);
        } else if constexpr (std::is_same<TX, __nv_bfloat16>::value) {
            const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = to_float(e[i]);
        }
    }
};

// Codes of N values, four bytes a word: round(y / s) with the FP32 quotient, halves
// to even.  Adding 1.5 2^23 rounds y times 1 / s and leaves the code in the low
// byte.  That product is within 6e-5 of the quotient (|q| <= 127; 2^-22 for r and
// three roundings of 2^-24), so only values next to a half need s and the division:
// one in five thousand, looked for once in N.  Not finite: zeros.
template <int N>
__device__ __forceinline__ void encode(const float (&y)[N], float top, float r, uint32_t (&word)[N / 4]) {
    constexpr float MAGIC = 12582912.f;
    const float2 r2 = make_float2(r, r), up = make_float2(MAGIC, MAGIC), minus = make_float2(-1.f, -1.f);
    uint32_t q[N];
    float off = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 t = make_float2(y[i], y[i + 1]), m = fma2(t, r2, up), d = fma2(t, r2, fma2(m, minus, up));
        q[i] = __float_as_uint(m.x), q[i + 1] = __float_as_uint(m.y);
        off = max3_abs(off, d.x, d.y);
    }
    if (off > 0.4999f) {
        const float s = step_of(top);
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = __float_as_uint(__fadd_rn(__fdiv_rn(y[i], s), MAGIC));
    }
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
        word[h] = __byte_perm(__byte_perm(q[4 * h], q[4 * h + 1], 0x0040), __byte_perm(q[4 * h + 2], q[4 * h + 3], 0x0040), 0x5410);
        if (!(top <= 3.402823466e38f)) word[h] = 0;
    }
}
template <int N>
__device__ __forceinline__ void put_codes(int8_t* q, const uint32_t (&word)[N / 4]) {
    if constexpr (N == 4) *reinterpret_cast<uint32_t*>(q) = word[0];
    else *reinterpret_cast<uint2*>(q) = make_uint2(word[0], word[1]);
}

// A row's sum of squares, added in one order that depends on nothing but the row, so that
// its scale is the same in any batch and from every kernel.  A group of G threads holds a
// row's 16-byte vectors 32 j + lane, j = c W + warp for a thread's c-th one (W = G / 32).
// Vectors of a lane with equal j mod 8 are one chain, j ascending, even and odd values
// apart; a chain's lanes are added in a butterfly, then the eight chains in order.  W
// divides eight: a thread of a small group holds N chains, and none of them crosses a warp.
// What is not there adds an exact zero.
template <int G, int CH>
struct Squares {
    static constexpr int W = G / 32, N = CH < 8 / W ? CH : 8 / W, CHAINS = W * N;
    static_assert(W <= 8 && 8 % W == 0 && N <= 2 && CH % N == 0, "chains of a thread");
    float2 s[N];
    __device__ __forceinline__ Squares() {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = make_float2(0.f, 0.f);
    }
    __device__ __forceinline__ void add(int c, float2 x) { s[c % N] = fma2(x, x, s[c % N]); }
    // This thread's chains, even and odd values together.
    __device__ __forceinline__ float2 ends() const { return make_float2(s[0].x + s[0].y, N == 2 ? s[N - 1].x + s[N - 1].y : 0.f); }
    // Over the warp: chain `warp` in lane 0, and, of two, chain W + warp in lane 16.
    __device__ __forceinline__ static float over_lanes(float2 ends, int lane) {
        float a = ends.x;
        if constexpr (N == 2) {
            const bool second = lane & 16;
            const float other = __shfl_xor_sync(FULL, second ? ends.x : ends.y, 16);
            a = (second ? ends.y : ends.x) + other;
        } else {
            a += __shfl_xor_sync(FULL, a, 16);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(FULL, a, o);
        return a;
    }
    // Where a row's chains have the one that thread t holds then: lane 0, and, of two, lane 16.
    __device__ __forceinline__ static int place(int t) { return N == 2 ? (t >> 5) + W * ((t >> 4) & 1) : t >> 5; }
    __device__ __forceinline__ static bool holds(int t) { return (t & (N == 2 ? 15 : 31)) == 0; }
    __device__ __forceinline__ static float total(const float* chains) {  // on 16 bytes
        float sum = 0.f;
        if constexpr (CHAINS % 4 == 0) {
#pragma unroll
            for (int i = 0; i < CHAINS; i += 4) {
                const float4 c = *reinterpret_cast<const float4*>(chains + i);
                sum = (((sum + c.x) + c.y) + c.z) + c.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < CHAINS; ++i) sum += chains[i];
        }
        return sum;
    }
};

// Floats that a row's threads leave for each other: largest of their warps, chains.
constexpr int ROW_RED = 16;

// One row by a group of G threads (G a multiple of 32; `t`: place in it):
// codes to `q` (16-byte aligned, zeros up to ceil16(K)), the scale returned to
// every thread.  A thread keeps CH vectors; longer rows are read twice, but for
// the last piece.  `red`: ROW_RED floats on 16 bytes; all threads of the CTA have to call this
// together.
template <class TX, int G, int CH>
__device__ __forceinline__ float quantize_row(const TX* __restrict__ x, const float* __restrict__ nw, float eps, int K,
                                              bool x_aligned, int8_t* q, int t, float* red) {
    constexpr int V = Vec<TX>::N;
    constexpr int PIECE = G * CH * V;
    using SQ = Squares<G, CH>;
    static_assert(G > 32 && CH * (G / 32) % 8 == 0, "a piece goes on with the chains of the one before");
    const bool w_aligned = (reinterpret_cast<uintptr_t>(nw) & 15) == 0;
    float v[CH][V];
    float top = 0.f, ss = 0.f;
    SQ squares;
    auto load = [&](int base) {
        Vec<TX> raw[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = base + (c * G + t) * V;
            raw[c].template load<true>(x + k, K - k, x_aligned);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) raw[c].get(v[c]);
    };
    auto weigh = [&](int base, bool first) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = base + (c * G + t) * V;
            if (nw != nullptr) {
#pragma unroll
                for (int h = 0; h < V / 4; ++h) {
                    Vec<float> raw;
                    raw.template load<true>(nw + k + 4 * h, K - k - 4 * h, w_aligned);
                    float w[4];
                    raw.get(w);
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        float &y0 = v[c][4 * h + i], &y1 = v[c][4 * h + i + 1];
                        if (first) squares.add(c, make_float2(y0, y1));
                        y0 = __fmul_rn(y0, w[i]), y1 = __fmul_rn(y1, w[i + 1]);
                    }
                }
            }
            if (first) {
#pragma unroll
                for (int i = 0; i < V; i += 2) top = max3_abs(top, v[c][i], v[c][i + 1]);
            }
        }
    };
    int base = 0;
    for (;; base += PIECE) {
        load(base);
        weigh(base, true);
        if (base + PIECE >= K) break;
    }
    top = warp_top(top);
    if ((t & 31) == 0) red[t >> 5] = top;
    if (nw != nullptr) {
        ss = SQ::over_lanes(squares.ends(), t & 31);
        if (SQ::holds(t)) red[8 + SQ::place(t)] = ss;
    }
    __syncthreads();
    top = 0.f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) top = max3_abs(top, red[w], 0.f);
    if (nw != nullptr) ss = SQ::total(red + 8);
    const float r = codes_per(top);
    for (;;) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = base + (c * G + t) * V;
            if (k >= ceil16(K)) continue;
            uint32_t word[V / 4];
            encode<V>(v[c], top, r, word);
            put_codes<V>(q + k, word);
        }
        if (base == 0) break;
        base -= PIECE;
        load(base);
        weigh(base, false);
    }
    const float s = step_of(top);
    return nw != nullptr ? s * rsqrtf(ss / (float)K + eps) : s;
}

// A sum's way to its result; the same operations in every kernel, so that from its
// codes and scale on a token's result does not depend on how many stand beside it.  `bias`: 0 without.
__device__ __forceinline__ float finish(int sum, float sx, float sw, float bias) {
    return fmaf(__fmul_rn((float)sum, sx), sw, bias);
}
// (float)v without the conversion unit, which a SwiGLU's exponentials and
// reciprocals share: two exact halves, rounded as they are joined.
__device__ __forceinline__ float whole_to_float(int v) {
    const float hi = __fsub_rn(__int_as_float(0x4b400000 + (v >> 16)), 12582912.f);
    const float lo = __fsub_rn(__int_as_float(0x4b000000 | (v & 0xffff)), 8388608.f);
    return fmaf(hi, 65536.f, lo);
}
// silu by the hardware's exponential and reciprocal: each is within 2^-22 of
// its value, where the product's own roundings are 2^-22 already, and the
// argument's rounding counts |g| 2^-24, as that of g itself does.  (The exact
// ones took 30 instructions more of each result.)
__device__ __forceinline__ float finish_glu(int gate, int up, float sx, float sg, float su) {
    const float g = finish(gate, sx, sg, 0.f);
    return __fmul_rn(__fdividef(g, __fadd_rn(1.0f, __expf(-g))), fmaf(__fmul_rn(whole_to_float(up), sx), su, 0.f));
}

template <class T>
__device__ __forceinline__ void store_out(T* p, float v) { *p = from_float<T>(v); }

__device__ __forceinline__ float load_as(const void* p, int type, long long i) {
    if (type == SKB_F32) return read(static_cast<const float*>(p) + i);
    if (type == SKB_BF16) return to_float(read(static_cast<const __nv_bfloat16*>(p) + i));
    return to_float(read(static_cast<const __half*>(p) + i));
}
__device__ __forceinline__ void store_as(void* p, int type, long long i, float v) {
    if (type == SKB_F32) store_out(static_cast<float*>(p) + i, v);
    else if (type == SKB_BF16) store_out(static_cast<__nv_bfloat16*>(p) + i, v);
    else store_out(static_cast<__half*>(p) + i, v);
}

// f(TO()) with the output's type.
template <class F>
inline cudaError_t with_type(int type, F f) {
    if (type == SKB_F32) return f(float());
    if (type == SKB_BF16) return f(__nv_bfloat16());
    return f(__half());
}

}  // namespace skb
