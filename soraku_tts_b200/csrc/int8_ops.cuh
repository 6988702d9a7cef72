// Shared pieces of the products in 8-bit integers (int8_rows.cu, int8_gemv.cu,
// int8_gemm.cu).
//
// A row y of K values becomes codes q_k = round(y_k / s), s = max |y| / 127,
// so that y is about q s.  The quotient is the FP32 one, rounded to even: a
// code is a definite number, the same from every kernel.  With a norm,
// y_k = x_k w_k and the row's scale is s / sqrt(mean x^2 + eps): the root mean
// square divides a whole row, so it moves the scale and no code, and codes do
// not depend on the order in which squares are added up.
//
// A product's sum over K is exact in 32 bits (K <= 131071), in any order;
//   out = (sum_k q_x q_w) s_x s_w + bias + residual
// is FP32 from there, rounded once to the output's type.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "ops.cuh"

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
constexpr int I8_FEW = 8;  // tokens that int8_gemv.cu serves
bool int8_gemv_fuses(int T, int K);
cudaError_t int8_gemv_launch(const Int8Args& a, bool glu, cudaStream_t s);
cudaError_t int8_gemm_launch(const Int8Args& a, bool glu, cudaStream_t s);

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// Largest of |a|, |b|; NaN if one of them is.
__device__ __forceinline__ float max_abs(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}
// s = max / 127, and no smaller than the smallest normal number, where the
// quotient by it stays finite.  NaN for a row that holds something not finite.
__device__ __forceinline__ float step_of(float top) {
    return top <= 3.402823466e38f ? fmaxf(__fdiv_rn(top, 127.f), 1.17549435e-38f) : __int_as_float(0x7fffffff);
}
// round(y / s) with the FP32 quotient: y times 1 / s is within 3e-5 of it
// (|q| <= 127, three roundings), so only near halves is it formed.
__device__ __forceinline__ int code_of(float y, float s, float r) {
    const float t = y * r;
    float q = rintf(t);
    if (fabsf(fabsf(t - q) - 0.5f) < 1e-4f) q = rintf(__fdiv_rn(y, s));
    return (int)q;
}

// VEC consecutive values: 16 bytes of the type.
template <class TX>
struct Vec {
    static constexpr int N = 16 / sizeof(TX);
};
template <class TX>
__device__ __forceinline__ void load_vec(const TX* p, int left, bool aligned, float (&v)[Vec<TX>::N]) {
    if (aligned && left >= Vec<TX>::N) {
        const uint4 u = __ldcg(reinterpret_cast<const uint4*>(p));
        const TX* e = reinterpret_cast<const TX*>(&u);
#pragma unroll
        for (int i = 0; i < Vec<TX>::N; ++i) v[i] = to_float(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < Vec<TX>::N; ++i) v[i] = i < left ? to_float(__ldcg(p + i)) : 0.f;
    }
}

// One row by a group of G threads (G a multiple of 32; `t`: place in it):
// codes to `q` (16-byte aligned, zeros up to ceil16(K)), the scale returned to
// every thread.  A thread keeps CH vectors; longer rows are read twice, but for
// the last piece.  `red`: 2 floats a warp of the group, if G > 32; then all
// threads of the CTA have to call this together.
template <class TX, int G, int CH>
__device__ __forceinline__ float quantize_row(const TX* __restrict__ x, const float* __restrict__ nw, float eps, int K,
                                              bool x_aligned, int8_t* q, int t, float* red) {
    constexpr int V = Vec<TX>::N;
    constexpr int PIECE = G * CH * V;
    const bool w_aligned = (reinterpret_cast<uintptr_t>(nw) & 15) == 0;
    float v[CH][V];
    float top = 0.f, ss = 0.f;
    auto load = [&](int base) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = base + (c * G + t) * V;
            load_vec<TX>(x + k, K - k, x_aligned, v[c]);
        }
    };
    auto weigh = [&](int base, bool first) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = base + (c * G + t) * V;
            if (nw != nullptr) {
#pragma unroll
                for (int h = 0; h < V / 4; ++h) {
                    float w[4];
                    load_vec<float>(nw + k + 4 * h, K - k - 4 * h, w_aligned, w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float& y = v[c][4 * h + i];
                        if (first) ss = fmaf(y, y, ss);
                        y = k + 4 * h + i < K ? __fmul_rn(y, w[i]) : 0.f;
                    }
                }
            }
            if (first) {
#pragma unroll
                for (int i = 0; i < V; ++i) top = max_abs(top, v[c][i]);
            }
        }
    };
    int base = 0;
    for (;; base += PIECE) {
        load(base);
        weigh(base, true);
        if (base + PIECE >= K) break;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        top = max_abs(top, __shfl_xor_sync(FULL, top, o));
        ss += __shfl_xor_sync(FULL, ss, o);
    }
    if (G > 32) {
        if ((t & 31) == 0) red[2 * (t >> 5)] = top, red[2 * (t >> 5) + 1] = ss;
        __syncthreads();
        top = 0.f, ss = 0.f;
#pragma unroll
        for (int w = 0; w < G / 32; ++w) top = max_abs(top, red[2 * w]), ss += red[2 * w + 1];
    }
    const float s = step_of(top);
    const bool bad = !(s == s);
    const float r = __fdiv_rn(1.f, s);
    for (;;) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = base + (c * G + t) * V;
            if (k >= ceil16(K)) continue;
            uint32_t word[V / 4];
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                word[h] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int code = bad ? 0 : code_of(v[c][4 * h + i], s, r);
                    word[h] |= (uint32_t)(code & 0xff) << (8 * i);
                }
            }
            if (V == 4)
                *reinterpret_cast<uint32_t*>(q + k) = word[0];
            else
                *reinterpret_cast<uint2*>(q + k) = make_uint2(word[0], word[V / 4 - 1]);
        }
        if (base == 0) break;
        base -= PIECE;
        load(base);
        weigh(base, false);
    }
    return nw != nullptr ? s * rsqrtf(ss / (float)K + eps) : s;
}

__device__ __forceinline__ float load_as_float(const void* p, int type, long long i) {
    if (type == SKB_F32) return __ldcg(static_cast<const float*>(p) + i);
    if (type == SKB_BF16) return __bfloat162float(__ldcg(static_cast<const __nv_bfloat16*>(p) + i));
    return __half2float(__ldcg(static_cast<const __half*>(p) + i));
}
__device__ __forceinline__ void store_as(void* p, int type, long long i, float v) {
    if (type == SKB_F32) static_cast<float*>(p)[i] = v;
    else if (type == SKB_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

}  // namespace skb
