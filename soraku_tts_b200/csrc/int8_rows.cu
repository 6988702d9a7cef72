// Rows of values to rows of 8-bit codes, each with its scale (int8_ops.cuh has
// the definition).  Activations before a product, weights once.
#include "int8_ops.cuh"

namespace skb {

// Rows of up to 1024 values: a warp each, the values in its registers between
// the largest's search and the codes.  Longer ones: a CTA each, up to 8192
// values in registers, the rest read again from L2.
template <class TX, int G>
__global__ void __launch_bounds__(256) quantize_kernel(const RowsIn in, int8_t* __restrict__ q, long long ldq,
                                                       float* __restrict__ scale) {
    __shared__ float red[16];
    pdl_wait();
    pdl_trigger();
    const long long row = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (G < 256 && row >= in.T) return;  // whole warps
    const int t = threadIdx.x % G;
    const TX* x = static_cast<const TX*>(in.x) + row * in.ld;
    const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    const float s = quantize_row<TX, G, 32 / Vec<TX>::N>(x, in.nw, in.eps, in.K, aligned, q + row * ldq, t, red);
    if (t == 0) scale[row] = s;
}

template <class TX>
static cudaError_t quantize_typed(const RowsIn& in, int8_t* q, long long ldq, float* scale, cudaStream_t s) {
    if (in.K <= 1024)
        return launch(quantize_kernel<TX, 32>, dim3((in.T + 7) / 8), dim3(256), 0, s, true, in, q, ldq, scale);
    return launch(quantize_kernel<TX, 256>, dim3(in.T), dim3(256), 0, s, true, in, q, ldq, scale);
}

cudaError_t quantize_launch(const RowsIn& in, int8_t* q, long long ldq, float* scale, cudaStream_t s) {
    if (in.type == SKB_F32) return quantize_typed<float>(in, q, ldq, scale, s);
    if (in.type == SKB_BF16) return quantize_typed<__nv_bfloat16>(in, q, ldq, scale, s);
    return quantize_typed<__half>(in, q, ldq, scale, s);
}

}  // namespace skb
