// C entries of the products in 8-bit integers: their checks, and which kernels
// serve a call.
#include "int8_ops.cuh"

namespace skb {

static int check_rows(const char* what, const RowsIn& in, bool codes_too) {
    if (in.T < 0 || in.T > 1 << 30 || in.K < 1 || in.K > I8_MAX_K)
        return fail(SKB_ERR_ARG, "%s: bad sizes (%d rows of %d; at most 2^30, of 1 to %d values)", what, in.T, in.K, I8_MAX_K);
    if (in.type < SKB_F32 || in.type > (codes_too ? SKB_I8 : SKB_F16))
        return fail(SKB_ERR_ARG, "%s: unknown type %d of the rows", what, in.type);
    if (!in.x) return fail(SKB_ERR_ARG, "%s: null pointer", what);
    if (in.type == SKB_I8) {
        if (!in.scale) return fail(SKB_ERR_ARG, "%s: codes need their scales", what);
        if (in.nw) return fail(SKB_ERR_ARG, "%s: codes take no norm", what);
        if (!aligned16(in.x) || in.ld % 16 != 0 || in.ld < ceil16(in.K))
            return fail(SKB_ERR_ARG, "%s: rows of codes must begin on 16 bytes", what);
    } else {
        if (in.scale) return fail(SKB_ERR_ARG, "%s: scales belong to codes", what);
        if (in.ld < in.K) return fail(SKB_ERR_ARG, "%s: rows overlap", what);
        if (reinterpret_cast<uintptr_t>(in.x) % type_size(in.type) != 0 || reinterpret_cast<uintptr_t>(in.nw) % 4 != 0)
            return fail(SKB_ERR_ARG, "%s: misaligned pointer", what);
        if (!(in.eps >= 0.f) || in.eps > 3e38f) return fail(SKB_ERR_ARG, "%s: eps must be finite and not negative", what);
    }
    return SKB_OK;
}

static int check_product(const char* what, const Int8Args& a, int parts) {
    const int st = check_rows(what, a.in, true);
    if (st) return st;
    if (a.N < 1 || a.N > 1 << 30) return fail(SKB_ERR_ARG, "%s: bad output width %d", what, a.N);
    for (int i = 0; i < parts; ++i) {
        if (!a.w[i] || !a.ws[i]) return fail(SKB_ERR_ARG, "%s: null pointer", what);
        if (!aligned16(a.w[i]) || a.ldw[i] % 16 != 0 || a.ldw[i] < ceil16(a.in.K))
            return fail(SKB_ERR_ARG, "%s: rows of weights must begin on 16 bytes", what);
        if (reinterpret_cast<uintptr_t>(a.ws[i]) % 4 != 0) return fail(SKB_ERR_ARG, "%s: misaligned pointer", what);
    }
    if (a.out_type < SKB_F32 || a.out_type > SKB_F16) return fail(SKB_ERR_ARG, "%s: unknown type %d of the output", what, a.out_type);
    if (!a.out) return fail(SKB_ERR_ARG, "%s: null pointer", what);
    if (a.ldo < a.N || (a.residual && a.ldr < a.N)) return fail(SKB_ERR_ARG, "%s: rows overlap", what);
    const int size = type_size(a.out_type);
    if (reinterpret_cast<uintptr_t>(a.out) % size != 0 || reinterpret_cast<uintptr_t>(a.residual) % size != 0 ||
        reinterpret_cast<uintptr_t>(a.bias) % 4 != 0)
        return fail(SKB_ERR_ARG, "%s: misaligned pointer", what);
    return SKB_OK;
}

static int64_t workspace_of(int T, int K, int type) {
    return type == SKB_I8 || int8_gemv_fuses(T, K) ? 0 : (int64_t)T * ceil16(K) + (int64_t)T * 4;
}

static int product(const char* what, Int8Args& a, bool glu, void* work, int64_t bytes, cudaStream_t s) {
    const int st = check_product(what, a, glu ? 2 : 1);
    if (st || a.in.T == 0) return st;
    const int64_t need = workspace_of(a.in.T, a.in.K, a.in.type);
    if (need > 0) {
        if (!work || bytes < need || !aligned16(work)) return fail(SKB_ERR_ARG, "%s: workspace too small or misaligned", what);
        const int kp = ceil16(a.in.K);
        int8_t* q = static_cast<int8_t*>(work);
        float* scale = reinterpret_cast<float*>(q + (int64_t)a.in.T * kp);
        const cudaError_t e = quantize_launch(a.in, q, kp, scale, s);
        if (e != cudaSuccess) return fail(SKB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
        a.in = {q, SKB_I8, kp, scale, nullptr, 0.f, a.in.T, a.in.K};
    }
    const cudaError_t e = int8_gemv_serves(a, glu) ? int8_gemv_launch(a, glu, need > 0, s) : int8_gemm_launch(a, glu, need > 0, s);
    return e == cudaSuccess ? SKB_OK : fail(SKB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace skb

using namespace skb;

extern "C" {

int skb_quantize_rows(const void* x, int x_type, int64_t ldx, int rows, int K, const float* norm_weight, float eps,
                      int8_t* q, int64_t ldq, float* scale, cudaStream_t stream) {
    const RowsIn in = {x, x_type, ldx, nullptr, norm_weight, eps, rows, K};
    const int st = check_rows("quantize_rows", in, false);
    if (st) return st;
    if (!q || !scale) return fail(SKB_ERR_ARG, "quantize_rows: null pointer");
    if (!aligned16(q) || ldq % 16 != 0 || ldq < ceil16(K) || reinterpret_cast<uintptr_t>(scale) % 4 != 0)
        return fail(SKB_ERR_ARG, "quantize_rows: rows of codes must begin on 16 bytes");
    if (rows == 0) return SKB_OK;
    const cudaError_t e = quantize_launch(in, q, ldq, scale, stream);
    return e == cudaSuccess ? SKB_OK : fail(SKB_ERR_CUDA, "quantize_rows: %s", cudaGetErrorString(e));
}

int64_t skb_int8_workspace(int T, int K, int x_type) {
    return T < 1 || K < 1 || K > I8_MAX_K ? 0 : workspace_of(T, K, x_type);
}

int skb_int8_linear(const void* x, int x_type, int64_t ldx, const float* x_scale, const float* norm_weight, float eps,
                    int T, int K, const int8_t* w, int64_t ldw, const float* w_scale, int N, const float* bias,
                    const void* residual, int64_t ldr, void* out, int out_type, int64_t ldo, void* workspace,
                    int64_t workspace_bytes, cudaStream_t stream) {
    Int8Args a = {{x, x_type, ldx, x_scale, norm_weight, eps, T, K}, {w, nullptr}, {ldw, 0}, {w_scale, nullptr}, N, bias,
                  residual, ldr, out, out_type, ldo};
    return product("int8_linear", a, false, workspace, workspace_bytes, stream);
}

int skb_int8_swiglu(const void* x, int x_type, int64_t ldx, const float* x_scale, const float* norm_weight, float eps,
                    int T, int K, const int8_t* gate, int64_t ldg, const float* gate_scale, const int8_t* up, int64_t ldu,
                    const float* up_scale, int I, void* out, int out_type, int64_t ldo, void* workspace,
                    int64_t workspace_bytes, cudaStream_t stream) {
    Int8Args a = {{x, x_type, ldx, x_scale, norm_weight, eps, T, K}, {gate, up}, {ldg, ldu}, {gate_scale, up_scale}, I,
                  nullptr, nullptr, 0, out, out_type, ldo};
    return product("int8_swiglu", a, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
