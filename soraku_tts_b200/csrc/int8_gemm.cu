// Products of 8-bit codes on the 5th-generation tensor cores
// (tcgen05.mma kind::i8, sums in 32-bit integers in tensor memory):
//   D[n][t] = sum_k W[n][k] X[t][k]
// Weights are the M operand, so that a product of few tokens costs few columns,
// and a thread of the epilogue holds one output channel: its scale and bias
// stay in registers, and a warp writes 32 neighbouring channels of a token.
//
// A CTA takes tiles of 128 channels x TN tokens (for SwiGLU the 128 gate rows
// and the 128 up rows of the same channels, two accumulators).  Warps:
//   0 (one thread)   TMA: K in blocks of 128 bytes, the width of the 128-byte
//                    swizzle, into a ring of stages; rows and bytes past the
//                    end arrive as zeros, which add nothing;
//   1 (one thread)   four MMAs of 32 bytes a block and part;
//   4-11             the epilogue of one tile while the next one is added up
//                    (two accumulators take turns).
// Where tiles are fewer than SMs, a cluster of CTAs splits a tile's K: whole
// numbers, so that the order of their sum does not matter.  Every CTA leaves
// its sums in its shared memory and finishes its share of the tile's tokens.
//
// What bounds it, 128 tokens of 1024 to 4096 channels (128 CTAs of 128 x 32, 5.1 us): the
// products take 0.3 us and the bytes 1.0; the rest is a chain of latencies, launch and
// barriers, the first copy, eight blocks, the sums out.  77 tokens to 2 x 2048 channels
// 5.7 to 6.0 us.
#include <cudaTypedefs.h>

#include <cstddef>

#include "int8_ops.cuh"
#include "umma.cuh"

namespace skb {

constexpr int GM_THREADS = 384, GM_EPI = 256;
constexpr int GM_MAX_SPLIT = 8;
constexpr int GM_RING = 196 * 1024;

struct GemmMaps {
    CUtensorMap x, w[2];
};

template <int TN, bool GLU>
struct GemmShape {
    static constexpr int PARTS = GLU ? 2 : 1;
    static constexpr int A_BYTES = 128 * 128, B_BYTES = TN * 128;
    static constexpr int STAGE = PARTS * A_BYTES + B_BYTES;
    static constexpr int STAGES = GM_RING / STAGE < 8 ? GM_RING / STAGE : 8;
    static constexpr int COLS = PARTS * TN;       // of one accumulator
    static constexpr int TMEM = 2 * COLS < 32 ? 32 : 2 * COLS;
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE;
    static_assert(COLS * 512 <= STAGES * STAGE, "a split's sums fit the ring");
};

struct GemmShared {
    uint64_t full[8], empty[8], acc_full[2], acc_free[2];
    uint32_t tmem;
    int abort;
    alignas(16) float sx[GM_EPI / 32][128];  // scales of a warp's tokens, read four at a time
};
static_assert(offsetof(GemmShared, sx) % 16 == 0 && alignof(GemmShared) % 16 == 0, "16-byte reads");

__device__ __forceinline__ void gm_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
// D S32, A and B S8, both K-major, M = 128.
__host__ __device__ constexpr uint32_t gm_idesc(int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void gm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ int gm_peer_load(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ int4 gm_peer_load4(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

template <int TN, bool GLU, class TO>
__global__ void __launch_bounds__(GM_THREADS, 1) int8_gemm_kernel(const Int8Args a, const __grid_constant__ GemmMaps maps, int split,
                                                                  bool early) {
    using S = GemmShape<TN, GLU>;
    extern __shared__ unsigned char gm_raw[];
    __shared__ GemmShared sm;
    unsigned char* base = gm_raw + ((1024u - (smem_u32(gm_raw) & 1023u)) & 1023u);
    const uint32_t ring = smem_u32(base);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) mbar_init(&sm.full[i], 1), mbar_init(&sm.empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&sm.acc_full[i], 1), mbar_init(&sm.acc_free[i], GM_EPI / 32);
        sm.abort = 0;
        mbar_fence_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.x)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.w[0])) : "memory");
        if (GLU) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.w[1])) : "memory");
    }
    if (warp == 2) ut_alloc<S::TMEM>(&sm.tmem);
    ut_fence_before();
    __syncthreads();
    ut_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* abort = &sm.abort;

    const int tiles_n = (a.N + 127) / 128, tiles_t = (a.in.T + TN - 1) / TN;
    const int tiles = tiles_n * tiles_t;  // the launch has seen that they are fewer than 2^30
    const int blocks = (a.in.K + 127) / 128;
    const int z = blockIdx.x % split;  // rank in the cluster
    const int k0 = (int)((long long)z * blocks / split), k1 = (int)((long long)(z + 1) * blocks / split);
    const int first = blockIdx.x / split, step = gridDim.x / split;
    // blocks whose weights are asked for before the wait
    int ahead = 0;
    auto load_w = [&](int n0, int kb, uint32_t at, uint64_t* bar) {
        gm_load(at, &maps.w[0], kb * 128, n0, bar);
        if (GLU) gm_load(at + S::A_BYTES, &maps.w[1], kb * 128, n0, bar);
    };
    if (early && tid == 0 && first < tiles) {
        for (; ahead < S::STAGES && k0 + ahead < k1; ++ahead) {
            mbar_expect_tx(&sm.full[ahead], S::STAGE);
            load_w(first % tiles_n * 128, k0 + ahead, ring + ahead * S::STAGE, &sm.full[ahead]);
        }
    }
    pdl_wait();
    pdl_trigger();

    // One thread issues a copy or a product, against whatever the other warps run: no
    // division on its way, stages and phases are counted along.
    if (warp == 0) {
        if (lane == 0) {
            int s = 0, asked = 0;  // stage; blocks asked for, of the first round alone
            uint32_t phase = 1;    // of the ring's barriers: the first round waits for nothing
            bool go = true;
            for (int tile = first; tile < tiles && go; tile += step) {
                const int n0 = tile % tiles_n * 128, t0 = tile / tiles_n * TN;
                for (int kb = k0; kb < k1; ++kb) {
                    if (asked >= S::STAGES && !ut_wait(&sm.empty[s], phase, abort)) {
                        go = false;
                        break;
                    }
                    const uint32_t at = ring + s * S::STAGE;
                    if (asked >= ahead) {
                        mbar_expect_tx(&sm.full[s], S::STAGE);
                        load_w(n0, kb, at, &sm.full[s]);
                    }
                    gm_load(at + S::PARTS * S::A_BYTES, &maps.x, kb * 128, t0, &sm.full[s]);
                    asked = min(asked + 1, S::STAGES);
                    if (++s == S::STAGES) s = 0, phase ^= 1;
                }
            }
            // no copy may land after the CTA has gone: the MMAs wait for each of
            // them; where those gave up, wait here, from the oldest on
            if (*abort)
                for (int i = 0; i < asked; ++i) {
                    const bool wrapped = asked == S::STAGES && s + i >= S::STAGES;
                    const int at = asked < S::STAGES ? i : (wrapped ? s + i - S::STAGES : s + i);
                    mbar_wait(&sm.full[at], asked < S::STAGES ? 0u : (wrapped ? phase ^ 1 : phase), nullptr);
                }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int s = 0, i = 0;
            uint32_t phase = 0;
            bool go = true;
            for (int tile = first; tile < tiles && go; tile += step, ++i) {
                const int b = i & 1;
                if (i >= 2 && !ut_wait(&sm.acc_free[b], (uint32_t)((i >> 1) - 1) & 1u, abort)) break;
                ut_fence_after();
                const uint32_t d = tmem + b * S::COLS;
                for (int kb = k0; kb < k1; ++kb) {
                    if (!ut_wait(&sm.full[s], phase, abort)) {
                        go = false;
                        break;
                    }
                    ut_fence_after();
                    const uint32_t at = ring + s * S::STAGE;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint64_t x = ut_desc(at + S::PARTS * S::A_BYTES, k * 32, false);
#pragma unroll
                        for (int p = 0; p < S::PARTS; ++p)
                            gm_mma(d + p * TN, ut_desc(at + p * S::A_BYTES, k * 32, false), x, gm_idesc(TN), kb > k0 || k > 0);
                    }
                    ut_commit(&sm.empty[s]);
                    if (++s == S::STAGES) s = 0, phase ^= 1;
                }
                if (go) ut_commit(&sm.acc_full[b]);
            }
            // what was issued ends before tensor memory is given back
            if (*abort) {
                ut_commit(&sm.acc_full[0]);
                for (int n = 0; n < 2; ++n) mbar_wait_limit(&sm.acc_full[0], n, nullptr, 1000000ull);
            }
        }
    } else if (warp >= 4) {
        const int q = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);
        constexpr int CH = 16;  // columns at a time
        float* sx = sm.sx[warp - 4];
        int i = 0;
        for (int tile = first; tile < tiles; tile += step, ++i) {
            const int n = tile % tiles_n * 128 + 32 * q + lane, t0 = tile / tiles_n * TN + half * (TN / 2);
            const int b = i & 1;
            const bool in = n < a.N;
            const float s0 = in ? __ldcg(a.ws[0] + n) : 0.f, s1 = GLU && in ? __ldcg(a.ws[1] + n) : 0.f;
            const float bias = !GLU && a.bias != nullptr && in ? __ldcg(a.bias + n) : 0.f;
            const TO* res = GLU ? nullptr : static_cast<const TO*>(a.residual);
            __syncwarp();
            for (int j = lane; j < TN / 2; j += 32) sx[j] = t0 + j < a.in.T ? __ldcg(a.in.scale + t0 + j) : 0.f;
            TO r_next[GLU ? 1 : CH];  // as it came: a conversion would wait for it
            auto residual_of = [&](int c) {
                const TO* p = res + (long long)(t0 + c) * a.ldr + n;
#pragma unroll
                for (int j = 0; j < CH; ++j, p += a.ldr) r_next[GLU ? 0 : j] = in && t0 + c + j < a.in.T ? read(p) : from_float<TO>(0.f);
            };
            if (!GLU && split == 1 && res != nullptr) residual_of(0);
            // a wait that ran out shows as NaN
            const float poison = ut_wait(&sm.acc_full[b], (uint32_t)(i >> 1) & 1u, abort) ? 1.f : __int_as_float(0x7fffffff);
            __syncwarp();
            ut_fence_after();
#pragma unroll 1
            for (int c = 0; c < TN / 2 && t0 + c < a.in.T; c += CH) {
                uint32_t v[CH], u[GLU ? CH : 1];
                const uint32_t col = lanes + b * S::COLS + half * (TN / 2) + c;
                ut_ld16(col, v);
                if constexpr (GLU) ut_ld16(col + TN, u);
                if (split > 1) {
                    ut_wait_ld();
                    int* sums = reinterpret_cast<int*>(base) + (half * (TN / 2) + c) * 128 + 32 * q + lane;
#pragma unroll
                    for (int j = 0; j < CH; ++j) {
                        sums[j * 128] = (int)v[j];
                        if constexpr (GLU) sums[(TN + j) * 128] = (int)u[j];
                    }
                    continue;
                }
                const int left = in ? a.in.T - t0 - c : 0;  // tokens there are
                float r[GLU ? 1 : CH];
                if (!GLU && res != nullptr) {
#pragma unroll
                    for (int j = 0; j < CH; ++j) r[GLU ? 0 : j] = to_float(r_next[GLU ? 0 : j]);
                    if (c + CH < TN / 2) residual_of(c + CH);  // on their way while these are used
                }
                ut_wait_ld();
                TO* p = static_cast<TO*>(a.out) + (long long)(t0 + c) * a.ldo + n;
                auto put = [&](bool all, bool add) {
#pragma unroll
                    for (int j0 = 0; j0 < CH; j0 += 4) {
                        const float4 s4 = *reinterpret_cast<const float4*>(sx + c + j0);
                        const float sj[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k, p += a.ldo) {
                            const int j = j0 + k;
                            float y;
                            if constexpr (GLU) y = finish_glu((int)v[j], (int)u[j], sj[k], s0 * poison, s1);
                            else y = finish((int)v[j], sj[k], s0 * poison, bias);
                            if (add) y += r[GLU ? 0 : j];
                            if (all || j < left) store_out(p, y);
                        }
                    }
                };
                if (!GLU && res != nullptr) put(false, true);
                else if (left >= CH) put(true, false);
                else put(false, false);
            }
            ut_fence_before();
            __syncwarp();
            if (lane == 0) ut_arrive(&sm.acc_free[b]);
        }
    }
    if (split > 1) {
        __syncwarp();
        cluster_sync();
        const int n0 = first % tiles_n * 128, t0 = first / tiles_n * TN;
        if (warp >= 4) {
            bool bad = false;
            for (int p = 0; p < split; ++p) bad |= gm_peer_load(cluster_addr(smem_u32(&sm.abort), p)) != 0;
            // a warp takes a token, a lane four channels; two tokens' sums are on their way
            const int nt = min(TN, a.in.T - t0), c = 4 * lane, n = n0 + c;
            const TO* res = GLU ? nullptr : static_cast<const TO*>(a.residual);
            float s0[4], s1[4], bias[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool in = n + k < a.N;
                s0[k] = in ? __ldcg(a.ws[0] + n + k) : 0.f;
                s1[k] = GLU && in ? __ldcg(a.ws[1] + n + k) : 0.f;
                bias[k] = !GLU && a.bias != nullptr && in ? __ldcg(a.bias + n + k) : 0.f;
                if (bad) s0[k] = __int_as_float(0x7fffffff);
            }
            constexpr int W = GM_EPI / 32;
            const int t_end = (z + 1) * nt / split;
            for (int t = z * nt / split + warp - 4; t < t_end; t += 2 * W) {
                int v[2][4] = {}, u[2][4] = {};
#pragma unroll
                for (int p = 0; p < GM_MAX_SPLIT; ++p) {
                    if (p >= split) break;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (t + h * W >= t_end) continue;
                        const int4 x = gm_peer_load4(cluster_addr(ring + ((t + h * W) * 128 + c) * 4, p));
                        v[h][0] += x.x, v[h][1] += x.y, v[h][2] += x.z, v[h][3] += x.w;
                        if constexpr (GLU) {
                            const int4 y = gm_peer_load4(cluster_addr(ring + ((TN + t + h * W) * 128 + c) * 4, p));
                            u[h][0] += y.x, u[h][1] += y.y, u[h][2] += y.z, u[h][3] += y.w;
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int tt = t + h * W;
                    if (tt >= t_end) break;
                    const float sx = __ldcg(a.in.scale + t0 + tt);
                    TO* o = static_cast<TO*>(a.out) + (long long)(t0 + tt) * a.ldo + n;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (n + k >= a.N) break;
                        float y;
                        if constexpr (GLU) y = finish_glu(v[h][k], u[h][k], sx, s0[k], s1[k]);
                        else y = finish(v[h][k], sx, s0[k], bias[k]) + (res ? to_float(read(res + (long long)(t0 + tt) * a.ldr + n + k)) : 0.f);
                        store_out(o + k, y);
                    }
                }
            }
        }
        __syncwarp();
        cluster_sync();  // peers have read this CTA's sums
    }
    __syncwarp();
    ut_fence_before();
    __syncthreads();
    if (warp == 2) ut_free<S::TMEM>(tmem);
}

static PFN_cuTensorMapEncodeTiled_v12000 gm_encoder() {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> known{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 f = known.load(std::memory_order_acquire);
    if (f) return f;
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    known.store(f, std::memory_order_release);
    return f;
}

bool int8_map(CUtensorMap* m, const void* p, int K, int rows, long long ld, int box) {
    const PFN_cuTensorMapEncodeTiled_v12000 encode = gm_encoder();
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t size[2] = {128, (cuuint32_t)box}, es[2] = {1, 1};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, size, es,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool out_map(CUtensorMap* m, void* p, int type, int N, int T, long long ld, int tokens) {
    const PFN_cuTensorMapEncodeTiled_v12000 encode = gm_encoder();
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)T};
    const cuuint64_t strides[1] = {(cuuint64_t)(ld * type_size(type))};
    const cuuint32_t size[2] = {32, (cuuint32_t)tokens}, es[2] = {1, 1};
    return encode(m, type == SKB_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                     : type == SKB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  2, p, dims, strides, size, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TN, bool GLU, class TO>
static cudaError_t gemm_launch(const Int8Args& a, int split, bool early, cudaStream_t s) {
    using S = GemmShape<TN, GLU>;
    const cudaError_t e = prepare_kernel<int8_gemm_kernel<TN, GLU, TO>>(S::SMEM);
    if (e != cudaSuccess) return e;
    GemmMaps maps;
    if (!int8_map(&maps.x, a.in.x, a.in.K, a.in.T, a.in.ld, TN) || !int8_map(&maps.w[0], a.w[0], a.in.K, a.N, a.ldw[0], 128))
        return cudaErrorNotSupported;
    if (GLU) {
        if (!int8_map(&maps.w[1], a.w[1], a.in.K, a.N, a.ldw[1], 128)) return cudaErrorNotSupported;
    } else {
        maps.w[1] = maps.w[0];
    }
    constexpr int SMS = 148;
    const long long tiles = (long long)((a.N + 127) / 128) * ((a.in.T + TN - 1) / TN);
    if (tiles >= 1 << 30) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(split > 1 ? tiles * split : tiles < SMS ? tiles : SMS));
    cfg.blockDim = dim3(GM_THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = split;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, int8_gemm_kernel<TN, GLU, TO>, a, maps, split, early);
}

// How many clusters of `split` CTAs run at once on the current device.
template <int TN, bool GLU, class TO>
static int clusters_at_once(int split) {
    static std::atomic<int> known[64][GM_MAX_SPLIT + 1];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    const int k = known[dev][split].load(std::memory_order_relaxed);
    if (k > 0) return k - 1;
    using S = GemmShape<TN, GLU>;
    if (prepare_kernel<int8_gemm_kernel<TN, GLU, TO>>(S::SMEM) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split);
    cfg.blockDim = dim3(GM_THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = split;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, int8_gemm_kernel<TN, GLU, TO>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    known[dev][split].store(n + 1, std::memory_order_relaxed);
    return n;
}

// Which tiles: their width in tokens, how many CTAs split K, or pairs (width 0,
// int8_wide.cu).  Of those that run at once the least time by what was measured at 9 to
// 512 tokens, 1024 to 4096 channels and K of 1024 to 8192, in us: 0.22 + width / 1000 a
// block of K, half as much again with two weights; a split 0.5 and 0.025 a token to hand
// sums over, a token's finish 0.004 without.  Narrow tiles go in one turn alone; in several
// they are not measured.  Where nothing fits, tiles are as wide as they get and CTAs take
// them in turn, which is dear for few tokens: 5 to 100 of 1024 to 32816 channels 16 us with
// most columns empty, 128 13.1, where four go by four-byte products in 11.0.  The model: a
// turn of a pair 1 to begin with, then 0.39 a block or its finish, 4 (SwiGLU 5.8, with a
// residual 8), whichever is longer; of a single CTA 0.48 a block (0.52) or 4.3 (3.9, 10).
template <class TO, bool GLU>
static void gemm_choose(const Int8Args& a, int& width, int& split) {
    const long long cols = (a.N + 127) / 128;
    const int blocks = (a.in.K + 127) / 128, T = a.in.T;
    float best = 3e38f;
    auto look = [&](int tn, int at_once, int s) {
        if (s > blocks || cols * ((T + tn - 1) / tn) > at_once) return;
        const float tokens = (float)(T < tn ? T : tn);
        const float t = (float)((blocks + s - 1) / s) * (0.22f + 0.001f * tn) * (GLU ? 1.5f : 1.f) +
                        (s > 1 ? 0.5f + 0.025f * tokens * (GLU ? 2 : 1) : 0.004f * tokens);
        if (t < best) best = t, width = tn, split = s;
    };
    look(32, 148, 1), look(64, 148, 1), look(128, 148, 1);
    for (int s = 2; s <= GM_MAX_SPLIT && cols * s <= 148; s *= 2) {
        look(32, clusters_at_once<32, GLU, TO>(s), s);
        look(64, clusters_at_once<64, GLU, TO>(s), s);
        look(128, clusters_at_once<128, GLU, TO>(s), s);
    }
    if (best < 3e38f) return;
    split = 1, width = GLU ? 128 : 256;
    if (!int8_wide_serves(a)) return;
    auto turn = [&](float block, float finish) { return (float)blocks * block > finish ? (float)blocks * block : finish; };
    const long long singles = (cols * ((T + width - 1) / width) + 147) / 148;
    const long long pairs = ((a.N + (GLU ? 127 : 255)) / (GLU ? 128 : 256) * (long long)((T + 255) / 256) + 73) / 74;
    if (1.f + (float)pairs * turn(0.39f, GLU ? 5.8f : a.residual ? 8.f : 4.f) <
        (float)singles * turn(GLU ? 0.52f : 0.48f, GLU ? 3.9f : a.residual ? 10.f : 4.3f))
        width = 0;
}

template <class TO>
static cudaError_t gemm_typed(const Int8Args& a, bool glu, bool early, cudaStream_t s) {
    int width = 0, split = 1;
    if (glu) {
        gemm_choose<TO, true>(a, width, split);
        if (width == 0) return int8_wide_launch(a, true, early, s);
        if (width == 32) return gemm_launch<32, true, TO>(a, split, early, s);
        if (width == 64) return gemm_launch<64, true, TO>(a, split, early, s);
        return gemm_launch<128, true, TO>(a, split, early, s);
    }
    gemm_choose<TO, false>(a, width, split);
    if (width == 0) return int8_wide_launch(a, false, early, s);
    if (width == 32) return gemm_launch<32, false, TO>(a, split, early, s);
    if (width == 64) return gemm_launch<64, false, TO>(a, split, early, s);
    if (width == 128) return gemm_launch<128, false, TO>(a, split, early, s);
    return gemm_launch<256, false, TO>(a, 1, early, s);
}

// Rows as codes; early: see int8_gemv_launch.
cudaError_t int8_gemm_launch(const Int8Args& a, bool glu, bool early, cudaStream_t s) {
    return with_type(a.out_type, [&](auto to) { return gemm_typed<decltype(to)>(a, glu, early, s); });
}

}  // namespace skb
