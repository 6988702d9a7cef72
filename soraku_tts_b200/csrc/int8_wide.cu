// Products of 8-bit codes for many tokens: pairs of CTAs on one tile
// (tcgen05.mma.cta_group::2 kind::i8), 256 weight rows x 256 tokens.
//
// One CTA alone reads 48 KB of operands into shared memory for every 2^25 products,
// and the tensor core reads them again: more than shared memory passes in the time of
// the products (measured: 57 % of the rate).  A pair halves the tokens' part: each
// CTA holds its own 128 weight rows and half of the tokens, 32 KB a stage.
//
// Warps of each CTA: 0 copies (into its own memory, on the first CTA's barriers), 1 of
// the first CTA issues the products for both, 4-19 finish one tile while the next
// is added up.  A thread of these holds a channel; its results go to shared memory,
// 32 channels x 16 tokens a warp, and out by TMA, which knows the output's edges.
// For SwiGLU a CTA's rows are 64 of the gate and the same 64 of up: the warps of a
// gate row and of its up row hand each other half of their tokens.
//
// From codes: 4096 tokens of 4096 to 4096 channels (BF16 out) 48 to 50 us in bursts of a few
// ms, 2.7 to 2.9 POPS, 61 % of the tensor pipe's cycles, 58 in a run of 20 ms and more (with
// all-zero operands 4.3 POPS: power).  6541 of 1024 to 4096 (FP32 out, 107 MB, which a fill
// writes in 15.5 us) 32 to 37 us: six turns of 3.1 us of products beside 4 us of results,
// which share shared memory and issue slots.  5003 of 2048 to 2 x 4096 64 to 75 us, 2.2 to
// 2.6 POPS.  Not faster: 8 epilogue
// warps in place of 16, their loop unrolled with an early hand-back, tensor memory read
// one step ahead.
#include <cudaTypedefs.h>

#include <cstddef>

#include "int8_ops.cuh"
#include "umma.cuh"

namespace skb {

constexpr int WD_THREADS = 640, WD_EPI_WARPS = 16;
constexpr int WD_CH = 16;  // tokens a warp takes at a time
constexpr int WD_STAGE = 32 * 1024, WD_A = 16 * 1024;
constexpr int WD_MAX_STAGES = 6;

struct WideMaps {
    CUtensorMap x, w[2], out;
};

template <bool GLU, class TO>
struct WideShape {
    static constexpr int TOKENS = GLU ? WD_CH / 2 : WD_CH;           // of one store
    static constexpr int OUT = 32 * TOKENS * (int)sizeof(TO);        // bytes of one store
    static constexpr int SWAP = GLU ? WD_CH / 2 * 32 * 4 : 0;        // sums for the other warp
    static constexpr int WARP = 2 * OUT + 2 * SWAP;
    static constexpr int STAGES = (224 * 1024 - WD_EPI_WARPS * WARP) / WD_STAGE;
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * WD_STAGE + WD_EPI_WARPS * WARP;
    static_assert(STAGES <= WD_MAX_STAGES && STAGES >= 4 && WARP % 512 == 0, "ring");
};

struct WideShared {
    uint64_t full[WD_MAX_STAGES], empty[WD_MAX_STAGES], acc_full[2], acc_free[2];
    uint32_t tmem;
    int abort;
    alignas(16) float sx[WD_EPI_WARPS][WD_CH];  // scales of a warp's tokens, read four at a time
};
static_assert(offsetof(WideShared, sx) % 16 == 0, "16-byte reads");

// Into this CTA's memory, counted by a barrier of this CTA or its peer.
__device__ __forceinline__ void wd_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void wd_store(const CUtensorMap* map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(src)
                 : "memory");
}
// D S32, A and B S8, both K-major, M = 256 (128 rows of each CTA), N = 256.
constexpr uint32_t WD_IDESC = (2u << 4) | (1u << 7) | (1u << 10) | (32u << 17) | (16u << 24);
__device__ __forceinline__ void wd_mma(uint32_t d, uint64_t a, uint64_t b, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(WD_IDESC), "r"((uint32_t)acc)
        : "memory");
}
// On the barrier at this place in both CTAs, once the products issued so far are done.
__device__ __forceinline__ void wd_commit(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// What it hands over is tensor memory, behind tcgen05's own fence: a release to the
// cluster would wait for all stores on their way (1900 cycles a tile).
__device__ __forceinline__ void wd_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <bool GLU, class TO>
__global__ void __launch_bounds__(WD_THREADS, 1) int8_wide_kernel(const Int8Args a, const __grid_constant__ WideMaps maps, bool early) {
    using S = WideShape<GLU, TO>;
    extern __shared__ unsigned char wd_raw[];
    __shared__ WideShared sm;
    unsigned char* base = wd_raw + ((1024u - (smem_u32(wd_raw) & 1023u)) & 1023u);
    const uint32_t ring = smem_u32(base);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x & 1;
    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) mbar_init(&sm.full[i], 1), mbar_init(&sm.empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&sm.acc_full[i], 1), mbar_init(&sm.acc_free[i], 2 * WD_EPI_WARPS);
        sm.abort = 0;
        mbar_fence_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.x)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.w[0])) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.out)) : "memory");
        if (GLU) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.w[1])) : "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "n"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    ut_fence_before();
    __syncthreads();
    cluster_sync();  // the peer's barriers and tensor memory are there
    ut_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* abort = &sm.abort;

    constexpr int COLS = GLU ? 128 : 256;  // output columns of a tile
    const int tiles_n = (a.N + COLS - 1) / COLS, tiles_t = (a.in.T + 255) / 256;
    const int tiles = tiles_n * tiles_t;  // the launch has seen that they are fewer than 2^30
    const int blocks = (a.in.K + 127) / 128;
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const uint32_t full0 = cluster_addr(smem_u32(&sm.full[0]), 0);  // the first CTA's
    auto load_w = [&](int n0, int kb, int s) {
        const uint32_t at = ring + s * WD_STAGE;
        if (GLU) {
            wd_load(at, &maps.w[0], kb * 128, n0, full0 + s * 8);
            wd_load(at + WD_A / 2, &maps.w[1], kb * 128, n0, full0 + s * 8);
        } else {
            wd_load(at, &maps.w[0], kb * 128, n0, full0 + s * 8);
        }
    };
    // blocks whose weights are asked for before the wait
    int ahead = 0;
    if (early && tid == 0 && first < tiles)
        for (; ahead < S::STAGES && ahead < blocks; ++ahead) {
            if (rank == 0) mbar_expect_tx(&sm.full[ahead], 2 * WD_STAGE);
            load_w(first % tiles_n * COLS + rank * (COLS / 2), ahead, ahead);
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
                const int n0 = tile % tiles_n * COLS + rank * (COLS / 2), t0 = tile / tiles_n * 256 + rank * 128;
                for (int kb = 0; kb < blocks; ++kb) {
                    if (asked >= S::STAGES && !ut_wait(&sm.empty[s], phase, abort)) {
                        go = false;
                        break;
                    }
                    if (asked >= ahead) {
                        if (rank == 0) mbar_expect_tx(&sm.full[s], 2 * WD_STAGE);
                        load_w(n0, kb, s);
                    }
                    wd_load(ring + s * WD_STAGE + WD_A, &maps.x, kb * 128, t0, full0 + s * 8);
                    asked = min(asked + 1, S::STAGES);
                    if (++s == S::STAGES) s = 0, phase ^= 1;
                }
            }
            // no copy may land after the CTAs have gone: the products wait for each of
            // them; where those gave up, wait here, from the oldest on
            if (*abort && rank == 0)
                for (int i = 0; i < asked; ++i) {
                    const bool wrapped = asked == S::STAGES && s + i >= S::STAGES;
                    const int at = asked < S::STAGES ? i : (wrapped ? s + i - S::STAGES : s + i);
                    mbar_wait(&sm.full[at], asked < S::STAGES ? 0u : (wrapped ? phase ^ 1 : phase), nullptr);
                }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int s = 0, i = 0;
            uint32_t phase = 0;
            bool go = true;
            for (int tile = first; tile < tiles && go; tile += step, ++i) {
                const int b = i & 1;
                if (i >= 2 && !ut_wait(&sm.acc_free[b], (uint32_t)((i >> 1) - 1) & 1u, abort)) break;
                ut_fence_after();
                for (int kb = 0; kb < blocks; ++kb) {
                    if (!ut_wait(&sm.full[s], phase, abort)) {
                        go = false;
                        break;
                    }
                    ut_fence_after();
                    const uint32_t at = ring + s * WD_STAGE;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        wd_mma(tmem + b * 256, ut_desc(at, k * 32, false), ut_desc(at + WD_A, k * 32, false), kb > 0 || k > 0);
                    wd_commit(&sm.empty[s]);
                    if (++s == S::STAGES) s = 0, phase ^= 1;
                }
                if (go) wd_commit(&sm.acc_full[b]);
            }
            // what was issued ends before tensor memory is given back
            if (*abort) {
                wd_commit(&sm.acc_full[0]);
                for (int n = 0; n < 2; ++n) mbar_wait_limit(&sm.acc_full[0], n, nullptr, 1000000ull);
            }
        }
    } else if (warp >= 4) {
        const int e = warp - 4, q = e & 3, part = e >> 2;  // lanes 32 q, tokens 64 part of the tile
        const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16) + part * 64;
        unsigned char* mine = base + S::STAGES * WD_STAGE + e * S::WARP;
        TO* stage = reinterpret_cast<TO*>(mine);
        int* give = reinterpret_cast<int*>(mine + 2 * S::OUT);
        // SwiGLU: the warp that has this one's gate or up rows
        const int* take = reinterpret_cast<const int*>(base + S::STAGES * WD_STAGE + (e ^ 2) * S::WARP + 2 * S::OUT);
        const bool is_up = GLU && q >= 2;
        float* sx = sm.sx[e];
        const uint32_t free0 = cluster_addr(smem_u32(&sm.acc_free[0]), 0);
        int i = 0, turn = 0;
        for (int tile = first; tile < tiles; tile += step, ++i) {
            const int n0 = tile % tiles_n * COLS + rank * (COLS / 2) + 32 * (GLU ? q & 1 : q), n = n0 + lane;
            const int t0 = tile / tiles_n * 256 + part * 64;
            const int b = i & 1;
            const bool in = n < a.N;
            float s0 = in ? __ldcg(a.ws[0] + n) : 0.f, s1 = GLU && in ? __ldcg(a.ws[1] + n) : 0.f;
            const float bias = !GLU && a.bias != nullptr && in ? __ldcg(a.bias + n) : 0.f;
            const TO* res = GLU ? nullptr : static_cast<const TO*>(a.residual);
            auto scale_of = [&](int t) { return lane < WD_CH && t + lane < a.in.T ? __ldcg(a.in.scale + t + lane) : 0.f; };
            float next = scale_of(t0);
            TO r_next[GLU ? 1 : WD_CH];  // as it came: a conversion would wait for it
            auto residual_of = [&](int t) {
                const TO* p = res + (long long)t * a.ldr + n;
#pragma unroll
                for (int j = 0; j < WD_CH; ++j, p += a.ldr) r_next[GLU ? 0 : j] = in && t + j < a.in.T ? read(p) : from_float<TO>(0.f);
            };
            if (!GLU && res != nullptr) residual_of(t0);
            // a wait that ran out shows as NaN
            if (!ut_wait(&sm.acc_full[b], (uint32_t)(i >> 1) & 1u, abort)) s0 = __int_as_float(0x7fffffff);
            __syncwarp();
            ut_fence_after();
            const int chunks = min(64 / WD_CH, (a.in.T - t0 + WD_CH - 1) / WD_CH);
#pragma unroll 1
            for (int c = 0; c < chunks; ++c, ++turn) {
                const int t = t0 + WD_CH * c;
                uint32_t v[WD_CH];
                ut_ld16(lanes + b * 256 + WD_CH * c, v);
                if (lane < WD_CH) sx[lane] = next;
                next = scale_of(t + WD_CH);
                TO* out = stage + (turn & 1) * (S::OUT / (int)sizeof(TO));
                // the store that read this buffer two turns ago has read it
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                if constexpr (GLU) {
                    constexpr int H = WD_CH / 2;
                    int* to = give + (turn & 1) * (S::SWAP / 4);
                    const int* from = take + (turn & 1) * (S::SWAP / 4);
                    ut_wait_ld();
#pragma unroll
                    for (int j = 0; j < H; ++j) to[j * 32 + lane] = (int)v[is_up ? j : H + j];
                    asm volatile("bar.sync %0, 64;" ::"r"(1 + part * 2 + (q & 1)) : "memory");
#pragma unroll
                    for (int j0 = 0; j0 < H; j0 += 4) {
                        const float4 s4 = *reinterpret_cast<const float4*>(sx + (is_up ? H : 0) + j0);
                        const float sj[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int j = j0 + k, own = (int)v[is_up ? H + j : j], other = from[j * 32 + lane];
                            store_out(out + j * 32 + lane, finish_glu(is_up ? other : own, is_up ? own : other, sj[k], s0, s1));
                        }
                    }
                } else {
                    float r[WD_CH];
                    if (res != nullptr) {
#pragma unroll
                        for (int j = 0; j < WD_CH; ++j) r[j] = to_float(r_next[j]);
                        if (c + 1 < chunks) residual_of(t + WD_CH);  // on their way while these are used
                    }
                    ut_wait_ld();
                    __syncwarp();
                    auto put = [&](bool add) {
#pragma unroll
                        for (int j0 = 0; j0 < WD_CH; j0 += 4) {
                            const float4 s4 = *reinterpret_cast<const float4*>(sx + j0);
                            const float sj[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                float y = finish((int)v[j0 + k], sj[k], s0, bias);
                                if (add) y += r[j0 + k];
                                store_out(out + (j0 + k) * 32 + lane, y);
                            }
                        }
                    };
                    if (res != nullptr) put(true);
                    else put(false);
                }
                if (c == chunks - 1) {  // the sums are out of tensor memory
                    ut_fence_before();
                    __syncwarp();
                    if (lane == 0) wd_arrive(free0 + b * 8);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    const int y = t + (is_up ? S::TOKENS : 0);
                    if (n0 < a.N && y < a.in.T) wd_store(&maps.out, n0, y, smem_u32(out));
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
            if (chunks <= 0) {
                ut_fence_before();
                __syncwarp();
                if (lane == 0) wd_arrive(free0 + b * 8);
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    ut_fence_before();
    cluster_sync();  // neither CTA goes while the other's copies, products or arrivals reach it
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}

// Where the output's rows are what TMA can write: on 16 bytes.  Against single CTAs
// (int8_gemm.cu), us: 5000 tokens to 4096 channels of 64 20.1 and 22.7, of 2048 55 and 57;
// 1500 to 2048 of 1024 11.1 and 10.2.  A SwiGLU's hand-over pays where its products
// last: 5000 to 4096 of 1024 64 and 57, of 2048 81 and 94.
bool int8_wide_serves(const Int8Args& a) { return aligned16(a.out) && a.ldo * type_size(a.out_type) % 16 == 0; }

template <bool GLU, class TO>
static cudaError_t wide_typed(const Int8Args& a, bool early, cudaStream_t s) {
    using S = WideShape<GLU, TO>;
    const cudaError_t e = prepare_kernel<int8_wide_kernel<GLU, TO>>(S::SMEM);
    if (e != cudaSuccess) return e;
    WideMaps maps;
    const int rows = GLU ? 64 : 128;
    if (!int8_map(&maps.x, a.in.x, a.in.K, a.in.T, a.in.ld, 128) || !int8_map(&maps.w[0], a.w[0], a.in.K, a.N, a.ldw[0], rows) ||
        !int8_map(&maps.w[1], a.w[GLU], a.in.K, a.N, a.ldw[GLU], rows) ||
        !out_map(&maps.out, a.out, a.out_type, a.N, a.in.T, a.ldo, S::TOKENS))
        return cudaErrorNotSupported;
    const long long tiles = (long long)((a.N + (GLU ? 127 : 255)) / (GLU ? 128 : 256)) * ((a.in.T + 255) / 256);
    if (tiles >= 1 << 30) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)(tiles < 74 ? tiles : 74));
    cfg.blockDim = dim3(WD_THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 2;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, int8_wide_kernel<GLU, TO>, a, maps, early);
}

// Rows as codes; early: see int8_gemv_launch.
cudaError_t int8_wide_launch(const Int8Args& a, bool glu, bool early, cudaStream_t s) {
    return with_type(a.out_type, [&](auto to) {
        return glu ? wide_typed<true, decltype(to)>(a, early, s) : wide_typed<false, decltype(to)>(a, early, s);
    });
}

}  // namespace skb
