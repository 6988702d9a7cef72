// fp16 tensor-core pieces of the cache operators: FP32 operands as pairs of
// fp16 tiles, the shared-memory and instruction descriptors of
// tcgen05.mma kind::f16, tensor-memory loads and stores, bounded waits.
//
// An FP32 row x is scaled by a power of two to a largest magnitude in
// [2^13, 2^14) and split into hi = fp16(x) and lo = fp16(x - hi): 22 bits,
// and an absolute floor 2^-38 of the row's largest.  A product of two such
// operands is hi.hi + hi.lo + lo.hi in FP32 (the dropped lo.lo is 2^-22
// relative): three fp16 products at twice the rate of TF32 in half its shared
// memory, where three TF32 products give the same bits.
//
// Tiles are [two halves of 64 columns][128 rows][128 bytes], each half in the
// 128-byte swizzle (16-byte chunk c of row r at c ^ (r & 7)).  The same bytes
// serve as a K-major operand whose rows are M or N (queries, keys) and as an
// MN-major one whose rows are K (values).
#pragma once

#include "cache_ops.cuh"

namespace skb {

constexpr uint32_t UT_HALF = 128 * 128;       // bytes of 64 columns
constexpr uint32_t UT_BYTES = 2 * UT_HALF;    // one fp16 tile
constexpr float UT_POISON_E = -200.f;         // exponent of a row of zeros

// ------------------------------------------------------------- descriptors
// Shared-memory operand, 128-byte swizzle.  K-major: 8-row groups 1024 bytes
// apart.  MN-major: 64-column halves `UT_HALF` apart (leading offset), 8-row
// groups along K 1024 bytes apart (stride offset).
// `off`: bytes added to the address, known when compiled.
__device__ __forceinline__ uint64_t ut_desc(uint32_t saddr, uint32_t off, bool mn_major) {
    const uint32_t lo = ((saddr >> 4) & 0x3FFFu) + (off >> 4) + ((mn_major ? (UT_HALF >> 4) : 1u) << 16);
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return (uint64_t)hi << 32 | lo;
}
// kind::f16, D FP32, A and B fp16, M = 128.
__host__ __device__ constexpr uint32_t ut_idesc(int n, bool b_mn_major) {
    return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void ut_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// The accumulation in tensor memory cuts towards zero (measured: about 1e-8 of
// the sum per step of 16 at full size, all of one sign), so the small
// products come first, where the sum is still 2^-11 of its size, and no sum
// runs on from tile to tile: that grew to 1.3e-5 over 8000 slots.

// D[128 x N] = A B^T over 128 columns: A in tensor memory (hi | lo, 64 columns
// each), which halves what the products read from shared memory; B as a hi | lo
// pair of [two halves of 64 columns][N rows] tiles (K-major).
template <int N>
__device__ __forceinline__ void ut_mma_qk(uint32_t d, uint32_t a_tmem, uint32_t b) {
    asm volatile("" : "+r"(a_tmem), "+r"(b));  // keeps 24 descriptors from being held across a caller's loop
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const uint32_t pa = a_tmem + (p == 1 ? 64 : 0);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            umma_f16_ts(d, pa + k * 8, ut_desc(b, (p == 0 ? 256 * N : 0) + (k >> 2) * (128 * N) + (k & 3) * 32, false),
                        ut_idesc(N, false), p > 0 || k > 0);
    }
}
// D[128 x 128] = P V: P in tensor memory, for each 16 keys 8 columns of hi,
// then 8 of lo; V as hi | lo tiles (MN-major).
__device__ __forceinline__ void ut_mma_pv(uint32_t d, uint32_t p_tmem, uint32_t v) {
    asm volatile("" : "+r"(p_tmem), "+r"(v));
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const uint32_t pa = p_tmem + (p == 1 ? 8 : 0);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            umma_f16_ts(d, pa + k * 16, ut_desc(v, (p == 0 ? UT_BYTES : 0) + k * 2048, true), ut_idesc(128, true), p > 0 || k > 0);
    }
}

// ---------------------------------------------------------- tensor memory
__device__ __forceinline__ void ut_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
          "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]),
          "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void ut_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}
__device__ __forceinline__ void ut_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void ut_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]),
        "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
        "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void ut_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ut_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ut_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ut_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <int COLUMNS>
__device__ __forceinline__ void ut_alloc(uint32_t* slot) {  // by one warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "n"(COLUMNS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLUMNS>
__device__ __forceinline__ void ut_free(uint32_t tmem) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLUMNS) : "memory");
}
// Row `row` of one fp16 tile of 128 rows into 64 columns of tensor memory, a
// lane its row.
__device__ __forceinline__ void ut_row_to_tmem(const unsigned char* tile, int row, uint32_t taddr) {
#pragma unroll
    for (int ch = 0; ch < 2; ++ch) {
        uint32_t w[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint4 y = *reinterpret_cast<const uint4*>(tile + ch * UT_HALF + row * 128 + ((j ^ (row & 7)) * 16));
            w[4 * j] = y.x;
            w[4 * j + 1] = y.y;
            w[4 * j + 2] = y.z;
            w[4 * j + 3] = y.w;
        }
        ut_st32(taddr + ch * 32, w);
    }
    ut_wait_st();
}

// ----------------------------------------------------------------- waits
__device__ __forceinline__ void ut_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Waits for phase `parity`, at most about 2 s and no longer than *abort stays
// 0; false (and *abort set) when it gave up.  Every wait of a kernel goes
// through here, so that one that runs out ends all the others.  A test first,
// which costs least when the phase is over (a try with a time to sleep took
// 230 cycles then); after a few of them tries that sleep up to 20 us in hardware,
// so that a waiting warp takes no issue slots.
__device__ __forceinline__ bool ut_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
    const uint32_t addr = smem_u32(bar);
    uint32_t done;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(addr), "r"(parity)
            : "memory");
        if (done) return true;
    }
    uint64_t t0 = 0;
    for (;;) {
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(addr), "r"(parity), "r"(20000u)
            : "memory");
        if (done) return true;
        const uint64_t now = globaltimer_ns();
        if (t0 == 0) t0 = now;
        if (*abort || now - t0 > SKB_WAIT_LIMIT_NS) {
            *abort = 1;
            return false;
        }
    }
}

// ------------------------------------------------------- splitting a row
// Pairs of FP32 in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
        " fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
// The same on pairs that stay 64-bit registers.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float2 unpack2(uint64_t a) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
    return d;
}
__device__ __forceinline__ uint64_t fma2p(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// hi = fp16 pair of x, lo = fp16 pair of what is left.
__device__ __forceinline__ void split2(float2 x, uint32_t& hi, uint32_t& lo) {
    asm("{\n .reg .b16 p, q, m;\n .reg .f32 u, v;\n"
        " cvt.rn.f16x2.f32 %0, %3, %2;\n mov.b32 {p, q}, %0;\n mov.b16 m, 0xBC00;\n"  // -1
        " fma.rn.f32.f16 u, p, m, %2;\n fma.rn.f32.f16 v, q, m, %3;\n cvt.rn.f16x2.f32 %1, v, u;\n}"
        : "=&r"(hi), "=r"(lo)
        : "f"(x.x), "f"(x.y));
}
// Largest of |a|, |b|, |c|; NaN if one of them is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Exponent floor(log2) of a row's largest magnitude as a whole number in
// [-100, 127]; UT_POISON_E for a row of zeros, NaN for one that holds
// something not finite.
__device__ __forceinline__ float top_exponent(float top) {
    const unsigned t = __float_as_uint(top);
    const float e = (float)max((int)(t >> 23) - 127, -100);
    return t >= 0x7f800000u ? __int_as_float(0x7fffffff) : (t == 0 ? UT_POISON_E : e);
}
// 2^e for whole e in [-126, 127].
__device__ __forceinline__ float pow2_whole(float e) { return __int_as_float(((int)e + 127) << 23); }
// The scale 2^(13 - e) of a row with exponent e; 0 for rows that become zeros
// (of zeros, or not finite).
__device__ __forceinline__ float row_scale(float e) { return e >= -100.f ? pow2_whole(13.f - e) : 0.f; }
// 8 bytes at row r, columns 4c .. 4c+3 of the tile pair at `tile` (hi, then lo
// UT_BYTES further).
__device__ __forceinline__ uint32_t ut_at(int r, int c) {
    return (uint32_t)(c >> 4) * UT_HALF + (uint32_t)r * 128u + ((((uint32_t)(c & 15) >> 1) ^ (uint32_t)(r & 7)) * 16u) +
           (uint32_t)(c & 1) * 8u;
}
__device__ __forceinline__ void put4(unsigned char* at, float4 x, float s) {
    uint2 hi, lo;
    const float2 s2 = make_float2(s, s);
    split2(mul2(make_float2(x.x, x.y), s2), hi.x, lo.x);
    split2(mul2(make_float2(x.z, x.w), s2), hi.y, lo.y);
    *reinterpret_cast<uint2*>(at) = hi;
    *reinterpret_cast<uint2*>(at + UT_BYTES) = lo;
}

// 4 NQ rows of a tile in the registers of a warp, on their way from the pool
// to a tile pair.  Lane 8 i + t holds, of rows i, 4 + i, ..., columns
// 8 t .. 8 t + 7 of either half: 32 bytes a load, and 16 bytes of hi or
// lo a store, whose four rows are whole 128-byte lines.
template <int NQ>
struct RowSet {
    float d[NQ][2][8];
    // `unit`: where this lane's row 4 q + i lies in the pool, or UT_NONE / UT_BAD: zeros
    // Read once, so first to leave L2: room for the tiles (512 tokens behind 8192
    // slots 113.3 us a call, 114.3 without; 16 ragged rows 87.0 and 86.7).
    __device__ __forceinline__ void load(int q, const float* pool, uint32_t unit, int lane) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* x = d[q][h];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = 0.f;
            asm volatile(
                "{\n .reg .pred p;\n setp.lt.u32 p, %8, 0xfffffffe;\n"
                " @p ld.global.L1::no_allocate.L2::evict_first.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%9];\n}"
                : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7])
                : "r"(unit), "l"(pool + (long long)unit * 128 + 64 * h + 8 * (lane & 7)));
        }
    }
    // Exponent of this lane's row 4 q + i (the same in its 8 lanes).
    __device__ __forceinline__ float exponent(int q, uint32_t unit) const {
        float m = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 8; k += 2) m = max3_abs(m, d[q][h][k], d[q][h][k + 1]);
        m = max3_abs(m, __shfl_xor_sync(FULL, m, 1), 0.f);
        m = max3_abs(m, __shfl_xor_sync(FULL, m, 2), 0.f);
        m = max3_abs(m, __shfl_xor_sync(FULL, m, 4), 0.f);
        return unit == UT_NONE ? UT_POISON_E : unit == UT_BAD ? __int_as_float(0x7fffffff) : top_exponent(m);
    }
    // Rows 4 q + i, scaled, into the tile at its row `row0` (a multiple of
    // 16).  A scale of 0 makes zeros of anything.
    __device__ __forceinline__ void put(int q, unsigned char* tile, int row0, float s, int lane) {
        const int i = lane >> 3, row = row0 + 4 * q + i;
        unsigned char* at = tile + row * 128 + (((lane & 7) ^ (row & 7)) * 16);
        const float2 s2 = make_float2(s, s);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint4 hi, lo;
            float* x = d[q][h];
            if (s == 0.f) {
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = 0.f;
            }
            split2(mul2(make_float2(x[0], x[1]), s2), hi.x, lo.x);
            split2(mul2(make_float2(x[2], x[3]), s2), hi.y, lo.y);
            split2(mul2(make_float2(x[4], x[5]), s2), hi.z, lo.z);
            split2(mul2(make_float2(x[6], x[7]), s2), hi.w, lo.w);
            *reinterpret_cast<uint4*>(at + h * UT_HALF) = hi;
            *reinterpret_cast<uint4*>(at + h * UT_HALF + UT_BYTES) = lo;
        }
    }
};

}  // namespace skb
