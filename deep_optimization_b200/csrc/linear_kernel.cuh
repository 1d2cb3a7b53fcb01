// Matrix product with bias, activation and residual in its epilogue, sm_100a: the tensor-core kernel.
//
//     C[i, j] = f( sum_k A[i, k] B[j, k] + bias[j] ) + r[i, j]        and, where asked,  f'( ... )
//
// A and B are bf16 or fp16 (the same type), the sum is fp32.  Each operand is K-major (the reduction
// index contiguous: x and the weight of a linear layer's forward pass) or MN-major (the reduction
// index is the row: the operands of dx = dz W and dW = dz^T x as they lie in memory), so that one
// kernel serves the forward pass and both gradients and nothing is transposed.
//
// CG = 2: a cluster of two CTAs on the two SMs of a TPC computes 256 x 256 tiles with
// tcgen05.mma.cta_group::2 (each CTA stages its own 128 rows of A and its own half of B, and keeps the
// accumulators of its own rows in its own tensor memory).  CG = 1: one CTA per 128 x BN tile, for
// problems with too few rows or columns to fill the GPU with pairs.
// Roles of a CTA's warps:
//   warp 0      TMA producer: 64 k of both operands per stage, as rows of 128 bytes with the 128-byte
//               swizzle, completion counted on the leader's barrier (no multicast);
//   warp 1      MMA issuer (the leader's): four tcgen05.mma of K = 16 per stage, fp32 accumulators in
//               tensor memory, two of them, so that the next tile's MMAs overlap this tile's epilogue;
//   warps 2..   epilogue (eight, four for 64 columns): tcgen05.ld a 32 x 64 piece, bias, activation and its derivative, residual,
//               one rounding, a swizzled staging buffer, a bulk tensor store of full 128-byte rows.
//               The residual comes in through the same staging buffer by bulk tensor load, asked for
//               a tile ahead.  Outputs or residuals whose rows are not multiples of 16 bytes go through
//               the staging buffer too and are moved by ordinary two-byte accesses.
// A split of the reduction into slices (dW, whose reduction is the batch) writes fp32 partial tiles,
// one plane per slice, that a second kernel adds in slice order: the result does not depend on timing.
// Every wait is bounded; on a timeout the kernel records a reason, tells its peer, and leaves.
// Bound: 16-bit tensor throughput, 2 M N K operations: 1361 to 1571 TFLOP/s without an activation (cuBLAS on
// the same box 1258 to 1474), 1107 to 1462 with GELU and its derivative written as well.
#pragma once

#include <cuda.h>

#include "act_common.cuh"

namespace act {
namespace linear {

constexpr int BM = 128;                         // rows of A per CTA
constexpr int BK = 64;                          // reduction per stage: 128 bytes of a 16-bit type
constexpr int UMMA_K = 16;
constexpr int CHUNK = BK * 128;                 // MN-major: 64 columns x BK rows
constexpr int PIECE = 32 * 128;                 // staging buffer: 32 rows of 128 bytes
constexpr int TMEM_COLS = 512;
constexpr uint32_t SPIN_LIMIT = 1u << 24;

template <int CG, int BN> struct Cfg {
    static constexpr int BNC = BN / CG;                          // rows of B per CTA
    static constexpr int A_STAGE = BM * 128, B_STAGE = BNC * 128;
    // a warp drains 32 rows of a tile's left or right half, or of all 64 columns
    static constexpr int EPI_WARPS = BN == 64 ? 4 : 8, THREADS = 64 + EPI_WARPS * 32;
    // what two 4 KB staging buffers per epilogue warp leave of an SM's 227 KB
    static constexpr int STAGES = BNC == 128 ? 5 : 8;
    static constexpr int TILE_M = BM * CG;
};

template <int CG, int BN> struct __align__(1024) Smem {
    uint8_t a[Cfg<CG, BN>::STAGES][Cfg<CG, BN>::A_STAGE];
    uint8_t b[Cfg<CG, BN>::STAGES][Cfg<CG, BN>::B_STAGE];
    uint8_t stage[Cfg<CG, BN>::EPI_WARPS][2][PIECE];          // 128-byte rows, 16-byte pieces xor-swizzled by row & 7
    float bias[Cfg<CG, BN>::EPI_WARPS][64];       // of the piece a warp works on
    uint64_t full[Cfg<CG, BN>::STAGES], empty[Cfg<CG, BN>::STAGES], acc_full[2], acc_empty[2], res[Cfg<CG, BN>::EPI_WARPS][2];
    uint32_t tmem_base;
    volatile uint32_t abort;
};
static_assert(sizeof(Smem<2, 256>) <= 227 * 1024 && sizeof(Smem<1, 128>) <= 227 * 1024 && sizeof(Smem<1, 64>) <= 227 * 1024,
              "shared memory of the linear kernel exceeds one SM");

struct Params {
    int M, N, K;                                 // C is M x N
    int a_mn, b_mn;                              // operand is MN-major
    int slices;                                  // of the reduction; fp32 partial planes when out_f32
    int dtype;                                   // of A, B, the residual and 16-bit outputs
    int out_f32, tma_out, has_res;
    const void* bias; int bias_dtype;            // NULL or [N]
    const void* res; int64_t ld_res;
    void* y; int64_t ld_y;
    void* d; int64_t ld_d;
};

static __device__ unsigned int g_linear_error = 0;   // last abort reason of this file's kernels (0 = none)

// ---------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r;
}
// address of the same shared-memory location in CTA `rank` of this cluster
__device__ __forceinline__ uint32_t map_to_cta(uint32_t smem_addr, uint32_t rank) {
    uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank)); return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" :: "r"(cluster_addr), "r"(v) : "memory");
}
template <int CG> __device__ __forceinline__ void sync_all() {
    if (CG == 2) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
}
__device__ __forceinline__ void fence_barrier_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// operand load; the bytes are counted on the leader's barrier (`bar`: its cluster address)
// (`dst`: its shared-memory address)
template <int CG> __device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    if (CG == 2)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     :: "r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     :: "r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" :: "l"(map) : "memory"); }
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
                 :: "l"(map), "r"(smem_u32(src)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                 :: "l"(map), "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void tma_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int KEEP> __device__ __forceinline__ void tma_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" :: "n"(KEEP) : "memory"); }
template <int CG> __device__ __forceinline__ void tmem_alloc(uint32_t* dst_smem) {
    if (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(dst_smem)), "n"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(dst_smem)), "n"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int CG> __device__ __forceinline__ void tmem_dealloc(uint32_t taddr) {
    if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(taddr), "n"(TMEM_COLS) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(taddr), "n"(TMEM_COLS) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <int CG> __device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives, once the MMAs issued so far are done, on the barrier at this offset (in both CTAs of a pair)
template <int CG> __device__ __forceinline__ void umma_commit(uint32_t bar) {
    if (CG == 2) {
        const uint16_t both = 3;
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" :: "r"(bar), "h"(both) : "memory");
    } else {
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
    }
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// A wait that runs out records why and raises this CTA's abort flag and its peer's.  Every lane of the
// warp waits, so that the loops around it stay uniform over the warp (one lane's wait and a broadcast of
// its outcome took 130 cycles more per stage).
template <int CG, typename S>
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, S* s, uint32_t code, uint32_t peer_abort) {
    bool ok = mbar_try_wait(bar, parity);
    for (uint32_t i = 0; !ok && i < SPIN_LIMIT && !s->abort; ++i) ok = mbar_try_wait(bar, parity);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok && !s->abort && (threadIdx.x & 31) == 0) {
        s->abort = 1;
        if (CG == 2) st_cluster_u32(peer_abort, 1u);
        atomicExch(&g_linear_error, code);
    }
    return ok;
}
// warp-wide: lane 0 polls with a short sleep in between, everybody learns the outcome
template <int CG, typename S>
__device__ __forceinline__ bool wait_bar_warp(uint64_t* bar, uint32_t parity, S* s, uint32_t code, uint32_t peer_abort) {
    uint32_t ok = 1;
    if ((threadIdx.x & 31) == 0) {
        ok = 0;
        for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
            if (mbar_try_wait(smem_u32(bar), parity)) { ok = 1; break; }
            if (s->abort) break;
            __nanosleep(32);
        }
        if (!ok && !s->abort) { s->abort = 1; if (CG == 2) st_cluster_u32(peer_abort, 1u); atomicExch(&g_linear_error, code); }
    }
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// Shared-memory descriptor of an operand tile with the 128-byte swizzle.  K-major: rows of the M or N
// index, eight-row groups 1024 bytes apart, the leading offset unused.  MN-major: rows of the
// reduction index, eight-row groups 1024 bytes apart, chunks of 64 columns CHUNK bytes apart.
__device__ __forceinline__ uint64_t make_desc(uint32_t tile, bool mn_major) {
    uint64_t d = (uint64_t)((tile & 0x3FFFF) >> 4);
    d |= (mn_major ? (uint64_t)(CHUNK >> 4) : (uint64_t)1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;                          // descriptor version
    d |= (uint64_t)2 << 61;                          // 128-byte swizzle
    return d;
}

// ---------------------------------------------------------------- activations
__device__ __forceinline__ float ex2_approx(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp_approx(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ f32x2 ex2_approx2(f32x2 v) {
    uint32_t a, b;
    unpack2u(v, a, b);
    return pack2(ex2_approx(__uint_as_float(a)), ex2_approx(__uint_as_float(b)));
}
__device__ __forceinline__ f32x2 rcp_approx2(f32x2 v) {
    uint32_t a, b;
    unpack2u(v, a, b);
    return pack2(rcp_approx(__uint_as_float(a)), rcp_approx(__uint_as_float(b)));
}
__device__ __forceinline__ f32x2 both(float v) { return pack2(v, v); }

// f(z) and f'(z) of two values, on packed fp32 pairs: as single operations the GELU with its derivative
// took more issue slots per tile than K = 768 of MMAs last (bf16 50432 x 768 x 2304: 192 us, 171 on pairs; 161 in all with what follows below).
// The exponential and reciprocal instructions are within 2^-22, which a 16-bit result does not show.
//
// GELU in its tanh form is z times the logistic function s of 2u, u = k (z + c z^3).  z^2 is held to
// 256 in the polynomials: beyond |z| = 16 s is 0 or 1 to the last bit whatever they say, and 0 times an
// overflow would be NaN.
// The exact GELU's erfc(|z| / sqrt 2) is Hastings' approximation, Abramowitz and Stegun 7.1.26 (error
// at most 1.5e-7): a polynomial in 1 / (1 + p x) times exp(-x^2), the exponential f' needs anyway.
template <int KIND, bool DERIV>
__device__ __forceinline__ void activate2(f32x2 z, f32x2& y, f32x2& d) {
    if (KIND == ACT_KIND_NONE) { y = z; return; }
    if (KIND == ACT_KIND_RELU) {
        uint32_t a, b;
        unpack2u(z, a, b);
        y = pack2(fmax_nan(__uint_as_float(a), 0.0f), fmax_nan(__uint_as_float(b), 0.0f));
        return;
    }
    const f32x2 one = both(1.0f), minus = both(-1.0f);
    if (KIND == ACT_KIND_SILU) {
        const f32x2 s = rcp_approx2(add2_rn(one, ex2_approx2(mul2_rn(z, both(-1.4426950408889634f)))));
        y = mul2_rn(z, s);
        if (DERIV) d = fma2_rn(y, fma2_rn(s, minus, one), s);
    }
    if (KIND == ACT_KIND_GELU) {
        constexpr float k = 0.7978845608028654f, c = 0.044715f;          // sqrt(2 / pi)
        constexpr float p = -2.0f * k * 1.4426950408889634f, q = p * c;  // exp(-2u) = 2^(z (p + q z^2))
        uint32_t a, b;
        unpack2u(mul2_rn(z, z), a, b);
        const f32x2 z2 = pack2(fmin_nan(__uint_as_float(a), 256.0f), fmin_nan(__uint_as_float(b), 256.0f));
        const f32x2 s = rcp_approx2(add2_rn(one, ex2_approx2(mul2_rn(z, fma2_rn(z2, both(q), both(p))))));
        y = mul2_rn(z, s);
        if (DERIV)
            d = fma2_rn(mul2_rn(y, fma2_rn(s, minus, one)), fma2_rn(z2, both(6.0f * k * c), both(2.0f * k)), s);
    }
    if (KIND == ACT_KIND_GELU_ERF) {
        uint32_t a, b;
        unpack2u(z, a, b);
        const f32x2 size = pack2u(a & 0x7FFFFFFFu, b & 0x7FFFFFFFu);
        const f32x2 t = rcp_approx2(fma2_rn(size, both(0.3275911f * 0.7071067811865476f), one));
        // half of erfc's polynomial
        f32x2 h = fma2_rn(t, both(0.5f * 1.061405429f), both(0.5f * -1.453152027f));
        h = fma2_rn(h, t, both(0.5f * 1.421413741f));
        h = fma2_rn(h, t, both(0.5f * -0.284496736f));
        h = fma2_rn(h, t, both(0.5f * 0.254829592f));
        const f32x2 e = ex2_approx2(mul2_rn(mul2_rn(z, both(-0.7213475204444817f)), z));   // exp(-z^2 / 2)
        h = mul2_rn(mul2_rn(h, t), e);                                   // Phi(-|z|)
        uint32_t h0, h1, u0, u1;
        unpack2u(h, h0, h1);
        unpack2u(fma2_rn(h, minus, one), u0, u1);
        const f32x2 cdf = pack2u(__uint_as_float(a) >= 0.0f ? u0 : h0, __uint_as_float(b) >= 0.0f ? u1 : h1);
        y = mul2_rn(z, cdf);
        if (DERIV) d = fma2_rn(mul2_rn(z, e), both(0.3989422804014327f), cdf);
    }
}
template <int KIND, bool DERIV>
__device__ __forceinline__ void activate(float z, float& y, float& d) {
    f32x2 y2 = 0, d2 = 0;
    activate2<KIND, DERIV>(both(z), y2, d2);
    uint32_t a, b;
    unpack2u(y2, a, b);
    y = __uint_as_float(a);
    if (DERIV) { unpack2u(d2, a, b); d = __uint_as_float(a); }
}

__device__ __forceinline__ float widen16(uint32_t h, int dtype) {
    return dtype == ACT_DTYPE_F16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16);
}
__device__ __forceinline__ uint32_t round_pair(float a, float b, int dtype) {
    if (dtype == ACT_DTYPE_F16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// the two halves of a 16-bit pair in fp32, and two fp32 rounded to such a pair
template <int DT> __device__ __forceinline__ f32x2 widen_pair(uint32_t h) { return pack2(widen_lo<DT>(h), widen_hi<DT>(h)); }
template <int DT> __device__ __forceinline__ uint32_t narrow_pair(f32x2 v) {
    uint32_t a, b;
    unpack2u(v, a, b);
    return round_pair(__uint_as_float(a), __uint_as_float(b), DT);
}
__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
    if (dtype == ACT_DTYPE_F32) return static_cast<const float*>(p)[i];
    return widen16(static_cast<const unsigned short*>(p)[i], dtype);
}

// A 32 x 64 piece between its staging buffer and a tensor whose rows are not multiples of 16 bytes:
// lane l moves columns l and l + 32 of each row.
__device__ __forceinline__ void piece_out(const uint8_t* buf, unsigned short* dst, int64_t ld, int rows, int cols, int lane) {
    for (int r = 0; r < rows; ++r) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int c = lane + 32 * half;
            const int at = r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2;
            if (c < cols) dst[(int64_t)r * ld + c] = *reinterpret_cast<const unsigned short*>(buf + at);
        }
    }
}
__device__ __forceinline__ void piece_in(uint8_t* buf, const unsigned short* src, int64_t ld, int rows, int cols, int lane) {
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int c = lane + 32 * half;
            const int at = r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2;
            if (c < cols) *reinterpret_cast<unsigned short*>(buf + at) = src[(int64_t)r * ld + c];
        }
    }
}

// ------------------------------------------------------------------ the kernel
// Work item w = (tile, slice), w = (mt * n_tiles + nt) * slices + slice, dealt out round-robin to the
// clusters: those that run together share rows of A and read all of B out of L2.
template <int CG, int BN, int DT, int KIND, bool DERIV>
__global__ void __launch_bounds__(Cfg<CG, BN>::THREADS, 1)
linear_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
              const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_d,
              const __grid_constant__ CUtensorMap map_r, const __grid_constant__ Params p)
{
    using C = Cfg<CG, BN>;
    using S = Smem<CG, BN>;
    constexpr int EPI_WARPS = C::EPI_WARPS;
    extern __shared__ __align__(1024) uint8_t smem_raw_linear[];
    S* s = reinterpret_cast<S*>(smem_raw_linear);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // warp: uniform, and known to be
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;      // 0 = leader
    const int m_tiles = (p.M + C::TILE_M - 1) / C::TILE_M, n_tiles = (p.N + BN - 1) / BN;
    const int n_work = m_tiles * n_tiles * p.slices;
    const int k_blocks = (p.K + BK - 1) / BK;
    const int first = (int)blockIdx.x / CG, stride = (int)gridDim.x / CG;
    const uint32_t peer_abort = CG == 2 ? map_to_cta(smem_u32((const void*)&s->abort), rank ^ 1u) : 0u;

    if (smem_u32(s) & 1023u) {                                    // the swizzled tiles need this alignment
        if (threadIdx.x == 0) atomicExch(&g_linear_error, 5u);
        return;                                                   // uniform over the grid: nobody waits for anybody
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(&s->full[i], 1); mbar_init(&s->empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&s->acc_full[i], 1); mbar_init(&s->acc_empty[i], CG * EPI_WARPS); }
        for (int i = 0; i < EPI_WARPS; ++i) { mbar_init(&s->res[i][0], 1); mbar_init(&s->res[i][1], 1); }
        s->abort = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_map(&map_a);
        prefetch_map(&map_b);
        if (p.out_f32 || p.tma_out) prefetch_map(&map_y);
    }
    if (warp == 1) tmem_alloc<CG>(&s->tmem_base);                 // the same warp of both CTAs
    tc_fence_before();
    sync_all<CG>();                                               // barriers of both CTAs exist from here on
    tc_fence_after();
    const uint32_t tmem_base = s->tmem_base;
    grid_dependency_wait();                                       // from here on global memory is touched
    grid_launch_dependents();

    // blocks [lo, hi) of the reduction belong to slice sl
    auto slice_range = [&](int sl, int& lo, int& hi) {
        const int per = k_blocks / p.slices, extra = k_blocks % p.slices;
        lo = sl * per + (sl < extra ? sl : extra);
        hi = lo + per + (sl < extra ? 1 : 0);
    };

    // The producer's and the issuer's loops run on a whole warp, uniform over it, and elect.sync picks
    // the lane that issues the loads, MMAs and commits: these take their operands from uniform
    // registers.  Under any other predicate (`lane == 0`) an MMA cost the issuing warp 68 cycles, so 21.
    // What a stage costs that warp all the same, a wait (95), four MMAs (85) and the commit (130), is
    // more than the MMAs of a 128 x 64 or 128 x 128 tile last: about 380 cycles per 64 of the reduction
    // bound those shapes; the pair's 256 x 256 tile, 512 cycles of MMAs, hides it.  A second producer
    // warp, or a look at the next stage's barrier ahead of the MMAs, gained nothing.
    const uint32_t full0 = smem_u32(&s->full[0]), empty0 = smem_u32(&s->empty[0]);
    const uint32_t a0 = smem_u32(&s->a[0][0]), b0 = smem_u32(&s->b[0][0]);
    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        const uint32_t lead_full0 = CG == 2 ? map_to_cta(full0, 0) : full0;
        for (int w = first; ok && w < n_work; w += stride) {
            const int tile = w / p.slices, m0 = (tile / n_tiles) * C::TILE_M + (int)rank * BM;
            const int n0 = (tile % n_tiles) * BN + (int)rank * C::BNC;
            int lo, hi;
            slice_range(w % p.slices, lo, hi);
            for (int kb = lo; kb < hi; ++kb) {
                if (!(ok = wait_bar<CG>(empty0 + 8 * stage, phase ^ 1, s, 1, peer_abort))) break;
                if (elect_one()) {
                    // the leader's barrier counts the bytes of both CTAs; parts out of range arrive as zeros
                    if (rank == 0) mbar_expect_tx(full0 + 8 * stage, CG * (C::A_STAGE + C::B_STAGE));
                    const uint32_t bar = lead_full0 + 8 * stage, at = a0 + stage * C::A_STAGE, bt = b0 + stage * C::B_STAGE;
                    if (p.a_mn) {
#pragma unroll
                        for (int c = 0; c < BM / 64; ++c) tma_load<CG>(at + c * CHUNK, &map_a, bar, m0 + c * 64, kb * BK);
                    } else {
                        tma_load<CG>(at, &map_a, bar, kb * BK, m0);
                    }
                    if (p.b_mn) {
#pragma unroll
                        for (int c = 0; c < C::BNC / 64; ++c) tma_load<CG>(bt + c * CHUNK, &map_b, bar, n0 + c * 64, kb * BK);
                    } else {
                        tma_load<CG>(bt, &map_b, bar, kb * BK, n0);
                    }
                }
                __syncwarp();
                if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
            }
        }
        // every slot handed out has come back: no arrival of the leader's commits is still on its
        // way to this CTA's barriers when it leaves
        for (int i = 0; ok && i < C::STAGES; ++i) {
            ok = wait_bar<CG>(empty0 + 8 * stage, phase ^ 1, s, 6, peer_abort);
            if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
        }
    } else if (warp == 1) {
        // -------------------------------------------------------------- MMA issuer (the leader's)
        if (rank == 0) {
            // fp32 accumulate; A and B f16 (0) or bf16 (1); operand majors; N / 8; M / 16
            const uint32_t t16 = DT == ACT_DTYPE_BF16 ? 1u : 0u;
            const uint32_t idesc = (1u << 4) | (t16 << 7) | (t16 << 10) | ((uint32_t)(p.a_mn != 0) << 15) | ((uint32_t)(p.b_mn != 0) << 16) |
                                   ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(C::TILE_M >> 4) << 24);
            // K = 16 further on: 32 bytes of a K-major row, or 16 rows of 128 bytes
            const uint64_t a_step = p.a_mn ? (uint64_t)((UMMA_K * 128) >> 4) : 2ull;
            const uint64_t b_step = p.b_mn ? (uint64_t)((UMMA_K * 128) >> 4) : 2ull;
            const uint64_t adesc0 = make_desc(a0, p.a_mn != 0), bdesc0 = make_desc(b0, p.b_mn != 0);
            const uint32_t acc_full0 = smem_u32(&s->acc_full[0]), acc_empty0 = smem_u32(&s->acc_empty[0]);
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            int t = 0;
            for (int w = first; ok && w < n_work; w += stride, ++t) {
                const uint32_t buf = t & 1, use = (uint32_t)t >> 1;               // the buffer's use-th tile
                int lo, hi;
                slice_range(w % p.slices, lo, hi);
                if (!(ok = wait_bar<CG>(acc_empty0 + 8 * buf, (use & 1) ^ 1, s, 2, peer_abort))) break;
                tc_fence_after();
                const uint32_t d = tmem_base + buf * BN;
                for (int kb = lo; kb < hi; ++kb) {
                    if (!(ok = wait_bar<CG>(full0 + 8 * stage, phase, s, 3, peer_abort))) break;
                    tc_fence_after();
                    const uint64_t adesc = adesc0 + stage * (C::A_STAGE >> 4), bdesc = bdesc0 + stage * (C::B_STAGE >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; ++k)
                            umma<CG>(d, adesc + a_step * k, bdesc + b_step * k, idesc, (kb > lo || k) ? 1u : 0u);
                        umma_commit<CG>(empty0 + 8 * stage);      // frees the slot (in both CTAs)
                        if (kb == hi - 1) umma_commit<CG>(acc_full0 + 8 * buf);
                    }
                    __syncwarp();
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        const int ew = warp - 2;
        const int q = warp & 3;                                   // TMEM lane quarter this warp may read
        const int half = ew >> 2;                                 // which half of the tile's pieces
        constexpr int PIECES = BN / 64;                           // 64-column pieces of a tile
        constexpr int MINE = PIECES >= 2 ? PIECES / 2 : 1;        // this warp's: half * MINE ...
        uint8_t* const my_stage = &s->stage[ew][0][0];
        uint32_t full_phase[2] = {0, 0}, res_phase[2] = {0, 0};
        uint32_t seq = 0;                                         // pieces done: buffer seq & 1
        bool ok = true;
        // the residual of the piece at (row0, col0) into staging buffer b
        auto fetch_residual = [&](int row0, int col0, int b) {
            mbar_expect_tx(smem_u32(&s->res[ew][b]), PIECE);
            tma_load<1>(smem_u32(my_stage + b * PIECE), &map_r, smem_u32(&s->res[ew][b]), col0, row0);
        };
        const bool ahead = p.has_res && p.tma_out && !DERIV;      // residual pieces fetched one ahead
        if (ahead && lane == 0 && first < n_work) {
            const int tile = first / p.slices;
            fetch_residual((tile / n_tiles) * C::TILE_M + (int)rank * BM + q * 32, (tile % n_tiles) * BN + half * MINE * 64, 0);
        }
        int t = 0;
        for (int w = first; ok && w < n_work; w += stride, ++t) {
            const int buf = t & 1, tile = w / p.slices;
            const int row0 = (tile / n_tiles) * C::TILE_M + (int)rank * BM + q * 32, n0 = (tile % n_tiles) * BN;
            // the bias of this warp's columns, two a lane and piece, on its way while the tile's MMAs run.
            // Each warp keeps its own copy: with one per tile, and a barrier for it, the warps waited for
            // one another (GELU with derivative, K = 768: 174 us, 161 without).
            float bias_lo[MINE], bias_hi[MINE];
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int c = n0 + (half * MINE + i) * 64 + lane;
                bias_lo[i] = p.bias && c < p.N ? load_any(p.bias, c, p.bias_dtype) : 0.0f;
                bias_hi[i] = p.bias && c + 32 < p.N ? load_any(p.bias, c + 32, p.bias_dtype) : 0.0f;
            }
            if (ahead && MINE == 2 && lane == 0) {
                // the second piece's residual as early as its buffer, which the last tile's second piece
                // left through, is free; the first one's was asked for at the end of that tile
                tma_wait_read<0>();
                fetch_residual(row0, n0 + (half * MINE + 1) * 64, 1);
            }
            ok = wait_bar_warp<CG>(&s->acc_full[buf], full_phase[buf], s, 4, peer_abort);
            if (!ok) break;
            full_phase[buf] ^= 1;
            tc_fence_after();
            const uint32_t t_base = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN + half * MINE * 64);
            const int rows = p.M - row0 < 32 ? p.M - row0 : 32;   // may be <= 0
#pragma unroll 1
            for (int i = 0; i < MINE; ++i) {
                const int col0 = n0 + (half * MINE + i) * 64;
                uint32_t r[64];
                tmem_ld32(t_base + (uint32_t)(i * 64), r);
                tmem_ld32(t_base + (uint32_t)(i * 64 + 32), r + 32);
                tmem_ld_wait();
                if (i == MINE - 1) {
                    // the accumulator now lives in registers: hand the buffer back to the leader
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&s->acc_empty[buf]), 0));
                }
                if (p.out_f32) {
                    // fp32 partial plane: two 32 x 32 pieces, one staging buffer each
                    const int slice = w % p.slices;
                    if (lane == 0) tma_wait_read<0>();
                    __syncwarp();
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        *reinterpret_cast<uint4*>(my_stage + (v >> 3) * PIECE + lane * 128 + (((v & 7) ^ (lane & 7)) << 4)) =
                            make_uint4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0 && rows > 0) {
                        if (col0 < p.N) tma_store_3d(&map_y, my_stage, col0, row0, slice);
                        if (col0 + 32 < p.N) tma_store_3d(&map_y, my_stage + PIECE, col0 + 32, row0, slice);
                        tma_commit();
                    }
                    continue;
                }
                // y (and the residual) in buffer b; the derivative in buffer 1 when there is one
                const int b = DERIV ? 0 : (int)(seq & 1);
                uint8_t* const yb = my_stage + b * PIECE;
                if (p.has_res) {
                    if (p.tma_out) {
                        if (!ahead && lane == 0) { tma_wait_read<0>(); fetch_residual(row0, col0, b); }
                        ok = wait_bar_warp<CG>(&s->res[ew][b], res_phase[b], s, 7, peer_abort);
                        res_phase[b] ^= 1;
                    } else {
                        piece_in(yb, static_cast<const unsigned short*>(p.res) + (int64_t)row0 * p.ld_res + col0, p.ld_res, rows, p.N - col0, lane);
                        __syncwarp();
                    }
                }
                // the stores that last read the buffers must be done with them: waited for here when there
                // are two outputs, whose words would else fill the registers (GELU with derivative, K = 768:
                // 182 us after the arithmetic, 174 before it), and after the arithmetic when there is one
                if (DERIV) {
                    if (p.tma_out && lane == 0) tma_wait_read<0>();
                    __syncwarp();
                }
                float* const bias = s->bias[ew];
                bias[lane] = i == 0 ? bias_lo[0] : bias_lo[MINE - 1];
                bias[lane + 32] = i == 0 ? bias_hi[0] : bias_hi[MINE - 1];
                __syncwarp();
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    const ulonglong2 b0 = *reinterpret_cast<const ulonglong2*>(bias + v * 8), b1 = *reinterpret_cast<const ulonglong2*>(bias + v * 8 + 4);
                    const f32x2 bb[4] = {b0.x, b0.y, b1.x, b1.y};
                    f32x2 y[4], d[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        activate2<KIND, DERIV>(add2_rn(pack2u(r[v * 8 + 2 * j], r[v * 8 + 2 * j + 1]), bb[j]), y[j], d[j]);
                    if (p.has_res) {
                        const uint4 rr = *reinterpret_cast<const uint4*>(yb + lane * 128 + ((v ^ (lane & 7)) << 4));
                        const uint32_t h[4] = {rr.x, rr.y, rr.z, rr.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = add2_rn(y[j], widen_pair<DT>(h[j]));
                    }
                    const int at = lane * 128 + ((v ^ (lane & 7)) << 4);
                    if (DERIV) {
                        *reinterpret_cast<uint4*>(yb + at) = make_uint4(narrow_pair<DT>(y[0]), narrow_pair<DT>(y[1]), narrow_pair<DT>(y[2]), narrow_pair<DT>(y[3]));
                        *reinterpret_cast<uint4*>(my_stage + PIECE + at) =
                            make_uint4(narrow_pair<DT>(d[0]), narrow_pair<DT>(d[1]), narrow_pair<DT>(d[2]), narrow_pair<DT>(d[3]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) r[v * 8 + j] = narrow_pair<DT>(y[j]);   // eight columns of z become four words
                    }
                }
                if (!DERIV) {
                    if (p.tma_out && lane == 0 && !p.has_res) tma_wait_read<1>();    // a residual's own buffer was free before
                    __syncwarp();
#pragma unroll
                    for (int v = 0; v < 8; ++v)
                        *reinterpret_cast<uint4*>(yb + lane * 128 + ((v ^ (lane & 7)) << 4)) = make_uint4(r[v * 8], r[v * 8 + 1], r[v * 8 + 2], r[v * 8 + 3]);
                }
                if (p.tma_out) {
                    // the 32 x 64 piece leaves as one bulk tensor store, clipped at the tensor's edges
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        if (ok && rows > 0 && col0 < p.N) {
                            tma_store_2d(&map_y, yb, col0, row0);
                            if (DERIV) tma_store_2d(&map_d, my_stage + PIECE, col0, row0);
                        }
                        tma_commit();                         // also when nothing was stored: the groups count pieces
                        if (ahead && i == MINE - 1 && ok && w + stride < n_work) {
                            // the next tile's first residual goes into the other buffer once its store has read it
                            const int nt = (w + stride) / p.slices;
                            tma_wait_read<1>();
                            fetch_residual((nt / n_tiles) * C::TILE_M + (int)rank * BM + q * 32,
                                           (nt % n_tiles) * BN + half * MINE * 64, b ^ 1);
                        }
                    }
                } else {
                    __syncwarp();
                    if (ok && rows > 0 && col0 < p.N) {
                        piece_out(yb, static_cast<unsigned short*>(p.y) + (int64_t)row0 * p.ld_y + col0, p.ld_y, rows, p.N - col0, lane);
                        if (DERIV)
                            piece_out(my_stage + PIECE, static_cast<unsigned short*>(p.d) + (int64_t)row0 * p.ld_d + col0, p.ld_d, rows, p.N - col0, lane);
                    }
                    __syncwarp();
                }
                ++seq;
            }
        }
        if (lane == 0) tma_wait_read<0>();                        // the staging buffers are read before the CTA leaves
    }

    __syncwarp();                                                 // lanes that had no role wait for the one that had
    if (s->abort) {
        // give copies and MMAs still in flight time to land before the memory is released
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    tc_fence_before();
    sync_all<CG>();                                               // neither CTA's memory is needed by the other any more
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<CG>(tmem_base);
    }
}

// launches the kernel for (kind, derivative); false if CUDA refused (linear_inst_*.cu)
struct Maps { CUtensorMap a, b, y, d, r; };
template <int CG, int BN> bool launch_kernel(int kind, bool deriv, const Maps& m, const Params& p, int grid, cudaStream_t st);
// the abort reason of that file's kernels on the current device; synchronises
template <int CG, int BN> bool kernel_error(unsigned int* out, bool clear);

template <int CG, int BN, int DT, int KIND, bool DERIV>
bool launch_one(const Maps& m, const Params& p, int grid, cudaStream_t st) {
    auto* k = linear_kernel<CG, BN, DT, KIND, DERIV>;
    const int smem = (int)sizeof(Smem<CG, BN>);
    // the shared-memory opt-in is an attribute of the kernel on each device: set on the first launch there
    static bool ready[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return false;
        ready[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    cfg.blockDim = dim3(Cfg<CG, BN>::THREADS, 1, 1);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CG; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = CG == 2 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, m.a, m.b, m.y, m.d, m.r, p) == cudaSuccess;
}

// instantiated once per tile shape, in a file of its own so that they compile in parallel
#define ACT_LINEAR_INSTANTIATE(CG, BN)                                                                                   \
    template <int DT> bool launch_kind(int kind, bool deriv, const Maps& m, const Params& p, int grid, cudaStream_t st) { \
        switch (kind) {                                                                                                  \
            case ACT_KIND_NONE: return launch_one<CG, BN, DT, ACT_KIND_NONE, false>(m, p, grid, st);                     \
            case ACT_KIND_RELU: return launch_one<CG, BN, DT, ACT_KIND_RELU, false>(m, p, grid, st);                     \
            case ACT_KIND_GELU: return deriv ? launch_one<CG, BN, DT, ACT_KIND_GELU, true>(m, p, grid, st)               \
                                             : launch_one<CG, BN, DT, ACT_KIND_GELU, false>(m, p, grid, st);             \
            case ACT_KIND_SILU: return deriv ? launch_one<CG, BN, DT, ACT_KIND_SILU, true>(m, p, grid, st)               \
                                             : launch_one<CG, BN, DT, ACT_KIND_SILU, false>(m, p, grid, st);             \
            case ACT_KIND_GELU_ERF: return deriv ? launch_one<CG, BN, DT, ACT_KIND_GELU_ERF, true>(m, p, grid, st)       \
                                                 : launch_one<CG, BN, DT, ACT_KIND_GELU_ERF, false>(m, p, grid, st);     \
            default: return false;                                                                                       \
        }                                                                                                                \
    }                                                                                                                    \
    template <> bool launch_kernel<CG, BN>(int kind, bool deriv, const Maps& m, const Params& p, int grid, cudaStream_t st) { \
        return p.dtype == ACT_DTYPE_BF16 ? launch_kind<ACT_DTYPE_BF16>(kind, deriv, m, p, grid, st)                      \
                                         : launch_kind<ACT_DTYPE_F16>(kind, deriv, m, p, grid, st);                      \
    }                                                                                                                    \
    template <> bool kernel_error<CG, BN>(unsigned int* out, bool clear) {                                               \
        const unsigned int zero = 0;                                                                                     \
        return cudaMemcpyFromSymbol(out, g_linear_error, sizeof(zero)) == cudaSuccess &&                                 \
               (!clear || cudaMemcpyToSymbol(g_linear_error, &zero, sizeof(zero)) == cudaSuccess);                       \
    }

}  // namespace linear
}  // namespace act
