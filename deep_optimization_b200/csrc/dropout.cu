// Dropout whose mask is never stored, sm_100a:
//
//     y[e] = (keep(e) ? x[e] * 65536 / (65536 - t) : 0) + r[e]          (r: an optional residual)
//
// The mask is a function of (seed, offset, e) alone, so the backward pass is this kernel again on
// dy: nothing is saved between the two (PyTorch's dropout keeps a byte per element).  Eight
// consecutive elements share one block of Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel
// random numbers: as easy as 1, 2, 3", 2011): counter (block number, offset), key = seed; element
// e takes the e & 7th sixteen bits h of block e >> 3 and is kept when h >= t.  t is the dropping
// probability in 2^-16, and the survivors' factor is that of the rounded probability, so E[y] = x
// exactly.  A dropped element contributes 0 whatever it held, infinities and NaN included.
//
// Bound: HBM, each input read once and y written once.  A thread moves 32-byte vectors (16 elements
// of 16 bits, 8 of 32) and runs the generator while its loads are on their way: ten rounds are about
// 60 integer instructions for eight elements, a third of what the SMs issue in the time the bytes take.
// bf16 [50432, 768]: 27 us (5.7 TB/s), with a residual 38 us (6.1 TB/s); 768 elements: 1.3 us.
#include "act_common.cuh"

namespace act {
namespace drop {

constexpr int kThreads = 256;

struct Key { uint32_t k0, k1, c2, c3; };

__device__ __forceinline__ void philox(uint64_t block, const Key& key, uint32_t (&w)[4]) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = key.c2, c3 = key.c3;
    uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = (uint64_t)0xD2511F53u * c0, q = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)q;
        c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// factor of element j of a block: `scale` when its sixteen bits reach the threshold, else 0
__device__ __forceinline__ bool kept(const uint32_t (&w)[4], int j, uint32_t threshold) {
    return ((w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu) >= threshold;
}

struct V32 { uint32_t u[8]; };               // 32 bytes
// plain (not read-only) loads: y may be x or r
__device__ __forceinline__ V32 ld32(const uint8_t* p) {
    V32 v;
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v.u[0]), "=r"(v.u[1]), "=r"(v.u[2]), "=r"(v.u[3]), "=r"(v.u[4]), "=r"(v.u[5]), "=r"(v.u[6]), "=r"(v.u[7])
                 : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void st32(uint8_t* p, const V32& v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 :: "l"(p), "r"(v.u[0]), "r"(v.u[1]), "r"(v.u[2]), "r"(v.u[3]), "r"(v.u[4]), "r"(v.u[5]), "r"(v.u[6]), "r"(v.u[7])
                 : "memory");
}

template <int DT> __device__ __forceinline__ float load1(const uint8_t* p, int64_t e) {
    if (DT == ACT_DTYPE_F32) return reinterpret_cast<const float*>(p)[e];
    const uint32_t h = reinterpret_cast<const unsigned short*>(p)[e];
    constexpr int D16 = (DT == ACT_DTYPE_F32) ? ACT_DTYPE_BF16 : DT;
    return widen_lo<D16>(h);
}
template <int DT> __device__ __forceinline__ uint32_t round2(float a, float b) {
    if (DT == ACT_DTYPE_F16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int DT> __device__ __forceinline__ void store1(uint8_t* p, int64_t e, float v) {
    if (DT == ACT_DTYPE_F32) reinterpret_cast<float*>(p)[e] = v;
    else reinterpret_cast<unsigned short*>(p)[e] = (unsigned short)round2<DT>(v, 0.0f);
}

// one 32-byte vector starting at element e0 (a multiple of 8)
template <int DT, bool RES>
__device__ __forceinline__ V32 apply(const V32& x, const V32& r, int64_t e0, const Key& key, uint32_t threshold, float scale) {
    V32 y;
    uint32_t w[4];
    if (DT == ACT_DTYPE_F32) {
        philox((uint64_t)e0 >> 3, key, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = kept(w, j, threshold) ? __fmul_rn(__uint_as_float(x.u[j]), scale) : 0.0f;
            y.u[j] = __float_as_uint(RES ? __fadd_rn(a, __uint_as_float(r.u[j])) : a);
        }
    } else {
        constexpr int D16 = (DT == ACT_DTYPE_F32) ? ACT_DTYPE_BF16 : DT;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            philox(((uint64_t)e0 >> 3) + half, key, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t v = x.u[half * 4 + j], q = RES ? r.u[half * 4 + j] : 0u;
                float a = kept(w, 2 * j, threshold) ? __fmul_rn(widen_lo<D16>(v), scale) : 0.0f;
                float b = kept(w, 2 * j + 1, threshold) ? __fmul_rn(widen_hi<D16>(v), scale) : 0.0f;
                if (RES) { a = __fadd_rn(a, widen_lo<D16>(q)); b = __fadd_rn(b, widen_hi<D16>(q)); }
                y.u[half * 4 + j] = round2<D16>(a, b);
            }
        }
    }
    return y;
}

// VEC: all pointers 32-byte aligned.  A thread owns UNROLL vectors, kThreads apart; the vector that
// the end of the tensor cuts, and everything when !VEC, goes element by element.
template <int DT, bool RES, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const uint8_t* x, const uint8_t* r, uint8_t* y, int64_t n, uint32_t threshold, float scale,
               uint64_t seed, uint64_t offset, const uint64_t* rng)
{
    constexpr int E = 32 / ElemT<DT>::bytes;                  // elements of a vector
    constexpr int UNROLL = VEC ? 2 : 1;
    grid_dependency_wait();
    if (rng) { seed = rng[0]; offset = rng[1]; }
    const Key key = {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
    const int64_t v0 = (int64_t)blockIdx.x * (kThreads * UNROLL) + threadIdx.x;
    if (VEC && (v0 - threadIdx.x + kThreads * UNROLL) * E <= n) {         // a whole block of whole vectors
        V32 a[UNROLL], b[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int64_t at = (v0 + u * kThreads) * 32;
            a[u] = ld32(x + at);
            if (RES) b[u] = ld32(r + at);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int64_t v = v0 + u * kThreads;
            st32(y + v * 32, apply<DT, RES>(a[u], b[u], v * E, key, threshold, scale));
        }
        return;
    }
    for (int u = 0; u < UNROLL; ++u) {
        const int64_t v = v0 + u * kThreads, e0 = v * E;
        if (e0 >= n) return;
        if (VEC && e0 + E <= n) {
            V32 a = ld32(x + v * 32), b = a;
            if (RES) b = ld32(r + v * 32);
            st32(y + v * 32, apply<DT, RES>(a, b, e0, key, threshold, scale));
            continue;
        }
        uint32_t w[4];
        for (int j = 0; j < E && e0 + j < n; ++j) {
            if ((j & 7) == 0) philox((uint64_t)(e0 + j) >> 3, key, w);
            float a = ((w[(j & 7) >> 1] >> (16 * (j & 1))) & 0xFFFFu) >= threshold ? __fmul_rn(load1<DT>(x, e0 + j), scale) : 0.0f;
            if (RES) a = __fadd_rn(a, load1<DT>(r, e0 + j));
            store1<DT>(y, e0 + j, a);
        }
    }
}

// Hands out the next number of a stream that lives on the device: a captured launch of this kernel
// takes a new one at every replay, and two graphs that replay at once never the same.
__global__ void rng_ticket_kernel(unsigned long long* state, unsigned long long* out) {
    out[0] = state[0];
    out[1] = atomicAdd(state + 1, 1ull);
}

template <int DT, bool RES>
cudaError_t launch(const void* x, const void* r, void* y, int64_t n, uint32_t threshold, float scale, uint64_t seed,
                   uint64_t offset, const void* rng, cudaStream_t st) {
    constexpr int E = 32 / ElemT<DT>::bytes;
    const bool vec = !(((uintptr_t)x | (uintptr_t)r | (uintptr_t)y) & 31);
    const int64_t vectors = (n + E - 1) / E;
    const int64_t per_block = kThreads * (vec ? 2 : 1);
    const int64_t blocks = (vectors + per_block - 1) / per_block;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
    auto* k = vec ? dropout_kernel<DT, RES, true> : dropout_kernel<DT, RES, false>;
    return launch_overlapped(k, (int)blocks, kThreads, st, static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(r),
                             static_cast<uint8_t*>(y), n, threshold, scale, seed, offset, static_cast<const uint64_t*>(rng));
}

template <int DT>
cudaError_t launch_any(const void* x, const void* r, void* y, int64_t n, uint32_t threshold, float scale, uint64_t seed,
                       uint64_t offset, const void* rng, cudaStream_t st) {
    return r ? launch<DT, true>(x, r, y, n, threshold, scale, seed, offset, rng, st)
             : launch<DT, false>(x, nullptr, y, n, threshold, scale, seed, offset, rng, st);
}

}  // namespace drop
}  // namespace act

extern "C" int act_dropout(const void* x, const void* residual, int dtype, int64_t n, unsigned threshold, uint64_t seed,
                           uint64_t offset, const void* rng, void* y, void* stream)
{
    using namespace act::drop;
    if (dtype != ACT_DTYPE_F32 && dtype != ACT_DTYPE_BF16 && dtype != ACT_DTYPE_F16) return ACT_ERR_DTYPE;
    if (n < 0 || n > ((int64_t)1 << 40) || threshold > 65536u) return ACT_ERR_SIZE;
    if (n == 0) return ACT_OK;
    if (!x || !y) return ACT_ERR_NULL;
    const uintptr_t es = dtype == ACT_DTYPE_F32 ? 4 : 2;
    if ((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) & (es - 1)) || ((uintptr_t)rng & 7)) return ACT_ERR_ALIGN;
    const float scale = threshold >= 65536u ? 0.0f : 65536.0f / (float)(65536u - threshold);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == ACT_DTYPE_F32) e = launch_any<ACT_DTYPE_F32>(x, residual, y, n, threshold, scale, seed, offset, rng, st);
    else if (dtype == ACT_DTYPE_BF16) e = launch_any<ACT_DTYPE_BF16>(x, residual, y, n, threshold, scale, seed, offset, rng, st);
    else e = launch_any<ACT_DTYPE_F16>(x, residual, y, n, threshold, scale, seed, offset, rng, st);
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ACT_ERR_LAUNCH; }
    return ACT_OK;
}

extern "C" int act_rng_ticket(void* state, void* out, void* stream)
{
    if (!state || !out) return ACT_ERR_NULL;
    if (((uintptr_t)state | (uintptr_t)out) & 7) return ACT_ERR_ALIGN;
    act::drop::rng_ticket_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<unsigned long long*>(state), static_cast<unsigned long long*>(out));
    return cudaGetLastError() == cudaSuccess ? ACT_OK : ACT_ERR_LAUNCH;
}
