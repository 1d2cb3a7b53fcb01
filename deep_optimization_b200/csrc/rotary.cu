// Rotary positions with several axes, sm_100a.  The first 2 P elements of a head are P pairs; pair j
// belongs to one axis (time, height, width, ...) and is turned by
//
//     angle(t, j) = pos[t, axis(j)] * turns[j]          (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin)
//
// Pairs are (j, P + j), or (2 j, 2 j + 1) when interleaved; elements from 2 P on pass through.  The
// backward pass is the same kernel with the angles negated.
//
// turns[j] is a frequency as a 64-bit binary fraction of a turn per position: the low 64 bits of its
// product with an integer position are the angle modulo a whole turn with an error of |pos| / 2
// units of 2^-64 turns, so a position of 10^9 costs nothing in accuracy (a float32 product would be
// off by whole turns) and no table of positions bounds them.  The quarter turn is taken off in
// integers; sincospi sees |x| <= 1/4.
//
// Up to three tensors of one [B, T] (q, k and v with their own head counts, strides and destinations)
// go through in one pass: forward this is the q/k/v split of a fused projection with the rotation
// in it, backward the merge of the three gradients into the projection's.  Bound: HBM, every
// element read once and written once.  A block takes a run of (b, t) rows, computes cos and sin of
// the rows' pairs once for all heads into shared memory, and every thread keeps its (tensor, head,
// 16-byte vector or pair of vectors) and walks the rows.
#include "act_common.cuh"

namespace act {

int stream_grid_for(int64_t n_blocks_wanted, int blocks_per_sm, int waves = 1);   // cabi.cu

namespace rotary {

// Rows in flight per thread, and rows it walks in all.  Measured on bf16 [256, 197, 3 x 12 x 64] each way
// (floor 71 us) and fp32 [2, 4601, 24 x 80] interleaved (floor 22 us): depth 1, 2, 3, 4 = 93, 82, 113, 112 us
// (beyond 64 registers a thread the SM holds too few of them); 2, 4, 8, 16 rows = 118, 93, 81, 87 us (fewer
// do not pay for the block's start, more leave SMs idle at the end).
constexpr int kDepth = 2, kRows = 8;
constexpr int kParts = 3, kAxes = 4;
constexpr int kTableBytes = 32 * 1024;       // cos/sin of a block's rows

struct Part {
    const uint8_t* src;
    uint8_t* dst;
    int64_t sb, sh, st, db, dh, dt;          // element strides of batch, head, token
    int rotate, units, per_head;             // work items of one (b, t) row, of one head of it
};
struct Args {
    Part part[kParts];
    const void* pos;
    int64_t pb, pt, pa;                      // element strides of pos
    const uint64_t* turns;
    int first[kAxes + 1];                    // pairs of axis a: first[a] .. first[a + 1]
    int64_t rows;
    int T, P, units, lanes, rows_per_block, pos64, interleaved, inverse;
};

// cos and sin of `a` units of 2^-64 turns
__device__ __forceinline__ float2 cos_sin(uint64_t a) {
    const uint64_t shifted = a + (1ull << 61);
    const int quarter = (int)(shifted >> 62);                             // nearest quarter turn
    const int64_t rest = (int64_t)(a - ((uint64_t)quarter << 62));        // [-2^61, 2^61)
    // rest * 2^-64 turns = rest * 2^-63 * pi
    const float half_turns = __fmul_rn((float)rest, 1.0842021724855044e-19f);   // 2^-63
    float s, c;
    sincospif(half_turns, &s, &c);
    if (quarter & 1) { const float x = c; c = -s; s = x; }
    if (quarter & 2) { c = -c; s = -s; }
    return make_float2(c, s);
}

// what one access brings: W 32-bit words of a 16- or 32-byte vector, or one element in the low bits (W = 1)
template <int W> struct Raw { uint32_t u[W]; };

template <int DT, int W> __device__ __forceinline__ Raw<W> fetch(const uint8_t* p) {
    Raw<W> v;
    if (W == 1) {
        v.u[0] = DT == ACT_DTYPE_F32 ? *reinterpret_cast<const uint32_t*>(p) : (uint32_t)*reinterpret_cast<const unsigned short*>(p);
    } else if (W == 4) {
        asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(v.u[0]), "=r"(v.u[1 % W]), "=r"(v.u[2 % W]), "=r"(v.u[3 % W]) : "l"(p) : "memory");
    } else {
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(v.u[0]), "=r"(v.u[1 % W]), "=r"(v.u[2 % W]), "=r"(v.u[3 % W]), "=r"(v.u[4 % W]), "=r"(v.u[5 % W]),
                       "=r"(v.u[6 % W]), "=r"(v.u[7 % W]) : "l"(p) : "memory");
    }
    return v;
}
template <int DT, int W> __device__ __forceinline__ void put(uint8_t* p, const Raw<W>& v) {
    if (W == 1) {
        if (DT == ACT_DTYPE_F32) *reinterpret_cast<uint32_t*>(p) = v.u[0];
        else *reinterpret_cast<unsigned short*>(p) = (unsigned short)v.u[0];
    } else if (W == 4) {
        stg_stream_v4(p, make_uint4(v.u[0], v.u[1 % W], v.u[2 % W], v.u[3 % W]));
    } else {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                     :: "l"(p), "r"(v.u[0]), "r"(v.u[1 % W]), "r"(v.u[2 % W]), "r"(v.u[3 % W]), "r"(v.u[4 % W]), "r"(v.u[5 % W]),
                        "r"(v.u[6 % W]), "r"(v.u[7 % W]) : "memory");
    }
}
template <int DT> __device__ __forceinline__ uint32_t round2(float a, float b) {
    if (DT == ACT_DTYPE_F16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// a pair turned: products and sums rounded one by one but for the fused second product
__device__ __forceinline__ void turn(float& a, float& b, float2 cs) {
    const float x = __fmaf_rn(a, cs.x, -__fmul_rn(b, cs.y)), y = __fmaf_rn(b, cs.x, __fmul_rn(a, cs.y));
    a = x; b = y;
}
// pairs split over two vectors: element i of a with element i of b, angles cs[i]
template <int DT, int W> __device__ __forceinline__ void turn_split(Raw<W>& a, Raw<W>& b, const float2* cs) {
    constexpr int D16 = (DT == ACT_DTYPE_F32) ? ACT_DTYPE_BF16 : DT;
    if (W == 1) {
        float x = DT == ACT_DTYPE_F32 ? __uint_as_float(a.u[0]) : widen_lo<D16>(a.u[0]);
        float y = DT == ACT_DTYPE_F32 ? __uint_as_float(b.u[0]) : widen_lo<D16>(b.u[0]);
        turn(x, y, cs[0]);
        a.u[0] = DT == ACT_DTYPE_F32 ? __float_as_uint(x) : round2<DT>(x, 0.0f);
        b.u[0] = DT == ACT_DTYPE_F32 ? __float_as_uint(y) : round2<DT>(y, 0.0f);
        return;
    }
    const float4* cs2 = reinterpret_cast<const float4*>(cs);  // the pair count is a multiple of a vector's elements
#pragma unroll
    for (int k = 0; k < W; ++k) {
        if (DT == ACT_DTYPE_F32) {
            if (k & 1) continue;
            const float4 c = cs2[k / 2];
            float x0 = __uint_as_float(a.u[k]), x1 = __uint_as_float(a.u[(k + 1) % W]);
            float y0 = __uint_as_float(b.u[k]), y1 = __uint_as_float(b.u[(k + 1) % W]);
            turn(x0, y0, make_float2(c.x, c.y));
            turn(x1, y1, make_float2(c.z, c.w));
            a.u[k] = __float_as_uint(x0); a.u[(k + 1) % W] = __float_as_uint(x1);
            b.u[k] = __float_as_uint(y0); b.u[(k + 1) % W] = __float_as_uint(y1);
        } else {
            const float4 c = cs2[k];
            float x0 = widen_lo<D16>(a.u[k]), x1 = widen_hi<D16>(a.u[k]), y0 = widen_lo<D16>(b.u[k]), y1 = widen_hi<D16>(b.u[k]);
            turn(x0, y0, make_float2(c.x, c.y));
            turn(x1, y1, make_float2(c.z, c.w));
            a.u[k] = round2<DT>(x0, x1);
            b.u[k] = round2<DT>(y0, y1);
        }
    }
}
// pairs side by side in one vector, the first `left` of them turned
template <int DT, int W> __device__ __forceinline__ void turn_adjacent(Raw<W>& a, const float2* cs, int left) {
    constexpr int D16 = (DT == ACT_DTYPE_F32) ? ACT_DTYPE_BF16 : DT;
#pragma unroll
    for (int k = 0; k < W; ++k) {
        if (DT == ACT_DTYPE_F32) {
            if ((k & 1) || k / 2 >= left) continue;
            float x = __uint_as_float(a.u[k]), y = __uint_as_float(a.u[(k + 1) % W]);
            turn(x, y, cs[k / 2]);
            a.u[k] = __float_as_uint(x); a.u[(k + 1) % W] = __float_as_uint(y);
        } else {
            if (k >= left) continue;
            float x = widen_lo<D16>(a.u[k]), y = widen_hi<D16>(a.u[k]);
            turn(x, y, cs[k]);
            a.u[k] = round2<DT>(x, y);
        }
    }
}

// W words per access: 32 or 16 bytes, or one element where strides, bases or the pair count allow no more.
// A block takes rows_per_block consecutive (b, t) rows.  Its threads are lanes x work items of a row;
// thread (l, u) walks rows l, l + lanes, ... of item u with two rows' loads in flight, the first two
// issued before the angles are computed, which hides the latency of both.
template <int DT, int W, bool INTER>
__global__ void __launch_bounds__(512, 2)
rotary_kernel(const __grid_constant__ Args g)
{
    extern __shared__ __align__(16) float2 table[];          // [rows of the block][P]
    constexpr int ES = ElemT<DT>::bytes, V = W == 1 ? 1 : 4 * W / ES;      // elements of an access
    const int64_t row0 = (int64_t)blockIdx.x * g.rows_per_block;
    const int n_rows = (int)(g.rows - row0 < g.rows_per_block ? g.rows - row0 : g.rows_per_block);
    // the block's first row: batch b0, token t0 (a 64-bit division only where the rows need it)
    const int64_t b0 = g.rows >> 32 ? row0 / g.T : (int64_t)((uint32_t)row0 / (uint32_t)g.T);
    const int t0 = (int)(row0 - b0 * g.T);
    const int per_pass = g.units < (int)blockDim.x ? g.units : (int)blockDim.x;
    const int lane = threadIdx.x / per_pass, lanes = g.lanes;
    for (int u0 = threadIdx.x - lane * per_pass, pass = 0; pass * per_pass < g.units; ++pass, u0 += per_pass) {
        const bool works = lane < lanes && u0 < g.units && lane < n_rows;
        int e0 = 0, e1 = -1, j0 = 0;
        bool turned = false;
        const uint8_t* src = nullptr;
        uint8_t* dst = nullptr;
        int64_t s_row = 0, d_row = 0, s_wrap = 0, d_wrap = 0;
        int t = 0;
        if (works) {
            int s = 0, u = u0;
            if (u >= g.part[0].units) { u -= g.part[0].units; s = 1; }
            if (s == 1 && u >= g.part[1].units) { u -= g.part[1].units; s = 2; }
            const Part& p = g.part[s];
            const int per_head = p.per_head;
            const int h = (int)((uint32_t)u / (uint32_t)per_head), q = u - h * per_head;
            // where the item's elements lie in the head, and whether they are turned
            turned = p.rotate && (INTER ? (V == 1 ? q < g.P : q * V < 2 * g.P) : q * V < g.P);
            if (!p.rotate) e0 = q * V;
            else if (INTER) {
                if (V == 1) { j0 = q; e0 = turned ? 2 * q : q + g.P; e1 = turned ? 2 * q + 1 : -1; }
                else { e0 = q * V; j0 = e0 / 2; }
            } else if (turned) { e0 = j0 = q * V; e1 = g.P + e0; }
            else e0 = q * V + g.P;                            // the P / V items before these cover 2 P elements
            const uint32_t over = (uint32_t)(t0 + lane) / (uint32_t)g.T;
            const int64_t b = b0 + over;
            t = (int)((uint32_t)(t0 + lane) - over * (uint32_t)g.T);
            src = p.src + ((int64_t)h * p.sh + b * p.sb + t * p.st + e0) * ES;
            dst = p.dst + ((int64_t)h * p.dh + b * p.db + t * p.dt + e0) * ES;
            s_row = p.st * ES; s_wrap = (p.sb - g.T * p.st) * ES;
            d_row = p.dt * ES; d_wrap = (p.db - g.T * p.dt) * ES;
        }
        const int e_off = (e1 - e0) * ES;
        const bool two = (V == 1 || !INTER) && e1 >= 0;       // interleaved vectors hold whole pairs
        Raw<W> a[kDepth], b[kDepth];
        int ts = t;                                           // token that src points at
        auto next = [&](int& tok, int64_t& step, int64_t row, int64_t wrap) {
            step = row * lanes;
            tok += lanes;
            if (tok >= g.T) {
                const int over = tok / g.T;
                tok -= over * g.T;
                step += over * wrap;
            }
        };
        int left = works ? (n_rows - lane + lanes - 1) / lanes : 0;       // rows not yet fetched
        int todo = left;
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
            if (left > 0) {
                a[i] = fetch<DT, W>(src);
                if (two) b[i] = fetch<DT, W>(src + e_off);
                int64_t step;
                next(ts, step, s_row, s_wrap);
                src += step;
                --left;
            }
        }
        if (pass == 0) {
            for (int i = threadIdx.x; i < n_rows * g.P; i += blockDim.x) {
                const int r = (int)((uint32_t)i / (uint32_t)g.P), j = i - r * g.P;
                const uint32_t over = (uint32_t)(t0 + r) / (uint32_t)g.T;
                const int64_t bb = b0 + over;
                const uint32_t tt = (uint32_t)(t0 + r) - over * (uint32_t)g.T;
                int axis = 0;
#pragma unroll
                for (int x = 1; x < kAxes; ++x) axis += j >= g.first[x] ? 1 : 0;
                const int64_t at = bb * g.pb + tt * g.pt + axis * g.pa;
                const int64_t pos = g.pos64 ? static_cast<const int64_t*>(g.pos)[at] : (int64_t)static_cast<const int32_t*>(g.pos)[at];
                float2 cs = cos_sin((uint64_t)pos * g.turns[j]);
                if (g.inverse) cs.y = -cs.y;
                table[i] = cs;
            }
            __syncthreads();
        }
        const float2* cs = table + lane * g.P + j0;
        int td = t;
        while (todo > 0) {
#pragma unroll
            for (int i = 0; i < kDepth; ++i) {
                if (todo <= 0) break;
                Raw<W> va = a[i], vb = b[i];
                if (left > 0) {
                    a[i] = fetch<DT, W>(src);
                    if (two) b[i] = fetch<DT, W>(src + e_off);
                    int64_t step;
                    next(ts, step, s_row, s_wrap);
                    src += step;
                    --left;
                }
                if (turned) {
                    if (V == 1 || !INTER) turn_split<DT, W>(va, vb, cs);
                    else turn_adjacent<DT, W>(va, cs, g.P - j0);
                }
                put<DT, W>(dst, va);
                if (two) put<DT, W>(dst + e_off, vb);
                int64_t step;
                next(td, step, d_row, d_wrap);
                dst += step;
                cs += lanes * g.P;
                --todo;
            }
        }
    }
}

template <int DT, int W>
cudaError_t launch(const Args& g, int blocks, int threads, int smem, cudaStream_t st) {
    if (g.interleaved) rotary_kernel<DT, W, true><<<blocks, threads, smem, st>>>(g);
    else rotary_kernel<DT, W == 8 ? 4 : W, false><<<blocks, threads, smem, st>>>(g);        // 8 is interleaved only
    return cudaGetLastError();
}

}  // namespace rotary
}  // namespace act

extern "C" int act_rotary_heads(const void* const* srcs, const int64_t* src_strides, void* const* dsts,
                                const int64_t* dst_strides, const int* heads, const int* rotate, int parts, int dtype,
                                int64_t B, int64_t T, int Dh, const void* pos, int pos_bytes, const int64_t* pos_strides,
                                const void* turns, const int* sections, int axes, int interleaved, int inverse,
                                void* stream)
{
    using namespace act;
    using namespace act::rotary;
    if (dtype != ACT_DTYPE_F32 && dtype != ACT_DTYPE_BF16 && dtype != ACT_DTYPE_F16) return ACT_ERR_DTYPE;
    if (pos_bytes != 4 && pos_bytes != 8) return ACT_ERR_DTYPE;
    if (parts < 1 || parts > kParts || axes < 1 || axes > kAxes || B < 0 || T < 0 || Dh < 1 || Dh > 1024) return ACT_ERR_SIZE;
    if (T > 0x7FFFFFFF || (T > 0 && B > ((int64_t)1 << 40) / T)) return ACT_ERR_SIZE;
    if (!heads || !rotate || !sections) return ACT_ERR_NULL;
    int64_t P = 0;
    Args g = {};
    for (int a = 0; a < kAxes; ++a) {
        if (a < axes && (sections[a] < 0 || sections[a] > Dh)) return ACT_ERR_SIZE;
        g.first[a] = (int)P;
        if (a < axes) P += sections[a];
    }
    g.first[kAxes] = (int)P;
    if (2 * P > Dh) return ACT_ERR_SIZE;
    int total_heads = 0;
    for (int s = 0; s < parts; ++s) {
        if (heads[s] < 0 || heads[s] > 65536) return ACT_ERR_SIZE;
        total_heads += heads[s];
    }
    if (B == 0 || T == 0 || total_heads == 0) return ACT_OK;
    if (!srcs || !src_strides || !dsts || !dst_strides) return ACT_ERR_NULL;
    if (P > 0 && (!pos || !pos_strides || !turns)) return ACT_ERR_NULL;
    if (P > 0 && (((uintptr_t)pos & (pos_bytes - 1)) || ((uintptr_t)turns & 7))) return ACT_ERR_ALIGN;

    const int es = dtype == ACT_DTYPE_F32 ? 4 : 2;
    uint64_t low = 0;                        // low bits of every base and stride, in bytes
    for (int s = 0; s < parts; ++s) {
        if (heads[s] == 0) continue;
        if (!srcs[s] || !dsts[s]) return ACT_ERR_NULL;
        low |= (uintptr_t)srcs[s] | (uintptr_t)dsts[s];
        if (low & (es - 1)) return ACT_ERR_ALIGN;
        for (int i = 0; i < 3; ++i) low |= (uint64_t)(src_strides[3 * s + i] * es) | (uint64_t)(dst_strides[3 * s + i] * es);
    }
    // the widest access that every base, stride and the pair count allow: 32, 16 bytes or one element
    auto allows = [&](int bytes) { return !(low & (bytes - 1)) && (Dh * es) % bytes == 0 && (interleaved || (P * es) % bytes == 0); };
    // (32 only interleaved: there it takes the video case above from 30 to 23 us; pairs split over two
    // vectors would need 96 registers, 100 us instead of 81)
    const int words = interleaved && allows(32) ? 8 : (allows(16) ? 4 : 1);
    const int v = words == 1 ? 1 : 4 * words / es;
    int k = 0;
    for (int s = 0; s < parts; ++s) {
        if (heads[s] == 0) continue;
        Part& p = g.part[k++];
        p.src = static_cast<const uint8_t*>(srcs[s]);
        p.dst = static_cast<uint8_t*>(dsts[s]);
        p.sb = src_strides[3 * s]; p.sh = src_strides[3 * s + 1]; p.st = src_strides[3 * s + 2];
        p.db = dst_strides[3 * s]; p.dh = dst_strides[3 * s + 1]; p.dt = dst_strides[3 * s + 2];
        p.rotate = rotate[s] && P > 0;
        // a unit is one access, or the two of a pair (j, P + j) / (2 j, 2 j + 1)
        const bool paired = p.rotate && (!interleaved || v == 1);
        p.per_head = (paired ? Dh - (int)P : Dh) / v;
        p.units = heads[s] * p.per_head;
        g.units += p.units;
    }
    g.pos = pos;
    if (P > 0) { g.pb = pos_strides[0]; g.pt = pos_strides[1]; g.pa = pos_strides[2]; }
    g.turns = static_cast<const uint64_t*>(turns);
    g.rows = B * T; g.T = (int)T; g.P = (int)P;
    g.pos64 = pos_bytes == 8; g.interleaved = interleaved != 0; g.inverse = inverse != 0;

    // Blocks of up to 512 threads; a row with few work items shares its block with other rows.  A thread
    // walks kRows rows, fewer where that would leave SMs without a full set of threads.
    g.lanes = g.units >= 128 ? 1 : 256 / g.units;
    if (g.lanes > g.rows) g.lanes = (int)g.rows;
    const int threads = g.units > 512 ? 512 : ((g.units * g.lanes + 31) & ~31);
    const int64_t target = stream_grid_for((int64_t)1 << 40, 1024 / threads, 1);
    int64_t per = (g.rows + target * g.lanes - 1) / (target * g.lanes);
    per = (per < kRows ? per : kRows) * g.lanes;
    const int64_t most = P > 0 ? kTableBytes / (8 * P) : 4096;
    if (per > most) per = most;
    const int64_t blocks = (g.rows + per - 1) / per;
    if (blocks > 0x7FFFFFFF) return ACT_ERR_SIZE;
    g.rows_per_block = (int)per;
    const int smem = (int)(per * P * 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define ACT_ROTARY(DT) \
    (words == 8 ? launch<DT, 8>(g, (int)blocks, threads, smem, st) \
                : words == 4 ? launch<DT, 4>(g, (int)blocks, threads, smem, st) : launch<DT, 1>(g, (int)blocks, threads, smem, st))
    const cudaError_t e = dtype == ACT_DTYPE_F32 ? ACT_ROTARY(ACT_DTYPE_F32)
                          : dtype == ACT_DTYPE_BF16 ? ACT_ROTARY(ACT_DTYPE_BF16) : ACT_ROTARY(ACT_DTYPE_F16);
#undef ACT_ROTARY
    return e == cudaSuccess ? ACT_OK : ACT_ERR_LAUNCH;
}

// qkv and dst contiguous [B, T, (heads + 2 kv_heads) Dh]
extern "C" int act_rotary_split(const void* qkv, void* dst, int heads, int kv_heads, int dtype, int64_t B, int64_t T, int Dh,
                                const void* pos, int pos_bytes, int64_t pos_sb, int64_t pos_st, int64_t pos_sa,
                                const void* turns, const int* sections, int axes, int interleaved, void* stream)
{
    if (heads < 0 || kv_heads < 0 || heads > 65536 || kv_heads > 65536 || Dh < 1 || Dh > 1024 || T < 0) return ACT_ERR_SIZE;
    const int64_t es = dtype == ACT_DTYPE_F32 ? 4 : 2, W = (int64_t)(heads + 2 * kv_heads) * Dh;
    const uint8_t* s = static_cast<const uint8_t*>(qkv);
    uint8_t* d = static_cast<uint8_t*>(dst);
    const int64_t at[3] = {0, (int64_t)heads * Dh * es, (int64_t)(heads + kv_heads) * Dh * es};
    const void* srcs[3];
    void* dsts[3];
    int64_t strides[9];
    for (int i = 0; i < 3; ++i) {
        srcs[i] = s ? s + at[i] : nullptr;
        dsts[i] = d ? d + at[i] : nullptr;
        strides[3 * i] = T * W; strides[3 * i + 1] = Dh; strides[3 * i + 2] = W;
    }
    const int counts[3] = {heads, kv_heads, kv_heads}, rotate[3] = {1, 1, 0};
    const int64_t ps[3] = {pos_sb, pos_st, pos_sa};
    return act_rotary_heads(srcs, strides, dsts, strides, counts, rotate, 3, dtype, B, T, Dh, pos, pos_bytes, ps, turns,
                            sections, axes, interleaved, 0, stream);
}

extern "C" int act_rotary_merge(const void* dq, const void* dk, const void* dv, const int64_t* src_strides, void* dst,
                                int heads, int kv_heads, int dtype, int64_t B, int64_t T, int Dh, const void* pos,
                                int pos_bytes, int64_t pos_sb, int64_t pos_st, int64_t pos_sa, const void* turns,
                                const int* sections, int axes, int interleaved, void* stream)
{
    if (heads < 0 || kv_heads < 0 || heads > 65536 || kv_heads > 65536 || Dh < 1 || Dh > 1024 || T < 0) return ACT_ERR_SIZE;
    const int64_t es = dtype == ACT_DTYPE_F32 ? 4 : 2, W = (int64_t)(heads + 2 * kv_heads) * Dh;
    uint8_t* d = static_cast<uint8_t*>(dst);
    const int64_t at[3] = {0, (int64_t)heads * Dh * es, (int64_t)(heads + kv_heads) * Dh * es};
    const void* srcs[3] = {dq, dk, dv};
    void* dsts[3];
    int64_t strides[9];
    for (int i = 0; i < 3; ++i) {
        dsts[i] = d ? d + at[i] : nullptr;
        strides[3 * i] = T * W; strides[3 * i + 1] = Dh; strides[3 * i + 2] = W;
    }
    const int counts[3] = {heads, kv_heads, kv_heads}, rotate[3] = {1, 1, 0};
    const int64_t ps[3] = {pos_sb, pos_st, pos_sa};
    return act_rotary_heads(srcs, src_strides, dsts, strides, counts, rotate, 3, dtype, B, T, Dh, pos, pos_bytes, ps, turns,
                            sections, axes, interleaved, 1, stream);
}
