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

constexpr int kParts = 3, kAxes = 4;
constexpr int kTableBytes = 32 * 1024;       // cos/sin of a block's rows

struct Part {
    const uint8_t* src;
    uint8_t* dst;
    int64_t sb, sh, st, db, dh, dt;          // element strides of batch, head, token
    int heads, rotate, units;                // units: work items of one (b, t) row
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

// what one access brings: 16 bytes, or one element in the low bits of x
template <int DT, int V> __device__ __forceinline__ uint4 fetch(const uint8_t* p) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (V == 1) {
        v.x = DT == ACT_DTYPE_F32 ? *reinterpret_cast<const uint32_t*>(p) : (uint32_t)*reinterpret_cast<const unsigned short*>(p);
    } else {
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    }
    return v;
}
template <int DT, int V> __device__ __forceinline__ void widen(uint4 v, float (&f)[V]) {
    constexpr int D16 = (DT == ACT_DTYPE_F32) ? ACT_DTYPE_BF16 : DT;
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < V; ++i)
        f[i] = DT == ACT_DTYPE_F32 ? __uint_as_float(u[i & 3]) : ((i & 1) ? widen_hi<D16>(u[(i >> 1) & 3]) : widen_lo<D16>(u[(i >> 1) & 3]));
}
template <int DT> __device__ __forceinline__ uint32_t round2(float a, float b) {
    if (DT == ACT_DTYPE_F16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int DT, int V> __device__ __forceinline__ uint4 narrow(const float (&f)[V]) {
    if (DT == ACT_DTYPE_F32)
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1 % V]), __float_as_uint(f[2 % V]), __float_as_uint(f[3 % V]));
    if (V == 1) return make_uint4(round2<DT>(f[0], 0.0f), 0u, 0u, 0u);
    return make_uint4(round2<DT>(f[0], f[1 % V]), round2<DT>(f[2 % V], f[3 % V]), round2<DT>(f[4 % V], f[5 % V]), round2<DT>(f[6 % V], f[7 % V]));
}
template <int DT, int V> __device__ __forceinline__ void put(uint8_t* p, uint4 v) {
    if (V > 1) stg_stream_v4(p, v);
    else if (DT == ACT_DTYPE_F32) *reinterpret_cast<uint32_t*>(p) = v.x;
    else *reinterpret_cast<unsigned short*>(p) = (unsigned short)v.x;
}
// a pair turned: products and sums rounded one by one but for the fused second product
__device__ __forceinline__ void turn(float& a, float& b, float2 cs) {
    const float x = __fmaf_rn(a, cs.x, -__fmul_rn(b, cs.y)), y = __fmaf_rn(b, cs.x, __fmul_rn(a, cs.y));
    a = x; b = y;
}

// V elements per access (16 bytes, or 1 element where strides, bases or the pair count do not allow it).
// A block takes rows_per_block consecutive (b, t) rows.  Its threads are lanes x work items of a row;
// thread (l, u) walks rows l, l + lanes, ... of item u with two rows' loads in flight, the first two
// issued before the angles are computed, which hides the latency of both.
template <int DT, int V>
__global__ void __launch_bounds__(512)
rotary_kernel(const __grid_constant__ Args g)
{
    extern __shared__ __align__(16) float2 table[];          // [rows of the block][P]
    constexpr int ES = ElemT<DT>::bytes;
    const int64_t row0 = (int64_t)blockIdx.x * g.rows_per_block;
    const int n_rows = (int)(g.rows - row0 < g.rows_per_block ? g.rows - row0 : g.rows_per_block);
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
            const int per_head = p.units / p.heads;
            const int h = u / per_head, q = u - h * per_head;
            // where the item's elements lie in the head, and whether they are turned
            turned = p.rotate && (g.interleaved ? (V == 1 ? q < g.P : q * V < 2 * g.P) : q * V < g.P);
            if (!p.rotate) e0 = q * V;
            else if (g.interleaved) {
                if (V == 1) { j0 = q; e0 = turned ? 2 * q : q + g.P; e1 = turned ? 2 * q + 1 : -1; }
                else { e0 = q * V; j0 = e0 / 2; }
            } else if (turned) { e0 = j0 = q * V; e1 = g.P + e0; }
            else e0 = q * V + g.P;                            // the P / V items before these cover 2 P elements
            const int64_t b = (row0 + lane) / g.T;
            t = (int)(row0 + lane - b * g.T);
            src = p.src + ((int64_t)h * p.sh + b * p.sb + t * p.st + e0) * ES;
            dst = p.dst + ((int64_t)h * p.dh + b * p.db + t * p.dt + e0) * ES;
            s_row = p.st * ES; s_wrap = (p.sb - g.T * p.st) * ES;
            d_row = p.dt * ES; d_wrap = (p.db - g.T * p.dt) * ES;
        }
        const int e_off = (e1 - e0) * ES;
        const bool two = e1 >= 0;
        uint4 a[2], b[2];
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
        for (int i = 0; i < 2; ++i) {
            if (left > 0) {
                a[i] = fetch<DT, V>(src);
                if (two) b[i] = fetch<DT, V>(src + e_off);
                int64_t step;
                next(ts, step, s_row, s_wrap);
                src += step;
                --left;
            }
        }
        if (pass == 0) {
            for (int i = threadIdx.x; i < n_rows * g.P; i += blockDim.x) {
                const int r = i / g.P, j = i - r * g.P;
                const int64_t row = row0 + r, bb = row / g.T, tt = row - bb * g.T;
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
            for (int i = 0; i < 2; ++i) {
                if (todo <= 0) break;
                uint4 va = a[i], vb = b[i];
                if (left > 0) {
                    a[i] = fetch<DT, V>(src);
                    if (two) b[i] = fetch<DT, V>(src + e_off);
                    int64_t step;
                    next(ts, step, s_row, s_wrap);
                    src += step;
                    --left;
                }
                if (turned) {
                    float x[V], y[V];
                    widen<DT, V>(va, x);
                    if (two) {
                        widen<DT, V>(vb, y);
#pragma unroll
                        for (int k = 0; k < V; ++k) turn(x[k], y[k], cs[k]);
                        vb = narrow<DT, V>(y);
                    } else {
                        // interleaved vectors: the one that the end of the pairs cuts keeps its rest
#pragma unroll
                        for (int k = 0; k + 1 < V; k += 2)
                            if (j0 + k / 2 < g.P) turn(x[k], x[(k + 1) % V], cs[k / 2]);
                    }
                    va = narrow<DT, V>(x);
                }
                put<DT, V>(dst, va);
                if (two) put<DT, V>(dst + e_off, vb);
                int64_t step;
                next(td, step, d_row, d_wrap);
                dst += step;
                cs += lanes * g.P;
                --todo;
            }
        }
    }
}

template <int DT, int V>
cudaError_t launch(const Args& g, int blocks, int threads, int smem, cudaStream_t st) {
    rotary_kernel<DT, V><<<blocks, threads, smem, st>>>(g);
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
    const int V = 16 / es;
    // sixteen bytes at a time where every base, stride and the pair count allow it
    bool vec = Dh % V == 0 && (interleaved || P % V == 0);
    for (int s = 0; s < parts; ++s) {
        if (heads[s] == 0) continue;
        if (!srcs[s] || !dsts[s]) return ACT_ERR_NULL;
        uint64_t low = (uintptr_t)srcs[s] | (uintptr_t)dsts[s];
        if (low & (es - 1)) return ACT_ERR_ALIGN;
        for (int i = 0; i < 3; ++i) low |= (uint64_t)(src_strides[3 * s + i] * es) | (uint64_t)(dst_strides[3 * s + i] * es);
        if (low & 15) vec = false;
    }
    const int v = vec ? V : 1;
    int k = 0;
    for (int s = 0; s < parts; ++s) {
        if (heads[s] == 0) continue;
        Part& p = g.part[k++];
        p.src = static_cast<const uint8_t*>(srcs[s]);
        p.dst = static_cast<uint8_t*>(dsts[s]);
        p.sb = src_strides[3 * s]; p.sh = src_strides[3 * s + 1]; p.st = src_strides[3 * s + 2];
        p.db = dst_strides[3 * s]; p.dh = dst_strides[3 * s + 1]; p.dt = dst_strides[3 * s + 2];
        p.heads = heads[s];
        p.rotate = rotate[s] && P > 0;
        // a unit is one access, or the two of a pair (j, P + j) / (2 j, 2 j + 1)
        const bool paired = p.rotate && (!interleaved || v == 1);
        p.units = heads[s] * ((paired ? Dh - (int)P : Dh) / v);
        g.units += p.units;
    }
    for (int s = k; s < kParts; ++s) g.part[s].heads = 1;
    g.pos = pos;
    if (P > 0) { g.pb = pos_strides[0]; g.pt = pos_strides[1]; g.pa = pos_strides[2]; }
    g.turns = static_cast<const uint64_t*>(turns);
    g.rows = B * T; g.T = (int)T; g.P = (int)P;
    g.pos64 = pos_bytes == 8; g.interleaved = interleaved != 0; g.inverse = inverse != 0;

    // Blocks of up to 512 threads; a row with few work items shares its block with other rows.  A block
    // takes enough rows to make about three resident waves of blocks (2048 threads per SM), at most
    // what kTableBytes hold.
    g.lanes = g.units >= 128 ? 1 : 256 / g.units;
    if (g.lanes > g.rows) g.lanes = (int)g.rows;
    const int threads = g.units > 512 ? 512 : ((g.units * g.lanes + 31) & ~31);
    int64_t blocks = stream_grid_for(g.rows, 2048 / threads, 3);
    int64_t per = (g.rows + blocks - 1) / blocks;
    per = (per + g.lanes - 1) / g.lanes * g.lanes;
    const int64_t most = P > 0 ? kTableBytes / (8 * P) : 4096;
    if (per > most) per = most;
    blocks = (g.rows + per - 1) / per;
    if (blocks > 0x7FFFFFFF) return ACT_ERR_SIZE;
    g.rows_per_block = (int)per;
    const int smem = (int)(per * P * 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == ACT_DTYPE_F32) e = vec ? launch<ACT_DTYPE_F32, 4>(g, (int)blocks, threads, smem, st) : launch<ACT_DTYPE_F32, 1>(g, (int)blocks, threads, smem, st);
    else if (dtype == ACT_DTYPE_BF16) e = vec ? launch<ACT_DTYPE_BF16, 8>(g, (int)blocks, threads, smem, st) : launch<ACT_DTYPE_BF16, 1>(g, (int)blocks, threads, smem, st);
    else e = vec ? launch<ACT_DTYPE_F16, 8>(g, (int)blocks, threads, smem, st) : launch<ACT_DTYPE_F16, 1>(g, (int)blocks, threads, smem, st);
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
