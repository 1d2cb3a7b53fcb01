// Linear layer with bias, activation and residual in its epilogue, and its backward pass: the entry
// points, the choice of kernel, and the small kernels around linear_kernel.cuh.
//
//   act_linear_fwd:   y = f(x W^T + b) + r, and optionally f'(x W^T + b)
//   act_mul_col_sum:  dz = dy * d and db = column sums of dy * d, one pass
//   act_linear_bwd:   dx = dz W, dW = dz^T x
#include <string.h>

#include "linear_kernel.cuh"

namespace act {

int stream_grid_for(int64_t n_blocks_wanted, int blocks_per_sm, int waves = 1);   // cabi.cu

namespace linear {

// ------------------------------------------------------------------ few rows: warps per column
// For a few rows of x the product reads W once and does next to nothing else: bound by HBM (or,
// when W is small, by the launch).  Warps walk rows of W (COLS of them each, so that x is widened once
// for both) in 16-byte pieces, two bytes where rows are not aligned, several pieces in flight; x comes
// out of L1.  Where there are few columns, KS warps share each column's reduction and join their sums
// through shared memory in a fixed order.  KS is chosen so that the GPU has work for about sixteen
// warps per SM ([1, 4096] x [4096, 1024]: 10.2 us with one warp per column, 4.5 so).  One row of 768 against
// 2304 columns takes 2.9 us, against [4096, 4096] out of HBM 9.2 us (33.6 MB, floor 5.1).
constexpr int kFewWarps = 8;

template <int DT, int MB, int COLS, bool VEC>
__global__ void __launch_bounds__(kFewWarps * 32)
few_rows_kernel(const unsigned short* __restrict__ x, int64_t ld_x, const unsigned short* __restrict__ w, int64_t ld_w,
                const void* __restrict__ bias, int bias_dtype, const unsigned short* __restrict__ res, int64_t ld_res,
                int M, int N, int K, int ks_count, int kind, unsigned short* __restrict__ y, int64_t ld_y,
                unsigned short* __restrict__ d, int64_t ld_d)
{
    constexpr int V = VEC ? 8 : 1, U = COLS == 1 ? 4 : 2;     // elements per access, accesses in flight per column
    __shared__ float part[kFewWarps][COLS * MB];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ks = warp % ks_count, group = warp / ks_count, groups = kFewWarps / ks_count;
    const int64_t n0 = ((int64_t)blockIdx.x * groups + group) * COLS;
    float acc[COLS][MB];
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[c][m] = 0.0f;
    const int64_t step = (int64_t)ks_count * 32 * V;
    for (int64_t k = ((int64_t)ks * 32 + lane) * V; k < K && n0 < N; k += U * step) {     // VEC: K is a multiple of 8
        uint4 wv[U][COLS];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                wv[u][c] = make_uint4(0u, 0u, 0u, 0u);
                if (k + u * step < K && n0 + c < N) {
                    const unsigned short* at = w + (n0 + c) * ld_w + k + u * step;
                    if (VEC) wv[u][c] = ldg_stream_v4(at);
                    else wv[u][c].x = __ldg(at);
                }
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k + u * step >= K) break;
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                if (m >= M) continue;
                uint4 xv = make_uint4(0u, 0u, 0u, 0u);
                if (VEC) xv = ldg_nc_v4(x + m * ld_x + k + u * step);
                else xv.x = __ldg(x + m * ld_x + k + u * step);
                const uint32_t xu[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    const uint32_t wu[4] = {wv[u][c].x, wv[u][c].y, wv[u][c].z, wv[u][c].w};
#pragma unroll
                    for (int i = 0; i < (VEC ? 4 : 1); ++i) {
                        acc[c][m] = __fmaf_rn(widen_lo<DT>(xu[i]), widen_lo<DT>(wu[i]), acc[c][m]);
                        if (VEC) acc[c][m] = __fmaf_rn(widen_hi<DT>(xu[i]), widen_hi<DT>(wu[i]), acc[c][m]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            float a = acc[c][m];
#pragma unroll
            for (int o = 16; o; o >>= 1) a = __fadd_rn(a, __shfl_xor_sync(0xffffffffu, a, o));
            if (lane == 0) part[warp][c * MB + m] = a;
        }
    __syncthreads();
    // one thread per output of the block
    const int t = threadIdx.x;
    if (t >= groups * COLS * MB) return;
    const int g = t / (COLS * MB), cm = t - g * (COLS * MB), c = cm / MB, m = cm - c * MB;
    const int64_t n = ((int64_t)blockIdx.x * groups + g) * COLS + c;
    if (m >= M || n >= N) return;
    float z = part[g * ks_count][cm];
    for (int i = 1; i < ks_count; ++i) z = __fadd_rn(z, part[g * ks_count + i][cm]);
    if (bias) z = __fadd_rn(z, load_any(bias, n, bias_dtype));
    float yv = z, dv = 0.0f;
    switch (kind) {
        case ACT_KIND_RELU: activate<ACT_KIND_RELU, false>(z, yv, dv); break;
        case ACT_KIND_GELU: activate<ACT_KIND_GELU, true>(z, yv, dv); break;
        case ACT_KIND_SILU: activate<ACT_KIND_SILU, true>(z, yv, dv); break;
        case ACT_KIND_GELU_ERF: activate<ACT_KIND_GELU_ERF, true>(z, yv, dv); break;
        default: break;
    }
    if (res) yv = __fadd_rn(yv, widen_lo<DT>(res[m * ld_res + n]));
    y[m * ld_y + n] = (unsigned short)round_pair(yv, 0.0f, DT);
    if (d) d[m * ld_d + n] = (unsigned short)round_pair(dv, 0.0f, DT);
}

struct FewArgs {
    const unsigned short *x, *w, *res;
    const void* bias;
    unsigned short *y, *d;
    int64_t ld_x, ld_w, ld_r, ld_y, ld_d;
    int bias_dtype, M, N, K, kind;
};
template <int DT, int MB, int COLS>
void few_rows(const FewArgs& a, bool vec, int sms, cudaStream_t st) {
    const int64_t units = ((int64_t)a.N + COLS - 1) / COLS;
    int ks = 1;
    while (ks < kFewWarps && units * ks < (int64_t)sms * 16 && (int64_t)a.K > (int64_t)ks * 512) ks *= 2;
    const int64_t grid = (units * ks + kFewWarps - 1) / kFewWarps;
    if (vec) few_rows_kernel<DT, MB, COLS, true><<<(unsigned)grid, kFewWarps * 32, 0, st>>>(a.x, a.ld_x, a.w, a.ld_w, a.bias, a.bias_dtype,
                 a.res, a.ld_r, a.M, a.N, a.K, ks, a.kind, a.y, a.ld_y, a.d, a.ld_d);
    else few_rows_kernel<DT, MB, COLS, false><<<(unsigned)grid, kFewWarps * 32, 0, st>>>(a.x, a.ld_x, a.w, a.ld_w, a.bias, a.bias_dtype,
                 a.res, a.ld_r, a.M, a.N, a.K, ks, a.kind, a.y, a.ld_y, a.d, a.ld_d);
}
template <int DT> void few_rows_any(const FewArgs& a, bool vec, int sms, cudaStream_t st) {
    if (a.M == 1) few_rows<DT, 1, 1>(a, vec, sms, st);
    else if (a.M == 2) few_rows<DT, 2, 2>(a, vec, sms, st);
    else if (a.M <= 4) few_rows<DT, 4, 2>(a, vec, sms, st);
    else few_rows<DT, 8, 2>(a, vec, sms, st);
}

// Rows of 16-bit elements copied to a pitch that a bulk tensor copy can read (a multiple of 16 bytes):
// all operands of a call that need it in one launch.
struct PadJob { const unsigned short* src; unsigned short* dst; int64_t ld, ld_dst, end; int cols; };   // end: 16-byte pieces up to here
struct PadJobs { PadJob job[3]; };

__global__ void __launch_bounds__(256)
pad_rows_kernel(const __grid_constant__ PadJobs jobs)
{
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < jobs.job[2].end; i += (int64_t)gridDim.x * blockDim.x) {
        const int k = i < jobs.job[0].end ? 0 : (i < jobs.job[1].end ? 1 : 2);
        const PadJob& j = jobs.job[k];
        const int64_t at = k ? i - jobs.job[k - 1].end : i, pieces = j.ld_dst >> 3;
        const int64_t r = at >> 32 ? at / pieces : (int64_t)((uint32_t)at / (uint32_t)pieces);
        const int c = (int)(at - r * pieces) * 8;
        const unsigned short* src = j.src + r * j.ld + c;
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = c + e < j.cols ? __ldg(src + e) : 0u;
        *reinterpret_cast<uint4*>(j.dst + r * j.ld_dst + c) = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
}

// out[i, j] = sum over slices, in their order, of part[slice][i][j]
__global__ void __launch_bounds__(256)
sum_slices_kernel(const float* __restrict__ part, int64_t ld_part, int64_t plane, int slices, int64_t rows, int cols,
                  void* __restrict__ out, int64_t ld_out, int out_dtype)
{
    const int64_t vecs = ld_part >> 2;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < rows * vecs; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / vecs;
        const int c = (int)(i - r * vecs) * 4;
        const float* p = part + r * ld_part + c;
        float4 a = *reinterpret_cast<const float4*>(p);
#pragma unroll 4
        for (int s = 1; s < slices; ++s) {
            const float4 b = *reinterpret_cast<const float4*>(p + s * plane);
            a.x = __fadd_rn(a.x, b.x); a.y = __fadd_rn(a.y, b.y); a.z = __fadd_rn(a.z, b.z); a.w = __fadd_rn(a.w, b.w);
        }
        const float f[4] = {a.x, a.y, a.z, a.w};
        const int n = cols - c < 4 ? cols - c : 4;
        if (out_dtype == ACT_DTYPE_F32) {
            float* o = static_cast<float*>(out) + r * ld_out + c;
            for (int j = 0; j < n; ++j) o[j] = f[j];
        } else {
            unsigned short* o = static_cast<unsigned short*>(out) + r * ld_out + c;
            if (n == 4 && !((uintptr_t)o & 7)) {
                *reinterpret_cast<uint2*>(o) = make_uint2(round_pair(f[0], f[1], out_dtype), round_pair(f[2], f[3], out_dtype));
            } else {
                for (int j = 0; j < n; ++j) o[j] = (unsigned short)round_pair(f[j], 0.0f, out_dtype);
            }
        }
    }
}

// ------------------------------------------------------------------ dz = dy * d, db = column sums
// A thread owns V consecutive columns and walks the rows of its block's slice; the block's partial
// sums go to part[slice][N] and a second kernel adds the slices in order: no atomics, the same sums
// every time.  Bound: HBM, dy and d read once, dz written once.  bf16 [50432, 2304]: 120 us (5.8 TB/s)
// and 3.7 us for the second kernel.
constexpr int kMulThreads = 256;

// W 32-bit words (2 W elements) per access, or one element (W = 0); ROWS rows' loads in flight
template <int W>
__global__ void __launch_bounds__(kMulThreads)
mul_col_sum_kernel(const unsigned short* __restrict__ dy, const unsigned short* __restrict__ d, unsigned short* __restrict__ dz,
                   float* __restrict__ part, int64_t M, int N, int dtype, int tpr)
{
    constexpr int V = W ? 2 * W : 1, ROWS = 4;
    __shared__ float sums[kMulThreads * V];
    const int rpi = kMulThreads / tpr;                       // rows per step of the block
    const int ql = threadIdx.x % tpr, rl = threadIdx.x / tpr;
    const int64_t c = ((int64_t)blockIdx.x * tpr + ql) * V;
    const int64_t r0 = M * blockIdx.y / gridDim.y, r1 = M * (blockIdx.y + 1) / gridDim.y;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    if (rl < rpi && c < N) {
        for (int64_t r = r0 + rl; r < r1; r += ROWS * rpi) {
            if (W) {
                uint4 a[ROWS], b[ROWS];
#pragma unroll
                for (int u = 0; u < ROWS; ++u)
                    if (r + u * rpi < r1) {
                        a[u] = ldg_stream_v4(dy + (r + u * rpi) * N + c);
                        b[u] = ldg_stream_v4(d + (r + u * rpi) * N + c);
                    }
#pragma unroll
                for (int u = 0; u < ROWS; ++u) {
                    if (r + u * rpi >= r1) break;
                    const uint32_t ua[4] = {a[u].x, a[u].y, a[u].z, a[u].w}, ub[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float lo = __fmul_rn(widen16(ua[i] & 0xFFFFu, dtype), widen16(ub[i] & 0xFFFFu, dtype));
                        const float hi = __fmul_rn(widen16(ua[i] >> 16, dtype), widen16(ub[i] >> 16, dtype));
                        acc[(2 * i) % V] = __fadd_rn(acc[(2 * i) % V], lo);
                        acc[(2 * i + 1) % V] = __fadd_rn(acc[(2 * i + 1) % V], hi);
                        o[i] = round_pair(lo, hi, dtype);
                    }
                    stg_stream_v4(dz + (r + u * rpi) * N + c, make_uint4(o[0], o[1], o[2], o[3]));
                }
            } else {
                float va[ROWS], vb[ROWS];
#pragma unroll
                for (int u = 0; u < ROWS; ++u)
                    if (r + u * rpi < r1) {
                        va[u] = widen16(__ldg(dy + (r + u * rpi) * N + c), dtype);
                        vb[u] = widen16(__ldg(d + (r + u * rpi) * N + c), dtype);
                    }
#pragma unroll
                for (int u = 0; u < ROWS; ++u) {
                    if (r + u * rpi >= r1) break;
                    const float v = __fmul_rn(va[u], vb[u]);
                    acc[0] = __fadd_rn(acc[0], v);
                    dz[(r + u * rpi) * N + c] = (unsigned short)round_pair(v, 0.0f, dtype);
                }
            }
        }
    }
    if (!part) return;
#pragma unroll
    for (int j = 0; j < V; ++j) sums[threadIdx.x * V + j] = acc[j];
    __syncthreads();
    if (rl == 0 && c < N) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float a = sums[ql * V + j];
            for (int r = 1; r < rpi; ++r) a = __fadd_rn(a, sums[(r * tpr + ql) * V + j]);
            part[(int64_t)blockIdx.y * N + c + j] = a;
        }
    }
}

// out[c] = sum over s of part[s][c]: 32 columns per block, 32 threads per column
__global__ void __launch_bounds__(1024)
col_sum_slices_kernel(const float* __restrict__ part, int slices, int N, float* __restrict__ out)
{
    __shared__ float t[32][33];
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float a = 0.0f;
    if (c < N)
        for (int s = row; s < slices; s += 32) a = __fadd_rn(a, part[(int64_t)s * N + c]);
    t[row][lane] = a;
    __syncthreads();
    float v = t[lane][row];                                   // column row of this block, partial `lane`
#pragma unroll
    for (int o = 16; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0 && blockIdx.x * 32 + row < N) out[blockIdx.x * 32 + row] = v;
}

}  // namespace linear
}  // namespace act

// ------------------------------------------------------------------- host side
namespace {

using namespace act::linear;

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn() {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    return fn;
}

// [rows, cols] of 16-bit elements, pitch ld elements, box 64 columns (128 bytes) x box_rows, 128-byte swizzle
bool map_16(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, bool operand) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               operand ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_NONE,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// fp32 [planes, rows, cols], pitch ld elements, box 1 x 32 x 32
bool map_f32(CUtensorMap* map, void* base, int64_t planes, int64_t rows, int64_t cols, int64_t ld) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 4, (cuuint64_t)(ld * rows) * 4};
    const cuuint32_t box[3] = {32, 32, 1}, estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t v, int64_t m) { return ceil_div(v, m) * m; }
size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// a stored 16-bit matrix [rows, cols], rows ld elements apart
struct Mat { const void* p; int64_t ld, rows, cols; };
bool tma_ready(const Mat& m) { return !((uintptr_t)m.p & 15) && !(m.ld & 7); }
size_t pad_bytes(const Mat& m) { return tma_ready(m) ? 0 : align256((size_t)m.rows * (size_t)round_up(m.cols, 8) * 2); }

struct Plan { int variant; int slices; };

// Tile shape and split of the reduction, by a model of the time in microseconds: a start, then waves of
// (64-deep blocks of the reduction + the tile's own cost).  Measured at K = 768, N = 768 to 2304, both sides
// of each choice: [197, 768] x [768, 768] 8.2 us with pairs, 6.3 with 128 x 128 tiles, 5.7 with 128 x 64;
// [1024, 768] x [768, 2304] 8.8, 7.1, 9.4; [6304, 768] x [768, 2304] 20.2, 25.1, 39.5.
// Partial planes (the split) cost their bytes, written and read at L2's pace, and one more launch.
Plan choose(int64_t M, int64_t N, int64_t K, bool may_slice, int variant) {
    const int sms = act::stream_grid_for((int64_t)1 << 40, 1, 1);
    struct Shape { int id; int tm, tn, units; double start, per_block, per_tile; };
    const Shape shapes[3] = {{ACT_LINEAR_PAIR, 256, 256, sms / 2 < 1 ? 1 : sms / 2, 3.7, 0.27, 0.5},
                             {ACT_LINEAR_128, 128, 128, sms, 2.8, 0.225, 0.3},
                             {ACT_LINEAR_64, 128, 64, sms, 2.7, 0.18, 0.2}};
    const int64_t kb = ceil_div(K, BK);
    Plan best = {ACT_LINEAR_PAIR, 1};
    double best_cost = 1e300;
    for (const Shape& s : shapes) {
        if (variant && s.id != variant) continue;
        const int64_t tiles = ceil_div(M, s.tm) * ceil_div(N, s.tn);
        for (int sl = 1; sl <= (may_slice ? 148 : 1) && sl <= kb; ++sl) {
            // a slice is at least four blocks deep, the planes stay within 64 MB, so that they live in L2
            if (sl > 1 && ((double)sl * M * N * 4 > 64e6 || kb / sl < 4)) break;
            const double waves = (double)ceil_div(tiles * sl, s.units);
            double cost = s.start + waves * ((double)ceil_div(kb, sl) * s.per_block + s.per_tile);
            if (sl > 1) cost += 2.5 + (double)(2 * sl + 1) * M * N * 4 / 6e6;
            if (cost < best_cost) { best_cost = cost; best = {s.id, sl}; }
        }
    }
    return best;
}

// copies those of the n operands that a bulk copy cannot read into the workspace, moving ws on
int pad_rows(Mat* const* mats, int n, uint8_t*& ws, cudaStream_t st) {
    PadJobs jobs = {};
    int64_t end = 0;
    int k = 0;
    for (int i = 0; i < n; ++i) {
        Mat& m = *mats[i];
        if (tma_ready(m)) continue;
        const int64_t ld = round_up(m.cols, 8);
        end += m.rows * (ld / 8);
        jobs.job[k++] = PadJob{static_cast<const unsigned short*>(m.p), reinterpret_cast<unsigned short*>(ws), m.ld, ld, end, (int)m.cols};
        m = Mat{ws, ld, m.rows, m.cols};
        ws += align256((size_t)m.rows * (size_t)ld * 2);
    }
    if (k == 0) return ACT_OK;
    for (; k < 3; ++k) jobs.job[k].end = end;
    pad_rows_kernel<<<act::stream_grid_for(ceil_div(end, 256), 8, 4), 256, 0, st>>>(jobs);
    return cudaGetLastError() == cudaSuccess ? ACT_OK : ACT_ERR_LAUNCH;
}

// C [M, N] = A B^T in p's epilogue; a and b as stored (K-major: rows of the output index; MN-major: rows
// of the reduction index), both ready for bulk copies
int launch(const Mat& a, const Mat& b, Params& p, int variant, int kind, bool deriv, cudaStream_t st) {
    const int bm = BM, bn = variant == ACT_LINEAR_64 ? 64 : 128;         // rows staged per CTA
    Maps m;
    memset(&m, 0, sizeof(m));
    if (!map_16(&m.a, a.p, a.rows, a.cols, a.ld, p.a_mn ? BK : bm, true) ||
        !map_16(&m.b, b.p, b.rows, b.cols, b.ld, p.b_mn ? BK : bn, true)) return ACT_ERR_DEVICE;
    if (p.out_f32) {
        if (!map_f32(&m.y, p.y, p.slices, p.M, p.N, p.ld_y)) return ACT_ERR_DEVICE;
    } else if (p.tma_out) {
        if (!map_16(&m.y, p.y, p.M, p.N, p.ld_y, 32, false)) return ACT_ERR_DEVICE;
        if (deriv && !map_16(&m.d, p.d, p.M, p.N, p.ld_d, 32, false)) return ACT_ERR_DEVICE;
        if (p.has_res && !map_16(&m.r, p.res, p.M, p.N, p.ld_res, 32, false)) return ACT_ERR_DEVICE;
    }
    const int tm = variant == ACT_LINEAR_PAIR ? 256 : 128, tn = variant == ACT_LINEAR_PAIR ? 256 : bn;
    const int64_t work = ceil_div(p.M, tm) * ceil_div(p.N, tn) * p.slices;
    if (work > 0x3FFFFFFF) return ACT_ERR_SIZE;
    const int sms = act::stream_grid_for((int64_t)1 << 40, 1, 1);
    bool ok;
    if (variant == ACT_LINEAR_PAIR) {
        const int pairs = sms / 2 < 1 ? 1 : sms / 2;
        ok = launch_kernel<2, 256>(kind, deriv, m, p, 2 * (int)(work < pairs ? work : pairs), st);
    } else if (variant == ACT_LINEAR_128) {
        ok = launch_kernel<1, 128>(kind, deriv, m, p, (int)(work < sms ? work : sms), st);
    } else {
        ok = launch_kernel<1, 64>(kind, deriv, m, p, (int)(work < sms ? work : sms), st);
    }
    if (!ok) { (void)cudaGetLastError(); return ACT_ERR_LAUNCH; }
    return ACT_OK;
}

bool is_16bit(int dtype) { return dtype == ACT_DTYPE_BF16 || dtype == ACT_DTYPE_F16; }
bool tensor_ready(const void* p, int64_t ld) { return !((uintptr_t)p & 15) && !(ld & 7); }

constexpr int kFewRows = 8;
// Warps per column or tensor-core tiles.  Measured, columns / 128 x 64 tiles, us: one row [768 -> 768] 2.5 / 5.4,
// [4096 -> 1024] 4.5 / 16, [4096 -> 4096] 9.2 / 22; four rows 4.0 / 5.4, 6.1 / 16, 15 / 22; eight rows 6.2 / 5.4,
// 9.0 / 16, 24 / 22.  Above four rows only a reduction longer than the row of outputs, which leaves few
// tiles with much to do each, is better served by columns.
bool use_columns(int M, int N, int K, int variant) {
    if (variant) return variant == ACT_LINEAR_FEW_ROWS;
    return M <= 4 || (M <= kFewRows && K > N);
}
constexpr int kMostRows = 0x7FFFFC00;

}  // namespace

extern "C" size_t act_linear_fwd_workspace(const void* x, int64_t ld_x, const void* w, int64_t ld_w, int M, int N, int K, int variant)
{
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    if (use_columns(M, N, K, variant)) return 0;
    return pad_bytes(Mat{x, ld_x, M, K}) + pad_bytes(Mat{w, ld_w, N, K});
}

extern "C" int act_linear_fwd(const void* x, int64_t ld_x, const void* w, int64_t ld_w, const void* bias, int bias_dtype,
                              const void* residual, int64_t ld_r, int dtype, int M, int N, int K, int kind,
                              void* y, int64_t ld_y, void* deriv, int64_t ld_d, int variant,
                              void* workspace, size_t ws_bytes, void* stream)
{
    if (!is_16bit(dtype) || (bias && !is_16bit(bias_dtype) && bias_dtype != ACT_DTYPE_F32)) return ACT_ERR_DTYPE;
    // tile corners are 32-bit numbers
    if (M > kMostRows || N > kMostRows || K > kMostRows) return ACT_ERR_SIZE;
    if (M < 0 || N < 0 || K < 1 || ld_x < K || ld_w < K || ld_y < N || (residual && ld_r < N) || (deriv && ld_d < N)) return ACT_ERR_SIZE;
    if (kind < ACT_KIND_NONE || kind > ACT_KIND_RELU || variant < 0 || variant > ACT_LINEAR_FEW_ROWS) return ACT_ERR_UNSUPPORTED;
    if (deriv && (kind == ACT_KIND_NONE || kind == ACT_KIND_RELU)) return ACT_ERR_UNSUPPORTED;
    if (variant == ACT_LINEAR_FEW_ROWS && M > kFewRows) return ACT_ERR_UNSUPPORTED;
    if (M == 0 || N == 0) return ACT_OK;
    if (!x || !w || !y) return ACT_ERR_NULL;
    if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)y | (uintptr_t)residual | (uintptr_t)deriv) & 1) return ACT_ERR_ALIGN;
    if (bias && ((uintptr_t)bias & (bias_dtype == ACT_DTYPE_F32 ? 3 : 1))) return ACT_ERR_ALIGN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (use_columns(M, N, K, variant)) {
        const FewArgs f = {static_cast<const unsigned short*>(x), static_cast<const unsigned short*>(w),
                           static_cast<const unsigned short*>(residual), bias, static_cast<unsigned short*>(y),
                           static_cast<unsigned short*>(deriv), ld_x, ld_w, ld_r, ld_y, ld_d, bias_dtype, M, N, K, kind};
        const bool vec = !((K | ld_x | ld_w) & 7) && !(((uintptr_t)x | (uintptr_t)w) & 15);
        const int sms = act::stream_grid_for((int64_t)1 << 40, 1, 1);
        if (dtype == ACT_DTYPE_BF16) few_rows_any<ACT_DTYPE_BF16>(f, vec, sms, st);
        else few_rows_any<ACT_DTYPE_F16>(f, vec, sms, st);
        return cudaGetLastError() == cudaSuccess ? ACT_OK : ACT_ERR_LAUNCH;
    }
    Mat a = {x, ld_x, M, K}, b = {w, ld_w, N, K};
    const size_t need = pad_bytes(a) + pad_bytes(b);
    if (need && (!workspace || ws_bytes < need)) return ACT_ERR_WORKSPACE;
    if (need && ((uintptr_t)workspace & 15)) return ACT_ERR_ALIGN;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    Mat* const operands[2] = {&a, &b};
    const int rc = pad_rows(operands, 2, ws, st);
    if (rc != ACT_OK) return rc;
    Params p = {};
    p.M = M; p.N = N; p.K = K; p.slices = 1; p.dtype = dtype;
    p.bias = bias; p.bias_dtype = bias_dtype;
    p.res = residual; p.ld_res = ld_r; p.has_res = residual != nullptr;
    p.y = y; p.ld_y = ld_y; p.d = deriv; p.ld_d = ld_d;
    p.tma_out = tensor_ready(y, ld_y) && (!deriv || tensor_ready(deriv, ld_d)) && (!residual || tensor_ready(residual, ld_r));
    return launch(a, b, p, choose(M, N, K, false, variant).variant, kind, deriv != nullptr, st);
}

extern "C" size_t act_linear_bwd_workspace(const void* dz, int64_t ld_dz, const void* x, int64_t ld_x, const void* w, int64_t ld_w,
                                           int M, int N, int K, int dw_dtype, int need_dx, int need_dw, int variant)
{
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    size_t n = 0;
    if (need_dx || need_dw) n += pad_bytes(Mat{dz, ld_dz, M, N});
    if (need_dx) n += pad_bytes(Mat{w, ld_w, N, K});
    if (need_dw) {
        n += pad_bytes(Mat{x, ld_x, M, K});
        const Plan plan = choose(N, K, M, true, variant);
        if (plan.slices > 1 || dw_dtype == ACT_DTYPE_F32) n += align256((size_t)plan.slices * N * (size_t)round_up(K, 4) * 4);
    }
    return n;
}

extern "C" int act_linear_bwd(const void* dz, int64_t ld_dz, const void* x, int64_t ld_x, const void* w, int64_t ld_w, int dtype,
                              int M, int N, int K, void* dx, int64_t ld_dx, void* dw, int64_t ld_dw, int dw_dtype, int variant,
                              void* workspace, size_t ws_bytes, void* stream)
{
    if (!is_16bit(dtype) || (dw && dw_dtype != dtype && dw_dtype != ACT_DTYPE_F32)) return ACT_ERR_DTYPE;
    if (M > kMostRows || N > kMostRows || K > kMostRows) return ACT_ERR_SIZE;
    if (M < 1 || N < 1 || K < 1 || ld_dz < N || (dw && (ld_x < K || ld_dw < K)) || (dx && (ld_w < K || ld_dx < K))) return ACT_ERR_SIZE;
    if (variant < 0 || variant > ACT_LINEAR_64) return ACT_ERR_UNSUPPORTED;
    if (!dx && !dw) return ACT_OK;
    if (!dz || (dx && !w) || (dw && !x)) return ACT_ERR_NULL;
    if (((uintptr_t)dz | (uintptr_t)x | (uintptr_t)w | (uintptr_t)dx) & 1) return ACT_ERR_ALIGN;
    if (dw && ((uintptr_t)dw & (dw_dtype == ACT_DTYPE_F32 ? 3 : 1))) return ACT_ERR_ALIGN;
    const size_t need = act_linear_bwd_workspace(dz, ld_dz, x, ld_x, w, ld_w, M, N, K, dw_dtype, dx != nullptr, dw != nullptr, variant);
    if (need && (!workspace || ws_bytes < need)) return ACT_ERR_WORKSPACE;
    if (need && ((uintptr_t)workspace & 15)) return ACT_ERR_ALIGN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    Mat g = {dz, ld_dz, M, N}, wm = {w, ld_w, N, K}, xm = {x, ld_x, M, K};
    Mat* operands[3];
    int n = 0;
    operands[n++] = &g;
    if (dx) operands[n++] = &wm;
    if (dw) operands[n++] = &xm;
    int rc = pad_rows(operands, n, ws, st);
    if (rc != ACT_OK) return rc;
    if (dx) {
        // dx[m, k] = sum_n dz[m, n] W[n, k]: dz K-major, W MN-major
        Params p = {};
        p.M = M; p.N = K; p.K = N; p.b_mn = 1; p.slices = 1; p.dtype = dtype;
        p.y = dx; p.ld_y = ld_dx; p.tma_out = tensor_ready(dx, ld_dx);
        if ((rc = launch(g, wm, p, choose(M, K, N, false, variant).variant, ACT_KIND_NONE, false, st)) != ACT_OK) return rc;
    }
    if (dw) {
        // dW[n, k] = sum_m dz[m, n] x[m, k]: both MN-major, the reduction is the batch
        const Plan plan = choose(N, K, M, true, variant);
        Params p = {};
        p.M = N; p.N = K; p.K = M; p.a_mn = p.b_mn = 1; p.slices = plan.slices; p.dtype = dtype;
        const bool planes = plan.slices > 1 || dw_dtype == ACT_DTYPE_F32;
        if (planes) { p.out_f32 = 1; p.y = ws; p.ld_y = round_up(K, 4); }
        else { p.y = dw; p.ld_y = ld_dw; p.tma_out = tensor_ready(dw, ld_dw); }
        if ((rc = launch(g, xm, p, plan.variant, ACT_KIND_NONE, false, st)) != ACT_OK) return rc;
        if (planes) {
            const int64_t blocks = ceil_div((int64_t)N * (p.ld_y / 4), 256);
            sum_slices_kernel<<<act::stream_grid_for(blocks, 8, 4), 256, 0, st>>>(
                static_cast<const float*>(p.y), p.ld_y, p.ld_y * N, plan.slices, N, K, dw, ld_dw, dw_dtype);
            if (cudaGetLastError() != cudaSuccess) return ACT_ERR_LAUNCH;
        }
    }
    return ACT_OK;
}

namespace {
// slices of the rows for the column sums: about six blocks per SM
void mul_grid(int64_t M, int N, bool vec, int& tpr, int& gx, int& gy) {
    const int v = vec ? 8 : 1;
    const int64_t vecs = ceil_div(N, v);
    tpr = (int)(vecs < kMulThreads ? vecs : kMulThreads);
    gx = (int)ceil_div(vecs, tpr);
    const int rpi = kMulThreads / tpr;
    int64_t want = ceil_div(act::stream_grid_for((int64_t)1 << 40, 6, 1), gx);
    const int64_t most = ceil_div(M, (int64_t)rpi * 4);
    if (want > most) want = most;
    // up to four steps of the block: one slice, whose sums are the result, and no second launch
    if (most <= 4) want = 1;
    gy = (int)(want < 1 ? 1 : (want > 65535 ? 65535 : want));
}
bool mul_vec(const void* dy, const void* d, const void* dz, int N) {
    return !(N & 7) && !(((uintptr_t)dy | (uintptr_t)d | (uintptr_t)dz) & 15);
}
}  // namespace

extern "C" size_t act_mul_col_sum_workspace(int64_t M, int N)
{
    if (M <= 0 || N <= 0) return 0;
    int tpr, gx, gy, gy1;
    mul_grid(M, N, false, tpr, gx, gy);
    mul_grid(M, N, true, tpr, gx, gy1);
    if (gy < gy1) gy = gy1;
    return gy == 1 ? 0 : (size_t)gy * (size_t)N * 4;
}

extern "C" int act_mul_col_sum(const void* dy, const void* d, int dtype, int64_t M, int N, void* dz, float* db,
                               void* workspace, size_t ws_bytes, void* stream)
{
    if (!is_16bit(dtype)) return ACT_ERR_DTYPE;
    if (M < 0 || N < 0) return ACT_ERR_SIZE;
    if (N == 0) return ACT_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (M == 0) {
        if (!db) return ACT_OK;
        return cudaMemsetAsync(db, 0, (size_t)N * 4, st) == cudaSuccess ? ACT_OK : ACT_ERR_LAUNCH;
    }
    if (!dy || !d || !dz) return ACT_ERR_NULL;
    if (((uintptr_t)dy | (uintptr_t)d | (uintptr_t)dz) & 1) return ACT_ERR_ALIGN;
    if (((uintptr_t)db | (db ? (uintptr_t)workspace : 0)) & 3) return ACT_ERR_ALIGN;
    const size_t need = db ? act_mul_col_sum_workspace(M, N) : 0;
    if (need && (!workspace || ws_bytes < need)) return ACT_ERR_WORKSPACE;
    const bool vec = mul_vec(dy, d, dz, N);
    int tpr, gx, gy;
    mul_grid(M, N, vec, tpr, gx, gy);
    const auto* a = static_cast<const unsigned short*>(dy);
    const auto* b = static_cast<const unsigned short*>(d);
    auto* o = static_cast<unsigned short*>(dz);
    float* part = !db ? nullptr : (gy == 1 ? db : static_cast<float*>(workspace));
    const dim3 grid((unsigned)gx, (unsigned)gy);
    if (vec) mul_col_sum_kernel<4><<<grid, kMulThreads, 0, st>>>(a, b, o, part, M, N, dtype, tpr);
    else mul_col_sum_kernel<0><<<grid, kMulThreads, 0, st>>>(a, b, o, part, M, N, dtype, tpr);
    if (cudaGetLastError() != cudaSuccess) return ACT_ERR_LAUNCH;
    if (db && gy > 1) {
        col_sum_slices_kernel<<<(unsigned)ceil_div(N, 32), 1024, 0, st>>>(part, gy, N, db);
        if (cudaGetLastError() != cudaSuccess) return ACT_ERR_LAUNCH;
    }
    return ACT_OK;
}

extern "C" int act_linear_status(unsigned int* out, int clear)
{
    if (!out) return ACT_ERR_NULL;
    unsigned int e[3] = {0, 0, 0};
    if (!kernel_error<2, 256>(&e[0], clear != 0) || !kernel_error<1, 128>(&e[1], clear != 0) || !kernel_error<1, 64>(&e[2], clear != 0))
        return ACT_ERR_DEVICE;
    *out = e[0] ? e[0] : (e[1] ? e[1] : e[2]);
    return ACT_OK;
}
