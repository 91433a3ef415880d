// Linear layers: y = act(x W^T + b) + r and the gradients
//   dz = dy act'(z),  db = sum over rows of dz,  dx = dz W,  dW = dz^T x      (dr = dy).
#include "activation.cuh"
#include "common.cuh"
#include "kernels.h"

namespace aq
{
namespace
{
// ------------------------------------------------------------------------------------------------
// out[i, j] = sum_k A[i, k] B[j, k] with float32 fused multiply-adds.  An operand is read as rows over k (KMAJOR:
// element (i, k) at i * ld + k) or as columns (element (i, k) at k * ld + i).
// ------------------------------------------------------------------------------------------------
constexpr int kTile = 64, kDepth = 16, kSimtThreads = 256;

template <typename T, bool KMAJOR>
__device__ __forceinline__ void simt_load(const T* p, int64_t ld, int64_t rows, int64_t k, int64_t row0, int64_t k0,
                                          float (*dst)[kTile + 4])
{
#pragma unroll
    for (int s = 0; s < kTile * kDepth / kSimtThreads; ++s)
    {
        const int e = s * kSimtThreads + threadIdx.x;
        const int r = KMAJOR ? e / kDepth : e % kTile;
        const int c = KMAJOR ? e % kDepth : e / kTile;
        const int64_t gr = row0 + r, gk = k0 + c;
        float v = 0.f;
        if (gr < rows && gk < k)
            v = to_f32(p[KMAJOR ? gr * ld + gk : gk * ld + gr]);
        dst[c][r] = v;
    }
}

template <typename T, bool AK, bool BK, int ACT>
__global__ void __launch_bounds__(kSimtThreads) simt_gemm_kernel(GemmArgs a)
{
    __shared__ float sa[kDepth][kTile + 4], sb[kDepth][kTile + 4];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t tiles_j = (a.cols + kTile - 1) / kTile;
    const int64_t i0 = (int64_t) (blockIdx.x / tiles_j) * kTile, j0 = (int64_t) (blockIdx.x % tiles_j) * kTile;
    const int ti = (threadIdx.x / 16) * 4, tj = (threadIdx.x % 16) * 4;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < a.depth; k0 += kDepth)
    {
        simt_load<T, AK>((const T*) a.a, a.lda, a.rows, a.depth, i0, k0, sa);
        simt_load<T, BK>((const T*) a.b, a.ldb, a.cols, a.depth, j0, k0, sb);
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kDepth; ++kk)
        {
            float av[4], bv[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
            {
                av[u] = sa[kk][ti + u];
                bv[u] = sb[kk][tj + u];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    acc[u][v] = fmaf(av[u], bv[v], acc[u][v]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v)
        {
            const int64_t i = i0 + ti + u, j = j0 + tj + v;
            if (i >= a.rows || j >= a.cols)
                continue;
            float z = acc[u][v];
            if (a.bias)
                z += to_f32(((const T*) a.bias)[j]);
            if (a.z)
                ((T*) a.z)[i * a.ldz + j] = from_f32<T>(z);
            float y = act_value<ACT, false>(z);
            if (a.residual)
                y += to_f32(((const T*) a.residual)[i * a.ldr + j]);
            ((T*) a.out)[i * a.ldo + j] = from_f32<T>(y);
        }
}

template <typename T, bool AK, bool BK>
int simt_gemm(const GemmArgs& a, cudaStream_t st)
{
    const int64_t grid = ((a.rows + kTile - 1) / kTile) * ((a.cols + kTile - 1) / kTile);
    if (grid > 0x7fffffff)
        return AQ_ERR_TOO_LARGE;
    return with_activation(a.act, [&](auto act) {
        const cudaError_t e =
            launch_pdl(simt_gemm_kernel<T, AK, BK, decltype(act)::value>, dim3((unsigned) grid), kSimtThreads, 0, st, a);
        note_launch();
        return e == cudaSuccess ? AQ_OK : cuda_fail(e);
    });
}

template <typename T>
int simt_dispatch(const GemmArgs& a, cudaStream_t st)
{
    if (a.a_kmajor && a.b_kmajor)
        return simt_gemm<T, true, true>(a, st);
    if (a.a_kmajor)
        return simt_gemm<T, true, false>(a, st);
    return simt_gemm<T, false, false>(a, st);
}

// ------------------------------------------------------------------------------------------------
// dz = dy act'(z) and the partial sums of db.  A thread owns VEC neighbouring columns, a warp 32 VEC of them, and the
// 8 warps of a CTA take the rows of its band in turn, four of them in flight per thread; the sums stay in registers
// until the band ends.  Bound by memory (dy and z in, dz out) once the slope costs few instructions: with erff and
// expf the gelu form of a bf16 16384 x 11008 layer is bound by issue.
// ------------------------------------------------------------------------------------------------
constexpr int kBandRowsAtOnce = 4;

template <typename T, int ACT, int VEC>
__global__ void __launch_bounds__(256) grad_z_kernel(GradZArgs a, int64_t band_rows)
{
    constexpr bool FAST = sizeof(T) == 2;
    __shared__ float sh[8][32 * VEC + 4];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col  = ((int64_t) blockIdx.x * 32 + lane) * VEC;
    const int64_t row0 = (int64_t) blockIdx.y * band_rows;
    const int64_t row1 = row0 + band_rows < a.rows ? row0 + band_rows : a.rows;
    float db[VEC]      = {};
    if (col < a.cols)   // VEC divides the number of columns
    {
        const T* dy = (const T*) a.dy + col;
        const T* z  = (const T*) a.z + col;
        T* dz       = (T*) a.dz + col;
        for (int64_t row = row0 + warp; row < row1; row += 8 * kBandRowsAtOnce)
        {
            Pack<T, VEC> g[kBandRowsAtOnce], h[kBandRowsAtOnce];
#pragma unroll
            for (int u = 0; u < kBandRowsAtOnce; ++u)
                if (row + 8 * u < row1)
                {
                    g[u] = load_pack<T, VEC>(dy + (row + 8 * u) * a.lddy);
                    if (ACT != AQ_ACT_NONE)
                        h[u] = load_pack<T, VEC>(z + (row + 8 * u) * a.ldz);
                }
#pragma unroll
            for (int u = 0; u < kBandRowsAtOnce; ++u)
                if (row + 8 * u < row1)
                {
                    Pack<T, VEC> o;
#pragma unroll
                    for (int c = 0; c < VEC; ++c)
                    {
                        float v = to_f32(g[u].v[c]);
                        if (ACT != AQ_ACT_NONE)
                            v = act_grad<ACT, FAST>(v, to_f32(h[u].v[c]));
                        o.v[c] = from_f32<T>(v);
                        db[c] += v;
                    }
                    if (a.dz)
                        store_pack<T, VEC>(dz + (row + 8 * u) * a.lddz, o);
                }
        }
    }
    if (!a.part)
        return;
#pragma unroll
    for (int c = 0; c < VEC; ++c)
        sh[warp][lane * VEC + c] = db[c];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * VEC; c += 256)
    {
        const int64_t out = (int64_t) blockIdx.x * 32 * VEC + c;
        if (out < a.cols)
        {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                s += sh[i][c];
            a.part[(int64_t) blockIdx.y * a.cols + out] = s;
        }
    }
}

// Bands for `ctas` column tiles: enough CTAs for 8 per SM, at least 64 rows each.
int64_t grad_bands(int64_t rows, int64_t ctas)
{
    int64_t bands      = (8 * kNumSMs + ctas - 1) / ctas;
    const int64_t most = (rows + 63) / 64;
    bands              = bands < most ? bands : most;
    return bands < 1 ? 1 : bands;
}

template <typename T, int VEC>
int grad_z_v(const GradZArgs& a, cudaStream_t st)
{
    const int64_t ctas      = (a.cols + 32 * VEC - 1) / (32 * VEC);
    const int64_t bands     = grad_bands(a.rows, ctas);
    const int64_t band_rows = (a.rows + bands - 1) / bands;
    const int rc            = with_activation(a.act, [&](auto act) {
        const cudaError_t e = launch_pdl(grad_z_kernel<T, decltype(act)::value, VEC>, dim3((unsigned) ctas, (unsigned) bands),
                                                    256, 0, st, a, band_rows);
        note_launch();
        return e == cudaSuccess ? AQ_OK : cuda_fail(e);
    });
    if (rc != AQ_OK || !a.db)
        return rc;
    return fold_columns(a.part, bands, a.cols, a.cols, a.db, nullptr, a.dtype, st);
}

template <typename T>
int grad_z_t(const GradZArgs& a, cudaStream_t st)
{
    // 16 bytes per access where every row of every matrix starts on such a boundary, else element by element
    constexpr int W = 16 / (int) sizeof(T);
    auto fits       = [&](const void* p, int64_t ld) { return !p || ((uintptr_t) p % 16 == 0 && ld % W == 0); };
    const bool wide = a.cols % W == 0 && fits(a.dy, a.lddy) && fits(a.dz, a.lddz) && (a.act == AQ_ACT_NONE || fits(a.z, a.ldz));
    return wide ? grad_z_v<T, W>(a, st) : grad_z_v<T, 1>(a, st);
}

// ------------------------------------------------------------------------------------------------
// Sums over the bands: out0[c] = sum_b part[b * stride + c], out1[c] the same at column cols + c.
// ------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(1024) fold_columns_kernel(const float* part, int64_t bands, int64_t stride, int64_t cols,
                                                            T* out0, T* out1)
{
    __shared__ float sh[32][32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = (int64_t) blockIdx.x * 32 + lane;
    T* out            = blockIdx.y ? out1 : out0;
    float s           = 0.f;
    if (out && col < cols)
#pragma unroll 4
        for (int64_t b = warp; b < bands; b += 32)
            s += part[b * stride + (int64_t) blockIdx.y * cols + col];
    sh[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && out && col < cols)
    {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i)
            s += sh[i][lane];
        out[col] = from_f32<T>(s);
    }
}

template <typename T>
int fold_columns_t(const float* part, int64_t bands, int64_t stride, int64_t cols, void* out0, void* out1, cudaStream_t st)
{
    const cudaError_t e = launch_pdl(fold_columns_kernel<T>, dim3((unsigned) ((cols + 31) / 32), out1 ? 2 : 1), 1024, 0, st,
                                     part, bands, stride, cols, (T*) out0, (T*) out1);
    note_launch();
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
}

// Row copies to a pitch the tensor cores can read from; the pad becomes 0.
template <typename T>
__global__ void __launch_bounds__(256) align_rows_kernel(const T* src, int64_t ld_src, T* dst, int64_t ld_dst, int64_t rows,
                                                         int64_t cols)
{
    pdl_launch_dependents();
    pdl_wait();
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
        for (int64_t c = threadIdx.x; c < ld_dst; c += 256)
            dst[row * ld_dst + c] = c < cols ? src[row * ld_src + c] : T(0);
}

template <typename T>
int align_rows_t(const void* src, int64_t ld_src, void* dst, int64_t ld_dst, int64_t rows, int64_t cols, cudaStream_t st)
{
    const int64_t grid  = rows < 8 * kNumSMs ? rows : 8 * kNumSMs;
    const cudaError_t e = launch_pdl(align_rows_kernel<T>, dim3((unsigned) grid), 256, 0, st, (const T*) src, ld_src, (T*) dst,
                                     ld_dst, rows, cols);
    note_launch();
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
}
}   // namespace

int align_rows(const void* src, int64_t ld_src, void* dst, int64_t ld_dst, int dtype, int64_t rows, int64_t cols,
               cudaStream_t st)
{
    if (dtype == AQ_F32)
        return align_rows_t<float>(src, ld_src, dst, ld_dst, rows, cols, st);
    return align_rows_t<uint16_t>(src, ld_src, dst, ld_dst, rows, cols, st);
}

int fold_columns(const float* part, int64_t bands, int64_t stride, int64_t cols, void* out0, void* out1, int dtype,
                 cudaStream_t st)
{
    switch (dtype)
    {
    case AQ_F32: return fold_columns_t<float>(part, bands, stride, cols, out0, out1, st);
    case AQ_F16: return fold_columns_t<__half>(part, bands, stride, cols, out0, out1, st);
    default: return fold_columns_t<__nv_bfloat16>(part, bands, stride, cols, out0, out1, st);
    }
}

int64_t grad_z_workspace_bytes(int64_t rows, int64_t cols)
{
    // the number of bands falls with the number of column tiles: the widest tiles need the most
    return grad_bands(rows, (cols + 255) / 256) * cols * (int64_t) sizeof(float);
}

int grad_z(const GradZArgs& a, cudaStream_t st)
{
    switch (a.dtype)
    {
    case AQ_F32: return grad_z_t<float>(a, st);
    case AQ_F16: return grad_z_t<__half>(a, st);
    default: return grad_z_t<__nv_bfloat16>(a, st);
    }
}

int gemm(const GemmArgs& a, cudaStream_t st)
{
    if (a.dtype == AQ_F32)
        return simt_dispatch<float>(a, st);
    if (a.depth == 0)
    {
        const cudaError_t e = cudaMemset2DAsync(a.out, (size_t) a.ldo * 2, 0, (size_t) a.cols * 2, (size_t) a.rows, st);
        return e == cudaSuccess ? AQ_OK : cuda_fail(e);
    }
    return tensor_gemm(a, st);
}

}   // namespace aq
