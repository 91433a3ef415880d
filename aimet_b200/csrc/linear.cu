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
            float y = act_value<ACT>(z);
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
// dz = dy act'(z) and the partial sums of db: a CTA of 8 warps takes 32 columns and every 8th row of its band per warp.
// ------------------------------------------------------------------------------------------------
template <typename T, int ACT>
__global__ void __launch_bounds__(256) grad_z_kernel(GradZArgs a, int64_t band_rows)
{
    __shared__ float sh[8][32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col  = (int64_t) blockIdx.x * 32 + lane;
    const int64_t row0 = (int64_t) blockIdx.y * band_rows;
    const int64_t row1 = row0 + band_rows < a.rows ? row0 + band_rows : a.rows;
    float db = 0.f;
    if (col < a.cols)
        for (int64_t row = row0 + warp; row < row1; row += 8)
        {
            const float dy = to_f32(((const T*) a.dy)[row * a.lddy + col]);
            const float dz = ACT == AQ_ACT_NONE ? dy : act_grad<ACT>(dy, to_f32(((const T*) a.z)[row * a.ldz + col]));
            if (a.dz)
                ((T*) a.dz)[row * a.lddz + col] = from_f32<T>(dz);
            db += dz;
        }
    sh[warp][lane] = db;
    __syncthreads();
    if (warp == 0 && col < a.cols && a.part)
    {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            s += sh[i][lane];
        a.part[(int64_t) blockIdx.y * a.cols + col] = s;
    }
}

template <typename T>
int grad_z_t(const GradZArgs& a, cudaStream_t st)
{
    const int64_t bands     = norm_bands(a.rows, a.cols);
    const int64_t band_rows = (a.rows + bands - 1) / bands;
    const int rc            = with_activation(a.act, [&](auto act) {
        const cudaError_t e = launch_pdl(grad_z_kernel<T, decltype(act)::value>,
                                         dim3((unsigned) ((a.cols + 31) / 32), (unsigned) bands), 256, 0, st, a, band_rows);
        note_launch();
        return e == cudaSuccess ? AQ_OK : cuda_fail(e);
    });
    if (rc != AQ_OK || !a.db)
        return rc;
    return fold_columns(a.part, bands, a.cols, a.cols, a.db, nullptr, a.dtype, st);
}

// ------------------------------------------------------------------------------------------------
// Sums over the bands: out0[c] = sum_b part[b * stride + c], out1[c] the same at column cols + c.
// ------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) fold_columns_kernel(const float* part, int64_t bands, int64_t stride, int64_t cols,
                                                           T* out0, T* out1)
{
    __shared__ float sh[8][32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = (int64_t) blockIdx.x * 32 + lane;
    T* out            = blockIdx.y ? out1 : out0;
    float s           = 0.f;
    if (out && col < cols)
        for (int64_t b = warp; b < bands; b += 8)
            s += part[b * stride + (int64_t) blockIdx.y * cols + col];
    sh[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && out && col < cols)
    {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            s += sh[i][lane];
        out[col] = from_f32<T>(s);
    }
}

template <typename T>
int fold_columns_t(const float* part, int64_t bands, int64_t stride, int64_t cols, void* out0, void* out1, cudaStream_t st)
{
    const cudaError_t e = launch_pdl(fold_columns_kernel<T>, dim3((unsigned) ((cols + 31) / 32), out1 ? 2 : 1), 256, 0, st,
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
    return norm_bands(rows, cols) * cols * (int64_t) sizeof(float);
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
