// Layer norm over rows of `dim` elements, forward and backward.
//
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) rstd, y = h w + b
//   g = dy w, dx = rstd (g - mean(g) - h mean(g h)), dw = sum over rows of dy h, db = sum over rows of dy
//
// The variance is the mean of squared differences from the mean (never E[x^2] - mu^2, which cancels when |mu| is large
// against the spread); every sum is float32.  All of it is bound by memory: x is read and y written once forward, x and
// dy read and dx written once backward.
#include "common.cuh"
#include "kernels.h"

namespace aq
{
namespace
{
constexpr int kLoopThreads = 256;

// Sum of one float (or two) over the CTA; every thread gets the result.  `red` holds 2 * 32 floats.
template <int THREADS>
__device__ __forceinline__ float2 block_sum2(float a, float b, float* red)
{
    constexpr int WARPS = THREADS / 32;
#pragma unroll
    for (int o = 16; o; o >>= 1)
    {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (WARPS > 1)
    {
        const int warp = threadIdx.x >> 5;
        __syncthreads();   // the previous use of `red` is over
        if ((threadIdx.x & 31) == 0)
        {
            red[warp]      = a;
            red[32 + warp] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i)
        {
            a += red[i];
            b += red[32 + i];
        }
    }
    return make_float2(a, b);
}

// Rows of any length: the CTA walks its row three times (the second and third time out of the caches).
template <typename T>
__global__ void __launch_bounds__(kLoopThreads) norm_fwd_loop_kernel(LayerNormArgs a)
{
    __shared__ float red[64];
    pdl_launch_dependents();
    pdl_wait();
    const T* w = (const T*) a.w;
    const T* b = (const T*) a.b;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x)
    {
        const T* x = (const T*) a.x + row * a.ldx;
        T* y       = (T*) a.y + row * a.dim;
        float s    = 0.f;
        for (int64_t i = threadIdx.x; i < a.dim; i += kLoopThreads)
            s += to_f32(x[i]);
        const float mu = block_sum2<kLoopThreads>(s, 0.f, red).x / (float) a.dim;
        s              = 0.f;
        for (int64_t i = threadIdx.x; i < a.dim; i += kLoopThreads)
        {
            const float d = to_f32(x[i]) - mu;
            s             = fmaf(d, d, s);
        }
        const float rstd = 1.f / sqrtf(block_sum2<kLoopThreads>(s, 0.f, red).x / (float) a.dim + a.eps);
        for (int64_t i = threadIdx.x; i < a.dim; i += kLoopThreads)
        {
            const float h = (to_f32(x[i]) - mu) * rstd;
            y[i]          = from_f32<T>(fmaf(h, w ? to_f32(w[i]) : 1.f, b ? to_f32(b[i]) : 0.f));
        }
        if (threadIdx.x == 0 && a.mean)
        {
            a.mean[row] = mu;
            a.rstd[row] = rstd;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kLoopThreads) norm_bwd_loop_kernel(LayerNormGradArgs a)
{
    __shared__ float red[64];
    pdl_launch_dependents();
    pdl_wait();
    const T* w = (const T*) a.w;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x)
    {
        const T* x       = (const T*) a.x + row * a.ldx;
        const T* dy      = (const T*) a.dy + row * a.lddy;
        T* dx            = (T*) a.dx + row * a.dim;
        const float mu   = a.mean[row];
        const float rstd = a.rstd[row];
        float sg = 0.f, sgh = 0.f;
        for (int64_t i = threadIdx.x; i < a.dim; i += kLoopThreads)
        {
            const float g = to_f32(dy[i]) * (w ? to_f32(w[i]) : 1.f);
            sg += g;
            sgh = fmaf(g, (to_f32(x[i]) - mu) * rstd, sgh);
        }
        const float2 s  = block_sum2<kLoopThreads>(sg, sgh, red);
        const float mg  = s.x / (float) a.dim;
        const float mgh = s.y / (float) a.dim;
        for (int64_t i = threadIdx.x; i < a.dim; i += kLoopThreads)
        {
            const float g = to_f32(dy[i]) * (w ? to_f32(w[i]) : 1.f);
            const float h = (to_f32(x[i]) - mu) * rstd;
            dx[i]         = from_f32<T>(rstd * (g - mg - h * mgh));
        }
    }
}

// Partial sums of dy h and dy over a band of rows: a CTA of 8 warps takes 32 columns (one per lane) and every 8th row
// of its band per warp, and writes one row of `part` [bands][2][dim].
template <typename T>
__global__ void __launch_bounds__(256) norm_param_kernel(LayerNormGradArgs a, int64_t band_rows)
{
    __shared__ float sh[2][8][32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col  = (int64_t) blockIdx.x * 32 + lane;
    const int64_t row0 = (int64_t) blockIdx.y * band_rows;
    const int64_t row1 = row0 + band_rows < a.rows ? row0 + band_rows : a.rows;
    float dw = 0.f, db = 0.f;
    if (col < a.dim)
        for (int64_t row = row0 + warp; row < row1; row += 8)
        {
            const float dy = to_f32(((const T*) a.dy)[row * a.lddy + col]);
            const float h  = (to_f32(((const T*) a.x)[row * a.ldx + col]) - a.mean[row]) * a.rstd[row];
            dw             = fmaf(dy, h, dw);
            db += dy;
        }
    sh[0][warp][lane] = dw;
    sh[1][warp][lane] = db;
    __syncthreads();
    if (warp < 2 && col < a.dim)
    {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            s += sh[warp][i][lane];
        a.part[((int64_t) blockIdx.y * 2 + warp) * a.dim + col] = s;
    }
}

template <typename T>
int norm_fwd_t(const LayerNormArgs& a, cudaStream_t st)
{
    const int64_t grid = a.rows < 8 * kNumSMs ? a.rows : 8 * kNumSMs;
    const cudaError_t e = launch_pdl(norm_fwd_loop_kernel<T>, dim3((unsigned) grid), kLoopThreads, 0, st, a);
    note_launch();
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
}

template <typename T>
int norm_bwd_t(const LayerNormGradArgs& a, cudaStream_t st)
{
    if (a.dx)
    {
        const int64_t grid = a.rows < 8 * kNumSMs ? a.rows : 8 * kNumSMs;
        const cudaError_t e = launch_pdl(norm_bwd_loop_kernel<T>, dim3((unsigned) grid), kLoopThreads, 0, st, a);
        note_launch();
        if (e != cudaSuccess)
            return cuda_fail(e);
    }
    if (a.dw || a.db)
    {
        const int64_t bands = norm_bands(a.rows, a.dim);
        const int64_t band_rows = (a.rows + bands - 1) / bands;
        const cudaError_t e = launch_pdl(norm_param_kernel<T>, dim3((unsigned) ((a.dim + 31) / 32), (unsigned) bands), 256, 0,
                                         st, a, band_rows);
        note_launch();
        if (e != cudaSuccess)
            return cuda_fail(e);
        return fold_columns(a.part, bands, 2 * a.dim, a.dim, a.dw, a.db, a.dtype, st);
    }
    return AQ_OK;
}
}   // namespace

// Bands of rows whose partial sums are joined afterwards: enough of them to fill the GPU, at least 64 rows each.
int64_t norm_bands(int64_t rows, int64_t dim)
{
    const int64_t col_ctas = (dim + 31) / 32;
    int64_t bands          = (8 * kNumSMs + col_ctas - 1) / col_ctas;
    const int64_t most     = (rows + 63) / 64;
    bands                  = bands < most ? bands : most;
    return bands < 1 ? 1 : bands;
}

int64_t norm_bwd_workspace_bytes(int64_t rows, int64_t dim)
{
    return norm_bands(rows, dim) * 2 * dim * (int64_t) sizeof(float);
}

int norm_fwd(const LayerNormArgs& a, cudaStream_t st)
{
    switch (a.dtype)
    {
    case AQ_F32: return norm_fwd_t<float>(a, st);
    case AQ_F16: return norm_fwd_t<__half>(a, st);
    default: return norm_fwd_t<__nv_bfloat16>(a, st);
    }
}

int norm_bwd(const LayerNormGradArgs& a, cudaStream_t st)
{
    switch (a.dtype)
    {
    case AQ_F32: return norm_bwd_t<float>(a, st);
    case AQ_F16: return norm_bwd_t<__half>(a, st);
    default: return norm_bwd_t<__nv_bfloat16>(a, st);
    }
}

}   // namespace aq
