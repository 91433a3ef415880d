// Layer norm over rows of `dim` elements, forward and backward.
//
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) rstd, y = h w + b
//   g = dy w, dx = rstd (g - mean(g) - h mean(g h)), dw = sum over rows of dy h, db = sum over rows of dy
//
// The variance is the mean of squared differences from the mean (never E[x^2] - mu^2, which cancels when |mu| is large
// against the spread); every sum is float32.  All of it is bound by memory: x is read and y written once forward, x and
// dy read and dx written once backward.
//
// Rows that fit into the registers of 32 to 512 threads take the kernels that hold them there (one pass over memory);
// longer rows take the *_loop_* kernels, which walk a row two or three times (again out of L2), and norm_param_kernel.
#include "common.cuh"
#include "kernels.h"

namespace aq
{
namespace
{
constexpr int kLoopThreads = 256;

// Sum of two floats over the TPR threads of a row (a warp, or the whole CTA); every thread gets both.  `red` holds
// 2 * 32 floats; consecutive calls of a CTA have to use different ones (one barrier each).
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float* red)
{
#pragma unroll
    for (int o = 16; o; o >>= 1)
    {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (TPR > 32)
    {
        constexpr int WARPS = TPR / 32;
        const int warp      = threadIdx.x >> 5;
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

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> splat(float v)
{
    Pack<T, VEC> p;
#pragma unroll
    for (int c = 0; c < VEC; ++c)
        p.v[c] = from_f32<T>(v);
    return p;
}

// ------------------------------------------------------------------------------------------------------------------
// Forward, row in registers: TPR threads hold PACKS packets of VEC elements each, packet k of thread t at (k TPR + t) VEC.
// TPR = 32: four rows per CTA, one per warp.  w and b come out of L1 for every row.
// ------------------------------------------------------------------------------------------------------------------
template <typename T, int VEC, int TPR, int PACKS>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_fwd_kernel(LayerNormArgs a)
{
    constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
    __shared__ float red[2][64];
    pdl_launch_dependents();
    pdl_wait();
    const int t       = threadIdx.x % TPR;
    const int64_t row = (int64_t) blockIdx.x * ROWS + threadIdx.x / TPR;
    if (ROWS > 1 && row >= a.rows)
        return;   // whole warps, and no barrier follows
    const T* x = (const T*) a.x + row * a.ldx;
    Pack<T, VEC> v[PACKS];
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
    {
        const int64_t i = ((int64_t) k * TPR + t) * VEC;
        v[k]            = i < a.dim ? load_pack<T, VEC>(x + i) : splat<T, VEC>(0.f);
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c)
            s += to_f32(v[k].v[c]);
    const float mu = row_sum2<TPR>(s, 0.f, red[0]).x / (float) a.dim;
    s              = 0.f;
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
        if (((int64_t) k * TPR + t) * VEC < a.dim)
#pragma unroll
            for (int c = 0; c < VEC; ++c)
            {
                const float d = to_f32(v[k].v[c]) - mu;
                s             = fmaf(d, d, s);
            }
    const float rstd = 1.f / sqrtf(row_sum2<TPR>(s, 0.f, red[1]).x / (float) a.dim + a.eps);
    T* y             = (T*) a.y + row * a.dim;
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
    {
        const int64_t i = ((int64_t) k * TPR + t) * VEC;
        if (i < a.dim)
        {
            const Pack<T, VEC> w = a.w ? load_pack<T, VEC>((const T*) a.w + i) : splat<T, VEC>(1.f);
            const Pack<T, VEC> b = a.b ? load_pack<T, VEC>((const T*) a.b + i) : splat<T, VEC>(0.f);
            Pack<T, VEC> o;
#pragma unroll
            for (int c = 0; c < VEC; ++c)
                o.v[c] = from_f32<T>(fmaf((to_f32(v[k].v[c]) - mu) * rstd, to_f32(w.v[c]), to_f32(b.v[c])));
            store_pack<T, VEC>(y + i, o);
        }
    }
    if (t == 0 && a.mean)
    {
        a.mean[row] = mu;
        a.rstd[row] = rstd;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Backward, row in registers.  A thread keeps the same columns for every row its CTA takes, so the sums for dw and db
// stay in its registers; the next row is fetched while the current one is reduced.  Each CTA leaves one row of partial
// sums, part [gridDim.x][2][dim] (TPR = 32: the warps of the CTA are added up in shared memory first).
// ------------------------------------------------------------------------------------------------------------------
template <typename T, int VEC, int TPR, int PACKS>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) norm_bwd_kernel(LayerNormGradArgs a)
{
    constexpr int ROWS = TPR < 256 ? 256 / TPR : 1;
    static_assert(ROWS == 1 || TPR == 32, "a row belongs to a warp or to the CTA");
    __shared__ float red[2][64];
    __shared__ float sums[ROWS > 1 ? ROWS : 1][ROWS > 1 ? TPR * PACKS * VEC + 1 : 1];
    pdl_launch_dependents();
    pdl_wait();
    const int t          = threadIdx.x % TPR;
    const int64_t stride = (int64_t) gridDim.x * ROWS;
    const T* w           = (const T*) a.w;
    const bool params    = a.part != nullptr;
    float dw[PACKS][VEC], db[PACKS][VEC];
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
#pragma unroll
        for (int c = 0; c < VEC; ++c)
            dw[k][c] = db[k][c] = 0.f;
    Pack<T, VEC> x[PACKS], g[PACKS];
    float mu = 0.f, rstd = 0.f;
    auto fetch = [&](int64_t row) {
        mu   = a.mean[row];
        rstd = a.rstd[row];
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
        {
            const int64_t i = ((int64_t) k * TPR + t) * VEC;
            if (i < a.dim)
            {
                x[k] = load_pack<T, VEC>((const T*) a.x + row * a.ldx + i);
                g[k] = load_pack<T, VEC>((const T*) a.dy + row * a.lddy + i);
            }
            else
            {
                x[k] = splat<T, VEC>(0.f);
                g[k] = splat<T, VEC>(0.f);
            }
        }
    };
    int64_t row = (int64_t) blockIdx.x * ROWS + threadIdx.x / TPR;
    if (row < a.rows)
        fetch(row);
    for (int slot = 0; row < a.rows; row += stride, slot ^= 1)
    {
        const float m = mu, r = rstd;
        float sg = 0.f, sgh = 0.f;
        Pack<T, VEC> cx[PACKS], cg[PACKS];
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
        {
            cx[k] = x[k];
            cg[k] = g[k];
        }
        if (row + stride < a.rows)
            fetch(row + stride);
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
        {
            const int64_t i = ((int64_t) k * TPR + t) * VEC;
            if (i >= a.dim)
                continue;
            const Pack<T, VEC> wk = w ? load_pack<T, VEC>(w + i) : splat<T, VEC>(1.f);
#pragma unroll
            for (int c = 0; c < VEC; ++c)
            {
                const float dy = to_f32(cg[k].v[c]);
                const float h  = (to_f32(cx[k].v[c]) - m) * r;
                const float gw = dy * to_f32(wk.v[c]);
                dw[k][c]       = fmaf(dy, h, dw[k][c]);
                db[k][c] += dy;
                sg += gw;
                sgh = fmaf(gw, h, sgh);
            }
        }
        if (!a.dx)
            continue;
        const float2 s  = row_sum2<TPR>(sg, sgh, red[slot]);
        const float mg  = s.x / (float) a.dim;
        const float mgh = s.y / (float) a.dim;
        T* dx           = (T*) a.dx + row * a.dim;
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
        {
            const int64_t i = ((int64_t) k * TPR + t) * VEC;
            if (i >= a.dim)
                continue;
            const Pack<T, VEC> wk = w ? load_pack<T, VEC>(w + i) : splat<T, VEC>(1.f);
            Pack<T, VEC> o;
#pragma unroll
            for (int c = 0; c < VEC; ++c)
            {
                const float h = (to_f32(cx[k].v[c]) - m) * r;
                o.v[c]        = from_f32<T>(r * (to_f32(cg[k].v[c]) * to_f32(wk.v[c]) - mg - h * mgh));
            }
            store_pack<T, VEC>(dx + i, o);
        }
    }
    if (!params)
        return;
    float* part = a.part + (int64_t) blockIdx.x * 2 * a.dim;
    if constexpr (ROWS == 1)
    {
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
        {
            const int64_t i = ((int64_t) k * TPR + t) * VEC;
            if (i >= a.dim)
                continue;
#pragma unroll
            for (int c = 0; c < VEC; ++c)
            {
                part[i + c]         = dw[k][c];
                part[a.dim + i + c] = db[k][c];
            }
        }
    }
    else
    {
        const int warp = threadIdx.x / TPR;
#pragma unroll
        for (int which = 0; which < 2; ++which)
        {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < PACKS; ++k)
#pragma unroll
                for (int c = 0; c < VEC; ++c)
                    sums[warp][(k * TPR + t) * VEC + c] = which ? db[k][c] : dw[k][c];
            __syncthreads();
            for (int i = threadIdx.x; i < a.dim; i += 256)
            {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < ROWS; ++j)
                    s += sums[j][i];
                part[which * a.dim + i] = s;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Rows of any length: the CTA walks its row three times (the second and third time out of the caches).
// ------------------------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kLoopThreads) norm_fwd_loop_kernel(LayerNormArgs a)
{
    __shared__ float red[2][64];
    pdl_launch_dependents();
    pdl_wait();
    const T* w = (const T*) a.w;
    const T* b = (const T*) a.b;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x)
    {
        const T* x = (const T*) a.x + row * a.ldx;
        T* y       = (T*) a.y + row * a.dim;
        float s    = 0.f;
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < a.dim; i += kLoopThreads)
            s += to_f32(x[i]);
        const float mu = row_sum2<kLoopThreads>(s, 0.f, red[0]).x / (float) a.dim;
        s              = 0.f;
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < a.dim; i += kLoopThreads)
        {
            const float d = to_f32(x[i]) - mu;
            s             = fmaf(d, d, s);
        }
        const float rstd = 1.f / sqrtf(row_sum2<kLoopThreads>(s, 0.f, red[1]).x / (float) a.dim + a.eps);
#pragma unroll 4
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
    __shared__ float red[2][64];
    pdl_launch_dependents();
    pdl_wait();
    const T* w = (const T*) a.w;
    int slot   = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, slot ^= 1)
    {
        const T* x       = (const T*) a.x + row * a.ldx;
        const T* dy      = (const T*) a.dy + row * a.lddy;
        T* dx            = (T*) a.dx + row * a.dim;
        const float mu   = a.mean[row];
        const float rstd = a.rstd[row];
        float sg = 0.f, sgh = 0.f;
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < a.dim; i += kLoopThreads)
        {
            const float g = to_f32(dy[i]) * (w ? to_f32(w[i]) : 1.f);
            sg += g;
            sgh = fmaf(g, (to_f32(x[i]) - mu) * rstd, sgh);
        }
        const float2 s  = row_sum2<kLoopThreads>(sg, sgh, red[slot]);
        const float mg  = s.x / (float) a.dim;
        const float mgh = s.y / (float) a.dim;
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < a.dim; i += kLoopThreads)
        {
            const float g = to_f32(dy[i]) * (w ? to_f32(w[i]) : 1.f);
            const float h = (to_f32(x[i]) - mu) * rstd;
            dx[i]         = from_f32<T>(rstd * (g - mg - h * mgh));
        }
    }
}

// Partial sums of dy h and dy over a band of rows, for rows that norm_bwd_loop_kernel takes: a CTA of 8 warps takes 32
// columns (one per lane) and every 8th row of its band per warp, and writes one row of part [bands][2][dim].
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
#pragma unroll 4
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

// ------------------------------------------------------------------------------------------------------------------
// dispatch
// ------------------------------------------------------------------------------------------------------------------
// f(TPR, PACKS) for the smallest shape that holds `packets` packets, AQ_ERR_TOO_LARGE (and no call) when none does.
// MAX_PACKS bounds the registers a thread gives to its columns.
template <int MAX_PACKS, typename F>
int with_row_shape(int64_t packets, F&& f)
{
    auto go = [&](auto tpr, auto packs) { return f(tpr, packs); };
    using std::integral_constant;
#define AQ_SHAPE(TPR, PACKS)                                                                       \
    if constexpr (PACKS <= MAX_PACKS)                                                              \
        if (packets <= (TPR) * (PACKS))                                                            \
            return go(integral_constant<int, TPR> {}, integral_constant<int, PACKS> {});
    AQ_SHAPE(32, 1)
    AQ_SHAPE(32, 2)
    AQ_SHAPE(32, 4)
    AQ_SHAPE(256, 1)
    AQ_SHAPE(256, 2)
    AQ_SHAPE(256, 3)
    AQ_SHAPE(256, 4)
    AQ_SHAPE(512, 3)
    AQ_SHAPE(512, 4)
    AQ_SHAPE(512, 6)
    AQ_SHAPE(512, 8)
    AQ_SHAPE(512, 12)
    AQ_SHAPE(512, 16)
    AQ_SHAPE(512, 24)
#undef AQ_SHAPE
    return AQ_ERR_TOO_LARGE;
}

template <typename T>
bool wide_rows(const void* a, int64_t lda, const void* b, int64_t ldb, const void* w, const void* bias, const void* out,
               int64_t dim)
{
    constexpr int W = 16 / (int) sizeof(T);
    auto fits       = [&](const void* p, int64_t ld) { return !p || ((uintptr_t) p % 16 == 0 && ld % W == 0); };
    return dim % W == 0 && fits(a, lda) && fits(b, ldb) && fits(w, W) && fits(bias, W) && fits(out, dim);
}

template <typename T, int VEC>
int norm_fwd_v(const LayerNormArgs& a, cudaStream_t st)
{
    return with_row_shape<VEC == 1 ? 24 : 8>((a.dim + VEC - 1) / VEC, [&](auto tpr, auto packs) {
        constexpr int TPR = decltype(tpr)::value;
        constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
        const cudaError_t e = launch_pdl(norm_fwd_kernel<T, VEC, TPR, decltype(packs)::value>,
                                         dim3((unsigned) ((a.rows + ROWS - 1) / ROWS)), TPR < 128 ? 128 : TPR, 0, st, a);
        note_launch();
        return e == cudaSuccess ? AQ_OK : cuda_fail(e);
    });
}

template <typename T>
int norm_fwd_t(const LayerNormArgs& a, cudaStream_t st)
{
    const bool wide = wide_rows<T>(a.x, a.ldx, nullptr, 0, a.w, a.b, a.y, a.dim);
    const int rc    = wide ? norm_fwd_v<T, 16 / (int) sizeof(T)>(a, st) : norm_fwd_v<T, 1>(a, st);
    if (rc != AQ_ERR_TOO_LARGE)
        return rc;
    const int64_t grid  = a.rows < 8 * kNumSMs ? a.rows : 8 * kNumSMs;
    const cudaError_t e = launch_pdl(norm_fwd_loop_kernel<T>, dim3((unsigned) grid), kLoopThreads, 0, st, a);
    note_launch();
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
}

constexpr int kBwdCtasPerSm = 2;

template <typename T, int VEC>
int norm_bwd_v(const LayerNormGradArgs& a, cudaStream_t st)
{
    // at most 24 columns per thread (48 running sums)
    return with_row_shape<24 / VEC>((a.dim + VEC - 1) / VEC, [&](auto tpr, auto packs) {
        constexpr int TPR  = decltype(tpr)::value;
        constexpr int ROWS = TPR < 256 ? 256 / TPR : 1;
        const int64_t most = (a.rows + ROWS - 1) / ROWS;
        int64_t grid       = most < kBwdCtasPerSm * kNumSMs ? most : kBwdCtasPerSm * kNumSMs;
        grid               = grid < 1 ? 1 : grid;
        cudaError_t e = launch_pdl(norm_bwd_kernel<T, VEC, TPR, decltype(packs)::value>, dim3((unsigned) grid),
                                   TPR < 256 ? 256 : TPR, 0, st, a);
        note_launch();
        if (e != cudaSuccess)
            return cuda_fail(e);
        return a.part ? fold_columns(a.part, grid, 2 * a.dim, a.dim, a.dw, a.db, a.dtype, st) : AQ_OK;
    });
}

// Bands of rows of norm_param_kernel: enough of them to fill the GPU, at least 64 rows each.
int64_t norm_bands(int64_t rows, int64_t dim)
{
    const int64_t col_ctas = (dim + 31) / 32;
    int64_t bands          = (8 * kNumSMs + col_ctas - 1) / col_ctas;
    const int64_t most     = (rows + 63) / 64;
    bands                  = bands < most ? bands : most;
    return bands < 1 ? 1 : bands;
}

template <typename T>
int norm_bwd_t(const LayerNormGradArgs& a, cudaStream_t st)
{
    const bool wide = wide_rows<T>(a.x, a.ldx, a.dy, a.lddy, a.w, nullptr, a.dx, a.dim);
    const int rc    = wide ? norm_bwd_v<T, 16 / (int) sizeof(T)>(a, st) : norm_bwd_v<T, 1>(a, st);
    if (rc != AQ_ERR_TOO_LARGE)
        return rc;
    if (a.dx)
    {
        const int64_t grid  = a.rows < 8 * kNumSMs ? a.rows : 8 * kNumSMs;
        const cudaError_t e = launch_pdl(norm_bwd_loop_kernel<T>, dim3((unsigned) grid), kLoopThreads, 0, st, a);
        note_launch();
        if (e != cudaSuccess)
            return cuda_fail(e);
    }
    if (!a.part)
        return AQ_OK;
    const int64_t bands     = norm_bands(a.rows, a.dim);
    const int64_t band_rows = (a.rows + bands - 1) / bands;
    const cudaError_t e     = launch_pdl(norm_param_kernel<T>, dim3((unsigned) ((a.dim + 31) / 32), (unsigned) bands), 256, 0, st,
                                         a, band_rows);
    note_launch();
    if (e != cudaSuccess)
        return cuda_fail(e);
    return fold_columns(a.part, bands, 2 * a.dim, a.dim, a.dw, a.db, a.dtype, st);
}
}   // namespace

int64_t norm_bwd_workspace_bytes(int64_t rows, int64_t dim)
{
    // one row of sums per CTA of norm_bwd_kernel or per band of norm_param_kernel
    int64_t n           = rows < kBwdCtasPerSm * kNumSMs ? rows : kBwdCtasPerSm * kNumSMs;
    const int64_t bands = norm_bands(rows, dim);
    n                   = n < bands ? bands : n;
    return (n < 1 ? 1 : n) * 2 * dim * (int64_t) sizeof(float);
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
