// Linear layers: y = act(x W^T + b) + r and the gradients
//   dz = dy act'(z),  db = sum over rows of dz,  dx = dz W,  dW = dz^T x      (dr = dy).
#include "activation.cuh"
#include "common.cuh"
#include "kernels.h"
#include "tensor_core.cuh"

namespace aq
{
namespace
{
// ------------------------------------------------------------------------------------------------
// float32 products: out[i, j] = sum_k A[i, k] B[j, k] with fused multiply-adds, two lanes per instruction.  (The tensor
// cores would round the operands to 10 bits.)  An operand is read as rows over k (KMAJOR: element (i, k) at i * ld + k)
// or as columns (element (i, k) at k * ld + i); either way a slice of 16 k lies in shared memory as [k][row].  The
// copies are asynchronous and element-wise: they need no alignment, turn rows into columns on the way, and cost one
// instruction per 32 fused multiply-adds.
//
// TM x TN results per CTA, 8 x 16 (128 x 128) or 4 x 4 per thread; the depth can be split over a cluster,
// whose CTAs then add up their partial tiles in a fixed order through distributed shared memory.
// ------------------------------------------------------------------------------------------------
constexpr int kDepth = 16;

template <int TM, int TN>
struct SimtShape
{
    static constexpr int kM = TM == 128 ? 8 : 4, kN = TM == 128 ? 16 : 4;   // results of a thread
    static constexpr int kTx = TN / kN, kTy = TM / kM, kThreads = kTx * kTy;
    static constexpr int kPitchA = TM + 4, kPitchB = TN + 4;   // [k][row]; the pad spreads the turned copies over the banks
    static constexpr int kStages = 4;
    static constexpr int kOffB   = kDepth * kPitchA;              // floats
    static constexpr int kStage  = kOffB + kDepth * kPitchB;
    static constexpr int kSmem   = kStages * kStage * 4;
    static_assert(TM * TN * 4 <= kSmem, "the partial tile takes the place of the operands");
};

__device__ __forceinline__ void copy_async4(uint32_t dst, const float* src, bool in)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}

// Slice of TILE rows x 16 k, element (r, c) to dst + c * PITCH + r; what lies outside the matrix (rows beyond
// `rows`, k beyond `depth`) becomes 0, and the address then is the start of the slice.
template <int TILE, int PITCH, int THREADS, bool KMAJOR>
__device__ __forceinline__ void simt_load(const float* p, int64_t ld, int rows, int depth, uint32_t dst)
{
    constexpr int STEP = KMAJOR ? THREADS / kDepth : THREADS / TILE;   // rows, or k, from one copy to the next
    const int r = KMAJOR ? threadIdx.x / kDepth : threadIdx.x % TILE, c = KMAJOR ? threadIdx.x % kDepth : threadIdx.x / TILE;
    const float* src = p + (KMAJOR ? r * ld + c : c * ld + r);
    uint32_t at      = dst + (c * PITCH + r) * 4;
#pragma unroll
    for (int s = 0; s < TILE * kDepth / THREADS; ++s)
    {
        const bool in = KMAJOR ? r + s * STEP < rows && c < depth : r < rows && c + s * STEP < depth;
        copy_async4(at, in ? src : p, in);
        src += STEP * ld;
        at += STEP * (KMAJOR ? 1 : PITCH) * 4;
    }
}

template <int TM, int TN, bool AK, bool BK, int ACT>
__global__ void __launch_bounds__(SimtShape<TM, TN>::kThreads, 2) simt_gemm_kernel(GemmArgs a)
{
    using S = SimtShape<TM, TN>;
    constexpr int M = S::kM, N = S::kN;   // rows ty 4 + {0..3} (and 4 kTy further), columns alike
    extern __shared__ __align__(16) float simt_smem[];
    pdl_launch_dependents();
    uint32_t splits;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
    const uint32_t rank   = tc::cluster_rank();
    const int64_t tile    = blockIdx.x / splits;
    const int64_t tiles_j = (a.cols + TN - 1) / TN;
    const int64_t i0 = tile / tiles_j * TM, j0 = tile % tiles_j * TN;
    const int64_t slices = (a.depth + kDepth - 1) / kDepth;
    const int64_t s0 = slices * rank / splits, s1 = slices * (rank + 1) / splits;
    const float* pa = (const float*) a.a;
    const float* pb = (const float*) a.b;
    const int tx = threadIdx.x % S::kTx, ty = threadIdx.x / S::kTx;
    const uint32_t base = tc::smem_addr(simt_smem);
    const int rows_left = a.rows - i0 < TM ? (int) (a.rows - i0) : TM, cols_left = a.cols - j0 < TN ? (int) (a.cols - j0) : TN;
    auto load = [&](int64_t slice) {
        if (slice < s1)
        {
            const uint32_t dst = base + (uint32_t) ((slice - s0) % S::kStages) * S::kStage * 4;
            const int64_t k0   = slice * kDepth;
            const int left     = a.depth - k0 < kDepth ? (int) (a.depth - k0) : kDepth;
            simt_load<TM, S::kPitchA, S::kThreads, AK>(pa + (AK ? i0 * a.lda + k0 : k0 * a.lda + i0), a.lda, rows_left, left, dst);
            simt_load<TN, S::kPitchB, S::kThreads, BK>(pb + (BK ? j0 * a.ldb + k0 : k0 * a.ldb + j0), a.ldb, cols_left, left,
                                               dst + S::kOffB * 4);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    pdl_wait();
    f32x2_t acc[M][N / 2];
#pragma unroll
    for (int u = 0; u < M; ++u)
#pragma unroll
        for (int v = 0; v < N / 2; ++v)
            acc[u][v] = pair(0.f, 0.f);
    for (int s = 0; s < S::kStages - 1; ++s)
        load(s0 + s);
    for (int64_t slice = s0; slice < s1; ++slice)
    {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
        __syncthreads();   // the slice is there, and everybody is done with the one that is overwritten next
        load(slice + S::kStages - 1);
        const float* sa = simt_smem + ((slice - s0) % S::kStages) * S::kStage + ty * 4;
        const float* sb = simt_smem + ((slice - s0) % S::kStages) * S::kStage + S::kOffB + tx * 4;
#pragma unroll
        for (int kk = 0; kk < kDepth; ++kk)
        {
            float av[M];
            ulonglong2 bv[N / 4];   // the register pairs (b0, b1), (b2, b3)
#pragma unroll
            for (int h = 0; h < M / 4; ++h)
                *reinterpret_cast<float4*>(av + 4 * h) = *reinterpret_cast<const float4*>(sa + kk * S::kPitchA + 4 * S::kTy * h);
#pragma unroll
            for (int h = 0; h < N / 4; ++h)
                bv[h] = *reinterpret_cast<const ulonglong2*>(sb + kk * S::kPitchB + 4 * S::kTx * h);
#pragma unroll
            for (int u = 0; u < M; ++u)
            {
                const f32x2_t a2 = pair(av[u], av[u]);
#pragma unroll
                for (int v = 0; v < N / 2; ++v)
                    acc[u][v] = fma2(a2, v % 2 ? bv[v / 2].y : bv[v / 2].x, acc[u][v]);
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    auto finish = [&](float z, int64_t i, int64_t j) {
        if (i >= a.rows || j >= a.cols)
            return;
        if (a.bias)
            z += ((const float*) a.bias)[j];
        if (a.z)
            ((float*) a.z)[i * a.ldz + j] = z;
        float y = act_value<ACT>(z);
        if (a.residual)
            y += ((const float*) a.residual)[i * a.ldr + j];
        ((float*) a.out)[i * a.ldo + j] = y;
    };
    if (splits == 1)
    {
#pragma unroll
        for (int u = 0; u < M; ++u)
#pragma unroll
            for (int v = 0; v < N / 2; ++v)
            {
                float lo, hi;
                unpair(acc[u][v], lo, hi);
                const int64_t i = i0 + u / 4 * 4 * S::kTy + ty * 4 + u % 4, j = j0 + v / 2 * 4 * S::kTx + tx * 4 + v % 2 * 2;
                finish(lo, i, j);
                finish(hi, i, j + 1);
            }
        return;
    }
    __syncthreads();   // the operands are no longer needed
#pragma unroll
    for (int u = 0; u < M; ++u)
#pragma unroll
        for (int v = 0; v < N / 2; ++v)
        {
            float lo, hi;
            unpair(acc[u][v], lo, hi);
            float* at = simt_smem + (u / 4 * 4 * S::kTy + ty * 4 + u % 4) * TN + v / 2 * 4 * S::kTx + tx * 4 + v % 2 * 2;
            at[0]     = lo;
            at[1]     = hi;
        }
    tc::cluster_sync();
    // every CTA finishes its share of the tile, four neighbouring results per thread at a time
    constexpr int THREADS = S::kThreads, QUADS = TM * TN / 4 / THREADS, AT = 2;
    const int e0 = QUADS * (int) rank / (int) splits, e1 = QUADS * (int) (rank + 1) / (int) splits;
#pragma unroll 1
    for (int q = e0; q < e1; q += AT)
    {
        float4 z[AT];
#pragma unroll
        for (int u = 0; u < AT; ++u)
            z[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (uint32_t r = 0; r < splits; r += 4)
        {
            float4 w[4][AT];   // on their way together
#pragma unroll
            for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int u = 0; u < AT; ++u)
                    if (r + v < splits && q + u < e1)
                        w[v][u] = tc::ld_cluster4(tc::map_to(base + ((q + u) * THREADS + threadIdx.x) * 16, r + v));
#pragma unroll
            for (int v = 0; v < 4; ++v)   // always in this order: the same bits on every run
#pragma unroll
                for (int u = 0; u < AT; ++u)
                    if (r + v < splits && q + u < e1)
                    {
                        z[u].x += w[v][u].x;
                        z[u].y += w[v][u].y;
                        z[u].z += w[v][u].z;
                        z[u].w += w[v][u].w;
                    }
        }
#pragma unroll
        for (int u = 0; u < AT; ++u)
            if (q + u < e1)
            {
                const int e = ((q + u) * THREADS + threadIdx.x) * 4;
                const int64_t i = i0 + e / TN, j = j0 + e % TN;
                finish(z[u].x, i, j);
                finish(z[u].y, i, j + 1);
                finish(z[u].z, i, j + 2);
                finish(z[u].w, i, j + 3);
            }
    }
    tc::cluster_meet();   // nobody leaves while its partial tile may be read
}

template <int TM, int TN, bool AK, bool BK>
int simt_gemm(const GemmArgs& a, int splits, cudaStream_t st)
{
    const int64_t grid = ((a.rows + TM - 1) / TM) * ((a.cols + TN - 1) / TN) * splits;
    if (grid > 0x7fffffff)
        return AQ_ERR_TOO_LARGE;
    auto run = [&](auto act) -> int {
        auto kernel   = simt_gemm_kernel<TM, TN, AK, BK, decltype(act)::value>;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SimtShape<TM, TN>::kSmem);
        if (e == cudaSuccess)
            e = launch_cluster(kernel, (unsigned) grid, splits, SimtShape<TM, TN>::kThreads, SimtShape<TM, TN>::kSmem, st, a);
        note_launch();
        return e == cudaSuccess ? AQ_OK : cuda_fail(e);
    };
    if constexpr (AK && BK)
        return with_activation(a.act, run);
    else   // the backward products have no epilogue
        return run(std::integral_constant<int, AQ_ACT_NONE> {});
}

template <bool AK, bool BK>
int simt_dispatch(const GemmArgs& a, cudaStream_t st)
{
    // Two CTAs per SM.  A 128 x 128 tile costs 0.6 of what its four 64 x 64 ones do, if these CTAs fill at least half of the
    // GPU's 296 places, with the depth split where the tiles alone do not: 1024^3 56 us in 64 tiles by four, 86 us in 256
    // small ones; 512 x 4096 -> 4096 390 and 648 us; 128 x 2048 -> 1000, 8 large or 32 small tiles by eight, 37 and 26 us.
    const int64_t places = 2 * kNumSMs, slices = (a.depth + kDepth - 1) / kDepth;
    auto splits_for = [&](int64_t tiles, int64_t room) {
        const int64_t s = room / tiles < slices / 4 ? room / tiles : slices / 4;
        return s < 1 ? 1 : s > 8 ? 8 : (int) s;
    };
    const int64_t large = ((a.rows + 127) / 128) * ((a.cols + 127) / 128);
    const int splits    = splits_for(large, places);
    if (a.rows > 64 && a.cols > 64 && large * splits >= places / 2)
        return simt_gemm<128, 128, AK, BK>(a, splits, st);
    if (a.rows <= 32)   // half the products of a 64-row tile would be for rows that do not exist
        return simt_gemm<32, 128, AK, BK>(a, splits_for((a.cols + 127) / 128, 2 * places), st);
    const int64_t small = ((a.rows + 63) / 64) * ((a.cols + 63) / 64);
    return simt_gemm<64, 64, AK, BK>(a, splits_for(small, 2 * places), st);
}

int simt_any(const GemmArgs& a, cudaStream_t st)
{
    if (a.a_kmajor && a.b_kmajor)
        return simt_dispatch<true, true>(a, st);
    if (a.a_kmajor)
        return simt_dispatch<true, false>(a, st);
    return simt_dispatch<false, false>(a, st);
}

// ------------------------------------------------------------------------------------------------
// Products for at most 8 rows of A, both operands rows over k: what counts is reading B once, in whole rows.  A CTA takes
// few_b rows of B and every row of A; its four warps share the depth (2 KB of every row per step with 16-byte accesses)
// and add up in shared memory.  A comes out of L1.  No alignment is needed: VEC = 1 reads element by element.
//
// One row, 4096 -> 11008 in bf16 (90 MB, 13.8 us at the copy bandwidth): 16.8 us, against 23.4 us on the tensor cores'
// kernel for few rows, which has a pipeline to fill and parts to join between SMs; two rows 19.2 against 23.4, four 27.1
// against 23.5.  A warp per row group instead of four: 21.7 us; half the loads in flight: the same here, 17.4 against
// 16.5 us for 11008 -> 4096.
// ------------------------------------------------------------------------------------------------
constexpr int kFewRows = AQ_LINEAR_FEW_ROWS;

// rows of B per warp
template <int M>
constexpr int few_b = M <= 4 ? 4 : 2;

template <typename T, int VEC, int M>
__global__ void __launch_bounds__(128) few_rows_kernel(GemmArgs a)
{
    constexpr int kFewB = few_b<M>;
    __shared__ float sh[4][kFewB * M];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t j0 = (int64_t) blockIdx.x * kFewB;
    float sums[kFewB][M];
    if constexpr (VEC > 1)
    {
        constexpr int Q = VEC / 2, AHEAD = M == 1 ? 4 : 2, STEP = 128;   // in packets of 16 bytes
        const uint4* pb[kFewB];
        const uint4* pa[M];
#pragma unroll
        for (int r = 0; r < kFewB; ++r)
            pb[r] = reinterpret_cast<const uint4*>((const T*) a.b + (j0 + r < a.cols ? j0 + r : a.cols - 1) * a.ldb);
#pragma unroll
        for (int m = 0; m < M; ++m)
            pa[m] = reinterpret_cast<const uint4*>((const T*) a.a + (m < a.rows ? m : 0) * a.lda);
        f32x2_t acc[kFewB][M];
#pragma unroll
        for (int r = 0; r < kFewB; ++r)
#pragma unroll
            for (int m = 0; m < M; ++m)
                acc[r][m] = pair(0.f, 0.f);
        auto add = [&](const uint4 (&b)[kFewB], int at) {
            uint4 x[M];
#pragma unroll
            for (int m = 0; m < M; ++m)
                x[m] = pa[m][at];
            f32x2_t bf[kFewB][Q];
#pragma unroll
            for (int r = 0; r < kFewB; ++r)
                expand<T>(b[r], bf[r]);
#pragma unroll
            for (int m = 0; m < M; ++m)
            {
                f32x2_t af[Q];
                expand<T>(x[m], af);
#pragma unroll
                for (int r = 0; r < kFewB; ++r)
#pragma unroll
                    for (int q = 0; q < Q; ++q)
                        acc[r][m] = fma2(af[q], bf[r][q], acc[r][m]);
            }
        };
        const int packets = (int) (a.depth / VEC);
        int at            = threadIdx.x;
        for (; at + STEP * (AHEAD - 1) < packets; at += STEP * AHEAD)
        {
            uint4 b[AHEAD][kFewB];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int r = 0; r < kFewB; ++r)
                    b[u][r] = pb[r][at + u * STEP];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                add(b[u], at + u * STEP);
        }
        for (; at < packets; at += STEP)
        {
            uint4 b[kFewB];
#pragma unroll
            for (int r = 0; r < kFewB; ++r)
                b[r] = pb[r][at];
            add(b, at);
        }
#pragma unroll
        for (int r = 0; r < kFewB; ++r)
#pragma unroll
            for (int m = 0; m < M; ++m)
            {
                float lo, hi;
                unpair(acc[r][m], lo, hi);
                sums[r][m] = lo + hi;
            }
    }
    else
    {
        constexpr int AHEAD = 8, STEP = 128;
        const T* pb[kFewB];
        const T* pa[M];
#pragma unroll
        for (int r = 0; r < kFewB; ++r)
            pb[r] = (const T*) a.b + (j0 + r < a.cols ? j0 + r : a.cols - 1) * a.ldb;
#pragma unroll
        for (int m = 0; m < M; ++m)
            pa[m] = (const T*) a.a + (m < a.rows ? m : 0) * a.lda;
#pragma unroll
        for (int r = 0; r < kFewB; ++r)
#pragma unroll
            for (int m = 0; m < M; ++m)
                sums[r][m] = 0.f;
        auto add = [&](const T (&b)[kFewB], int at) {
#pragma unroll
            for (int m = 0; m < M; ++m)
            {
                const float x = to_f32(pa[m][at]);
#pragma unroll
                for (int r = 0; r < kFewB; ++r)
                    sums[r][m] = fmaf(x, to_f32(b[r]), sums[r][m]);
            }
        };
        int at = threadIdx.x;
        for (; at + STEP * (AHEAD - 1) < a.depth; at += STEP * AHEAD)
        {
            T b[AHEAD][kFewB];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int r = 0; r < kFewB; ++r)
                    b[u][r] = pb[r][at + u * STEP];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                add(b[u], at + u * STEP);
        }
        for (; at < a.depth; at += STEP)
        {
            T b[kFewB];
#pragma unroll
            for (int r = 0; r < kFewB; ++r)
                b[r] = pb[r][at];
            add(b, at);
        }
    }
    float mine = 0.f;   // lane r M + m ends up with the sum of (r, m)
#pragma unroll
    for (int r = 0; r < kFewB; ++r)
#pragma unroll
        for (int m = 0; m < M; ++m)
        {
            float s = sums[r][m];
#pragma unroll
            for (int o = 16; o; o >>= 1)
                s += __shfl_xor_sync(0xffffffffu, s, o);
            mine = lane == r * M + m ? s : mine;
        }
    if (lane < kFewB * M)
        sh[warp][lane] = mine;
    __syncthreads();
    if (warp || lane >= kFewB * M)
        return;
    mine = sh[0][lane] + sh[1][lane] + sh[2][lane] + sh[3][lane];
    const int64_t i = lane % M, j = j0 + lane / M;
    if (i >= a.rows || j >= a.cols)
        return;
    if (a.bias)
        mine += to_f32(((const T*) a.bias)[j]);
    if (a.z)
        ((T*) a.z)[i * a.ldz + j] = from_f32<T>(mine);
    float v = mine;
    switch (a.act)
    {
    case AQ_ACT_RELU: v = act_as<T, AQ_ACT_RELU>(v); break;
    case AQ_ACT_GELU: v = act_as<T, AQ_ACT_GELU>(v); break;
    case AQ_ACT_GELU_TANH: v = act_as<T, AQ_ACT_GELU_TANH>(v); break;
    case AQ_ACT_SILU: v = act_as<T, AQ_ACT_SILU>(v); break;
    default: break;
    }
    if (a.residual)
        v += to_f32(((const T*) a.residual)[i * a.ldr + j]);
    ((T*) a.out)[i * a.ldo + j] = from_f32<T>(v);
}

template <typename T, int VEC, int M>
int few_rows_m(const GemmArgs& a, cudaStream_t st)
{
    const cudaError_t e =
        launch_pdl(few_rows_kernel<T, VEC, M>, dim3((unsigned) ((a.cols + few_b<M> - 1) / few_b<M>)), 128, 0, st, a);
    note_launch();
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
}

template <typename T>
bool few_wide(const GemmArgs& a)
{
    constexpr int W = 16 / (int) sizeof(T);
    return (uintptr_t) a.a % 16 == 0 && (uintptr_t) a.b % 16 == 0 && a.depth % W == 0 && a.ldb % W == 0 &&
           (a.lda % W == 0 || a.rows == 1);
}

template <typename T>
int few_rows(const GemmArgs& a, cudaStream_t st)
{
    constexpr int W = 16 / (int) sizeof(T);
    auto by_rows = [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        return a.rows == 1 ? few_rows_m<T, VEC, 1>(a, st) :
               a.rows == 2 ? few_rows_m<T, VEC, 2>(a, st) :
               a.rows <= 4 ? few_rows_m<T, VEC, 4>(a, st) :
                             few_rows_m<T, VEC, 8>(a, st);
    };
    return few_wide<T>(a) ? by_rows(std::integral_constant<int, W> {}) : by_rows(std::integral_constant<int, 1> {});
}

// ------------------------------------------------------------------------------------------------
// dz = dy act'(z) and the partial sums of db.  A thread owns VEC neighbouring columns, a warp 32 VEC of them, and the
// 8 warps of a CTA take the rows of its band in turn, two of them in flight per thread; the sums stay in registers
// until the band ends.  Bound by memory (dy and z in, dz out) once the slope costs few instructions and registers: 16384
// x 11008 bf16 gelu 739 us element by element with erff and expf, 236 us with 27 instructions per element and 16 warps
// per SM, 165 us at the copy bandwidth.
// ------------------------------------------------------------------------------------------------
template <typename T, int ACT, int VEC>
__global__ void __launch_bounds__(256, VEC > 1 ? 4 : 2) grad_z_kernel(GradZArgs a, int64_t band_rows)
{
    __shared__ float sh[8][32 * VEC + 4];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col  = ((int64_t) blockIdx.x * 32 + lane) * VEC;
    const int64_t row0 = (int64_t) blockIdx.y * band_rows;
    const int64_t row1 = row0 + band_rows < a.rows ? row0 + band_rows : a.rows;
    const T* dy = (const T*) a.dy + col;
    const T* z  = (const T*) a.z + col;
    T* dz       = (T*) a.dz + col;
    if constexpr (VEC > 1)
    {
        constexpr int Q = VEC / 2, AT = 2;
        f32x2_t db[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q)
            db[q] = pair(0.f, 0.f);
        auto one = [&](const uint4& g, const uint4& h, int64_t row) {
            f32x2_t v[Q];
            expand<T>(g, v);
            if constexpr (ACT != AQ_ACT_NONE)
            {
                f32x2_t zz[Q];
                expand<T>(h, zz);
#pragma unroll
                for (int q = 0; q < Q; ++q)
                {
                    if constexpr (sizeof(T) == 2)
                        v[q] = act_grad2<ACT>(v[q], zz[q]);
                    else
                    {
                        float d0, d1, z0, z1;
                        unpair(v[q], d0, d1);
                        unpair(zz[q], z0, z1);
                        v[q] = pair(act_grad<ACT>(d0, z0), act_grad<ACT>(d1, z1));
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < Q; ++q)
                db[q] = add2(db[q], v[q]);
            if (a.dz)
                *reinterpret_cast<uint4*>(dz + row * a.lddz) = ACT == AQ_ACT_NONE ? g : compress<T>(v);
        };
        if (col < a.cols)   // VEC divides the number of columns
        {
            int64_t row = row0 + warp;
            for (; row + 8 * (AT - 1) < row1; row += 8 * AT)
            {
                uint4 g[AT], h[AT];
#pragma unroll
                for (int u = 0; u < AT; ++u)
                {
                    g[u] = *reinterpret_cast<const uint4*>(dy + (row + 8 * u) * a.lddy);
                    if (ACT != AQ_ACT_NONE)
                        h[u] = *reinterpret_cast<const uint4*>(z + (row + 8 * u) * a.ldz);
                }
#pragma unroll
                for (int u = 0; u < AT; ++u)
                    one(g[u], h[u], row + 8 * u);
            }
            for (; row < row1; row += 8)
                one(*reinterpret_cast<const uint4*>(dy + row * a.lddy),
                    ACT != AQ_ACT_NONE ? *reinterpret_cast<const uint4*>(z + row * a.ldz) : uint4 {}, row);
        }
#pragma unroll
        for (int q = 0; q < Q; ++q)
        {
            float lo, hi;
            unpair(db[q], lo, hi);
            sh[warp][lane * VEC + 2 * q]     = lo;
            sh[warp][lane * VEC + 2 * q + 1] = hi;
        }
    }
    else
    {
        float db = 0.f;
        if (col < a.cols)
#pragma unroll 4
            for (int64_t row = row0 + warp; row < row1; row += 8)
            {
                const float g = to_f32(dy[row * a.lddy]);
                const float v = ACT == AQ_ACT_NONE ? g : act_grad<ACT>(g, to_f32(z[row * a.ldz]));
                if (a.dz)
                    dz[row * a.lddz] = from_f32<T>(v);
                db += v;
            }
        sh[warp][lane] = db;
    }
    if (!a.part)
        return;
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

// Bands for `ctas` column tiles: whole waves of four CTAs per SM as far as that goes, at least 64 rows each.
int64_t grad_bands(int64_t rows, int64_t ctas)
{
    const int64_t wave = 4 * kNumSMs;
    int64_t bands      = wave / ctas;
    if (bands < 8)   // few bands fit into one wave: the loss at its end is smaller with two
        bands = 2 * wave / ctas;
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

// Row copies to a pitch the tensor cores can read from; the pad becomes 0.  Eight elements in flight per thread.
template <typename T>
__global__ void __launch_bounds__(256) align_rows_kernel(const T* src, int64_t ld_src, T* dst, int64_t ld_dst, int64_t rows,
                                                         int64_t cols)
{
    pdl_launch_dependents();
    pdl_wait();
    constexpr int AT = 8;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
        for (int64_t c = threadIdx.x; c < ld_dst; c += 256 * AT)
        {
            T v[AT];
#pragma unroll
            for (int u = 0; u < AT; ++u)
                v[u] = c + 256 * u < cols ? src[row * ld_src + c + 256 * u] : T(0);
#pragma unroll
            for (int u = 0; u < AT; ++u)
                if (c + 256 * u < ld_dst)
                    dst[row * ld_dst + c + 256 * u] = v[u];
        }
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
    int64_t bands = 1;
    for (int64_t width : {32, 128, 256})   // of a CTA, by type and alignment
    {
        const int64_t n = grad_bands(rows, (cols + width - 1) / width);
        bands           = n > bands ? n : bands;
    }
    return bands * cols * (int64_t) sizeof(float);
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
    if (a.rows <= kFewRows && a.a_kmajor && a.b_kmajor)
    {
        if (a.dtype == AQ_F32)
            return few_rows<float>(a, st);
        // rows that the tensor cores could read go to them from the third on
        if (a.rows <= 2 || !few_wide<__half>(a))
            return a.dtype == AQ_F16 ? few_rows<__half>(a, st) : few_rows<__nv_bfloat16>(a, st);
    }
    if (a.dtype == AQ_F32)
        return simt_any(a, st);
    if (a.depth == 0)
    {
        const cudaError_t e = cudaMemset2DAsync(a.out, (size_t) a.ldo * 2, 0, (size_t) a.cols * 2, (size_t) a.rows, st);
        return e == cudaSuccess ? AQ_OK : cuda_fail(e);
    }
    return tensor_gemm(a, st);
}

}   // namespace aq
