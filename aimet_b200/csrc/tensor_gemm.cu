// Matrix products of 16-bit operands on the tensor cores: out[i, j] = act(sum_k A[i, k] B[j, k] + bias[j]) + r[i, j].
//
// Two kernels.  pair_kernel: tiles of 256 x 256 or 256 x 128 results, one pair of SMs (cta_group::2) per tile,
// persistent -- for products whose time is arithmetic.  slim_kernel: tiles of 128 columns x 16 ... 128 rows with the
// depth split over a cluster -- for few rows, where the time is reading B once, and for products too small to
// fill the GPU with large tiles.  Both read either operand as rows over k or as columns (GemmArgs), so the forward
// product and the two of the backward pass need no transposed copies.
#include <atomic>

#include "activation.cuh"
#include "kernels.h"
#include "tensor_core.cuh"

namespace aq
{
namespace
{
using namespace tc;

__device__ int g_stuck;   // raised when a bounded wait ran out; read by aq_layers_stuck

struct TcArgs
{
    const void* bias;
    const void* residual;
    void* z;
    void* out;
    int64_t ldr, ldz, ldo;
    int64_t rows, cols;
    int k_blocks;        // ceil(depth / 64)
    int act;
    uint32_t idesc;
    int a_kmajor, b_kmajor;
    int tiles_i, tiles_j;
    int vec;             // pair_kernel: elements per access of out / z / residual: 16, 8, or 0 (through shared memory)
};

constexpr int kBlockK   = 64;   // one 128-byte row of the swizzle
constexpr int kPairWarps = 8;   // epilogue warps of pair_kernel

template <int ACT, int N>
__device__ __forceinline__ void activate_as(float (&v)[N])
{
#pragma unroll
    for (int c = 0; c < N; c += 2)
        unpair(act_value2<ACT>(pair(v[c], v[c + 1])), v[c], v[c + 1]);
}
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act)
{
    switch (act)
    {
    case AQ_ACT_RELU: activate_as<AQ_ACT_RELU>(v); break;
    case AQ_ACT_GELU: activate_as<AQ_ACT_GELU>(v); break;
    case AQ_ACT_GELU_TANH: activate_as<AQ_ACT_GELU_TANH>(v); break;
    case AQ_ACT_SILU: activate_as<AQ_ACT_SILU>(v); break;
    default: break;
    }
}

// N (8 or 16) 16-bit elements as one access of 16 or 32 bytes
template <typename T, int N>
__device__ __forceinline__ void load_wide(const T* p, T (&v)[N])
{
    uint32_t w[N / 2];
    if constexpr (N == 16)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(p)
                     : "memory");
    else
        asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "l"(p)
                     : "memory");
    memcpy(v, w, sizeof w);
}
template <typename T, int N>
__device__ __forceinline__ void store_wide(T* p, const float (&f)[N])
{
    T v[N];
#pragma unroll
    for (int c = 0; c < N; ++c)
        v[c] = from_f32<T>(f[c]);
    uint32_t w[N / 2];
    memcpy(w, v, sizeof w);
    if constexpr (N == 16)
        asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "l"(p)
                     : "memory");
    else
        asm volatile("st.global.v4.b32 [%4], {%0, %1, %2, %3};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "l"(p)
                     : "memory");
}

// ------------------------------------------------------------------------------------------------------------------
// pair_kernel
// ------------------------------------------------------------------------------------------------------------------
template <int BN>
struct PairShape
{
    static constexpr int kStageBytes = 128 * 128 + BN / 2 * 128;   // a CTA's half of A and of B
    static constexpr int kStages     = BN == 256 ? 6 : 8;
    static constexpr int kPatch      = 32 * 33 * 4;                // per epilogue warp: 32 x 32 results on their way to memory
    static constexpr int kBars       = kStages * kStageBytes + kPairWarps * kPatch;
    static constexpr int kSmem       = 1024 + kBars + 256;
};

// tile number -> (row tile, column tile): bands of 8 row tiles, walked column by column, so that the tiles in flight
// share rows of A and of B in L2
__device__ __forceinline__ void tile_at(int t, int tiles_i, int tiles_j, int& ti, int& tj)
{
    const int band = t / (8 * tiles_j), in_band = t - band * 8 * tiles_j;
    const int left = tiles_i - band * 8, h = left < 8 ? left : 8;
    tj             = in_band / h;
    ti             = band * 8 + in_band - tj * h;
}

// One epilogue chunk of N columns for a thread that holds one row of them.
template <typename T, int N>
__device__ __forceinline__ void row_chunk(const TcArgs& p, const float* acc, int64_t i, int64_t j, bool row_ok)
{
    if (j >= p.cols || !row_ok)
        return;
    float f[N];
#pragma unroll
    for (int c = 0; c < N; ++c)
        f[c] = acc[c];
    if (p.bias)
    {
#pragma unroll
        for (int c = 0; c < N; ++c)
            f[c] += to_f32(((const T*) p.bias)[j + c]);
    }
    if (p.z)
        store_wide<T, N>((T*) p.z + i * p.ldz + j, f);
    activate<N>(f, p.act);
    if (p.residual)
    {
        T r[N];
        load_wide<T, N>((const T*) p.residual + i * p.ldr + j, r);
#pragma unroll
        for (int c = 0; c < N; ++c)
            f[c] += to_f32(r[c]);
    }
    store_wide<T, N>((T*) p.out + i * p.ldo + j, f);
}

// One epilogue chunk of N rows (the first `most` of them exist) for a thread that holds one column of them; z is acc.
// The residuals are fetched together: one at a time their latency is what the epilogue waits for (a 777 x 1537 result:
// 30 us against 8 us).
template <typename T, int N>
__device__ __forceinline__ void column_chunk(const TcArgs& p, float (&acc)[N], int64_t i, int most, int64_t j)
{
    T r[N];
    if (p.residual)
    {
        const T* src = (const T*) p.residual + i * p.ldr + j;
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (u < most)
                r[u] = src[u * p.ldr];
    }
    if (p.z)
    {
        T* dst = (T*) p.z + i * p.ldz + j;
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (u < most)
                dst[u * p.ldz] = from_f32<T>(acc[u]);
    }
    activate<N>(acc, p.act);
    T* dst = (T*) p.out + i * p.ldo + j;
#pragma unroll
    for (int u = 0; u < N; ++u)
        if (u < most)
            dst[u * p.ldo] = from_f32<T>(p.residual ? acc[u] + to_f32(r[u]) : acc[u]);
}

template <typename T, int BN>
__global__ void __launch_bounds__(128 + 32 * kPairWarps, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const TcArgs p)
{
    using S = PairShape<BN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int stuck_smem;
    volatile int* stuck   = &stuck_smem;
    const uint32_t base   = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars   = base + S::kBars;
    const uint32_t full   = bars, empty = full + 8 * S::kStages, tfull = empty + 8 * S::kStages, tempty = tfull + 16,
                   tmem_at = tempty + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();

    pdl_launch_dependents();
    if (threadIdx.x == 0)
    {
        stuck_smem = 0;
        for (int s = 0; s < S::kStages; ++s)
        {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b)
        {
            mbar_init(tfull + 8 * b, 1);
            mbar_init(tempty + 8 * b, 2 * kPairWarps);
        }
        mbar_init_fence();
        tma_prefetch_map(&map_a);
        tma_prefetch_map(&map_b);
    }
    if (warp == 2)
        tmem_alloc<2>(tmem_at, 2 * BN);
    tmem_fence_before();
    __syncthreads();
    cluster_sync();
    tmem_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at) : "memory");
    pdl_wait();

    const int tiles = p.tiles_i * p.tiles_j;
    const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

    if (warp == 0 && lane == 0)
    {
        // ---- producer: this CTA's 128 rows of A and BN / 2 rows of B per stage, reported to the leader's barrier ----
        int s = 0;
        uint32_t phase = 0;
        bool ok        = true;
        int used       = 0;
        for (int t = first; t < tiles && ok; t += stride)
        {
            int ti, tj;
            tile_at(t, p.tiles_i, p.tiles_j, ti, tj);
            const int i0 = ti * 256 + (int) rank * 128, j0 = tj * BN + (int) rank * (BN / 2);
            for (int kb = 0; kb < p.k_blocks; ++kb)
            {
                ok = mbar_wait(empty + 8 * s, phase ^ 1u, stuck);
                if (!ok)
                    break;
                if (rank == 0)
                    mbar_expect(full + 8 * s, 2 * S::kStageBytes);
                const uint32_t bar = map_to(full + 8 * s, 0);
                const uint32_t sa = base + s * S::kStageBytes, sb = sa + 128 * 128;
                const int k0 = kb * kBlockK;
                if (p.a_kmajor)
                    tma_load_pair(sa, &map_a, k0, i0, bar);
                else
                {
                    tma_load_pair(sa, &map_a, i0, k0, bar);
                    tma_load_pair(sa + 8192, &map_a, i0 + 64, k0, bar);
                }
                if (p.b_kmajor)
                    tma_load_pair(sb, &map_b, k0, j0, bar);
                else
                {
                    tma_load_pair(sb, &map_b, j0, k0, bar);
                    if constexpr (BN == 256)
                        tma_load_pair(sb + 8192, &map_b, j0 + 64, k0, bar);
                }
                used = used < S::kStages ? used + 1 : used;
                if (++s == S::kStages)
                {
                    s = 0;
                    phase ^= 1u;
                }
            }
        }
        // every stage in use is handed back before the CTA may end: the releases arrive in this CTA's memory
        for (int u = 0; u < used && ok; ++u)
        {
            ok = mbar_wait(empty + 8 * s, phase ^ 1u, stuck);
            if (++s == S::kStages)
            {
                s = 0;
                phase ^= 1u;
            }
        }
    }
    else if (warp == 1 && lane == 0 && rank == 0)
    {
        // ---- one thread of the leader issues the matrix instructions of both SMs ----
        int s = 0;
        uint32_t phase = 0;
        bool ok        = true;
        int n          = 0;
        const uint32_t step_a = operand_step(p.a_kmajor), step_b = operand_step(p.b_kmajor);
        for (int t = first; t < tiles && ok; t += stride, ++n)
        {
            const int buf    = n & 1;
            const uint32_t d = tmem + buf * BN;
            ok               = mbar_wait(tempty + 8 * buf, ((n >> 1) & 1) ^ 1u, stuck);
            tmem_fence_after();
            for (int kb = 0; kb < p.k_blocks && ok; ++kb)
            {
                ok = mbar_wait(full + 8 * s, phase, stuck);
                if (!ok)
                    break;
                tmem_fence_after();
                const uint32_t sa = base + s * S::kStageBytes;
                const uint64_t da = operand_desc(sa, p.a_kmajor), db = operand_desc(sa + 128 * 128, p.b_kmajor);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    mma<2>(d, da + u * step_a, db + u * step_b, p.idesc, kb > 0 || u > 0);
                mma_commit_pair(empty + 8 * s, 3);
                if (++s == S::kStages)
                {
                    s = 0;
                    phase ^= 1u;
                }
            }
            if (ok)
                mma_commit_pair(tfull + 8 * buf, 3);
        }
    }
    else if (warp >= 4)
    {
        // ---- epilogue: a warp reads its quarter of the 128 rows (lanes of tensor memory) and half of the columns ----
        const int ew = warp - 4, quarter = warp & 3, half = ew >> 2;
        float* patch = reinterpret_cast<float*>(smem_raw + (base - smem_addr(smem_raw)) + S::kStages * S::kStageBytes + ew * S::kPatch);
        const uint32_t release0 = map_to(tempty, 0);
        int n = 0;
        for (int t = first; t < tiles; t += stride, ++n)
        {
            int ti, tj;
            tile_at(t, p.tiles_i, p.tiles_j, ti, tj);
            const int buf     = n & 1;
            const bool ok     = mbar_wait(tfull + 8 * buf, (n >> 1) & 1, stuck);
            const bool poison = __any_sync(0xffffffffu, !ok);
            tmem_fence_after();
            const int64_t row0 = (int64_t) ti * 256 + rank * 128 + quarter * 32;
            const int64_t col0 = (int64_t) tj * BN + half * (BN / 2);
            for (int c0 = 0; c0 < BN / 2; c0 += 32)
            {
                uint32_t raw[32];
                tmem_load32(tmem + buf * BN + half * (BN / 2) + c0 + ((uint32_t) (quarter * 32) << 16), raw);
                tmem_load_wait();
                if (c0 + 32 == BN / 2)
                {
                    // everything this warp needs is in registers: the next tile may overwrite the accumulators
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive_cluster(release0 + 8 * buf);
                }
                float acc[32];
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    acc[c] = __uint_as_float(raw[c]);
                if (poison)
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        acc[c] = __int_as_float(0x7fffffff);
                const int64_t j = col0 + c0;
                if (p.vec == 16)
                {
                    const int64_t i = row0 + lane;
                    row_chunk<T, 16>(p, acc, i, j, i < p.rows);
                    row_chunk<T, 16>(p, acc + 16, i, j + 16, i < p.rows);
                }
                else if (p.vec == 8)
                {
                    const int64_t i = row0 + lane;
#pragma unroll
                    for (int g = 0; g < 32; g += 8)
                        row_chunk<T, 8>(p, acc + g, i, j + g, i < p.rows);
                }
                else
                {
                    // rows that no wide access fits: turn the patch in shared memory and write along the rows
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        patch[lane * 33 + c] = acc[c];
                    __syncwarp();
                    const int64_t jj = j + lane;
                    if (jj < p.cols)
                    {
                        const float bias = p.bias ? to_f32(((const T*) p.bias)[jj]) : 0.f;
                        const int most   = p.rows - row0 < 32 ? (int) (p.rows - row0) : 32;
#pragma unroll 1
                        for (int r = 0; r < most; r += 16)
                        {
                            float v[16];
#pragma unroll
                            for (int u = 0; u < 16; ++u)
                                v[u] = patch[(r + u) * 33 + lane] + bias;
                            column_chunk<T, 16>(p, v, row0 + r, most - r, jj);
                        }
                    }
                }
            }
        }
    }
    __syncwarp();
    stuck_exit(stuck, &g_stuck);
    tmem_fence_before();
    __syncthreads();
    cluster_sync();
    tmem_fence_after();
    if (warp == 2)
        tmem_free<2>(tmem, 2 * BN);
}

// ------------------------------------------------------------------------------------------------------------------
// slim_kernel: the columns (contiguous in the result) are the 128 lanes, the rows the BN columns of tensor memory, so
// that a warp writes 32 neighbouring results; CTA r of a cluster takes the r-th share of the depth.
// ------------------------------------------------------------------------------------------------------------------
template <int BN>
struct SlimShape
{
    static constexpr int kStageBytes = 128 * 128 + BN * 128;
    static constexpr int kStages     = BN == 16 ? 6 : BN == 32 ? 5 : BN == 64 ? 4 : 3;   // two CTAs per SM
    static constexpr int kBars       = kStages * kStageBytes;
    static constexpr int kSmem       = 1024 + kBars + 256;
    static constexpr int kTmemCols   = BN < 32 ? 32 : BN;
    static_assert(BN * 128 * 4 <= kBars, "the partial results of a CTA take the place of its operand tiles");
};

template <typename T, int BN>
__global__ void __launch_bounds__(192, 2)
    slim_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const TcArgs p)
{
    using S = SlimShape<BN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int stuck_smem;
    volatile int* stuck = &stuck_smem;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = base + S::kBars;
    const uint32_t full = bars, empty = full + 8 * S::kStages, tfull = empty + 8 * S::kStages, tmem_at = tfull + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t splits;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
    const uint32_t rank = cluster_rank();

    pdl_launch_dependents();
    if (threadIdx.x == 0)
    {
        stuck_smem = 0;
        for (int s = 0; s < S::kStages; ++s)
        {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        mbar_init(tfull, 1);
        mbar_init_fence();
        tma_prefetch_map(&map_a);
        tma_prefetch_map(&map_b);
    }
    if (warp == 2)
        tmem_alloc<1>(tmem_at, S::kTmemCols);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at) : "memory");
    pdl_wait();

    const int tile = blockIdx.x / splits;
    const int ti = tile / p.tiles_j, tj = tile - ti * p.tiles_j;
    const int i0 = ti * BN, j0 = tj * 128;
    const int kb0 = (int) ((int64_t) p.k_blocks * rank / splits), kb1 = (int) ((int64_t) p.k_blocks * (rank + 1) / splits);

    if (warp == 0 && lane == 0)
    {
        int s = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb)
        {
            if (!mbar_wait(empty + 8 * s, phase ^ 1u, stuck))
                break;
            mbar_expect(full + 8 * s, S::kStageBytes);
            const uint32_t sf = base + s * S::kStageBytes, sr = sf + 128 * 128;
            const int k0 = kb * kBlockK;
            if (p.b_kmajor)
                tma_load(sf, &map_b, k0, j0, full + 8 * s);
            else
            {
                tma_load(sf, &map_b, j0, k0, full + 8 * s);
                tma_load(sf + 8192, &map_b, j0 + 64, k0, full + 8 * s);
            }
            if (p.a_kmajor)
                tma_load(sr, &map_a, k0, i0, full + 8 * s);
            else
            {
#pragma unroll
                for (int u = 0; u < BN / 64; ++u)   // column operands have BN of 64 or more
                    tma_load(sr + 8192 * u, &map_a, i0 + 64 * u, k0, full + 8 * s);
            }
            if (++s == S::kStages)
            {
                s = 0;
                phase ^= 1u;
            }
        }
    }
    else if (warp == 1 && lane == 0)
    {
        int s = 0;
        uint32_t phase = 0;
        bool ok        = true;
        const uint32_t step_f = operand_step(p.b_kmajor), step_r = operand_step(p.a_kmajor);
        for (int kb = kb0; kb < kb1; ++kb)
        {
            ok = mbar_wait(full + 8 * s, phase, stuck);
            if (!ok)
                break;
            tmem_fence_after();
            const uint32_t sf = base + s * S::kStageBytes;
            const uint64_t df = operand_desc(sf, p.b_kmajor), dr = operand_desc(sf + 128 * 128, p.a_kmajor);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                mma<1>(tmem, df + u * step_f, dr + u * step_r, p.idesc, kb > kb0 || u > 0);
            mma_commit(empty + 8 * s);
            if (++s == S::kStages)
            {
                s = 0;
                phase ^= 1u;
            }
        }
        if (ok)
            mma_commit(tfull);
    }
    __syncwarp();
    float* part = reinterpret_cast<float*>(smem_raw + (base - smem_addr(smem_raw)));   // [BN][128]
    const int quarter = warp & 3, f = quarter * 32 + lane;
    const int64_t j   = (int64_t) j0 + f;
    float bias        = 0.f;
    bool poison       = false;
    if (warp >= 2)
    {
        if (p.bias && j < p.cols)
            bias = to_f32(((const T*) p.bias)[j]);
        poison = __any_sync(0xffffffffu, !mbar_wait(tfull, 0, stuck));
        tmem_fence_after();
    }
    const float bad = __int_as_float(0x7fffffff);
    const int rows  = p.rows - i0 < BN ? (int) (p.rows - i0) : BN;
    if (warp >= 2)
    {
#pragma unroll 1
        for (int c0 = 0; c0 < rows; c0 += 16)
        {
            uint32_t raw[16];
            tmem_load16(tmem + c0 + ((uint32_t) (quarter * 32) << 16), raw);
            tmem_load_wait();
            if (splits > 1)
            {
#pragma unroll
                for (int c = 0; c < 16; ++c)
                    part[(c0 + c) * 128 + f] = poison ? bad : __uint_as_float(raw[c]);
            }
            else if (j < p.cols)
            {
                float v[16];
#pragma unroll
                for (int c = 0; c < 16; ++c)
                    v[c] = (poison ? bad : __uint_as_float(raw[c])) + bias;
                column_chunk<T, 16>(p, v, i0 + c0, rows - c0, j);
            }
        }
    }
    if (splits > 1)
    {
        __syncwarp();
        cluster_sync();
        if (warp >= 2 && j < p.cols)
        {
            const int c0 = rows * (int) rank / (int) splits, c1 = rows * (int) (rank + 1) / (int) splits;
            const uint32_t mine = smem_addr(part) + f * 4;
            constexpr int AT = BN < 8 * 8 ? 4 : 8;   // rows joined at a time
#pragma unroll 1
            for (int c = c0; c < c1; c += AT)
            {
                float v[AT] = {};
                for (uint32_t r = 0; r < splits; ++r)   // always in this order: the same bits on every run
                {
                    const uint32_t from = map_to(mine + c * 512, r);
                    float w[AT];
#pragma unroll
                    for (int u = 0; u < AT; ++u)
                        w[u] = c + u < c1 ? ld_cluster(from + u * 512) : 0.f;
#pragma unroll
                    for (int u = 0; u < AT; ++u)
                        v[u] += w[u];
                }
#pragma unroll
                for (int u = 0; u < AT; ++u)
                    v[u] += bias;
                column_chunk<T, AT>(p, v, i0 + c, c1 - c, j);
            }
        }
        __syncwarp();
        cluster_sync();   // nobody leaves while its partial results may be read
    }
    stuck_exit(stuck, &g_stuck);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == 2)
        tmem_free<1>(tmem, S::kTmemCols);
}

// ------------------------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled()
{
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (EncodeTiled) f;
    }();
    return fn;
}

// Boxes of 64 columns x box_rows of a [rows, cols] matrix; what a box covers outside the matrix reads as 0.
int make_map(CUtensorMap* map, const void* base, int dtype, int64_t rows, int64_t cols, int64_t ld, int box_rows)
{
    const EncodeTiled fn = encode_tiled();
    if (!fn)
        return AQ_ERR_UNSUPPORTED;
    const cuuint64_t dims[2]    = {(cuuint64_t) cols, (cuuint64_t) rows};
    const cuuint64_t pitch[1]   = {(cuuint64_t) ld * 2};
    const cuuint32_t box[2]     = {(cuuint32_t) kBlockK, (cuuint32_t) box_rows};
    const cuuint32_t strides[2] = {1, 1};
    const CUresult r =
        fn(map, dtype == AQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base),
           dims, pitch, box, strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? AQ_OK : AQ_ERR_INVALID_ARG;
}

TcArgs tc_args(const GemmArgs& a)
{
    TcArgs p   = {};
    p.bias     = a.bias;
    p.residual = a.residual;
    p.z        = a.z;
    p.out      = a.out;
    p.ldr      = a.ldr;
    p.ldz      = a.ldz;
    p.ldo      = a.ldo;
    p.rows     = a.rows;
    p.cols     = a.cols;
    p.k_blocks = (int) ((a.depth + kBlockK - 1) / kBlockK);
    p.act      = a.act;
    p.a_kmajor = a.a_kmajor;
    p.b_kmajor = a.b_kmajor;
    return p;
}

int operand_map(CUtensorMap* map, const void* base, int64_t ld, bool kmajor, int64_t rows, int64_t depth, int tile_rows, int dtype)
{
    return kmajor ? make_map(map, base, dtype, rows, depth, ld, tile_rows) : make_map(map, base, dtype, depth, rows, ld, kBlockK);
}

// elements per access that out, z and residual (where there are any) and the number of columns allow
int wide_access(const GemmArgs& a)
{
    for (int v : {16, 8})
    {
        auto fits = [&](const void* p, int64_t ld) { return !p || ((uintptr_t) p % (2 * v) == 0 && ld % v == 0); };
        if (a.cols % v == 0 && fits(a.out, a.ldo) && fits(a.z, a.ldz) && fits(a.residual, a.ldr))
            return v;
    }
    return 0;
}

template <typename Kernel>
int launch(Kernel kernel, int64_t grid, int cluster, int threads, int smem, cudaStream_t st, const CUtensorMap& ma,
           const CUtensorMap& mb, const TcArgs& p)
{
    if (grid > 0x7fffffff)
        return AQ_ERR_TOO_LARGE;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
        e = launch_cluster(kernel, (unsigned) grid, cluster, threads, smem, st, ma, mb, p);
    note_launch();
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
}

template <typename T, int BN>
int run_pair(const GemmArgs& a, cudaStream_t st)
{
    CUtensorMap ma, mb;
    int rc = operand_map(&ma, a.a, a.lda, a.a_kmajor, a.rows, a.depth, 128, a.dtype);
    if (rc == AQ_OK)
        rc = operand_map(&mb, a.b, a.ldb, a.b_kmajor, a.cols, a.depth, BN / 2, a.dtype);
    if (rc != AQ_OK)
        return rc;
    TcArgs p   = tc_args(a);
    p.tiles_i  = (int) ((a.rows + 255) / 256);
    p.tiles_j  = (int) ((a.cols + BN - 1) / BN);
    p.idesc    = instruction_desc(a.dtype == AQ_BF16, a.a_kmajor, a.b_kmajor, 256, BN);
    p.vec      = wide_access(a);
    const int64_t tiles = (int64_t) p.tiles_i * p.tiles_j;
    if (tiles > 0x3fffffff)
        return AQ_ERR_TOO_LARGE;
    const int64_t pairs = tiles < kNumSMs / 2 ? tiles : kNumSMs / 2;
    return launch(pair_kernel<T, BN>, 2 * pairs, 2, 128 + 32 * kPairWarps, PairShape<BN>::kSmem, st, ma, mb, p);
}

template <typename T, int BN>
int run_slim(const GemmArgs& a, int splits, cudaStream_t st)
{
    CUtensorMap ma, mb;
    int rc = operand_map(&ma, a.a, a.lda, a.a_kmajor, a.rows, a.depth, BN, a.dtype);
    if (rc == AQ_OK)
        rc = operand_map(&mb, a.b, a.ldb, a.b_kmajor, a.cols, a.depth, 128, a.dtype);
    if (rc != AQ_OK)
        return rc;
    TcArgs p  = tc_args(a);
    p.tiles_i = (int) ((a.rows + BN - 1) / BN);
    p.tiles_j = (int) ((a.cols + 127) / 128);
    // the columns' operand is the instruction's A
    p.idesc = instruction_desc(a.dtype == AQ_BF16, a.b_kmajor, a.a_kmajor, 128, BN);
    return launch(slim_kernel<T, BN>, (int64_t) p.tiles_i * p.tiles_j * splits, splits, 192, SlimShape<BN>::kSmem, st, ma, mb, p);
}

// Clusters of `splits` CTAs of slim_kernel that the current device holds at once (a cluster lives inside one GPC, so this
// is less than the SMs' room divided by the cluster: 30 of the 37 that 296 CTAs by eight would be).  Asked once.
template <typename T, int BN>
int resident_clusters(int splits)
{
    static std::atomic<int> known[16][9];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16)
        dev = 0;
    int n = known[dev][splits].load(std::memory_order_relaxed);
    if (n == 0)
    {
        cudaFuncSetAttribute(slim_kernel<T, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, SlimShape<BN>::kSmem);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim            = dim3(splits);
        cfg.blockDim           = dim3(192);
        cfg.dynamicSmemBytes   = SlimShape<BN>::kSmem;
        cudaLaunchAttribute attr[1];
        attr[0].id               = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = splits;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs                = attr;
        cfg.numAttrs             = 1;
        if (cudaOccupancyMaxActiveClusters(&n, slim_kernel<T, BN>, &cfg) != cudaSuccess || n < 1)
        {
            cudaGetLastError();
            n = 2 * kNumSMs / splits;
        }
        known[dev][splits].store(n, std::memory_order_relaxed);
    }
    return n;
}

// CTAs of a cluster that share the depth, and the blocks of 64 k that the kernel's longest chain of CTAs then walks: a
// second wave costs more than a larger cluster gains (24 x 11008 -> 4096: 32 tiles by eight CTAs are two waves and 37 us,
// by seven one).  Filling the pipeline and joining the parts is worth about 8 blocks.
template <typename T, int BN>
int64_t slim_plan(int64_t tiles, int64_t k_blocks, int& splits)
{
    int64_t best = INT64_MAX;
    splits       = 1;
    for (int s = 1; s <= 8 && (s == 1 || k_blocks >= 4 * s); ++s)
    {
        const int64_t room = resident_clusters<T, BN>(s);
        const int64_t cost = (tiles + room - 1) / room * ((k_blocks + s - 1) / s + 8);
        if (cost < best)
        {
            best   = cost;
            splits = s;
        }
    }
    return best;
}

template <typename T>
int tensor_gemm_t(const GemmArgs& a, cudaStream_t st)
{
    const int64_t kb    = (a.depth + kBlockK - 1) / kBlockK;
    auto slim_tiles     = [&](int bn) { return (a.rows + bn - 1) / bn * ((a.cols + 127) / 128); };
    int splits          = 1;
    if (a.rows <= 64 && a.a_kmajor)
    {
        if (a.rows <= 16)
        {
            slim_plan<T, 16>(slim_tiles(16), kb, splits);
            return run_slim<T, 16>(a, splits, st);
        }
        if (a.rows <= 32)
        {
            slim_plan<T, 32>(slim_tiles(32), kb, splits);
            return run_slim<T, 32>(a, splits, st);
        }
        slim_plan<T, 64>(slim_tiles(64), kb, splits);
        return run_slim<T, 64>(a, splits, st);
    }
    // Estimated cycles: a stage of pair_kernel costs 512 (BN 256) or 384 (BN 128), one of slim_kernel 1024 with two CTAs on
    // the SM; the other term of pair_kernel stands for filling the pipeline and the epilogue.
    auto waves = [](int64_t n, int64_t slots) { return (n + slots - 1) / slots; };
    const int64_t rt = (a.rows + 255) / 256;
    const int64_t p256 = waves(rt * ((a.cols + 255) / 256), kNumSMs / 2) * (kb * 512 + 1500);
    const int64_t p128 = waves(rt * ((a.cols + 127) / 128), kNumSMs / 2) * (kb * 384 + 1000);
    const int64_t s128 = slim_plan<T, 128>(slim_tiles(128), kb, splits) * 1024;
    if (s128 < p256 && s128 < p128)
        return run_slim<T, 128>(a, splits, st);
    return p256 <= p128 ? run_pair<T, 256>(a, st) : run_pair<T, 128>(a, st);
}
}   // namespace

int tensor_gemm(const GemmArgs& a, cudaStream_t st)
{
    return a.dtype == AQ_F16 ? tensor_gemm_t<__half>(a, st) : tensor_gemm_t<__nv_bfloat16>(a, st);
}

int gemm_stuck(int* out)
{
    const cudaError_t e = cudaMemcpyFromSymbol(out, g_stuck, sizeof(int));
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
}

}   // namespace aq
