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
    int vec;             // elements per access that out, z and residual allow: 16, 8, or 0
    int stages;          // slim_kernel
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

// 16 neighbouring elements as float32 lanes.  `wide`: one access of 32 bytes, else two of 16, of which the second only if
// `all` 16 exist.
template <typename T>
__device__ __forceinline__ void load16(const T* p, f32x2_t (&f)[8], bool wide, bool all)
{
    uint4 lo, hi = make_uint4(0, 0, 0, 0);
    if (wide)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w), "=r"(hi.x), "=r"(hi.y), "=r"(hi.z), "=r"(hi.w)
                     : "l"(p));
    else
    {
        lo = *reinterpret_cast<const uint4*>(p);
        if (all)
            hi = *reinterpret_cast<const uint4*>(p + 8);
    }
    expand<T>(lo, reinterpret_cast<f32x2_t(&)[4]>(f[0]));
    expand<T>(hi, reinterpret_cast<f32x2_t(&)[4]>(f[4]));
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const f32x2_t (&f)[8], bool wide, bool all)
{
    const uint4 lo = compress<T>(reinterpret_cast<const f32x2_t(&)[4]>(f[0]));
    const uint4 hi = compress<T>(reinterpret_cast<const f32x2_t(&)[4]>(f[4]));
    if (wide)
        asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(lo.x), "r"(lo.y), "r"(lo.z), "r"(lo.w),
                     "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w), "l"(p)
                     : "memory");
    else
    {
        *reinterpret_cast<uint4*>(p) = lo;
        if (all)
            *reinterpret_cast<uint4*>(p + 8) = hi;
    }
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

// 16 columns from j of row i, which the thread holds; rows start on 16-byte boundaries everywhere (32 when `wide`).
template <typename T, int ACT>
__device__ __forceinline__ void row_chunk(const TcArgs& p, f32x2_t (&v)[8], int64_t i, int64_t j, bool wide)
{
    const bool all = j + 16 <= p.cols;   // the number of columns is a multiple of 8
    f32x2_t r[8];
    if (p.residual)
        load16<T>((const T*) p.residual + i * p.ldr + j, r, wide, all);
    if (p.bias)
    {
        const T* b = (const T*) p.bias + j;
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (q < 4 || all)
                v[q] = add2(v[q], pair(to_f32(b[2 * q]), to_f32(b[2 * q + 1])));
    }
    if (p.z)
        store16<T>((T*) p.z + i * p.ldz + j, v, wide, all);
    if constexpr (ACT != AQ_ACT_NONE)
    {
#pragma unroll
        for (int q = 0; q < 8; ++q)
            v[q] = act_value2<ACT>(v[q]);
    }
    if (p.residual)
    {
#pragma unroll
        for (int q = 0; q < 8; ++q)
            v[q] = add2(v[q], r[q]);
    }
    store16<T>((T*) p.out + i * p.ldo + j, v, wide, all);
}

// One epilogue chunk of N rows (the first `most` of them exist) for a thread that holds one column of them; z is acc.
// ACT = -1: the activation comes with the arguments.
// The residuals are fetched together: one at a time their latency is what the epilogue waits for (a 777 x 1537 result:
// 30 us against 8 us).
template <typename T, int N, int ACT = -1>
__device__ __forceinline__ void column_chunk(const TcArgs& p, float (&acc)[N], int64_t i, int most, int64_t j)
{
    T r[N];
    if (p.residual)
    {
        const T* src = (const T*) p.residual + i * p.ldr + j;
#pragma unroll
        for (int u = 0; u < N; ++u, src += p.ldr)
            if (u < most)
                r[u] = *src;
    }
    if (p.z)
    {
        T* dst = (T*) p.z + i * p.ldz + j;
#pragma unroll
        for (int u = 0; u < N; ++u, dst += p.ldz)
            if (u < most)
                *dst = from_f32<T>(acc[u]);
    }
    if constexpr (ACT < 0)
        activate<N>(acc, p.act);
    else if constexpr (ACT != AQ_ACT_NONE)
        activate_as<ACT, N>(acc);
    T* dst = (T*) p.out + i * p.ldo + j;
#pragma unroll
    for (int u = 0; u < N; ++u, dst += p.ldo)
        if (u < most)
            *dst = from_f32<T>(p.residual ? acc[u] + to_f32(r[u]) : acc[u]);
}

// A warp's 32 x 32 patch of z without bias in shared memory, [row][33], to rows that no wide access fits.  Not inlined: its
// addresses would push the registers of the other path out to memory.
template <typename T, int ACT>
__device__ __noinline__ void write_patch(const TcArgs& p, const float* patch, int64_t row0, int64_t j)
{
    const int lane = threadIdx.x & 31;
    j += lane;
    if (j >= p.cols)
        return;
    const float bias = p.bias ? to_f32(((const T*) p.bias)[j]) : 0.f;
    const int most   = p.rows - row0 < 32 ? (int) (p.rows - row0) : 32;
#pragma unroll 1
    for (int r = 0; r < most; r += 16)
    {
        float v[16];
#pragma unroll
        for (int u = 0; u < 16; ++u)
            v[u] = patch[(r + u) * 33 + lane] + bias;
        column_chunk<T, 16, ACT>(p, v, row0 + r, most - r, j);
    }
}

template <typename T, int BN, int ACT>
__global__ void __launch_bounds__(128 + 32 * kPairWarps, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ TcArgs p)
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

    if (warp == 0)
    {
        // ---- producer: this CTA's 128 rows of A and BN / 2 rows of B per stage, reported to the leader's barrier ----
        int s = 0;
        uint32_t phase = 0;
        bool ok        = true;
        int used       = 0;
        const uint32_t full0 = map_to(full, 0);
        for (int t = first; t < tiles && ok; t += stride)
        {
            int ti, tj;
            tile_at(t, p.tiles_i, p.tiles_j, ti, tj);
            const int i0 = ti * 256 + (int) rank * 128, j0 = tj * BN + (int) rank * (BN / 2);
            for (int kb = 0; kb < p.k_blocks; ++kb)
            {
                ok = mbar_wait_warp(empty + 8 * s, phase ^ 1u, stuck);
                if (!ok)
                    break;
                if (elect_one())
                {
                    if (rank == 0)
                        mbar_expect(full + 8 * s, 2 * S::kStageBytes);
                    const uint32_t bar = full0 + 8 * s;
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
                }
                __syncwarp();
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
            ok = mbar_wait_warp(empty + 8 * s, phase ^ 1u, stuck);
            if (++s == S::kStages)
            {
                s = 0;
                phase ^= 1u;
            }
        }
    }
    else if (warp == 1 && rank == 0)
    {
        // ---- one lane of the leader issues the matrix instructions of both SMs ----
        int s = 0;
        uint32_t phase = 0;
        bool ok        = true;
        int n          = 0;
        const uint32_t step_a = operand_step(p.a_kmajor), step_b = operand_step(p.b_kmajor);
        const uint64_t desc_a = operand_desc(base, p.a_kmajor), desc_b = operand_desc(base + 128 * 128, p.b_kmajor);
        for (int t = first; t < tiles && ok; t += stride, ++n)
        {
            const int buf    = n & 1;
            const uint32_t d = tmem + buf * BN;
            ok               = mbar_wait_warp(tempty + 8 * buf, ((n >> 1) & 1) ^ 1u, stuck);
            tmem_fence_after();
            for (int kb = 0; kb < p.k_blocks && ok; ++kb)
            {
                ok = mbar_wait_warp(full + 8 * s, phase, stuck);
                if (!ok)
                    break;
                if (elect_one())
                {
                    const uint64_t da = desc_a + s * (S::kStageBytes >> 4), db = desc_b + s * (S::kStageBytes >> 4);
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        mma<2>(d, da + u * step_a, db + u * step_b, p.idesc, kb > 0 || u > 0);
                    mma_commit_pair(empty + 8 * s, 3);
                    if (kb + 1 == p.k_blocks)
                        mma_commit_pair(tfull + 8 * buf, 3);
                }
                __syncwarp();
                if (++s == S::kStages)
                {
                    s = 0;
                    phase ^= 1u;
                }
            }
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
            const bool poison = !mbar_wait_warp(tfull + 8 * buf, (n >> 1) & 1, stuck);
            tmem_fence_after();
            const int64_t row0 = (int64_t) ti * 256 + rank * 128 + quarter * 32;
            const int64_t col0 = (int64_t) tj * BN + half * (BN / 2);
#pragma unroll 1
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
                if (poison)
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        raw[c] = 0x7fffffff;
                const int64_t j = col0 + c0;
                if (p.vec)
                {
                    const int64_t i = row0 + lane;
#pragma unroll
                    for (int g = 0; g < 32; g += 16)
                        if (i < p.rows && j + g < p.cols)
                        {
                            f32x2_t v[8];
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                v[q] = pair(__uint_as_float(raw[g + 2 * q]), __uint_as_float(raw[g + 2 * q + 1]));
                            row_chunk<T, ACT>(p, v, i, j + g, p.vec == 16);
                        }
                }
                else
                {
                    // rows that no wide access fits: turn the patch in shared memory and write along the rows
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        patch[lane * 33 + c] = __uint_as_float(raw[c]);
                    __syncwarp();
                    write_patch<T, ACT>(p, patch, row0, j);
                }
            }
        }
    }
    __syncwarp();
    stuck_exit(stuck, &g_stuck);
    tmem_fence_before();
    __syncthreads();
    cluster_meet();
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
    // shallow: two CTAs per SM; deep: one, with as much of B on its way as the two would have.  (With 16 or 32 rows a deeper
    // pipeline only crowds the memory: 8 x 4096 -> 11008 24.2 us with twelve stages, 19.4 with six.)
    static constexpr int kShallow = BN == 16 ? 6 : BN == 32 ? 5 : BN == 64 ? 4 : 3;
    static constexpr int kDeep    = BN >= 64 ? 2 * kShallow : kShallow;
    static constexpr int smem(int stages)
    {
        return 1024 + stages * kStageBytes + 256;
    }
    static constexpr int kTmemCols   = BN < 32 ? 32 : BN;
    static_assert(BN * 128 * 4 <= kShallow * kStageBytes, "the partial results of a CTA take the place of its operand tiles");
    static_assert(smem(kDeep) <= 232448 - 16 && 16 * kDeep + 16 <= 256, "shared memory, barriers");
};

// Four results of row i from column j.  With p.vec every row starts on a 16-byte boundary and the number of columns is a
// multiple of 8.
template <typename T>
__device__ __forceinline__ void quad(const TcArgs& p, const float4& z, int64_t i, int64_t j)
{
    float v[4] = {z.x, z.y, z.z, z.w};
    if (p.vec)
    {
        if (j >= p.cols)
            return;
        auto store = [&](T* dst) {
            Pack<T, 4> o;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                o.v[u] = from_f32<T>(v[u]);
            store_pack<T, 4>(dst, o);
        };
        Pack<T, 4> r;
        if (p.residual)
            r = load_pack<T, 4>((const T*) p.residual + i * p.ldr + j);
        if (p.z)
            store((T*) p.z + i * p.ldz + j);
        activate<4>(v, p.act);
        if (p.residual)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                v[u] += to_f32(r.v[u]);
        store((T*) p.out + i * p.ldo + j);
    }
    else
    {
        T r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j + u < p.cols)
            {
                if (p.residual)
                    r[u] = ((const T*) p.residual)[i * p.ldr + j + u];
                if (p.z)
                    ((T*) p.z)[i * p.ldz + j + u] = from_f32<T>(v[u]);
            }
        activate<4>(v, p.act);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j + u < p.cols)
                ((T*) p.out)[i * p.ldo + j + u] = from_f32<T>(p.residual ? v[u] + to_f32(r[u]) : v[u]);
    }
}

template <typename T, int BN>
__global__ void __launch_bounds__(192, 2)
    slim_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ TcArgs p)
{
    using S = SlimShape<BN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int stuck_smem;
    volatile int* stuck = &stuck_smem;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const int stages    = p.stages;
    const uint32_t bars = base + stages * S::kStageBytes;
    const uint32_t full = bars, empty = full + 8 * stages, tfull = empty + 8 * stages, tmem_at = tfull + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t splits;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
    const uint32_t rank = cluster_rank();

    pdl_launch_dependents();
    if (threadIdx.x == 0)
    {
        stuck_smem = 0;
        for (int s = 0; s < stages; ++s)
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

    if (warp == 0)
    {
        int s = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb)
        {
            if (!mbar_wait_warp(empty + 8 * s, phase ^ 1u, stuck))
                break;
            if (elect_one())
            {
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
            }
            __syncwarp();
            if (++s == stages)
            {
                s = 0;
                phase ^= 1u;
            }
        }
    }
    else if (warp == 1)
    {
        int s = 0;
        uint32_t phase = 0;
        const uint32_t step_f = operand_step(p.b_kmajor), step_r = operand_step(p.a_kmajor);
        const uint64_t desc_f = operand_desc(base, p.b_kmajor), desc_r = operand_desc(base + 128 * 128, p.a_kmajor);
        for (int kb = kb0; kb < kb1; ++kb)
        {
            if (!mbar_wait_warp(full + 8 * s, phase, stuck))
                break;
            if (elect_one())
            {
                const uint64_t df = desc_f + s * (S::kStageBytes >> 4), dr = desc_r + s * (S::kStageBytes >> 4);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    mma<1>(tmem, df + u * step_f, dr + u * step_r, p.idesc, kb > kb0 || u > 0);
                mma_commit(empty + 8 * s);
                if (kb + 1 == kb1)
                    mma_commit(tfull);
            }
            __syncwarp();
            if (++s == stages)
            {
                s = 0;
                phase ^= 1u;
            }
        }
    }
    __syncwarp();
    float* part = reinterpret_cast<float*>(smem_raw + (base - smem_addr(smem_raw)));   // [BN][128]
    const int quarter = warp & 3, f = quarter * 32 + lane;
    const int64_t j   = (int64_t) j0 + f;
    float bias        = 0.f;
    bool poison       = false;
    if (warp >= 2)
    {
        if (p.bias && splits == 1 && j < p.cols)
            bias = to_f32(((const T*) p.bias)[j]);
        poison = !mbar_wait_warp(tfull, 0, stuck);
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
        if (warp >= 2)
        {
            // every CTA finishes its share of the rows: a warp takes a row, a lane four columns of it, four rows at a time
            const int c0 = rows * (int) rank / (int) splits, c1 = rows * (int) (rank + 1) / (int) splits;
            const int64_t jq = (int64_t) j0 + lane * 4;
            const uint32_t from = smem_addr(part) + lane * 16;
            float4 b4 = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p.bias)
            {
                const T* b = (const T*) p.bias + jq;
                b4         = make_float4(jq < p.cols ? to_f32(b[0]) : 0.f, jq + 1 < p.cols ? to_f32(b[1]) : 0.f,
                                         jq + 2 < p.cols ? to_f32(b[2]) : 0.f, jq + 3 < p.cols ? to_f32(b[3]) : 0.f);
            }
#pragma unroll 1
            for (int c = c0 + warp - 2; c < c1; c += 16)
            {
                float4 v[4] = {b4, b4, b4, b4};
#pragma unroll 1
                for (uint32_t r = 0; r < splits; r += 4)
                {
                    float4 w[4][4];   // [part][row], all on their way together
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (r + q < splits)
                        {
                            const uint32_t at = map_to(from + c * 512, r + q);
#pragma unroll
                            for (int u = 0; u < 4; ++u)
                                if (c + 4 * u < c1)
                                    w[q][u] = ld_cluster4(at + 4 * u * 512);
                        }
#pragma unroll
                    for (int q = 0; q < 4; ++q)   // always in this order: the same bits on every run
                        if (r + q < splits)
#pragma unroll
                            for (int u = 0; u < 4; ++u)
                                if (c + 4 * u < c1)
                                {
                                    v[u].x += w[q][u].x;
                                    v[u].y += w[q][u].y;
                                    v[u].z += w[q][u].z;
                                    v[u].w += w[q][u].w;
                                }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (c + 4 * u < c1)
                        quad<T>(p, v[u], i0 + c + 4 * u, jq);
            }
        }
        __syncwarp();
        cluster_meet();   // nobody leaves while its partial results may be read
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
    auto encode = [&] {
        return fn(map, dtype == AQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base),
                  dims, pitch, box, strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED)
    {
        // the first CUDA call of this host thread: the driver has no context for it until the runtime binds one
        int dev       = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e == cudaSuccess)
            e = cudaSetDevice(dev);
        if (e != cudaSuccess)
            return cuda_fail(e);
        r = encode();
    }
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

// `most`: the most shared memory that any call of the kernel asks for.  The limit belongs to the kernel, not to the launch,
// so every call sets it to the same value: a smaller one would refuse the launch that another host thread is about to make.
template <typename Kernel>
int launch(Kernel kernel, int64_t grid, int cluster, int threads, int smem, int most, cudaStream_t st, const CUtensorMap& ma,
           const CUtensorMap& mb, const TcArgs& p)
{
    if (grid > 0x7fffffff)
        return AQ_ERR_TOO_LARGE;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
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
    return with_activation(a.act, [&](auto act) {
        return launch(pair_kernel<T, BN, decltype(act)::value>, 2 * pairs, 2, 128 + 32 * kPairWarps, PairShape<BN>::kSmem,
                      PairShape<BN>::kSmem, st, ma, mb, p);
    });
}

template <typename T, int BN>
int run_slim(const GemmArgs& a, int splits, cudaStream_t st)
{
    using S = SlimShape<BN>;
    CUtensorMap ma, mb;
    int rc = operand_map(&ma, a.a, a.lda, a.a_kmajor, a.rows, a.depth, BN, a.dtype);
    if (rc == AQ_OK)
        rc = operand_map(&mb, a.b, a.ldb, a.b_kmajor, a.cols, a.depth, 128, a.dtype);
    if (rc != AQ_OK)
        return rc;
    TcArgs p  = tc_args(a);
    p.tiles_i = (int) ((a.rows + BN - 1) / BN);
    p.tiles_j = (int) ((a.cols + 127) / 128);
    p.vec     = wide_access(a);
    // the columns' operand is the instruction's A
    p.idesc            = instruction_desc(a.dtype == AQ_BF16, a.b_kmajor, a.a_kmajor, 128, BN);
    const int64_t ctas = (int64_t) p.tiles_i * p.tiles_j * splits;
    p.stages           = ctas <= kNumSMs ? S::kDeep : S::kShallow;
    return launch(slim_kernel<T, BN>, ctas, splits, 192, S::smem(p.stages), S::smem(S::kDeep), st, ma, mb, p);
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
        cudaFuncSetAttribute(slim_kernel<T, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, SlimShape<BN>::smem(SlimShape<BN>::kDeep));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim            = dim3(splits);
        cfg.blockDim           = dim3(192);
        cfg.dynamicSmemBytes   = SlimShape<BN>::smem(SlimShape<BN>::kShallow);
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

// How many CTAs share the depth.  `cost` is what the kernel's longest chain of CTAs takes, in cycles: 64 k of a tile cost 290
// of them (BN 16 to 64) or 560 (BN 128; both operands then keep the shared memory as busy as the tensor cores could make
// it) with one CTA on the SM, twice that with two, joining the parts 5000 (BN 128: 9000), the rest 3500.  A second wave of
// clusters costs more than a larger cluster gains (24 x 11008 -> 4096: 32 tiles by eight CTAs are two waves and 37 us, by
// seven one and 22).
template <typename T, int BN>
int slim_plan(int64_t tiles, int64_t k_blocks, int64_t& cost)
{
    const int64_t block = BN == 128 ? 560 : 290, join = BN == 128 ? 9000 : 5000;
    int best = 1;
    cost     = INT64_MAX;
    for (int s = 1; s <= 8 && (s == 1 || k_blocks >= 4 * s); ++s)
    {
        const int64_t room  = resident_clusters<T, BN>(s);
        const int64_t waves = (tiles + room - 1) / room;
        const int64_t per   = tiles * s > kNumSMs ? 2 * block : block;
        const int64_t c     = waves * ((k_blocks + s - 1) / s) * per + (s > 1 ? join : 0) + 3500;
        if (c < cost)
        {
            cost = c;
            best = s;
        }
    }
    return best;
}

template <typename T>
int tensor_gemm_t(const GemmArgs& a, cudaStream_t st)
{
    const int64_t kb = (a.depth + kBlockK - 1) / kBlockK;
    auto slim_tiles  = [&](int bn) { return (a.rows + bn - 1) / bn * ((a.cols + 127) / 128); };
    int64_t slim     = 0;
    if (a.rows <= 64 && a.a_kmajor)
    {
        if (a.rows <= 16)
            return run_slim<T, 16>(a, slim_plan<T, 16>(slim_tiles(16), kb, slim), st);
        if (a.rows <= 32)
            return run_slim<T, 32>(a, slim_plan<T, 32>(slim_tiles(32), kb, slim), st);
        return run_slim<T, 64>(a, slim_plan<T, 64>(slim_tiles(64), kb, slim), st);
    }
    // The same estimate for pair_kernel: 512 cycles for 64 k of a 256 x 256 tile (the tensor cores' own rate), 400 of a
    // 256 x 128 one (issue and handshakes).  512 x 4096 -> 4096: 23.8 and 20.5 us, slim_kernel 22.9.
    auto waves = [](int64_t n, int64_t slots) { return (n + slots - 1) / slots; };
    const int64_t rt = (a.rows + 255) / 256;
    const int64_t p256 = waves(rt * ((a.cols + 255) / 256), kNumSMs / 2) * kb * 512 + 4500;
    const int64_t p128 = waves(rt * ((a.cols + 127) / 128), kNumSMs / 2) * kb * 400 + 4000;
    const int splits   = slim_plan<T, 128>(slim_tiles(128), kb, slim);
    if (slim < p256 && slim < p128)
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
