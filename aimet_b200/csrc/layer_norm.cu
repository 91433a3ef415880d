// Layer norm over rows of `dim` elements, forward and backward.
//
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) rstd, y = h w + b
//   g = dy w, dx = rstd (g - mean(g) - h mean(g h)), dw = sum over rows of dy h, db = sum over rows of dy
//
// The variance is the mean of squared differences from the mean (never E[x^2] - mu^2, which cancels when |mu| is large
// against the spread); every sum is float32.  All of it is bound by memory: x is read and y written once forward, x and
// dy read and dx written once backward.
//
// Which kernel takes a call:
//   norm_fwd_kernel        forward, a row in the registers of 4 to 512 threads
//   norm_fwd_any_kernel    the same in 16-byte packets for many long rows off 16-byte boundaries
//   norm_bwd_ring_kernel   backward: rows arrive in shared memory by bulk copies, several ahead; the sums for dw and db
//                          stay in registers
//   norm_bwd_kernel        backward of short rows, and of few rows off 16-byte boundaries: the next row is fetched into
//                          registers instead
//   *_loop_kernel, norm_param_kernel   rows too long for the registers of 512 threads
// (A forward ring was slower than enough rows in registers: 16384 x 4096 bf16 53 us against 46.)
#include <cfloat>

#include "common.cuh"
#include "kernels.h"
#include "tensor_core.cuh"

namespace aq
{
namespace
{
constexpr int kLoopThreads = 256;

// CTAs per SM that registers allow when a thread needs about `regs`
constexpr int ctas_for(int regs, int threads)
{
    const int n = 65536 / ((regs + 7) / 8 * 8 * threads);
    return n < 1 ? 1 : n > 8 ? 8 : n;
}

// Sum of two floats over the TPR threads of a row (part of a warp, a warp, or the whole CTA); every thread gets both.  Consecutive calls
// of a CTA have to use different `red` (one barrier each).
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float4 (&red)[8])
{
#pragma unroll
    for (int o = TPR < 32 ? TPR / 2 : 16; o; o >>= 1)
    {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (TPR > 32)
    {
        constexpr int WARPS = TPR / 32;
        static_assert(WARPS <= 16 && WARPS % 2 == 0, "two warps per 16 bytes");
        if ((threadIdx.x & 31) == 0)
            reinterpret_cast<float2*>(red)[threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS / 2; ++i)
        {
            const float4 r = red[i];
            a += r.x;
            b += r.y;
            a += r.z;
            b += r.w;
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

// Elements 2q and 2q + 1 of a thread's packets as two float32 lanes (the last lane of an odd count is 0).
template <typename T, int VEC, int PACKS>
__device__ __forceinline__ f32x2_t lanes(const Pack<T, VEC> (&p)[PACKS], int q)
{
    const int i = 2 * q, j = 2 * q + 1;
    return pair(to_f32(p[i / VEC].v[i % VEC]), j < PACKS * VEC ? to_f32(p[j / VEC].v[j % VEC]) : 0.f);
}
template <typename T, int VEC, int PACKS>
__device__ __forceinline__ void set_lanes(Pack<T, VEC> (&p)[PACKS], int q, f32x2_t v)
{
    float lo, hi;
    unpair(v, lo, hi);
    const int i = 2 * q, j = 2 * q + 1;
    p[i / VEC].v[i % VEC] = from_f32<T>(lo);
    if (j < PACKS * VEC)
        p[j / VEC].v[j % VEC] = from_f32<T>(hi);
}
__device__ __forceinline__ float lane_sum(f32x2_t v)
{
    float lo, hi;
    unpair(v, lo, hi);
    return lo + hi;
}

// A packet, or `fill` in every element.  Through whole registers: element-wise selects would make the compiler wait for
// each load before it issues the next.
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_or(const T* p, bool in, float fill)
{
    Pack<T, VEC> r = splat<T, VEC>(fill);
    if constexpr (sizeof(r) == 16)
    {
        uint4 u;
        memcpy(&u, &r, 16);
        if (in)
            u = *reinterpret_cast<const uint4*>(p);
        memcpy(&r, &u, 16);
    }
    else if (in)
        r = load_pack<T, VEC>(p);
    return r;
}

// A thread's packets of one row: packet k of thread t starts at element (k TPR + t) VEC; what lies beyond the row is `fill`.
template <typename T, int VEC, int TPR, int PACKS>
__device__ __forceinline__ void load_row(Pack<T, VEC> (&p)[PACKS], const T* row, int t, int64_t dim, float fill)
{
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
    {
        const int64_t i = ((int64_t) k * TPR + t) * VEC;
        p[k]            = load_or<T, VEC>(row + i, row && i < dim, fill);
    }
}
template <typename T, int VEC, int TPR, int PACKS>
__device__ __forceinline__ void store_row(const Pack<T, VEC> (&p)[PACKS], T* row, int t, int64_t dim)
{
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
    {
        const int64_t i = ((int64_t) k * TPR + t) * VEC;
        if (i < dim)
            store_pack<T, VEC>(row + i, p[k]);
    }
}

// ---- rows that do not start or end on 16-byte boundaries -----------------------------------------------------------
// Packets are laid on the 16-byte boundaries of the row that is written.  What is left before the first and behind the last
// of them, fewer than VEC elements each, goes to the first 2 VEC threads, one element each: with packets that were in part
// outside the row, the warps that held them set the pace (16384 x 4097 bf16 forward 138 us, backward 146 us).  An input
// with other boundaries is read as the two aligned pieces that hold a packet.  Now 78 and 105 us (float32 93 and 140);
// element by element 196 and 369 us (175 and 292).
struct Cut
{
    int head, end;   // the packets hold elements head to end - 1
    int mine;        // this thread's single element, -1 without one

    template <typename T>
    static __device__ __forceinline__ Cut of(const T* row, int t, int dim)
    {
        constexpr int VEC = 16 / (int) sizeof(T);
        Cut c;
        c.head = (VEC - (int) ((uintptr_t) row % 16 / sizeof(T))) % VEC;
        c.end  = c.head + (dim - c.head) / VEC * VEC;
        c.mine = t < c.head ? t : t >= VEC && t - VEC < dim - c.end ? c.end + t - VEC : -1;
        return c;
    }
};
// Elements of T between the last 16-byte boundary and p.
template <typename T>
__device__ __forceinline__ int elements_in(const T* p)
{
    return (int) ((uintptr_t) p % 16 / sizeof(T));
}
// 16 of the 32 bytes (lo, hi), from byte `from` (0 to 15, even) on
__device__ __forceinline__ uint4 piece(uint4 lo, uint4 hi, uint32_t from)
{
    uint32_t u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int j = 0; j < 6; ++j)
        u[j] = from & 8 ? u[j + 2] : u[j];
#pragma unroll
    for (int j = 0; j < 5; ++j)
        u[j] = from & 4 ? u[j + 1] : u[j];
    const uint32_t bits = (from & 2) * 8;
    return make_uint4(__funnelshift_r(u[0], u[1], bits), __funnelshift_r(u[1], u[2], bits), __funnelshift_r(u[2], u[3], bits),
                      __funnelshift_r(u[3], u[4], bits));
}
// The packets at at[k] < end of p, by the element.
template <typename T, int VEC, int N>
__device__ __forceinline__ void load_elements(Pack<T, VEC> (&r)[N], const T* p, const int (&at)[N], int end, float fill)
{
#pragma unroll
    for (int k = 0; k < N; ++k)
    {
        r[k] = splat<T, VEC>(fill);
        if (p && at[k] < end)
#pragma unroll
            for (int c = 0; c < VEC; ++c)
                r[k].v[c] = p[at[k] + c];
    }
}
// The packets of a row, and zeros.  Between two other rows that lie at least 2 VEC elements from it whole pieces are read:
// what they hold besides the packets lies between elements of x.
template <typename T, int VEC, int N>
__device__ __forceinline__ void load_row_any(uint4 (&r)[N], const T* row, const int (&at)[N], int end, bool between)
{
    if (!between)
    {
        Pack<T, VEC> p[N];
        load_elements(p, row, at, end, 0.f);
#pragma unroll
        for (int k = 0; k < N; ++k)
            memcpy(&r[k], &p[k], 16);
        return;
    }
    const int off = elements_in(row + at[0]);
#pragma unroll
    for (int k = 0; k < N; ++k)
    {
        r[k] = make_uint4(0, 0, 0, 0);
        if (at[k] < end)
            r[k] = *reinterpret_cast<const uint4*>(row + at[k] - off);
    }
    if (off)
    {
        uint4 hi[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
        {
            hi[k] = make_uint4(0, 0, 0, 0);
            if (at[k] < end)
                hi[k] = *reinterpret_cast<const uint4*>(row + at[k] - off + VEC);
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
            r[k] = piece(r[k], hi[k], off * sizeof(T));
    }
}

// Statistics and result of a row whose packets are in v.  w and b come out of L1.  The arithmetic runs two float32 lanes per instruction.
template <typename T, int VEC, int TPR, int PACKS>
__device__ __forceinline__ void norm_row(const LayerNormArgs& a, const Pack<T, VEC> (&v)[PACKS], int64_t row, int t,
                                         float4 (&red)[2][8], bool live)
{
    constexpr int Q = (PACKS * VEC + 1) / 2;
    f32x2_t s2 = pair(0.f, 0.f);
#pragma unroll
    for (int q = 0; q < Q; ++q)
        s2 = add2(s2, lanes(v, q));
    const float mu   = row_sum2<TPR>(lane_sum(s2), 0.f, red[0]).x / (float) a.dim;
    const f32x2_t m2 = pair(mu, mu);
    s2               = pair(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
        if (((int64_t) k * TPR + t) * VEC < a.dim)   // what lies beyond the row holds zeros, not the mean
        {
            const Pack<T, VEC> one[1] = {v[k]};
#pragma unroll
            for (int q = 0; q < (VEC + 1) / 2; ++q)
            {
                const f32x2_t d = sub2(lanes(one, q), VEC > 1 ? m2 : pair(mu, 0.f));
                s2              = fma2(d, d, s2);
            }
        }
    const float rstd = 1.f / sqrtf(row_sum2<TPR>(lane_sum(s2), 0.f, red[1]).x / (float) a.dim + a.eps);
    const f32x2_t r2 = pair(rstd, rstd);
    // eight lanes' worth of w and b at a time, so that they need few registers beside the row
    constexpr int AT = PACKS < 2 ? PACKS : 2;
#pragma unroll
    for (int k0 = 0; k0 < PACKS; k0 += AT)
    {
        Pack<T, VEC> w[AT], b[AT], o[AT];
#pragma unroll
        for (int k = 0; k < AT; ++k)
        {
            const int64_t i = ((int64_t) (k0 + k) * TPR + t) * VEC;
            const bool in   = k0 + k < PACKS && i < a.dim;
            w[k]            = load_or<T, VEC>((const T*) a.w + i, a.w && in, 1.f);
            b[k]            = load_or<T, VEC>((const T*) a.b + i, a.b && in, 0.f);
            if (k0 + k < PACKS)
                o[k] = v[k0 + k];
        }
#pragma unroll
        for (int q = 0; q < (AT * VEC + 1) / 2; ++q)
            set_lanes(o, q, fma2(mul2(sub2(lanes(o, q), m2), r2), lanes(w, q), lanes(b, q)));
#pragma unroll
        for (int k = 0; k < AT; ++k)
        {
            const int64_t i = ((int64_t) (k0 + k) * TPR + t) * VEC;
            if (k0 + k < PACKS && i < a.dim && live)
                store_pack<T, VEC>((T*) a.y + row * a.dim + i, o[k]);
        }
    }
    if (t == 0 && a.mean && live)
    {
        a.mean[row] = mu;
        a.rstd[row] = rstd;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Forward, row in registers.  Up to TPR = 32 a warp takes 32 / TPR neighbouring rows.
// ------------------------------------------------------------------------------------------------------------------
template <typename T, int VEC, int TPR, int PACKS>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_fwd_kernel(LayerNormArgs a)
{
    constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
    __shared__ float4 red[2][8];
    pdl_launch_dependents();
    pdl_wait();
    const int t       = threadIdx.x % TPR;
    const int64_t row = (int64_t) blockIdx.x * ROWS + threadIdx.x / TPR;
    const bool live   = row < a.rows;   // the others of a warp go along with nothing
    Pack<T, VEC> v[PACKS];
    load_row<T, VEC, TPR>(v, live ? (const T*) a.x + row * a.ldx : nullptr, t, a.dim, 0.f);
    norm_row<T, VEC, TPR>(a, v, row, t, red, live);
}

// The same for rows off 16-byte boundaries.  A group of threads keeps its columns from row to row (the rows it takes are a
// multiple of 16 bytes apart), so it reads and shifts its part of w and b once; the next row is on its way while one is
// reduced.  4000 x 5001 bf16 34 us in 320 threads with two packets each, 40 us in 192 with four.
template <int TPR, int PACKS>
struct AnyShape
{
    static constexpr int kThreads = TPR < 128 ? 128 : TPR;
    static constexpr int kRows    = TPR < 128 ? 128 / TPR : 1;
    static constexpr int kCtas    = ctas_for(16 * PACKS + 48, kThreads);
};

template <typename T, int TPR, int PACKS>
__global__ void __launch_bounds__(AnyShape<TPR, PACKS>::kThreads, AnyShape<TPR, PACKS>::kCtas) norm_fwd_any_kernel(LayerNormArgs a)
{
    constexpr int VEC = 16 / (int) sizeof(T), ROWS = AnyShape<TPR, PACKS>::kRows;
    __shared__ float4 red[2][8];
    pdl_launch_dependents();
    pdl_wait();
    const int t          = threadIdx.x % TPR, dim = (int) a.dim;
    const int64_t stride = (int64_t) gridDim.x * ROWS;
    int64_t row          = (int64_t) blockIdx.x * ROWS + threadIdx.x / TPR;
    const Cut cut        = Cut::of((const T*) a.y + row * a.dim, t, dim);
    int at[PACKS];
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
        at[k] = cut.head + (k * TPR + t) * VEC;
    Pack<T, VEC> w[PACKS], b[PACKS];
    load_elements(w, (const T*) a.w, at, cut.end, 1.f);
    load_elements(b, (const T*) a.b, at, cut.end, 0.f);
    const bool one_more = cut.mine >= 0;
    const float w1 = one_more && a.w ? to_f32(((const T*) a.w)[cut.mine]) : 1.f;
    const float b1 = one_more && a.b ? to_f32(((const T*) a.b)[cut.mine]) : 0.f;
    uint4 next[PACKS];
    T next1    = from_f32<T>(0.f);
    auto fetch = [&](int64_t r) {
        const T* x = (const T*) a.x + r * a.ldx;
        load_row_any<T, VEC>(next, x, at, cut.end, r > 0 && r + 1 < a.rows);
        if (one_more)
            next1 = x[cut.mine];
    };
    if (row < a.rows)
        fetch(row);
    for (; row < a.rows; row += stride)
    {
        Pack<T, VEC> v[PACKS];
        memcpy(v, next, sizeof(v));
        const float x1 = to_f32(next1);
        if (row + stride < a.rows)
            fetch(row + stride);
        f32x2_t s2 = pair(x1, 0.f);
#pragma unroll
        for (int q = 0; q < PACKS * VEC / 2; ++q)
            s2 = add2(s2, lanes(v, q));
        const float mu   = row_sum2<TPR>(lane_sum(s2), 0.f, red[0]).x / (float) a.dim;
        const f32x2_t m2 = pair(mu, mu);
        const float d1   = one_more ? x1 - mu : 0.f;
        s2               = pair(d1 * d1, 0.f);
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
            if (at[k] < cut.end)   // the others hold zeros, not the mean
            {
                const Pack<T, VEC> one[1] = {v[k]};
#pragma unroll
                for (int q = 0; q < VEC / 2; ++q)
                {
                    const f32x2_t d = sub2(lanes(one, q), m2);
                    s2              = fma2(d, d, s2);
                }
            }
        const float rstd = 1.f / sqrtf(row_sum2<TPR>(lane_sum(s2), 0.f, red[1]).x / (float) a.dim + a.eps);
        const f32x2_t r2 = pair(rstd, rstd);
        T* y             = (T*) a.y + row * a.dim;
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
            if (at[k] < cut.end)
            {
                const Pack<T, VEC> one[1] = {v[k]}, wk[1] = {w[k]}, bk[1] = {b[k]};
                Pack<T, VEC> o[1];
#pragma unroll
                for (int q = 0; q < VEC / 2; ++q)
                    set_lanes(o, q, fma2(mul2(sub2(lanes(one, q), m2), r2), lanes(wk, q), lanes(bk, q)));
                store_pack<T, VEC>(y + at[k], o[0]);
            }
        if (one_more)
            y[cut.mine] = from_f32<T>(fmaf(d1 * rstd, w1, b1));
        if (t == 0 && a.mean)
        {
            a.mean[row] = mu;
            a.rstd[row] = rstd;
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Backward with a ring of rows in shared memory.  One thread of a row's group (a warp, or the CTA) keeps
// `stages` rows on their way with bulk copies, so that the memory system sees 100 to 200 KB in flight per SM however
// long the reductions of a row take; with the next row in registers alone it was 16 KB, and the backward pass of 16384
// x 4096 bf16 took 168 us.  The waits are bounded (see mbar_wait).
// ------------------------------------------------------------------------------------------------------------------
__device__ int g_stuck;

template <int TPR>
struct RingShape
{
    static constexpr int kThreads = TPR < 128 ? 256 : TPR;
    static constexpr int kGroups  = TPR < 128 ? 256 / TPR : 1;
    static_assert(kGroups == 1 || TPR == 32, "a row belongs to a warp or to the CTA");
};

// Bytes of a row of the ring: in a ring of any rows 16 in front and 16 behind (the two pieces of a packet may begin before
// the row and end after it), and the row from a 16-byte boundary to another.
__host__ __device__ constexpr int64_t ring_row_bytes(int64_t bytes, bool any)
{
    return any ? (bytes + 15) / 16 * 16 + 80 : bytes;
}

// dynamic shared memory: [group][stage][x, dy][ring_row_bytes], then the barriers [group][stage]
template <typename T, bool ANY>
struct Ring
{
    uint32_t data, bars, row_bytes, pitch;
    int stages, stage = 0;
    uint32_t phase    = 0;
    volatile int* stuck;

    __device__ __forceinline__ Ring(uint32_t base, int groups, int group, int stages_, int64_t dim, volatile int* stuck_)
        : row_bytes((uint32_t) dim * sizeof(T)), pitch((uint32_t) ring_row_bytes(dim * sizeof(T), ANY)), stages(stages_),
          stuck(stuck_)
    {
        data = base + group * stages * 2 * pitch;
        bars = base + groups * stages * 2 * pitch + group * stages * 8;
    }
    // where the row, or the 16-byte boundary before it, lies
    __device__ __forceinline__ uint32_t at(int s, int matrix) const
    {
        return data + (s * 2 + matrix) * pitch + (ANY ? 16 : 0);
    }
    __device__ __forceinline__ void request(int s, const T* p0, const T* p1)
    {
        const uint32_t bar = bars + 8 * s;
        tc::mbar_expect(bar, 2 * row_bytes);
        tc::bulk_load(at(s, 0), p0, row_bytes, bar);
        tc::bulk_load(at(s, 1), p1, row_bytes, bar);
    }
    // Rows off the boundaries.  Between two other rows the copy takes whole pieces, with some of its neighbours' elements
    // (or what lies between them); of the first and the last row it takes the whole pieces inside, and this thread the rest.
    __device__ __forceinline__ void request_any(int s, const T* p0, const T* p1, bool between)
    {
        const T* p[2] = {p0, p1};
        uintptr_t from[2];
        uint32_t bytes[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            const uintptr_t begin = (uintptr_t) p[i], end = begin + row_bytes;
            from[i]               = between ? begin / 16 * 16 : (begin + 15) / 16 * 16;
            const uintptr_t to    = between ? (end + 15) / 16 * 16 : end / 16 * 16;
            bytes[i]              = (uint32_t) (to - from[i]);
            if (!between)
            {
                const uint32_t row = at(s, i) + (uint32_t) (begin % 16);
                for (uintptr_t e = begin; e < from[i]; e += sizeof(T))
                    put(row + (uint32_t) (e - begin), *reinterpret_cast<const T*>(e));
                for (uintptr_t e = to; e < end; e += sizeof(T))
                    put(row + (uint32_t) (e - begin), *reinterpret_cast<const T*>(e));
            }
        }
        if (!between)   // a later copy may write there
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        const uint32_t bar = bars + 8 * s;
        tc::mbar_expect(bar, bytes[0] + bytes[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            tc::bulk_load(at(s, i) + (uint32_t) (from[i] - (uintptr_t) p[i] / 16 * 16), (const void*) from[i], bytes[i], bar);
    }
    static __device__ __forceinline__ void put(uint32_t at, T v)
    {
        if constexpr (sizeof(T) == 2)
        {
            uint16_t u;
            memcpy(&u, &v, 2);
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(u) : "memory");
        }
        else
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
    }
    __device__ __forceinline__ bool wait()
    {
        return tc::mbar_wait(bars + 8 * stage, phase, stuck);
    }
    __device__ __forceinline__ void advance()
    {
        if (++stage == stages)
        {
            stage = 0;
            phase ^= 1u;
        }
    }
};

__device__ __forceinline__ uint4 shared16(uint32_t at)
{
    uint4 u;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at) : "memory");
    return u;
}
// Elements i and on of the row whose first one lies at `row` in shared memory
template <typename T, int VEC, bool ANY>
__device__ __forceinline__ Pack<T, VEC> read_packet(uint32_t row, int i)
{
    const uint32_t at = row + i * (uint32_t) sizeof(T), off = ANY ? at % 16 : 0;
    uint4 u           = shared16(at - off);
    if (off)
        u = piece(u, shared16(at - off + 16), off);
    Pack<T, VEC> p;
    memcpy(&p, &u, 16);
    return p;
}
template <typename T>
__device__ __forceinline__ float read_element(uint32_t row, int i)
{
    if constexpr (sizeof(T) == 4)
    {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(row + i * 4) : "memory");
        return v;
    }
    else
    {
        uint16_t u;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(row + i * 2) : "memory");
        T v;
        memcpy(&v, &u, 2);
        return to_f32(v);
    }
}

// A thread keeps the same columns for every row its group takes; their sums for dw and db stay in its registers.  Up to
// 16 columns h and dy w stay there too between the sums of the row and dx; with more they are formed twice, from the
// packets in shared memory.  16 columns per thread is where the work beside them (reductions, barriers, addresses) stops
// mattering: 8 columns on 512 threads took 107 us for 16384 x 4096 bf16.  Each CTA leaves one row of partial sums,
// part [gridDim.x][2][dim] (TPR = 32: its warps are added up in shared memory first).
template <typename T, int PACKS>
struct BwdColumns
{
    static constexpr int N     = PACKS * (16 / (int) sizeof(T));
    static constexpr bool KEEP = N <= 16;
    static constexpr int kRegs = (KEEP ? 4 : 2) * N + 48;
};

// ANY: rows off 16-byte boundaries.  The rows of a group are a multiple of 16 bytes apart, so that it keeps its columns.
template <typename T, int TPR, int PACKS, bool ANY>
__global__ void __launch_bounds__(RingShape<TPR>::kThreads, ctas_for(BwdColumns<T, PACKS>::kRegs, RingShape<TPR>::kThreads))
    norm_bwd_ring_kernel(LayerNormGradArgs a, int stages)
{
    constexpr int VEC = 16 / (int) sizeof(T), GROUPS = RingShape<TPR>::kGroups;
    constexpr int N = PACKS * VEC, Q = N / 2;
    constexpr bool KEEP = BwdColumns<T, PACKS>::KEEP;
    extern __shared__ __align__(128) uint8_t ring_smem[];
    __shared__ float4 red[2][8];
    __shared__ int stuck_smem;
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    Ring<T, ANY> ring(tc::smem_addr(ring_smem), GROUPS, group, stages, a.dim, &stuck_smem);
    pdl_launch_dependents();
    if (threadIdx.x == 0)
        stuck_smem = 0;
    if (t < stages)
        tc::mbar_init(ring.bars + 8 * t, 1);
    tc::mbar_init_fence();
    __syncthreads();
    pdl_wait();
    const int64_t stride = (int64_t) gridDim.x * GROUPS;
    int64_t row          = (int64_t) blockIdx.x * GROUPS + group;
    auto request         = [&](int s, int64_t r) {
        const T *x = (const T*) a.x + r * a.ldx, *dy = (const T*) a.dy + r * a.lddy;
        if constexpr (ANY)
            ring.request_any(s, x, dy, r > 0 && r + 1 < a.rows);
        else
            ring.request(s, x, dy);
    };
    const int dim  = (int) a.dim;
    Cut cut        = {0, dim, -1};
    uint32_t off_x = 0, off_g = 0;   // bytes of the rows behind a boundary
    if constexpr (ANY)
    {
        off_x = (uint32_t) elements_in((const T*) a.x + row * a.ldx) * sizeof(T);
        off_g = (uint32_t) elements_in((const T*) a.dy + row * a.lddy) * sizeof(T);
        cut   = Cut::of(a.dx ? (const T*) a.dx + row * a.dim : (const T*) a.x + row * a.ldx, t, dim);
    }
    // a stage is requested again behind the barrier of the row that it held, or, if dx is formed from it after that barrier,
    // behind the next row's
    constexpr bool LATE = !KEEP && GROUPS == 1;
    const int ahead     = LATE ? stages - 1 : stages;
    if (t == 0)
        for (int s = 0; s < ahead && row + s * stride < a.rows; ++s)
            request(s, row + s * stride);
    const f32x2_t zero = pair(0.f, 0.f);
    f32x2_t dw[Q], db[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q)
        dw[q] = db[q] = zero;
    Pack<T, VEC> w[PACKS];
    if constexpr (ANY)
    {
        int at[PACKS];
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
            at[k] = cut.head + (k * TPR + t) * VEC;
        load_elements(w, (const T*) a.w, at, cut.end, 1.f);
    }
    else
        load_row<T, VEC, TPR>(w, (const T*) a.w, t, a.dim, 1.f);
    const bool one_more = ANY && cut.mine >= 0;
    const float w1      = one_more && a.w ? to_f32(((const T*) a.w)[cut.mine]) : 1.f;
    float dw1 = 0.f, db1 = 0.f;
    float mu = 0.f, rstd = 0.f;
    if (row < a.rows)
    {
        mu   = a.mean[row];
        rstd = a.rstd[row];
    }
    for (int slot = 0; row < a.rows; row += stride, slot ^= 1)
    {
        const float r = rstd, mean = mu;
        const f32x2_t m2 = pair(mu, mu), r2 = pair(r, r);
        if (row + stride < a.rows)
        {
            mu   = a.mean[row + stride];
            rstd = a.rstd[row + stride];
        }
        const bool ok = ring.wait();
        const uint32_t at_x = ring.at(ring.stage, 0) + off_x, at_g = ring.at(ring.stage, 1) + off_g;
        float h1 = 0.f, g1 = 0.f;
        if (one_more)
        {
            const float dy = read_element<T>(at_g, cut.mine);
            h1             = (read_element<T>(at_x, cut.mine) - mean) * r;
            g1             = dy * w1;
            dw1            = fmaf(dy, h1, dw1);
            db1 += dy;
        }
        f32x2_t sg = pair(g1, 0.f), sgh = pair(g1 * h1, 0.f), kept_h[KEEP ? Q : 1], kept_g[KEEP ? Q : 1];
#pragma unroll
        for (int k = 0; k < PACKS; ++k)
        {
            const int at = cut.head + (k * TPR + t) * VEC;
            if (at >= cut.end)
                continue;
            const Pack<T, VEC> x[1] = {read_packet<T, VEC, ANY>(at_x, at)}, wk[1] = {w[k]};
            const Pack<T, VEC> g[1] = {read_packet<T, VEC, ANY>(at_g, at)};
#pragma unroll
            for (int q = 0; q < VEC / 2; ++q)
            {
                const int i      = k * (VEC / 2) + q;
                const f32x2_t dy = lanes(g, q);
                const f32x2_t h  = mul2(sub2(lanes(x, q), m2), r2);
                const f32x2_t gw = mul2(dy, lanes(wk, q));
                dw[i]            = fma2(dy, h, dw[i]);
                db[i]            = add2(db[i], dy);
                sg               = add2(sg, gw);
                sgh              = fma2(gw, h, sgh);
                if constexpr (KEEP)
                {
                    kept_h[i] = h;
                    kept_g[i] = gw;
                }
            }
        }
        float2 sum = row_sum2<TPR>(lane_sum(sg), lane_sum(sgh), red[slot]);
        if (!ok)
            sum.x = __int_as_float(0x7fffffff);
        // not after a wait that ran out: the barrier's phase is still open, and a second arrival in it is not allowed
        if ((KEEP || LATE) && t == 0 && ok && row + ahead * stride < a.rows)
            request(LATE ? (ring.stage == 0 ? stages - 1 : ring.stage - 1) : ring.stage, row + ahead * stride);
        if (a.dx)
        {
            // dx = r gw - r mean(g) - h r mean(g h)
            const float c0 = -r * (sum.x / (float) a.dim), c1 = -r * (sum.y / (float) a.dim);
            const f32x2_t c02 = pair(c0, c0), c12 = pair(c1, c1);
#pragma unroll
            for (int k = 0; k < PACKS; ++k)
            {
                const int i = cut.head + (k * TPR + t) * VEC;
                if (i >= cut.end)
                    continue;
                Pack<T, VEC> o[1];
                if constexpr (KEEP)
                {
#pragma unroll
                    for (int q = 0; q < VEC / 2; ++q)
                        set_lanes(o, q, fma2(kept_h[k * (VEC / 2) + q], c12, fma2(kept_g[k * (VEC / 2) + q], r2, c02)));
                }
                else
                {
                    const Pack<T, VEC> x[1] = {read_packet<T, VEC, ANY>(at_x, i)}, wk[1] = {w[k]};
                    const Pack<T, VEC> g[1] = {read_packet<T, VEC, ANY>(at_g, i)};
#pragma unroll
                    for (int q = 0; q < VEC / 2; ++q)
                        set_lanes(o, q,
                                  fma2(mul2(sub2(lanes(x, q), m2), r2), c12, fma2(mul2(lanes(g, q), lanes(wk, q)), r2, c02)));
                }
                store_pack<T, VEC>((T*) a.dx + row * a.dim + i, o[0]);
            }
            if (one_more)
                ((T*) a.dx)[row * a.dim + cut.mine] = from_f32<T>(fmaf(h1, c1, fmaf(g1, r, c0)));
        }
        if (!KEEP && !LATE)
        {
            __syncwarp();
            if (t == 0 && ok && row + ahead * stride < a.rows)
                request(ring.stage, row + ahead * stride);
        }
        ring.advance();
    }
    __syncthreads();
    tc::stuck_exit(&stuck_smem, &g_stuck);
    if (!a.part)
        return;
    if (stuck_smem)   // rows that never arrived are in the sums
    {
        dw1 = db1 = __int_as_float(0x7fffffff);
#pragma unroll
        for (int q = 0; q < Q; ++q)
            dw[q] = db[q] = pair(dw1, dw1);
    }
    float* part = a.part + (int64_t) blockIdx.x * 2 * a.dim;
    float* sums = reinterpret_cast<float*>(ring_smem);   // [GROUPS][dim]: the ring is no longer needed
#pragma unroll
    for (int which = 0; which < 2; ++which)
    {
        Pack<float, VEC> o[PACKS];
#pragma unroll
        for (int q = 0; q < Q; ++q)
            set_lanes(o, q, which ? db[q] : dw[q]);
        auto put = [&](float* to) {
            if constexpr (ANY)
            {
#pragma unroll
                for (int k = 0; k < PACKS; ++k)
                {
                    const int i = cut.head + (k * TPR + t) * VEC;
                    if (i < cut.end)
#pragma unroll
                        for (int c = 0; c < VEC; ++c)
                            to[i + c] = o[k].v[c];
                }
                if (one_more)
                    to[cut.mine] = which ? db1 : dw1;
            }
            else
                store_row<float, VEC, TPR>(o, to, t, a.dim);
        };
        if constexpr (GROUPS == 1)
            put(part + which * a.dim);
        else
        {
            __syncthreads();
            put(sums + group * a.dim);
            __syncthreads();
            for (int i = threadIdx.x; i < a.dim; i += 256)
            {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < GROUPS; ++j)
                    s += sums[j * a.dim + i];
                part[which * a.dim + i] = s;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Backward of short rows, and of few rows off 16-byte boundaries: as norm_bwd_ring_kernel, but the next row is fetched into
// registers while the current one is reduced.  Up to TPR = 32 a warp takes 32 / TPR neighbouring rows at a time.
// ------------------------------------------------------------------------------------------------------------------
template <int TPR, int COLUMNS>
struct BwdShape
{
    static constexpr int kThreads = TPR < 128 ? 256 : TPR;
    static constexpr int kRows    = TPR < 128 ? 256 / TPR : 1;
    static constexpr int kCtas    = ctas_for(5 * COLUMNS + 40, kThreads);
};

template <typename T, int VEC, int TPR, int PACKS>
__global__ void __launch_bounds__(BwdShape<TPR, PACKS * VEC>::kThreads, BwdShape<TPR, PACKS * VEC>::kCtas)
    norm_bwd_kernel(LayerNormGradArgs a)
{
    constexpr int ROWS = BwdShape<TPR, PACKS * VEC>::kRows;
    constexpr int N = PACKS * VEC, Q = (N + 1) / 2;
    constexpr bool AHEAD = N <= 16;   // with more columns the registers of 512 threads do not hold the next row
    static_assert(ROWS == 1 || TPR <= 32, "a row belongs to (part of) a warp or to the CTA");
    __shared__ float4 red[2][8];
    __shared__ float sums[ROWS > 1 ? ROWS : 1][ROWS > 1 ? TPR * N + 1 : 1];
    pdl_launch_dependents();
    pdl_wait();
    const int t          = threadIdx.x % TPR;
    const int64_t stride = (int64_t) gridDim.x * ROWS;
    const f32x2_t zero   = pair(0.f, 0.f);
    f32x2_t dw[Q], db[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q)
        dw[q] = db[q] = zero;
    Pack<T, VEC> x[PACKS], g[PACKS];
    float mu = 0.f, rstd = 0.f;
    auto fetch = [&](int64_t row) {   // beyond the last row, and beyond a row's end: no part in any sum
        const bool live = row < a.rows;
        mu              = live ? a.mean[row] : 0.f;
        rstd            = live ? a.rstd[row] : 0.f;
        load_row<T, VEC, TPR>(x, live ? (const T*) a.x + row * a.ldx : nullptr, t, a.dim, 0.f);
        load_row<T, VEC, TPR>(g, live ? (const T*) a.dy + row * a.lddy : nullptr, t, a.dim, 0.f);
    };
    int64_t row     = (int64_t) blockIdx.x * ROWS + threadIdx.x / TPR;
    const int above = TPR < 32 ? (threadIdx.x & 31) / TPR : 0;   // rows of this warp above this one
    if (AHEAD)
        fetch(row);
    for (int slot = 0; row - above < a.rows; row += stride, slot ^= 1)
    {
        if (!AHEAD)
            fetch(row);
        const float r = rstd, mean = mu;
        const f32x2_t m2 = pair(mu, mu), r2 = pair(r, r);
        f32x2_t h[Q], gw[Q], sg = zero, sgh = zero;
        Pack<T, VEC> w[PACKS];
        load_row<T, VEC, TPR>(w, (const T*) a.w, t, a.dim, 1.f);
#pragma unroll
        for (int q = 0; q < Q; ++q)
        {
            const f32x2_t dy = lanes(g, q);
            const f32x2_t hq = mul2(sub2(lanes(x, q), m2), r2);
            const f32x2_t gq = mul2(dy, lanes(w, q));
            dw[q]            = fma2(dy, hq, dw[q]);
            db[q]            = add2(db[q], dy);
            sg               = add2(sg, gq);
            sgh              = fma2(gq, hq, sgh);
            h[q]             = hq;
            gw[q]            = gq;
        }
        if (AHEAD && row + stride - above < a.rows)
            fetch(row + stride);
        if (!a.dx)
            continue;
        if (!(fabsf(mean * r) <= FLT_MAX))   // outside the row h is not finite, and 0 h no 0
        {
            sgh = zero;
#pragma unroll
            for (int q = 0; q < Q; ++q)
            {
                float h0, h1, g0, g1;
                unpair(h[q], h0, h1);
                unpair(gw[q], g0, g1);
                const int i = 2 * q, j = 2 * q + 1;
                const bool in0 = ((int64_t) (i / VEC) * TPR + t) * VEC + i % VEC < a.dim;
                const bool in1 = j < N && ((int64_t) (j / VEC) * TPR + t) * VEC + j % VEC < a.dim;
                sgh            = add2(sgh, pair(in0 ? g0 * h0 : 0.f, in1 ? g1 * h1 : 0.f));
            }
        }
        const float2 s = row_sum2<TPR>(lane_sum(sg), lane_sum(sgh), red[slot]);
        // dx = r gw - r mean(g) - h r mean(g h)
        const float c0 = -r * (s.x / (float) a.dim), c1 = -r * (s.y / (float) a.dim);
        const f32x2_t c02 = pair(c0, c0), c12 = pair(c1, c1);
        Pack<T, VEC> o[PACKS];
#pragma unroll
        for (int q = 0; q < Q; ++q)
            set_lanes(o, q, fma2(h[q], c12, fma2(gw[q], r2, c02)));
        if (row < a.rows)
            store_row<T, VEC, TPR>(o, (T*) a.dx + row * a.dim, t, a.dim);
    }
    if (!a.part)
        return;
    float* part = a.part + (int64_t) blockIdx.x * 2 * a.dim;
#pragma unroll
    for (int which = 0; which < 2; ++which)
    {
        if constexpr (ROWS == 1)
        {
            Pack<float, VEC> o[PACKS];
#pragma unroll
            for (int q = 0; q < Q; ++q)
                set_lanes(o, q, which ? db[q] : dw[q]);
            store_row<float, VEC, TPR>(o, part + which * a.dim, t, a.dim);
        }
        else
        {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < Q; ++q)
            {
                float lo, hi;
                unpair(which ? db[q] : dw[q], lo, hi);
                const int i = 2 * q, j = 2 * q + 1;
                sums[threadIdx.x / TPR][((i / VEC) * TPR + t) * VEC + i % VEC] = lo;
                if (j < N)
                    sums[threadIdx.x / TPR][((j / VEC) * TPR + t) * VEC + j % VEC] = hi;
            }
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
    __shared__ float4 red[2][8];
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
    __shared__ float4 red[2][8];
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
#define AQ_SHAPE(TPR, PACKS)                                                                                        \
    if constexpr (PACKS <= MAX_PACKS)                                                                               \
        if (packets <= (TPR) * (PACKS))                                                                             \
            return f(std::integral_constant<int, TPR> {}, std::integral_constant<int, PACKS> {});

// f(TPR, PACKS) for the first shape that holds `packets` packets, AQ_ERR_TOO_LARGE (and no call) when none does.
// Rows in registers, few of them: many threads per row.
template <int MAX_PACKS, typename F>
int with_row_shape(int64_t packets, F&& f)
{
    AQ_SHAPE(4, 1)
    AQ_SHAPE(8, 1)
    AQ_SHAPE(16, 1)
    AQ_SHAPE(32, 1)
    AQ_SHAPE(32, 2)
    AQ_SHAPE(128, 1)
    AQ_SHAPE(256, 1)
    AQ_SHAPE(512, 1)
    AQ_SHAPE(512, 2)
    AQ_SHAPE(512, 4)
    AQ_SHAPE(512, 8)
    AQ_SHAPE(512, 16)
    AQ_SHAPE(512, 24)
    return AQ_ERR_TOO_LARGE;
}
// many rows of single elements
template <typename F>
int with_odd_shape(int64_t packets, F&& f)
{
    constexpr int MAX_PACKS = 24;
    AQ_SHAPE(4, 1)
    AQ_SHAPE(4, 4)
    AQ_SHAPE(4, 8)
    AQ_SHAPE(8, 8)
    AQ_SHAPE(16, 8)
    AQ_SHAPE(32, 8)
    AQ_SHAPE(32, 16)
    AQ_SHAPE(128, 8)
    AQ_SHAPE(128, 16)
    AQ_SHAPE(256, 16)
    AQ_SHAPE(512, 16)
    AQ_SHAPE(512, 24)
    return AQ_ERR_TOO_LARGE;
}
// many rows of packets
template <typename F>
int with_even_shape(int64_t packets, F&& f)
{
    constexpr int MAX_PACKS = 8;
    AQ_SHAPE(4, 1)
    AQ_SHAPE(4, 2)
    AQ_SHAPE(4, 4)
    AQ_SHAPE(8, 4)
    AQ_SHAPE(16, 4)
    AQ_SHAPE(32, 4)
    AQ_SHAPE(128, 2)
    AQ_SHAPE(128, 4)
    AQ_SHAPE(256, 4)
    AQ_SHAPE(512, 4)
    AQ_SHAPE(512, 8)
    return AQ_ERR_TOO_LARGE;
}
// Many rows of packets off 16-byte boundaries.  The shapes between the powers of two keep most of a CTA's threads on the row;
// without them bf16, 2^26 elements: 2501 columns in 128 x 4 111 us, in 128 x 3 98; 5001 in 256 x 4 113, in 320 x 2 102; 6001 102
// and in 384 x 2 94; 9001 in 512 x 4 145, in 320 x 4 119; 11001 125 and in 384 x 4 109.
template <typename F>
int with_any_shape(int64_t packets, F&& f)
{
    constexpr int MAX_PACKS = 4;
    AQ_SHAPE(32, 1)
    AQ_SHAPE(32, 2)
    AQ_SHAPE(32, 4)
    AQ_SHAPE(128, 2)
    AQ_SHAPE(128, 3)
    AQ_SHAPE(128, 4)
    AQ_SHAPE(320, 2)
    AQ_SHAPE(384, 2)
    AQ_SHAPE(256, 4)
    AQ_SHAPE(320, 4)
    AQ_SHAPE(384, 4)
    AQ_SHAPE(512, 4)
    return AQ_ERR_TOO_LARGE;
}
// short rows of packets with sums: at most 16 columns per thread
template <int MAX_PACKS, typename F>
int with_short_shape(int64_t packets, F&& f)
{
    AQ_SHAPE(4, 1)
    AQ_SHAPE(4, 2)
    AQ_SHAPE(4, 4)
    AQ_SHAPE(8, 2)
    AQ_SHAPE(8, 4)
    AQ_SHAPE(16, 2)
    AQ_SHAPE(16, 4)
    return AQ_ERR_TOO_LARGE;
}
// The backward ring: 16 columns per thread where the row's length allows; a warp takes up to 768 elements of 16 bits or 512 of
// 32 alone.  As above, backward pass with sums, 2^26 elements: bf16 600 columns in 128 threads 82 us, in a warp with three packets 67;
// 11008 in 512 x 4 108, in 512 x 3 84 (float32 8500 in 512 x 8 157, in 512 x 6 138); off boundaries 5001 in 512 x 2 150, in
// 320 x 2 121 (float32 4999 160 and 133).  192 threads for the rows between those of 128 and 256 were slower than 256 (bf16 2501
// 181 and 144, float32 261 and 154).
template <typename T, bool ANY, typename F>
int with_sums_shape(int64_t packets, F&& f)
{
    constexpr int MAX_PACKS = 8;
    AQ_SHAPE(32, 1)
    AQ_SHAPE(32, 2)
    if constexpr (sizeof(T) == 2)
    {
        AQ_SHAPE(32, 3)
        AQ_SHAPE(128, 1)
        AQ_SHAPE(128, 2)
        AQ_SHAPE(256, 2)
        if constexpr (ANY)
        {
            AQ_SHAPE(320, 2)
        }
        AQ_SHAPE(512, 2)
        AQ_SHAPE(512, 3)
        AQ_SHAPE(512, 4)
    }
    else
    {
        AQ_SHAPE(32, 4)
        AQ_SHAPE(128, 4)
        AQ_SHAPE(256, 4)
        if constexpr (ANY)
        {
            AQ_SHAPE(320, 4)
        }
        AQ_SHAPE(512, 4)
        AQ_SHAPE(512, 6)
        AQ_SHAPE(512, 8)
    }
    return AQ_ERR_TOO_LARGE;
}
#undef AQ_SHAPE

constexpr int kRingBudget = 208 * 1024;   // shared memory of an SM for the rings of its CTAs

// Stages of a ring: as many as fit with `ctas` CTAs on an SM (or fewer CTAs), 2 to 6; 0 when two do not fit.
int ring_stages(int64_t stage_bytes, int groups, int& ctas)
{
    for (; ctas >= 1; --ctas)
    {
        const int64_t n = kRingBudget / ctas / (stage_bytes * groups + 8 * groups);
        if (n >= (ctas > 1 ? 3 : 2))
            return (int) (n < 6 ? n : 6);
    }
    return 0;
}

template <typename Kernel>
int launch_ring(Kernel kernel, const LayerNormGradArgs& a, int stages, int groups, int64_t stage_bytes, int64_t grid, int threads,
                cudaStream_t st)
{
    const int64_t smem = groups * stages * (stage_bytes + 8);
    // the same limit on every call: it belongs to the kernel, and another host thread may be about to launch with more
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBudget);
    if (e == cudaSuccess)
        e = launch_pdl(kernel, dim3((unsigned) grid), threads, (size_t) smem, st, a, stages);
    note_launch();
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
}

template <typename T>
bool wide_rows(const void* a, int64_t lda, const void* b, int64_t ldb, const void* w, const void* bias, const void* out,
               int64_t dim)
{
    constexpr int W = 16 / (int) sizeof(T);
    auto fits       = [&](const void* p, int64_t ld) { return !p || ((uintptr_t) p % 16 == 0 && ld % W == 0); };
    return dim % W == 0 && fits(a, lda) && fits(b, ldb) && fits(w, W) && fits(bias, W) && fits(out, dim);
}

// Rows off 16-byte boundaries in packets all the same (see Cut), where that pays, forward and backward: 1024 x 4097 bf16
// 12 + 18 us against 15 + 24 us element by element, 5000 x 513 9.4 + 9.8 against 10.2 + 12.3, but 297 x 1001 5.9 + 5.8
// against 4.2 + 3.6 (a group's first row waits for its part of w and b), and 100000 x 65 31 + 58 against 22 + 34.
template <typename T>
bool any_rows(int64_t rows, int64_t dim, int64_t ld, int64_t ld2)
{
    constexpr int64_t W = 32 / (int) sizeof(T);
    return rows >= 5 * kNumSMs && dim >= 512 && ld >= W && ld2 >= W;
}
template <typename T, int VEC>
int norm_fwd_v(const LayerNormArgs& a, cudaStream_t st)
{
    const int64_t packets = (a.dim + VEC - 1) / VEC;
    auto in_registers     = [&](auto tpr, auto packs) {
        constexpr int TPR   = decltype(tpr)::value;
        constexpr int ROWS  = TPR < 128 ? 128 / TPR : 1;
        const cudaError_t e = launch_pdl(norm_fwd_kernel<T, VEC, TPR, decltype(packs)::value>,
                                         dim3((unsigned) ((a.rows + ROWS - 1) / ROWS)), TPR < 128 ? 128 : TPR, 0, st, a);
        note_launch();
        return e == cudaSuccess ? AQ_OK : cuda_fail(e);
    };
    // Many rows: few threads per row, so that each has several loads in flight (2048 x 4096 bf16: 8.8 us with 128 threads
    // and four packets each, 14.7 us with 512 and one).  Few rows: the other way round, one row ends sooner.
    if constexpr (VEC > 1)
        return a.rows > 2 * kNumSMs ? with_even_shape(packets, in_registers) : with_row_shape<8>(packets, in_registers);
    else
        return a.rows > 2 * kNumSMs ? with_odd_shape(packets, in_registers) : with_row_shape<24>(packets, in_registers);
}

template <typename T>
int norm_fwd_t(const LayerNormArgs& a, cudaStream_t st)
{
    const bool wide = wide_rows<T>(a.x, a.ldx, nullptr, 0, a.w, a.b, a.y, a.dim);
    int rc          = AQ_ERR_TOO_LARGE;
    if (wide)
        rc = norm_fwd_v<T, 16 / (int) sizeof(T)>(a, st);
    else if (any_rows<T>(a.rows, a.dim, a.ldx, a.ldx))
        rc = with_any_shape(a.dim / (16 / (int) sizeof(T)), [&](auto tpr, auto packs) {
            using S      = AnyShape<decltype(tpr)::value, decltype(packs)::value>;
            int64_t grid = (a.rows + S::kRows - 1) / S::kRows;
            if (grid > S::kCtas * kNumSMs)
            {
                constexpr int VEC = 16 / (int) sizeof(T);
                grid              = S::kCtas * kNumSMs;
                grid -= grid * S::kRows % VEC;   // rows of a group a multiple of 16 bytes apart
            }
            const cudaError_t e = launch_pdl(norm_fwd_any_kernel<T, decltype(tpr)::value, decltype(packs)::value>,
                                             dim3((unsigned) grid), S::kThreads, 0, st, a);
            note_launch();
            return e == cudaSuccess ? AQ_OK : cuda_fail(e);
        });
    if (rc != AQ_ERR_TOO_LARGE)
        return rc;
    if (!wide)
        rc = norm_fwd_v<T, 1>(a, st);
    if (rc != AQ_ERR_TOO_LARGE)
        return rc;
    const int64_t grid  = a.rows < 8 * kNumSMs ? a.rows : 8 * kNumSMs;
    const cudaError_t e = launch_pdl(norm_fwd_loop_kernel<T>, dim3((unsigned) grid), kLoopThreads, 0, st, a);
    note_launch();
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
}

// Most CTAs of the backward kernels, each with one row of partial sums: what the registers let reside anyway.
int64_t bwd_ctas(int64_t rows, int64_t dim)
{
    const int64_t n = kNumSMs * (dim <= 1024 ? 8 : dim <= 2048 ? 4 : dim <= 8192 ? 2 : 1);
    return rows < 1 ? 1 : rows < n ? rows : n;
}

template <typename T, bool ANY>
int norm_bwd_ring(const LayerNormGradArgs& a, cudaStream_t st)
{
    constexpr int VEC = 16 / (int) sizeof(T);
    return with_sums_shape<T, ANY>(a.dim / VEC, [&](auto tpr, auto packs) -> int {
        constexpr int TPR = decltype(tpr)::value, PACKS = decltype(packs)::value;
        using S             = RingShape<TPR>;
        const int64_t bytes = 2 * ring_row_bytes(a.dim * (int64_t) sizeof(T), ANY);
        int ctas            = ctas_for(BwdColumns<T, PACKS>::kRegs, S::kThreads);
        const int n         = ring_stages(bytes, S::kGroups, ctas);
        if (n == 0)
            return AQ_ERR_TOO_LARGE;
        const int64_t most = bwd_ctas((a.rows + S::kGroups - 1) / S::kGroups, a.dim);
        int64_t grid       = most < (int64_t) ctas * kNumSMs ? most : (int64_t) ctas * kNumSMs;
        if (ANY && grid * S::kGroups < a.rows)   // rows of a group a multiple of 16 bytes apart
            grid -= grid * S::kGroups % VEC;
        const int rc = launch_ring(norm_bwd_ring_kernel<T, TPR, PACKS, ANY>, a, n, S::kGroups, bytes, grid, S::kThreads, st);
        if (rc != AQ_OK || !a.part)
            return rc;
        return fold_columns(a.part, grid, 2 * a.dim, a.dim, a.dw, a.db, a.dtype, st);
    });
}

template <typename T, int VEC>
int norm_bwd_registers(const LayerNormGradArgs& a, cudaStream_t st)
{
    auto run = [&](auto tpr, auto packs) {
        using S            = BwdShape<decltype(tpr)::value, decltype(packs)::value * VEC>;
        const int64_t most = bwd_ctas((a.rows + S::kRows - 1) / S::kRows, a.dim);
        const int64_t grid = most < (int64_t) S::kCtas * kNumSMs ? most : (int64_t) S::kCtas * kNumSMs;
        cudaError_t e      = launch_pdl(norm_bwd_kernel<T, VEC, decltype(tpr)::value, decltype(packs)::value>,
                                        dim3((unsigned) grid), S::kThreads, 0, st, a);
        note_launch();
        if (e != cudaSuccess)
            return cuda_fail(e);
        return a.part ? fold_columns(a.part, grid, 2 * a.dim, a.dim, a.dw, a.db, a.dtype, st) : AQ_OK;
    };
    if constexpr (VEC > 1)
        return with_short_shape<16 / VEC>(a.dim / VEC, run);
    else
        return with_odd_shape(a.dim, run);
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
    int rc          = AQ_ERR_TOO_LARGE;
    if (wide)
    {
        rc = norm_bwd_registers<T, 16 / (int) sizeof(T)>(a, st);
        if (rc == AQ_ERR_TOO_LARGE)
            rc = norm_bwd_ring<T, false>(a, st);
    }
    else
    {
        if (any_rows<T>(a.rows, a.dim, a.ldx, a.lddy))
            rc = norm_bwd_ring<T, true>(a, st);
        if (rc == AQ_ERR_TOO_LARGE)
            rc = norm_bwd_registers<T, 1>(a, st);
    }
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
    // one row of sums per CTA of the register kernels or per band of norm_param_kernel
    const int64_t ctas = bwd_ctas(rows, dim), bands = norm_bands(rows, dim);
    return (ctas < bands ? bands : ctas) * 2 * dim * (int64_t) sizeof(float);
}

int norm_stuck(int* out)
{
    const cudaError_t e = cudaMemcpyFromSymbol(out, g_stuck, sizeof(int));
    return e == cudaSuccess ? AQ_OK : cuda_fail(e);
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
