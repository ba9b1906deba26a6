// Root-mean-square norm with the residual's addition in front of it and the GEMM's A operand behind it:
//     s = x + r                               (fp32; r_out = s rounded to r's type)
//     y = s * w / sqrt(mean(s^2) + eps)       (fp32)
//     one scale per row and 128 columns of y, e4m3 bytes A[m + M*k], inverse scales a_scale[m + M*kb] (as quantize.cuh)
// The norm and the scales see the sum before it is rounded to r's type: there is one rounding between the inputs and each output.
//
// The norm needs a whole row before the first byte can be written, and the bytes of a column of A want many rows side by side.
// So 16 rows are spread over a cluster: a warp owns 16 rows x 128 columns, one scale block of each row, in registers (a lane four
// consecutive columns of every row); the warps of up to eight CTAs hold the row, which is read once.  The CTAs exchange their rows'
// sums of squares through distributed shared memory (64 bytes from each to each, counted by an mbarrier of the receiver).  All
// that does not need the norm is done before the exchange: s * w and its largest magnitude per row and block; after it one factor
// per row and block is left, 1 / rms times the scale.  The 16 rows of a lane's column are 16 neighbouring bytes of A, so the
// quantised values leave the registers as one 16-byte store per column, without going through shared memory.
// The clusters are persistent and their rows arrive by bulk copies: a CTA's buffer is requested anew as soon as its warps have it in
// registers, so that the next 16 rows are on their way while these are reduced, exchanged and stored.
// Sums are added in a fixed order (lanes, warps, CTAs).
// Rows that do not fit (more than 128 blocks, or 16 rows of a CTA's share above SMEM_LIMIT: from 13440 columns in fp32 with an
// fp32 residual) are read twice.
#pragma once
#include "quantize.cuh"
#include <type_traits>

namespace fp8bs {

constexpr int NORM_ROWS = 16;              // rows of a cluster
constexpr int NORM_WARPS = 8;              // per CTA ...
constexpr int NORM_MOST_WARPS = 16;        // ... and where eight CTAs of eight do not hold a row
constexpr int NORM_MAX_CLUSTER = 8;        // the portable limit
constexpr int NORM_SMEM_LIMIT = 220 * 1024;
// behind the buffers: [2][warps] and [2][CTAs] sums of 16 rows, barriers and control words
constexpr int NORM_FIXED_SMEM = 2 * (NORM_MOST_WARPS + NORM_MAX_CLUSTER) * NORM_ROWS * 4 + 64;

struct NormParams {
    const void* x;
    const void* r;                     // may be NULL
    void* r_out;                       // r's type, row pitch K; may be r or x themselves
    const void* w;
    uint8_t* out;                      // [K][M]
    float* scale_out;                  // [K / 128][M]
    unsigned int* status;
    long long ldx, ldr;                // row pitches in elements
    int rows, M, K;                    // M: rows rounded up to 16
    int cluster;
    int w_is_bf16;
    float eps, fp8_max;
};

// torch's maximum: NaN if either is (fmaxf drops it), so that a NaN in a row shows in its bytes and scales.
__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// Reduces 16 values per lane, one per row, over the 32 lanes: the halving butterfly of quantize.cuh (16 shuffles).  Lanes 2 r
// and 2 r + 1 return row r's.
template <class Op>
__device__ __forceinline__ float reduce_16_rows(const float (&a)[16], int lane, Op op)
{
    const bool b4 = (lane & 16) != 0, b3 = (lane & 8) != 0, b2 = (lane & 4) != 0, b1 = (lane & 2) != 0;
    float h8[8], h4[4], h2[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float give = b4 ? a[j] : a[j + 8], keep = b4 ? a[j + 8] : a[j];
        h8[j] = op(keep, __shfl_xor_sync(0xffffffffu, give, 16));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float give = b3 ? h8[j] : h8[j + 4], keep = b3 ? h8[j + 4] : h8[j];
        h4[j] = op(keep, __shfl_xor_sync(0xffffffffu, give, 8));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float give = b2 ? h4[j] : h4[j + 2], keep = b2 ? h4[j + 2] : h4[j];
        h2[j] = op(keep, __shfl_xor_sync(0xffffffffu, give, 4));
    }
    const float give = b1 ? h2[0] : h2[1], keep = b1 ? h2[1] : h2[0];
    const float one = op(keep, __shfl_xor_sync(0xffffffffu, give, 2));
    return op(one, __shfl_xor_sync(0xffffffffu, one, 1));
}

typedef unsigned long long f32x2;      // two fp32 values, the operand of the packed instructions

__device__ __forceinline__ f32x2 mul_f32x2(f32x2 a, f32x2 b)
{
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 add_f32x2(f32x2 a, f32x2 b)
{
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Four consecutive elements of a type, and as two pairs of fp32.
template <class T>
struct Quad;
template <>
struct Quad<float> {
    uint4 v;
    __device__ __forceinline__ void from_global(const void* p, long long at) { v = __ldcs(reinterpret_cast<const uint4*>(static_cast<const float*>(p) + at)); }
    __device__ __forceinline__ void from_shared(const void* p) { v = *static_cast<const uint4*>(p); }
    __device__ __forceinline__ f32x2 pair(int j) const
    {
        return j ? (static_cast<f32x2>(v.w) << 32 | v.z) : (static_cast<f32x2>(v.y) << 32 | v.x);
    }
    static __device__ __forceinline__ void store(void* p, long long at, f32x2 a, f32x2 b)
    {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + at) = make_float4(f32x2_lo(a), f32x2_hi(a), f32x2_lo(b), f32x2_hi(b));
    }
};
template <>
struct Quad<__nv_bfloat16> {
    uint2 v;
    __device__ __forceinline__ void from_global(const void* p, long long at) { v = __ldcs(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + at)); }
    __device__ __forceinline__ void from_shared(const void* p) { v = *static_cast<const uint2*>(p); }
    __device__ __forceinline__ f32x2 pair(int j) const
    {
        const uint32_t w = j ? v.y : v.x;
        return static_cast<f32x2>(w & 0xffff0000u) << 32 | (w << 16);
    }
    static __device__ __forceinline__ void store(void* p, long long at, f32x2 a, f32x2 b)
    {
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + at) =
            make_uint2(pack_bf16x2(f32x2_lo(a), f32x2_hi(a)), pack_bf16x2(f32x2_lo(b), f32x2_hi(b)));
    }
};

// s = x + r of 16 rows and four columns.  From shared memory, where the rows behind the last hold zeros ...
template <class X, class R>
__device__ __forceinline__ void norm_read_shared(const uint8_t* xs, const uint8_t* rs, int width, int col, f32x2 (&s)[16][2])
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        Quad<X> x;
        x.from_shared(xs + (i * width + col) * static_cast<int>(sizeof(X)));
        s[i][0] = x.pair(0);
        s[i][1] = x.pair(1);
        if constexpr (!std::is_void<R>::value) {
            Quad<R> r;
            r.from_shared(rs + (i * width + col) * static_cast<int>(sizeof(R)));
            s[i][0] = add_f32x2(s[i][0], r.pair(0));
            s[i][1] = add_f32x2(s[i][1], r.pair(1));
        }
    }
}
// ... and from global memory.
template <class X, class R>
__device__ __forceinline__ void norm_read(const NormParams& p, int r0, int k, f32x2 (&s)[16][2])
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        Quad<X> x{};
        if (r0 + i < p.rows) x.from_global(p.x, (r0 + i) * p.ldx + k);
        s[i][0] = x.pair(0);
        s[i][1] = x.pair(1);
    }
    if constexpr (!std::is_void<R>::value) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            Quad<R> r{};
            if (r0 + i < p.rows) r.from_global(p.r, (r0 + i) * p.ldr + k);
            s[i][0] = add_f32x2(s[i][0], r.pair(0));
            s[i][1] = add_f32x2(s[i][1], r.pair(1));
        }
    }
}

__device__ __forceinline__ float sum_of_squares(f32x2 a, f32x2 b)
{
    const f32x2 q = ptx::fma_f32x2(b, b, mul_f32x2(a, a));
    return f32x2_lo(q) + f32x2_hi(q);
}

__device__ __forceinline__ void norm_weights(const NormParams& p, int k, f32x2 (&w)[2])
{
    if (p.w_is_bf16) {
        Quad<__nv_bfloat16> q;
        q.v = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.w) + k));
        w[0] = q.pair(0);
        w[1] = q.pair(1);
    } else {
        Quad<float> q;
        q.v = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(p.w) + k));
        w[0] = q.pair(0);
        w[1] = q.pair(1);
    }
}

// s -> r_out; s = s * w; returns the largest |s * w| of the block in row lane / 2.
template <class R>
__device__ __forceinline__ float norm_weigh(const NormParams& p, int r0, int k, int lane, const f32x2 (&w)[2], f32x2 (&s)[16][2])
{
    float amax[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if constexpr (!std::is_void<R>::value)
            if (r0 + i < p.rows) Quad<R>::store(p.r_out, static_cast<long long>(r0 + i) * p.K + k, s[i][0], s[i][1]);
        s[i][0] = mul_f32x2(s[i][0], w[0]);
        s[i][1] = mul_f32x2(s[i][1], w[1]);
        amax[i] = max_nan(max_nan(fabsf(f32x2_lo(s[i][0])), fabsf(f32x2_hi(s[i][0]))),
                          max_nan(fabsf(f32x2_lo(s[i][1])), fabsf(f32x2_hi(s[i][1]))));
    }
    return reduce_16_rows(amax, lane, [](float a, float b) { return max_nan(a, b); });
}

// The bytes and scales of one 16 x 128 block from t = s * w.  rstd, amax: 1 / rms and the largest |t| of row lane / 2.
__device__ __forceinline__ void norm_store(const NormParams& p, int r0, int kb, int lane, const f32x2 (&t)[16][2], float rstd, float amax)
{
    // the rows behind the last are zeros whatever eps is
    const float rs = r0 + (lane >> 1) < p.rows ? rstd : 0.0f;
    const float m = max_nan(__fmul_rn(amax, rs), 1e-12f);
    const float sc = __fmul_rn(__fdiv_rn(1.0f, m), p.fp8_max);                       // as in quantize.cuh
    if ((lane & 1) == 0) p.scale_out[static_cast<size_t>(kb) * p.M + r0 + (lane >> 1)] = __fdiv_rn(1.0f, sc);
    // No product below may round to more than fp8_max: the factor is five roundings off at most, and eight are taken off where the
    // largest product shows one.
    float mine = __fmul_rn(rs, sc);
    if (__fmul_rn(amax, mine) > p.fp8_max) mine = __fmul_rn(mine, 1.0f - 0x1p-21f);
    uint8_t* dst = p.out + static_cast<size_t>(kb * 128 + lane * 4) * p.M + r0;
    uint32_t q[4][4];                                                                // [column][four rows]
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float v[4][4];                                                               // [row][column]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = __shfl_sync(0xffffffffu, mine, 2 * (4 * g + i));
            const f32x2 ff = pack_f32x2(f, f), a = mul_f32x2(t[4 * g + i][0], ff), b = mul_f32x2(t[4 * g + i][1], ff);
            v[i][0] = f32x2_lo(a); v[i][1] = f32x2_hi(a); v[i][2] = f32x2_lo(b); v[i][3] = f32x2_hi(b);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j][g] = cvt_e4m3x2(v[0][j], v[1][j]) | (cvt_e4m3x2(v[2][j], v[3][j]) << 16);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(dst + static_cast<size_t>(j) * p.M) = make_uint4(q[j][0], q[j][1], q[j][2], q[j][3]);
}

__device__ __forceinline__ float norm_rstd(const NormParams& p, float total)
{
    return __frsqrt_rn(__fadd_rn(__fdiv_rn(total, static_cast<float>(p.K)), p.eps));
}

// Rows that a cluster holds.  grid = a multiple of the cluster size, 32 threads per block of a CTA's share.
template <class X, class R>
__global__ void __launch_bounds__(32 * NORM_MOST_WARPS, 1)
rmsnorm_quantize_kernel(const NormParams p)
{
    constexpr bool ADD = !std::is_void<R>::value;
    using RT = typename std::conditional<ADD, R, float>::type;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, C = p.cluster;
    const int rank = C > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const int width = warps * 128, KB = p.K / 128, kb = rank * warps + warp;
    const int cols = min(warps, KB - rank * warps) * 128;              // of this CTA's share, at least one block
    uint8_t* xs = smem;
    uint8_t* rs = xs + NORM_ROWS * width * sizeof(X);
    float* warp_sums = reinterpret_cast<float*>(rs + (ADD ? NORM_ROWS * width * sizeof(RT) : 0));       // [2][warps][16]
    float* cta_sums = warp_sums + 2 * NORM_MOST_WARPS * NORM_ROWS;                                      // [2][CTAs][16]
    uint64_t* bars = reinterpret_cast<uint64_t*>(cta_sums + 2 * NORM_MAX_CLUSTER * NORM_ROWS);          // rows, sums even, sums odd
    const uint32_t rows_bar = ptx::smem_u32(bars), sums_bar = rows_bar + 8;
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(bars + 3);

    const int groups = p.M / NORM_ROWS, step = static_cast<int>(gridDim.x) / C;
    // 16 rows of x and of r, a copy per row, by warp 0
    auto request = [&](int g) {
        const int rows = min(NORM_ROWS, p.rows - g * NORM_ROWS);
        if (rows < NORM_ROWS) {                      // the last 16 rows: zeros behind the last
            for (uint32_t i = static_cast<uint32_t>(rows * width) * sizeof(X) + lane * 16; i < NORM_ROWS * width * sizeof(X); i += 512)
                *reinterpret_cast<uint4*>(xs + i) = make_uint4(0u, 0u, 0u, 0u);
            if (ADD)
                for (uint32_t i = static_cast<uint32_t>(rows * width) * sizeof(RT) + lane * 16; i < NORM_ROWS * width * sizeof(RT); i += 512)
                    *reinterpret_cast<uint4*>(rs + i) = make_uint4(0u, 0u, 0u, 0u);
            __syncwarp();
        }
        if (lane == 0) ptx::mbar_arrive_expect_tx(rows_bar, static_cast<uint32_t>(rows * cols * (sizeof(X) + (ADD ? sizeof(RT) : 0))));
        __syncwarp();
        const long long row = g * NORM_ROWS + (lane & 15), col = rank * width;
        if ((lane & 15) < rows) {
            if (lane < 16)
                ptx::bulk_load(ptx::smem_u32(xs) + (lane & 15) * width * static_cast<int>(sizeof(X)),
                               static_cast<const X*>(p.x) + row * p.ldx + col, static_cast<uint32_t>(cols * sizeof(X)), rows_bar);
            else if (ADD)
                ptx::bulk_load(ptx::smem_u32(rs) + (lane & 15) * width * static_cast<int>(sizeof(RT)),
                               static_cast<const RT*>(p.r) + row * p.ldr + col, static_cast<uint32_t>(cols * sizeof(RT)), rows_bar);
        }
    };
    if (threadIdx.x == 0) {
        ptx::mbar_init(rows_bar, 1);
        ptx::mbar_init(sums_bar, 1);
        ptx::mbar_init(sums_bar + 8, 1);
        *abort_flag = 0u;
        ptx::fence_mbar_init();
    }
    __syncthreads();
    if (C > 1) ptx::cluster_arrive();                // waited for before anything is sent to a peer: its barriers exist
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    if (warp == 0) request(static_cast<int>(blockIdx.x) / C);          // grid <= C * groups
    if (C > 1) ptx::cluster_wait();

    auto cta_sum = [&](const float* ws, int row) {
        float v[NORM_MOST_WARPS], sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NORM_MOST_WARPS; ++j) v[j] = j < warps ? ws[j * NORM_ROWS + row] : 0.0f;
#pragma unroll
        for (int j = 0; j < NORM_MOST_WARPS; ++j) sum += v[j];
        return sum;
    };
    const bool mine = kb < KB;
    const int k = kb * 128 + lane * 4, col = warp * 128 + lane * 4;
    f32x2 w[2] = {0ull, 0ull};
    if (mine) norm_weights(p, k, w);
    bool ok = true;
    uint32_t n = 0;
    for (int g = static_cast<int>(blockIdx.x) / C; g < groups; g += step, ++n) {
        const int r0 = g * NORM_ROWS;
        const uint32_t odd = n & 1u;
        ok = ok && wait_bounded(rows_bar, odd, abort_flag, p.status, DS_TIMEOUT_STAGE_FULL);
        f32x2 t[16][2];
        float part[16];
        if (mine) norm_read_shared<X, R>(xs, rs, width, col, t);
#pragma unroll
        for (int i = 0; i < 16; ++i) part[i] = mine ? sum_of_squares(t[i][0], t[i][1]) : 0.0f;
        const float sum = reduce_16_rows(part, lane, [](float a, float b) { return a + b; });
        float* ws = warp_sums + odd * NORM_MOST_WARPS * NORM_ROWS;
        if ((lane & 1) == 0) ws[warp * NORM_ROWS + (lane >> 1)] = sum;
        // everybody has read the rows, and the sums are there.  A set of sums is written again two rounds later, which the barrier of
        // the round between keeps apart (for the peers': a CTA sends round n + 2 after it has round n + 1 from everybody).
        ok = __syncthreads_and(ok);
        if (!ok) break;
        if (warp == 0 && g + step < groups) request(g + step);
        float total = 0.0f;
        if (C > 1) {
            const uint32_t bar = sums_bar + 8u * odd;
            if (threadIdx.x == 0) ptx::mbar_arrive_expect_tx(bar, static_cast<uint32_t>(C * NORM_ROWS * 4));
            for (int i = static_cast<int>(threadIdx.x); i < NORM_ROWS * C; i += static_cast<int>(blockDim.x)) {
                const int row = i % NORM_ROWS;
                const uint32_t peer = static_cast<uint32_t>(i / NORM_ROWS);
                ptx::st_async_f32(ptx::mapa(ptx::smem_u32(cta_sums + (odd * NORM_MAX_CLUSTER + rank) * NORM_ROWS + row), peer), cta_sum(ws, row),
                                  ptx::mapa(bar, peer));
            }
        } else {
            total = cta_sum(ws, lane >> 1);
        }
        float amax = 0.0f;
        if (mine) amax = norm_weigh<R>(p, r0, k, lane, w, t);
        if (C > 1) {
            ok = wait_bounded(sums_bar + 8u * odd, (n >> 1) & 1u, abort_flag, p.status, DS_TIMEOUT_PEER_PARTIAL);
            ok = __all_sync(0xffffffffu, ok);
            float v[NORM_MAX_CLUSTER];
#pragma unroll
            for (int c = 0; c < NORM_MAX_CLUSTER; ++c) v[c] = c < C ? cta_sums[(odd * NORM_MAX_CLUSTER + c) * NORM_ROWS + (lane >> 1)] : 0.0f;
#pragma unroll
            for (int c = 0; c < NORM_MAX_CLUSTER; ++c) total += v[c];
        }
        if (mine && ok) norm_store(p, r0, kb, lane, t, norm_rstd(p, total), amax);
    }
    if (!ok) {
        // giving up with copies possibly in flight: a bounded time to land
        const long long c0 = clock64();
        while (clock64() - c0 < 2000000LL) __nanosleep(1000);
    }
    if (C > 1) ptx::cluster_sync();                  // what this CTA has sent has arrived before a peer leaves
}

// Rows that no cluster holds: 16 rows to a cluster of eight CTAs of eight warps, each of which walks its blocks twice.
template <class X, class R>
__global__ void __launch_bounds__(32 * NORM_WARPS, 2)
rmsnorm_quantize_long_kernel(const NormParams p)
{
    __shared__ float warp_sums[NORM_WARPS][NORM_ROWS];
    __shared__ float cta_sums[NORM_MAX_CLUSTER][NORM_ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(ptx::cluster_ctarank());
    const int r0 = static_cast<int>(blockIdx.x) / NORM_MAX_CLUSTER * NORM_ROWS;
    const int KB = p.K / 128, kb0 = rank * NORM_WARPS + warp;
    constexpr int STEP = NORM_MAX_CLUSTER * NORM_WARPS;
    ptx::cluster_arrive();                           // waited for before anything is written into a peer: it has started
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    f32x2 t[16][2];
    float part[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) part[i] = 0.0f;
    for (int kb = kb0; kb < KB; kb += STEP) {
        norm_read<X, R>(p, r0, kb * 128 + lane * 4, t);
#pragma unroll
        for (int i = 0; i < 16; ++i) part[i] += sum_of_squares(t[i][0], t[i][1]);
    }
    const float sum = reduce_16_rows(part, lane, [](float a, float b) { return a + b; });
    if ((lane & 1) == 0) warp_sums[warp][lane >> 1] = sum;
    __syncthreads();
    ptx::cluster_wait();
    if (threadIdx.x < NORM_ROWS * NORM_MAX_CLUSTER) {
        const int row = threadIdx.x % NORM_ROWS;
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < NORM_WARPS; ++i) mine += warp_sums[i][row];
        ptx::st_shared_cluster_f32(ptx::mapa(ptx::smem_u32(&cta_sums[rank][row]), threadIdx.x / NORM_ROWS), mine);
    }
    ptx::cluster_sync();
    float total = 0.0f;
#pragma unroll
    for (int c = 0; c < NORM_MAX_CLUSTER; ++c) total += cta_sums[c][lane >> 1];
    const float rstd = norm_rstd(p, total);
    for (int kb = kb0; kb < KB; kb += STEP) {
        const int k = kb * 128 + lane * 4;
        norm_read<X, R>(p, r0, k, t);
        f32x2 w[2];
        norm_weights(p, k, w);
        const float amax = norm_weigh<R>(p, r0, k, lane, w, t);
        norm_store(p, r0, kb, lane, t, rstd, amax);
    }
}

}  // namespace fp8bs
