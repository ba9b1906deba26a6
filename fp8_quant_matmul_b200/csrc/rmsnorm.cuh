// Root-mean-square norm with the residual's addition in front of it and the GEMM's A operand behind it:
//     s = x + r                               (fp32; r_out = s rounded to r's type)
//     y = s * w / sqrt(mean(s^2) + eps)       (fp32)
//     one scale per row and 128 columns of y, e4m3 bytes A[m + M*k], inverse scales a_scale[m + M*kb] (as quantize.cuh)
// The norm and the scales see the sum before it is rounded to r's type: there is one rounding between the inputs and each output.
//
// The norm needs a whole row before the first byte can be written, and the bytes of a column of A want many rows side by side.
// So 16 rows are spread over a cluster: a warp owns 16 rows x 128 columns, one scale block of each row, in registers (a lane four
// consecutive columns of every row); the warps of up to eight CTAs hold the row, which is read once.  A warp sends its rows' sums of squares
// to every CTA (16 x 4 bytes each, st.async onto an mbarrier of the receiver that counts all blocks' bytes) and adds up all blocks' itself, in
// a fixed order.  All that does not need the norm is done before: s * w and its largest magnitude per row and block; after it one factor
// per row and block is left, 1 / rms times the scale.  The 16 rows of a lane's column are 16 neighbouring bytes of A, so the
// quantised values leave straight from the registers, two groups of 16 rows (a 32-byte sector) at a time.
// The clusters are persistent and a warp's rows arrive by TMA, a box of 16 x 128 (zeros behind the last row) on an mbarrier of its own: the next
// box is requested as soon as this one is in registers.  The warps of a CTA have nothing else to do with one another; with copies per row for the
// CTA as a whole, two barriers and sums per CTA a round took up to 15 % longer.
// Measured (CUDA graph, cold inputs, outputs of their own): 4096 x 7168 bf16 43-44 us with residual (206 MB: 4.7 TB/s; a copy reaches 6.4), 28
// without (3.2 TB/s); 6144 x 4608 bf16 with residual 39 (5.1), fp32 with residual 67 (5.5); one row of 7168 3.3, with residual 3.9, the chain of a
// launch and one round.  What bounds it: in bf16 the instructions of a round and the waits between them, 16 warps per SM at most
// with 128 registers each; in fp32 nearly the memory.
// Rows that do not fit (more than 16384 columns; in fp32 with an fp32 residual more than 13312) are read twice: 512 x
// 20480 bf16 23-24 us, with residual 34-35 (5.0 and 11.5 at a copy's rate, reading once).
#pragma once
#include "quantize.cuh"
#include <type_traits>

namespace fp8bs {

constexpr int NORM_ROWS = 16;              // rows of a cluster
constexpr int NORM_WARPS = 8;              // per CTA of the kernel for long rows
constexpr int NORM_MOST_WARPS = 16;        // of the other
constexpr int NORM_MAX_CLUSTER = 8;        // the portable limit
constexpr int NORM_SMEM_LIMIT = 227 * 1024;
// behind the buffers: two sets of sums, barriers, control word
constexpr int norm_fixed_smem(int blocks) { return 2 * blocks * NORM_ROWS * 4 + (2 + NORM_MOST_WARPS) * 8 + 16; }

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
    float inv_K, eps, fp8_max;
};

// Adds up 16 values per lane, one per row, over the 32 lanes: the halving butterfly of quantize.cuh (16 shuffles).  Lanes 2 r and
// 2 r + 1 return row r's.
__device__ __forceinline__ float sum_16_rows(const float (&a)[16], int lane)
{
    const bool b4 = (lane & 16) != 0, b3 = (lane & 8) != 0, b2 = (lane & 4) != 0, b1 = (lane & 2) != 0;
    float h8[8], h4[4], h2[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float give = b4 ? a[j] : a[j + 8], keep = b4 ? a[j + 8] : a[j];
        h8[j] = keep + __shfl_xor_sync(0xffffffffu, give, 16);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float give = b3 ? h8[j] : h8[j + 4], keep = b3 ? h8[j + 4] : h8[j];
        h4[j] = keep + __shfl_xor_sync(0xffffffffu, give, 8);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float give = b2 ? h4[j] : h4[j + 2], keep = b2 ? h4[j + 2] : h4[j];
        h2[j] = keep + __shfl_xor_sync(0xffffffffu, give, 4);
    }
    const float give = b1 ? h2[0] : h2[1], keep = b1 ? h2[1] : h2[0];
    const float one = keep + __shfl_xor_sync(0xffffffffu, give, 2);
    return one + __shfl_xor_sync(0xffffffffu, one, 1);
}

using ptx::add_f32x2;
using ptx::mul_f32x2;
typedef unsigned long long f32x2;      // two fp32 values, the operand of the packed instructions

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

// Which of the 16 rows a lane answers for once the sums are in (lanes that differ in bit 2: the same one), and the first lane that does.
__device__ __forceinline__ int row_of(int lane) { return 4 * (lane & 3) + (lane >> 3); }
__device__ constexpr int lane_of(int row) { return (row >> 2) | ((row & 3) << 3); }

// 1 / x and 1 / sqrt(x): the hardware's approximation (2^-22) and a step of Newton's method, off by 2^-24 and 1.5 times that.  Without the branches of
// the exactly rounded forms, which were a twelfth of a round.  Where the approximation is 0 or infinite the step gives NaN, and it stays.
__device__ __forceinline__ float reciprocal(float x)
{
    float y;
    asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    const float e = __fmaf_rn(-x, y, 1.0f);
    return fabsf(e) < 1.0f ? __fmaf_rn(y, e, y) : y;
}
__device__ __forceinline__ float reciprocal_root(float x)
{
    float y;
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    const float e = __fmaf_rn(-__fmul_rn(x, y), y, 1.0f);
    return fabsf(e) < 1.0f ? __fmaf_rn(__fmul_rn(0.5f, y), e, y) : y;
}

// s -> r_out (`rows` of the 16); s = s * w; returns the largest |s * w| of the block in row row_of(lane).
template <class R>
__device__ __forceinline__ float norm_weigh(const NormParams& p, int r0, int k, int lane, const f32x2 (&w)[2], f32x2 (&s)[16][2])
{
    if constexpr (!std::is_void<R>::value) {
        const long long at = static_cast<long long>(r0) * p.K + k;
        const int rows = p.rows - r0;
        if (rows >= NORM_ROWS) {
#pragma unroll
            for (int i = 0; i < 16; ++i) Quad<R>::store(p.r_out, at + static_cast<long long>(i) * p.K, s[i][0], s[i][1]);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < rows) Quad<R>::store(p.r_out, at + static_cast<long long>(i) * p.K, s[i][0], s[i][1]);
        }
    }
    float mine = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        s[i][0] = mul_f32x2(s[i][0], w[0]);
        s[i][1] = mul_f32x2(s[i][1], w[1]);
        const float m = warp_absmax_nan(max_nan(max_nan(fabsf(f32x2_lo(s[i][0])), fabsf(f32x2_hi(s[i][0]))),
                                                max_nan(fabsf(f32x2_lo(s[i][1])), fabsf(f32x2_hi(s[i][1])))));
        if (row_of(lane) == i) mine = m;
    }
    return mine;
}

// What t = s * w is multiplied with in row row_of(lane) of a 16 x 128 block before it is rounded to 8 bits; stores the inverse scale.
// rstd, amax: 1 / rms and the largest |t| of that row.
__device__ __forceinline__ float norm_factor(const NormParams& p, int r0, int kb, int lane, float rstd, float amax)
{
    // the rows behind the last have the scale of zeros, whatever eps and the weight are, and their bytes are masked
    const int row = row_of(lane);
    const float m = r0 + row < p.rows ? max_nan(__fmul_rn(amax, rstd), 1e-12f) : 1e-12f;
    const float sc = __fmul_rn(reciprocal(m), p.fp8_max);                            // as in quantize.cuh
    if ((lane & 4) == 0) p.scale_out[static_cast<size_t>(kb) * p.M + r0 + row] = reciprocal(sc);
    // No product may round to more than fp8_max: the factor is five roundings off at most, and eight are taken off where the
    // largest product shows one.
    const float f = __fmul_rn(rstd, sc);
    return __fmul_rn(amax, f) > p.fp8_max ? __fmul_rn(f, 1.0f - 0x1p-21f) : f;
}
// t = t * factor
__device__ __forceinline__ void norm_scale(float factor, f32x2 (&t)[16][2])
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float f = __shfl_sync(0xffffffffu, factor, lane_of(i));
        t[i][0] = mul_f32x2(t[i][0], pack_f32x2(f, f));
        t[i][1] = mul_f32x2(t[i][1], pack_f32x2(f, f));
    }
}
// Which bytes of a column's 16 are rows that exist: those behind the last are +0, which a product with a negative weight, or one that is not
// finite, is not.
__device__ __forceinline__ void norm_rows_mask(int rows, uint32_t (&mask)[4])
{
#pragma unroll
    for (int g = 0; g < 4; ++g) asm("shl.b32 %0, -1, %1;" : "=r"(mask[g]) : "r"(max(8 * (rows - 4 * g), 0)));      // by 32 or more: 0
#pragma unroll
    for (int g = 0; g < 4; ++g) mask[g] = ~mask[g];
}
// The bytes of column j of a lane's four, 16 rows; those that exist of the last 16 (WHOLE false).
template <bool WHOLE>
__device__ __forceinline__ void norm_bytes(const f32x2 (&t)[16][2], const uint32_t (&mask)[4], int j, uint32_t (&q)[4])
{
    auto v = [&](int i) { return (j & 1) ? f32x2_hi(t[i][j >> 1]) : f32x2_lo(t[i][j >> 1]); };
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        q[g] = cvt_e4m3x2(v(4 * g), v(4 * g + 1)) | (cvt_e4m3x2(v(4 * g + 2), v(4 * g + 3)) << 16);
        if constexpr (!WHOLE) q[g] &= mask[g];
    }
}

__device__ __forceinline__ void store_16(uint8_t* dst, const uint32_t (&q)[4])
{
    *reinterpret_cast<uint4*>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
}
__device__ __forceinline__ void store_32(uint8_t* dst, const uint32_t (&a)[4], const uint32_t (&b)[4])
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(__cvta_generic_to_global(dst)), "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "r"(b[2]), "r"(b[3])
                 : "memory");
}

__device__ __forceinline__ float norm_rstd(const NormParams& p, float total)
{
    return reciprocal_root(__fadd_rn(__fmul_rn(total, p.inv_K), p.eps));
}

// The sum over all blocks of row row_of(lane); sums: [KB][16].  A lane adds up four rows of every eighth block, then the lanes theirs.
__device__ __forceinline__ float sum_of_blocks(const float* sums, int KB, int lane)
{
    const float4* from = reinterpret_cast<const float4*>(sums) + (lane & 3);
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j0 = lane >> 2; j0 < KB; j0 += 32) {
        float4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = j0 + 8 * j < KB ? from[(j0 + 8 * j) * (NORM_ROWS / 4)] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) a = make_float4(a.x + v[j].x, a.y + v[j].y, a.z + v[j].z, a.w + v[j].w);
    }
    const bool b4 = (lane & 16) != 0, b3 = (lane & 8) != 0;
    const float h0 = (b4 ? a.z : a.x) + __shfl_xor_sync(0xffffffffu, b4 ? a.x : a.z, 16);
    const float h1 = (b4 ? a.w : a.y) + __shfl_xor_sync(0xffffffffu, b4 ? a.y : a.w, 16);
    const float one = (b3 ? h1 : h0) + __shfl_xor_sync(0xffffffffu, b3 ? h0 : h1, 8);
    return one + __shfl_xor_sync(0xffffffffu, one, 4);
}

// Rows that a cluster holds.  grid = a multiple of the cluster size, 32 threads per block of a CTA's share.  x_map, r_map: [rows, K] in boxes of
// 16 rows x 128 columns, zeros behind the last row (r_map is not looked at without R).
template <class X, class R>
__global__ void __launch_bounds__(32 * NORM_MOST_WARPS, 1)
rmsnorm_quantize_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap r_map, const NormParams p)
{
    constexpr bool ADD = !std::is_void<R>::value;
    using RT = typename std::conditional<ADD, R, float>::type;
    constexpr int X_BYTES = NORM_ROWS * 128 * static_cast<int>(sizeof(X)), R_BYTES = ADD ? NORM_ROWS * 128 * static_cast<int>(sizeof(RT)) : 0;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, C = p.cluster;
    const int rank = C > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const int KB = p.K / 128, kb = rank * warps + warp;
    const bool mine = kb < KB;                                         // of every CTA's warps the first has a block at least
    uint8_t* const xs = smem + warp * X_BYTES;
    uint8_t* const rs = smem + warps * X_BYTES + warp * R_BYTES;
    float* const sums = reinterpret_cast<float*>(smem + warps * (X_BYTES + R_BYTES));                   // [2][KB][16]
    uint64_t* const bars = reinterpret_cast<uint64_t*>(sums + 2 * KB * NORM_ROWS);                      // sums even, sums odd, rows of each warp
    const uint32_t sums_bar = ptx::smem_u32(bars), rows_bar = sums_bar + 16u + 8u * static_cast<uint32_t>(warp);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(bars + 2 + warps);

    // the groups of 16 rows that this cluster does, one after the other
    const int groups = p.M / NORM_ROWS, clusters = static_cast<int>(gridDim.x) / C, id = static_cast<int>(blockIdx.x) / C;
    const int g0 = static_cast<int>(static_cast<long long>(groups) * id / clusters);
    const int g1 = static_cast<int>(static_cast<long long>(groups) * (id + 1) / clusters);
    // this warp's block of 16 rows, of x and of r
    auto request = [&](int g) {
        if (ptx::elect_one()) {
            ptx::mbar_arrive_expect_tx(rows_bar, X_BYTES + R_BYTES);
            ptx::tma_load_2d(ptx::smem_u32(xs), &x_map, kb * 128, g * NORM_ROWS, rows_bar);
            if (ADD) ptx::tma_load_2d(ptx::smem_u32(rs), &r_map, kb * 128, g * NORM_ROWS, rows_bar);
        }
        __syncwarp();
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 + warps; ++i) ptx::mbar_init(sums_bar + 8u * static_cast<uint32_t>(i), 1);
        *abort_flag = 0u;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&x_map);
        if (ADD) ptx::prefetch_tensormap(&r_map);
    }
    __syncthreads();
    if (C > 1) ptx::cluster_arrive();                // waited for before anything is sent to a peer: its barriers exist
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    if (mine) request(g0);                           // clusters <= groups
    if (C > 1) ptx::cluster_wait();

    const int k = kb * 128 + lane * 4;
    f32x2 w[2] = {0ull, 0ull};
    if (mine) norm_weights(p, k, w);
    bool ok = true;
    uint32_t n = 0;
    // Bytes of a column leave 32 at a time: the first 16 of an aligned 32 wait in registers for the next 16 rows.  Which rows are first
    // depends on the column where a column is not a multiple of 32 bytes long.
    uint8_t* const dst = p.out + static_cast<size_t>(k) * p.M;
    uint32_t held[4][4];
    const uint32_t start = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(dst) >> 4), long_by = static_cast<uint32_t>(groups);
    for (int g = mine ? g0 : g1; g < g1; ++g, ++n) {
        const int r0 = g * NORM_ROWS;
        const uint32_t odd = n & 1u, bar = sums_bar + 8u * odd;
        float* const row_sums = sums + odd * static_cast<uint32_t>(KB * NORM_ROWS);
        ok = wait_bounded(rows_bar, odd, abort_flag, p.status, DS_TIMEOUT_STAGE_FULL);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        f32x2 t[16][2];
        norm_read_shared<X, R>(xs, rs, 128, lane * 4, t);
        float part[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) part[i] = sum_of_squares(t[i][0], t[i][1]);
        const float sum = sum_16_rows(part, lane);
        // The box may be filled again once its values are in registers, which nothing says but an instruction that needs them: a load may still wait
        // for its turn when a copy that was issued after it arrives.  A sum of squares is never -0, so the vote is always for it.
        if (__any_sync(0xffffffffu, __float_as_uint(sum) != 0x80000000u) && g + 1 < g1) request(g + 1);
        // The block's 16 sums to every CTA, four of them from a lane.  A set of sums is written again two rounds later: whoever sends round n + 2
        // has round n + 1 from every warp, which sent it after it had read the sums of round n.
        {
            const int q = lane & 3;
            const uint32_t peer = static_cast<uint32_t>(lane >> 2);
            float4 v;
            v.x = __shfl_sync(0xffffffffu, sum, 8 * q);
            v.y = __shfl_sync(0xffffffffu, sum, 8 * q + 2);
            v.z = __shfl_sync(0xffffffffu, sum, 8 * q + 4);
            v.w = __shfl_sync(0xffffffffu, sum, 8 * q + 6);
            if (static_cast<int>(peer) < C)
                ptx::st_async_v4(ptx::mapa(ptx::smem_u32(row_sums + kb * NORM_ROWS + 4 * q), peer), v, ptx::mapa(bar, peer));
            if (threadIdx.x == 0) ptx::mbar_arrive_expect_tx(bar, static_cast<uint32_t>(KB * NORM_ROWS * 4));
            __syncwarp();
        }
        const float amax = norm_weigh<R>(p, r0, k, lane, w, t);
        ok = wait_bounded(bar, (n >> 1) & 1u, abort_flag, p.status, DS_TIMEOUT_PEER_PARTIAL);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const float total = sum_of_blocks(row_sums, KB, lane);
        norm_scale(norm_factor(p, r0, kb, lane, norm_rstd(p, total), amax), t);
        // FIRST bit j: the bytes of column j are the first 16 of an aligned 32.  (The mask in every round, with its registers, was 4 % of 4096 x 7168 bf16
        // without residual.)
        auto leave_rows = [&](auto first, auto whole) {
            constexpr int FIRST = decltype(first)::value;
            constexpr bool WHOLE = decltype(whole)::value;
            uint32_t mask[4];
            if constexpr (!WHOLE) norm_rows_mask(p.rows - r0, mask);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint8_t* to = dst + static_cast<size_t>(j) * p.M + r0;
                if ((FIRST >> j) & 1) {
                    norm_bytes<WHOLE>(t, mask, j, held[j]);
                    if (g + 1 == g1) store_16(to, held[j]);
                } else {
                    uint32_t q[4];
                    norm_bytes<WHOLE>(t, mask, j, q);
                    if (g > g0) store_32(to - 16, held[j], q);
                    else store_16(to, q);
                }
            }
        };
        auto leave = [&](auto first) {
            if (p.rows - r0 >= NORM_ROWS) leave_rows(first, std::true_type{});
            else leave_rows(first, std::false_type{});
        };
        const uint32_t even = (start + static_cast<uint32_t>(g)) & 1u, next = (even + long_by) & 1u;     // of columns 0, 2 and 1, 3
        if (even == 0u && next == 0u) leave(std::integral_constant<int, 15>{});
        else if (even != 0u && next != 0u) leave(std::integral_constant<int, 0>{});
        else if (even == 0u) leave(std::integral_constant<int, 5>{});
        else leave(std::integral_constant<int, 10>{});
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
    const float sum = sum_16_rows(part, lane);
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
    for (int c = 0; c < NORM_MAX_CLUSTER; ++c) total += cta_sums[c][row_of(lane)];
    const float rstd = norm_rstd(p, total);
    for (int kb = kb0; kb < KB; kb += STEP) {
        const int k = kb * 128 + lane * 4;
        norm_read<X, R>(p, r0, k, t);
        f32x2 w[2];
        norm_weights(p, k, w);
        const float amax = norm_weigh<R>(p, r0, k, lane, w, t);
        norm_scale(norm_factor(p, r0, kb, lane, rstd, amax), t);
        auto leave = [&](auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            uint32_t mask[4];
            if constexpr (!WHOLE) norm_rows_mask(p.rows - r0, mask);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t q[4];
                norm_bytes<WHOLE>(t, mask, j, q);
                store_16(p.out + static_cast<size_t>(k + j) * p.M + r0, q);
            }
        };
        if (p.rows - r0 >= NORM_ROWS) leave(std::true_type{});
        else leave(std::false_type{});
    }
}

}  // namespace fp8bs
