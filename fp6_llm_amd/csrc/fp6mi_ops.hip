// Operators around the FPx linear layer that are the same for every weight format, and the C ABI of all of them (include/fp6mi.h): the gated
// feed-forward block, the input gradient, low-rank adapters beside a projection.  No counterpart in the reference.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "fp6mi_internal.h"
#include "fp6mi_activation.inc"
#include "fp6mi_scale.inc"

namespace {

typedef _Float16 half_t;
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float    v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---------------------------------------------------------------------------------------------------------------
// The gated block element by element: rows of pre-activations in pair order (16 of gate, the same 16 of up, ...).  HBM-bound.
// ---------------------------------------------------------------------------------------------------------------
// The EACH outputs of thread t, which follow one another, as the place and the column of the gate's pre-activations; those of up lie 16 behind.  (A division in 32 bits.)
struct Place { size_t p; uint32_t m; };
template <int EACH> __device__ __forceinline__ Place pair_place(uint32_t t, uint32_t F)
{
    const uint32_t row = F / EACH, n = t / row, r = t - n * row, m = r / (16 / EACH) * 32 + r % (16 / EACH) * EACH;
    return { (size_t)n * 2 * F + m, m };
}

// What the kernels of fp6mi_block.hip do on their way out, for a split product: the outputs from its partial sums, which it adds up in split order, with the bias and, where they are wanted, the pre-activations.
template <int ACT>
__global__ __launch_bounds__(256) void gated_reduce(half_t *__restrict__ out, float *__restrict__ preact, const float *__restrict__ ws, const half_t *__restrict__ bias, size_t count,
                                                    uint32_t F, int splits)
{
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    const size_t   i = (size_t)t * 4, stride = count * 2;
    if (i >= count) return;
    const auto [p, m] = pair_place<4>(t, F);
    v4f          g = { 0.f, 0.f, 0.f, 0.f }, u = g;
#pragma unroll 4
    for (int s = 0; s < splits; s++) {
        g += *reinterpret_cast<const v4f *>(ws + s * stride + p);
        u += *reinterpret_cast<const v4f *>(ws + s * stride + p + 16);
    }
    v4h o;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (bias) g[j] += (float)bias[m + j], u[j] += (float)bias[m + 16 + j];
        o[j] = (half_t)(activation<ACT>(g[j]) * u[j]);
    }
    *reinterpret_cast<v4h *>(out + i) = o;
    if (preact) {
        *reinterpret_cast<v4f *>(preact + p) = g;
        *reinterpret_cast<v4f *>(preact + p + 16) = u;
    }
}

// dg = dh * u * act'(g), du = dh * act(g), in pair order: rounded to fp16 as they are (dpre, unless null) and as their products with the mantissas of the row scales, which
// the product with the weights takes (scaled; one rounding for both instead of one behind the other).  Eight outputs a thread, which makes every
// store 16 bytes wide: 4096 rows of 22016 pre-activations take 148 us (5.5 TB/s; four a thread 213).
template <int ACT>
__global__ __launch_bounds__(256) void gated_grad(half_t *__restrict__ dpre, half_t *__restrict__ scaled, const half_t *__restrict__ dout, const float *__restrict__ preact,
                                                  const half_t *__restrict__ scales, size_t count, uint32_t F)
{
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    const size_t   i = (size_t)t * 8;
    if (i >= count) return;
    const auto [p, m] = pair_place<8>(t, F);
    const v8h d = *reinterpret_cast<const v8h *>(dout + i);
    v8h       cg, cu;
    v4f       g[2], u[2];
    if ((reinterpret_cast<uintptr_t>(scales) & 15u) == 0) { // (they need not be)
        cg = *reinterpret_cast<const v8h *>(scales + m), cu = *reinterpret_cast<const v8h *>(scales + m + 16);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) cg[j] = scales[m + j], cu[j] = scales[m + 16 + j];
    }
#pragma unroll
    for (int h = 0; h < 2; h++) g[h] = *reinterpret_cast<const v4f *>(preact + p + 4 * h), u[h] = *reinterpret_cast<const v4f *>(preact + p + 16 + 4 * h);
    v8h dg, du, sg, su;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float       slope;
        const float a = activation_slope<ACT>(g[j / 4][j % 4], slope), vg = (float)d[j] * u[j / 4][j % 4] * slope, vu = (float)d[j] * a;
        dg[j] = (half_t)vg, du[j] = (half_t)vu;
        sg[j] = (half_t)(vg * (float)scale_mantissa(cg[j])), su[j] = (half_t)(vu * (float)scale_mantissa(cu[j]));
    }
    if (dpre) {
        *reinterpret_cast<v8h *>(dpre + p) = dg;
        *reinterpret_cast<v8h *>(dpre + p + 16) = du;
    }
    *reinterpret_cast<v8h *>(scaled + p) = sg;
    *reinterpret_cast<v8h *>(scaled + p + 16) = su;
}

constexpr size_t kMostOutputs = (size_t)1 << 33; // (a grid has fewer than 2^32 threads, of four outputs each)

template <typename F> int by_activation(int activation, const F &f)
{
    if (activation == FP6MI_ACT_SILU) return f(std::integral_constant<int, FP6MI_ACT_SILU>{});
    if (activation == FP6MI_ACT_GELU) return f(std::integral_constant<int, FP6MI_ACT_GELU>{});
    return f(std::integral_constant<int, FP6MI_ACT_GELU_TANH>{});
}
inline bool known_activation(int a) { return a == FP6MI_ACT_SILU || a == FP6MI_ACT_GELU || a == FP6MI_ACT_GELU_TANH; }

// The launch shape of the gated block: the GEMM's, or the nearest that holds its row tiles in pairs (gemm_stream's odd numbers of them, gemm_tile's single ones) or that its kernels have.
fp6mi::LaunchCfg gated_shape(int E, int Mb, size_t M, size_t N, size_t K, bool grouped)
{
    fp6mi::LaunchCfg c = fp6mi::linear_shape(E, Mb, M, N, K, 1, grouped);
    if (c.kind == 0) {
        c.rt += c.rt & 1;
        if (c.rt == 8 || (c.rt == 6 && c.nt == 2)) c.wk = 4;
        if (c.rt >= 4 && c.wk == 16) c.wk = 8;
        return c;
    }
    if (c.kind == 2 && c.wk == 4 && c.nt == 2) return { 1, 2, 2, 4, 2 };                           // gemm_ws 256 x 32
    if ((c.kind == 2 && c.wr == 2) || (c.kind == 1 && c.nt == 8))                                    // gemm_prefill, gemm_tile 256 x 128; the wide tiles end at K = 2^20
        return K <= (size_t)1 << 20 ? fp6mi::LaunchCfg{ 2, 8, 4, 4, 1 } : fp6mi::LaunchCfg{ 1, 4, 2, 8, 1 };
    if (c.kind == 2) return c;
    if (c.nt == 2) return { 1, 2, 2, 4, c.wk >= 4 ? 4 : c.wk };
    if (c.nt == 4 && c.wk == 2) return { 1, 4, 2, 4, 2 };
    return { 1, c.nt, 2, 8, 1 };
}

// ---------------------------------------------------------------------------------------------------------------
// Low-rank adapters of many requests: y[n] += s[a] * (x[n] . A[a]^T) . B[a]^T, a = index[n] (none where it is no slot's number).
// Batch rows are taken 16 or 64 at a time, in their order, a lane holding the adapter of a row.  The lowest row that is left names the adapter of the next pass, a comparison of all
// lanes the rows that share it, and the MFMA's other columns go along for the ride.  So no sorting and no lists are needed, an adapter's matrices are read once for
// every tile that holds it, and a tile of one request takes one pass.  Passes of a tile are shared out over the grid's third dimension: they write different rows.
// ---------------------------------------------------------------------------------------------------------------

// the adapter of row (lane) of a tile of ROWS rows, or -1
template <int ROWS> __device__ __forceinline__ int adapter_of(const int *__restrict__ index, uint32_t tile, uint32_t N, uint32_t slots)
{
    const uint32_t lane = threadIdx.x & 63, n = tile * ROWS + lane;
    const int      v = lane < ROWS && n < N ? index[n] : -1;
    return (uint32_t)v < slots ? v : -1;
}
// The passes of this workgroup, numbered from the tile's first: blockIdx.z-th share of gridDim.z, of TOGETHER at least.  A workgroup without any ends before it has asked for anything but
// the index.  (A further pass of a workgroup waits for the adapter's matrix alone, a further workgroup for everything: with tiles of 64 rows and 11 requests of random lengths
// in 2048 rows, 10240 x 8192 at rank 64, one pass a workgroup and sixteen side by side made the call 366 us, four and three 343.)
struct Passes { uint32_t first, end; };
template <uint32_t TOGETHER> __device__ __forceinline__ Passes passes_of(int mine)
{
    uint32_t count = 0;
    for (uint64_t todo = __ballot(mine >= 0); todo; count++) todo &= ~__ballot(mine == __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo)));
    const uint32_t share = (count + gridDim.z - 1) / gridDim.z, per = share > TOGETHER ? share : TOGETHER, first = blockIdx.z * per;
    return { first < count ? first : count, first + per < count ? first + per : count };
}
// f(adapter, rows that have it) for each of them.  The same in all wavefronts of a workgroup.
template <typename F> __device__ __forceinline__ void each_adapter(int mine, Passes p, const F &f)
{
    uint32_t z = 0;
    for (uint64_t todo = __ballot(mine >= 0); z < p.end; z++) {
        const int      a = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
        const uint64_t same = __ballot(mine == a);
        todo &= ~same;
        if (z >= p.first) f(a, same);
    }
}

// shrink: part[range][n][r] = sum over a range of K of x[n, k] * A[a, r, k], fp32.  grid = (tiles, K ranges, passes side by side).  Ranks are taken RT * 16 at a time, in
// adapter_shrink by workgroups of their own (in the grid's second dimension, behind the ranges).
//
// adapter_shrink, for few rows: tiles of sixteen, operands straight from memory, the four wavefronts of a workgroup taking every fourth 64 columns of its range and meeting in LDS.
// Bound by latency: three round trips, to the index, to the operands and to the output (4096 columns, 32 rows of 32 requests, rank 16: 4.6 to 4.9 us).
template <int RT>
__global__ __launch_bounds__(256) void adapter_shrink(float *__restrict__ part, const half_t *__restrict__ x, const half_t *__restrict__ A, const int *__restrict__ index, uint32_t N,
                                                      uint32_t K, uint32_t R, uint32_t slots, uint32_t ranges)
{
    __shared__ __attribute__((aligned(16))) float sums[3][RT][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, q = lane >> 4;
    const int mine = adapter_of<16>(index, blockIdx.x, N, slots), here = __shfl(mine, col);
    const Passes mypasses = passes_of<1>(mine);
    if (mypasses.first == mypasses.end) return;

    const uint32_t range = blockIdx.y % ranges, r0 = blockIdx.y / ranges * (RT * 16), pieces = K / 64, avg = pieces / ranges, extra = pieces % ranges;
    const uint32_t p0 = range * avg + (range < extra ? range : extra), p1 = p0 + avg + (range < extra ? 1u : 0u);
    const uint32_t n = blockIdx.x * 16 + col;
    const half_t  *xrow = x + (size_t)(n < N ? n : N - 1) * K + 8 * q;
    each_adapter(mine, mypasses, [&](int a, uint64_t) {
        const half_t *rows[RT];
        v4f           acc[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const uint32_t row = r0 + r * 16 + col < R ? r0 + r * 16 + col : R - 1; // (rows beyond the rank are not stored)
            rows[r] = A + ((size_t)a * R + row) * K + 8 * q;
            acc[r] = (v4f){ 0.f, 0.f, 0.f, 0.f };
        }
        for (uint32_t p = p0 + wave; p < p1; p += 4) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const v8h b = *reinterpret_cast<const v8h *>(xrow + (size_t)p * 64 + 32 * h);
#pragma unroll
                for (int r = 0; r < RT; r++)
                    acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const v8h *>(rows[r] + (size_t)p * 64 + 32 * h), b, acc[r], 0, 0, 0);
            }
        }
        if (wave > 0)
#pragma unroll
            for (int r = 0; r < RT; r++) *reinterpret_cast<v4f *>(&sums[wave - 1][r][lane * 4]) = acc[r];
        __syncthreads();
        if (wave == 0 && here == a) { // acc[r][i]: rank r0 + 16 r + 4 q + i of batch row n
#pragma unroll
            for (int r = 0; r < RT; r++) {
#pragma unroll
                for (int w = 0; w < 3; w++) acc[r] += *reinterpret_cast<const v4f *>(&sums[w][r][lane * 4]);
                const uint32_t rank = r0 + r * 16 + 4 * q;
                if (rank < R) *reinterpret_cast<v4f *>(part + ((size_t)range * N + n) * R + rank) = acc[r];
            }
        }
        __syncthreads();
    });
}

// Tiles that follow one another, and so have adapters in common more often than not, on one XCD, whose L2 they share: workgroup x runs on XCD x % 8 where there are tiles by the eight.
__device__ __forceinline__ uint32_t neighbouring_tile()
{
    const uint32_t xcd = blockIdx.x & 7, extra = gridDim.x & 7;
    return xcd * (gridDim.x >> 3) + (xcd < extra ? xcd : extra) + (blockIdx.x >> 3);
}

// adapter_shrink_tile, for many: tiles of 64 rows, sixteen a wavefront.  Rows and adapter pass through LDS in chunks of 128 columns, loaded as whole rows of 256 bytes a chunk ahead: in
// operand order sixteen lanes ask for sixteen rows, whose addresses share an L2 channel where K is a power of two (8192 columns, N 2048, rank 64: 41 us, this 22 to 30).  LDS rows
// are 272 bytes apart, the stride at which the operand reads are free of bank conflicts.
template <int RT>
__global__ __launch_bounds__(256) void adapter_shrink_tile(float *__restrict__ part, const half_t *__restrict__ x, const half_t *__restrict__ A, const int *__restrict__ index, uint32_t N,
                                                           uint32_t K, uint32_t R, uint32_t slots)
{
    constexpr int kRow = 272, kX = 4, kA = RT; // bytes of an LDS row; loads of a thread
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][(64 + RT * 16) * kRow];
    const uint32_t tile = neighbouring_tile();
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, q = lane >> 4;
    const int mine = adapter_of<64>(index, tile, N, slots), here = __shfl(mine, wave * 16 + col);
    const Passes mypasses = passes_of<4>(mine);
    if (mypasses.first == mypasses.end) return;

    const uint32_t pieces = (K + 127) / 128, avg = pieces / gridDim.y, extra = pieces % gridDim.y;
    const uint32_t p0 = blockIdx.y * avg + (blockIdx.y < extra ? blockIdx.y : extra), p1 = p0 + avg + (blockIdx.y < extra ? 1u : 0u);
    const uint32_t at = (tid & 15) * 8; // this thread's columns of a chunk, of rows tid / 16, tid / 16 + 16, ...
    const half_t  *xrow[kX];
#pragma unroll
    for (int j = 0; j < kX; j++) {
        const uint32_t n = tile * 64 + (tid >> 4) + 16 * j;
        xrow[j] = x + (size_t)(n < N ? n : N - 1) * K;
    }
    each_adapter(mine, mypasses, [&](int a, uint64_t) {
        for (uint32_t r0 = 0; r0 < R; r0 += RT * 16) {
            const half_t *arow[kA];
            v4f           acc[RT];
            v8h           xr[kX], ar[kA];
#pragma unroll
            for (int j = 0; j < RT; j++) {
                const uint32_t row = r0 + (tid >> 4) + 16 * j;
                arow[j] = A + ((size_t)a * R + (row < R ? row : R - 1)) * K; // (rows beyond the rank are not stored)
                acc[j] = (v4f){ 0.f, 0.f, 0.f, 0.f };
            }
            auto load = [&](uint32_t p) { // (columns beyond K, the second half of a last chunk, are read at the row's start and count as zeros in both)
                const uint32_t k = p * 128 + at, kk = k < K ? k : 0;
#pragma unroll
                for (int j = 0; j < kX; j++) xr[j] = *reinterpret_cast<const v8h *>(xrow[j] + kk);
#pragma unroll
                for (int j = 0; j < kA; j++) ar[j] = *reinterpret_cast<const v8h *>(arow[j] + kk);
                if (k >= K) {
#pragma unroll
                    for (int j = 0; j < kX; j++) xr[j] = (v8h)(half_t)0.f;
#pragma unroll
                    for (int j = 0; j < kA; j++) ar[j] = (v8h)(half_t)0.f;
                }
            };
            auto store = [&](int buf) {
#pragma unroll
                for (int j = 0; j < kX; j++) *reinterpret_cast<v8h *>(lds[buf] + ((tid >> 4) + 16 * j) * kRow + (tid & 15) * 16) = xr[j];
#pragma unroll
                for (int j = 0; j < kA; j++) *reinterpret_cast<v8h *>(lds[buf] + (64 + (tid >> 4) + 16 * j) * kRow + (tid & 15) * 16) = ar[j];
            };
            if (p0 < p1) load(p0), store(0);
            __syncthreads();
            int buf = 0;
            for (uint32_t p = p0; p < p1; p++, buf ^= 1) {
                if (p + 1 < p1) load(p + 1);
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const v8h b = *reinterpret_cast<const v8h *>(lds[buf] + (wave * 16 + col) * kRow + s * 64 + q * 16);
#pragma unroll
                    for (int r = 0; r < RT; r++)
                        acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const v8h *>(lds[buf] + (64 + r * 16 + col) * kRow + s * 64 + q * 16), b, acc[r], 0, 0, 0);
                }
                if (p + 1 < p1) store(buf ^ 1);
                __syncthreads();
            }
            if (here == a) {
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    const uint32_t rank = r0 + r * 16 + 4 * q;
                    if (rank < R) *reinterpret_cast<v4f *>(part + ((size_t)blockIdx.y * N + tile * 64 + wave * 16 + col) * R + rank) = acc[r];
                }
            }
        }
    });
}

// The sums over the K ranges of a row's ranks as the MFMA takes them: fp16, scaled by a power of two that puts the row's largest magnitude below 2^15.  Nothing overflows, what is
// rounded away is 2^-11 of a value at most (2^-39 of the row's largest one for the smallest), and the factor is taken off the fp32 sums.
// v: the ranks that this lane of GROUP holds of the row
template <int GROUP, int COUNT> __device__ __forceinline__ int common_exponent(const float (&v)[COUNT])
{
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < COUNT; j++) top = fmaxf(top, fabsf(v[j]));
#pragma unroll
    for (int d = 1; d < GROUP; d *= 2) top = fmaxf(top, __shfl_xor(top, d, GROUP));
    const int e = top > 0.f && top < __builtin_inff() ? __builtin_amdgcn_frexp_expf(top) - 15 : 0; // top < 2^(e + 15)
    return e < -120 ? -120 : e;
}

// For many rows that is a kernel of its own, a wavefront a row: ranks[n][R rounded up to 32], factor[n] = the power of two times the adapter's scaling
__global__ __launch_bounds__(256) void adapter_ranks(half_t *__restrict__ ranks, float *__restrict__ factor, const float *__restrict__ part, const float *__restrict__ scaling,
                                                     const int *__restrict__ index, uint32_t N, uint32_t R, uint32_t slots, uint32_t ranges)
{
    const uint32_t lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6), Rp = (R + 31) & ~31u;
    if (n >= N) return;
    const int a = index[n];
    if ((uint32_t)a >= slots) return;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        v[j] = 0.f;
        if (lane + 64 * j < R) {
            const float *at = part + (size_t)n * R + lane + 64 * j;
            for (uint32_t s0 = 0; s0 < ranges; s0 += 8) { // eight ranges' sums on their way at once
                float t[8];
#pragma unroll
                for (int u = 0; u < 8; u++) t[u] = at[(size_t)(s0 + u < ranges ? s0 + u : 0) * N * R];
#pragma unroll
                for (int u = 0; u < 8; u++) v[j] += s0 + u < ranges ? t[u] : 0.f;
            }
        }
    }
    const int e = common_exponent<64>(v);
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (lane + 64 * j < Rp) ranks[(size_t)n * Rp + lane + 64 * j] = (half_t)ldexpf(v[j], -e);
    if (lane == 0) factor[n] = ldexpf(1.f, e) * scaling[a];
}

// expand: y[n, m] += factor[n] * sum over r of t[n, r] * B[a, m, r].  grid = (tiles, blocks of 256 outputs, passes side by side); 64 outputs a wavefront.
//
// adapter_expand, for few rows: tiles of sixteen; forms t in LDS from the ranges' sums, which saves a launch and is bound by the latency of it (4096 outputs, 32 rows of 32 requests,
// rank 16: 7.1 to 7.7 us).  The sums are held as two halfs, 22 bits: with few rows of few ranks a rounding of one of them is a rounding of the whole row, and two more MFMAs a step are not to be
// seen in the time.
template <int RT>
__global__ __launch_bounds__(256) void adapter_expand(half_t *__restrict__ y, const float *__restrict__ part, const half_t *__restrict__ B, const float *__restrict__ scaling,
                                                      const int *__restrict__ index, uint32_t M, uint32_t N, uint32_t R, uint32_t slots, uint32_t ranges)
{
    constexpr int kRow = 256 + 8; // halfs
    __shared__ __attribute__((aligned(16))) half_t t16[2][16 * kRow]; // what fp16 holds of a sum, and of the rest
    __shared__ float                               row_factor[16];
    const int      lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, q = lane >> 4;
    const int      mine = adapter_of<16>(index, blockIdx.x, N, slots), here = __shfl(mine, col);
    const uint32_t m0 = blockIdx.y * 256 + wave * 64, Rp = (R + 31) & ~31u, n = blockIdx.x * 16 + col;
    const Passes mypasses = passes_of<1>(mine);
    if (mypasses.first == mypasses.end) return;
    half_t *const  yrow = y + (size_t)(n < N ? n : N - 1) * M + m0 + 4 * q;
    v4h            yv[4];
#pragma unroll
    for (int o = 0; o < 4; o++) yv[o] = *reinterpret_cast<const v4h *>(yrow + o * 16);
    each_adapter(mine, mypasses, [&](int a, uint64_t same) {
        const half_t *rows = B + ((size_t)a * M + m0 + col) * R;
        v8h           w[4]; // of the next step; beyond the rank the row's start, and zeros
        auto          load_w = [&](uint32_t r) {
#pragma unroll
            for (int o = 0; o < 4; o++) {
                w[o] = *reinterpret_cast<const v8h *>(rows + (size_t)o * 16 * R + (r < R ? r : 0));
                if (r >= R) w[o] = (v8h)(half_t)0.f;
            }
        };
        load_w(8 * q);
        { // thread (row i = tid / 16, piece c = tid % 16) sums ranks c, c + 16, ...
            const int      i = threadIdx.x >> 4, c = threadIdx.x & 15;
            const bool     has = same >> i & 1;
            const float   *src = part + (size_t)(has ? blockIdx.x * 16 + i : 0) * R; // (row 0 is there to be read)
            float          v[16];
            __syncthreads(); // (the pass before has read its ranks)
#pragma unroll
            for (int j = 0; j < 16; j++) v[j] = 0.f;
#pragma unroll
            for (int j0 = 0; j0 < 16; j0 += RT)
                if (16 * j0 < (int)R) {
                    for (uint32_t s0 = 0; s0 < ranges; s0 += 8) { // the sums of RT x 16 ranks over eight ranges on their way at once
                        float t[RT][8];
#pragma unroll
                        for (int j = 0; j < RT; j++) {
                            const float *at = src + (c + 16 * (j0 + j) < (int)R ? c + 16 * (j0 + j) : 0);
#pragma unroll
                            for (int u = 0; u < 8; u++) t[j][u] = at[(size_t)(s0 + u < ranges ? s0 + u : 0) * N * R];
                        }
#pragma unroll
                        for (int j = 0; j < RT; j++)
#pragma unroll
                            for (int u = 0; u < 8; u++) v[j0 + j] += s0 + u < ranges ? t[j][u] : 0.f;
                    }
                }
#pragma unroll
            for (int j = 0; j < 16; j++) v[j] = has && c + 16 * j < (int)R ? v[j] : 0.f;
            const int e = common_exponent<16>(v);
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (c + 16 * j < (int)Rp) {
                    const float  sum = ldexpf(v[j], -e);
                    const half_t most = (half_t)sum;
                    const float  rest = sum - (float)most;
                    t16[0][i * kRow + c + 16 * j] = most;
                    t16[1][i * kRow + c + 16 * j] = fabsf(rest) < 64.f ? (half_t)rest : (half_t)0.f; // (no rest to an infinity or a NaN)
                }
            if (c == 0) row_factor[i] = ldexpf(1.f, e) * scaling[a];
            __syncthreads();
        }
        v4f acc[4];
#pragma unroll
        for (int o = 0; o < 4; o++) acc[o] = (v4f){ 0.f, 0.f, 0.f, 0.f };
        for (uint32_t r = 8 * q; r < R + 8 * q; r += 32) { // (the same number of steps in every lane)
            const v8h t = *reinterpret_cast<const v8h *>(t16[0] + col * kRow + r), rest = *reinterpret_cast<const v8h *>(t16[1] + col * kRow + r);
#pragma unroll
            for (int o = 0; o < 4; o++) acc[o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[o], t, acc[o], 0, 0, 0);
#pragma unroll
            for (int o = 0; o < 4; o++) acc[o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[o], rest, acc[o], 0, 0, 0);
            load_w(r + 32);
        }
        if (here == a) {
            const float f = row_factor[col];
#pragma unroll
            for (int o = 0; o < 4; o++) {
                v4h h;
#pragma unroll
                for (int i = 0; i < 4; i++) h[i] = (half_t)((float)yv[o][i] + f * acc[o][i]);
                *reinterpret_cast<v4h *>(yrow + o * 16) = h;
            }
        }
    });
}

// adapter_expand_tile, for many: tiles of 64 rows; t lies in memory (adapter_ranks).  An operand of B feeds four MFMAs.  A row's products are kept from the pass that is its own (a
// selection: another adapter's infinities must not reach it), so y is read and written once for all passes of a workgroup, as whole row pieces of 512 bytes, the products reaching
// them through LDS (sixteen rows a wavefront at once, 32 bytes each, where the row length is a multiple of 4 KB all of one L2 channel: 62 us for 10240 outputs at N 2048, rank 64).
// Bound by the operands' way through L2: 25 us with one adapter a tile (3.4 TB/s of y), 30 to 42 for eleven requests of random lengths, 48 to 58 with four adapters in every tile; with
// y read and written in every pass 25, 49 to 66 and 62 to 72.
constexpr int kExpandRow = 256 * 4 + 16;
// STEPS: of 32 ranks, asked for at once
template <int STEPS>
__global__ __launch_bounds__(256, 3) void adapter_expand_tile(half_t *__restrict__ y, const half_t *__restrict__ ranks, const float *__restrict__ factors, const half_t *__restrict__ B,
                                                              const int *__restrict__ index, uint32_t M, uint32_t N, uint32_t R, uint32_t slots)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[32 * kExpandRow]; // 32 of the rows at a time
    const uint32_t tile = neighbouring_tile();
    const int      tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, q = lane >> 4;
    const int      mine = adapter_of<64>(index, tile, N, slots);
    const uint32_t m0 = blockIdx.y * 256, Rp = (R + 31) & ~31u;
    const Passes   mypasses = passes_of<4>(mine);
    if (mypasses.first == mypasses.end) return;
    // this thread's pieces of y: eight outputs each of rows tid / 32, tid / 32 + 8, ...
    half_t *const  ybase = y + (size_t)tile * 64 * M + m0 + (tid & 31) * 8;
    const uint32_t nlast = N - tile * 64 < 64 ? N - 1 - tile * 64 : 63;
    auto           yp = [&](int j) { const uint32_t n = (tid >> 5) + 8 * j; return ybase + (size_t)(n < nlast ? n : nlast) * M; };
    const half_t *trow[4];
    float         f[4];
    int           here[4];
    v4f           acc[4][4];
#pragma unroll
    for (int s = 0; s < 4; s++) { // (rows without an adapter hold anything, and are not stored)
        const uint32_t n = tile * 64 + (16 * s + col < (int)nlast ? 16 * s + col : nlast);
        trow[s] = ranks + (size_t)n * Rp;
        f[s] = factors[n];
        here[s] = __shfl(mine, 16 * s + col);
#pragma unroll
        for (int o = 0; o < 4; o++) acc[s][o] = (v4f){ 0.f, 0.f, 0.f, 0.f };
    }
    uint64_t done = 0; // rows of this workgroup's passes
    each_adapter(mine, mypasses, [&](int a, uint64_t same) {
        const half_t *rows = B + ((size_t)a * M + m0 + wave * 64 + col) * R;
        done |= same;
        for (uint32_t r0 = 0; r0 < R; r0 += 32 * STEPS) { // (the same number of steps in every lane; beyond the rank zeros count)
            v8h w[STEPS][4], t[STEPS][4];
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                const uint32_t r = r0 + 32 * i + 8 * q;
#pragma unroll
                for (int o = 0; o < 4; o++) w[i][o] = *reinterpret_cast<const v8h *>(rows + (size_t)o * 16 * R + (r < R ? r : 0));
#pragma unroll
                for (int s = 0; s < 4; s++) t[i][s] = *reinterpret_cast<const v8h *>(trow[s] + (r < Rp ? r : 0));
            }
#pragma unroll
            for (int i = 0; i < STEPS; i++)
                if (r0 + 32 * i + 8 * q >= R)
#pragma unroll
                    for (int o = 0; o < 4; o++) w[i][o] = t[i][o] = (v8h)(half_t)0.f;
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int o = 0; o < 4; o++) {
                    v4f sum = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
                    for (int i = 0; i < STEPS; i++) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[i][o], t[i][s], sum, 0, 0, 0);
#pragma unroll
                    for (int k = 0; k < 4; k++) acc[s][o][k] += here[s] == a ? sum[k] : 0.f;
                }
        }
    });
#pragma unroll
    for (int h = 0; h < 2; h++) {
        v8h yv[4];
#pragma unroll
        for (int j = 0; j < 4; j++) yv[j] = *reinterpret_cast<const v8h *>(yp(4 * h + j));
        if (h) __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int o = 0; o < 4; o++) *reinterpret_cast<v4f *>(lds + (16 * s + col) * kExpandRow + (wave * 64 + o * 16 + 4 * q) * 4) = acc[2 * h + s][o] * f[2 * h + s];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = (tid >> 5) + 8 * j;
            if (done >> (32 * h + row) & 1) {
                const v4f lo = *reinterpret_cast<const v4f *>(lds + row * kExpandRow + (tid & 31) * 32), hi = *reinterpret_cast<const v4f *>(lds + row * kExpandRow + (tid & 31) * 32 + 16);
                v8h       out;
#pragma unroll
                for (int i = 0; i < 8; i++) out[i] = (half_t)((float)yv[j][i] + (i < 4 ? lo[i & 3] : hi[i & 3]));
                *reinterpret_cast<v8h *>(yp(4 * h + j)) = out;
            }
        }
    }
}

// How an adapter call is cut.  Tiles of 64 rows where there are many: with every batch row a request of its own, 4096 x 4096, rank 16, tiles of 16 / 64 take 36 / 38 us of 192 rows, 40 / 39 of
// 256, 52 / 43 of 384 (with eight runs of rows 30 / 37 of 256 and 46 / 46 of 768); 10240 x 8192, rank 64, where a row's ranks weigh more, 53 / 57 of 96, 66 / 62 of 128, 94 / 80 of 256.
// K ranges of 256 columns at least that fill the chip (of 512 in small tiles above rank 64, whose sums the second kernel has to add up: 8192 x 8192, rank 128, us of 1 / 64 rows 24.5 / 59
// -> 23.8 / 53; at rank 64 4096 x 4096, 8 rows, 17.9 -> 19.2), and passes of a tile side by side as far as that leaves no crowd of workgroups that find nothing to do (a round of them takes 2 us).
struct AdapterPlan { uint32_t rows, tiles, ranges, shrink_side, expand_side; };
inline AdapterPlan adapter_plan(size_t M, size_t N, size_t K, size_t R, size_t slots)
{
    AdapterPlan p;
    p.rows = N > (R > 32 ? 112u : 256u) ? 64 : 16;
    p.tiles = (uint32_t)((N + p.rows - 1) / p.rows);
    const size_t fill = 512, cols = p.rows == 16 && R > 64 ? 512 : 256, most = K / cols > 0 ? K / cols : 1, want = (fill + p.tiles - 1) / p.tiles;
    p.ranges = (uint32_t)(want < most ? want : most);
    const size_t rows = N < p.rows ? N : p.rows, passes = rows < slots ? rows : slots;
    auto         side = [&](size_t workgroups, size_t room) { return (uint32_t)(workgroups * passes <= room ? passes : workgroups < room ? room / workgroups : 1); };
    p.shrink_side = side((size_t)p.tiles * p.ranges, 2048);
    p.expand_side = side(p.tiles * (M / 256), 4096);
    return p;
}
inline size_t round16(size_t bytes) { return (bytes + 15) & ~(size_t)15; }
// workspace, the same for any number of slots: the ranges' sums, then (tiles of 64 rows) the ranks in fp16 and the rows' factors, then the layer's own
struct AdapterSpace { size_t part, ranks, factors, total; };
inline AdapterSpace adapter_space(const AdapterPlan &p, size_t N, size_t R)
{
    AdapterSpace s;
    s.part = 0;
    s.ranks = round16((size_t)p.ranges * N * R * sizeof(float));
    s.factors = s.ranks + (p.rows == 64 ? round16(N * ((R + 31) / 32 * 32) * 2) : 0);
    s.total = s.factors + (p.rows == 64 ? round16(N * sizeof(float)) : 0);
    return s;
}

int adapter_ranks_of(hipStream_t st, const AdapterPlan &p, float *part, const void *x, const void *A, const int *index, size_t N, size_t K, size_t R, size_t slots)
{
    auto go = [&](auto rt_c) {
        constexpr int RT = decltype(rt_c)::value;
        if (p.rows == 64)
            hipLaunchKernelGGL(adapter_shrink_tile<RT>, dim3(p.tiles, p.ranges, p.shrink_side), dim3(256), 0, st, part, static_cast<const half_t *>(x), static_cast<const half_t *>(A), index,
                               (uint32_t)N, (uint32_t)K, (uint32_t)R, (uint32_t)slots);
        else
            hipLaunchKernelGGL(adapter_shrink<RT>, dim3(p.tiles, p.ranges * (uint32_t)((R + RT * 16 - 1) / (RT * 16)), p.shrink_side), dim3(256), 0, st, part, static_cast<const half_t *>(x),
                               static_cast<const half_t *>(A), index, (uint32_t)N, (uint32_t)K, (uint32_t)R, (uint32_t)slots, p.ranges);
        return (int)hipGetLastError();
    };
    return R <= 16 ? go(std::integral_constant<int, 1>{}) : R <= 32 ? go(std::integral_constant<int, 2>{}) : go(std::integral_constant<int, 4>{});
}
int adapter_expand_of(hipStream_t st, const AdapterPlan &p, void *y, const float *part, const half_t *ranks, const float *factors, const void *B, const float *scaling, const int *index, size_t M,
                      size_t N, size_t R, size_t slots)
{
    const dim3 grid(p.tiles, (uint32_t)(M / 256), p.expand_side);
    if (p.rows == 64) {
        hipLaunchKernelGGL(R <= 32 ? adapter_expand_tile<1> : adapter_expand_tile<2>, grid, dim3(256), 0, st, static_cast<half_t *>(y), ranks, factors, static_cast<const half_t *>(B), index, (uint32_t)M, (uint32_t)N,
                           (uint32_t)R, (uint32_t)slots);
    } else {
        hipLaunchKernelGGL(R <= 16 ? adapter_expand<1> : R <= 32 ? adapter_expand<2> : adapter_expand<4>, grid, dim3(256), 0, st, static_cast<half_t *>(y), part, static_cast<const half_t *>(B), scaling, index, (uint32_t)M, (uint32_t)N, (uint32_t)R,
                           (uint32_t)slots, p.ranges);
    }
    return (int)hipGetLastError();
}

// ---------------------------------------------------------------------------------------------------------------
// Which kernel takes an input gradient, named by the batch rows of its workgroup: grad_stream (16, 32) up to 32 rows, else the tile of grad_tile (128, 192, 256) that is the
// fastest by this model of its time, us: rounds of one workgroup to a CU, each of which takes so long for 32 weight rows, and with a split the partial sums' way to memory and back.
// Fitted to 7 matrices (1024x8192 to 28672x8192) x N 48 to 4096 x splits 1 to 32, off by 9 % rms; its choice of tile and split takes 1.01 times the fastest measured (at worst 1.14).
// ---------------------------------------------------------------------------------------------------------------
constexpr size_t kGradWorkspace = (size_t)256 << 20; // what a split of the heuristic's may take

double grad_time(size_t M, size_t N, size_t K, int splits, int cus, int *rows)
{
    static const struct { int rows; double per32; } tiles[] = { { 128, 0.503 }, { 192, 0.690 }, { 256, 0.906 } };
    double best = 0;
    for (const auto &t : tiles) {
        const size_t wgs = (K + 255) / 256 * ((N + t.rows - 1) / t.rows) * (size_t)splits, rounds = (wgs + cus - 1) / cus, steps = (M / 32 + splits - 1) / splits;
        const double us = 6.1 + t.per32 * (double)rounds * (double)steps + (splits > 1 ? 2.75 + (double)splits * N * K * 8 / 6.08e6 : 0.0);
        if (best == 0 || us < best) {
            best = us;
            if (rows) *rows = t.rows;
        }
    }
    return best;
}
int grad_rows(size_t M, size_t N, size_t K, int splits)
{
    if (N <= 32) return N <= 16 ? 16 : 32;
    int rows = 128;
    grad_time(M, N, K, splits, 256, &rows);
    return rows;
}

} // namespace

// ------------------------------------------------------------------------------------------------ C ABI
extern "C" {

size_t fp6mi_grad_workspace_bytes(size_t N, size_t K, int splits) { return splits > 1 ? (size_t)splits * N * K * sizeof(float) : 0; }

int fp6mi_heuristic_grad_splits(int E, int Mb, size_t M, size_t N, size_t K, int num_cus)
{
    (void)E, (void)Mb;
    if (M == 0 || N == 0 || K == 0 || num_cus <= 0) return 1;
    if (N <= 32) { // a workgroup to a CU and never more (43 blocks of features, us at N 8: four splits 14.5, five 13.7, six 19.4), whose wavefronts have 32 rows at least
        const size_t units = (K + 255) / 256, s = (size_t)num_cus / units, most = M / 256;
        return (int)(s < 1 ? 1 : s < most ? s : most > 0 ? most : 1);
    }
    int    best = 1;
    double t = grad_time(M, N, K, 1, num_cus, nullptr);
    for (int s = 2; s <= 32 && (size_t)s * 128 <= M && fp6mi_grad_workspace_bytes(N, K, s) <= kGradWorkspace; s++)
        if (const double ts = grad_time(M, N, K, s, num_cus, nullptr); ts < t) best = s, t = ts;
    return best;
}

int fp6mi_query_grad_launch(int E, int Mb, size_t M, size_t N, size_t K, int splits)
{
    if (!fp6mi::supported(E, Mb)) return FP6MI_ERR_FORMAT;
    if (M == 0 || M % 256 || M > (size_t)1 << 20 || K == 0 || K % 64 || N == 0) return FP6MI_ERR_SHAPE;
    return splits < 1 ? FP6MI_ERR_SPLITK : grad_rows(M, N, K, splits);
}

static int check_grad(int E, int Mb, const void *W, const void *sc, const void *gexp, const void *dY, const void *dX, size_t M, size_t N, size_t K, const float *ws, int splits)
{
    const int rc = fp6mi::check_linear(E, Mb, W, sc, gexp, nullptr, dY, dX, M, N, K, ws, splits);
    if (rc != FP6MI_OK) return rc;
    return M > (size_t)1 << 20 || K > (size_t)1 << 28 ? FP6MI_ERR_SHAPE : FP6MI_OK; // (32-bit offsets over the rows of a tile, over a row of native blocks)
}

static int run_grad(int E, int Mb, void *stream, const void *W, const void *sc, const void *gexp, const void *dY, bool premultiplied, void *dX, size_t M, size_t N, size_t K, float *ws, int splits)
{
    const int rc = fp6mi::block_ops_for(E, Mb)->grad(grad_rows(M, N, K, splits), stream, W, sc, gexp, dY, premultiplied, dX, ws, M, N, K, splits);
    return rc != 0 || splits == 1 ? rc : fp6mi::reduce_partials(stream, dX, ws, K, N, splits);
}

int fp6mi_linear_grad_native(int E, int Mb, void *stream, const void *W, const void *sc, const void *group_exps, const void *dY, void *dX, size_t M, size_t N, size_t K, float *ws, int splits)
{
    const int rc = check_grad(E, Mb, W, sc, group_exps, dY, dX, M, N, K, ws, splits);
    return rc != FP6MI_OK ? rc : run_grad(E, Mb, stream, W, sc, group_exps, dY, false, dX, M, N, K, ws, splits);
}

size_t fp6mi_gated_workspace_bytes(size_t M, size_t N, int splitK) { return fp6mi_workspace_bytes(M, N, splitK); }

int fp6mi_query_gated_launch(int E, int Mb, size_t M, size_t N, size_t K, int grouped, int *shape)
{
    if (!fp6mi::supported(E, Mb)) return FP6MI_ERR_FORMAT;
    if (M == 0 || M % 256 || K == 0 || K % 64 || N == 0) return FP6MI_ERR_SHAPE;
    if (!shape) return FP6MI_ERR_NULL;
    const fp6mi::LaunchCfg c = gated_shape(E, Mb, M, N, K, grouped != 0);
    shape[0] = c.kind, shape[1] = c.nt, shape[2] = c.rt, shape[3] = c.wr, shape[4] = c.wk;
    return FP6MI_OK;
}

int fp6mi_gated_native(int E, int Mb, void *stream, const void *W, const void *sc, const void *group_exps, const void *bias, const void *B, void *C, float *preact, size_t M, size_t N, size_t K,
                       int activation, float *ws, int splitK)
{
    const int rc = fp6mi::check_linear(E, Mb, W, sc, group_exps, bias, B, C, M, N, K, ws, splitK);
    if (rc != FP6MI_OK) return rc;
    if (!known_activation(activation)) return FP6MI_ERR_ACTIVATION;
    if (preact && !aligned16(preact)) return FP6MI_ERR_ALIGN;
    if (N * (M / 2) > kMostOutputs) return FP6MI_ERR_SHAPE;
    if (splitK == 1) return fp6mi::block_ops_for(E, Mb)->gated(gated_shape(E, Mb, M, N, K, group_exps != nullptr), stream, W, sc, group_exps, bias, B, C, preact, M, N, K, activation);
    const size_t count = N * (M / 2);
    if (const int e = fp6mi::run_linear(E, Mb, stream, W, sc, group_exps, nullptr, B, C, M, N, K, ws, splitK, true)) return e;
    return by_activation(activation, [&](auto act) {
        hipLaunchKernelGGL(gated_reduce<decltype(act)::value>, dim3((uint32_t)((count / 4 + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<half_t *>(C), preact, ws,
                           static_cast<const half_t *>(bias), count, (uint32_t)(M / 2), splitK);
        return (int)hipGetLastError();
    });
}

size_t fp6mi_gated_backward_workspace_bytes(size_t M, size_t N, size_t K, int splits) { return round16(N * M * 2) + fp6mi_grad_workspace_bytes(N, K, splits); }

int fp6mi_gated_backward_native(int E, int Mb, void *stream, const void *W, const void *sc, const void *group_exps, const void *grad_out, const float *preact, void *grad_preact, void *grad_in,
                                size_t M, size_t N, size_t K, int activation, float *ws, int splits)
{
    const int rc = check_grad(E, Mb, W, sc, group_exps, grad_out, grad_in, M, N, K, ws, splits);
    if (rc != FP6MI_OK) return rc;
    if (!preact) return FP6MI_ERR_NULL;
    if (!ws) return FP6MI_ERR_WORKSPACE;
    if (!known_activation(activation)) return FP6MI_ERR_ACTIVATION;
    if (!aligned16(preact) || !aligned16(grad_preact)) return FP6MI_ERR_ALIGN;
    if (N * (M / 2) > kMostOutputs) return FP6MI_ERR_SHAPE;
    const size_t count = N * (M / 2);
    half_t      *scaled = reinterpret_cast<half_t *>(ws);
    const int    e = by_activation(activation, [&](auto act) {
        hipLaunchKernelGGL(gated_grad<decltype(act)::value>, dim3((uint32_t)((count / 8 + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<half_t *>(grad_preact), scaled,
                           static_cast<const half_t *>(grad_out), preact, static_cast<const half_t *>(sc), count, (uint32_t)(M / 2));
        return (int)hipGetLastError();
    });
    return e != 0 ? e : run_grad(E, Mb, stream, W, sc, group_exps, scaled, true, grad_in, M, N, K, ws + round16(N * M * 2) / sizeof(float), splits);
}

size_t fp6mi_adapter_workspace_bytes(size_t M, size_t N, size_t K, size_t R, int splitK)
{
    return N == 0 ? 0 : adapter_space(adapter_plan(M, N, K, R, 1), N, R).total + fp6mi_workspace_bytes(M, N, splitK);
}

int fp6mi_adapter_native(int E, int Mb, void *stream, const void *W, const void *sc, const void *group_exps, const void *bias, const void *B, void *C, const void *lora_a, const void *lora_b,
                         const float *scaling, const int *index, size_t M, size_t N, size_t K, size_t R, size_t slots, float *ws, int splitK)
{
    const int rc = fp6mi::check_linear(E, Mb, W, sc, group_exps, bias, B, C, M, N, K, ws, splitK);
    if (rc != FP6MI_OK) return rc;
    if (!lora_a || !lora_b || !scaling || !index) return FP6MI_ERR_NULL;
    if (!ws) return FP6MI_ERR_WORKSPACE;
    if (R == 0 || R % 8 || R > 256 || slots == 0 || slots > 0x7fffffffu) return FP6MI_ERR_SHAPE;
    if (M / 256 > 65535) return FP6MI_ERR_SHAPE; // (a grid dimension)
    if (!aligned16(lora_a) || !aligned16(lora_b) || (reinterpret_cast<uintptr_t>(scaling) & 3u) || (reinterpret_cast<uintptr_t>(index) & 3u)) return FP6MI_ERR_ALIGN;
    hipStream_t        st = static_cast<hipStream_t>(stream);
    const AdapterPlan  p = adapter_plan(M, N, K, R, slots);
    const AdapterSpace s = adapter_space(p, N, R);
    uint8_t           *base = reinterpret_cast<uint8_t *>(ws);
    half_t            *ranks = reinterpret_cast<half_t *>(base + s.ranks);
    float             *factors = reinterpret_cast<float *>(base + s.factors);
    if (const int e = adapter_ranks_of(st, p, ws, B, lora_a, index, N, K, R, slots)) return e;
    if (p.rows == 64) {
        hipLaunchKernelGGL(adapter_ranks, dim3((uint32_t)((N + 3) / 4)), dim3(256), 0, st, ranks, factors, ws, scaling, index, (uint32_t)N, (uint32_t)R, (uint32_t)slots, p.ranges);
        if (const hipError_t e = hipGetLastError()) return (int)e;
    }
    if (const int e = fp6mi::run_linear(E, Mb, stream, W, sc, group_exps, bias, B, C, M, N, K, splitK > 1 ? reinterpret_cast<float *>(base + s.total) : nullptr, splitK, false)) return e;
    return adapter_expand_of(st, p, C, ws, ranks, factors, lora_b, scaling, index, M, N, R, slots);
}

} // extern "C"
