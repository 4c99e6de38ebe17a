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
__device__ __forceinline__ size_t pair_index(size_t i, uint32_t F) // of output i = n * F + f: its gate pre-activation; the one of up lies 16 behind
{
    const size_t n = i / F, f = i - n * F;
    return n * 2 * F + (f >> 4) * 32 + (f & 15);
}

// What the kernels of fp6mi_block.hip do on their way out, for a split product: the outputs from its partial sums, which it adds up in split order, with the bias and, where they are wanted, the pre-activations.
template <int ACT>
__global__ __launch_bounds__(256) void gated_reduce(half_t *__restrict__ out, float *__restrict__ preact, const float *__restrict__ ws, const half_t *__restrict__ bias, size_t count,
                                                    uint32_t F, int splits)
{
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= count) return;
    const size_t p = pair_index(i, F), stride = count * 2;
    const uint32_t m = (uint32_t)(p % (2 * (size_t)F));
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
// the product with the weights takes (scaled; one rounding for both instead of one behind the other)
template <int ACT>
__global__ __launch_bounds__(256) void gated_grad(half_t *__restrict__ dpre, half_t *__restrict__ scaled, const half_t *__restrict__ dout, const float *__restrict__ preact,
                                                  const half_t *__restrict__ scales, size_t count, uint32_t F)
{
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= count) return;
    const size_t   p = pair_index(i, F);
    const uint32_t m = (uint32_t)(p % (2 * (size_t)F));
    const v4f      g = *reinterpret_cast<const v4f *>(preact + p), u = *reinterpret_cast<const v4f *>(preact + p + 16);
    const v4h      d = *reinterpret_cast<const v4h *>(dout + i);
    v4h            dg, du, sg, su;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float       slope;
        const float a = activation_slope<ACT>(g[j], slope), vg = (float)d[j] * u[j] * slope, vu = (float)d[j] * a;
        dg[j] = (half_t)vg, du[j] = (half_t)vu;
        sg[j] = (half_t)(vg * (float)scale_mantissa(scales[m + j])), su[j] = (half_t)(vu * (float)scale_mantissa(scales[m + 16 + j]));
    }
    if (dpre) {
        *reinterpret_cast<v4h *>(dpre + p) = dg;
        *reinterpret_cast<v4h *>(dpre + p + 16) = du;
    }
    *reinterpret_cast<v4h *>(scaled + p) = sg;
    *reinterpret_cast<v4h *>(scaled + p + 16) = su;
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
    if (c.kind == 2 && c.wr == 2) return { 2, 8, 4, 4, 1 };                                          // gemm_prefill
    if (c.kind == 2) return c;
    if (c.nt == 8) return K <= (size_t)1 << 20 ? fp6mi::LaunchCfg{ 2, 8, 4, 4, 1 } : fp6mi::LaunchCfg{ 1, 4, 2, 8, 1 };
    if (c.nt == 2) return { 1, 2, 2, 4, c.wk >= 4 ? 4 : c.wk };
    if (c.nt == 4 && c.wk == 2) return { 1, 4, 2, 4, 2 };
    return { 1, c.nt, 2, 8, 1 };
}

// ---------------------------------------------------------------------------------------------------------------
// Low-rank adapters of many requests: y[n] += s[a] * (x[n] . A[a]^T) . B[a]^T, a = index[n] (none where it is no slot's number).
// Batch rows are taken sixteen at a time, in their order; the distinct adapters among the sixteen are found by comparing their numbers, and each gets its own pass
// with the MFMA's other fifteen columns along for the ride.  So no sorting and no lists are needed, an adapter's matrices are read once for each sixteen rows that hold it,
// and sixteen rows of one request take one pass.
// ---------------------------------------------------------------------------------------------------------------

// The distinct adapters of batch rows 16 * tile ..: `mine` is the adapter of row (lane & 15) or -1, and the result has bit i set where row i is the first with its adapter.
__device__ __forceinline__ uint32_t distinct_adapters(const int *__restrict__ index, uint32_t tile, uint32_t N, uint32_t slots, int &mine)
{
    const int      i = threadIdx.x & 15;
    const uint32_t n = tile * 16 + i;
    const int      v = n < N ? index[n] : -1;
    mine = (uint32_t)v < slots ? v : -1;
    bool first = mine >= 0;
#pragma unroll
    for (int j = 0; j < 15; j++) {
        const int other = __shfl(mine, j, 16); // (every lane takes part)
        first = first & !((j < i) & (other == mine));
    }
    return (uint32_t)__ballot(first) & 0xffffu;
}

// shrink: part[s][n][r] = sum over K range s of x[n, k] * A[a, r, k], fp32.  grid = (row tiles, K ranges, passes side by side); the four wavefronts of a workgroup take every fourth
// 64 columns of its range and add up through LDS.
template <int RT>
__global__ __launch_bounds__(256) void adapter_shrink(float *__restrict__ part, const half_t *__restrict__ x, const half_t *__restrict__ A, const int *__restrict__ index, uint32_t N,
                                                      uint32_t K, uint32_t R, uint32_t slots)
{
    __shared__ __attribute__((aligned(16))) float sums[3][RT][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, q = lane >> 4;
    int       mine;
    uint32_t  firsts = distinct_adapters(index, blockIdx.x, N, slots, mine);
    for (uint32_t z = blockIdx.z; z > 0 && firsts; z--) firsts &= firsts - 1;

    const uint32_t pieces = K / 64, avg = pieces / gridDim.y, extra = pieces % gridDim.y;
    const uint32_t p0 = blockIdx.y * avg + (blockIdx.y < extra ? blockIdx.y : extra), p1 = p0 + avg + (blockIdx.y < extra ? 1u : 0u);
    const uint32_t n = blockIdx.x * 16 + col;
    const half_t  *xrow = x + (size_t)(n < N ? n : N - 1) * K + 8 * q;
    while (firsts) {
        const int     a = __builtin_amdgcn_readlane(mine, __builtin_ctz(firsts));
        const half_t *rows = A + (size_t)a * R * K + 8 * q;
        v4f           acc[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) acc[r] = (v4f){ 0.f, 0.f, 0.f, 0.f };
        for (uint32_t p = p0 + wave; p < p1; p += 4) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const v8h b = *reinterpret_cast<const v8h *>(xrow + p * 64 + 32 * h);
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    const uint32_t row = r * 16 + col < R ? r * 16 + col : R - 1; // (rows beyond the rank are not stored)
                    const v8h      w = *reinterpret_cast<const v8h *>(rows + (size_t)row * K + p * 64 + 32 * h);
                    acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, b, acc[r], 0, 0, 0);
                }
            }
        }
        if (wave > 0)
#pragma unroll
            for (int r = 0; r < RT; r++) *reinterpret_cast<v4f *>(&sums[wave - 1][r][lane * 4]) = acc[r];
        __syncthreads();
        if (wave == 0) { // acc[r][i]: rank 16 r + 4 q + i of batch row n
#pragma unroll
            for (int r = 0; r < RT; r++) {
#pragma unroll
                for (int w = 0; w < 3; w++) acc[r] += *reinterpret_cast<const v4f *>(&sums[w][r][lane * 4]);
                if (mine == a && r * 16 + 4 * q < R) *reinterpret_cast<v4f *>(part + ((size_t)blockIdx.y * N + n) * R + r * 16 + 4 * q) = acc[r];
            }
        }
        __syncthreads();
        for (uint32_t z = gridDim.z; z > 0 && firsts; z--) firsts &= firsts - 1;
    }
}

// expand: y[n, m] += s[a] * sum over r of t[n, r] * B[a, m, r], t = the sum of part over the K ranges.  grid = (row tiles, blocks of 256 outputs).
// t is held in fp16 for the MFMA, each row scaled by a power of two that puts its largest magnitude below 2^15: nothing overflows, what is rounded away is 2^-11 of a value at
// most (2^-39 of the row's largest one for the smallest), and the factor is taken off the fp32 sums.
__global__ __launch_bounds__(256) void adapter_expand(half_t *__restrict__ y, const float *__restrict__ part, const half_t *__restrict__ B, const float *__restrict__ scaling,
                                                      const int *__restrict__ index, uint32_t M, uint32_t N, uint32_t R, uint32_t slots, uint32_t ranges)
{
    constexpr int kRow = 256 + 8; // halfs
    __shared__ __attribute__((aligned(16))) half_t t16[16 * kRow];
    __shared__ float                               factor[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, q = lane >> 4;
    int       mine;
    uint32_t  firsts = distinct_adapters(index, blockIdx.x, N, slots, mine);
    if (!firsts) return;
    // thread (row i = tid / 16, piece c = tid % 16) sums ranks c, c + 16, ...
    {
        const int      i = threadIdx.x >> 4, c = threadIdx.x & 15;
        const uint32_t n = blockIdx.x * 16 + i;
        const bool     has = __shfl(mine, i & 15, 16) >= 0; // (lane i of any sixteen holds row i's)
        const uint32_t Rp = (R + 31) & ~31u;
        float          v[16], top = 0.f;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            v[j] = 0.f;
            const uint32_t r = c + 16 * j;
            if (has && r < R)
                for (uint32_t s = 0; s < ranges; s++) v[j] += part[((size_t)s * N + n) * R + r];
            top = fmaxf(top, fabsf(v[j]));
        }
#pragma unroll
        for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor(top, d, 16));
        int e = top > 0.f && top < __builtin_inff() ? __builtin_amdgcn_frexp_expf(top) - 15 : 0; // top < 2^(e + 15)
        e = e < -120 ? -120 : e;
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (c + 16 * j < (int)Rp) t16[i * kRow + c + 16 * j] = (half_t)ldexpf(v[j], -e);
        if (c == 0) factor[i] = ldexpf(1.f, e);
    }
    __syncthreads();
    const uint32_t n = blockIdx.x * 16 + col;
    const float    f = mine >= 0 ? factor[col] * scaling[mine] : 0.f;
    const uint32_t m0 = blockIdx.y * 256 + wave * 64;
    v4f            out[4];
#pragma unroll
    for (int o = 0; o < 4; o++) out[o] = (v4f){ 0.f, 0.f, 0.f, 0.f };
    while (firsts) {
        const int     a = __builtin_amdgcn_readlane(mine, __builtin_ctz(firsts));
        const half_t *rows = B + ((size_t)a * M + m0 + col) * R;
        v4f           acc[4];
#pragma unroll
        for (int o = 0; o < 4; o++) acc[o] = (v4f){ 0.f, 0.f, 0.f, 0.f };
        for (uint32_t r = 8 * q; r < R + 8 * q; r += 32) { // (the same number of steps in every lane; beyond the rank zeros meet zeros)
            const v8h t = *reinterpret_cast<const v8h *>(t16 + col * kRow + r);
#pragma unroll
            for (int o = 0; o < 4; o++) {
                const v8h w = r < R ? *reinterpret_cast<const v8h *>(rows + (size_t)o * 16 * R + r) : (v8h)(half_t)0.f;
                acc[o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, t, acc[o], 0, 0, 0);
            }
        }
#pragma unroll
        for (int o = 0; o < 4; o++) out[o] = mine == a ? acc[o] : out[o]; // (not a sum: another adapter's infinities stay out)
        firsts &= firsts - 1;
    }
    if (mine >= 0) {
#pragma unroll
        for (int o = 0; o < 4; o++) {
            half_t   *p = y + (size_t)n * M + m0 + o * 16 + 4 * q;
            const v4h v = *reinterpret_cast<const v4h *>(p);
            v4h       w;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = (half_t)((float)v[i] + f * out[o][i]);
            *reinterpret_cast<v4h *>(p) = w;
        }
    }
}

// K ranges of the shrink: as many workgroups as fill the chip twice, each with 256 columns at least
inline uint32_t shrink_ranges(size_t N, size_t K)
{
    const size_t tiles = (N + 15) / 16, most = K / 256 > 0 ? K / 256 : 1;
    const size_t want = tiles >= 512 ? 1 : (512 + tiles - 1) / tiles;
    return (uint32_t)(want < most ? want : most);
}
inline size_t round16(size_t bytes) { return (bytes + 15) & ~(size_t)15; }

int shrink(hipStream_t st, float *part, const void *x, const void *A, const int *index, size_t N, size_t K, size_t R, size_t slots, uint32_t ranges)
{
    const uint32_t tiles = (uint32_t)((N + 15) / 16), side = tiles >= 64 ? 1 : (uint32_t)(N < 16 ? N : 16);
    const dim3     grid(tiles, ranges, side < slots ? side : (uint32_t)slots);
    auto           go = [&](auto rt_c) {
        hipLaunchKernelGGL((adapter_shrink<decltype(rt_c)::value>), grid, dim3(256), 0, st, part, static_cast<const half_t *>(x), static_cast<const half_t *>(A), index, (uint32_t)N, (uint32_t)K,
                           (uint32_t)R, (uint32_t)slots);
        return (int)hipGetLastError();
    };
    if (R <= 16) return go(std::integral_constant<int, 1>{});
    if (R <= 32) return go(std::integral_constant<int, 2>{});
    if (R <= 64) return go(std::integral_constant<int, 4>{});
    if (R <= 128) return go(std::integral_constant<int, 8>{});
    return go(std::integral_constant<int, 16>{});
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
    if (N <= 32) { // a workgroup to a CU, of which every wavefront has 32 rows at least
        const size_t units = (K + 255) / 256, s = ((size_t)num_cus + units / 2) / units, most = M / 256;
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
    return M > (size_t)1 << 20 ? FP6MI_ERR_SHAPE : FP6MI_OK;
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
        hipLaunchKernelGGL(gated_grad<decltype(act)::value>, dim3((uint32_t)((count / 4 + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<half_t *>(grad_preact), scaled,
                           static_cast<const half_t *>(grad_out), preact, static_cast<const half_t *>(sc), count, (uint32_t)(M / 2));
        return (int)hipGetLastError();
    });
    return e != 0 ? e : run_grad(E, Mb, stream, W, sc, group_exps, scaled, true, grad_in, M, N, K, ws + round16(N * M * 2) / sizeof(float), splits);
}

size_t fp6mi_adapter_workspace_bytes(size_t M, size_t N, size_t K, size_t R, int splitK)
{
    return round16(shrink_ranges(N, K) * N * R * sizeof(float)) + fp6mi_workspace_bytes(M, N, splitK);
}

int fp6mi_adapter_native(int E, int Mb, void *stream, const void *W, const void *sc, const void *group_exps, const void *bias, const void *B, void *C, const void *lora_a, const void *lora_b,
                         const float *scaling, const int *index, size_t M, size_t N, size_t K, size_t R, size_t slots, float *ws, int splitK)
{
    const int rc = fp6mi::check_linear(E, Mb, W, sc, group_exps, bias, B, C, M, N, K, ws, splitK);
    if (rc != FP6MI_OK) return rc;
    if (!lora_a || !lora_b || !scaling || !index) return FP6MI_ERR_NULL;
    if (!ws) return FP6MI_ERR_WORKSPACE;
    if (R == 0 || R % 8 || R > 256 || slots == 0 || slots > 0x7fffffffu) return FP6MI_ERR_SHAPE;
    if (!aligned16(lora_a) || !aligned16(lora_b) || (reinterpret_cast<uintptr_t>(scaling) & 3u) || (reinterpret_cast<uintptr_t>(index) & 3u)) return FP6MI_ERR_ALIGN;
    hipStream_t    st = static_cast<hipStream_t>(stream);
    const uint32_t ranges = shrink_ranges(N, K);
    float         *base_ws = ws + round16(ranges * N * R * sizeof(float)) / sizeof(float);
    if (const int e = shrink(st, ws, B, lora_a, index, N, K, R, slots, ranges)) return e;
    if (const int e = fp6mi::run_linear(E, Mb, stream, W, sc, group_exps, bias, B, C, M, N, K, splitK > 1 ? base_ws : nullptr, splitK, false)) return e;
    hipLaunchKernelGGL(adapter_expand, dim3((uint32_t)((N + 15) / 16), (uint32_t)(M / 256)), dim3(256), 0, st, static_cast<half_t *>(C), ws, static_cast<const half_t *>(lora_b), scaling, index,
                       (uint32_t)M, (uint32_t)N, (uint32_t)R, (uint32_t)slots, ranges);
    return (int)hipGetLastError();
}

} // extern "C"
