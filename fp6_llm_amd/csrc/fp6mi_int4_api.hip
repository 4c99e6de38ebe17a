// Layout and C ABI of the products with 4-bit integer weights (fp6mi_int4.hip; include/fp6mi.h).  No counterpart in the reference.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "fp6mi_internal.h"
#include "fp6mi_int4.inc"

namespace {

#include "fp6mi_grid.inc"

inline bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The nibble of a dword that column j (0..7) of its eight is held in: even ones in the lower 16 bits, odd ones in the upper.
inline uint32_t nibble_of(uint32_t j) { return (j & 1) * 4 + j / 2; }

// Dword i of the native layout of one matrix from its codes, two to a byte, the even column in the low half.
inline uint32_t native_dword(const uint8_t *codes, size_t i, uint32_t K, uint32_t KB)
{
    const uint32_t s = i & 3, lane = i >> 2 & 63, k = (uint32_t)((i >> 8) % KB) * 128 + s * 32 + (lane >> 4) * 8;
    const size_t   row = (i >> 8) / KB * 16 + (lane & 15);
    uint32_t       d = 0;
    if (k < K) // (K is a multiple of 32)
        for (uint32_t j = 0; j < 8; j++) d |= (codes[(row * K + k + j) / 2] >> 4 * (j & 1) & 15u) << 4 * nibble_of(j);
    return d;
}

// A zero point as a number of the scales' type, which holds it exactly.
__host__ __device__ inline uint16_t zero_bits(uint32_t z, int bf16)
{
    z &= 15;
    if (z == 0) return 0;
    uint32_t e = 3;
    while (!(z >> e)) e--;
    return bf16 ? (uint16_t)((127 + e) << 7 | (z << (7 - e) & 127)) : (uint16_t)((15 + e) << 10 | (z << (10 - e) & 1023));
}

// The scales (with zero points: {scale, zero point}) of 16 rows, `each` columns (32, 64 or 128) to a native group: j from `first` in strides up to their number, [column block][row][group of the block].
__host__ __device__ inline void native_scales_of(uint16_t *to, const uint16_t *scales, const uint8_t *zeros, int bf16, uint32_t K, uint32_t KB, uint32_t group, uint32_t each, uint32_t first, uint32_t stride)
{
    const uint32_t per = 128 / each, groups = (K + group - 1) / group;
    for (uint32_t j = first; j < KB * 16 * per; j += stride) {
        const uint32_t k = j / (16 * per) * 128 + j % per * each;
        const size_t   at = (size_t)(j / per % 16) * groups + k / group;
        const uint16_t scale = k < K ? scales[at] : 0;
        if (zeros)
            to[2 * (size_t)j] = scale, to[2 * (size_t)j + 1] = k < K ? zero_bits(zeros[at], bf16) : 0;
        else
            to[j] = scale;
    }
}

// A wavefront to a block of 16 rows x 128 columns: lane c + 16 s reads the 16 bytes of row c from column 32 s on, puts the nibbles of each dword in order, and the four lanes of a row trade dwords by way of LDS.
// (28672x8192 with its scales: 39 us, 6 TB/s read and written; with a thread to a dword that reads its bytes one by one 390.)
template <bool ALIGNED> __global__ __launch_bounds__(256) void pack_codes(uint32_t *__restrict__ out, const uint8_t *__restrict__ codes, uint32_t blocks, uint32_t K, uint32_t KB)
{
    __shared__ uint32_t stage[4][256];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, s = lane >> 4, b = workgroup() * 4 + wave, k = b % KB * 128 + s * 32;
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    v4u d = { 0, 0, 0, 0 };
    if (b < blocks && k < K) { // (K is a multiple of 32)
        const uint8_t *row = codes + (((size_t)(b / KB) * 16 + c) * K + k) / 2;
        if constexpr (ALIGNED)
            d = *reinterpret_cast<const v4u *>(row);
        else
            for (int i = 0; i < 16; i++) d[i / 4] |= (uint32_t)row[i] << i % 4 * 8;
    }
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
        uint32_t even = d[q] & 0x0f0f0f0fu, odd = d[q] >> 4 & 0x0f0f0f0fu;
        even = (even | even >> 4) & 0x00ff00ffu, odd = (odd | odd >> 4) & 0x00ff00ffu;
        stage[wave][(c + 16 * q) * 4 + s] = ((even | even >> 8) & 0xffffu) | (odd | odd >> 8) << 16;
    }
    __syncthreads();
    if (b < blocks) reinterpret_cast<v4u *>(out)[(size_t)b * 64 + lane] = *reinterpret_cast<const v4u *>(&stage[wave][lane * 4]);
}

// A workgroup to 16 rows.
__global__ __launch_bounds__(256) void pack_scales(uint16_t *__restrict__ out, const uint16_t *__restrict__ scales, const uint8_t *__restrict__ zeros, uint32_t tiles, int bf16, uint32_t K, uint32_t KB, uint32_t group, uint32_t each)
{
    if (workgroup() >= tiles) return;
    const size_t rows = (size_t)workgroup() * 16, groups = (K + group - 1) / group;
    native_scales_of(out + rows * KB * (128 / each) * (zeros ? 2 : 1), scales + rows * groups, zeros ? zeros + rows * groups : nullptr, bf16, K, KB, group, each, threadIdx.x, 256);
}

inline uint32_t native_group(size_t group) { return group % 128 == 0 ? 128 : group % 64 == 0 ? 64 : 32; }

int check_shape(size_t experts, size_t M, size_t K)
{
    if (M == 0 || M % 16 || K == 0 || K % 32 || K > (size_t)1 << 24 || M > (size_t)1 << 24 || experts == 0 || experts > 1024) return FP6MI_ERR_SHAPE;
    return experts * (M / 16) * ((K + 127) / 128) > (size_t)1 << 31 ? FP6MI_ERR_SHAPE : FP6MI_OK;
}

int check_pack(const void *native, const void *native_scales, const void *codes, const void *scales, int dtype, size_t experts, size_t M, size_t K, size_t group)
{
    if (dtype != 0 && dtype != 1) return FP6MI_ERR_TYPE;
    if (const int e = check_shape(experts, M, K)) return e;
    if (group == 0 || group % 32 || group > (size_t)1 << 24) return FP6MI_ERR_SHAPE;
    if (!native || !native_scales || !codes || !scales) return FP6MI_ERR_NULL;
    return aligned(native, 16) && aligned(native_scales, 16) && aligned(scales, 2) ? FP6MI_OK : FP6MI_ERR_ALIGN;
}

// Which kernel takes a product (an index of kInt4Kernels): the fastest by this model of its time, us.  A workgroup's column blocks one after another take `step` each while every CU has one at the most,
// `share` times the workgroups of a CU beyond; and no kernel reads the weights faster than memory.  Rows of experts are taken to be spread evenly, with half a tile to spare for each expert.
// Fitted to 4372 times of 407 products in graphs, weights from HBM (512x2048 to 28672x8192 at 1 to 1000 rows, 8 to 128 experts at 1 to 700 tokens, fp16 and bf16): a kernel's own time is off by 17 to 31 % rms, the
// choice takes 1.01 times the fastest measured in the mean, at worst 1.29; for 100 other products 1.02 and 1.25.
struct Times { double base, step, share, rows; }; // rows: how much longer a step takes with 16 rows than with none
constexpr Times kTimes[] = { { 1.25, 1.19, 1.28, 1.12 }, { 1.78, 0.87, 1.13, 0 }, { 2.65, 1.17, 1.35, 0.10 }, { 1.61, 1.64, 1.93, 0 }, { 2.01, 1.08, 0.70, 0 }, { 3.25, 0.99, 0.97, 0 },
                             { 2.78, 1.05, 1.20, 0 },    { 3.07, 1.35, 1.57, 0 }, { 2.18, 1.75, 2.14, 0 },    { 6.59, 0.99, 0.78, 0 }, { 2.58, 1.26, 1.44, 0 }, { 2.18, 1.03, 1.10, 0 } };

constexpr int    kKernels = sizeof(kTimes) / sizeof(kTimes[0]);
static_assert(kKernels == sizeof(fp6mi::kInt4Kernels) / sizeof(fp6mi::kInt4Kernels[0]), "");
constexpr size_t kMostTileColumns = (size_t)1 << 20; // (offsets in a tile have 32 bits)

double time_of(int kernel, int dtype, size_t experts, bool grouped, size_t M, size_t N, size_t K)
{
    const fp6mi::Int4Kernel &k = fp6mi::kInt4Kernels[kernel];
    const Times             &t = kTimes[kernel];
    const double used = grouped ? experts * (1 - std::exp(-(double)N / experts)) : 1.0, tiles = grouped ? std::max(used, (double)N / k.cols + 0.5 * used) : (double)((N + k.cols - 1) / k.cols);
    const double load = (double)((M / 16 + k.row_tiles - 1) / k.row_tiles) * tiles / 256, steps = (double)(((K + 127) / 128 + k.k_split - 1) / k.k_split);
    const double more = 1 + t.rows * std::min(16.0, (double)N / used) / 16;
    const double among = load <= 1 ? load : (load + std::ceil(load)) / 2;
    double       us = t.base + steps * more * std::max(t.step, t.share * among);
    if (dtype == 1 && k.tile) us += 3 + (double)N * K * 4 / 4.0e6; // (the rows on their way to fp16)
    return std::max(us, used * M * K * 0.515 / 5.1e6 + 1.5);
}

// Whether a kernel has the problem.
bool lacks(int kernel, int group, size_t K, bool gated)
{
    const fp6mi::Int4Kernel &k = fp6mi::kInt4Kernels[kernel];
    return (k.tile && K > kMostTileColumns) || (gated && !k.pairs) || (k.group128 && group != 128);
}

// Whether a kernel's grid would not hold the tiles of N that there are by those of M.
bool too_many(int kernel, size_t tiles, size_t M)
{
    const fp6mi::Int4Kernel &k = fp6mi::kInt4Kernels[kernel];
    return k.tile ? tiles * ((M / 16 + k.row_tiles - 1) / k.row_tiles) > fp6mi::kInt4MostTiles : tiles > fp6mi::kInt4MostStreams;
}

int choice(int dtype, int group, size_t experts, bool grouped, size_t M, size_t N, size_t K, bool gated)
{
    int       best = -1;
    double    least = 0;
    for (int k = 0; k < kKernels; k++) {
        if (lacks(k, group, K, gated)) continue;
        const size_t tiles = fp6mi::int4_tiles(N, grouped ? experts : 0, fp6mi::kInt4Kernels[k].cols);
        if (too_many(k, tiles, M)) continue;
        const double us = time_of(k, dtype, experts, grouped, M, N, K);
        if (best < 0 || us < least) best = k, least = us;
    }
    return best;
}

// Scratch of a product by kernel `kernel`: of bf16 tiles the rows of X as halfs, behind their exponents.
size_t round16(size_t n) { return (n + 15) / 16 * 16; }
size_t scratch_bytes(int dtype, int kernel, size_t N, size_t K) { return dtype == 1 && kernel >= 0 && fp6mi::kInt4Kernels[kernel].tile ? round16(N * sizeof(int)) + N * K * 2 : 0; }

} // namespace

extern "C" {

size_t fp6mi_int4_weight_bytes(size_t experts, size_t M, size_t K) { return check_shape(experts, M, K) ? 0 : experts * (M / 16) * ((K + 127) / 128) * 1024; }

size_t fp6mi_int4_scale_bytes(size_t experts, size_t M, size_t K, size_t group, int zeros)
{
    if (check_shape(experts, M, K) || group == 0 || group % 32) return 0;
    return experts * M * ((K + 127) / 128) * (128 / native_group(group)) * (zeros ? 4 : 2);
}

int fp6mi_int4_pack(void *native, void *native_scales, const void *codes, const void *scales, const void *zeros, int dtype, size_t experts, size_t M, size_t K, size_t group)
{
    if (const int e = check_pack(native, native_scales, codes, scales, dtype, experts, M, K, group)) return e;
    const uint32_t KB = (uint32_t)((K + 127) / 128);
    const size_t   matrix = M / 16 * KB * 256, tiles = experts * (M / 16), groups = (K + group - 1) / group, of_tile = fp6mi_int4_scale_bytes(1, 16, K, group, zeros != nullptr) / 2;
    for (size_t e = 0; e < experts; e++)
        for (size_t i = 0; i < matrix; i++) static_cast<uint32_t *>(native)[e * matrix + i] = native_dword(static_cast<const uint8_t *>(codes) + e * M * (K / 2), i, (uint32_t)K, KB);
    for (size_t t = 0; t < tiles; t++)
        native_scales_of(static_cast<uint16_t *>(native_scales) + t * of_tile, static_cast<const uint16_t *>(scales) + t * 16 * groups,
                         zeros ? static_cast<const uint8_t *>(zeros) + t * 16 * groups : nullptr, dtype, (uint32_t)K, KB, (uint32_t)group, native_group(group), 0, 1);
    return FP6MI_OK;
}

int fp6mi_int4_pack_gpu(void *stream, void *native, void *native_scales, const void *codes, const void *scales, const void *zeros, int dtype, size_t experts, size_t M, size_t K, size_t group)
{
    if (const int e = check_pack(native, native_scales, codes, scales, dtype, experts, M, K, group)) return e;
    const uint32_t KB = (uint32_t)((K + 127) / 128);
    const size_t   tiles = experts * (M / 16), blocks = tiles * KB; // up to 2^31
    hipStream_t    st = static_cast<hipStream_t>(stream);
    if (aligned(codes, 16))
        hipLaunchKernelGGL(pack_codes<true>, grid_of((blocks + 3) / 4), dim3(256), 0, st, static_cast<uint32_t *>(native), static_cast<const uint8_t *>(codes), (uint32_t)blocks, (uint32_t)K, KB);
    else
        hipLaunchKernelGGL(pack_codes<false>, grid_of((blocks + 3) / 4), dim3(256), 0, st, static_cast<uint32_t *>(native), static_cast<const uint8_t *>(codes), (uint32_t)blocks, (uint32_t)K, KB);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    hipLaunchKernelGGL(pack_scales, grid_of(tiles), dim3(256), 0, st, static_cast<uint16_t *>(native_scales), static_cast<const uint16_t *>(scales), static_cast<const uint8_t *>(zeros), (uint32_t)tiles, dtype,
                       (uint32_t)K, KB, (uint32_t)group, native_group(group));
    return (int)hipGetLastError();
}

size_t fp6mi_int4_workspace_bytes(int dtype, int group, size_t experts, int grouped, size_t M, size_t N, size_t K, int gated, int kernel)
{
    if ((dtype != 0 && dtype != 1) || (group != 32 && group != 64 && group != 128) || check_shape(experts, M, K) || N == 0 || N > (size_t)1 << 30 || kernel >= kKernels) return 0;
    return scratch_bytes(dtype, kernel >= 0 ? kernel : choice(dtype, group, experts, grouped != 0, M, N, K, gated != 0), N, K);
}

int fp6mi_int4_query_kernel(int dtype, int group, size_t experts, int grouped, size_t M, size_t N, size_t K, int gated, int *shape)
{
    if (dtype != 0 && dtype != 1) return FP6MI_ERR_TYPE;
    if ((group != 32 && group != 64 && group != 128) || check_shape(experts, M, K) || N == 0 || N > (size_t)1 << 30) return FP6MI_ERR_SHAPE;
    const int k = choice(dtype, group, experts, grouped != 0, M, N, K, gated != 0);
    if (k < 0) return FP6MI_ERR_SHAPE;
    const fp6mi::Int4Kernel &c = fp6mi::kInt4Kernels[k];
    if (shape) shape[0] = c.tile, shape[1] = c.cols, shape[2] = c.row_tiles, shape[3] = c.k_split;
    return k;
}

int fp6mi_int4_linear_cfg(void *stream, int dtype, const void *W_native, const void *scales_native, int group, int zeros, const void *bias, const void *X, void *Y, int out_f32, int activation,
                          const int *offsets, size_t experts, size_t M, size_t N, size_t K, void *workspace, int kernel)
{
    if (dtype != 0 && dtype != 1) return FP6MI_ERR_TYPE;
    if (const int e = check_shape(experts, M, K)) return e;
    if ((group != 32 && group != 64 && group != 128) || N > (size_t)1 << 30 || (!offsets && experts != 1) || kernel >= kKernels) return FP6MI_ERR_SHAPE;
    if (activation > FP6MI_ACT_GELU_TANH) return FP6MI_ERR_ACTIVATION;
    if (activation >= 0 && M % 32) return FP6MI_ERR_SHAPE;
    if (N == 0) return FP6MI_OK;
    if (!W_native || !scales_native || !X || !Y) return FP6MI_ERR_NULL;
    if (!aligned(W_native, 16) || !aligned(scales_native, 16) || !aligned(X, 16) || !aligned(Y, 16) || !aligned(bias, 2) || !aligned(offsets, 4) || !aligned(workspace, 16)) return FP6MI_ERR_ALIGN;
    if (kernel < 0) kernel = choice(dtype, group, experts, offsets != nullptr, M, N, K, activation >= 0);
    if (kernel < 0 || lacks(kernel, group, K, activation >= 0) || too_many(kernel, fp6mi::int4_tiles(N, offsets ? experts : 0, fp6mi::kInt4Kernels[kernel].cols), M)) return FP6MI_ERR_SHAPE;
    fp6mi::Int4Args a = { W_native, scales_native, X, bias, Y, offsets, (uint32_t)N, (uint32_t)K, (uint32_t)((K + 127) / 128), (uint32_t)(M / 16), (uint32_t)experts, activation, out_f32, nullptr };
    if (scratch_bytes(dtype, kernel, N, K)) {
        if (!workspace) return FP6MI_ERR_WORKSPACE;
        int  *exponents = static_cast<int *>(workspace);
        void *halfs = static_cast<uint8_t *>(workspace) + round16(N * sizeof(int));
        if (const int e = fp6mi::int4_rows_to_halfs(stream, halfs, exponents, X, N, K)) return e;
        a.X = halfs, a.exponents = exponents;
    }
    if (dtype == 0) return group == 128 ? fp6mi::int4_run_0_1(stream, a, zeros != 0, kernel) : group == 64 ? fp6mi::int4_run_0_2(stream, a, zeros != 0, kernel) : fp6mi::int4_run_0_4(stream, a, zeros != 0, kernel);
    return group == 128 ? fp6mi::int4_run_1_1(stream, a, zeros != 0, kernel) : group == 64 ? fp6mi::int4_run_1_2(stream, a, zeros != 0, kernel) : fp6mi::int4_run_1_4(stream, a, zeros != 0, kernel);
}

int fp6mi_int4_linear(void *stream, int dtype, const void *W_native, const void *scales_native, int group, int zeros, const void *bias, const void *X, void *Y, int out_f32, int activation,
                      const int *offsets, size_t experts, size_t M, size_t N, size_t K, void *workspace)
{
    return fp6mi_int4_linear_cfg(stream, dtype, W_native, scales_native, group, zeros, bias, X, Y, out_f32, activation, offsets, experts, M, N, K, workspace, -1);
}

} // extern "C"
