// Products with 4-bit integer weights and a scale (and zero point) for each group of columns: y[n,m] = sum_k x[n,k] * s[m,g(k)] * (q[m,k] - z[m,g(k)]), for one matrix or, with rows that
// are sorted by expert, for the matrix of each row's expert; optionally act(gate) * up of the pairs of 16 rows.  Compiled once per activation type (FP6MI_TYPE 0: fp16, 1: bf16).
// No counterpart in the reference.
//
// q - z is an integer from -15 to 15, exact in fp16, so the matrix instructions' products are exact and their sums float32; a group's sum is multiplied by its scale in float32.
// (Scaling the weights before the product would round each of them to 16 bits, and 16-bit sums would be no cheaper.)  bf16 has no packed arithmetic that would make q - z of codes: the kernel of
// few rows multiplies 16 + q, which are bits, from sums that start at -(16 + z) times those of X; the one of many rows is given X in fp16 with an exponent for each row (rows_to_halfs).
//
// Layout (fp6mi_int4_pack): blocks of 16 rows x 128 columns of 1024 bytes, [expert][row tile][column block]; lane c + 16 q of a wavefront holds 16 bytes of a block, dword s of which are the
// columns 32 s + 8 q to 32 s + 8 q + 7 of row c: the operand of one v_mfma_f32_16x16x32.  In a dword the nibbles 0..7 are the columns 0, 2, 4, 6, 1, 3, 5, 7, so that a mask leaves two neighbours
// 16 bits apart.  Scales: [expert][row tile][column block][row][group of the block], with zero points {scale, zero point} in pairs, both of the activations' type.
#include <hip/hip_runtime.h>

#include <atomic>
#include <type_traits>

#include "fp6mi_internal.h"
#include "fp6mi_activation.inc"
#include "fp6mi_int4.inc"

namespace {

#if FP6MI_TYPE == 0
typedef _Float16 T;
#else
typedef __bf16 T;
#endif
#include "fp6mi_lds.inc"

typedef _Float16 half_t;
typedef half_t   v2h __attribute__((ext_vector_type(2)));
typedef half_t   v8h __attribute__((ext_vector_type(8)));
typedef T        v8t __attribute__((ext_vector_type(8)));
typedef float    v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

using fp6mi::Int4Args;

__device__ __forceinline__ v4f mfma(v8t x, v8t w, v4f acc)
{
#if FP6MI_TYPE == 0
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, w, acc, 0, 0, 0);
#else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, w, acc, 0, 0, 0);
#endif
}

__device__ __forceinline__ v4f mfma_halfs(v8h x, v8h w, v4f acc) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, w, acc, 0, 0, 0); }

// f(0), ..., f(N - 1) with the index as a compile-time constant
template <int N, int I = 0, typename F> __device__ __forceinline__ void sections(const F &f)
{
    f(std::integral_constant<int, I>{});
    if constexpr (I + 1 < N) sections<N, I + 1>(f);
}

// What the codes are cut out with.  (w & mask) | bits is one instruction where of the two constants one is in a vector register, of which the compiler has to be told.
struct Cutter {
    uint32_t low = 0x000f000fu, high = 0x00f000f0u, bits = 0x64006400u;
    __device__ __forceinline__ Cutter() { asm("" : "+s"(low), "+s"(high), "+v"(bits)); }
};

// What a group's zero point (8 without one) makes of the codes: -(1024 + z), -(64 + z).
struct Zero {
    v2h low, high;
    __device__ __forceinline__ void set(T zero)
    {
        const half_t z = (half_t)(float)zero, l = (half_t)-1024.f - z, h = (half_t)-64.f - z;
        low = (v2h){ l, l }, high = (v2h){ h, h };
    }
};

// Eight codes as q - z in fp16, columns 0..7, or (half) four of them: 1024 + q and 1024 + 16 q are read off the bits 0x6400 | nibble, 9 instructions.
union Codes { uint32_t d[4]; v8h v; };
__device__ __forceinline__ void codes_half(Codes &to, uint32_t w, const Zero &zero, const Cutter &cut, int half)
{
    const v2h sixteenth = { (half_t)0.0625f, (half_t)0.0625f };
    if (half) w >>= 8;
    to.d[2 * half] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, (w & cut.low) | cut.bits) + zero.low);
    to.d[2 * half + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(v2h, (w & cut.high) | cut.bits), sixteenth, zero.high));
}

// The operands of the kernel of few rows.  fp16: q - z.  bf16: 16 + q, the bits 0x4180 | nibble << 3, 8 instructions (q - z by way of float32 takes 23, which bound that kernel); what is too much, 16 + z times
// the sum of a group's X, is where the products start from, a sum that a matrix instruction with ones makes for all row tiles (28672x8192 at 4 rows with groups of 64 and zero points 26.7 -> 24.9 us
// against one with -(16 + z) for each).  That costs float32 sums a factor of some five in rounding: of 8192 columns they are off by 1e-7 to 3e-7 rms (values of mean 0 or 1, one of 3000 among them), where
// a product in float32 is by 4e-7 to 8e-7; 128 + q, the nibble as it stands, takes an instruction less (26.1 us, with these 26.6) and is off by 7e-7 to 3e-6.  Sums that leave float32's range on the way
// are made again at the end, with q - z.
#if FP6MI_TYPE == 0
struct FewCutter : Cutter { };
struct FewZero : Zero { };
__device__ __forceinline__ v8t codes_of(uint32_t w, const FewZero &zero, const FewCutter &cut)
{
    Codes r;
    codes_half(r, w, zero, cut, 0);
    codes_half(r, w, zero, cut, 1);
    return r.v;
}
#else
struct FewCutter {
    uint32_t mask = 0x00780078u, bits = 0x41804180u;
    __device__ __forceinline__ FewCutter() { asm("" : "+s"(mask), "+v"(bits)); }
};
struct FewZero {
    float all; // -(16 + z)
    __device__ __forceinline__ void set(T zero) { all = -16.f - (float)zero; }
};
__device__ __forceinline__ v8t codes_of(uint32_t w, const FewZero &, const FewCutter &cut)
{
    union { uint32_t d[4]; v8t v; } r;
#pragma unroll
    for (int i = 0; i < 4; i++) r.d[i] = ((i ? w >> (4 * i - 3) : w << 3) & cut.mask) | cut.bits;
    return r.v;
}
#endif

// The scales (and zero points) of one row in one block.
template <int GPB, bool Z> struct alignas(2 * GPB * (Z ? 2 : 1)) Scales { T v[GPB * (Z ? 2 : 1)]; };

// Rows [row, row + rows) of X against the weights of an expert; or rows that no expert has (expert < 0), which get zeros.
struct Tile { int expert; uint32_t row, rows; };

// Tile number i of `each` rows: those of one matrix, or of the experts one after another, then of the rows behind them; rows = 0: there are fewer.  The same for all lanes.
__device__ __forceinline__ Tile tile_of(const Int4Args &a, uint32_t i, uint32_t each)
{
    if (!a.offsets) {
        const uint32_t row = i * each;
        return { 0, row, row < a.N ? (a.N - row < each ? a.N - row : each) : 0 };
    }
    const int lane = threadIdx.x & 63;
    uint32_t  first = 0; // tiles of the experts before these 64
    for (uint32_t b = 0; b <= a.E; b += 64) {
        const uint32_t e = b + lane, lo = e <= a.E ? (uint32_t)a.offsets[e] : a.N, hi = e < a.E ? (uint32_t)a.offsets[e + 1] : a.N, n = hi > lo ? (hi - lo + each - 1) / each : 0;
        uint32_t       s = n;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t o = __shfl_up(s, m);
            if (lane >= m) s += o;
        }
        const uint64_t reached = __ballot(first + s > i);
        if (reached) {
            const int      at = __builtin_ctzll(reached);
            const uint32_t row = __builtin_amdgcn_readlane(lo, at) + (i - first - __builtin_amdgcn_readlane(s - n, at)) * each, end = __builtin_amdgcn_readlane(hi, at);
            return { b + at < a.E ? (int)(b + at) : -1, row, row < end && end <= a.N ? (end - row < each ? end - row : each) : 0 };
        }
        first += __builtin_amdgcn_readlane(s, 63);
    }
    return { 0, 0, 0 };
}

__device__ __forceinline__ void store(const Int4Args &a, uint32_t row, uint32_t m, uint32_t ld, float v)
{
    const size_t at = (size_t)row * ld + m;
    if (a.out_f32)
        static_cast<float *>(a.Y)[at] = v;
    else
        static_cast<T *>(a.Y)[at] = (T)v;
}

// Zeros for the rows of a tile that no expert has, in the columns of row tiles [m0, m0 + mt).
__device__ __forceinline__ void store_zeros(const Int4Args &a, const Tile &t, uint32_t m0, uint32_t mt, uint32_t threads)
{
    const uint32_t per = a.act >= 0 ? 8 : 16, ld = a.Mt * per, lo = m0 * per, w = (m0 + mt < a.Mt ? mt : a.Mt - m0) * per;
    for (uint32_t i = threadIdx.x; i < t.rows * w; i += threads) store(a, t.row + i / w, lo + i % w, ld, 0.f);
}

// ---------------------------------------------------------------------------------------------------------------
// Few rows: RT row tiles and 16 rows of X to a workgroup of WK wavefronts, which share K: a wavefront takes every WK-th column block, its weights straight from HBM to registers (the next block's on their
// way meanwhile) and its part of X from L2; the partial sums meet in LDS.  X is read in whole rows, two blocks ahead, and turned into operands through LDS a block ahead: as operands, 64 bytes of each of 16
// rows to a load, 8192x8192 at 16 rows took 11.8 us and 28672x8192 27.8, in whole rows 10.2 and 24.8.  (Only the kernel of one row tile, which is for few blocks, reads operands: to turn them
// takes it 0.4 us, and at one row there is nothing to be won.)
// Bound by the bytes of the weights where there are many (28672x8192: 22.4 us at 1 row, 24.8 at 16, of which the bytes take 23.6 at a copy's rate; 8192x8192: 8.5 and 10.2 of 6.8), by a wavefront's few blocks
// one after another where there are few (4096x4096 at 1 row: 4.3 us with 16 wavefronts to a row tile, 5.2 with 8 to two).  Three and four blocks of weights on their way were no faster, nor were two
// tiles of rows of X to a workgroup.
// ---------------------------------------------------------------------------------------------------------------
template <int GPB, bool Z, int RT> struct Block {
    v4u            w[RT];
    Scales<GPB, Z> s[RT];
};

template <int GPB, bool Z, int RT, int WK> __global__ __launch_bounds__(WK * 64, WK > 4 ? 1 : 2) void int4_stream(const Int4Args a)
{
    static_assert(RT <= 4, "");
    __shared__ v4f shared[WK][RT > 1 ? 4 : 1][64]; // of a wavefront: a block of X on its way into operand order, in the end its sums
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, q = lane >> 4;
    const uint32_t m0 = blockIdx.x * RT;
    const Tile     t = tile_of(a, blockIdx.y, 16);
    if (t.rows == 0) return;
    if (t.expert < 0) return store_zeros(a, t, m0, RT, WK * 64);

    const v4u            *w[RT];
    const Scales<GPB, Z> *s[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) { // (a last workgroup with fewer row tiles takes the last one again)
        const size_t at = ((size_t)t.expert * a.Mt + (m0 + r < a.Mt ? m0 + r : a.Mt - 1)) * a.KB;
        w[r] = static_cast<const v4u *>(a.W) + at * 64 + lane;
        s[r] = static_cast<const Scales<GPB, Z> *>(a.S) + at * 16 + c;
    }
    // X: in whole rows, four of 256 bytes to a load, lane c + 16 q with piece c of row 4 i + q, or (one row tile) as operands, piece 4 i + q of row c.  Rows behind the last one are behind the buffer: they read as zeros and ask for nothing.
    constexpr bool kTurn = RT > 1;
    const auto     xbuf = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(static_cast<const T *>(a.X) + (size_t)t.row * a.K), 0, (int)(t.rows * a.K * 2), 0x00027000);
    uint32_t       xoff[4], beyond[4]; // (beyond: what puts an offset in the last block behind the buffer, which reads as zeros)
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
        const uint32_t row = kTurn ? 4 * i + q : c, piece = kTurn ? c : 4 * i + q;
        xoff[i] = row * a.K * 2 + piece * 16;
        beyond[i] = (a.KB - 1) * 128 + piece * 8 < a.K ? 0 : 0x80000000u;
    }

    typedef Block<GPB, Z, RT> B;
    const FewCutter           cut;
    auto load = [&](B &b, uint32_t kb) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RT; r++) b.w[r] = __builtin_nontemporal_load(w[r] + (size_t)kb * 64);
#pragma unroll
        for (int r = 0; r < RT; r++) b.s[r] = s[r][(size_t)kb * 16];
    };
    auto load_x = [&](v8t(&rows)[4], uint32_t kb) __attribute__((always_inline)) {
        const uint32_t last = kb + 1 < a.KB ? 0 : ~0u;
        kb = kb < a.KB ? kb : a.KB - 1;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) rows[i] = __builtin_bit_cast(v8t, __builtin_amdgcn_raw_buffer_load_b128(xbuf, xoff[i] + (beyond[i] & last), kb * 256, 0));
    };
    // rows to operands; in LDS the pieces of a row stand in the order piece ^ row, which gives reads and writes all banks (within a wavefront, whose accesses to LDS keep their order)
    v8t *const stage = reinterpret_cast<v8t *>(shared[wave]);
    auto       turn = [&](v8t(&x)[4], const v8t(&rows)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) stage[(4 * i + q) * 16 + (c ^ (4 * i + q))] = rows[i];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) x[i] = stage[c * 16 + ((4 * i + q) ^ c)];
    };
    v4f sum[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) sum[r] = (v4f){ 0.f, 0.f, 0.f, 0.f };
    auto multiply = [&](const B &b, const v8t(&x)[4]) __attribute__((always_inline)) {
        constexpr int kEach = 4 / GPB; // steps of a group
        constexpr bool kStart = FP6MI_TYPE == 1;
        FewZero        zero;
        zero.set((T)8.f);
        v4f start[GPB]; // the groups' sums of X; without zero points -24 times that, which all rows' products start from
#if FP6MI_TYPE == 1
        const T   each = (T)(Z ? 1.f : -24.f);
        const v8t ones = { each, each, each, each, each, each, each, each };
#pragma unroll
        for (int g = 0; g < GPB; g++) {
            start[g] = (v4f){ 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int i = 0; i < kEach; i++) start[g] = mfma(x[g * kEach + i], ones, start[g]);
        }
#endif
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int g = 0; g < GPB; g++) {
                const float scale = (float)b.s[r].v[Z ? 2 * g : g];
                if constexpr (Z) zero.set(b.s[r].v[2 * g + 1]);
                v8t v[kEach];
#pragma unroll
                for (int i = 0; i < kEach; i++) v[i] = codes_of(b.w[r][g * kEach + i], zero, cut);
                v4f y = { 0.f, 0.f, 0.f, 0.f };
#if FP6MI_TYPE == 1
                y = Z ? start[g] * zero.all : start[g];
#endif
#pragma unroll
                for (int i = 0; i < kEach; i++) y = mfma(x[g * kEach + i], v[i], y);
#pragma unroll
                for (int i = 0; i < 4; i++) sum[r][i] += scale * y[i];
                if (kStart && Z && GPB == 4 && RT == 4 && g == GPB - 1 && r % 2 == 1) __builtin_amdgcn_sched_barrier(0); // (or conversions come so early that registers spill: 16 -> 28 us for 8192x8192)
            }
    };
    B        b[2];
    v8t      x[2][4], rows[4]; // operands of this block and the next, rows of the one behind it
    uint32_t kb = wave;
    auto next = [&](v8t(&to)[4], uint32_t kb) __attribute__((always_inline)) {
        if constexpr (kTurn) {
            turn(to, rows);
            load_x(rows, kb + WK);
        } else {
            load_x(to, kb);
        }
    };
    if (kb < a.KB) {
        load_x(x[kTurn], kb);
        load(b[0], kb);
        if constexpr (kTurn) {
            load_x(rows, kb + WK);
            turn(x[0], x[1]);
        }
        for (; kb + 2 * WK < a.KB; kb += 2 * WK) {
            load(b[1], kb + WK);
            next(x[1], kb + WK);
            multiply(b[0], x[0]);
            __builtin_amdgcn_sched_barrier(0); // (or loads sink behind the next block's conversions: 37.6 -> 32.2 us for 64 experts of 2560x2048 at 320 rows)
            load(b[0], kb + 2 * WK);
            next(x[0], kb + 2 * WK);
            multiply(b[1], x[1]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (kb + WK < a.KB) {
            load(b[1], kb + WK);
            if constexpr (kTurn)
                turn(x[1], rows);
            else
                load_x(x[1], kb + WK);
            multiply(b[0], x[0]);
            multiply(b[1], x[1]);
        } else {
            multiply(b[0], x[0]);
        }
    }
#if FP6MI_TYPE == 1
    // Sums that are no numbers: 16 + q times a value of X has left float32's range, or there are infinities or NaN in X (or the scales).  The wavefront goes over its blocks again with (q - z) / 4096, which is exact in
    // bf16 and keeps any sum of 128 products in range, so that what is finite comes out finite and an infinity as one, as from the tiles; finite sums stay as they are.  (28672x8192, 4 rows, one of which holds an
    // infinity: 76 us instead of 26.6.)
    bool lost = false;
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) lost |= !__builtin_isfinite(sum[r][i]);
    if (__builtin_expect(__any(lost), 0)) {
        constexpr int kEach = 4 / GPB;
        uint32_t      expert = t.expert;
        asm("" : "+s"(expert)); // (addresses of their own: those above need not be kept for this)
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const size_t at = ((size_t)expert * a.Mt + (m0 + r < a.Mt ? m0 + r : a.Mt - 1)) * a.KB;
            v4f          whole = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll 1
            for (uint32_t k = wave; k < a.KB; k += WK) {
                const v4u            codes = static_cast<const v4u *>(a.W)[(at + k) * 64 + lane];
                const Scales<GPB, Z> of = static_cast<const Scales<GPB, Z> *>(a.S)[(at + k) * 16 + c];
#pragma unroll
                for (int g = 0; g < GPB; g++) {
                    const float zero = Z ? (float)of.v[2 * g + 1] : 8.f;
                    v4f         y = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
                    for (uint32_t i = g * kEach; i < (g + 1) * kEach; i++) {
                        const uint32_t column = k * 128 + i * 32 + q * 8;
                        const v8t      x = __builtin_bit_cast(v8t, __builtin_amdgcn_raw_buffer_load_b128(xbuf, column < a.K ? (c * a.K + column) * 2 : 0x80000000u, 0, 0));
                        v8t            v;
#pragma unroll
                        for (int j = 0; j < 8; j++) v[j] = (T)(((float)(codes[i] >> 4 * (j % 2 * 4 + j / 2) & 15u) - zero) * 0x1p-12f);
                        y = mfma(x, v, y);
                    }
                    const float scale = (float)of.v[Z ? 2 * g : g];
#pragma unroll
                    for (int i = 0; i < 4; i++) whole[i] += scale * y[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!__builtin_isfinite(sum[r][i])) sum[r][i] = whole[i] * 0x1p12f;
        }
    }
#endif
#pragma unroll
    for (int r = 0; r < RT; r++) shared[wave][r][lane] = sum[r];
    __syncthreads();

    // the sums of row tile r: lane c + 16 q has weight row c and rows 4 q + i of X
    auto total = [&](int r) __attribute__((always_inline)) {
        v4f y = shared[0][r][lane];
#pragma unroll
        for (int k = 1; k < WK; k++) y += shared[k][r][lane];
        return y;
    };
    const T *bias = a.bias ? static_cast<const T *>(a.bias) + (size_t)t.expert * a.Mt * 16 : nullptr;
    if (a.act < 0) {
        for (uint32_t r = wave; r < RT; r += WK) {
            const uint32_t m = (m0 + r) * 16 + c;
            if (m0 + r >= a.Mt) continue;
            v4f         y = total(r);
            const float add = bias ? (float)bias[m] : 0.f;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                if (4 * q + i < t.rows) store(a, t.row + 4 * q + i, m, a.Mt * 16, y[i] + add);
        }
    } else if constexpr (RT % 2 == 0) {
        for (uint32_t r = 2 * wave; r < RT; r += 2 * WK) {
            const uint32_t m = (m0 + r) * 16 + c;
            if (m0 + r >= a.Mt) continue;
            v4f         g = total(r), u = total(r + 1);
            const float bg = bias ? (float)bias[m] : 0.f, bu = bias ? (float)bias[m + 16] : 0.f;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                if (4 * q + i < t.rows) store(a, t.row + 4 * q + i, (m0 + r) * 8 + c, a.Mt * 8, activated(a.act, g[i] + bg) * (u[i] + bu));
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
template <int GPB, bool Z, int RT, int WK> int launch_stream(hipStream_t st, const Int4Args &a)
{
    const size_t tiles = fp6mi::int4_tiles(a.N, a.offsets ? a.E : 0, 16);
    hipLaunchKernelGGL((int4_stream<GPB, Z, RT, WK>), dim3((a.Mt + RT - 1) / RT, (uint32_t)tiles), dim3(WK * 64), 0, st, a);
    return (int)hipGetLastError();
}

#if FP6MI_TYPE == 1 && FP6MI_GROUPS == 1
// Rows in bf16 as fp16 times a power of two for each row, which puts the largest finite magnitude from 2^15 to 2^16 (65280 at most: eight bits).  What is smaller than 2^-32 of that loses bits, half of 2^-24
// and so 2^-40 of it at most: a float32 sum of such products has been rounded by more.  Infinities and NaN stay.  A workgroup to a row, which reads it twice (from L2); 4096 rows of 4096 take 15.4 us, 4.4 TB/s.
// (From 2^23 rows on a workgroup has more than one: a grid has fewer than 2^32 threads.)
__global__ __launch_bounds__(256) void rows_to_halfs(half_t *__restrict__ out, int *__restrict__ exponents, const T *__restrict__ X, uint32_t N, uint32_t K)
{
    __shared__ uint32_t most[4];
    const uint32_t tid = threadIdx.x, pieces = K / 8;
    for (uint32_t row = blockIdx.x; row < N; row += gridDim.x) {
        const v4u     *x = reinterpret_cast<const v4u *>(X + (size_t)row * K);
        uint32_t       top = 0; // exponent field and mantissa of the largest finite magnitude
        auto           field = [](uint32_t b) { return b < 0x7f80u ? b : 0u; };
        for (uint32_t i = tid; i < pieces; i += 256) {
            const v4u v = x[i];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t lo = field(v[j] & 0x7fffu), hi = field(v[j] >> 16 & 0x7fffu);
                top = top > lo ? top : lo, top = top > hi ? top : hi;
            }
        }
#pragma unroll
        for (int m = 32; m; m >>= 1) {
            const uint32_t o = __shfl_xor(top, m);
            top = top > o ? top : o;
        }
        if ((tid & 63) == 0) most[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; w++) top = top > most[w] ? top : most[w];
        const int e = top ? (int)(top >> 7 > 1 ? top >> 7 : 1) - 127 - 15 : 0;
        if (tid == 0) exponents[row] = e;
        for (uint32_t i = tid; i < pieces; i += 256) {
            const v4u v = x[i];
            v8h       h;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                h[2 * j] = (half_t)__builtin_ldexpf(__builtin_bit_cast(float, v[j] << 16), -e);
                h[2 * j + 1] = (half_t)__builtin_ldexpf(__builtin_bit_cast(float, v[j] & 0xffff0000u), -e);
            }
            reinterpret_cast<v8h *>(out + (size_t)row * K)[i] = h;
        }
        __syncthreads(); // (the maxima are overwritten)
    }
}
#endif

// ---------------------------------------------------------------------------------------------------------------
// More rows: tiles of WR * RT row tiles x NT * 16 rows of X to a workgroup of WR x WK wavefronts; the WK groups take every WK-th column block.  X goes to LDS by direct transfers, a K block ahead, two
// stages to a group; a row of a stage is 256 bytes whose 16 pieces stand in the order piece ^ (row & 15), which gives the reads of an MFMA operand all banks.  A wavefront holds its X of one block in
// registers and takes one of its RT row tiles after another: its codes become operands while the tile before is multiplied.
// Many rows are bound by the matrix units with the conversions and the scaling of the group sums beside them (3.6 VALU instructions to a matrix instruction; twice the columns to a wavefront, 2.6, was no
// faster, nor were 32x32x16 instructions, which draw more power): 8192x8192 at 777 rows takes 108 to 114 us, 8 experts of 22016x4096 at 4096 rows 720 to 750, 1.0 PFLOP/s, where a library's product of large
// dense fp16 matrices reaches 1.2.  Two workgroups to a CU where LDS allows, so that one multiplies while the other waits at its barrier.
// 17 to some 100 rows reach neither the matrix units nor memory: 11 to 14 bytes of the weights a ns and CU, of a copy 20.  Tiles are as many there as there are CUs, of three, four, six or eight row tiles
// (10240x4576 at 19 rows: 13.0 us in 160 workgroups of four row tiles, 11.1 in 214 of three), so that weights are loaded and converted again for every 32 rows; of 21.7 us of 8192x8192 at 64 rows, without
// codes and scales 13.0 were left, without the transfers of X 18.8, without conversions 19.4, and more stages or blocks ahead did nothing.
// ---------------------------------------------------------------------------------------------------------------
template <int RT, int NT, int WR, int WK> constexpr size_t tile_lds_bytes() // the stages; the sums of the groups on their way to the first; the outputs on their way out (a half at a time where they are float32)
{
    const size_t stages = (size_t)WK * 2 * NT * 4096, sums = (size_t)(WK - 1) * WR * RT * NT * 1024, outputs = NT * 16 * ((size_t)WR * RT * 32 + 16);
    return stages > outputs ? (stages > sums ? stages : sums) : (outputs > sums ? outputs : sums);
}

template <int GPB, bool Z, int RT, int NT, int WR, int WK> __global__ __launch_bounds__(WR *WK * 64, 2) void int4_tile(const Int4Args a, uint32_t col_tiles)
{
    static_assert((NT == 2 && RT >= 2 && RT <= 4) || (NT == 4 && RT == 4), "the steps of a block are written for these");
    constexpr int      A = WR == 1 && RT < 4 ? 2 : 1; // blocks of codes on their way: two where a wavefront asks for few at a time (10240x4576 at 19 rows 11.6 -> 11.1 us; 1 to 4 % slower elsewhere)
    constexpr int      kWaves = WR * WK, kCols = NT * 16, kTiles = WR * RT, kRows = kTiles * 16, kStage = kCols * 256, kDma = kCols / 4 / WR;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, q = lane >> 4, wr = wave % WR, wk = wave / WR;

    // Workgroups that an XCD runs side by side are panels of eight row blocks by a few column tiles, mostly of one expert.
    const uint32_t per = gridDim.x >> 3, rem = gridDim.x & 7u, xcd = blockIdx.x & 7u, id = xcd * per + (xcd < rem ? xcd : rem) + (blockIdx.x >> 3);
    const uint32_t row_blocks = gridDim.x / col_tiles, first = id / (8 * col_tiles) * 8, in = id - first * col_tiles, high = row_blocks - first < 8 ? row_blocks - first : 8;
    const uint32_t m0 = (first + in % high) * kTiles;
    const Tile     t = tile_of(a, in / high, kCols);
    if (t.rows == 0) return;
    if (t.expert < 0) return store_zeros(a, t, m0, kTiles, kWaves * 64);

    // transfers of X: four rows of one block each
    typedef __attribute__((address_space(3))) void lvoid;
    const auto     xbuf = __builtin_amdgcn_make_buffer_rsrc(const_cast<half_t *>(static_cast<const half_t *>(a.X) + (size_t)t.row * a.K), 0, (int)(t.rows * a.K * 2), 0x00027000);
    uint8_t *const xstage = lds + wk * 2 * kStage;
    const uint32_t xrow0 = (4 * wr + q) * a.K * 2; // 32 bits: the launcher bounds K
    auto           transfer = [&](uint32_t kb, uint32_t stage) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t j = 0; j < kDma; j++) {
            uint32_t row = xrow0, piece = c ^ q;
            if constexpr (kDma > 4) asm("" : "+v"(row), "+v"(piece)); // (each address for itself when it is needed: kept, they take the registers of a tile)
            row += j * WR * 8 * a.K, piece ^= 4 * ((j * WR + wr) & 3);
            const uint32_t k = kb * 128 + piece * 8, off = row + (k < a.K ? k * 2 : 0xc0000000u); // (beyond the buffer, as the rows behind the last one: reads as zeros and asks for nothing)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xbuf, (lvoid *)(xstage + stage * kStage + (j * WR + wr) * 1024), 16, off, 0, 0, 0);
        }
    };
    // operands of X: of the first two tiles of the next block while this one's are still in use, of the others in their place
    const uint8_t *xread = xstage + c * 256;
    v8h            early[2][2][4], late[NT > 2 ? NT - 2 : 1][4];
    auto           read_x = [&](v8h &to, int n, uint32_t i, uint32_t stage) __attribute__((always_inline)) {
        to = *reinterpret_cast<const v8h *>(xread + stage * kStage + n * 16 * 256 + ((4 * i + q) ^ c) * 16);
    };

    // codes and scales, by scalar offsets from the wavefront's first row tile (row tiles beyond the last one take it again); a row tile's are asked for again as soon as they are converted
    const uint32_t tile0 = m0 + wr * RT < a.Mt ? m0 + wr * RT : a.Mt - 1, tiles = a.Mt - tile0 < RT ? a.Mt - tile0 : RT;
    const size_t   at = ((size_t)t.expert * a.Mt + tile0) * a.KB;
    const auto     wbuf = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(static_cast<const uint8_t *>(a.W) + at * 1024), 0, (int)(tiles * a.KB * 1024), 0x00027000);
    constexpr int  kScaleBytes = sizeof(Scales<GPB, Z>) * 16;
    const auto     sbuf = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(static_cast<const uint8_t *>(a.S) + at * kScaleBytes), 0, (int)(tiles * a.KB * kScaleBytes), 0x00027000);
    v4u            raw[A][RT];
    Scales<GPB, Z> scales[A][RT];
    auto           load_w = [&](int set, int r, uint32_t kb) __attribute__((always_inline)) {
        const uint32_t block = (r < (int)tiles ? r : tiles - 1) * a.KB + (kb < a.KB ? kb : a.KB - 1);
        raw[set][r] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(wbuf, lane * 16, block * 1024, 0));
        if constexpr (sizeof(scales[set][r]) == 2) scales[set][r] = __builtin_bit_cast(Scales<GPB, Z>, __builtin_amdgcn_raw_buffer_load_b16(sbuf, c * 2, block * kScaleBytes, 0));
        if constexpr (sizeof(scales[set][r]) == 4) scales[set][r] = __builtin_bit_cast(Scales<GPB, Z>, __builtin_amdgcn_raw_buffer_load_b32(sbuf, c * 4, block * kScaleBytes, 0));
        if constexpr (sizeof(scales[set][r]) == 8) scales[set][r] = __builtin_bit_cast(Scales<GPB, Z>, __builtin_amdgcn_raw_buffer_load_b64(sbuf, c * 8, block * kScaleBytes, 0));
        if constexpr (sizeof(scales[set][r]) == 16) scales[set][r] = __builtin_bit_cast(Scales<GPB, Z>, __builtin_amdgcn_raw_buffer_load_b128(sbuf, c * 16, block * kScaleBytes, 0));
    };
    constexpr int kEach = 4 / GPB; // matrix instructions of a group
    Codes         op[2][4];
    Zero          zero;
    const Cutter  cut;
    float         scale[2][GPB];
    auto          convert = [&](int set, int to, int r, int i, int half) __attribute__((always_inline)) {
        if (half == 0 && i % kEach == 0) zero.set(Z ? scales[set][r].v[i / kEach * 2 + 1] : (T)8.f);
        codes_half(op[to][i], raw[set][r][i], zero, cut, half);
    };
    auto take_scales = [&](int set, int to, int r) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < GPB; g++) scale[to][g] = (float)scales[set][r].v[Z ? 2 * g : g];
    };
    v4f sum[RT][NT], y[2][2];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int n = 0; n < NT; n++) sum[r][n] = (v4f){ 0.f, 0.f, 0.f, 0.f };
    y[1][0] = y[1][1] = (v4f){ 0.f, 0.f, 0.f, 0.f };
#pragma unroll
    for (int g = 0; g < GPB; g++) scale[1][g] = 0.f;

    // A block is RT * NT / 2 steps of two tiles of X by one row tile; a step also converts its share of the next row tile, adds up the groups that the step before has multiplied, and reads some of the
    // next block's X.  The last row tile takes the early tiles of X last, so that the registers of the others are free for the next block's.
    constexpr int kPairs = NT / 2, kSteps = RT * kPairs;
    auto          step = [&](auto u_c, auto set_c, uint32_t kb) __attribute__((always_inline)) {
        constexpr int u = decltype(u_c)::value, set = decltype(set_c)::value, r = u / kPairs, p = u % kPairs, odd = set * RT; // (a block of three row tiles swaps what alternates)
        constexpr int n = 2 * (r == RT - 1 ? (p + 1) % kPairs : p), next = (r + 1) % RT, nset = A == 1 ? 0 : r + 1 < RT ? set : set ^ 1;
        constexpr int pu = u == 0 ? kSteps - 1 : u - 1, pr = pu / kPairs, pn = 2 * (pr == RT - 1 ? (pu % kPairs + 1) % kPairs : pu % kPairs); // the step before
        constexpr int before = r + odd - (p == 0 ? 1 : 0) + 2;
        if constexpr (u == kPairs) { // the next block's X has landed (behind its transfers come two loads for every row tile), and all have read this one's
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * RT) : "memory");
            transfer(kb + 2 * WK, set);
            asm volatile("" ::: "memory");
        }
        constexpr int kReads = RT == 2 ? 8 : NT == 2 ? 4 : 2; // of an early tile's operands in a step
        if constexpr (u >= kPairs && u < kPairs + 8 / kReads) {
#pragma unroll
            for (int e = (u - kPairs) * kReads; e < (u - kPairs + 1) * kReads; e++) read_x(early[set ^ 1][e / 4][e % 4], e / 4, e % 4, set ^ 1);
        }
        if constexpr (r == RT - 1 && p > 0) { // in the place of the step before
#pragma unroll
            for (int i = 0; i < 8; i++) read_x(late[pn - 2 + i / 4][i % 4], pn + i / 4, i % 4, set ^ 1);
        }
        // of the groups multiplied before: pair v of them, tiles n and n + 1 of X by row tile r, from tile `from` of the two on
        auto add = [&](int r, int s, int n, int g, int v, int from, int to) __attribute__((always_inline)) {
#pragma unroll
            for (int k = from; k < to; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) sum[r][n + k][i] += scale[s & 1][g] * y[v & 1][k][i];
        };
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int v = (u + odd) * GPB + i / kEach;
#pragma unroll
            for (int k = 0; k < 2; k++)
                y[v & 1][k] = mfma_halfs(n == 0 ? early[set][k][i] : late[n == 0 ? 0 : n - 2 + k][i], op[(r + odd) & 1][i].v, i % kEach == 0 ? (v4f){ 0.f, 0.f, 0.f, 0.f } : y[v & 1][k]);
            if constexpr (GPB == 1) {
                if (i == 1 || i == 2) add(pr, before, pn, 0, v + 1, i - 1, i);
            } else if constexpr (GPB == 2) {
                if (i == 1) add(pr, before, pn, 1, v + 1, 0, 2);
                if (i == 3) add(r, r + odd, n, 0, v + 1, 0, 2);
            } else {
                if (i == 0)
                    add(pr, before, pn, 3, v + 1, 0, 2);
                else
                    add(r, r + odd, n, i - 1, v + 1, 0, 2);
            }
            if constexpr (kPairs == 2) {
                convert(nset, (r + odd + 1) & 1, next, p * 2 + i / 2, i & 1);
            } else {
                convert(nset, (r + odd + 1) & 1, next, i, 0);
                convert(nset, (r + odd + 1) & 1, next, i, 1);
            }
            if (i < 3) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (p == kPairs - 1) {
            take_scales(nset, (r + odd + 1) & 1, next);
            if constexpr (A == 2) { // (the codes and scales are used before their registers are loaded again, or they would be loaded to others and waited for at the loop's end to be moved)
#pragma unroll
                for (int g = 0; g < GPB; g++) asm volatile("" : "+v"(scale[(r + odd + 1) & 1][g]));
                __builtin_amdgcn_sched_barrier(0);
            }
            load_w(nset, next, kb + (r + 1 < RT ? A : A + 1) * WK);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto block = [&](auto set_c, uint32_t kb) __attribute__((always_inline)) { sections<kSteps>([&](auto u_c) __attribute__((always_inline)) { step(u_c, set_c, kb); }); };
    transfer(wk, 0);
    load_w(0, 0, wk);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    transfer(wk + WK, 1);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; i++) read_x(early[0][i / 4][i % 4], i / 4, i % 4, 0);
#pragma unroll
    for (int i = 0; i < 4 * (NT - 2); i++) read_x(late[i / 4][i % 4], 2 + i / 4, i % 4, 0);
#pragma unroll
    for (int i = 0; i < 8; i++) convert(0, 0, 0, i / 2, i & 1);
    take_scales(0, 0, 0);
#pragma unroll
    for (int set = 0; set < A; set++)
#pragma unroll
        for (int r = 0; r < RT; r++) load_w(set, r, set == 0 && r == 0 ? wk + A * WK : wk + set * WK);
    uint32_t kb = wk, left = (a.KB + WK - 1) / WK; // blocks of every group (of those beyond the last one X reads as zeros)
    for (; left >= 2; left -= 2, kb += 2 * WK) {
        block(std::integral_constant<int, 0>{}, kb);
        block(std::integral_constant<int, 1>{}, kb + WK);
    }
    if (left) block(std::integral_constant<int, 0>{}, kb);
    const bool swapped = RT % 2 == 1 && left; // (of three row tiles an odd number of blocks)
#pragma unroll
    for (int k = 0; k < 2; k++) // the last pair
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float last = swapped ? scale[0][GPB - 1] * y[GPB % 2 == 1 ? 0 : 1][k][i] : scale[1][GPB - 1] * y[1][k][i];
            sum[RT - 1][k][i] += last;
        }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); // nothing is on its way to LDS any more

    if constexpr (WK > 1) { // the sums of the other groups to the first, [group][row wavefront][r][n][lane]
        auto at = [&](int g, int r, int n) { return reinterpret_cast<v4f *>(lds) + ((((g - 1) * WR + wr) * RT + r) * NT + n) * 64 + lane; };
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int n = 0; n < NT; n++)
                if (wk > 0) *at(wk, r, n) = sum[r][n];
        __syncthreads();
        if (wk == 0)
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int g = 1; g < WK; g++) sum[r][n] += *at(g, r, n);
        __syncthreads();
    }

    // outputs through LDS, so that a lane stores 16 bytes: [row of X][weight row], rows 16 bytes apart from a multiple of 128
    auto     exponent = [&](uint32_t n, uint32_t i) { return FP6MI_TYPE == 1 && n * 16 + 4 * q + i < t.rows ? a.exponents[t.row + n * 16 + 4 * q + i] : 0; };
    auto     scaled = [&](float v, int e) { return FP6MI_TYPE == 1 ? __builtin_ldexpf(v, e) : v; };
    const T *bias = a.bias ? static_cast<const T *>(a.bias) + (size_t)t.expert * a.Mt * 16 : nullptr;
    auto     out = [&](auto type, auto gated_c) __attribute__((always_inline)) {
        typedef decltype(type) O;
        constexpr bool     gated = decltype(gated_c)::value;
        constexpr uint32_t kHalves = sizeof(O) == 4 && !gated ? 2 : 1, kOut = gated ? kRows / 2 : kRows, kPitch = kOut * sizeof(O) + 16, kEach = 16 / sizeof(O), kNs = NT / kHalves;
        static_assert((size_t)kCols / kHalves * kPitch <= tile_lds_bytes<RT, NT, WR, WK>(), "");
        const uint32_t ld = a.Mt * (gated ? 8 : 16), col0 = m0 * (gated ? 8 : 16);
#pragma unroll
        for (uint32_t h = 0; h < kHalves; h++) {
            if (h) __syncthreads();
            if (wk == 0)
#pragma unroll
                for (uint32_t n = h * kNs; n < (h + 1) * kNs; n++)
#pragma unroll
                    for (uint32_t r = 0; r < RT; r += gated ? 2 : 1) {
                        const uint32_t m = (m0 + wr * RT + r) * 16 + c, row = (n - h * kNs) * 16 + 4 * q;
                        const bool     in = bias && m0 + wr * RT + r < a.Mt;
                        const float    b0 = in ? (float)bias[m] : 0.f, b1 = gated && in ? (float)bias[m + 16] : 0.f;
#pragma unroll
                        for (uint32_t i = 0; i < 4; i++) {
                            const int e = exponent(n, i);
                            float     v = scaled(sum[r][n][i], e) + b0;
                            if constexpr (gated) v = activated(a.act, v) * (scaled(sum[r + 1][n][i], e) + b1);
                            reinterpret_cast<O *>(lds + (row + i) * kPitch)[gated ? (wr * RT + r) * 8 + c : (wr * RT + r) * 16 + c] = (O)v;
                        }
                    }
            __syncthreads();
            constexpr uint32_t kPieces = kOut / kEach; // of a row
            for (uint32_t i = tid; i < kNs * 16 * kPieces; i += kWaves * 64) {
                const uint32_t row = i / kPieces, piece = i % kPieces, col = col0 + piece * kEach, n = h * kNs * 16 + row;
                if (n < t.rows && col < ld) // (ld is a multiple of 8)
                    *reinterpret_cast<v4u *>(static_cast<O *>(a.Y) + (size_t)(t.row + n) * ld + col) = *reinterpret_cast<const v4u *>(lds + row * kPitch + piece * 16);
            }
        }
    };
    if (a.act < 0) {
        if (a.out_f32)
            out(float{}, std::false_type{});
        else
            out(T{}, std::false_type{});
    } else if constexpr (RT % 2 == 0) {
        if (a.out_f32)
            out(float{}, std::true_type{});
        else
            out(T{}, std::true_type{});
    }
}

template <int GPB, bool Z, int RT, int NT, int WR, int WK> int launch_tile(hipStream_t st, const Int4Args &a)
{
    constexpr size_t bytes = tile_lds_bytes<RT, NT, WR, WK>();
    const size_t     cols = fp6mi::int4_tiles(a.N, a.offsets ? a.E : 0, NT * 16), rows = (a.Mt + WR * RT - 1) / (WR * RT);
    static_assert(WR * WK <= 8, "workgroups of up to 512 threads (fp6mi::kInt4MostTiles)");
    if constexpr (bytes > 65536)
        if (const int e = allow_dynamic_lds<int4_tile<GPB, Z, RT, NT, WR, WK>>(bytes)) return e;
    hipLaunchKernelGGL((int4_tile<GPB, Z, RT, NT, WR, WK>), dim3((uint32_t)(cols * rows)), dim3(WR * WK * 64), bytes, st, a, (uint32_t)cols);
    return (int)hipGetLastError();
}

template <int GPB, bool Z> int run(hipStream_t st, const Int4Args &a, int kernel)
{
    switch (kernel) { // (in the order of fp6mi::kInt4Kernels)
    case 0: return launch_stream<GPB, Z, 1, 16>(st, a);
    case 1: return launch_stream<GPB, Z, 2, 8>(st, a);
    case 2: return launch_stream<GPB, Z, 3, 8>(st, a);
    case 3: return launch_stream<GPB, Z, 4, 8>(st, a);
    case 4: return launch_stream<GPB, Z, 4, 4>(st, a);
    case 5: return launch_tile<GPB, Z, 3, 2, 1, 4>(st, a);
    case 6: return launch_tile<GPB, Z, 2, 2, 2, 4>(st, a);
    case 7: return launch_tile<GPB, Z, 3, 2, 2, 4>(st, a);
    case 8: return launch_tile<GPB, Z, 4, 2, 2, 4>(st, a);
    case 9: return launch_tile<GPB, Z, 4, 2, 2, 2>(st, a);
    case 10:
        if constexpr (GPB == 1) return launch_tile<GPB, Z, 4, 4, 2, 2>(st, a);
        break;
    case 11: return launch_tile<GPB, Z, 4, 4, 4, 1>(st, a);
    }
    return FP6MI_ERR_SHAPE;
}

} // namespace

#define FP6MI_NAME2(type, groups) int4_run_##type##_##groups
#define FP6MI_NAME(type, groups) FP6MI_NAME2(type, groups)
namespace fp6mi {
int FP6MI_NAME(FP6MI_TYPE, FP6MI_GROUPS)(void *stream, const Int4Args &a, bool zeros, int kernel)
{
    hipStream_t st = static_cast<hipStream_t>(stream);
    return zeros ? run<FP6MI_GROUPS, true>(st, a, kernel) : run<FP6MI_GROUPS, false>(st, a, kernel);
}

#if FP6MI_TYPE == 1 && FP6MI_GROUPS == 1
int int4_rows_to_halfs(void *stream, void *out, int *exponents, const void *X, size_t N, size_t K)
{
    hipLaunchKernelGGL(rows_to_halfs, dim3((uint32_t)(N < 1u << 23 ? N : 1u << 23)), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<half_t *>(out), exponents, static_cast<const T *>(X), (uint32_t)N,
                       (uint32_t)K);
    return (int)hipGetLastError();
}
#endif
} // namespace fp6mi
