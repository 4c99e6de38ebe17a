// gfx950 kernels around the FPx linear layer that read the native weight layout in another way than its GEMM, for ONE weight format per translation unit
// (compiled like fp6mi_gemm.hip, with -DFP6MI_FORMAT=<10*E+M>).  No counterpart in the reference, whose only operator is the forward product.
//   grad_tile   dX[N,K] = dY[N,M] . dequant(W)[M,K]: the input gradient of the linear layer
#include <hip/hip_runtime.h>

#include <atomic>
#include <type_traits>

#include "fp6mi_internal.h"

#ifndef FP6MI_FORMAT
#error "compile with -DFP6MI_FORMAT=32, 22, 23 or 21 (10*E + M of the weight format)"
#endif

namespace {

#include "fp6mi_device.inc"
#include "fp6mi_scale.inc"

// ---------------------------------------------------------------------------------------------------------------
// grad_tile: the product that contracts over the weights' rows.
//   dX[n, k] = sum over m of dY[n, m] * scale[m] * 2^(b-127) * value[m, k]
// The scale belongs to the contracted index, so it cannot wait for the epilogue as in the forward product.  It is taken apart, scale = mantissa * 2^e with
// 1 <= |mantissa| < 2: the conversion instruction applies 2^e along with the group's power of two, which leaves the weights exact (they have four significant bits), and
// the mantissa goes to dY, whose products are rounded to fp16 once (half a step, 2^-11; with a mantissa below two they keep dY's range).  PRE: dY comes multiplied already.
//   workgroup = 2 x WN wavefronts; tile = 256 input features (a native block's width) x (NT*WN*16) batch rows, 128 x (NT*16) of it per wavefront
// The native layout holds eight consecutive columns k of one row m in a lane, the MFMA wants eight consecutive rows m of one column.  So a chunk of OCC rows is
// converted once per workgroup, written to LDS as rows, and read back by the transposing read (ds_read_b64_tr_b16: of a 4 x 16 piece, lane l of
// sixteen gets column l).  Rows lie in LDS in the order in which those reads take them: row 8q + 4h + j of 32 is the (4q + j)-th of half h, 544 bytes apart, the
// halves 16 bytes more, which leaves both the writes (eight rows, 16 bytes each) and the reads (eight rows, 32 bytes each) free of bank conflicts.
// dY passes memory -> LDS without registers: piece p (16 bytes) of batch row n lies at slot p ^ swizzle(n) of its row.
// Two stages, one barrier a chunk; weights are asked for two chunks ahead.
// ---------------------------------------------------------------------------------------------------------------
typedef short v4s __attribute__((ext_vector_type(4)));
typedef _Float16 v4hh __attribute__((ext_vector_type(4)));

constexpr int kGradRow = 544, kGradHalf = 16 * kGradRow + 16, kGrad32 = 2 * kGradHalf; // bytes of a row, of 16 rows, of 32
template <int NT, int WN, int OCC> struct GradTile {
    static constexpr int TN = NT * WN * 16, kWStage = OCC / 32 * kGrad32, kXStage = TN * OCC * 2, kMant = kWStage + kXStage, kStage = kMant + OCC * 2;
    static constexpr int kOutFull = TN * (512 + 16), kOutPart = NT * 16 * (1024 + 16);
    static constexpr int kLds = 2 * kStage > kOutFull ? (2 * kStage > kOutPart ? 2 * kStage : kOutPart) : (kOutFull > kOutPart ? kOutFull : kOutPart);
};

// the 192-bit string of 6-bit fields of half a block, as convert_raw_half forms it
template <int FM, int H> __device__ __forceinline__ v6u raw_half_fields(const RawHalf &f)
{
    if constexpr (Fmt<FM>::bits == 6)
        return H == 0 ? (v6u){ f.p[0], f.p[1], f.p[2], f.p[3], f.s[0], f.s[1] } : (v6u){ f.s[0], f.s[1], f.p[0], f.p[1], f.p[2], f.p[3] };
    else if constexpr (Fmt<FM>::bits == 5)
        return fp5_expand(f.p[0], f.p[1], f.p[2], f.p[3], f.s[0]);
    else
        return fp4_expand(f.p);
}

// What the conversion of a row's codes applies, 2^(e + b - 127) (and the factor that the format's fields owe), and the rest of its scale.  A scale that is zero, infinite or no number is
// all mantissa.  (Powers of two beyond what the instruction takes have long left fp16.)
template <int FM, bool GS> __device__ __forceinline__ float grad_factor(half_t scale, uint32_t g, half_t &mantissa)
{
    int e = 0;
    mantissa = split_scale(scale, e);
    if constexpr (Fmt<FM>::post_scale == 4.0f) e += 2;
    static_assert(Fmt<FM>::post_scale == 1.0f || Fmt<FM>::post_scale == 4.0f, "a power of two");
    int field = e + (GS ? (int)g : 127);
    field = field < 0 ? 0 : field > 254 ? 254 : field;
    return __builtin_bit_cast(float, (uint32_t)field << 23);
}

// one lane's 4 x 16-bit share of a transposing read
__device__ __forceinline__ v4hh read_transposed(const uint8_t *p)
{
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    return __builtin_bit_cast(v4hh, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(p)));
}

template <int FM, bool GS, bool PRE, int NT, int WN, int OCC>
__global__ __launch_bounds__(2 * WN *kWave) void grad_tile(const uint8_t *W, const half_t *scales, const uint8_t *gexp, const half_t *dY, half_t *__restrict__ dX,
                                                           float *__restrict__ ws, uint32_t M, uint32_t N, uint32_t K, uint32_t units, uint32_t splits,
                                                           uint32_t nblocks)
{
    typedef GradTile<NT, WN, OCC> T;
    constexpr int TN = T::TN, RT = 8, WAVES = 2 * WN, NTHREADS = WAVES * kWave;
    constexpr int kPieces = OCC / 8;                    // 16-byte pieces of a batch row of a stage
    constexpr int kRowsPer = 64 / kPieces;              // batch rows of one transfer
    constexpr int kDma = TN / kRowsPer / WAVES, kUnits = OCC / 16 * 2 / WAVES; // transfers, and half blocks to convert, of a wavefront
    static_assert(kDma * WAVES * kRowsPer == TN && kUnits * WAVES == OCC / 8, "every wavefront does the same share");
    constexpr int kLoads = kUnits * ((Fmt<FM>::bits == 4 ? 1 : 2) + (GS ? 1 : 0) + 1); // (codes, group exponent, row scale)
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, q = lane >> 4, wi = wave & 1, wn = wave >> 1;

    const TileId   id = tile_of<256, TN>(splits, nblocks, N, M);
    const uint32_t kb = id.mb, nbase = id.nb * TN, chunks = M / OCC;
    uint32_t       c0 = 0, c1 = chunks;
    if (splits > 1) {
        const uint32_t avg = chunks / splits, extra = chunks % splits;
        c0 = id.split * avg + (id.split < extra ? id.split : extra);
        c1 = c0 + avg + (id.split < extra ? 1u : 0u);
    }

    v4f acc[RT][NT];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[r][t] = (v4f){ 0.f, 0.f, 0.f, 0.f };

    // half blocks of this wavefront: number u = wave + WAVES * i of a chunk is half u & 1 of row tile u >> 1
    struct Raw { RawHalf h; half_t sc; };
    auto load_raw = [&](Raw &f, int i, uint32_t c) __attribute__((always_inline)) {
        const uint32_t R = c * (OCC / 16) + ((wave + WAVES * i) >> 1);
        const size_t   blk = (size_t)R * units + kb;
        if (wi == 0)
            load_raw_half<FM, GS, 0>(f.h, W + blk * Fmt<FM>::block_bytes, GS ? gexp + blk * 32 : nullptr, lane);
        else
            load_raw_half<FM, GS, 1>(f.h, W + blk * Fmt<FM>::block_bytes, GS ? gexp + blk * 32 : nullptr, lane);
        f.sc = scales[R * 16 + col];
    };
    auto store_w = [&](const Raw &f, int i, uint32_t stage) __attribute__((always_inline)) {
        const int rt = (wave + WAVES * i) >> 1, o = 16 * (rt & 1) + col; // row within 32
        uint8_t  *dst = lds + stage * T::kStage + (rt >> 1) * kGrad32 + ((o >> 2) & 1) * kGradHalf + (4 * (o >> 3) + (o & 3)) * kGradRow + wi * 256 + q * 16;
        half_t       mantissa;
        const float  factor = grad_factor<FM, GS>(f.sc, f.h.g, mantissa);
        const v32h   v = fields_to_halfs<FM>(wi == 0 ? raw_half_fields<FM, 0>(f.h) : raw_half_fields<FM, 1>(f.h), factor);
#pragma unroll
        for (int s = 0; s < 4; s++) *reinterpret_cast<v8h *>(dst + 64 * s) = slice8(v, s);
        if (!PRE && wi == 0 && q == 0) *reinterpret_cast<half_t *>(lds + stage * T::kStage + T::kMant + (rt * 16 + col) * 2) = mantissa;
    };

    // transfer j of this wavefront fills batch rows kRowsPer * (wave + WAVES * j) .. of a stage; rows beyond N repeat the last one (never stored)
    typedef __attribute__((address_space(3))) void lvoid;
    auto swizzle = [](uint32_t n) { return kPieces == 8 ? n & 7 : (n >> 1) & 3; };
    const uint32_t xrow = lane / kPieces, xlast = N - nbase < (uint32_t)TN ? N - 1 - nbase : TN - 1;
    const auto     xbuf = __builtin_amdgcn_make_buffer_rsrc(const_cast<half_t *>(dY + (size_t)nbase * M), 0, (int)((xlast + 1) * M * 2), 0x00027000); // (the launcher bounds M)
    auto           transfer = [&](int j, uint32_t c, uint32_t stage) __attribute__((always_inline)) {
        uint32_t       n = kRowsPer * (wave + WAVES * j) + xrow;
        const uint32_t piece = (lane % kPieces) ^ swizzle(n);
        n = n < xlast ? n : xlast;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xbuf, (lvoid *)(lds + stage * T::kStage + T::kWStage + (wave + WAVES * j) * 1024), 16,
                                                 n * M * 2 + c * (OCC * 2) + piece * 16, 0, 0, 0);
    };

    const uint8_t *wread = lds + (4 * q + (col >> 2)) * kGradRow + (col & 3) * 8 + wi * 256;
    auto           compute = [&](uint32_t stage) __attribute__((always_inline)) {
#pragma unroll
        for (int kk = 0; kk < OCC / 32; kk++) {
            v8h a[RT], b[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int n = (wn * NT + t) * 16 + col;
                b[t] = *reinterpret_cast<const v8h *>(lds + stage * T::kStage + T::kWStage + n * (OCC * 2) + (((4 * kk + q) ^ swizzle(n)) * 16));
            }
            if constexpr (!PRE) {
                const v8h mant = *reinterpret_cast<const v8h *>(lds + stage * T::kStage + T::kMant + (32 * kk + 8 * q) * 2);
#pragma unroll
                for (int t = 0; t < NT; t++) b[t] = b[t] * mant;
            }
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const uint8_t *p = wread + stage * T::kStage + kk * kGrad32 + r * 32;
                const v4hh     lo = read_transposed(p), hi = read_transposed(p + kGradHalf);
                a[r] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int t = 0; t < NT; t++) acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[r], b[t], acc[r][t], 0, 0, 0);
        }
    };

    if (c0 < c1) { // (more splits than chunks leave some empty: their partial sums are zeros)
        Raw even[kUnits], odd[kUnits];
#pragma unroll
        for (int i = 0; i < kUnits; i++) load_raw(even[i], i, c0);
#pragma unroll
        for (int j = 0; j < kDma; j++) transfer(j, c0, 0);
#pragma unroll
        for (int i = 0; i < kUnits; i++) load_raw(odd[i], i, c0 + 1 < c1 ? c0 + 1 : c0);
#pragma unroll
        for (int i = 0; i < kUnits; i++) store_w(even[i], i, 0);
        wait_transfers_and_barrier<0>();
        // chunk c from stage `st`; `cur` holds the codes of the next one.  (After the last chunk one is fetched and converted once more, and not used: every chunk
        // has the same waits.  Two copies of the code, so that codes on their way are never moved between registers.)
        auto chunk = [&](auto st_c, uint32_t c, Raw(&cur)[kUnits], Raw(&after)[kUnits]) __attribute__((always_inline)) {
            constexpr int  st = decltype(st_c)::value;
            const uint32_t ct = c + 1 < c1 ? c + 1 : c, cr = c + 2 < c1 ? c + 2 : c1 - 1;
#pragma unroll
            for (int j = 0; j < kDma; j++) transfer(j, ct, st ^ 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kUnits; i++) load_raw(after[i], i, cr);
            __builtin_amdgcn_sched_barrier(0);
            compute(st);
#pragma unroll
            for (int i = 0; i < kUnits; i++) store_w(cur[i], i, st ^ 1);
            wait_transfers_and_barrier<kLoads>();
        };
        typedef std::integral_constant<int, 0> Stage0;
        typedef std::integral_constant<int, 1> Stage1;
        for (uint32_t c = c0; c < c1; c += 2) {
            chunk(Stage0{}, c, odd, even);
            if (c + 1 < c1) chunk(Stage1{}, c + 1, even, odd);
        }
    }
    wait_transfers_and_barrier<0>(); // nothing is on its way to LDS any more, and nobody reads operands

    // acc[r][t][i]: input feature 256 kb + 128 wi + 16 r + 4 q + i of batch row nbase + 16 (wn NT + t) + col.  Out through LDS as in the other tile kernels.
    const uint32_t k0 = kb * 256;
    if (splits == 1) {
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int t = 0; t < NT; t++)
                *reinterpret_cast<v4hh *>(lds + ((wn * NT + t) * 16 + col) * 528 + (wi * 128 + 16 * r + 4 * q) * 2) =
                    (v4hh){ (half_t)acc[r][t][0], (half_t)acc[r][t][1], (half_t)acc[r][t][2], (half_t)acc[r][t][3] };
        __syncthreads();
        for (int p = tid; p < TN * 32; p += NTHREADS) {
            const uint32_t n = nbase + (p >> 5), k = k0 + (p & 31) * 8;
            if (n < N && k < K) *reinterpret_cast<v4u *>(dX + (size_t)n * K + k) = *reinterpret_cast<const v4u *>(lds + (p >> 5) * 528 + (p & 31) * 16);
        }
    } else {
        float *out = ws + (size_t)id.split * N * K;
#pragma unroll
        for (int part = 0; part < WN; part++) { // (the columns of all wavefronts at once would not fit)
            if (wn == part)
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int t = 0; t < NT; t++) *reinterpret_cast<v4f *>(lds + (t * 16 + col) * 1040 + (wi * 128 + 16 * r + 4 * q) * 4) = acc[r][t];
            __syncthreads();
            for (int p = tid; p < NT * 16 * 64; p += NTHREADS) {
                const uint32_t n = nbase + part * NT * 16 + (p >> 6), k = k0 + (p & 63) * 4;
                if (n < N && k < K) *reinterpret_cast<v4u *>(out + (size_t)n * K + k) = *reinterpret_cast<const v4u *>(lds + (p >> 6) * 1040 + (p & 63) * 16);
            }
            __syncthreads();
        }
    }
}

template <int FM, bool GS, bool PRE, int NT, int WN, int OCC>
int launch_grad(hipStream_t st, const void *W, const void *sc, const void *gexp, const void *dY, void *dX, float *ws, size_t M, size_t N, size_t K, int splits)
{
    typedef GradTile<NT, WN, OCC> T;
    static_assert(T::kLds <= 160 * 1024, "tile does not fit in LDS");
    const uint32_t units = (uint32_t)((K + 255) / 256), nblocks = (uint32_t)((N + T::TN - 1) / T::TN);
    const size_t   wgs = (size_t)units * (size_t)splits * nblocks;
    if (wgs > 0x7fffffffu || M > (size_t)1 << 20) return FP6MI_ERR_SHAPE; // (M: 32-bit offsets over TN batch rows)
    if (T::kLds > 48 * 1024)
        if (int rc = allow_dynamic_lds<&grad_tile<FM, GS, PRE, NT, WN, OCC>>(T::kLds)) return rc;
    hipLaunchKernelGGL((grad_tile<FM, GS, PRE, NT, WN, OCC>), dim3((uint32_t)wgs), dim3(2 * WN * kWave), T::kLds, st, static_cast<const uint8_t *>(W),
                       static_cast<const half_t *>(sc), static_cast<const uint8_t *>(gexp), static_cast<const half_t *>(dY), static_cast<half_t *>(dX), ws,
                       (uint32_t)M, (uint32_t)N, (uint32_t)K, units, (uint32_t)splits, nblocks);
    return (int)hipGetLastError();
}

template <int FM, bool GS, bool PRE>
int grad_cfg(hipStream_t st, const void *W, const void *sc, const void *gexp, const void *dY, void *dX, float *ws, size_t M, size_t N, size_t K, int splits)
{
    if (N <= 32) return launch_grad<FM, GS, PRE, 1, 2, 64>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits);
    if (N <= 64) return launch_grad<FM, GS, PRE, 2, 2, 64>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits);
    return launch_grad<FM, GS, PRE, 4, 2, 32>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits);
}

template <int FM>
int op_grad(void *stream, const void *W, const void *sc, const void *gexp, const void *dY, bool premultiplied, void *dX, float *ws, size_t M, size_t N, size_t K, int splits)
{
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (premultiplied)
        return gexp ? grad_cfg<FM, true, true>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits) : grad_cfg<FM, false, true>(st, W, sc, nullptr, dY, dX, ws, M, N, K, splits);
    return gexp ? grad_cfg<FM, true, false>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits) : grad_cfg<FM, false, false>(st, W, sc, nullptr, dY, dX, ws, M, N, K, splits);
}

} // namespace

namespace fp6mi {
#define FP6MI_OPS_NAME_(f) block_ops_##f
#define FP6MI_OPS_NAME(f) FP6MI_OPS_NAME_(f)
const BlockOps &FP6MI_OPS_NAME(FP6MI_FORMAT)()
{
    static const BlockOps ops = { &op_grad<FP6MI_FORMAT> };
    return ops;
}
} // namespace fp6mi
