// gfx950 kernels around the FPx linear layer that read the native weight layout in another way than its GEMM, for ONE weight format per translation unit
// (compiled like fp6mi_gemm.hip, with -DFP6MI_FORMAT=<10*E+M>).  No counterpart in the reference, whose only operator is the forward product.
//   gated_stream, gated_tile, gated_ws, gated_wide   H = act(X . Wg^T + bg) * (X . Wu^T + bu): the gated feed-forward block, on weights in pair order
//   grad_tile, grad_stream   dX[N,K] = dY[N,M] . dequant(W)[M,K]: the input gradient of the linear layer
#include <hip/hip_runtime.h>

#include <atomic>
#include <type_traits>

#include "fp6mi_internal.h"

#ifndef FP6MI_FORMAT
#error "compile with -DFP6MI_FORMAT=32, 22, 23 or 21 (10*E + M of the weight format)"
#endif

namespace {

using fp6mi::LaunchCfg;

#include "fp6mi_device.inc"
#include "fp6mi_scale.inc"
#include "fp6mi_activation.inc"

// ---------------------------------------------------------------------------------------------------------------
// grad_tile: the product that contracts over the weights' rows.
//   dX[n, k] = sum over m of dY[n, m] * scale[m] * 2^(b-127) * value[m, k]
// The scale belongs to the contracted index, so it cannot wait for the epilogue as in the forward product.  It is taken apart, scale = mantissa * 2^e with
// 1/2 <= |mantissa| < 1: the conversion instruction applies 2^e along with the group's power of two, which leaves the weights exact (they have four significant bits), and
// the mantissa goes to dY, whose products are rounded to fp16 once (half a step, 2^-11) and stay within fp16 wherever dY does.  PRE: dY comes multiplied already.
//   workgroup = 2 x WN wavefronts; tile = 256 input features (a native block's width) x (NT*WN*16) batch rows, 128 x (NT*16) of it per wavefront
// The native layout holds eight consecutive columns k of one row m in a lane, the MFMA wants eight consecutive rows m of one column.  So a chunk of OCC rows is
// converted once per workgroup, written to LDS as rows, and read back by the transposing read (ds_read_b64_tr_b16: of a 4 x 16 piece, lane l of
// sixteen gets column l).  Rows lie in LDS in the order in which those reads take them: row 8q + 4h + j of 32 is the (4q + j)-th of half h, 544 bytes apart, the
// halves 16 bytes more, which leaves both the writes (eight rows, 16 bytes each) and the reads (eight rows, 32 bytes each) free of bank conflicts.
// Piece p (16 bytes) of batch row n of dY lies at slot p ^ swizzle(n) of its row.  It passes through registers, where the mantissas are multiplied in.  (Behind a transfer straight to LDS
// the compiler holds the next transposing read back until the transfer is there.)
// What bounds it: with 128 x 128 outputs a wavefront (256 x 256 a workgroup, one wavefront to a SIMD) the MFMAs, of which 64 take an operand read of 24 KB; the LDS unit is busy for a third
// of the time, bank conflicts are none.  What was gained on the way, 8192x8192 N 4096, us: 256 x 128 tiles, operands read as they are multiplied 1414; read a step ahead 498;
// 256 x 256 466; other instructions spread between the MFMAs 448 (1.23 PFLOP/s; the fp16 library product of the card reaches 1.41).  22016x4096 N 4096 598, N 512 100 to 108 (4 splits),
// 4608x4544 N 333 33 (4 splits).  Left out: 256 x 128 with two workgroups of four wavefronts to a CU (515) and chunks of 32 rows.
// Two stages, one barrier a chunk.
// ---------------------------------------------------------------------------------------------------------------
typedef short v4s __attribute__((ext_vector_type(4)));
typedef _Float16 v4hh __attribute__((ext_vector_type(4)));

constexpr int kGradRow = 544, kGradHalf = 16 * kGradRow + 16, kGrad32 = 2 * kGradHalf; // bytes of a row, of 16 rows, of 32
constexpr int kGradRows = 64; // weight rows of a chunk
template <int NT, int WN> struct GradTile {
    static constexpr int TN = NT * WN * 16, kWStage = kGradRows / 32 * kGrad32, kXStage = TN * kGradRows * 2, kStage = kWStage + kXStage;
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

// One lane's 32 weights of a row (fields: their codes; g: the exponent byte of their group) as they are multiplied: value * 2^(b-127) * 2^e, e the exponent of the row's scale, which
// the conversion instruction applies.  (Powers of two beyond what it takes have long left fp16.)
template <int FM, bool GS> __device__ __forceinline__ v32h grad_weights(v6u fields, half_t scale, uint32_t g)
{
    static_assert(Fmt<FM>::post_scale == 1.0f || Fmt<FM>::post_scale == 4.0f, "a power of two");
    int field = scale_exponent(scale) + (Fmt<FM>::post_scale == 4.0f ? 2 : 0) + (GS ? (int)g : 127);
    if constexpr (GS) field = field < 0 ? 0 : field > 254 ? 254 : field;
    return fields_to_halfs<FM>(fields, __builtin_bit_cast(float, (uint32_t)field << 23));
}

__device__ __forceinline__ void wait_lds_and_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// one lane's 4 x 16-bit share of a transposing read
__device__ __forceinline__ v4hh read_transposed(const uint8_t *p)
{
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    return __builtin_bit_cast(v4hh, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(p)));
}

template <int FM, bool GS, bool PRE, int NT, int WN>
__global__ __launch_bounds__(2 * WN *kWave, NT >= 6 ? 1 : 2) void grad_tile(const uint8_t *W, const half_t *scales, const uint8_t *gexp, const half_t *dY, half_t *__restrict__ dX,
                                                           float *__restrict__ ws, uint32_t M, uint32_t N, uint32_t K, uint32_t units, uint32_t splits,
                                                           uint32_t nblocks)
{
    typedef GradTile<NT, WN> T;
    constexpr int TN = T::TN, RT = 8, WAVES = 2 * WN, NTHREADS = WAVES * kWave;
    constexpr int OCC = kGradRows, kPieces = OCC / 8;                    // 16-byte pieces of a batch row of a stage
    constexpr int kRowsPer = 64 / kPieces;              // batch rows of one load
    constexpr int kX = TN / kRowsPer / WAVES, kUnits = OCC / 16 * 2 / WAVES; // loads of dY, and half blocks to convert, of a wavefront
    static_assert(kX * WAVES * kRowsPer == TN && kUnits * WAVES == OCC / 8, "every wavefront does the same share");
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

    // What is fetched for a chunk, from pointers that go from chunk to chunk and stay at the last one: past the end it is fetched, converted and stored once more, and not used.
    // Half blocks: number u = wave + WAVES * i of a chunk is half wi = u & 1 of row tile u >> 1.
    const uint32_t wstep = units * Fmt<FM>::block_bytes, lane16 = lane * 16, lane8 = lane * 8, col2 = col * 2;
    const uint8_t *wp = W + (size_t)(c0 * (OCC / 16) + (wave >> 1)) * wstep + (size_t)kb * Fmt<FM>::block_bytes;
    const uint8_t *gp = GS ? gexp + ((size_t)(c0 * (OCC / 16) + (wave >> 1)) * units + kb) * 32 : nullptr;
    const uint8_t *sp = reinterpret_cast<const uint8_t *>(scales) + ((size_t)c0 * OCC + (wave >> 1) * 16) * 2;
    uint32_t       wleft = c1 - c0;
    auto           load_codes = [&](auto half_c, RawHalf &f, half_t &sc, int i) __attribute__((always_inline)) {
        constexpr int  H = decltype(half_c)::value, kPiece = Fmt<FM>::bits == 6 ? 2048 : 1024; // pieces as in load_raw_half
        const uint8_t *block = wp + (size_t)(WAVES / 2 * i) * wstep;
        f.p = *reinterpret_cast<const v4u *>(block + H * kPiece + lane16);
        if constexpr (Fmt<FM>::bits == 6) f.s = *reinterpret_cast<const v2u *>(block + 1024 + 8 * H + lane16);
        if constexpr (Fmt<FM>::bits == 5) f.s[0] = *reinterpret_cast<const uint32_t *>(block + 2048 + 4 * H + lane8);
        if constexpr (GS) f.g = gp[(size_t)(WAVES / 2 * i) * units * 32 + H + col2];
        sc = *reinterpret_cast<const half_t *>(sp + WAVES / 2 * i * 32 + col2);
    };
    auto next_codes = [&]() __attribute__((always_inline)) {
        const bool more = --wleft > 0 && wleft < 0x80000000u;
        wp += more ? (size_t)(OCC / 16) * wstep : 0;
        if constexpr (GS) gp += more ? (size_t)(OCC / 16) * units * 32 : 0;
        sp += more ? OCC * 2 : 0;
    };
    v32h           converted;
    uint8_t *const wdst = lds + ((col >> 2) & 1) * kGradHalf + (4 * (col >> 3) + (col & 3)) * kGradRow + wi * 256 + q * 16; // row o = 16 * (rt & 1) + col of 32 is the (4 (o / 8) + o % 4)-th of its half
    auto           write_w = [&](int i, int s, int stage) __attribute__((always_inline)) {
        const int rt = (wave + WAVES * i) >> 1;
        *reinterpret_cast<v8h *>(wdst + stage * T::kStage + (rt >> 1) * kGrad32 + (rt & 1) * 8 * kGradRow + 64 * s) = slice8(converted, s);
    };

    // batch rows: load j of this wavefront is of rows kRowsPer * (wave + WAVES * j) ..; rows beyond N repeat the last one (never stored)
    auto           swizzle = [](uint32_t n) { return n & 7; };
    const uint32_t xrow = lane / kPieces, xpiece = ((lane % kPieces) ^ swizzle(xrow)) * 16, nlast = N - nbase < (uint32_t)TN ? N - 1 - nbase : TN - 1;
    uint32_t       xoff[kX]; // 32 bits: the launcher bounds M
#pragma unroll
    for (int j = 0; j < kX; j++) {
        const uint32_t n = kRowsPer * (wave + WAVES * j) + xrow;
        xoff[j] = (n < nlast ? n : nlast) * M * 2 + xpiece;
    }
    const uint8_t *xp = reinterpret_cast<const uint8_t *>(dY + (size_t)nbase * M + (size_t)c0 * OCC), *ep = reinterpret_cast<const uint8_t *>(scales + (size_t)c0 * OCC);
    uint32_t       xleft = c1 - c0;
    v4u            xr[kX], xs; // xs: the scales of this lane's eight rows of a chunk
    const bool     scales_aligned = (reinterpret_cast<uintptr_t>(scales) & 15u) == 0;
    auto           load_x = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kX; j++) xr[j] = *reinterpret_cast<const v4u *>(xp + xoff[j]);
        if constexpr (!PRE) {
            if (scales_aligned) {
                xs = *reinterpret_cast<const v4u *>(ep + xpiece);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) xs[i] = *reinterpret_cast<const uint16_t *>(ep + xpiece + 4 * i) | (uint32_t)*reinterpret_cast<const uint16_t *>(ep + xpiece + 4 * i + 2) << 16;
            }
        }
        const bool more = --xleft > 0 && xleft < 0x80000000u;
        xp += more ? OCC * 2 : 0, ep += more ? OCC * 2 : 0;
    };
    auto store_x = [&](int stage) __attribute__((always_inline)) {
        if constexpr (!PRE)
            scale_mantissas(xs);
#pragma unroll
        for (int j = 0; j < kX; j++) {
            if constexpr (!PRE) xr[j] = __builtin_bit_cast(v4u, __builtin_bit_cast(v8h, xr[j]) * __builtin_bit_cast(v8h, xs));
            *reinterpret_cast<v4u *>(lds + stage * T::kStage + T::kWStage + (wave + WAVES * j) * 1024 + lane16) = xr[j];
        }
    };

    // Operands of one MFMA step (32 rows).  A step is RT groups of NT MFMAs; behind a group's MFMAs its weights are replaced by the next step's, and the first half of the groups read
    // the next step's batch rows into the other set.
    v8h            a[RT], b[2][NT];
    const uint8_t *wread = lds + (4 * q + (col >> 2)) * kGradRow + (col & 3) * 8 + wi * 256;
    auto           read_a = [&](int r, int stage, int kk) __attribute__((always_inline)) {
        const uint8_t *p = wread + stage * T::kStage + kk * kGrad32 + r * 32;
        a[r] = __builtin_shufflevector(read_transposed(p), read_transposed(p + kGradHalf), 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto read_b = [&](auto set_c, int t, int stage, int kk) __attribute__((always_inline)) {
        const int n = (wn * NT + t) * 16 + col;
        b[decltype(set_c)::value][t] = *reinterpret_cast<const v8h *>(lds + stage * T::kStage + T::kWStage + n * (OCC * 2) + (((4 * kk + q) ^ swizzle(col)) * 16));
    };
    auto run = [&](auto half_c) __attribute__((always_inline)) {
        typedef std::integral_constant<int, 0> Zero;
        typedef std::integral_constant<int, 1> One;
        constexpr int H = decltype(half_c)::value;
        // a chunk is converted and stored in its predecessor's first step; the next one's batch rows and codes are asked for right behind
        RawHalf raw[kUnits];
        half_t  rsc[kUnits];
#pragma unroll
        for (int i = 0; i < kUnits; i++) load_codes(half_c, raw[i], rsc[i], i);
        next_codes();
        load_x();
#pragma unroll
        for (int i = 0; i < kUnits; i++) {
            converted = grad_weights<FM, GS>(raw_half_fields<FM, H>(raw[i]), rsc[i], raw[i].g);
#pragma unroll
            for (int j = 0; j < 4; j++) write_w(i, j, 0);
        }
        store_x(0);
#pragma unroll
        for (int i = 0; i < kUnits; i++) load_codes(half_c, raw[i], rsc[i], i);
        next_codes();
        load_x();
        wait_lds_and_barrier();
#pragma unroll
        for (int t = 0; t < NT; t++) read_b(Zero{}, t, 0, 0);
#pragma unroll
        for (int r = 0; r < RT; r++) read_a(r, 0, 0);
        // A chunk, two steps, lies in stage `st`.  Its second step begins with the chunk's barrier: what it multiplies is in registers by then, so stage `st` is free for the next chunk but
        // one, and the next chunk is there, whose first step is read now.
        auto chunk = [&](auto st_c) __attribute__((always_inline)) {
            constexpr int st = decltype(st_c)::value;
            sections<2>([&](auto kk_c) __attribute__((always_inline)) {
                constexpr int  kk = decltype(kk_c)::value;
                constexpr bool last = kk == 1;
                typedef std::integral_constant<int, kk ^ 1> Next;
                if constexpr (last) wait_lds_and_barrier();
                __builtin_amdgcn_sched_barrier(0);
                sections<RT>([&](auto r_c) __attribute__((always_inline)) {
                    constexpr int r = decltype(r_c)::value, rs = last ? st ^ 1 : st, rk = last ? 0 : kk + 1, kHalfRT = RT / 2;
                    if constexpr (r < kHalfRT) {
#pragma unroll
                        for (int t = r * NT / kHalfRT; t < (r + 1) * NT / kHalfRT; t++) read_b(Next{}, t, rs, rk);
                    }
                    if constexpr (kk == 0) { // half blocks to convert: each takes RT / kUnits groups, one for the conversion and two for its writes
                        constexpr int per = RT / kUnits, i = r / per, g = r % per, dst = st ^ 1;
                        static_assert(per >= 4, "a conversion, its writes and the next loads need four groups");
                        if constexpr (g == 0) converted = grad_weights<FM, GS>(raw_half_fields<FM, H>(raw[i]), rsc[i], raw[i].g);
                        if constexpr (g == 1) {
#pragma unroll
                            for (int s = 0; s < 2; s++) write_w(i, s, dst);
                        }
                        if constexpr (g == 2) {
#pragma unroll
                            for (int s = 2; s < 4; s++) write_w(i, s, dst);
                        }
                        if constexpr (g == 3) load_codes(half_c, raw[i], rsc[i], i);
                        if constexpr (r == RT - 2) store_x(dst);
                        if constexpr (r == RT - 1) next_codes(), load_x();
                    }
#pragma unroll
                    for (int t = 0; t < NT; t++) acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[r], b[kk][t], acc[r][t], 0, 0, 0);
                    read_a(r, rs, rk);
#pragma unroll
                    for (int t = 0; t < NT; t++) { // one other instruction behind every MFMA, as far as they go (8192x8192 N 4096 in 256 x 256 tiles: 466 -> 448 us)
                        __builtin_amdgcn_sched_group_barrier(0x08, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0xA6, 1, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
            });
        };
        for (uint32_t c = c0; c < c1; c += 2) {
            chunk(Zero{});
            if (c + 1 < c1) chunk(One{});
        }
    };
    if (c0 < c1) { // (more splits than chunks leave some empty: their partial sums are zeros)
        if (wi == 0)
            run(std::integral_constant<int, 0>{});
        else
            run(std::integral_constant<int, 1>{});
    }
    __syncthreads(); // nobody reads operands any more

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

// ---------------------------------------------------------------------------------------------------------------
// grad_stream: the same product for up to 32 batch rows, where the weights' way from memory is the bound.
//   grid = (blocks of 256 input features, splits)   block = WO wavefronts, which share the weight rows of a split among them, 32 rows (two native blocks) at a time in turn, half of
//   the columns each
// Every wavefront is by itself until the end: it converts its halves of two native blocks into an LDS area of its own (rows 288 bytes apart, in grad_tile's
// order; no barrier, the LDS unit serves a wavefront in order), reads them back transposed, and takes its batch rows from memory in operand order.  The codes of the next
// 32 rows are asked for before this one's are converted.  Sums meet in LDS.  us a call in a captured graph, the reduction of the splits among it, over weights that no cache holds (several
// matrices in turn, 300 to 600 MB), e3m2, N 8 / 32: 4096x4096 10.3 / 15.5 (16 splits), 8192x8192 15.8 / 21.4 (8), 28672x8192 36.7 / 46.8 (8, 4.8 TB/s); with whole blocks a wavefront, twice the sums to
// meet, and at N 32 four wavefronts everywhere, 10.8 / 17.3, 17.1 / 26.0, 34.9 / 55.3.  (4096x4096 N 8 over three matrices, which the memory-side cache holds: 9.6.  Half blocks of different workgroups 13.3 and 35.6 at N 8, 1:
// the codes that the halves share were fetched by two XCDs.)
// ---------------------------------------------------------------------------------------------------------------
constexpr int kStreamRow = 288, kStreamHalf = 16 * kStreamRow + 16, kStreamMant = 2 * kStreamHalf, kStreamWave = kStreamMant + 64;
template <int NT, int WO> constexpr int grad_stream_lds() { return WO * (NT * 8192 > kStreamWave ? NT * 8192 : kStreamWave); }

template <int FM, bool GS, bool PRE, int NT, int WO>
__global__ __launch_bounds__(WO *kWave) void grad_stream(const uint8_t *__restrict__ W, const half_t *__restrict__ scales, const uint8_t *__restrict__ gexp, const half_t *__restrict__ dY,
                                                         half_t *__restrict__ dX, float *__restrict__ ws, uint32_t M, uint32_t N, uint32_t K, uint32_t units, uint32_t splits)
{
    constexpr int RT = 8, WR = WO / 2, kWaveLds = grad_stream_lds<NT, WO>() / WO;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int      tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, q = lane >> 4, wi = wave & 1, wr = wave >> 1;
    const uint32_t kb = blockIdx.x, split = blockIdx.y, chunks = M / 32;
    const uint32_t avg = chunks / splits, extra = chunks % splits, c0 = split * avg + (split < extra ? split : extra), c1 = c0 + avg + (split < extra ? 1u : 0u);
    uint8_t       *mine = lds + wave * kWaveLds;

    v4f acc[RT][NT];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[r][t] = (v4f){ 0.f, 0.f, 0.f, 0.f };

    // (reads of other lanes' writes: the LDS unit serves a wavefront in order, the compiler has to leave them in this one)
    auto in_order = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    uint8_t *const       wdst = mine + (col >> 2 & 1) * kStreamHalf + (4 * (col >> 3) + (col & 3)) * kStreamRow + q * 16;
    const uint8_t *const wread = mine + (4 * q + (col >> 2)) * kStreamRow + (col & 3) * 8;
    auto run = [&](auto half_c) __attribute__((always_inline)) {
        constexpr int H = decltype(half_c)::value;
        // what is fetched for 32 rows: codes, exponent and scale of two native blocks, and the batch rows
        auto load_codes = [&](RawHalf &w, half_t &sc, uint32_t tile) __attribute__((always_inline)) {
            const size_t blk = (size_t)tile * units + kb;
            load_raw_half<FM, GS, H>(w, W + blk * Fmt<FM>::block_bytes, GS ? gexp + blk * 32 : nullptr, lane);
            sc = scales[tile * 16 + col];
        };
        auto load_rows = [&](v8h(&b)[NT], uint32_t c) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < NT; t++) { // (rows beyond N repeat the last one and are not stored)
                const uint32_t n = 16 * t + col < N ? 16 * t + col : N - 1;
                b[t] = *reinterpret_cast<const v8h *>(dY + (size_t)n * M + c * 32 + 8 * q);
            }
        };
        auto convert_rows = [&](const RawHalf &w, half_t sc, int i) __attribute__((always_inline)) { // row 16 i + col of 32: the (4 (2 i + col / 8) + col % 4)-th of its half
            const v32h v = grad_weights<FM, GS>(raw_half_fields<FM, H>(w), sc, w.g);
#pragma unroll
            for (int s = 0; s < 4; s++) *reinterpret_cast<v8h *>(wdst + i * 8 * kStreamRow + 64 * s) = slice8(v, s);
            if (!PRE && q == 0) *reinterpret_cast<half_t *>(mine + kStreamMant + (16 * i + col) * 2) = scale_mantissa(sc);
        };
        auto multiply = [&](v8h(&b)[NT]) __attribute__((always_inline)) {
            in_order();
            if constexpr (!PRE) {
                const v8h mant = *reinterpret_cast<const v8h *>(mine + kStreamMant + 16 * q);
#pragma unroll
                for (int t = 0; t < NT; t++) b[t] = b[t] * mant;
            }
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const v8h a = __builtin_shufflevector(read_transposed(wread + r * 32), read_transposed(wread + kStreamHalf + r * 32), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int t = 0; t < NT; t++) acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b[t], acc[r][t], 0, 0, 0);
            }
            in_order();
        };
        RawHalf  w00, w01, w10, w11; // (arrays or one struct of them go to scratch memory)
        half_t   s00, s01, s10, s11;
        v8h      b0[NT], b1[NT];
        uint32_t c = c0 + wr;
        if (c < c1) load_codes(w00, s00, 2 * c), load_codes(w01, s01, 2 * c + 1), load_rows(b0, c);
        while (c < c1) {
            if (c + WR < c1) load_codes(w10, s10, 2 * (c + WR)), load_codes(w11, s11, 2 * (c + WR) + 1), load_rows(b1, c + WR);
            convert_rows(w00, s00, 0), convert_rows(w01, s01, 1), multiply(b0);
            c += WR;
            if (c >= c1) break;
            if (c + WR < c1) load_codes(w00, s00, 2 * (c + WR)), load_codes(w01, s01, 2 * (c + WR) + 1), load_rows(b0, c + WR);
            convert_rows(w10, s10, 0), convert_rows(w11, s11, 1), multiply(b1);
            c += WR;
        }
    };
    if (wi == 0)
        run(std::integral_constant<int, 0>{});
    else
        run(std::integral_constant<int, 1>{});

    // every wavefront parks its sums in its own area, [r][t][lane] of four input features
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < NT; t++) *reinterpret_cast<v4f *>(mine + (r * NT + t) * 1024 + lane * 16) = acc[r][t];
    __syncthreads();
    for (uint32_t p = tid; p < N * 64; p += WO * kWave) { // input features 4 f .. of half h, batch row n
        const uint32_t f = p & 31, h = p >> 5 & 1, n = p >> 6, k = kb * 256 + h * 128 + 4 * f;
        const uint8_t *src = lds + h * kWaveLds + ((f >> 2) * NT + (n >> 4)) * 1024 + ((f & 3) * 16 + (n & 15)) * 16;
        v4f            sum = *reinterpret_cast<const v4f *>(src);
#pragma unroll
        for (int w = 1; w < WR; w++) sum += *reinterpret_cast<const v4f *>(src + 2 * w * kWaveLds);
        if (k < K) {
            if (splits == 1)
                *reinterpret_cast<v4hh *>(dX + (size_t)n * K + k) = (v4hh){ (half_t)sum[0], (half_t)sum[1], (half_t)sum[2], (half_t)sum[3] };
            else
                *reinterpret_cast<v4f *>(ws + ((size_t)split * N + n) * K + k) = sum;
        }
    }
}

template <int FM, bool GS, bool PRE, int NT, int WO>
int launch_grad_stream(hipStream_t st, const void *W, const void *sc, const void *gexp, const void *dY, void *dX, float *ws, size_t M, size_t N, size_t K, int splits)
{
    constexpr int kLds = grad_stream_lds<NT, WO>();
    static_assert(kLds <= 160 * 1024, "the wavefronts' areas do not fit in LDS");
    const uint32_t units = (uint32_t)((K + 255) / 256);
    if (kLds > 48 * 1024)
        if (int rc = allow_dynamic_lds<&grad_stream<FM, GS, PRE, NT, WO>>(kLds)) return rc;
    hipLaunchKernelGGL((grad_stream<FM, GS, PRE, NT, WO>), dim3(units, (uint32_t)splits), dim3(WO * kWave), kLds, st, static_cast<const uint8_t *>(W), static_cast<const half_t *>(sc),
                       static_cast<const uint8_t *>(gexp), static_cast<const half_t *>(dY), static_cast<half_t *>(dX), ws, (uint32_t)M, (uint32_t)N, (uint32_t)K, units, (uint32_t)splits);
    return (int)hipGetLastError();
}

template <int FM, bool GS, bool PRE, int NT, int WN>
int launch_grad(hipStream_t st, const void *W, const void *sc, const void *gexp, const void *dY, void *dX, float *ws, size_t M, size_t N, size_t K, int splits)
{
    typedef GradTile<NT, WN> T;
    static_assert(T::kLds <= 160 * 1024, "tile does not fit in LDS");
    const uint32_t units = (uint32_t)((K + 255) / 256), nblocks = (uint32_t)((N + T::TN - 1) / T::TN);
    const size_t   wgs = (size_t)units * (size_t)splits * nblocks;
    if (wgs > 0x7fffffffu || M > (size_t)1 << 20) return FP6MI_ERR_SHAPE; // (M: 32-bit offsets over TN batch rows)
    if (T::kLds > 48 * 1024)
        if (int rc = allow_dynamic_lds<&grad_tile<FM, GS, PRE, NT, WN>>(T::kLds)) return rc;
    hipLaunchKernelGGL((grad_tile<FM, GS, PRE, NT, WN>), dim3((uint32_t)wgs), dim3(2 * WN * kWave), T::kLds, st, static_cast<const uint8_t *>(W),
                       static_cast<const half_t *>(sc), static_cast<const uint8_t *>(gexp), static_cast<const half_t *>(dY), static_cast<half_t *>(dX), ws,
                       (uint32_t)M, (uint32_t)N, (uint32_t)K, units, (uint32_t)splits, nblocks);
    return (int)hipGetLastError();
}

// rows: the batch rows of a workgroup, which say which kernel (fp6mi::grad_rows)
template <int FM, bool GS, bool PRE>
int grad_cfg(int rows, hipStream_t st, const void *W, const void *sc, const void *gexp, const void *dY, void *dX, float *ws, size_t M, size_t N, size_t K, int splits)
{
    switch (rows) {
    case 16: return launch_grad_stream<FM, GS, PRE, 1, 8>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits);
    case 32: // (us at N 24, four / eight wavefronts: 8 of these 32 rows a split 14.3 / 15.4 and 13.2 / 13.3, 10 of them 16.1 / 16.1, 32 of them 25.2 / 20.1, 43 31.0 / 23.0, 112 64 / 45)
        return M / 32 / splits >= 16 ? launch_grad_stream<FM, GS, PRE, 2, 8>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits)
                                     : launch_grad_stream<FM, GS, PRE, 2, 4>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits);
    case 128: return launch_grad<FM, GS, PRE, 2, 4>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits);
    case 192: return launch_grad<FM, GS, PRE, 6, 2>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits);
    case 256: return launch_grad<FM, GS, PRE, 8, 2>(st, W, sc, gexp, dY, dX, ws, M, N, K, splits);
    default: return FP6MI_ERR_SHAPE;
    }
}

// ---------------------------------------------------------------------------------------------------------------
// The gated feed-forward block: the GEMM's kernels (fp6mi_gemm.hip: gemm_stream, gemm_tile, gemm_ws, gemm_wide and gemm_span) with another epilogue.
// The weights are one matrix of M rows in pair order: a 16-row tile of the gate projection, the same tile of the up projection, and so on.  An even number of row tiles to a
// workgroup then holds both pre-activations of every output, and no launch, no trip through memory follows: 2 * N * M bytes written and read less.
// The float32 sums are scaled and parked in LDS as the partial sums of a split are; on the way out a thread takes four rows of gate and the same four of up, adds the biases and
// writes act(g) * u, and the pre-activations themselves where a backward pass will want them.
// Parameters as in the GEMM's kernels; preact and bias may be null.
// ---------------------------------------------------------------------------------------------------------------
template <int NT, int RT, int WR, int NTHREADS>
__device__ __forceinline__ void gated_flush(half_t *__restrict__ out, float *__restrict__ preact, const half_t *__restrict__ bias, uint32_t activation_code, const uint8_t *stage, uint32_t M,
                                            uint32_t N, uint32_t mb, uint32_t nbase, int tid)
{
    constexpr int TM = WR * RT * 16, TN = NT * 16, kStride = TM * 4 + 16, kPerCol = TM / 8, kPieces = TN * kPerCol; // a piece: four outputs
    static_assert(TM % 32 == 0, "pairs of row tiles");
    for (int p = tid; p < kPieces; p += NTHREADS) {
        const int      c = p / kPerCol, i = p % kPerCol;
        const uint32_t ng = nbase + c, m = mb * TM + (i >> 2) * 32 + (i & 3) * 4;
        if (ng < N) {
            const uint8_t *src = stage + c * kStride + ((i >> 2) * 32 + (i & 3) * 4) * 4;
            v4f            g = *reinterpret_cast<const v4f *>(src), u = *reinterpret_cast<const v4f *>(src + 64);
            v4h            h;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (bias) g[k] += (float)bias[m + k], u[k] += (float)bias[m + 16 + k];
                h[k] = (half_t)(activated(activation_code, g[k]) * u[k]);
            }
            *reinterpret_cast<v4h *>(out + (size_t)ng * (M / 2) + (size_t)mb * (TM / 2) + i * 4) = h;
            if (preact) {
                *reinterpret_cast<v4f *>(preact + (size_t)ng * M + m) = g;
                *reinterpret_cast<v4f *>(preact + (size_t)ng * M + m + 16) = u;
            }
        }
    }
}

#define FP6MI_GATED 1
template <int FM, bool GS, int NT, int RT, int WAVES>
__global__ __launch_bounds__(WAVES *kWave) void gated_stream(const uint8_t *__restrict__ W, const half_t *__restrict__ scales, const uint8_t *__restrict__ gexp, const half_t *__restrict__ X,
                                                             half_t *__restrict__ C, float *__restrict__ preact, const half_t *__restrict__ bias, uint32_t M, uint32_t N, uint32_t K,
                                                             uint32_t units, uint32_t activation_code)
{
    static_assert(RT % 2 == 0, "pairs of row tiles");
    constexpr bool     SPLIT = false;
    constexpr uint32_t splitK = 1;
    float *const       ws = preact;
#include "fp6mi_stream_tile.inc"
}

template <int FM, bool GS, int NT, int RT, int WR, int WK>
__global__ __launch_bounds__(WR *WK *kWave) void gated_tile(const uint8_t *__restrict__ W, const half_t *__restrict__ scales, const uint8_t *__restrict__ gexp, const half_t *__restrict__ X,
                                                            half_t *__restrict__ C, float *__restrict__ preact, const half_t *__restrict__ bias, uint32_t M, uint32_t N, uint32_t K,
                                                            uint32_t units, uint32_t activation_code, uint32_t nblocks)
{
    constexpr int NTHREADS = WR * WK * kWave;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int      tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave % WR, wk = wave / WR, col = lane & 15, q = lane >> 4;
    const TileId   id = tile_of<WR * RT * 16, NT * 16>(1, nblocks, N, K);
    const uint32_t nbase = id.nb * NT * 16, R0 = (id.mb * WR + wr) * RT;
    v4f            acc[RT][NT];
    v4h            sc4[RT]; // fetched ahead of the K loop, as in gemm_tile
#pragma unroll
    for (int r = 0; r < RT; r++) {
        const half_t *p = scales + (R0 + r) * 16 + 4 * q;
        sc4[r] = (v4h){ p[0], p[1], p[2], p[3] };
    }
    tile_segment<FM, GS, NT, RT, WR, WK>(acc, W, gexp, X, N, K, units, id.mb, nbase, 0, units, lds, tid, lane, wr, wk, col, q);
    if (WK > 1) __syncthreads(); // (the sums are parked where the partial sums of the K wavefronts met)
    if (wk == 0) tile_park<FM, NT, RT, WR, float>(acc, sc4, lds, wr, col, q);
    __syncthreads();
    gated_flush<NT, RT, WR, NTHREADS>(C, preact, bias, activation_code, lds, M, N, id.mb, nbase, tid);
}

template <int FM, bool GS, int NT, int RT, int WR, int PW, int SW, int SX>
__global__ __launch_bounds__((WR + PW) * kWave) void gated_ws(const uint8_t *__restrict__ W, const half_t *__restrict__ scales, const uint8_t *__restrict__ gexp, const half_t *__restrict__ X,
                                                              half_t *__restrict__ C, float *__restrict__ preact, const half_t *__restrict__ bias, uint32_t M, uint32_t N, uint32_t K,
                                                              uint32_t units, uint32_t activation_code, uint32_t nblocks)
{
    constexpr uint32_t splitK = 1;
    float *const       ws = preact;
#include "fp6mi_ws_tile.inc"
}

template <int FM, bool GS, int NT, int RT, int WK>
__global__ __launch_bounds__(4 * WK *kWave, RT *NT <= 8 ? 4 : 2) void gated_wide(const uint8_t *W, const half_t *__restrict__ scales, const uint8_t *gexp, const half_t *X,
                                                                                 half_t *__restrict__ C, float *__restrict__ preact, const half_t *__restrict__ bias, uint32_t M, uint32_t N,
                                                                                 uint32_t K, uint32_t units, uint32_t activation_code, uint32_t nblocks)
{
    constexpr uint32_t splitK = 1;
#include "fp6mi_wide_tile.inc"
}
#undef FP6MI_GATED

struct GatedArgs {
    hipStream_t st;
    const void *W, *sc, *gexp, *B;
    void       *C;
    float      *preact;
    const void *bias;
    size_t      M, N, K;
    int         activation;
};

template <int FM, bool GS, int NT, int RT, int WAVES> int launch_gated_stream(const GatedArgs &a)
{
    constexpr size_t kMaxLds = (size_t)WAVES * stream_wave_bytes(16 * NT, RT, NT);
    static_assert(kMaxLds <= 160 * 1024, "the wavefronts' activation rows do not fit in LDS");
    const uint32_t units = (uint32_t)((a.K + 255) / 256);
    const dim3     grid((uint32_t)((a.M / 16 + RT - 1) / RT), 1, (uint32_t)((a.N + 16 * NT - 1) / (16 * NT)));
    const size_t   lds_bytes = NT == 1 && a.N <= 8 ? (size_t)WAVES * stream_wave_bytes(8, RT, NT) : kMaxLds;
    if (kMaxLds > 48 * 1024)
        if (int rc = allow_dynamic_lds<&gated_stream<FM, GS, NT, RT, WAVES>>(kMaxLds)) return rc;
    hipLaunchKernelGGL((gated_stream<FM, GS, NT, RT, WAVES>), grid, dim3(WAVES * kWave), lds_bytes, a.st, static_cast<const uint8_t *>(a.W), static_cast<const half_t *>(a.sc),
                       static_cast<const uint8_t *>(a.gexp), static_cast<const half_t *>(a.B), static_cast<half_t *>(a.C), a.preact, static_cast<const half_t *>(a.bias), (uint32_t)a.M,
                       (uint32_t)a.N, (uint32_t)a.K, units, (uint32_t)a.activation);
    return (int)hipGetLastError();
}
// the kernels of tiles: TM x TN outputs of the GEMM a workgroup of THREADS
template <auto Kernel, int TM, int TN, int THREADS> int launch_gated_tiles(const GatedArgs &a, size_t lds_bytes)
{
    if (a.M % TM) return FP6MI_ERR_SHAPE;
    if (lds_bytes > 48 * 1024)
        if (int rc = allow_dynamic_lds<Kernel>(lds_bytes)) return rc;
    const uint32_t units = (uint32_t)((a.K + 255) / 256), nblocks = (uint32_t)((a.N + TN - 1) / TN);
    const size_t   wgs = a.M / TM * nblocks;
    if (wgs > 0x7fffffffu) return FP6MI_ERR_SHAPE;
    hipLaunchKernelGGL(Kernel, dim3((uint32_t)wgs), dim3(THREADS), lds_bytes, a.st, static_cast<const uint8_t *>(a.W), static_cast<const half_t *>(a.sc), static_cast<const uint8_t *>(a.gexp),
                       static_cast<const half_t *>(a.B), static_cast<half_t *>(a.C), a.preact, static_cast<const half_t *>(a.bias), (uint32_t)a.M, (uint32_t)a.N, (uint32_t)a.K, units,
                       (uint32_t)a.activation, nblocks);
    return (int)hipGetLastError();
}
constexpr size_t most_of(size_t a, size_t b) { return a > b ? a : b; }
template <int FM, bool GS, int NT, int RT, int WR, int WK> int launch_gated_tile(const GatedArgs &a)
{
    constexpr size_t kLoop = most_of(2 * (size_t)WK * NT * 16 * kXsRowBytes, WK > 1 ? (size_t)WK * WR * RT * NT * 1024 : 0), kLds = most_of(kLoop, tile_stage_bytes<NT, RT, WR>(true));
    static_assert(kLds <= 160 * 1024, "tile does not fit in LDS");
    return launch_gated_tiles<&gated_tile<FM, GS, NT, RT, WR, WK>, WR * RT * 16, NT * 16, WR * WK * kWave>(a, kLds);
}
template <int FM, bool GS, int NT, int RT, int WR, int PW, int SW, int SX> int launch_gated_ws(const GatedArgs &a)
{
    constexpr size_t kLds = most_of(ws_ring_bytes<FM, NT, RT, WR, SW, SX>() + ws_exps_ring_bytes<GS, RT, WR, SW>(), tile_stage_bytes<NT, RT, WR>(true));
    static_assert(kLds <= 160 * 1024, "the rings do not fit in LDS");
    return launch_gated_tiles<&gated_ws<FM, GS, NT, RT, WR, PW, SW, SX>, WR * RT * 16, NT * 16, (WR + PW) * kWave>(a, kLds);
}
template <int FM, bool GS, int NT, int RT, int WK> int launch_gated_wide(const GatedArgs &a)
{
    constexpr size_t kSums = WK == 2 ? (size_t)4 * RT * 16 * ((NT + 1) / 2) * 128 : 0, kLds = most_of(most_of(WK * 2 * (size_t)NT * 16 * 256, tile_stage_bytes<(NT + 1) / 2, RT, 4>(true)), kSums);
    static_assert(kLds <= 160 * 1024 / (3 - WK), "two workgroups of four wavefronts or one of eight do not fit in LDS");
    if (a.K > (size_t)1 << 20) return FP6MI_ERR_SHAPE; // (32-bit offsets over TN rows)
    return launch_gated_tiles<&gated_wide<FM, GS, NT, RT, WK>, 4 * RT * 16, NT * 16, 4 * WK * kWave>(a, kLds);
}

template <int FM, bool GS> int gated_cfg(const LaunchCfg &c, const GatedArgs &a)
{
#define FP6MI_CASE(NT, RT, WV) \
    if (c.kind == 0 && c.nt == NT && c.rt == RT && c.wk == WV) return launch_gated_stream<FM, GS, NT, RT, WV>(a);
    FP6MI_CASE(1, 2, 4) FP6MI_CASE(1, 2, 8) FP6MI_CASE(1, 2, 16) FP6MI_CASE(1, 4, 4) FP6MI_CASE(1, 4, 8) FP6MI_CASE(1, 6, 4) FP6MI_CASE(1, 6, 8) FP6MI_CASE(1, 8, 4)
    FP6MI_CASE(2, 2, 4) FP6MI_CASE(2, 4, 4) FP6MI_CASE(2, 4, 8) FP6MI_CASE(2, 6, 4) FP6MI_CASE(2, 8, 4)
#undef FP6MI_CASE
#define FP6MI_CASE(NT, WR, WK) \
    if (c.kind == 1 && c.nt == NT && c.wr == WR && c.wk == WK) return launch_gated_tile<FM, GS, NT, 2, WR, WK>(a);
    FP6MI_CASE(2, 4, 1) FP6MI_CASE(2, 4, 2) FP6MI_CASE(2, 4, 4) FP6MI_CASE(3, 8, 1) FP6MI_CASE(4, 4, 2) FP6MI_CASE(4, 8, 1) FP6MI_CASE(5, 8, 1) FP6MI_CASE(6, 8, 1)
#undef FP6MI_CASE
    if (c.kind == 2 && c.wk == 4) { // (ring depths as in gemm_ws)
#define FP6MI_CASE(NT, WR) \
    if (c.nt == NT && c.wr == WR) return launch_gated_ws<FM, GS, NT, 2, WR, 4, WR == 4 && NT < 6 ? 3 : 2, WR == 4 && NT == 3 ? 3 : 2>(a);
        FP6MI_CASE(4, 8) FP6MI_CASE(3, 4) FP6MI_CASE(4, 4) FP6MI_CASE(5, 4) FP6MI_CASE(6, 4)
#undef FP6MI_CASE
    }
#define FP6MI_CASE(NT, RT, WK) \
    if (c.kind == 2 && c.wr == 4 && c.nt == NT && c.rt == RT && c.wk == WK) return launch_gated_wide<FM, GS, NT, RT, WK>(a);
    FP6MI_CASE(8, 4, 1) FP6MI_CASE(8, 4, 2) FP6MI_CASE(6, 4, 1) FP6MI_CASE(8, 2, 2) FP6MI_CASE(3, 2, 2) FP6MI_CASE(5, 2, 2) FP6MI_CASE(7, 2, 2) FP6MI_CASE(5, 4, 2) FP6MI_CASE(6, 4, 2)
    FP6MI_CASE(7, 4, 2) FP6MI_CASE(4, 2, 2) FP6MI_CASE(6, 2, 2)
#undef FP6MI_CASE
    return FP6MI_ERR_SHAPE;
}

template <int FM>
int op_gated(const LaunchCfg &c, void *stream, const void *W, const void *sc, const void *gexp, const void *bias, const void *B, void *C, float *preact, size_t M, size_t N, size_t K, int activation)
{
    const GatedArgs a = { static_cast<hipStream_t>(stream), W, sc, gexp, B, C, preact, bias, M, N, K, activation };
    return gexp ? gated_cfg<FM, true>(c, a) : gated_cfg<FM, false>(c, a);
}

template <int FM>
int op_grad(int rows, void *stream, const void *W, const void *sc, const void *gexp, const void *dY, bool premultiplied, void *dX, float *ws, size_t M, size_t N, size_t K, int splits)
{
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (premultiplied)
        return gexp ? grad_cfg<FM, true, true>(rows, st, W, sc, gexp, dY, dX, ws, M, N, K, splits) : grad_cfg<FM, false, true>(rows, st, W, sc, nullptr, dY, dX, ws, M, N, K, splits);
    return gexp ? grad_cfg<FM, true, false>(rows, st, W, sc, gexp, dY, dX, ws, M, N, K, splits) : grad_cfg<FM, false, false>(rows, st, W, sc, nullptr, dY, dX, ws, M, N, K, splits);
}

} // namespace

namespace fp6mi {
#define FP6MI_OPS_NAME_(f) block_ops_##f
#define FP6MI_OPS_NAME(f) FP6MI_OPS_NAME_(f)
const BlockOps &FP6MI_OPS_NAME(FP6MI_FORMAT)()
{
    static const BlockOps ops = { &op_gated<FP6MI_FORMAT>, &op_grad<FP6MI_FORMAT> };
    return ops;
}
} // namespace fp6mi
