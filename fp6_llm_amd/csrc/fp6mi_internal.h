// Internal declarations shared by the host code and the kernel translation unit.
#ifndef FP6MI_INTERNAL_H
#define FP6MI_INTERNAL_H

#include <cmath>
#include <cstddef>
#include <cstdint>

#include "../../include/fp6mi.h"

namespace fp6mi {

// FP6_e3m2 and FP5_e2m2 (the formats of the reference's entry points), FP6_e2m3 and FP4_e2m1 (through the same paths)
inline bool supported(int E, int Mbits) { return (E == 3 && Mbits == 2) || (E == 2 && (Mbits == 1 || Mbits == 2 || Mbits == 3)); }

// fp6mi_gemm.hip, compiled once per format: the entry functions of one weight format (stream = hipStream_t)
// kind 0: gemm_stream (wr == 1, wk = wavefronts per workgroup);  kind 1: gemm_tile (wr x wk wavefronts)
struct LaunchCfg { int kind, nt, rt, wr, wk; };
struct FormatOps {
    int bits;
    // gexp: group exponents in their native layout (one byte per row and 128 columns), or null; ws: the partial sums with a split, else an fp16 bias [M] or null
    int (*gemm)(const LaunchCfg &c, void *stream, const void *W, const void *sc, const void *gexp, const void *B, void *C, float *ws, size_t M,
                size_t N, size_t K, int splitK);
    int (*relayout)(void *stream, void *native, const void *packed_ref, size_t M, size_t K);
    int (*dequant)(void *stream, void *out_f16, const void *W, const void *sc, const void *gexp, size_t M, size_t K);
    int (*quantize)(void *stream, void *native, void *scales, void *gexp, const void *weights, int dtype, size_t M, size_t K); // gexp may be null
};
const FormatOps &format_ops_32(), &format_ops_22(), &format_ops_23(), &format_ops_21(); // named by 10*E + M
inline const FormatOps *ops_for(int E, int Mbits)
{
    return E == 3 ? &format_ops_32() : Mbits == 2 ? &format_ops_22() : Mbits == 3 ? &format_ops_23() : &format_ops_21();
}

// fp6mi_block.hip, compiled once per format: the kernels that read the same weights for another product
struct BlockOps {
    // H[N,M/2] of the gated block on weights in pair order by launch shape c (FP6MI_ERR_SHAPE where its kernels lack it); gexp, bias and preact may be null
    int (*gated)(const LaunchCfg &c, void *stream, const void *W, const void *sc, const void *gexp, const void *bias, const void *B, void *C, float *preact, size_t M, size_t N, size_t K,
                 int activation);
    // dX[N,K] = dY[N,M] . dequant(W); rows: batch rows of a workgroup, from grad_rows; gexp as above; premultiplied: dY holds its products with the mantissas of the row scales (fp6mi_scale.inc); ws: splits * N * K partial sums with
    // splits > 1, which the caller reduces
    int (*grad)(int rows, void *stream, const void *W, const void *sc, const void *gexp, const void *dY, bool premultiplied, void *dX, float *ws, size_t M, size_t N, size_t K, int splits);
};
const BlockOps &block_ops_32(), &block_ops_22(), &block_ops_23(), &block_ops_21();
inline const BlockOps *block_ops_for(int E, int Mbits)
{
    return E == 3 ? &block_ops_32() : Mbits == 2 ? &block_ops_22() : Mbits == 3 ? &block_ops_23() : &block_ops_21();
}

// fp6mi_api.hip: parts of fp6mi_linear_native for the operators around it (fp6mi_ops.hip)
int  check_linear(int E, int Mbits, const void *W, const void *sc, const void *gexp, const void *bias, const void *B, const void *C, size_t M, size_t N, size_t K, const float *ws, int splitK);
// the launch shape of fp6mi_linear_native
LaunchCfg linear_shape(int E, int Mbits, size_t M, size_t N, size_t K, int splitK, bool grouped);
// the GEMM by the shape that fp6mi_linear_native takes; partial_only: with a split, the partial sums alone, [splitK][N][M] floats in ws (C is not touched)
int  run_linear(int E, int Mbits, void *stream, const void *W, const void *sc, const void *gexp, const void *bias, const void *B, void *C, size_t M, size_t N, size_t K, float *ws, int splitK,
                bool partial_only);
// C[N,M] = fp16_rn(sum over splits of ws[s])
int  reduce_partials(void *stream, void *C, const float *ws, size_t M, size_t N, int splits);

// fp6mi_host.cpp
int    prepack_ref(int E, int Mb, void *packed, const void *raw, size_t M, size_t K);
int    unpack_ref(int E, int Mb, void *raw, const void *packed, size_t M, size_t K);
int    dequant(int E, int Mb, void *out_f16, const void *raw, size_t M, size_t K, const void *scales_f16);
size_t native_block_bytes(int x);
size_t native_bytes(int E, int Mb, size_t M, size_t K);
int    prepack_native(int E, int Mb, void *native, const void *raw, size_t M, size_t K);
int    unpack_native(int E, int Mb, void *raw, const void *native, size_t M, size_t K);
int    relayout_ref_to_native(int E, int Mb, void *native, const void *packed_ref, size_t M, size_t K);
size_t group_exps_bytes(size_t M, size_t K);
int    pack_group_exps(void *native_exps, const void *exps, size_t M, size_t K);
int    dequant_grouped(int E, int Mb, void *out_f16, const void *raw, size_t M, size_t K, const void *scales_f16, const void *exps);

} // namespace fp6mi
#endif
