// Microscaled 4-bit floating point rows: their layout, quantisation and the tcgen05 product.
//
// Values are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte, the first in the low half, a row's
// K / 2 bytes after the row before. A block of consecutive values in a row shares one 8-bit scale:
//   mx  32 values, scale 2^e (byte e + 127; 255 stands for NaN)
//   nv  16 values, an e4m3 scale, and one fp32 scale a row
// The scale bytes lie in the order in which the tensor core takes them, so that the product copies them into TMEM
// without a shuffle: tiles of 128 rows x 4 blocks (512 bytes), the tiles of a row range one after another along K, byte
// (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4 inside. Tiles are whole: the bytes of rows and blocks past the
// tensor's are there and 0.
#pragma once
#include "gemm.cuh"

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace h3 {

enum class Fp4 : int { mx = 0, nv = 1 };
enum class Elem : int { bf16 = 0, f16 = 1, f32 = 2 };

#ifdef __CUDACC__
#define H3_FP4_HD __host__ __device__
#else
#define H3_FP4_HD
#endif

H3_FP4_HD constexpr int fp4_block(Fp4 f) { return f == Fp4::mx ? 32 : 16; }
// Scale tiles along a row of K values.
H3_FP4_HD constexpr int fp4_scale_tiles(int K, Fp4 f) { return (K + 4 * fp4_block(f) - 1) / (4 * fp4_block(f)); }
// Bytes of the scales of [rows][K].
inline size_t fp4_scale_bytes(int rows, int K, Fp4 f) { return size_t((rows + 127) / 128) * fp4_scale_tiles(K, f) * 512; }

// Quantises rows of K values (K a multiple of 32; x's rows ldx elements apart, 16-byte aligned). Writes all of the
// scale bytes, padding included; row_scale [rows] for nv only.
void quant_rows_fp4(const void* x, Elem type, int64_t ldx, int rows, int K, Fp4 f, void* codes, void* scales, float* row_scale,
                    cudaStream_t s);
// The values that the codes stand for, in fp32 and rounded to the output's type (rows ldo elements apart, 16-byte aligned).
// row_scale null: 1.
void dequant_rows_fp4(const void* codes, const void* scales, const float* row_scale, int rows, int K, Fp4 f, Elem type, void* out,
                      int64_t ldo, cudaStream_t s);
// D[M][N] = A[M][K] B[N][K]^T with the epilogues of gemm_bf16; p.a_scale / p.b_scale are the row scales (null: 1).
void gemm_fp4(const void* A, const void* a_scales, const void* B, const void* b_scales, Fp4 f, const GemmParams& p, Epi epi,
              cudaStream_t s);

} // namespace h3
