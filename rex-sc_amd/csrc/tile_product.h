// The product of two row-major operands on the matrix instructions, int8 -> int32 or binary16 -> float32, and its
// epilogue.  Operand rows are handled as bytes: 16 bytes are one lane's share of an instruction's operand in either type.
#pragma once
#include "lowp.h"

namespace rexsc {

struct TileArgs {
    const char *a, *b;              // y[m][n] = sum_piece sum_k a[piece][m][k] b[n][k]
    size_t a_stride, b_stride;      // bytes, multiples of 16; below MAX_ROW_BYTES
    int M, N;
    int kbytes;                     // length of a reduction row, 0: y is zeros; rows are readable to the next multiple of 16 bytes
    int pieces;                     // a is this many matrices, one behind the other, all multiplied by the same b
    size_t piece_stride;            // bytes
    const float *a_scale, *b_scale; // NULL: 1
    const void *bias;               // NULL: none
    int bias_dtype;
    void *y;                        // dense [M][N]
};

constexpr size_t MAX_ROW_BYTES = 8u << 20; // 256 rows stay within 32-bit offsets

// Bytes of workspace for partial results (0: the reduction is not split); 16-byte aligned.
size_t tile_product_workspace(int M, int N, int kbytes, int pieces);
// out_dtype: y's type; f16: the operands are binary16 and kbytes is a multiple of 128, else int8.
int launch_tile_product(const TileArgs &p, bool f16, int out_dtype, void *workspace, const char *name, hipStream_t stream);

} // namespace rexsc
