// The 8-bit product for a few tokens (a decoding step): bound by reading the weights once.
#pragma once
#include "tile_product.h"

namespace rexsc {

constexpr int FEW_ROWS = 48; // most tokens the kernel takes
bool few_rows_takes(int M, int N); // whether it is the faster one

// y = a b^T of int8 operands with their epilogue, as TileArgs says (one piece).
int launch_few_rows(const TileArgs &p, int out_dtype, hipStream_t stream);

// The same from float tokens x [M][K] (rows x_stride elements apart), taken to 8 bits in every block: where M K and N are
// small and the rows begin on 16 bytes.
bool few_rows_fuses(int M, int N, int K, const void *x, size_t x_stride, int dtype);
int launch_few_rows_fused(const TileArgs &p, const void *x, size_t x_stride, int dtype, hipStream_t stream);

} // namespace rexsc
