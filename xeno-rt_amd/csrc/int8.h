// Rows and weight matrices in 8-bit integers with scales.
//
// Rows: values[m][j] (signed bytes, a row every int8_stride(k) bytes) and scales[m] (float32); row m stands for values[m][j] * scales[m]. Behind the k
// columns the operators write zeros, and packed weights have zeros there in any case, so that every product runs in whole steps of 128 along k.
//
// A weight matrix w[rows][k] is kept in tiles of 16 rows x 64 columns, 1 KB each, the tiles of a group of 16 rows one after another along k, groups one
// after another. Inside a tile the 16-byte pieces (16 columns of one row) lie in the order in which the lanes of a wavefront hold the A operand of
// v_mfma_i32_16x16x64_i8: piece (row r, columns 16 c .. 16 c + 15) at place r + 16 c, so that one load instruction of a wavefront reads a whole
// contiguous tile. A gated matrix [gate rows | up rows] of n outputs has in group g the gate rows 8 g .. 8 g + 7, then the up rows of the same outputs.
// Rows that fill up a group hold zeros. The rows' scales lie in the order of the packed rows (zeros where there is no row).
#pragma once
#include "common.h"
#include "xrt_hip.h"

#define XRT_INT8_STEP 128                   // columns that a product takes at a time
#define XRT_INT8_MOST_K XRT_INT8_K_LIMIT    // 2^14 * k stays below 2^31: a sum of k products of two signed bytes fits 32 bits

#define XRT_INT8_GRID_THREADS (1L << 32)    // a launch takes the number of its threads modulo this, without an error: there are fewer

__host__ __device__ inline long int8_stride(long k) { return (k + XRT_INT8_STEP - 1) / XRT_INT8_STEP * XRT_INT8_STEP; }
// groups of 16 packed rows of a matrix with n outputs
__host__ __device__ inline long int8_groups(long n, bool gated) { return gated ? (n + 7) / 8 : (n + 15) / 16; }
