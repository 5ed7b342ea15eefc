// Where the kernels of gemm_int8.hip read and write, as functions of the sizes and of the workgroup's, wavefront's and lane's numbers. The kernels call them, and
// so does xrt_linear_int8_reach on the host, which says without a GPU what a workgroup reaches.
#pragma once
#include "int8.h"
#include "large_tiles.h"

namespace {

constexpr int STEP_A = XRT_INT8_STEP;             // bytes from a step of 128 columns to the next, in a row of a
constexpr int STEP_W = 16 * XRT_INT8_STEP;        // in a group of w

// Where the sums of a block (16 rows of a and a group of w) lie in a part of the workspace, in pieces of 16 bytes a lane.
__host__ __device__ __forceinline__ long sums_place(int part, int M, int block, int groups, int group) {
    return (((long)part * ((M + 15) / 16) + block) * groups + group) * XRT_WAVE;
}

// ---- the kernel of few rows
// A workgroup's tile and its part of k (cut: there are parts). once: the rows of a are one tile.
__host__ __device__ __forceinline__ PartPlace few_place(int id, int tiles_m, int tiles_n, bool cut, int parts, bool once) {
    if (cut && once) return PartPlace{TilePlace{id < tiles_n * parts ? 0 : -1, id % tiles_n}, id / tiles_n};
    return part_place(id, 0, tiles_m, tiles_n, cut ? parts : 0);
}

// The steps along k of one of a workgroup's wavefronts: dealt evenly to the parts and within a part to the wavefronts.
struct Share { int first, count; };
__host__ __device__ __forceinline__ Share few_share(int units, bool cut, int part, int parts, int wave, int waves) {
    const int begin = cut ? (int)((long)units * part / parts) : 0, end = cut ? (int)((long)units * (part + 1) / parts) : units;
    const int first = begin + (end - begin) * wave / waves;
    return Share{first, begin + (end - begin) * (wave + 1) / waves - first};
}

// A lane's 16 bytes of the first 64 columns of step `first`, of a group of w (one beyond the matrix: the last one again) and of its row of a block of a (likewise);
// the other 64 columns lie half a step of w, 64 bytes of a behind.
__host__ __device__ __forceinline__ long few_w_offset(int group, int groups, int stride, int first, int lane) {
    return (long)min(group, groups - 1) * 16 * stride + (long)first * STEP_W + lane * 16;
}
__host__ __device__ __forceinline__ long few_a_offset(int block, int M, int stride, int first, int lane) {
    return (long)min(block * 16 + lane % 16, M - 1) * stride + (long)first * STEP_A + lane / 16 * 16;
}

// ---- the kernel with tiles in LDS: bm rows of a by bn packed rows of w, eight wavefronts, two by four
constexpr int LARGE_WAVES_N = 4;

// What a tile and one of its wavefronts stand for.
struct LargeTile {
    int m0, first_group, end;         // the tile's first row of a and first group of w; the row behind its last
    int upper_blocks, blocks;         // of 16 rows of a: of the wavefronts 0 to 3, and of this one
    int wave_row, wave_group;         // the wavefront's first row of a and first group of w
    int missing;                      // rows of the first half of the bm that no wavefront has
};
__host__ __device__ __forceinline__ LargeTile large_tile(TilePlace at, int bm, int bn, int height, int M, int wave) {
    LargeTile t;
    const int wave_m = wave / LARGE_WAVES_N;
    t.m0 = at.m * height;
    t.first_group = at.n * (bn / 16);
    t.end = min(t.m0 + height, M);
    t.upper_blocks = (height / 16 + 1) / 2;
    t.blocks = wave_m == 0 ? t.upper_blocks : height / 16 - t.upper_blocks;
    t.wave_row = t.m0 + wave_m * t.upper_blocks * 16;
    t.wave_group = t.first_group + wave % LARGE_WAVES_N * (bn / LARGE_WAVES_N / 16);
    t.missing = bm / 2 - t.upper_blocks * 16;
    return t;
}
__host__ __device__ __forceinline__ int large_row_end(const LargeTile& t) { return min(t.wave_row + t.blocks * 16, t.end); }      // of the wavefront's rows

// The kilobyte of LDS (8 rows of a, or a packed tile of w) that a wavefront's load i of half h fills; rows: a wavefront's rows of the operand in the tile;
// blocks: kilobytes of a half.
__host__ __device__ __forceinline__ int large_block(int h, int i, int rows, int blocks, int wave) {
    const int per = rows / 16, p = min(i * 8 + wave, blocks - 1);
    return (p / per * rows + h * (rows / 2)) / 8 + p % per;
}

// A lane's 16 bytes of such a kilobyte at step 0, from the tile's first byte of a and of w. (They fit 32 bits: 256 rows of up to 131072 bytes.) Piece c of row r
// of a lies at place c ^ (r % 8) of the row in LDS; rows beyond the tile and groups beyond the matrix: the last one again.
__host__ __device__ __forceinline__ unsigned large_a_offset(const LargeTile& t, int block, int bm, int stride, int lane) {
    const int row = block * 8 + lane / 8 - (block * 8 >= bm / 2 ? t.missing : 0);
    return (unsigned)min(row, t.end - 1 - t.m0) * (unsigned)stride + (unsigned)((lane % 8) ^ (lane / 8)) * 16u;
}
__host__ __device__ __forceinline__ unsigned large_w_offset(const LargeTile& t, int block, int groups, int stride, int lane) {
    return (unsigned)min(block / 2, groups - 1 - t.first_group) * 16u * (unsigned)stride + (unsigned)(block % 2) * 1024u + (unsigned)lane * 16u;
}

// The scales of row i of the tile's rows of a and of its packed row i of w: from the tile's first one on (in 64 bits: 2^30 rows of scales are 2^32 bytes), bytes.
struct ScalePlace { long first; unsigned offset; };
__host__ __device__ __forceinline__ ScalePlace large_a_scale(const LargeTile& t, int i, int M) { return ScalePlace{t.m0, (unsigned)min(i, M - 1 - t.m0) * 4u}; }
__host__ __device__ __forceinline__ ScalePlace large_w_scale(const LargeTile& t, int i, int groups) {
    return ScalePlace{(long)t.first_group * 16, (unsigned)min(i, (groups - t.first_group) * 16 - 1) * 4u};
}

// The steps along k of a part: steps_a_part of them, the last part what is left.
__host__ __device__ __forceinline__ Share large_share(int units, int part, int steps_a_part) {
    const int first = part * steps_a_part;
    return Share{first, min(steps_a_part, units - first)};
}

}  // namespace
