// What the products with large tiles share (gemm_mfma.hip, gemm_int8.hip): which tile a workgroup takes, and how the sums of the matrix cores leave the
// registers in whole cache lines.
#pragma once
#include "common.h"

namespace {

typedef unsigned uint4v __attribute__((ext_vector_type(4)));

// Which tile of tiles_m x tiles_n a workgroup takes. Ids are dealt to the XCDs round-robin: each XCD gets a contiguous run of
// tiles, and a run is walked n-fastest inside panels of 8 n-tiles, so that the tiles that run at one time on an XCD share a
// and w in its L2; m-fastest where there are up to four rows of tiles (a panel's tiles of one n would often lie on two XCDs, which then both read their w), but not where k
// is no multiple of 64 (panels): operands then go through the registers, and tiles of one n that run side by side took up to 1.12 times as long as those of one m (331 rows of
// x, 12696 of w, k = 8480 160 -> 180 us; 150 such products otherwise the same). An id beyond the tiles (grids are whole rounds over the XCDs) has none: m is negative.
struct TilePlace { int m, n; };
__host__ __device__ __forceinline__ TilePlace tile_place(int id, int tiles_m, int tiles_n, bool panels = false) {
    const int total = tiles_m * tiles_n;
    const int xcds = 8;
    id = (id % xcds) * ((total + xcds - 1) / xcds) + id / xcds;
    if (id >= total) return TilePlace{-1, 0};
    if (tiles_m <= 4 && !panels) return TilePlace{id % tiles_m, id / tiles_m};
    constexpr int PANEL = 8;
    const int panel = id / (PANEL * tiles_m), in_panel = id % (PANEL * tiles_m);
    const int panel_width = min(PANEL, tiles_n - panel * PANEL);
    return TilePlace{in_panel / panel_width, panel * PANEL + in_panel % panel_width};
}

// The same of a product whose k is split into parts, in one of two orders. By columns: an XCD gets a run of tiles and all parts of them, a grid row each. By
// parts (by_parts: their number; else 0, and `row` is the workgroup's grid row): it gets a run of tiles and parts, part after part, so that it reads some
// slices of k of a, which its L2 holds, instead of all of a, and no XCD has more to do for a number of tiles that does not divide.
struct PartPlace { TilePlace tile; int part; };
__host__ __device__ __forceinline__ PartPlace part_place(int id, int row, int tiles_m, int tiles_n, int by_parts) {
    if (by_parts == 0) return PartPlace{tile_place(id, tiles_m, tiles_n), row};
    constexpr int XCDS = 8;
    const int tiles = tiles_m * tiles_n, total = tiles * by_parts;
    id = (id % XCDS) * ((total + XCDS - 1) / XCDS) + id / XCDS;
    if (id >= total) return PartPlace{TilePlace{-1, 0}, 0};
    const int tile = id % tiles;
    return PartPlace{TilePlace{tile % tiles_m, tile / tiles_m}, id / tiles};
}
// Workgroups that such a product's launch has, places that no tile is dealt to among them.
inline long part_ids(long tiles, int parts, bool by_parts) { return by_parts ? (tiles * parts + 7) / 8 * 8 : (tiles + 7) / 8 * 8 * parts; }

// The rows of a of each tile, where tiles of up to `most` rows (a multiple of 16) share M.
inline int even_height(int M, int most) {
    const long tiles = ((long)M + most - 1) / most;
    return (int)((M + tiles - 1) / tiles + 15) / 16 * 16;
}

// ---- the large tiles' small pieces
// The upper 32 lanes of `low` change places with the lower 32 lanes of `high`.
__device__ __forceinline__ void exchange_halves(float& low, float& high) {
    const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, low), __builtin_bit_cast(unsigned, high), false, false);
    const unsigned first = both[0], second = both[1];          // (a vector's element itself is not what a bit cast takes)
    low = __builtin_bit_cast(float, first);
    high = __builtin_bit_cast(float, second);
}
// In every row of 16 lanes the upper eight lanes of `low` change places with the lower eight lanes of `high`.
__device__ __forceinline__ void exchange_eights(unsigned& low, unsigned& high) {
    const unsigned l = low, h = high;
    low = __builtin_amdgcn_update_dpp(l, h, 0x128 /* row_ror:8 */, 0xf, 0xc /* lanes 8 to 15 */, false);
    high = __builtin_amdgcn_update_dpp(h, l, 0x128, 0xf, 0x3 /* lanes 0 to 7 */, false);
}
__device__ __forceinline__ void exchange_eights(float& low, float& high) {
    unsigned l = __builtin_bit_cast(unsigned, low), h = __builtin_bit_cast(unsigned, high);
    exchange_eights(l, h);
    low = __builtin_bit_cast(float, l);
    high = __builtin_bit_cast(float, h);
}
template <typename TO>
__device__ __forceinline__ unsigned two_bf16(float a, float b) {
    return (unsigned)__builtin_bit_cast(unsigned short, from_float<bf16>(a)) | (unsigned)__builtin_bit_cast(unsigned short, from_float<bf16>(b)) << 16;
}
// Four values of each of two blocks, rounded to bfloat16, exchanged between the two rows of 16 lanes of each half of the
// wavefront: the first row gets the first block's values of both rows (eight neighbours), the second row the second block's.
template <typename TO>
__device__ __forceinline__ uint4v join_rows(const float (&first)[4], const float (&second)[4]) {
    const auto low = __builtin_amdgcn_permlane16_swap(two_bf16<TO>(first[0], first[1]), two_bf16<TO>(second[0], second[1]), false, false);
    const auto high = __builtin_amdgcn_permlane16_swap(two_bf16<TO>(first[2], first[3]), two_bf16<TO>(second[2], second[3]), false, false);
    return uint4v{low[0], high[0], low[1], high[1]};
}

}  // namespace
