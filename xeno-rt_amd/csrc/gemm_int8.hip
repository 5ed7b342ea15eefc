// Products of rows and weights in 8-bit integers (int8.h), on the matrix cores:
//
//     out[m, n] (+)= float(sum_j a[m, j] * w[n, j]) * a_scales[m] * w_scales[n]
//
// The sum is exact: whole numbers of 32 bits (k is limited so that it cannot overflow). Every kernel here therefore gives the same bits for a row of a,
// however many other rows there are and however k is cut. It is rounded to float32 once, then multiplied by the row's and by the channel's scale.
//
// v_mfma_i32_16x16x64_i8 takes w as its A operand and a as its B operand: lane (r, c) = (lane % 16, lane / 16) holds columns 16 c .. 16 c + 15 of packed row
// r of w and of row r of a, and gets the sums of row r of a with packed rows 4 c .. 4 c + 3 of w. A "block" below is such a 16 x 16 piece of the result.
//
// Up to 64 rows the product is bound by reading w, and gemm_int8_few_kernel streams it through registers. More rows go through tiles in LDS
// (gemm_int8_large_kernel). Where there are too few workgroups for the chip, k is cut into parts whose sums, as the lanes hold them, go to a workspace;
// int8_finish_kernel adds them and does the rest.
#include <limits.h>

#include <algorithm>
#include <type_traits>
#include "int8.h"
#include "activation.h"
#include "int8_places.h"

namespace {

typedef int int4v __attribute__((ext_vector_type(4)));
enum { MODE_STORE = 0, MODE_ACCUMULATE = 1, MODE_GATED = 2 };

// Neighbouring columns of a row of out [M][N], in one piece wherever they lie (global memory wants no more than an element's alignment), and those that
// are there where the row ends inside the piece. (Four accesses of one element each instead: 1588 rows added to, 717 channels, k = 384 21.7 us, 13.9 so.)
template <typename T, int COUNT> struct Run { T e[COUNT]; };
template <typename TO>
__device__ __forceinline__ void load_run(const TO* out, long m, long n, int M, int N, float (&v)[4]) {
    const TO* row = out + min(m, (long)M - 1) * (long)N;       // (rows and columns beyond the matrix: something inside, not used)
    if (n + 4 <= N) {
        Run<TO, 4> run;
        __builtin_memcpy(&run, row + n, sizeof(run));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = to_float(run.e[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = to_float(row[min(n + e, (long)N - 1)]);
    }
}
template <typename TO, int COUNT>
__device__ __forceinline__ void store_run(TO* out, long m, long n, int M, int N, const Run<TO, COUNT>& run) {
    typedef unsigned Words __attribute__((ext_vector_type(COUNT * sizeof(TO) / 4)));
    typedef Words Anywhere __attribute__((aligned(2)));
    if (m >= M || n >= N) return;
    TO* row = out + m * (long)N + n;
    if (n + COUNT <= N) {
        *reinterpret_cast<Anywhere*>(row) = __builtin_bit_cast(Words, run);
    } else {
#pragma unroll
        for (int e = 0; e < COUNT; ++e)
            if (n + e < N) row[e] = run.e[e];
    }
}
template <typename TO>
__device__ __forceinline__ void store_run(TO* out, long m, long n, int M, int N, const float (&v)[4]) {
    Run<TO, 4> run;
#pragma unroll
    for (int e = 0; e < 4; ++e) run.e[e] = from_float<TO>(v[e]);
    store_run<TO, 4>(out, m, n, M, N, run);
}

// (Not contracted with an addition behind it, which one kernel would do and another not: the bits would go by the number of rows.)
__device__ __forceinline__ float scaled(int sum, float a_scale, float w_scale) {
#pragma clang fp contract(off)
    return (float)sum * a_scale * w_scale;
}

// What a product writes, and what the sums are multiplied by.
template <typename TO>
struct Result {
    const float* a_scales;
    const float* w_scales;      // in the order of the packed rows
    TO* out;                    // [M][N]
    int M, N, activation;
};

// Writes the block of rows m0 .. m0 + 15 of a and group `group` of w.
template <int MODE, typename TO>
__device__ __forceinline__ void finish_block(const int4v sum, long m0, long group, const Result<TO>& to) {
    const int lane = threadIdx.x % XRT_WAVE, r = lane % 16, c = lane / 16;
    const long m = m0 + r;
    const float a_scale = to.a_scales[m < to.M ? m : (long)to.M - 1];
    const float4 w_scale = *reinterpret_cast<const float4*>(to.w_scales + group * 16 + c * 4);
    float value[4] = {scaled(sum[0], a_scale, w_scale.x), scaled(sum[1], a_scale, w_scale.y), scaled(sum[2], a_scale, w_scale.z), scaled(sum[3], a_scale, w_scale.w)};
    long n = group * 16 + c * 4;
    bool mine = m < to.M;
    if constexpr (MODE == MODE_GATED) {
        // lanes c = 0, 1 hold the gate sums of outputs 8 group + 4 c + e, lanes c = 2, 3 the up sums of the same
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float up = of_other_half(value[e]);
            value[e] = gate_activation<sizeof(TO) == 2>(value[e], to.activation) * up;
        }
        n = group * 8 + c * 4;
        mine = mine && c < 2;
    }
    if (!mine || n >= to.N) return;
    if constexpr (MODE == MODE_ACCUMULATE) {
        float before[4];
        load_run<TO>(to.out, m, n, to.M, to.N, before);
#pragma unroll
        for (int e = 0; e < 4; ++e) value[e] = before[e] + value[e];
    }
    store_run<TO>(to.out, m, n, to.M, to.N, value);
}

// Adds the parts of every block, one wavefront a block: sums[part][16 rows of a][group][lane].
template <int MODE, typename TO>
__global__ void __launch_bounds__(256) int8_finish_kernel(const int4v* __restrict__ sums, int parts, int groups, long blocks, const Result<TO> to) {
    const long block = (long)blockIdx.x * 4 + threadIdx.x / XRT_WAVE;
    if (block >= blocks) return;
    const int4v* at = sums + block * XRT_WAVE + threadIdx.x % XRT_WAVE;
    int4v sum{0, 0, 0, 0};
    for (int first = 0; first < parts; first += 8) {            // eight parts asked for at once, however many there are
        int4v piece[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) piece[i] = first + i < parts ? at[(first + i) * blocks * XRT_WAVE] : int4v{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += piece[i];
    }
    finish_block<MODE, TO>(sum, block / groups * 16, block % groups, to);
}

// ---- up to 64 rows ----------------------------------------------------------------------------------------------------------------------------------------

constexpr int WAVES = 8;

// MT: blocks of 16 rows of a; G: groups of 16 packed rows of w a workgroup. Its wavefronts share out k, each with a run of its own, and add their sums
// through LDS. Nothing is read twice by a workgroup, so a's rows come from L2 as often as there are workgroups along n: with G groups a workgroup reads
// MT / G times as much of a as of w. PARTS: k is cut among workgroups. ONCE: the rows of a are one tile, so that every byte of w is read by one workgroup,
// and is asked for past the caches. Reading w bounds it: 8 rows, k = 4096, 14336 pairs 19.5 us, 6.0 TB/s; 128256 channels 83 us, 6.4 TB/s; a kernel that only reads 7.2.
template <int MT, int G, int MODE, typename TO, bool PARTS, bool ONCE>
__global__ void __launch_bounds__(WAVES * XRT_WAVE, MT * G <= 2 ? 4 : 2) gemm_int8_few_kernel(const signed char* __restrict__ a, const signed char* __restrict__ w,
                                                                                          int4v* __restrict__ sums, int M, int stride, int groups, int tiles_m,
                                                                                          int tiles_n, int parts, const Result<TO> to) {
    constexpr int AT_ONCE = G * MT < 8 ? G * MT : 8;            // blocks whose sums lie in LDS at one time
    __shared__ int4v shared[WAVES][AT_ONCE][XRT_WAVE];
    // An XCD gets a run of tiles; split over one tile of rows: tiles and parts in turn. (33 rows, k = 4096, 1792 groups 26.0 us in runs, 28.6 in turn, 8 rows 19.5 either way;
    // 64 rows, k = 14336, 4096 channels in four parts 19.2 and 17.9.)
    const PartPlace place = few_place(blockIdx.x, tiles_m, tiles_n, PARTS, parts, ONCE);
    if (place.tile.m < 0) return;
    const int lane = threadIdx.x % XRT_WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / XRT_WAVE);
    const int first_group = place.tile.n * G, first_block = place.tile.m * MT;

    // units of 128 columns
    const int part = PARTS ? place.part : 0;
    const Share share = few_share(stride / XRT_INT8_STEP, PARTS, part, parts, wave, WAVES);
    const int first = share.first, count = share.count;

    const signed char* w_at[G];
    const signed char* a_at[MT];
#pragma unroll
    for (int g = 0; g < G; ++g) w_at[g] = w + few_w_offset(first_group + g, groups, stride, first, lane);
#pragma unroll
    for (int i = 0; i < MT; ++i) a_at[i] = a + few_a_offset(first_block + i, M, stride, first, lane);

    struct Unit { int4v w[G][2], a[MT][2]; };
    auto load = [&](Unit& unit, int u) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) unit.a[i][j] = *reinterpret_cast<const int4v*>(a_at[i] + (long)u * STEP_A + j * (STEP_A / 2));
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int4v* from = reinterpret_cast<const int4v*>(w_at[g] + (long)u * STEP_W + j * (STEP_W / 2));
                unit.w[g][j] = ONCE ? __builtin_nontemporal_load(from) : *from;
            }
    };
    int4v acc[G][MT];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[g][i] = int4v{0, 0, 0, 0};
    auto multiply = [&](const Unit& unit) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[g][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(unit.w[g][j], unit.a[i][j], acc[g][i], 0, 0, 0);
    };
    // Two units in turn: while one is multiplied the other is on its way. (Three cost the workgroups that run beside this one their registers: 32 rows, k = 4096,
    // 14336 pairs 25.2 us with three, 23.1 with two; 64 rows, which then spill, 66.8 and 31.0.)
    constexpr int RING = 2;
    Unit ring[RING];
#pragma unroll
    for (int b = 0; b < RING; ++b)
        if (b < count) load(ring[b], b);
    int u = 0;
    for (; u + 2 * RING <= count; u += RING)
#pragma unroll
        for (int b = 0; b < RING; ++b) {
            multiply(ring[b]);
            load(ring[b], u + b + RING);
        }
#pragma unroll
    for (int b = 0; b < RING; ++b)
        if (u + b < count) {
            multiply(ring[b]);
            if (u + b + RING < count) load(ring[b], u + b + RING);
        }
#pragma unroll
    for (int b = 0; b < RING; ++b)
        if (u + RING + b < count) multiply(ring[b]);

    // the wavefronts' sums of a block, added by the wavefront that writes it
#pragma unroll
    for (int t0 = 0; t0 < G * MT; t0 += AT_ONCE) {
        if (t0 > 0) __syncthreads();
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t) shared[wave][t][lane] = acc[(t0 + t) / MT][(t0 + t) % MT];
        __syncthreads();
        if (wave >= AT_ONCE) continue;
        int4v sum = shared[0][wave][lane];
#pragma unroll
        for (int other = 1; other < WAVES; ++other) sum += shared[other][wave][lane];
        const int group = first_group + (t0 + wave) / MT, block = first_block + (t0 + wave) % MT;
        if (group >= groups || block * 16 >= M) continue;
        if constexpr (PARTS) sums[sums_place(part, M, block, groups, group) + lane] = sum;
        else finish_block<MODE, TO>(sum, (long)block * 16, group, to);
    }
}

// ---- more rows --------------------------------------------------------------------------------------------------------------------------------------------

// Tiles of BM (256, 192 or 128) rows of a by BN (256, or 128) packed rows of w: eight wavefronts, two to a SIMD, which take turns as those of the bfloat16 product's
// large tiles do. Power bounds it: 4096 rows, k = 14336, 8192 channels 310 to 329 us, 2.9 to 3.1 Pop/s; these instructions reach 3.1 on numbers that stay in registers; at
// k = 4096, 14336 pairs 342 to 373 us, of which a round's first loads and its results take a sixth. Of the two on a SIMD (one of each group of four) one reads the operands of its next products from LDS and asks for tiles to come while the other
// multiplies; a barrier ends a turn, and the second group runs one barrier behind the first. A wavefront's part (BM / 2 x BN / 4) is four quarters along k: (half
// h of its rows of a, half g of its rows of w) in the order (0,0) (0,1) (1,1) (1,0), so that every turn reads one new half: w0, w1, a1, and a0 of the next
// tile. A half is loaded into the place of the same half two tiles ago as soon as both groups have read that, seven quarters before it is needed, and the
// waits leave the newer six quarters' loads in flight.
//
// height: the rows of a that a tile stands for, a multiple of 16 up to BM (even_height): the first four wavefronts take half of the blocks of 16, or one
// more than the others, and a wavefront runs the loop made for its number of blocks (all, one or two fewer).
template <int BM, int BN, int MODE, typename TO, bool PARTS>
__global__ void __launch_bounds__(8 * XRT_WAVE) gemm_int8_large_kernel(const signed char* __restrict__ a, const signed char* __restrict__ w, int4v* __restrict__ sums,
                                                                       int stride, int groups, int tiles_m, int tiles_n, int height, int by_parts,
                                                                       int steps_a_part, const Result<TO> to) {
    constexpr int STEP = XRT_INT8_STEP, WAVES_N = LARGE_WAVES_N;
    constexpr int WAVE_M = BM / 2, WAVE_N = BN / WAVES_N;      // the wavefront's part of the tile
    constexpr int TM = WAVE_M / 16, TN = WAVE_N / 16, HM = TM / 2, HN = TN / 2;      // blocks of 16 rows of a and of w: all, and a half
    constexpr int BLOCKS_A = BM / 16;                          // kilobytes of one half of a: where they do not divide among the wavefronts, the spare loads fetch the last one again
    constexpr int LOADS_A = (BLOCKS_A + 7) / 8, LOADS_B = BN / 128;      // load instructions of a wavefront for one half
    extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
    unsigned char* stage_a = lds_raw;                          // [2][BM][128]: rows of eight 16-byte pieces, swizzled
    unsigned char* stage_b = stage_a + 2 * BM * STEP;          // [2][16 groups][2][1024]: packed tiles as they lie
    float* lds_a_scales = reinterpret_cast<float*>(stage_b + 2 * BN * STEP);      // [256] of the tile's rows
    float* lds_w_scales = lds_a_scales + 256;                  // [BN]

    const PartPlace dealt = PARTS ? part_place(blockIdx.x, blockIdx.y, tiles_m, tiles_n, by_parts) : PartPlace{tile_place(blockIdx.x, tiles_m, tiles_n), 0};
    if (dealt.tile.m < 0) return;
    const int M = to.M, N = to.N;
    const int lane = threadIdx.x % XRT_WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / XRT_WAVE);
    const int wave_m = wave / WAVES_N, wave_n = wave % WAVES_N;
    const int quad = lane / 16;                                // which four packed rows of a block this lane has the sums of
    const LargeTile tile = large_tile(dealt.tile, BM, BN, height, M, wave);
    const int m0 = tile.m0, first_group = tile.first_group, blocks = tile.blocks, wave_row = tile.wave_row;
    a += (long)m0 * stride;
    w += (long)first_group * 16 * stride;

    // (The pieces of a row of a change places: the lanes that a 16-byte read serves at once then take different banks.)
    auto block_of = [&](int h, int i, int rows, int blocks) { return large_block(h, i, rows, blocks, wave); };
    unsigned off_a[2][LOADS_A], off_b[2][LOADS_B];             // bytes
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < LOADS_A; ++i) off_a[h][i] = large_a_offset(tile, block_of(h, i, WAVE_M, BLOCKS_A), BM, stride, lane);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < LOADS_B; ++i) off_b[h][i] = large_w_offset(tile, block_of(h, i, WAVE_N, BN / 16), groups, stride, lane);
    const unsigned lds_a0 = lds_address(stage_a), lds_b0 = lds_address(stage_b);
    auto issue_a = [&](int h, int stage, int step) {
#pragma unroll
        for (int i = 0; i < LOADS_A; ++i)
            load_to_lds(a, off_a[h][i] + (unsigned)step * (unsigned)STEP_A, lds_a0 + (unsigned)(stage * BM * STEP + block_of(h, i, WAVE_M, BLOCKS_A) * 1024));
    };
    auto issue_b = [&](int h, int stage, int step) {
#pragma unroll
        for (int i = 0; i < LOADS_B; ++i)
            load_to_lds(w, off_b[h][i] + (unsigned)step * (unsigned)STEP_W, lds_b0 + (unsigned)(stage * BN * STEP + block_of(h, i, WAVE_N, BN / 16) * 1024));
    };
    // the tile's scales, ahead of the tiles themselves: wavefronts 0 to 3 those of 64 rows of a each, 4 to 7 those of 64 packed rows of w
    if constexpr (!PARTS) {
        if (wave < 4) {
            const ScalePlace at = large_a_scale(tile, wave * 64 + lane, M);
            load_dword_to_lds(to.a_scales + at.first, at.offset, lds_address(lds_a_scales + wave * 64));
        } else if ((wave - 4) * 64 < BN) {
            const ScalePlace at = large_w_scale(tile, (wave - 4) * 64 + lane, groups);
            load_dword_to_lds(to.w_scales + at.first, at.offset, lds_address(lds_w_scales + (wave - 4) * 64));
        }
    }
    // where this lane finds its 16 bytes of block 0 of its wavefront, for either 64 columns of the tile
    const unsigned char* place_a[2];
    const unsigned char* place_b[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        place_a[ks] = stage_a + (wave_m * WAVE_M + lane % 16) * STEP + (((ks * 4 + quad) ^ (lane % 8)) * 16);
        place_b[ks] = stage_b + wave_n * WAVE_N * STEP + ks * 1024 + lane * 16;
    }
    int4v xa[2][2][HM], wb[2][2][HN];                          // [half][64 columns][block]
    // (T: the blocks of the wavefront, TM or somewhat fewer; they are missing from the second half)
    auto read_a = [&](auto t, int h, int stage) {
        constexpr int T = decltype(t)::value;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < HM; ++i)
                if (h * HM + i < T) xa[h][ks][i] = *reinterpret_cast<const int4v*>(place_a[ks] + stage * BM * STEP + (h * HM + i) * 16 * STEP);
    };
    auto read_b = [&](int h, int stage) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < HN; ++j)
                wb[h][ks][j] = *reinterpret_cast<const int4v*>(place_b[ks] + stage * BN * STEP + (h * HN + j) * 16 * STEP);
    };
    int4v acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = int4v{0, 0, 0, 0};
    auto multiply = [&](auto t, int h, int g) {
        constexpr int T = decltype(t)::value;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < HM; ++i)
#pragma unroll
                for (int j = 0; j < HN; ++j)
                    if (h * HM + i < T)
                        acc[h * HM + i][g * HN + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wb[g][ks][j], xa[h][ks][i], acc[h * HM + i][g * HN + j], 0, 0, 0);
    };
    const Share share = large_share(stride / STEP, dealt.part, steps_a_part);
    const int first_step = share.first, steps = share.count, last_step = first_step + steps - 1;
    auto step_of = [&](int t) { return min(first_step + t, last_step); };        // (tiles beyond the end: the last one again, into a place nobody reads)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        issue_a(0, t, step_of(t));
        issue_b(0, t, step_of(t));
        issue_b(1, t, step_of(t));
        issue_a(1, t, step_of(t));
    }
    // Loads that may stay in flight behind a quarter's reads: those of the six quarters after the next one.
    constexpr int ALL = 2 * (LOADS_A + LOADS_B);
    auto barrier = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    auto walk = [&](auto t_blocks) {
        wait_loads_and_barrier<ALL + LOADS_A + LOADS_B>();     // a0 and w0 of tile 0 are in LDS
        read_a(t_blocks, 0, 0);
        wait_loads_and_barrier<ALL + LOADS_A + LOADS_B>();     // and a0 is read by all: the first turn fills its place again
        auto turn = [&](auto in_flight, int h, int g) {
            __builtin_amdgcn_sched_barrier(0);
            wait_loads_and_barrier<decltype(in_flight)::value>();  // this wavefront's reads are done: what it read may be overwritten
            __builtin_amdgcn_sched_barrier(0);
            multiply(t_blocks, h, g);
            barrier();
        };
        if (wave >= 4) barrier();
        for (int t = 0; t < steps; ++t) {
            const int now = t % 2, next = step_of(t + 2);
            read_b(0, now);
            issue_a(0, now, next);
            turn(std::integral_constant<int, ALL + 2 * LOADS_A>{}, 0, 0);           // in flight: a1 a0 w0 w1 a1 a0
            read_b(1, now);
            issue_b(0, now, next);
            turn(std::integral_constant<int, ALL + LOADS_A + LOADS_B>{}, 0, 1);     // a0 w0 w1 a1 a0 w0
            read_a(t_blocks, 1, now);
            issue_b(1, now, next);
            turn(std::integral_constant<int, ALL + 2 * LOADS_B>{}, 1, 1);           // w0 w1 a1 a0 w0 w1
            read_a(t_blocks, 0, now ^ 1);
            issue_a(1, now, next);
            turn(std::integral_constant<int, ALL + LOADS_A + LOADS_B>{}, 1, 0);     // w1 a1 a0 w0 w1 a1
        }
    };
    if (BM == 128 || blocks == TM) walk(std::integral_constant<int, TM>{});
    else if (blocks == TM - 1) walk(std::integral_constant<int, TM - 1>{});
    else walk(std::integral_constant<int, TM - 2>{});          // (fewer than that: some products that nobody writes)
    if (wave < 4) barrier();
    wait_loads_and_barrier<0>();                               // nothing lands in LDS after this

    // ---- epilogue: element e of acc[i][j] is row i * 16 + lane % 16 of a and packed row j * 16 + quad * 4 + e of w
    const int row_end = large_row_end(tile), wave_group = tile.wave_group;
    if constexpr (PARTS) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                if (wave_row + i * 16 < row_end && wave_group + j < groups)
                    sums[sums_place(dealt.part, M, wave_row / 16 + i, groups, wave_group + j) + lane] = acc[i][j];
        return;
    }
    float4 w_scale[TN];
    float a_scale[TM];
#pragma unroll
    for (int j = 0; j < TN; ++j) w_scale[j] = *reinterpret_cast<const float4*>(lds_w_scales + wave_n * WAVE_N + j * 16 + quad * 4);
#pragma unroll
    for (int i = 0; i < TM; ++i) a_scale[i] = lds_a_scales[min(wave_row - m0 + i * 16 + lane % 16, 255)];
    auto value = [&](int i, int j, int e) {
        const float of_channel = e == 0 ? w_scale[j].x : e == 1 ? w_scale[j].y : e == 2 ? w_scale[j].z : w_scale[j].w;
        return scaled(acc[i][j][e], a_scale[i], of_channel);
    };
    TO* out = to.out;
    typedef Run<TO, 8> Eight;
    if constexpr (MODE == MODE_GATED) {
        // A group of 16 packed rows holds the gate rows of 8 outputs, then their up rows: the lane with an output's up sum
        // is 32 lanes away. One exchange of half a register between the sums of two blocks of a leaves gate and up of
        // every output of both in one lane (lanes 0 to 31 the first block's outputs, the others the second's); for
        // bfloat16 another one between two groups of w brings eight neighbouring outputs together: 16 bytes a store.
        const long n_wave = (long)wave_group * 8;
#pragma unroll
        for (int i = 0; i < TM; i += 2) {
            const long m = wave_row + lane % 16 + i * 16 + lane / 32 * 16;
#pragma unroll
            for (int j = 0; j < TN; j += 2) {
                float made[2][4];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float gate = value(i, j + u, e), up = value(i + 1, j + u, e);
                        exchange_halves(gate, up);
                        made[u][e] = gate_activation<sizeof(TO) == 2>(gate, to.activation) * up;
                    }
                if constexpr (sizeof(TO) == 2) {
                    store_run<TO, 8>(out, m, n_wave + (j + quad % 2) * 8, row_end, N, __builtin_bit_cast(Eight, join_rows<TO>(made[0], made[1])));
                } else {
#pragma unroll
                    for (int u = 0; u < 2; ++u) store_run<TO>(out, m, n_wave + (j + u) * 8 + quad % 2 * 4, row_end, N, made[u]);
                }
            }
        }
    } else {
        // Two neighbouring blocks of columns change eight lanes with each other, so that an instruction takes eight rows of
        // 128 bytes, whole cache lines, instead of sixteen of 64.
        const long row8 = wave_row + lane % 8;
        const int upper = lane % 16 / 8;
        if constexpr (MODE == MODE_STORE && sizeof(TO) == 2) {
            if constexpr (TN == 2) {                           // (one piece of 32 columns: sixteen rows of 64 bytes)
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const float first[4] = {value(i, 0, 0), value(i, 0, 1), value(i, 0, 2), value(i, 0, 3)};
                    const float second[4] = {value(i, 1, 0), value(i, 1, 1), value(i, 1, 2), value(i, 1, 3)};
                    store_run<TO, 8>(out, wave_row + i * 16 + lane % 16, (long)wave_group * 16 + quad % 2 * 16 + quad / 2 * 8, row_end, N,
                                     __builtin_bit_cast(Eight, join_rows<TO>(first, second)));
                }
                return;
            } else {
            static_assert(TN == 4, "two pieces of 32 columns");
            const long n = (long)wave_group * 16 + (2 * upper + quad % 2) * 16 + quad / 2 * 8;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                uint4v piece[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float first[4] = {value(i, 2 * u, 0), value(i, 2 * u, 1), value(i, 2 * u, 2), value(i, 2 * u, 3)};
                    const float second[4] = {value(i, 2 * u + 1, 0), value(i, 2 * u + 1, 1), value(i, 2 * u + 1, 2), value(i, 2 * u + 1, 3)};
                    piece[u] = join_rows<TO>(first, second);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned low = piece[0][e], high = piece[1][e];
                    exchange_eights(low, high);
                    piece[0][e] = low;
                    piece[1][e] = high;
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) store_run<TO, 8>(out, row8 + i * 16 + u * 8, n, row_end, N, __builtin_bit_cast(Eight, piece[u]));
            }
            return;
            }
        }
        constexpr int RUN = TM % 4 == 0 ? 4 : 3;               // blocks of a whose old values are read in one go, before any is written
#pragma unroll
        for (int i0 = 0; i0 < TM; i0 += RUN) {
            float before[RUN][TN][4];
            if constexpr (MODE == MODE_ACCUMULATE) {
#pragma unroll
                for (int i = 0; i < RUN; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        load_run<TO>(out, row8 + (i0 + i) * 16 + j % 2 * 8, (long)(wave_group + j / 2 * 2 + upper) * 16 + quad * 4, row_end, N, before[i][j]);
            }
#pragma unroll
            for (int i = 0; i < RUN; ++i)
#pragma unroll
                for (int j = 0; j < TN; j += 2) {
                    float made[2][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        made[0][e] = value(i0 + i, j, e);
                        made[1][e] = value(i0 + i, j + 1, e);
                        exchange_eights(made[0][e], made[1][e]);
                        if constexpr (MODE == MODE_ACCUMULATE) {
                            made[0][e] = before[i][j][e] + made[0][e];
                            made[1][e] = before[i][j + 1][e] + made[1][e];
                        }
                    }
                    const long n = (long)(wave_group + j + upper) * 16 + quad * 4;
                    store_run<TO>(out, row8 + (i0 + i) * 16, n, row_end, N, made[0]);
                    store_run<TO>(out, row8 + (i0 + i) * 16 + 8, n, row_end, N, made[1]);
                }
        }
    }
}

// ---- which kernel -----------------------------------------------------------------------------------------------------------------------------------------

struct Plan {
    int tile;           // rows of a of a tile (256, 192, 128), or 0: the kernel of few rows
    int width;          // packed rows of w of a tile (256 or 128)
    int blocks;         // of 16 rows of a, of the kernel of few rows (1, 2 or 4)
    int groups;         // of w a workgroup, of the same (1, 2 or 4)
    int parts;          // of k
};

Plan plan_of(long M, long groups, long stride) {
    const long units = stride / XRT_INT8_STEP;
    // The kernel of few rows: up to 64, and more where its tiles of 64 x 64 find a compute unit each and no workgroup goes through many columns: a tile reads as much
    // of a as of w, and the larger tiles get k in the more parts the fewer of these there are. Without a cut 40 units of 128 columns to 56 of them by the number of
    // workgroups (us, and of the larger tiles: 217 rows, k = 384, 1312 channels 4.5 and 6.9; 1233, 5342, 497 15.7 and 17.9; 119, 5724, 4235 19.6 and 15.5; 225, 6021, 4037
    // 18.4 and 18.7; 92, 8327, 4784 23.4 and 16.4), else 32 a part (144, 15612, 928 14.1 and 15.4; 256, 13719, 1101 19.2 and 17.7; 480, 16494, 975 26.0 and 21.8).
    {
        // (two blocks of rows, 1792 groups of w: 26.8 us with two groups a workgroup, 23.0 with four; 384 groups: 8.6 and 10.7)
        Plan plan{0, 0, M <= 16 ? 1 : M <= 32 ? 2 : 4, M <= 16 ? 1 : M <= 32 && groups < 4 * XRT_COMPUTE_UNITS ? 2 : 4, 1};
        const long workgroups = (M + plan.blocks * 16 - 1) / (plan.blocks * 16) * ((groups + plan.groups - 1) / plan.groups);
        // k in as many parts as there are compute units for, each of 12 units of 128 columns by 16 rows at least, if the longest way along k gets shorter by 48 of them:
        // else the kernel that adds the parts takes what they save. (7 rows, k = 926, 297 channels 2.8 us whole, 4.6 in two; 3, 6640, 538 5.0 and 5.2 in six; 74, 6977, 330
        // pairs 8.5 in eight, 8.2 in nine; 16, 14336, 1024 11.6 whole, 9.5 in two, 7.7 in four; 239, 14602, 31 9.3 in eight, 7.9 in sixteen.)
        const int parts = (int)min(min(XRT_COMPUTE_UNITS / workgroups, units * plan.blocks / 12), 16L);
        if (parts > 1 && units * plan.blocks * (parts - 1) >= 48 * parts) plan.parts = parts;
        if (M <= 64 || (workgroups <= XRT_COMPUTE_UNITS && units <= (plan.parts == 1 ? 24 + workgroups / 8 : 32 * plan.parts))) return plan;
    }
    // What a tile height costs, fitted to products of 4096 rows, k = 4096 and 14336 (us): a step along k (256 rows: 1.31, 128: 0.80), and the first loads and the
    // epilogue. A partly filled round takes half of a full one and its share of the rest: power bounds the chip, and the compute units at work run faster.
    Plan plan{0, 256, 0, 0, 1};
    const long tiles_n = (groups + 15) / 16;
    double best = 0;
    for (const int tile : {256, 192, 128}) {
        const int height = even_height((int)M, tile);
        const long tiles = (M + tile - 1) / tile * tiles_n;
        const double rest = (double)(tiles % XRT_COMPUTE_UNITS) / XRT_COMPUTE_UNITS;
        const double cost = (tiles / XRT_COMPUTE_UNITS + (rest > 0 ? 0.55 + 0.45 * rest : 0)) * (units * (height + 73) * 0.004 + 2.7 + 0.0234 * tile);
        if (plan.tile == 0 || cost < best) plan.tile = tile, best = cost;
    }
    long tiles = (M + plan.tile - 1) / plan.tile * tiles_n;
    // Tiles half as wide where the others fill up to half of the chip, and k in parts as far as every compute unit gets one at most: a compute unit pulls no more
    // than some 29 GB/s of w, however much is asked for ahead (100 rows, k = 4096, 14336 pairs 34.5 us in 112 tiles, 28.7 in 224; three steps in LDS instead of two changed nothing).
    // A step along k takes 0.5 us, the parts' sums and the kernel that adds them 6 to 8, so a short k stays whole (416 rows, k = 987, 1705 pairs 8.9 us whole, 15.1 in two
    // parts; 423, 2293, 3037 channels 17.7 and 19.2; 375, 6572, 1709 pairs 33.2 and 25.4; 598, 10587, 851 pairs 31.6 in two, 26.2 in three).
    if (plan.tile == 128 && tiles * 2 <= XRT_COMPUTE_UNITS) plan.width = 128, tiles = (M + 127) / 128 * ((groups + 7) / 8);
    if (plan.width == 128 && units >= 32) plan.parts = (int)max(1L, min(XRT_COMPUTE_UNITS / tiles, 16L));
    const long steps = (units + plan.parts - 1) / plan.parts;
    plan.parts = (int)((units + steps - 1) / steps);           // (none is empty)
    return plan;
}

long sums_bytes(const Plan& plan, long M, long groups) { return plan.parts == 1 ? 0 : plan.parts * ((M + 15) / 16) * groups * XRT_WAVE * (long)sizeof(int4v); }

struct Operands { const signed char* a; const signed char* w; int4v* sums; int stride, groups; hipStream_t stream; };

template <int MT, int G, int MODE, typename TO, bool ONCE = true, bool SPLITS = true>
int launch_few(const Operands& o, const Plan& plan, const Result<TO>& to) {
    const int tiles_m = (to.M + MT * 16 - 1) / (MT * 16), tiles_n = (o.groups + G - 1) / G;
    const long ids = part_ids((long)tiles_m * tiles_n, plan.parts, true);        // a whole number of rounds over the XCDs
    XRT_REQUIRE(ids * WAVES * XRT_WAVE < XRT_INT8_GRID_THREADS, "linear_int8: too many tiles, %ld", ids);
    if (plan.parts == 1) gemm_int8_few_kernel<MT, G, MODE, TO, false, ONCE><<<(unsigned)ids, WAVES * XRT_WAVE, 0, o.stream>>>(o.a, o.w, nullptr, to.M, o.stride, o.groups, tiles_m, tiles_n, 1, to);
    else if constexpr (SPLITS) gemm_int8_few_kernel<MT, G, MODE_STORE, float, true, ONCE><<<(unsigned)ids, WAVES * XRT_WAVE, 0, o.stream>>>(o.a, o.w, o.sums, to.M, o.stride, o.groups, tiles_m, tiles_n, plan.parts, Result<float>{});
    XRT_REQUIRE(SPLITS || plan.parts == 1, "linear_int8: a product that is not cut, in %d parts", plan.parts);
    return 0;
}

template <int BM, int BN, int MODE, typename TO, bool PARTS>
int launch_large(const Operands& o, const Plan& plan, const Result<TO>& to) {
    constexpr size_t lds = (size_t)2 * (BM + BN) * XRT_INT8_STEP + 2 * 256 * sizeof(float);
    auto kernel = gemm_int8_large_kernel<BM, BN, MODE, TO, PARTS>;
    const int units = o.stride / XRT_INT8_STEP, steps = (units + plan.parts - 1) / plan.parts;
    const int height = even_height(to.M, BM), tiles_m = (to.M + height - 1) / height, tiles_n = (o.groups + BN / 16 - 1) / (BN / 16);
    const long ids = part_ids((long)tiles_m * tiles_n, plan.parts, true);        // a whole number of rounds over the XCDs
    XRT_REQUIRE(ids * WAVES * XRT_WAVE < XRT_INT8_GRID_THREADS, "linear_int8: too many tiles, %ld", ids);
    static bool configured[64] = {};                           // per instantiation and device
    int device = 0;
    XRT_REQUIRE(hipGetDevice(&device) == hipSuccess, "linear_int8: no current device");
    if (device < 0 || device >= 64 || !configured[device]) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        XRT_REQUIRE(e == hipSuccess, "linear_int8: cannot reserve %zu bytes of LDS: %s", lds, hipGetErrorString(e));
        if (device >= 0 && device < 64) configured[device] = true;
    }
    kernel<<<(unsigned)ids, 8 * XRT_WAVE, lds, o.stream>>>(o.a, o.w, o.sums, o.stride, o.groups, tiles_m, tiles_n, height, plan.parts, steps, to);
    return 0;
}

template <int MODE, typename TO>
int launch(const Operands& o, const Plan& plan, const Result<TO>& to) {
    int failed = 0;
    if (plan.tile == 0) {
        if (plan.blocks == 1) failed = launch_few<1, 1, MODE, TO>(o, plan, to);
        else if (plan.blocks == 2 && plan.groups == 2) failed = launch_few<2, 2, MODE, TO>(o, plan, to);
        else if (plan.blocks == 2) failed = launch_few<2, 4, MODE, TO, true, false>(o, plan, to);      // (1024 groups and more: never cut)
        else if (to.M <= 64) failed = launch_few<4, 4, MODE, TO>(o, plan, to);
        else failed = launch_few<4, 4, MODE, TO, false>(o, plan, to);
    } else if (plan.parts > 1) {
        Result<float> sizes{};
        sizes.M = to.M, sizes.N = to.N;
        XRT_REQUIRE(plan.tile == 128 && plan.width == 128, "linear_int8: tiles of %d x %d in parts", plan.tile, plan.width);
        failed = launch_large<128, 128, MODE_STORE, float, true>(o, plan, sizes);       // (products that are cut have few tiles: the small ones)
    } else if (plan.tile == 256) failed = launch_large<256, 256, MODE, TO, false>(o, plan, to);
    else if (plan.tile == 192) failed = launch_large<192, 256, MODE, TO, false>(o, plan, to);
    else if (plan.width == 256) failed = launch_large<128, 256, MODE, TO, false>(o, plan, to);
    else failed = launch_large<128, 128, MODE, TO, false>(o, plan, to);
    if (failed) return failed;
    if (plan.parts > 1) {
        const long blocks = (long)((to.M + 15) / 16) * o.groups;
        int8_finish_kernel<MODE, TO><<<(unsigned)((blocks + 3) / 4), 256, 0, o.stream>>>(o.sums, plan.parts, o.groups, blocks, to);
    }
    XRT_LAUNCH_CHECK("linear_int8");
    return 0;
}

}  // namespace

// Whether row numbers, and a tile's rows behind the last, fit 32 bits, and the packed rows of w (two for an output of a gated matrix) 30.
static bool sizes_fit(int M, int N, int mode) { return (long)M + 256 < (1L << 31) && int8_groups(N, mode_of(mode) == MODE_GATED) * 16 < (1L << 30); }

extern "C" long xrt_linear_int8_workspace(int M, int N, int K, int mode) {
    if (M <= 0 || N <= 0 || K <= 0 || K > XRT_INT8_MOST_K || !sizes_fit(M, N, mode)) return 0;
    const long groups = int8_groups(N, mode_of(mode) == MODE_GATED);
    return sums_bytes(plan_of(M, groups, int8_stride(K)), M, groups);
}

extern "C" int xrt_linear_int8_plan(int M, int N, int K, int mode, int* plan) {
    XRT_REQUIRE(plan && M > 0 && N > 0 && K > 0 && K <= XRT_INT8_MOST_K && sizes_fit(M, N, mode), "linear_int8: bad sizes M=%d N=%d K=%d", M, N, K);
    const Plan chosen = plan_of(M, int8_groups(N, mode_of(mode) == MODE_GATED), int8_stride(K));
    plan[0] = chosen.tile, plan[1] = chosen.width, plan[2] = chosen.blocks, plan[3] = chosen.groups, plan[4] = chosen.parts;
    return 0;
}

// What a workgroup of such a product reads and which blocks of the result it makes, by the functions that the kernels call (int8_places.h).
extern "C" int xrt_linear_int8_reach(int M, int N, int K, int mode, long workgroup, long* reach, int* made, int room) {
    XRT_REQUIRE(reach && made && M > 0 && N > 0 && K > 0 && K <= XRT_INT8_MOST_K && sizes_fit(M, N, mode) && workgroup >= 0, "linear_int8: bad sizes M=%d N=%d K=%d", M, N, K);
    const long long_groups = int8_groups(N, mode_of(mode) == MODE_GATED);
    const Plan plan = plan_of(M, long_groups, int8_stride(K));
    const int groups = (int)long_groups, stride = (int)int8_stride(K), units = stride / XRT_INT8_STEP;
    const bool in_lds = plan.tile > 0, once = M <= 64, cut = plan.parts > 1;
    const int bm = plan.tile, bn = plan.width, height = in_lds ? even_height(M, bm) : plan.blocks * 16, wide = in_lds ? bn / 16 : plan.groups;
    const int tiles_m = (M + height - 1) / height, tiles_n = (groups + wide - 1) / wide;
    for (int i = 0; i < 10; ++i) reach[i] = i % 2 == 0 ? LONG_MAX : 0;
    reach[10] = part_ids((long)tiles_m * tiles_n, plan.parts, true);
    reach[11] = plan.parts;
    XRT_REQUIRE(workgroup < reach[10] && reach[10] < (1L << 31), "linear_int8: workgroup %ld of %ld", workgroup, reach[10]);
    auto reads = [&](int operand, long offset, long size) { reach[2 * operand] = std::min(reach[2 * operand], offset), reach[2 * operand + 1] = std::max(reach[2 * operand + 1], offset + size); };
    int count = 0;
    auto makes = [&](int part, int block, int group) {
        if (cut) reads(4, sums_place(part, M, block, groups, group) * (long)sizeof(int4v), XRT_WAVE * sizeof(int4v));
        if (count < room) made[3 * count] = part, made[3 * count + 1] = block, made[3 * count + 2] = group;
        ++count;
    };
    const PartPlace at = !in_lds ? few_place((int)workgroup, tiles_m, tiles_n, cut, plan.parts, once)
                         : cut   ? part_place((int)workgroup, 0, tiles_m, tiles_n, plan.parts)
                                 : PartPlace{tile_place((int)workgroup, tiles_m, tiles_n), 0};
    reach[12] = 0;
    reach[13] = 0;
    if (at.tile.m < 0) return 0;
    for (int wave = 0; wave < 8; ++wave) {
        const Share share = in_lds ? large_share(units, at.part, (units + plan.parts - 1) / plan.parts) : few_share(units, cut, at.part, plan.parts, wave, WAVES);
        XRT_REQUIRE(share.count >= (in_lds ? 1 : 0) && share.first + share.count <= units, "linear_int8: steps %d to %d of %d", share.first, share.first + share.count, units);
        if (wave == 0 || !in_lds) reach[12] += share.count;
        const LargeTile tile = in_lds ? large_tile(at.tile, bm, bn, height, M, wave) : LargeTile{};
        for (int lane = 0; lane < XRT_WAVE; ++lane) {
            for (int step : {0, share.count - 1}) {
                if (step < 0) continue;
                if (!in_lds) {
                    for (int half = 0; half < 2; ++half) {
                        for (int i = 0; i < plan.blocks; ++i) reads(0, few_a_offset(at.tile.m * plan.blocks + i, M, stride, share.first, lane) + (long)step * STEP_A + half * (STEP_A / 2), 16);
                        for (int g = 0; g < wide; ++g) reads(1, few_w_offset(at.tile.n * wide + g, groups, stride, share.first, lane) + (long)step * STEP_W + half * (STEP_W / 2), 16);
                    }
                    continue;
                }
                for (int h = 0; h < 2; ++h) {
                    for (int i = 0; i < (bm / 16 + 7) / 8; ++i)
                        reads(0, (long)tile.m0 * stride + (large_a_offset(tile, large_block(h, i, bm / 2, bm / 16, wave), bm, stride, lane) + (unsigned)(share.first + step) * (unsigned)STEP_A), 16);
                    for (int i = 0; i < bn / 128; ++i)
                        reads(1, (long)tile.first_group * 16 * stride + (large_w_offset(tile, large_block(h, i, bn / LARGE_WAVES_N, bn / 16, wave), groups, stride, lane) + (unsigned)(share.first + step) * (unsigned)STEP_W), 16);
                }
            }
            if (in_lds && !cut && wave < 4) {
                const ScalePlace scale = large_a_scale(tile, wave * 64 + lane, M);
                reads(2, scale.first * 4 + scale.offset, 4);
            } else if (in_lds && !cut && (wave - 4) * 64 < bn) {
                const ScalePlace scale = large_w_scale(tile, (wave - 4) * 64 + lane, groups);
                reads(3, scale.first * 4 + scale.offset, 4);
            }
        }
        if (!in_lds) continue;
        for (int row = tile.wave_row; row < large_row_end(tile); row += 16)
            for (int j = 0; j < bn / LARGE_WAVES_N / 16; ++j)
                if (tile.wave_group + j < groups) makes(at.part, row / 16, tile.wave_group + j);
    }
    if (!in_lds)
        for (int i = 0; i < plan.blocks; ++i)
            for (int g = 0; g < wide; ++g)
                if ((at.tile.m * plan.blocks + i) * 16 < M && at.tile.n * wide + g < groups) makes(at.part, at.tile.m * plan.blocks + i, at.tile.n * wide + g);
    reach[13] = count;
    return 0;
}

extern "C" int xrt_linear_int8(const void* a, const float* a_scales, const void* w, const float* w_scales, void* out, int out_dtype, int M, int N, int K,
                               int mode, void* workspace, long workspace_bytes, void* stream) {
    XRT_REQUIRE(M >= 0 && N > 0 && K > 0 && K <= XRT_INT8_MOST_K && (M == 0 || (a && a_scales && w && w_scales && out)), "linear_int8: bad operands M=%d N=%d K=%d", M, N, K);
    const int kind = mode_of(mode);
    XRT_REQUIRE(kind >= MODE_STORE && kind <= MODE_GATED && activation_of(mode) >= 0 && activation_of(mode) < XRT_ACT_COUNT && (kind == MODE_GATED || activation_of(mode) == 0),
                "linear_int8: unknown mode %d", mode);
    XRT_REQUIRE(out_dtype == XRT_F32 || (out_dtype == XRT_BF16 && kind != MODE_ACCUMULATE), "linear_int8: unknown element type %d of out for mode %d", out_dtype, mode);
    XRT_REQUIRE(((uintptr_t)a | (uintptr_t)w | (uintptr_t)w_scales) % 16 == 0, "linear_int8: rows, weights and their scales start at multiples of 16 bytes");
    if (M == 0) return 0;
    XRT_REQUIRE(sizes_fit(M, N, mode), "linear_int8: too many rows, %d of a and %d of w", M, N);
    const long groups = int8_groups(N, kind == MODE_GATED);
    const Plan plan = plan_of(M, groups, int8_stride(K));
    const long need = sums_bytes(plan, M, groups);
    XRT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), "linear_int8: a workspace of %ld bytes is needed, %ld given", need, workspace ? workspace_bytes : 0);
    const Operands o{(const signed char*)a, (const signed char*)w, (int4v*)workspace, (int)int8_stride(K), (int)groups, (hipStream_t)stream};
    if (out_dtype == XRT_BF16) {
        const Result<bf16> to{a_scales, w_scales, (bf16*)out, M, N, activation_of(mode)};
        return kind == MODE_GATED ? launch<MODE_GATED, bf16>(o, plan, to) : launch<MODE_STORE, bf16>(o, plan, to);
    }
    const Result<float> to{a_scales, w_scales, (float*)out, M, N, activation_of(mode)};
    return kind == MODE_GATED ? launch<MODE_GATED, float>(o, plan, to) : kind == MODE_ACCUMULATE ? launch<MODE_ACCUMULATE, float>(o, plan, to) : launch<MODE_STORE, float>(o, plan, to);
}
