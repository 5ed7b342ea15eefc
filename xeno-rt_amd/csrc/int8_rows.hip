// Rows in 8-bit integers (int8.h): made from float rows, by themselves or behind an RMSNorm that adds to the residual stream first, and turned back; weight
// matrices packed for the products.
//
//     scale = max_j |y_j| / 127          q_j = round(y_j / scale), halves to even
//
// in float32, the division the exact one: a value next to a border between two integers falls to the side where float32 arithmetic written down plainly has
// it. A row of zeros has scale 0. A row that holds an infinity or a NaN has scale NaN and zeros for values, so that whatever is made of it is NaN.
#include <algorithm>

#include "int8.h"
#include "xrt_hip.h"

namespace {

// Eight neighbouring elements of a row, asked for in whole pieces whatever the row's alignment (global loads need none beyond the element's).
template <typename T> struct Eight { T e[8]; };
template <typename T>
__device__ __forceinline__ void load_eight(const T* row, int at, int width, float (&v)[8]) {
    if (at + 8 <= width) {
        Eight<T> piece;
        __builtin_memcpy(&piece, row + at, sizeof(piece));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = to_float(piece.e[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = at + e < width ? to_float(row[at + e]) : 0.f;
    }
}
// The same on the way back. (16384 rows of 4096 normed, with the sums written: 148 us; 163 where the compiler was left to find the pieces in a copy of the array.)
template <typename T>
__device__ __forceinline__ void store_eight(T* row, int at, int width, const float (&v)[8]) {
    typedef unsigned Words __attribute__((ext_vector_type(4)));
    typedef Words Anywhere __attribute__((aligned(2)));                // (in memory: aligned as the smallest element is)
    Eight<T> piece;
#pragma unroll
    for (int e = 0; e < 8; ++e) piece.e[e] = from_float<T>(v[e]);
    if (at + 8 <= width) {
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
            Words part;
            __builtin_memcpy(&part, piece.e + h * (16 / sizeof(T)), 16);
            reinterpret_cast<Anywhere*>(row + at)[h] = part;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (at + e < width) row[at + e] = piece.e[e];
    }
}

// The bits of |v|: as whole numbers they are ordered as the magnitudes are, infinity above all numbers and NaN above infinity.
__device__ __forceinline__ unsigned magnitude_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

__device__ __forceinline__ unsigned wave_max_bits(unsigned v) {
#pragma unroll
    for (int offset = XRT_WAVE / 2; offset > 0; offset >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, offset, XRT_WAVE));
    return v;
}

// The largest of a block's magnitudes; every thread comes here and gets it. `scratch` holds 16 words that nothing else uses.
__device__ __forceinline__ unsigned block_max_bits(unsigned v, unsigned* scratch) {
    v = wave_max_bits(v);
    if (threadIdx.x % XRT_WAVE == 0) scratch[threadIdx.x / XRT_WAVE] = v;
    __syncthreads();
    unsigned most = scratch[0];
    for (int w = 1; w < (int)blockDim.x / XRT_WAVE; ++w) most = max(most, scratch[w]);
    return most;
}

__device__ __forceinline__ float scale_of(unsigned most) {
    return most >= 0x7f800000u ? __builtin_nanf("") : __builtin_bit_cast(float, most) / 127.0f;
}

// Eight values as signed bytes. The quotient by the scale's reciprocal, corrected by what is left of the value (exact, by a fused multiply-add), is the
// division's own result where neither leaves the normal numbers: four instructions instead of twelve. Adding 1.5 * 2^23 rounds it to an integer, halves to
// even, whose two's complement then stands in the sum's lowest bits.
__device__ __forceinline__ uint2 eight_bytes(const float (&y)[8], float scale) {
    unsigned word[2] = {0u, 0u};
    if (scale >= 0x1p-100f && scale <= 0x1p100f) {
        const float inverse = 1.0f / scale;
        unsigned bits[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float near = y[e] * inverse;
            bits[e] = __builtin_bit_cast(unsigned, fmaf(fmaf(-near, scale, y[e]), inverse, near) + 0x1.8p23f);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)                             // the lowest bytes of four words, side by side
            word[h] = __builtin_amdgcn_perm(bits[4 * h + 1], bits[4 * h], 0x0c0c0400u) | __builtin_amdgcn_perm(bits[4 * h + 3], bits[4 * h + 2], 0x04000c0cu);
    } else if (scale > 0.f) {                                   // (neither zero nor NaN; a scale that is no normal number is off by up to half of itself)
#pragma unroll
        for (int e = 0; e < 8; ++e) word[e / 4] |= ((unsigned)(int)fminf(fmaxf(rintf(y[e] / scale), -127.f), 127.f) & 255u) << (e % 4 * 8);
    }
    return make_uint2(word[0], word[1]);
}

constexpr int MOST_THREADS = 1024;

// One workgroup a row; PIECES: pieces of eight elements that a thread keeps in registers. NORM: the row of x gets delta added (written back) and is normed before
// it is brought to 8 bits. A row wider than what the threads keep is read again for what comes after the sums. Memory bounds it, so a row is read once where that
// can be had: its scale depends on all of it, and a workgroup holds it while two sums over its threads (the squares, the largest) are made.
template <typename TX, typename TD, typename TW, bool NORM, int PIECES>
__global__ void __launch_bounds__(MOST_THREADS) int8_rows_kernel(TX* x, const TD* delta, const TW* __restrict__ weight, const int* __restrict__ rows,
                                                                 signed char* __restrict__ values, float* __restrict__ scales, long x_stride,
                                                                 int x_rows, int width, int stride, float eps) {
    __shared__ float sums[32];
    __shared__ unsigned maxima[2][16];
    const long r = blockIdx.x;
    const long source = rows ? rows[r] : r;
    signed char* out = values + r * stride;
    if (source < 0 || source >= x_rows) {                       // (an index that names no row)
        for (int at = threadIdx.x * 8; at < stride; at += blockDim.x * 8) *reinterpret_cast<uint2*>(out + at) = make_uint2(0u, 0u);
        if (threadIdx.x == 0) scales[r] = __builtin_nanf("");
        return;
    }
    TX* row = x + source * x_stride;
    const TD* add = NORM && delta ? delta + source * width : nullptr;
    const int step = blockDim.x * 8, first = threadIdx.x * 8;
    constexpr bool EARLY = NORM && PIECES <= 2;                 // the gains are asked for now, so that they arrive under the sum
    float kept[PIECES][8], gains[EARLY ? PIECES : 1][8];
    float inv_rms = 1.f, power = 1.f;                           // (power: of two, that the row is multiplied by where its squares do not fit float32)
#pragma unroll
    for (int i = 0; i < PIECES; ++i) load_eight(row, first + i * step, width, kept[i]);
    if constexpr (EARLY)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) load_eight(weight, first + i * step, width, gains[i]);
    if constexpr (NORM) {
        auto added = [&](int at, float (&v)[8]) {
            if (!add || at >= width) return;
            float d[8];
            load_eight(add, at, width, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += d[e];
            store_eight(row, at, width, v);
        };
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            added(first + i * step, kept[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(kept[i][e], kept[i][e], sum);
        }
        for (int at = first + PIECES * step; at < width; at += step) {
            float v[8];
            load_eight(row, at, width, v);
            added(at, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
        }
        sum = block_sum(sum, sums);
        const float mean = sum / (float)width + eps;
        inv_rms = 1.0f / sqrtf(mean);
        if (__builtin_expect(!(sum < __builtin_inff()) || mean < 0x1p-100f, 0)) {      // (the same for all threads)
            // The squares overflow (elements of 2^64 / sqrt(width) and more) or vanish (eps is next to nothing). Of finite elements that are not all zero they are summed
            // again, of the row times a power of two: the quotient does not change by it.
            unsigned largest = 0u;
            auto each = [&](auto look) {                        // (the thread's elements that are not kept, as they lie in memory)
                for (int at = first + PIECES * step; at < width; at += step) {
                    float v[8];
                    load_eight(row, at, width, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) look(v[e]);
                }
            };
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) largest = max(largest, magnitude_bits(kept[i][e]));
            each([&](float v) { largest = max(largest, magnitude_bits(v)); });
            largest = block_max_bits(largest, maxima[1]);
            if (largest > 0u && largest < 0x7f800000u) {
                power = sum < 1.f ? 0x1p100f : 0x1p-80f;
                sum = 0.f;
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        kept[i][e] *= power;
                        sum = fmaf(kept[i][e], kept[i][e], sum);
                    }
                each([&](float v) { sum = fmaf(v * power, v * power, sum); });
                inv_rms = 1.0f / sqrtf(block_sum(sum, sums) / (float)width + eps * power * power);
            }
        }
    }
    // what is brought to 8 bits, of what the row holds (a thread reads again only what it wrote itself)
    auto times = [&](float (&v)[8], const float (&gain)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * inv_rms * gain[e];
    };
    auto finished = [&](int at, float (&v)[8]) {
        if constexpr (NORM) {
            float gain[8];
            load_eight(weight, at, width, gain);
            times(v, gain);
        }
    };
    auto finished_again = [&](int at, float (&v)[8]) {          // the same of a row read again, which lies in memory as it was
        if constexpr (NORM)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= power;
        finished(at, v);
    };
    unsigned most = 0u;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        if constexpr (EARLY) times(kept[i], gains[i]);
        else finished(first + i * step, kept[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max(most, magnitude_bits(kept[i][e]));
    }
    for (int at = first + PIECES * step; at < width; at += step) {
        float v[8];
        load_eight(row, at, width, v);
        finished_again(at, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max(most, magnitude_bits(v[e]));
    }
    const float scale = scale_of(block_max_bits(most, maxima[0]));
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
        if (first + i * step < stride) *reinterpret_cast<uint2*>(out + first + i * step) = eight_bytes(kept[i], scale);
    for (int at = first + PIECES * step; at < stride; at += step) {
        float v[8];
        load_eight(row, at, width, v);
        finished_again(at, v);
        *reinterpret_cast<uint2*>(out + at) = eight_bytes(v, scale);
    }
    if (threadIdx.x == 0) scales[r] = scale;
}

// out[m][j] = values[m][j] * scales[m]: `lanes` threads a row (a power of two up to 256), a thread eight neighbouring columns. (8192 rows of 14336 to
// bfloat16 63 us, 5.6 TB/s; 8 rows of 4096 2.3 us, an empty kernel 2.)
template <typename TO>
__global__ void __launch_bounds__(256) int8_values_kernel(const signed char* __restrict__ values, const float* __restrict__ scales, TO* __restrict__ out,
                                                          int rows, int width, int stride, int lanes, unsigned chunks) {
    const long r = (long)(blockIdx.x / chunks) * (256 / lanes) + threadIdx.x / lanes;
    const int at = ((int)(blockIdx.x % chunks) * lanes + (int)threadIdx.x % lanes) * 8;
    if (r >= rows || at >= width) return;
    const float scale = scales[r];
    const uint2 bytes = *reinterpret_cast<const uint2*>(values + r * stride + at);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)(int)(signed char)((e < 4 ? bytes.x : bytes.y) >> (e % 4 * 8)) * scale;
    store_eight(out + r * width, at, width, v);
}

// A thread a 16-byte piece of the packed matrix; the threads of the first tile of a group see to its scales.
__global__ void __launch_bounds__(256) int8_pack_kernel(const signed char* __restrict__ values, const float* __restrict__ scales,
                                                        signed char* __restrict__ packed, float* __restrict__ packed_scales, int n, int k, int stride,
                                                        long pieces, int gated) {
    const long id = (long)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= pieces) return;
    const int lane = (int)(id % XRT_WAVE), tiles = stride / 64;
    const long tile = id / XRT_WAVE, group = tile / tiles;
    const int within = lane % 16;
    long row = gated ? group * 8 + within % 8 : group * 16 + within;
    const bool there = row < n;
    if (gated && within >= 8) row += n;
    const long column = tile % tiles * 64 + lane / 16 * 16;
    unsigned piece[4] = {0u, 0u, 0u, 0u};
    if (there) {
        const uint4 read = *reinterpret_cast<const uint4*>(values + row * stride + column);
        piece[0] = read.x, piece[1] = read.y, piece[2] = read.z, piece[3] = read.w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                           // zeros behind the k columns, whatever stood there: what rows hold there then does not count
            const long left = (long)k - column - i * 4;
            if (left < 4) piece[i] = left <= 0 ? 0u : piece[i] & ((1u << (left * 8)) - 1u);
        }
    }
    *reinterpret_cast<uint4*>(packed + id * 16) = make_uint4(piece[0], piece[1], piece[2], piece[3]);
    if (tile % tiles == 0 && lane < 16) packed_scales[group * 16 + within] = there ? scales[row] : 0.f;
}

// Threads of a row's workgroup, where each keeps up to `most` pieces.
int threads_for(int stride, int most) { return whole_wavefronts(min(MOST_THREADS, (stride / 8 + most - 1) / most)); }

// Calls launch(first, count) for runs of rows whose workgroups of `threads` threads (of `together` rows each) fit a launch.
template <typename Launch>
void in_runs(int rows, int threads, int together, Launch launch) {
    const long most = (XRT_INT8_GRID_THREADS - 1) / threads * together;
    for (long first = 0; first < rows; first += most) launch(first, (int)std::min(most, rows - first));
}

}  // namespace

extern "C" long xrt_int8_stride(int k) { return int8_stride(k); }
extern "C" long xrt_int8_packed_rows(int n, int gated) { return int8_groups(n, gated != 0) * 16; }

extern "C" int xrt_quantize_int8(const void* x, int dtype, long x_stride, void* values, float* scales, int rows, int k, void* stream) {
    XRT_REQUIRE(rows >= 0 && k > 0 && k <= XRT_INT8_MOST_K && (rows == 0 || (x && values && scales)), "quantize_int8: bad operands rows=%d k=%d", rows, k);
    XRT_REQUIRE(dtype == XRT_F32 || dtype == XRT_BF16, "quantize_int8: unknown dtype %d", dtype);
    XRT_REQUIRE((uintptr_t)values % 16 == 0, "quantize_int8: values start at a multiple of 16 bytes");
    XRT_REQUIRE(x_stride >= k, "quantize_int8: rows of %d elements %ld apart", k, x_stride);
    if (rows == 0) return 0;
    const int stride = (int)int8_stride(k);
    hipStream_t s = (hipStream_t)stream;
#define XRT_ROWS8(TX, PIECES)                                                                                                                            \
    in_runs(rows, threads_for(stride, PIECES), 1, [&](long first, int count) {                                                                            \
        int8_rows_kernel<TX, float, float, false, PIECES><<<count, threads_for(stride, PIECES), 0, s>>>(                                                  \
            (TX*)x + first * x_stride, nullptr, nullptr, nullptr, (signed char*)values + first * stride, scales + first, x_stride, count, k, stride, 0.f); \
    })
    // two pieces a thread up to 8192 columns, four beyond: more of a wide row is then in flight (bfloat16, three matrices in turn, 8192 rows of 14336: 96 us with one, 70
    // with two, 65 with four, 71 with eight; 33 of 25600: 7.0, 5.0, 4.5 and 5.1; 2048 of 8192: 18.1, 10.8, 11.4 and 11.3; 8192 of 513: 8.8, 5.8, 6.8 and 10.3. float32: 113, 102, 109 and
    // 110; 6.5, 4.8, 4.4 and 4.6; 19.2, 13.9, 14.0 and 14.3; 9.0, 7.1, 8.0 and 11.3. Behind other kernels, which leave less of the last cache to it, the first takes 79 us, in float32 125.)
    if (dtype == XRT_F32 && stride <= 8192) XRT_ROWS8(float, 2);
    else if (dtype == XRT_F32) XRT_ROWS8(float, 4);
    else if (stride <= 8192) XRT_ROWS8(bf16, 2);
    else XRT_ROWS8(bf16, 4);
#undef XRT_ROWS8
    XRT_LAUNCH_CHECK("quantize_int8");
    return 0;
}

extern "C" int xrt_rmsnorm_int8(float* x, const void* delta, int delta_dtype, const void* weight, int weight_dtype, float eps, void* values, float* scales,
                                const int* rows, int n_rows, int x_rows, int hidden, void* stream) {
    XRT_REQUIRE(n_rows >= 0 && x_rows >= 0 && hidden > 0 && hidden <= XRT_INT8_MOST_K && (n_rows == 0 || ((x || x_rows == 0) && weight && values && scales)),
                "rmsnorm_int8: bad operands rows=%d hidden=%d", n_rows, hidden);
    XRT_REQUIRE((weight_dtype == XRT_F32 || weight_dtype == XRT_BF16) && (!delta || delta_dtype == XRT_F32 || delta_dtype == XRT_BF16),
                "rmsnorm_int8: unknown dtype weight=%d delta=%d", weight_dtype, delta_dtype);
    XRT_REQUIRE((uintptr_t)values % 16 == 0, "rmsnorm_int8: values start at a multiple of 16 bytes");
    XRT_REQUIRE(!delta || !rows, "rmsnorm_int8: chosen rows of x cannot be added to (one might be chosen twice)");
    XRT_REQUIRE(n_rows == 0 || rows || n_rows == x_rows, "rmsnorm_int8: %d rows of results for %d rows of x", n_rows, x_rows);
    if (n_rows == 0) return 0;
    const int stride = (int)int8_stride(hidden);
    hipStream_t s = (hipStream_t)stream;
#define XRT_NORM8(TD, TW, PIECES)                                                                                                                           \
    in_runs(n_rows, threads_for(stride, PIECES), 1, [&](long first, int count) {                                                                            \
        int8_rows_kernel<float, TD, TW, true, PIECES><<<count, threads_for(stride, PIECES), 0, s>>>(                                                        \
            rows ? x : x + first * hidden, delta ? (const TD*)delta + first * hidden : nullptr, (const TW*)weight, rows ? rows + first : nullptr,           \
            (signed char*)values + first * stride, scales + first, hidden, rows ? x_rows : count, hidden, stride, eps);                                     \
    })
#define XRT_NORM8_OF(PIECES)                                                                      \
    do {                                                                                          \
        if (delta_dtype == XRT_BF16 && weight_dtype == XRT_BF16) XRT_NORM8(bf16, bf16, PIECES);   \
        else if (delta_dtype == XRT_BF16) XRT_NORM8(bf16, float, PIECES);                         \
        else if (weight_dtype == XRT_BF16) XRT_NORM8(float, bf16, PIECES);                        \
        else XRT_NORM8(float, float, PIECES);                                                     \
    } while (0)
    // two pieces a thread, with the gains in registers ahead of the sum (8 rows of 4096 4.3 us, 4.7 with one piece, 5.0 with four and the gains fetched behind
    // the sum; 333 of 5120 7.2, 8.9 and 7.9; 1001 of 2049 8.1, 9.8 and 8.8; 16384 of 4096 148 us, 148 and 154: 5.0 TB/s, the rate of a copy)
    if (stride <= 2 * 8 * MOST_THREADS) XRT_NORM8_OF(2);
    else XRT_NORM8_OF(4);
#undef XRT_NORM8_OF
#undef XRT_NORM8
    XRT_LAUNCH_CHECK("rmsnorm_int8");
    return 0;
}

extern "C" int xrt_dequantize_int8(const void* values, const float* scales, void* out, int out_dtype, int rows, int k, void* stream) {
    XRT_REQUIRE(rows >= 0 && k > 0 && k <= XRT_INT8_MOST_K && (rows == 0 || (values && scales && out)), "dequantize_int8: bad operands rows=%d k=%d", rows, k);
    XRT_REQUIRE(out_dtype == XRT_F32 || out_dtype == XRT_BF16, "dequantize_int8: unknown dtype %d", out_dtype);
    XRT_REQUIRE((uintptr_t)values % 16 == 0, "dequantize_int8: values start at a multiple of 16 bytes");
    if (rows == 0) return 0;
    int lanes = 8;
    while (lanes < 256 && lanes * 8 < k) lanes *= 2;
    const int chunks = (k + lanes * 8 - 1) / (lanes * 8), together = 256 / lanes, stride = (int)int8_stride(k);
    hipStream_t s = (hipStream_t)stream;
#define XRT_VALUES8(TO)                                                                                                                                    \
    in_runs(rows, 256 * chunks, together, [&](long first, int count) {                                                                                     \
        int8_values_kernel<TO><<<(unsigned)((count + together - 1) / together * (long)chunks), 256, 0, s>>>(                                               \
            (const signed char*)values + first * stride, scales + first, (TO*)out + first * k, count, k, stride, lanes, (unsigned)chunks);                 \
    })
    if (out_dtype == XRT_F32) XRT_VALUES8(float);
    else XRT_VALUES8(bf16);
#undef XRT_VALUES8
    XRT_LAUNCH_CHECK("dequantize_int8");
    return 0;
}

extern "C" int xrt_pack_int8(const void* values, const float* scales, void* packed, float* packed_scales, int n, int k, int gated, void* stream) {
    XRT_REQUIRE(values && scales && packed && packed_scales && n > 0 && k > 0 && k <= XRT_INT8_MOST_K, "pack_int8: bad operands n=%d k=%d", n, k);
    XRT_REQUIRE(((uintptr_t)values | (uintptr_t)packed) % 16 == 0, "pack_int8: values start at a multiple of 16 bytes");
    const long pieces = int8_groups(n, gated != 0) * int8_stride(k);             // 16 rows of stride bytes, 16 bytes a piece
    const long blocks = (pieces + 255) / 256;
    XRT_REQUIRE(blocks * 256 < XRT_INT8_GRID_THREADS, "pack_int8: too many elements, %d rows of %d columns", n, k);
    int8_pack_kernel<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>((const signed char*)values, scales, (signed char*)packed, packed_scales, n, k,
                                                                        (int)int8_stride(k), pieces, gated != 0);
    XRT_LAUNCH_CHECK("pack_int8");
    return 0;
}
