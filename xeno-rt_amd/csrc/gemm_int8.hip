// Products of rows and weights in 8-bit integers (int8.h), on the matrix cores:
//
//     out[m, n] (+)= float(sum_j a[m, j] * w[n, j]) * a_scales[m] * w_scales[n]
//
// The sum is exact: whole numbers of 32 bits (k is limited so that it cannot overflow). Every kernel here therefore gives the same bits for a row of a,
// however many other rows there are and however k is cut. It is rounded to float32 once, then multiplied by the row's and by the channel's scale.
#include "int8.h"
#include "activation.h"
#include "xrt_hip.h"

namespace {

typedef int int4v __attribute__((ext_vector_type(4)));
enum { MODE_STORE = 0, MODE_ACCUMULATE = 1, MODE_GATED = 2 };

// One value of the result; `before` is what out holds.
__device__ __forceinline__ float scaled(int sum, float a_scale, float w_scale) { return (float)sum * a_scale * w_scale; }

// The simple one: a wavefront has 16 packed rows of w and 64 rows of a, and loads its operands from global memory.
template <int MODE, typename TO>
__global__ void __launch_bounds__(256) gemm_int8_kernel(const signed char* __restrict__ a, const float* __restrict__ a_scales,
                                                        const signed char* __restrict__ w, const float* __restrict__ w_scales, TO* __restrict__ out,
                                                        int M, int N, int stride, int groups, int activation) {
    const int lane = threadIdx.x % XRT_WAVE, wave = threadIdx.x / XRT_WAVE;
    const int group = blockIdx.x * 4 + wave;
    if (group >= groups) return;
    const int r = lane % 16, c = lane / 16;
    const long m0 = (long)blockIdx.y * 64;
    const signed char* w_at = w + (long)group * 16 * stride + lane * 16;
    const signed char* a_at[4];
    int4v sum[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long m = m0 + i * 16 + r;
        a_at[i] = a + (m < M ? m : (long)M - 1) * stride + c * 16;
        sum[i] = int4v{0, 0, 0, 0};
    }
    for (int k = 0; k < stride; k += 64) {
        const int4v wk = *reinterpret_cast<const int4v*>(w_at + (long)k * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wk, *reinterpret_cast<const int4v*>(a_at[i] + k), sum[i], 0, 0, 0);
    }
    // element e of sum[i]: row m0 + i * 16 + r of a, packed row group * 16 + c * 4 + e of w
    float w_scale[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w_scale[e] = w_scales[group * 16 + c * 4 + e];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long m = m0 + i * 16 + r;
        const float a_scale = a_scales[m < M ? m : (long)M - 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float value = scaled(sum[i][e], a_scale, w_scale[e]);
            long n = (long)group * 16 + c * 4 + e;
            bool mine = m < M;
            if constexpr (MODE == MODE_GATED) {
                const float up = of_other_half(value);
                value = gate_activation<sizeof(TO) == 2>(value, activation) * up;
                n = (long)group * 8 + c * 4 + e;
                mine = mine && c < 2;
            }
            if (mine && n < N) {
                TO* to = out + m * N + n;
                if constexpr (MODE == MODE_ACCUMULATE) value += to_float(*to);
                *to = from_float<TO>(value);
            }
        }
    }
}

}  // namespace

extern "C" long xrt_linear_int8_workspace(int M, int N, int K, int mode) { return 0; }

extern "C" int xrt_linear_int8(const void* a, const float* a_scales, const void* w, const float* w_scales, void* out, int out_dtype, int M, int N, int K,
                               int mode, void* workspace, long workspace_bytes, void* stream) {
    XRT_REQUIRE(M >= 0 && N > 0 && K > 0 && K <= XRT_INT8_MOST_K && (M == 0 || (a && a_scales && w && w_scales && out)), "linear_int8: bad operands M=%d N=%d K=%d", M, N, K);
    XRT_REQUIRE(mode_of(mode) >= MODE_STORE && mode_of(mode) <= MODE_GATED && activation_of(mode) < XRT_ACT_COUNT && (mode_of(mode) == MODE_GATED || activation_of(mode) == 0),
                "linear_int8: unknown mode %d", mode);
    XRT_REQUIRE(out_dtype == XRT_F32 || (out_dtype == XRT_BF16 && mode_of(mode) != MODE_ACCUMULATE), "linear_int8: unknown element type %d of out for mode %d", out_dtype, mode);
    if (M == 0) return 0;
    const bool gated = mode_of(mode) == MODE_GATED;
    const int stride = (int)int8_stride(K), groups = (int)int8_groups(N, gated);
    XRT_REQUIRE((M + 63) / 64 <= XRT_GRID_ROWS, "linear_int8: too many rows, %d", M);
    const dim3 grid((groups + 3) / 4, (M + 63) / 64);
    hipStream_t s = (hipStream_t)stream;
#define XRT_INT8(MODE, TO) gemm_int8_kernel<MODE, TO><<<grid, 256, 0, s>>>((const signed char*)a, a_scales, (const signed char*)w, w_scales, (TO*)out, M, N, stride, groups, activation_of(mode))
    if (gated && out_dtype == XRT_F32) XRT_INT8(MODE_GATED, float);
    else if (gated) XRT_INT8(MODE_GATED, bf16);
    else if (mode_of(mode) == MODE_ACCUMULATE) XRT_INT8(MODE_ACCUMULATE, float);
    else if (out_dtype == XRT_F32) XRT_INT8(MODE_STORE, float);
    else XRT_INT8(MODE_STORE, bf16);
#undef XRT_INT8
    XRT_LAUNCH_CHECK("linear_int8");
    return 0;
}
