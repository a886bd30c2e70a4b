/* Rows in 8 bits times a matrix in e4m3 (q38hip_gemm_e4m3).
 *
 * Per output, the products of a block of 128 inputs are summed by the matrix
 * unit, 16 matrix rows by 16 tokens, with the tokens' powers of two applied to
 * its operands, and the matrix block's fp32 scale joins the result to the
 * running sum by one fma.  Lane i holds 32 codes of row (token) i % 16: 16
 * neighbours from 16 (i / 16) on and 16 from 64 + 16 (i / 16) on, in both operands
 * alike, so every load is a whole 64 bytes of a row.
 *
 * 16-bit outputs: one v_mfma_scale_f32_16x16x128_f8f6f4.  The unit adds products
 * of e4m3 codes at 13 bits below the largest of a group (measured with 2^8 -
 * 2^8 + t: t is kept down to 2^-5): 1.5e-5 to 3e-5 of the result's norm, a
 * hundredth of a bf16 output's rounding and a tenth of an fp16 output's.
 * fp32 outputs would keep that error, so for them codes become bf16 values
 * (exactly; four significant bits, the token's power of two in their exponent)
 * and four v_mfma_f32_16x16x32_bf16 sum their products with all 24 bits, at
 * half the rate. */
#include <type_traits>

#include "q38_kernels.h"
#include "q38_layer_device.h"

namespace q38 {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kWaves = 8;

__device__ __forceinline__ i32x8 both(i32x4 low, i32x4 high)
{
    return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
}

/* eight codes as bf16 times a power of two */
__device__ __forceinline__ bf16x8 decoded(int low, int high, float scale)
{
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, scale, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, scale, true);
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1,
                                   2, 3, 4, 5, 6, 7);
}

/* sum + factor * the products of a block: element r is matrix row 4 (lane / 16) +
 * r, token lane % 16.  `scale` is the token's scale byte. */
template <bool kExact>
__device__ __forceinline__ f32x4 add_block(f32x4 sum, i32x8 matrix, i32x8 token, uint32_t scale, float factor)
{
    f32x4 p = {};
    if constexpr (kExact) {
        const float power = __uint_as_float(scale << 23);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(decoded(matrix[2 * q], matrix[2 * q + 1], 1.0f),
                                                        decoded(token[2 * q], token[2 * q + 1], power), p, 0, 0, 0);
        factor = scale == 255u ? __uint_as_float(0x7fc00000u) : factor;
    } else {
        /* the scale of the matrix operand is 1 (127) */
        p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(matrix, token, p, 0, 0, 0, 127, 0, (int)scale);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[r] = fmaf(p[r], factor, sum[r]);
    return sum;
}

template <typename T>
__device__ __forceinline__ void store_output(const ProductE4M3 &a, uint32_t token, uint32_t row, float v)
{
    static_cast<T *>(a.output)[(uint64_t)token * a.output_row + row] = static_cast<T>(v);
}

/* 16 matrix rows by 16 * M tokens to a workgroup, whose eight wavefronts take
 * every eighth block of inputs and are summed in LDS in their order. */
template <typename T, int M>
__global__ void __launch_bounds__(kWaves * 64) few_kernel(ProductE4M3 a)
{
    __shared__ float sums[kWaves][M * 4][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t row0 = blockIdx.x * 16, token0 = blockIdx.y * (16 * M);
    const uint8_t *matrix = a.weight + (uint64_t)min(row0 + lane % 16, a.outputs - 1) * a.inputs;
    const uint8_t *codes[M], *scales[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        const uint64_t token = min(token0 + m * 16 + lane % 16, a.tokens - 1);
        codes[m] = a.codes + token * a.inputs;
        scales[m] = a.scales + token * a.pitch;
    }
    const float *weight_scales = a.weight_scales + (uint64_t)(row0 / kE4M3Block) * a.blocks;
    f32x4 sum[M] = {};
    for (uint32_t b = wave; b < a.blocks; b += kWaves) {
        const uint32_t at = b * kE4M3Block + lane / 16 * 16;
        const bool low = at < a.inputs, high = at + 64 < a.inputs;
        const auto load = [&](const uint8_t *row) {
            const i32x4 l = low ? *reinterpret_cast<const i32x4 *>(row + at) : i32x4{};
            const i32x4 h = high ? *reinterpret_cast<const i32x4 *>(row + at + 64) : i32x4{};
            return both(l, h);
        };
        const i32x8 w = load(matrix);
        const float s = weight_scales[b];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            sum[m] = add_block<std::is_same_v<T, float>>(sum[m], w, load(codes[m]), scales[m][b], s);
        }
    }
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[wave][m * 4 + r][lane] = sum[m][r];
    __syncthreads();
    /* output i of 256 M: token i / 16, matrix row i % 16 */
    for (uint32_t i = threadIdx.x; i < 256 * M; i += kWaves * 64) {
        const uint32_t r = i % 16, t = i / 16;
        float v = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) v += sums[w][t / 16 * 4 + r % 4][r / 4 * 16 + t % 16];
        if (token0 + t < a.tokens && row0 + r < a.outputs) store_output<T>(a, token0 + t, row0 + r, v);
    }
}

template <typename T>
bool product(const ProductE4M3 &a, hipStream_t stream)
{
    const uint32_t tiles = layer_up(a.outputs, 16);
    const int m = a.tokens <= 16 ? 1 : a.tokens <= 32 ? 2 : 4;
    const dim3 grid(tiles, layer_up(a.tokens, 16 * m));
    const auto kernel = m == 1 ? few_kernel<T, 1> : m == 2 ? few_kernel<T, 2> : few_kernel<T, 4>;
    return launch_kernel(kernel, grid, dim3(kWaves * 64), stream, a);
}

}  // namespace

uint64_t product_e4m3_workspace_bytes(uint32_t, uint64_t, uint32_t) { return 0; }

bool launch_product_e4m3(const ProductE4M3 &a, hipStream_t stream)
{
    return a.type == kLayerF32 ? product<float>(a, stream) : a.type == kLayerF16 ? product<_Float16>(a, stream)
                                                                                 : product<__bf16>(a, stream);
}

}  // namespace q38
