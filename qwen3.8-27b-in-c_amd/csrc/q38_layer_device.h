/* Device helpers of a decoder layer's operators: elements of three types, and
 * blocks of 128 values into e4m3 codes with a scale byte. */
#pragma once

#include "q38_device.h"
#include "q38_layer.h"

namespace q38 {

typedef uint32_t layer_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t layer_u32x2 __attribute__((ext_vector_type(2)));

/* N neighbours at any place of an element: the compiler makes wide accesses of it,
 * which this target takes at any address */
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) LayerSome {
    T e[N];
};

/* Eight neighbouring elements, or `some` of them.  Whole: 16-byte aligned and all there.
 * Otherwise only a row's end goes element by element (939 bf16 rows of 13396 into 8
 * bits: 23 us, 67 us if all do). */
template <typename T, bool kWhole>
__device__ __forceinline__ void layer_load8(float v[8], const T *from, uint32_t some)
{
    if constexpr (kWhole) {
        constexpr int kWords = sizeof(T) * 8 / 16;
        layer_u32x4 raw[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[i] = reinterpret_cast<const layer_u32x4 *>(from)[i];
        const T *e = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(e[i]);
    } else if (some == 8) {
        const LayerSome<T, 8> raw = *reinterpret_cast<const LayerSome<T, 8> *>(from);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(raw.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (uint32_t)i < some ? static_cast<float>(from[i]) : 0.0f;
    }
}

template <typename T, bool kWhole>
__device__ __forceinline__ void layer_store8(T *to, const float v[8], uint32_t some)
{
    if constexpr (kWhole) {
        constexpr int kWords = sizeof(T) * 8 / 16;
        layer_u32x4 raw[kWords];
        T *e = reinterpret_cast<T *>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = static_cast<T>(v[i]);
#pragma unroll
        for (int i = 0; i < kWords; ++i) reinterpret_cast<layer_u32x4 *>(to)[i] = raw[i];
    } else if (some == 8) {
        LayerSome<T, 8> raw;
#pragma unroll
        for (int i = 0; i < 8; ++i) raw.e[i] = static_cast<T>(v[i]);
        *reinterpret_cast<LayerSome<T, 8> *>(to) = raw;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((uint32_t)i < some) to[i] = static_cast<T>(v[i]);
    }
}

/* largest word of each 16 neighbouring lanes, in all of them; every lane is active */
__device__ __forceinline__ uint32_t row16_max(uint32_t v)
{
    v = max(v, (uint32_t)dpp_move<0xB1>(0, (int)v));
    v = max(v, (uint32_t)dpp_move<0x4E>(0, (int)v));
    v = max(v, (uint32_t)dpp_move<0x141>(0, (int)v));
    return max(v, (uint32_t)dpp_move<0x140>(0, (int)v));
}

/* The scale byte of a block whose largest magnitude has these bits: k + 127, k
 * >= -100 the least with it <= 448 * 2^k (448 = 1.75 * 2^8); 255 where it is
 * not finite (as integers, the bits of NaN and infinity are above all others). */
__device__ __forceinline__ uint32_t e4m3_scale_byte(uint32_t largest)
{
    if (largest >= 0x7f800000u) return 255u;
    const int e = (int)(largest >> 23) - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)max(e, 127 - 100);
}

/* Eight neighbours of a block into codes; the block's other values are with the
 * other 15 lanes of the same 16, which all call this.  Returns the scale byte.
 * The division by a power of two is exact but for values that fall below a
 * code's smallest step by far, and v_cvt_pk_fp8_f32 rounds once, ties to even. */
__device__ __forceinline__ uint32_t e4m3_encode8(layer_u32x2 &codes, const float v[8])
{
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max(largest, __float_as_uint(v[i]) & 0x7fffffffu);
    const uint32_t byte = e4m3_scale_byte(row16_max(largest));
    const float inverse = __uint_as_float((254u - min(byte, 253u)) << 23);
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = v[i] * inverse;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(u[4 * i], u[4 * i + 1], 0, false);
        word = __builtin_amdgcn_cvt_pk_fp8_f32(u[4 * i + 2], u[4 * i + 3], word, true);
        codes[i] = byte == 255u ? 0x7f7f7f7fu : (uint32_t)word;
    }
    return byte;
}

template <bool kWhole>
__device__ __forceinline__ void e4m3_store8(uint8_t *to, layer_u32x2 codes, uint32_t some)
{
    if constexpr (kWhole) {
        *reinterpret_cast<layer_u32x2 *>(to) = codes;
    } else if (some == 8) {
        *reinterpret_cast<LayerSome<uint8_t, 8> *>(to) = __builtin_bit_cast(LayerSome<uint8_t, 8>, codes);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((uint32_t)i < some) to[i] = (uint8_t)(codes[i / 4] >> 8 * (i % 4));
    }
}

/* the scale byte of block `block` of a row, and zeros behind the row's last */
__device__ __forceinline__ void e4m3_store_scale(uint8_t *row, uint32_t block, uint32_t byte, uint32_t blocks, uint32_t pitch)
{
    row[block] = (uint8_t)byte;
    if (block == blocks - 1)
        for (uint32_t i = blocks; i < pitch; ++i) row[i] = 0;
}

}  // namespace q38
