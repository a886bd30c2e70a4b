/* Rows of keys and values into the pages of the 8-bit cache.
 *
 * Per page, head and half (keys, values): with a the largest magnitude among
 * the page's new tokens, k the least exponent with a <= M 2^k (M = 127, or 448
 * for e4m3), the page's scale becomes 2^k where it holds no older token, else
 * the larger of 2^k and what it was; older codes follow a scale that grew, and
 * a new code is x / scale rounded to nearest, ties to even.  The scales are
 * powers of two, so the quotient is exact and every code is one rounding; an
 * e4m3 page that grows loses nothing but what falls below the type's smallest
 * values, an int8 page a rounding of its older codes per doubling.  A value
 * that is not finite makes the scale NaN, and the page reads as NaN until its
 * first token is written again.
 *
 * One workgroup per (page touched, head, half): no other writes there.  Keys
 * are [token][channel] and go out as they come; values are [channel][token],
 * so theirs turn in LDS and whole dwords of tokens go out. */
#include "q38_kernels.h"
#include "q38_device.h"
#include "q38_kv.h"

namespace q38 {

namespace {

constexpr int kThreads = 256;

struct KVAppend {
    Q38KVPages cache;     /* data and scales moved to the layer */
    KVRows rows;
    const void *key, *value;
    uint64_t row_stride;
    bool vector;          /* rows are aligned to four elements */
};

template <int TYPE>
__device__ __forceinline__ void load4(float *x, const void *base, uint64_t at, bool vector)
{
    if constexpr (TYPE == kElementF32) {
        const float *p = static_cast<const float *>(base) + at;
        if (vector) {
            const float4 v = *reinterpret_cast<const float4 *>(p);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
            for (int e = 0; e < 4; ++e) x[e] = p[e];
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(base) + at;
        uint16_t bits[4];
        if (vector) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            bits[0] = v.x & 0xffff, bits[1] = v.x >> 16, bits[2] = v.y & 0xffff, bits[3] = v.y >> 16;
        } else {
            for (int e = 0; e < 4; ++e) bits[e] = p[e];
        }
        for (int e = 0; e < 4; ++e)
            x[e] = TYPE == kElementF16 ? f16_to_f32(bits[e]) : __uint_as_float((uint32_t)bits[e] << 16);
    }
}

/* the code of v, |v| <= 127 or 448 */
template <bool E4M3>
__device__ __forceinline__ uint32_t encode(float v)
{
    if constexpr (E4M3) return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v, 0.0f, 0, false) & 0xffu;
    else return (uint32_t)(int)__builtin_rintf(v) & 0xffu;
}
template <bool E4M3>
__device__ __forceinline__ float decode(uint32_t code)
{
    if constexpr (E4M3) return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
    else return (float)(int8_t)code;
}

template <bool E4M3, int TYPE>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KVAppend a)
{
    extern __shared__ uint8_t turned[];       /* values: [channel][T + 4] codes */
    __shared__ uint32_t wave_largest[kThreads / 64];
    const uint32_t T = a.cache.page_tokens, D = a.cache.head_dim;
    const uint32_t slot = blockIdx.x, half = blockIdx.y & 1, head = blockIdx.y >> 1;
    const int i = kv_find_sequence(a.rows, slot, 1, T, 2);
    if (i < 0) return;
    const uint32_t begin = kv_row_start(a.rows, i), end = kv_row_start(a.rows, i + 1);
    if (end <= begin) return;
    const int32_t sequence = a.rows.sequences[i];
    const uint32_t tokens = kv_tokens(a.cache, sequence);
    /* rows that lie before the sequence's first token are left out */
    const uint32_t rows = min(end - begin, tokens), first = tokens - rows;
    const uint32_t entry = first / T + (slot - kv_slot_base(begin, i, 1, T, 2));
    if (!rows || entry * T >= tokens) return;
    const int32_t page = kv_page(a.cache, sequence, entry);
    if (page < 0) {
        if (threadIdx.x == 0) atomicOr(a.cache.status, Q38_KV_BAD_PAGE);
        return;
    }
    const uint32_t from = max(first, entry * T) - entry * T, to = min(tokens, entry * T + T) - entry * T;
    const uint32_t count = to - from;
    const void *source = half ? a.value : a.key;
    /* element of new token 0, channel 0 */
    const uint64_t origin = (uint64_t)(end - tokens + entry * T + from) * a.row_stride + (uint64_t)head * D;
    const uint64_t block = kv_block(a.cache, page, half, head);
    uint8_t *codes = a.cache.data + block * (T * D);
    const uint32_t quads = D / 4;

    uint32_t largest = 0;
    for (uint32_t at = threadIdx.x; at < count * quads; at += kThreads) {
        float x[4];
        load4<TYPE>(x, source, origin + (at / quads) * a.row_stride + at % quads * 4, a.vector);
        for (int e = 0; e < 4; ++e) largest = max(largest, __float_as_uint(x[e]) & 0x7fffffffu);
    }
    for (int by = 1; by < 64; by *= 2) largest = max(largest, (uint32_t)__shfl_xor((int)largest, by));
    if ((threadIdx.x & 63) == 0) wave_largest[threadIdx.x >> 6] = largest;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) largest = max(largest, wave_largest[w]);

    const bool finite = largest < 0x7f800000u;
    const float was = from ? a.cache.scales[block] : 0.0f;
    float scale = finite ? __uint_as_float((uint32_t)(kv_scale_exponent(largest, E4M3) + 127) << 23) : NAN;
    if (!(was <= scale) && finite) scale = was;        /* the larger, or an older NaN */
    __syncthreads();                                   /* every thread has read the old scale */
    if (threadIdx.x == 0) a.cache.scales[block] = scale;
    if (from && scale > was) {
        const float shrink = was / scale;
        for (uint32_t at = threadIdx.x; at < from * D; at += kThreads) {
            uint8_t *code = codes + (half ? at / from * T + at % from : at);
            *code = (uint8_t)encode<E4M3>(decode<E4M3>(*code) * shrink);
        }
    }
    const bool usable = scale == scale;
    const float inverse = usable ? 1.0f / scale : 0.0f;
    const bool turn = half && count >= 4;
    const uint32_t pitch = T + 4;
    for (uint32_t at = threadIdx.x; at < count * quads; at += kThreads) {
        const uint32_t t = at / quads, d = at % quads * 4;
        float x[4];
        load4<TYPE>(x, source, origin + t * a.row_stride + d, a.vector);
        uint32_t code[4];
        for (int e = 0; e < 4; ++e) code[e] = usable ? encode<E4M3>(x[e] * inverse) : 0u;
        if (!half)
            *reinterpret_cast<uint32_t *>(codes + (from + t) * D + d) = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
        else if (turn)
            for (int e = 0; e < 4; ++e) turned[(d + e) * pitch + from + t] = (uint8_t)code[e];
        else
            for (int e = 0; e < 4; ++e) codes[(d + e) * T + from + t] = (uint8_t)code[e];
    }
    if (!turn) return;
    __syncthreads();
    const uint32_t words = T / 4;
    for (uint32_t at = threadIdx.x; at < D * words; at += kThreads) {
        const uint32_t d = at / words, t = at % words * 4;
        if (t >= from && t + 4 <= to)
            *reinterpret_cast<uint32_t *>(codes + d * T + t) = *reinterpret_cast<const uint32_t *>(turned + d * pitch + t);
        else
            for (uint32_t e = t; e < t + 4; ++e)
                if (e >= from && e < to) codes[d * T + e] = turned[d * pitch + e];
    }
}

template <bool E4M3, int TYPE>
bool launch_typed(const KVAppend &a, uint32_t slots, hipStream_t stream)
{
    KVAppend call = a;
    void *arguments[] = {&call};
    const uint32_t lds = a.cache.head_dim * (a.cache.page_tokens + 4);
    return hipLaunchKernel(reinterpret_cast<const void *>(kv_append_kernel<E4M3, TYPE>),
                           dim3(slots, 2 * a.cache.kv_heads), dim3(kThreads), arguments, lds, stream) == hipSuccess;
}
template <bool E4M3>
bool launch_kind(const KVAppend &a, int type, uint32_t slots, hipStream_t stream)
{
    return type == kElementF32   ? launch_typed<E4M3, kElementF32>(a, slots, stream)
           : type == kElementF16 ? launch_typed<E4M3, kElementF16>(a, slots, stream)
                                 : launch_typed<E4M3, kElementBF16>(a, slots, stream);
}

}  // namespace

bool launch_kv_append(const Q38KVPages &cache, uint32_t layer, const void *key, const void *value, int type,
                      uint64_t row_stride, const KVRows &rows, hipStream_t stream)
{
    KVAppend a{cache, rows, key, value, row_stride, false};
    a.cache.data += (uint64_t)layer * cache.pages * kv_page_bytes(cache);
    a.cache.scales += (uint64_t)layer * cache.pages * 2 * cache.kv_heads;
    const uintptr_t step = type == kElementF32 ? 4 : 2;
    a.vector = row_stride % 4 == 0 && ((uintptr_t)key | (uintptr_t)value) % (4 * step) == 0;
    const uint32_t slots = (uint32_t)kv_slots(rows.total_rows, rows.count, 1, cache.page_tokens, 2);
    return cache.type == Q38_KV_E4M3 ? launch_kind<true>(a, type, slots, stream)
                                     : launch_kind<false>(a, type, slots, stream);
}

}  // namespace q38
