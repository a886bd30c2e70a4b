/* Attention over the paged 8-bit cache: the kernel template of one head
 * width (instantiated by q38_kv_attention{64,128,256}.hip).
 *
 * For a column (a row of the call times a query head of the key/value head's
 * group), with codes c, key scale sk and value scale sv of a token's page:
 *     u_t = log2(e) scale sk (q . ck_t) + log2 sv
 *     w_t = 2^(u_t - m),  O = sum w_t cv_t,  l = sum w_t / sv,  out = O / l
 * over the tokens the row sees; m follows the largest u.  The value scale, a
 * power of two, rides in the exponent, so a weight needs no multiplication
 * and stays in a range that fp16 holds for pages of any size of values.
 *
 * Everything stays transposed: S^T = K Q^T and O^T = V^T W^T, on
 * v_mfma_f32_16x16x32_f16.  Lane (n = lane & 15, g = lane >> 4) holds column
 * n in the results of both, so maximum, sum and rescaling are the lane's own
 * (one exchange over g for the maximum).  Row m of the i-th of four key tiles
 * is token 16 (m / 4) + 4 i + m % 4 of a 64-token step: lane g then has the
 * scores of tokens 16 g .. 16 g + 15, which are both its slice of the second
 * product and 16 consecutive bytes of a value channel.  Keys and values come
 * straight from memory as 16-byte loads, in the order the products use them:
 * no LDS and no exchange in the loop.
 *
 * 8-bit codes are exact in fp16, and so is a 16-bit query once its row is
 * scaled by a power of two to a maximum of 2^13..2^14.  For fp32 calls
 * (SPLIT) a column takes two lanes: n < 8 works with the fp16 value of its
 * queries and weights, n + 8 with what that leaves, 22 bits together.  16-bit
 * calls keep the fp16 weight alone: its error, 2^-12 of the weight, is an
 * eighth of a bf16 output's own rounding and, over many tokens, below an
 * fp16 output's. */
#pragma once

#include "q38_device.h"
#include "q38_kv.h"

namespace q38 {

using kv_half2 = _Float16 __attribute__((ext_vector_type(2)));
using kv_half8 = _Float16 __attribute__((ext_vector_type(8)));
using kv_float4 = float __attribute__((ext_vector_type(4)));

constexpr int kKVStep = 64;               /* tokens of a step */
/* exponent of the largest weight, and how far a column's maximum may be
 * passed before its sums are rescaled: weights stay below 2^15 (fp16 holds
 * 2^16) and one 2^20 below the largest is still a normal fp16 value */
constexpr float kKVWeightExponent = 6.0f;
constexpr float kKVMaximumSlack = 8.0f;

__device__ __forceinline__ float kv_other_rows(float v, bool maximum)
{
    /* over the four lanes of a column: rows of 16 lanes, then halves of 32 */
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = maximum ? fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])) : __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return maximum ? fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1])) : __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
/* l 2^d, d <= 0: a total counts pages without their value scales, so it can be
 * as large as 2^d is small, and 2^d alone may leave fp32 */
__device__ __forceinline__ float kv_lower(float l, float d)
{
    const float half = exp2f(0.5f * d);
    return l * half * half;
}
/* lane n ^ 8 of the same 16 lanes (row rotation by 8) */
__device__ __forceinline__ float kv_partner(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));
}

/* eight codes -> fp16, exactly */
template <bool E4M3>
__device__ __forceinline__ kv_half8 kv_decode8(uint32_t lo, uint32_t hi)
{
    union {
        kv_half2 pair[4];
        kv_half8 all;
    } r;
    if constexpr (E4M3) {
        r.pair[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
        r.pair[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
        r.pair[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
        r.pair[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    } else {
        /* the byte q + 128 in the low bits of fp16 1024 is 1152 + q */
        lo ^= 0x80808080u;
        hi ^= 0x80808080u;
        const kv_half2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
        r.pair[0] = __builtin_bit_cast(kv_half2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) - bias;
        r.pair[1] = __builtin_bit_cast(kv_half2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) - bias;
        r.pair[2] = __builtin_bit_cast(kv_half2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) - bias;
        r.pair[3] = __builtin_bit_cast(kv_half2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) - bias;
    }
    return r.all;
}

__device__ __forceinline__ float kv_element(const void *base, uint64_t at, int type)
{
    if (type == kElementF32) return static_cast<const float *>(base)[at];
    const uint16_t bits = static_cast<const uint16_t *>(base)[at];
    return type == kElementF16 ? f16_to_f32(bits) : __uint_as_float((uint32_t)bits << 16);
}

/* elements at .. at + 7 as fp32 */
__device__ __forceinline__ void kv_elements8(float *x, const void *base, uint64_t at, int type, bool vector)
{
    if (!vector) {
        for (int e = 0; e < 8; ++e) x[e] = kv_element(base, at + e, type);
    } else if (type == kElementF32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
        const float4 a = p[0], b = p[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + at);
        const uint32_t word[4] = {v.x, v.y, v.z, v.w};
        for (int e = 0; e < 8; ++e) {
            const uint32_t bits = e & 1 ? word[e / 2] >> 16 : word[e / 2] & 0xffffu;
            x[e] = type == kElementF16 ? f16_to_f32(bits) : __uint_as_float(bits << 16);
        }
    }
}

/* four consecutive outputs, rounded once */
__device__ __forceinline__ void kv_store4(void *base, uint64_t at, int type, const kv_float4 v)
{
    if (type == kElementF32) {
        float *p = static_cast<float *>(base) + at;
        for (int e = 0; e < 4; ++e) p[e] = v[e];
    } else {
        uint16_t *p = static_cast<uint16_t *>(base) + at;
        for (int e = 0; e < 4; ++e)
            p[e] = type == kElementF16 ? __builtin_bit_cast(uint16_t, (_Float16)v[e])
                                       : __builtin_bit_cast(uint16_t, (__bf16)v[e]);
    }
}

/* out[row][head][d .. d + 3] = O / l, times sigmoid(gate); 0 where the row saw nothing */
__device__ __forceinline__ void kv_finish4(const KVAttention &a, uint32_t row, uint32_t head, uint32_t d, kv_float4 o,
                                           float l)
{
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    for (int e = 0; e < 4; ++e) o[e] *= inverse;
    if (a.gate) {
        const uint64_t at = row * a.query_row + head * a.query_head + d;
        for (int e = 0; e < 4; ++e) o[e] = o[e] / (1.0f + expf(-kv_element(a.gate, at + e, a.type)));
    }
    kv_store4(a.output, row * a.output_row + (uint64_t)head * a.cache.head_dim + d, a.type, o);
}

/* what a work slot covers; false for a slot with nothing to do */
struct KVSlot {
    uint32_t first_row, rows, column, columns;   /* columns column .. column + columns - 1 of the sequence's rows x group */
    int32_t sequence, tokens;                    /* sequence -1 where the id is bad */
    int32_t seen;                                /* tokens the slot's last row sees */
    __device__ __forceinline__ int32_t seen_by(uint32_t column_at, uint32_t group) const
    {
        return tokens - (int32_t)rows + (int32_t)(column_at / group) + 1;
    }
};
__device__ __forceinline__ bool kv_slot(const KVAttention &a, uint32_t slot, KVSlot &s)
{
    const int i = kv_find_sequence(a.rows, slot, a.group, a.columns, 1);
    if (i < 0) return false;
    const uint32_t begin = kv_row_start(a.rows, i), end = kv_row_start(a.rows, i + 1);
    s.first_row = begin;
    s.rows = end > begin ? end - begin : 0;
    s.column = (slot - kv_slot_base(begin, i, a.group, a.columns, 1)) * a.columns;
    if (s.column >= s.rows * a.group) return false;
    s.columns = min(a.columns, s.rows * a.group - s.column);
    const int32_t id = a.rows.sequences[i];
    s.tokens = (int32_t)kv_tokens(a.cache, id);
    s.sequence = s.tokens > 0 ? id : -1;
    s.seen = max(0, s.seen_by(s.column + s.columns - 1, a.group));
    return true;
}
/* parts of the token axis that a slot is worked on in: at least
 * `least` steps each */
__device__ __forceinline__ uint32_t kv_parts(const KVAttention &a, uint32_t steps, uint32_t least)
{
    return max(1u, min(a.parts, (steps + least - 1) / least));
}
constexpr uint32_t kKVLeastStepsTokens = 4;   /* one per wavefront */
constexpr uint32_t kKVLeastStepsColumns = 8;

/* One workgroup of four wavefronts per (slot, part, key/value head).
 * COLUMNS false: the wavefronts take steps of the tokens in turn, over the
 * same NT tiles of columns, and are joined at the end.  COLUMNS true (prompt
 * chunks): every wavefront has NT column tiles of its own over all steps. */
template <bool E4M3, int D, int NT, bool SPLIT, bool COLUMNS>
__global__ __launch_bounds__(256) void kv_attention_kernel(KVAttention a)
{
    constexpr int kTile = SPLIT ? 8 : 16;
    constexpr int kChunks = D / 64, kChannels = D / 16;
    constexpr int kPitch = D + 4;
    __shared__ float merge_o[COLUMNS ? 1 : 4 * kTile * kPitch];
    __shared__ float merge_m[COLUMNS ? 1 : 4 * NT * kTile], merge_l[COLUMNS ? 1 : 4 * NT * kTile];

    const uint32_t slot = blockIdx.x, head = blockIdx.y, part = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const uint32_t T = a.cache.page_tokens;
    KVSlot s;
    if (!kv_slot(a, slot, s)) return;
    const uint32_t steps = (s.seen + kKVStep - 1) / kKVStep;
    const uint32_t parts = kv_parts(a, steps, COLUMNS ? kKVLeastStepsColumns : kKVLeastStepsTokens);
    if (part >= parts) return;
    uint32_t step = (uint64_t)steps * part / parts, end = (uint64_t)steps * (part + 1) / parts;

    /* the wavefront's columns */
    uint32_t column[NT];
    int32_t seen[NT], seen_least = 0x7fffffff, seen_most = 0;
    float to_u[NT];
    kv_half8 q[NT][2 * kChunks];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        column[t] = ((COLUMNS ? wave * NT : 0) + t) * kTile + (SPLIT ? n & 7 : n);
        const bool held = column[t] < s.columns;
        const uint32_t at = s.column + (held ? column[t] : 0);
        seen[t] = held ? s.seen_by(at, a.group) : 0;
        float x[kChunks * 16];
        uint32_t largest = 0;
        const uint64_t from = (s.first_row + at / a.group) * a.query_row + (head * a.group + at % a.group) * a.query_head;
#pragma unroll
        for (int c = 0; c < 2 * kChunks; ++c) {
            kv_elements8(x + 8 * c, a.query, from + (c / 2) * 64 + g * 16 + (c & 1) * 8, a.type, a.vector);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (!held) x[8 * c + e] = 0.0f;
                largest = max(largest, __float_as_uint(x[8 * c + e]) & 0x7fffffffu);
            }
        }
        /* non-negative floats order as their bits; NaN is above all of them */
        {
            auto r = __builtin_amdgcn_permlane16_swap(largest, largest, false, false);
            largest = max(r[0], r[1]);
            r = __builtin_amdgcn_permlane32_swap(largest, largest, false, false);
            largest = max(r[0], r[1]);
        }
        const uint32_t exponent = max(largest >> 23, 30u);
        const float scale = __uint_as_float((267u - exponent) << 23);       /* largest * scale in 2^13..2^14 */
        to_u[t] = a.scale * __uint_as_float((exponent - 13u) << 23);
#pragma unroll
        for (int c = 0; c < 2 * kChunks; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = x[8 * c + e] * scale;
                const _Float16 high = (_Float16)v;
                q[t][c][e] = SPLIT && n >= 8 ? (_Float16)(v - (float)high) : high;
            }
    }
    /* least and most over the wavefront's columns: columns are in row order */
    for (int t = 0; t < NT; ++t) {
        const uint32_t first = ((COLUMNS ? wave * NT : 0) + t) * kTile;
        if (first < s.columns) {
            seen_least = min(seen_least, s.seen_by(s.column + first, a.group));
            seen_most = max(seen_most, s.seen_by(s.column + min(first + kTile, s.columns) - 1, a.group));
        }
    }
    if (COLUMNS) end = min(end, (uint32_t)(max(seen_most, 0) + kKVStep - 1) / kKVStep);

    kv_float4 o[NT][kChannels];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.0f;
#pragma unroll
        for (int c = 0; c < kChannels; ++c) o[t][c] = {0.0f, 0.0f, 0.0f, 0.0f};
    }

    constexpr uint32_t kStride = COLUMNS ? 1 : 4;
    if (!COLUMNS) step += wave;
    /* the page of the 16 tokens of lane group `part_of` of a step; -1: none */
    auto page_of = [&](uint32_t at, int part_of) -> int32_t {
        const uint32_t token = at * kKVStep + 16 * part_of;
        if (s.sequence < 0 || token >= (uint32_t)s.seen) return -1;
        return kv_page(a.cache, s.sequence, token >> a.page_shift);
    };
    uint4 k[4][kChunks];
    auto load_keys = [&](uint32_t at, int32_t page) {
        const uint32_t token = at * kKVStep + 16 * (n >> 2);
        const uint8_t *from = a.cache.data + kv_block(a.cache, max(page, 0), 0, head) * (T * D) +
                              ((token & (T - 1)) + (n & 3)) * D + g * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < kChunks; ++j) k[i][j] = *reinterpret_cast<const uint4 *>(from + 4 * i * D + j * 64);
    };
    int32_t key_page = step < end ? page_of(step, n >> 2) : -1, page = step < end ? page_of(step, g) : -1;
    if (step < end) load_keys(step, key_page);
    for (; step < end; step += kStride) {
        const uint32_t token = step * kKVStep + 16 * g;
        /* this step's values and scales */
        const uint64_t block = kv_block(a.cache, max(page, 0), 1, head);
        uint4 v[kChannels];
        {
            const uint8_t *from = a.cache.data + block * (T * D) + n * T + (token & (T - 1));
#pragma unroll
            for (int c = 0; c < kChannels; ++c) v[c] = *reinterpret_cast<const uint4 *>(from + c * 16 * T);
        }
        float key_scale = 1.0f, value_scale = 1.0f;
        if (page >= 0) {
            key_scale = a.cache.scales[block - a.cache.kv_heads];
            value_scale = a.cache.scales[block];
        }
        const bool next = step + kStride < end;
        const int32_t next_key_page = next ? page_of(step + kStride, n >> 2) : -1;
        const int32_t next_page = next ? page_of(step + kStride, g) : -1;

        kv_float4 score[NT][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int t = 0; t < NT; ++t) score[t][i] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                const kv_half8 low = kv_decode8<E4M3>(k[i][j].x, k[i][j].y), high = kv_decode8<E4M3>(k[i][j].z, k[i][j].w);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    score[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(low, q[t][2 * j], score[t][i], 0, 0, 0);
                    score[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, q[t][2 * j + 1], score[t][i], 0, 0, 0);
                }
            }
        }
        if (next) load_keys(step + kStride, next_key_page);

        const uint32_t scale_bits = __float_as_uint(value_scale);
        const float value_log = value_scale == value_scale ? (float)((int)(scale_bits >> 23) - 127) : value_scale;
        const float inverse = __uint_as_float((254u << 23) - scale_bits);
        const bool whole = step * kKVStep + kKVStep <= (uint32_t)max(seen_least, 0) && __all(page >= 0);
        kv_half8 weight[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float factor = to_u[t] * key_scale;
            float u[16], most = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float dot = score[t][e / 4][e & 3];
                if (SPLIT) dot += kv_partner(dot);
                u[e] = fmaf(dot, factor, value_log);
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (page < 0 || (int32_t)(token + e) >= seen[t]) u[e] = -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) most = fmaxf(most, u[e]);
            most = kv_other_rows(most, true);
            if (__any(most > m[t] + kKVMaximumSlack)) {
                const float now = fmaxf(m[t], most);
                const float by = m[t] == now ? 0.0f : m[t] - now, keep = exp2f(by);
                m[t] = now;
                l[t] = kv_lower(l[t], by);
#pragma unroll
                for (int c = 0; c < kChannels; ++c) o[t][c] *= keep;
            }
            const float offset = kKVWeightExponent - (m[t] == -INFINITY ? 0.0f : m[t]);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float w = __builtin_amdgcn_exp2f(u[e] + offset);
                sum += w;
                const _Float16 high = (_Float16)w;
                weight[t][e / 8][e & 7] = SPLIT && n >= 8 ? (_Float16)(w - (float)high) : high;
            }
            /* weights of a page whose value scale lies that far below the sums'
             * largest leave fp32 before they leave the total: theirs is taken
             * without the scale */
            if (__any(value_log < m[t] - 64.0f && page >= 0)) {
                const float back = value_scale == value_scale ? offset - value_log : offset;
                sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f(u[e] + back);
                l[t] += sum;
            } else {
                l[t] = fmaf(sum, inverse, l[t]);
            }
        }
        if (!whole) {
            /* codes of tokens that no column of the slot sees may be any bytes */
            const int32_t good = page < 0 ? 0 : min(16, max(0, s.seen - (int32_t)token));
#pragma unroll
            for (int c = 0; c < kChannels; ++c) {
                uint32_t word[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int left = good - 4 * b;
                    word[b] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
                }
                v[c] = make_uint4(word[0], word[1], word[2], word[3]);
            }
        }
#pragma unroll
        for (int c = 0; c < kChannels; ++c) {
            const kv_half8 low = kv_decode8<E4M3>(v[c].x, v[c].y), high = kv_decode8<E4M3>(v[c].z, v[c].w);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                o[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(low, weight[t][0], o[t][c], 0, 0, 0);
                o[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, weight[t][1], o[t][c], 0, 0, 0);
            }
        }
        key_page = next_key_page;
        page = next_page;
    }

    const uint64_t partial = (((uint64_t)slot * a.cache.kv_heads + head) * a.parts + part) * a.columns;
    float *stats = a.partial + (uint64_t)a.slots * a.cache.kv_heads * a.parts * a.columns * D;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        l[t] = kv_other_rows(l[t], false);
        if (l[t] != l[t]) m[t] = INFINITY;      /* a NaN outweighs the other parts */
        if (SPLIT)
#pragma unroll
            for (int c = 0; c < kChannels; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t][c][e] += kv_partner(o[t][c][e]);
    }
    if (COLUMNS) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (column[t] >= s.columns || (SPLIT && n >= 8)) continue;
            const uint32_t at = s.column + column[t];
            if (parts == 1) {
#pragma unroll
                for (int c = 0; c < kChannels; ++c)
                    kv_finish4(a, s.first_row + at / a.group, head * a.group + at % a.group, c * 16 + 4 * g, o[t][c], l[t]);
            } else {
                float *to = a.partial + (partial + column[t]) * D + 4 * g;
#pragma unroll
                for (int c = 0; c < kChannels; ++c) *reinterpret_cast<kv_float4 *>(to + c * 16) = o[t][c];
                if (g == 0) {
                    stats[2 * (partial + column[t])] = m[t];
                    stats[2 * (partial + column[t]) + 1] = l[t];
                }
            }
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
        if (g == 0 && (!SPLIT || n < 8)) {
            merge_m[(wave * NT + t) * kTile + n] = m[t];
            merge_l[(wave * NT + t) * kTile + n] = l[t];
        }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t * kTile >= s.columns) break;
        if (!SPLIT || n < 8) {
            float top = -INFINITY;
            for (int w = 0; w < 4; ++w) top = fmaxf(top, merge_m[(w * NT + t) * kTile + n]);
            const float keep = m[t] == top ? (m[t] == -INFINITY ? 0.0f : 1.0f) : exp2f(m[t] - top);
#pragma unroll
            for (int c = 0; c < kChannels; ++c)
                *reinterpret_cast<kv_float4 *>(&merge_o[(wave * kTile + n) * kPitch + c * 16 + 4 * g]) = o[t][c] * keep;
        }
        __syncthreads();
        for (uint32_t at = threadIdx.x; at < kTile * (D / 4); at += 256) {
            const uint32_t c = at / (D / 4), d = at % (D / 4) * 4, of = t * kTile + c;
            if (of >= s.columns) break;
            float top = -INFINITY, total = 0.0f;
            kv_float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int w = 0; w < 4; ++w) top = fmaxf(top, merge_m[(w * NT + t) * kTile + c]);
            for (int w = 0; w < 4; ++w) {
                const float mw = merge_m[(w * NT + t) * kTile + c];
                if (mw == -INFINITY) continue;
                total += kv_lower(merge_l[(w * NT + t) * kTile + c], mw - top);
                sum += *reinterpret_cast<const kv_float4 *>(&merge_o[(w * kTile + c) * kPitch + d]);
            }
            if (parts == 1) {
                const uint32_t col = s.column + of;
                kv_finish4(a, s.first_row + col / a.group, head * a.group + col % a.group, d, sum, total);
            } else {
                *reinterpret_cast<kv_float4 *>(a.partial + (partial + of) * D + d) = sum;
                if (d == 0) {
                    stats[2 * (partial + of)] = top;
                    stats[2 * (partial + of) + 1] = total;
                }
            }
        }
        __syncthreads();
    }
}

template <int D>
bool launch_kv_attention_width(const KVAttention &a, hipStream_t stream);

}  // namespace q38
