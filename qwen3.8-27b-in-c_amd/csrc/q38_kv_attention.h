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
 * n in the results of both, so maximum, sum and rescaling are the lane's own.
 * Row m of the i-th of four key tiles is token 16 (m / 4) + 4 i + m % 4 of a
 * 64-token step: lane g then has the scores of tokens 16 g .. 16 g + 15, which
 * are both its slice of the second product and 16 consecutive bytes of a value
 * channel.
 *
 * Few columns (decode, verify): memory is the bound.  Codes go straight into
 * LDS (global_load_lds, 1 KiB each, whole rows of keys or values, so requests
 * are contiguous and no register waits for them); a wavefront asks for its next
 * keys when it has read the present ones, and for its next values channel by
 * channel.  48 sequences of up to 16384 tokens (32 heads, 8 of keys, 128 wide,
 * 339 MB): 63 us, 5.3 TB/s, what a large copy reaches here.  Four rows at 131075
 * tokens (24 heads, 4 of keys, 256 wide, 268 MB): 71 us, 3.8 TB/s; 9 us pass
 * before the first step's codes are there, 7 in the merge at the end.
 *
 * Many columns (prompts): the products are the bound.  512 rows behind 7679
 * tokens (24 heads, 4 of keys, 256 wide, 100 GFLOP): 146 us, 680 TFLOP/s; of
 * its cycles the matrix unit is busy in a third, LDS in over half.
 *
 * Short calls are instruction fetch: 37 tokens take 11 us, of which memory is
 * three; what runs once is kept short.
 *
 * 8-bit codes are exact in fp16, and so is a 16-bit query once its row is
 * scaled by a power of two to a maximum of 2^13..2^14 (but for what lies 2^37
 * below it).  For fp32 calls (SPLIT) a column takes two lanes: n < 8 works
 * with the fp16 value of its queries and weights, n + 8 with what that leaves,
 * 22 bits together.  16-bit calls keep the fp16 weight alone, for half the
 * products: its error, up to 2^-11 of the weight, is an eighth of a bf16 output's
 * own rounding and as large as an fp16 output's for one token, less over many
 * (off the 64-bit result, root of the mean square: 512 rows behind 7679 tokens,
 * bf16, 1.7e-3 as with fp32 weights; prompts of up to 300 tokens, fp16, 2.5e-4
 * instead of 2.1e-4).  The largest weight is 2^6 or more, fp16's least step 2^-24:
 * what lies 2^20 below the largest loses bits, what lies 2^31 below is nothing. */
#pragma once

#include "q38_device.h"
#include "q38_kv.h"
#include "q38_kv_plan.h"

namespace q38 {

using kv_half2 = _Float16 __attribute__((ext_vector_type(2)));
using kv_half8 = _Float16 __attribute__((ext_vector_type(8)));
using kv_float4 = float __attribute__((ext_vector_type(4)));

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
/* largest of 8, 16 or 32 neighbouring lanes: within quads, eights and rows of 16 by row operations */
template <int LANES>
__device__ __forceinline__ uint32_t kv_largest(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));      /* lane ^ 1 */
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));      /* lane ^ 2 */
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));     /* 7 - lane of eight */
    if (LANES >= 16) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));    /* 15 - lane */
    if (LANES == 32) {
        auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(r[0], r[1]);
    }
    return v;
}
/* l 2^d, d <= 0: a total counts pages without their value scales, so it can be
 * as large as 2^d is small, and 2^d alone may leave fp32 */
__device__ __forceinline__ float kv_lower(float l, float d)
{
    const float half = __builtin_amdgcn_exp2f(0.5f * d);
    return l * half * half;
}
/* lane n ^ 8 of the same 16 lanes (row rotation by 8) */
__device__ __forceinline__ float kv_partner(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));
}

using kv_float2 = float __attribute__((ext_vector_type(2)));
/* two values to fp16; LOW: what fp16 leaves of them in the lanes of `mask` -1 */
template <bool LOW>
__device__ __forceinline__ kv_half2 kv_round2(float a, float b, uint32_t mask)
{
    const kv_half2 high = __builtin_convertvector((kv_float2){a, b}, kv_half2);
    if constexpr (!LOW) return high;
    const kv_half2 taken = __builtin_bit_cast(kv_half2, __builtin_bit_cast(uint32_t, high) & mask);
    return __builtin_convertvector((kv_float2){a - (float)taken[0], b - (float)taken[1]}, kv_half2);
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

/* sums += A B for sums in accumulation registers, in place: the builtin lets
 * the compiler give the result other registers, and it moved all sums about once
 * a step.  What it cannot see it cannot guard, so the wait states are here: two
 * between a vector instruction that writes A or B, or the product that wrote the
 * sums, and this one; eight behind the last one of a step, before anything else
 * may touch its sums.  (A product takes three with its own, so those before it
 * are done by then.)  The compiler may copy the sums anywhere behind it. */
__device__ __forceinline__ void kv_accumulate(kv_float4 &sums, kv_half8 a, kv_half8 b, bool last)
{
    if (last) asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0\n\ts_nop 7" : "+a"(sums) : "v"(a), "v"(b));
    else asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(sums) : "v"(a), "v"(b));
}

/* Sums in accumulation registers times keep, by way of 16 bytes of LDS per
 * lane: vector instructions take no accumulation registers, and four of them
 * have no names of their own here.  Seldom done, and no product is under way. */
__device__ __forceinline__ void kv_scale(kv_float4 &sums, float keep, uint32_t lane_lds)
{
    float a, b, c, d;
    asm volatile("ds_write_b128 %6, %0\n\t"
                 "ds_read_b32 %1, %6\n\tds_read_b32 %2, %6 offset:4\n\tds_read_b32 %3, %6 offset:8\n\tds_read_b32 %4, %6 offset:12\n\t"
                 "s_waitcnt lgkmcnt(0)\n\tv_mul_f32 %1, %1, %5\n\tv_mul_f32 %2, %2, %5\n\tv_mul_f32 %3, %3, %5\n\tv_mul_f32 %4, %4, %5\n\t"
                 "ds_write_b32 %6, %1\n\tds_write_b32 %6, %2 offset:4\n\tds_write_b32 %6, %3 offset:8\n\tds_write_b32 %6, %4 offset:12\n\t"
                 "ds_read_b128 %0, %6\n\ts_waitcnt lgkmcnt(0)"
                 : "+a"(sums), "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d)
                 : "v"(keep), "v"(lane_lds)
                 : "memory");
}

/* 16, 8 and 4 bytes at any alignment of the element */
struct __attribute__((packed, aligned(2))) KVBytes16 {
    uint32_t word[4];
};
struct __attribute__((packed, aligned(2))) KVBytes8 {
    uint32_t word[2];
};
struct __attribute__((packed, aligned(4))) KVFloats4 {
    float v[4];
};

/* fp16 where `f16` is -1, bf16 where it is 0: no branch for each element */
__device__ __forceinline__ float kv_half(uint32_t bits, uint32_t f16)
{
    return __uint_as_float((__float_as_uint(f16_to_f32(bits)) & f16) | (bits << 16 & ~f16));
}
__device__ __forceinline__ uint32_t kv_f16(const KVAttention &a) { return a.type == kElementF16 ? 0xffffffffu : 0u; }

/* elements at .. at + 7 as stored: fp32 eight words, 16-bit types four */
template <bool F32>
__device__ __forceinline__ void kv_load8(uint32_t *raw, const void *base, uint64_t at)
{
    if constexpr (F32) {
        const KVFloats4 *p = reinterpret_cast<const KVFloats4 *>(static_cast<const float *>(base) + at);
        const KVFloats4 a = p[0], b = p[1];
        for (int e = 0; e < 4; ++e) raw[e] = __float_as_uint(a.v[e]), raw[4 + e] = __float_as_uint(b.v[e]);
    } else {
        const KVBytes16 v = *reinterpret_cast<const KVBytes16 *>(static_cast<const uint16_t *>(base) + at);
        for (int e = 0; e < 4; ++e) raw[e] = v.word[e];
    }
}
template <bool F32>
__device__ __forceinline__ float kv_element8(const uint32_t *raw, int e, uint32_t f16)
{
    if constexpr (F32) return __uint_as_float(raw[e]);
    else return kv_half(e & 1 ? raw[e / 2] >> 16 : raw[e / 2] & 0xffffu, f16);
}

/* elements at .. at + 3 */
__device__ __forceinline__ kv_float4 kv_load4(const void *base, uint64_t at, const KVAttention &a)
{
    if (a.type == kElementF32) {
        const KVFloats4 v = *reinterpret_cast<const KVFloats4 *>(static_cast<const float *>(base) + at);
        return {v.v[0], v.v[1], v.v[2], v.v[3]};
    }
    const KVBytes8 v = *reinterpret_cast<const KVBytes8 *>(static_cast<const uint16_t *>(base) + at);
    const uint32_t f16 = kv_f16(a);
    return {kv_half(v.word[0] & 0xffffu, f16), kv_half(v.word[0] >> 16, f16), kv_half(v.word[1] & 0xffffu, f16),
            kv_half(v.word[1] >> 16, f16)};
}
/* four consecutive outputs, rounded once */
__device__ __forceinline__ void kv_store4(void *base, uint64_t at, const KVAttention &a, const kv_float4 v)
{
    if (a.type == kElementF32) {
        *reinterpret_cast<KVFloats4 *>(static_cast<float *>(base) + at) = {{v[0], v[1], v[2], v[3]}};
    } else {
        const uint32_t f16 = kv_f16(a);
        uint32_t bits[4];
        for (int e = 0; e < 4; ++e)
            bits[e] = (__builtin_bit_cast(uint16_t, (_Float16)v[e]) & f16) | (__builtin_bit_cast(uint16_t, (__bf16)v[e]) & ~f16);
        *reinterpret_cast<KVBytes8 *>(static_cast<uint16_t *>(base) + at) = {{bits[0] | bits[1] << 16, bits[2] | bits[3] << 16}};
    }
}

/* 1 / (1 + e^-x) within 2^-21 of itself, or, where it is subnormal, 2^-149.
 * With E = e^-|x| it is 1 / (1 + E), for negative x E / (1 + E): nothing
 * overflows.  E = 2^(n + f), n whole, with log2(e) in two parts, so f's error
 * does not grow with x; E is 0 in fp32 from |x| = 104 on, so x ends at 128 (a NaN
 * stays one). */
__device__ __forceinline__ float kv_sigmoid(float x)
{
    constexpr float kHigh = 1.44269502f, kLow = 1.92596299e-8f;
    float a = fabsf(x);
    if (a > 128.0f) a = 128.0f;
    const float n = __builtin_rintf(-a * kHigh);
    const float f = fmaf(-a, kLow, fmaf(-a, kHigh, -n));
    const float e = ldexpf(__builtin_amdgcn_exp2f(f), (int)n), d = 1.0f + e;
    const float first = __builtin_amdgcn_rcpf(d), inverse = fmaf(first, fmaf(-d, first, 1.0f), first);
    return x < 0.0f ? e * inverse : inverse;
}

__device__ __forceinline__ kv_float4 kv_gate4(const KVAttention &a, uint32_t row, uint32_t head, uint32_t d)
{
    if (!a.gate) return {0.0f, 0.0f, 0.0f, 0.0f};
    return kv_load4(a.gate, row * a.query_row + head * a.query_head + d, a);
}
/* out[row][head][d .. d + 3] = O / l, times sigmoid(gate); 0 where the row saw
 * nothing.  The gate was asked for by kv_gate4 some time before. */
__device__ __forceinline__ void kv_finish4(const KVAttention &a, uint32_t row, uint32_t head, uint32_t d, kv_float4 o,
                                           float l, kv_float4 gate)
{
    o *= l == 0.0f ? 0.0f : 1.0f / l;
    if (a.gate)
        for (int e = 0; e < 4; ++e) o[e] *= kv_sigmoid(gate[e]);
    kv_store4(a.output, row * a.output_row + (uint64_t)head * a.cache.head_dim + d, a, o);
}

/* ---- work ---------------------------------------------------------------------- */

/* A slot: up to a.columns columns of one sequence, from the rem-th query head
 * of the group in its row `row` on. */
struct KVSlot {
    uint32_t index;                              /* among the call's slots */
    uint32_t first_row, row, rem, columns;       /* the sequence's first row in the call */
    int32_t sequence, seen_first, seen;          /* -1 where the id is bad; tokens that row `row`, and the last, sees */
    /* row of the slot's column c, from `row` on, and its head of the group */
    __device__ __forceinline__ uint32_t row_of(const KVAttention &a, uint32_t c) const { return kv_divide(rem + c, a.group_magic); }
    __device__ __forceinline__ uint32_t head_of(const KVAttention &a, uint32_t c) const
    {
        return rem + c - row_of(a, c) * a.group;
    }
    /* tokens that column c sees, none or fewer for a row before the sequence's first token */
    __device__ __forceinline__ int32_t seen_by(const KVAttention &a, uint32_t c) const
    {
        return seen_first + (int32_t)row_of(a, c);
    }
};

/* 64 sequences of the call, one per lane, and the prefix sums of their slots
 * and units (kv_slot_units) */
template <uint32_t COLUMNS>
struct KVLanes {
    uint32_t first;                              /* of the block */
    uint32_t begin, end, slots, each;            /* the lane's; units of each slot */
    int32_t id, tokens;
    uint32_t slots_upto, units_upto;             /* inclusive, within the block */
    uint32_t trouble;                            /* Q38_KV_*: row offsets that decrease, bad ids that own rows */

    __device__ __forceinline__ void load(const KVAttention &a, uint32_t at)
    {
        const uint32_t lane = threadIdx.x & 63, i = at + lane;
        first = at;
        begin = end = slots = each = 0;
        id = -1;
        tokens = 0;
        if (i < a.rows.count) {
            id = a.rows.sequences[i];
            begin = kv_row_start(a.rows, i);
            end = kv_row_start(a.rows, i + 1);
            tokens = (int32_t)kv_tokens(a.cache, id);
            slots = ((end - begin) * a.group + COLUMNS - 1) / COLUMNS;
            each = kv_slot_units(kv_steps((uint32_t)tokens), a.shift);
        }
        trouble = (__any(begin > end) ? Q38_KV_BAD_ROWS : 0) |
                  (__any(begin < end && (uint32_t)id >= a.cache.sequences) ? Q38_KV_BAD_SEQUENCE : 0);
        slots_upto = slots;
        units_upto = slots * each;
        if (a.rows.count == 1) {
            slots_upto = of(slots_upto, 0);
            units_upto = of(units_upto, 0);
            return;
        }
        for (int by = 1; by < 64; by *= 2) {
            const uint32_t s = (uint32_t)__shfl_up((int)slots_upto, by), u = (uint32_t)__shfl_up((int)units_upto, by);
            if (lane >= (uint32_t)by) slots_upto += s, units_upto += u;
        }
    }
    static __device__ __forceinline__ uint32_t of(uint32_t v, int lane)
    {
        return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
    }
};

/* What a workgroup does.  The slots' units, one after another, are cut into
 * equal ranges, one per workgroup (and key/value head); a slot of few units
 * goes whole to the range that it begins in. */
template <uint32_t COLUMNS>
struct KVWalk {
    using Lanes = KVLanes<COLUMNS>;
    Lanes block;
    uint32_t block_slots, block_units;           /* of the sequences before the block */
    uint32_t total_slots, total_units, chunk, small, at, end;

    __device__ __forceinline__ void start(const KVAttention &a, uint32_t workgroup)
    {
        total_slots = total_units = block_slots = block_units = 0;
        uint32_t trouble = 0;
        for (uint32_t first = (a.rows.count - 1) / 64 * 64 + 64; first; ) {
            first -= 64;
            block.load(a, first);
            total_slots += Lanes::of(block.slots_upto, 63);
            total_units += Lanes::of(block.units_upto, 63);
            trouble |= block.trouble;
        }
        if (trouble) {
            if (threadIdx.x == 0) atomicOr(a.cache.status, (int32_t)trouble);
            /* with bad offsets the sums mean nothing, and the workspace need not hold the slots */
            if (trouble & Q38_KV_BAD_ROWS) total_slots = total_units = 0;
        }
        chunk = kv_chunk(total_units, a.workgroups, a.workgroups_inverse, a.least);
        small = kv_small(chunk);
        at = min((uint64_t)workgroup * chunk, (uint64_t)total_units);
        end = min((uint64_t)at + chunk, (uint64_t)total_units);
    }

    /* the next piece of a slot; false when there is none */
    __device__ __forceinline__ bool next(const KVAttention &a, KVSlot &s, KVPiece &piece)
    {
        const uint32_t from = at;
        while (at < end) {
            while (at - block_units >= Lanes::of(block.units_upto, 63)) {
                block_slots += Lanes::of(block.slots_upto, 63);
                block_units += Lanes::of(block.units_upto, 63);
                block.load(a, block.first + 64);
            }
            const int i = __popcll(__ballot(block.units_upto <= at - block_units));
            const uint32_t slots = Lanes::of(block.slots, i), each = Lanes::of(block.each, i);
            const uint32_t base = block_units + Lanes::of(block.units_upto, i) - slots * each;
            uint32_t j = 0;
            if (slots != 1) {
                /* (opaque: a division that is skipped, not one that is begun ahead of the branch) */
                uint32_t by = each;
                asm volatile("" : "+v"(by));
                j = __builtin_amdgcn_readfirstlane((at - base) / by);
            }
            const uint32_t slot_at = base + j * each;
            const uint32_t rows = Lanes::of(block.end, i) - Lanes::of(block.begin, i), column = j * COLUMNS;
            const int32_t tokens = (int32_t)Lanes::of((uint32_t)block.tokens, i);
            s.first_row = Lanes::of(block.begin, i);
            s.index = block_slots + Lanes::of(block.slots_upto, i) - slots + j;
            s.row = 0;
            if (j) {
                uint32_t group = a.group;
                asm volatile("" : "+v"(group));
                s.row = __builtin_amdgcn_readfirstlane(column / group);
            }
            s.rem = column - s.row * a.group;
            s.columns = min(COLUMNS, rows * a.group - column);
            s.sequence = tokens > 0 ? (int32_t)Lanes::of((uint32_t)block.id, i) : -1;
            s.seen_first = tokens - (int32_t)rows + (int32_t)s.row + 1;
            s.seen = max(0, s.seen_by(a, s.columns - 1));
            at = slot_at + each;
            piece = kv_piece(slot_at, each, kv_steps((uint32_t)s.seen), from, end, small, a.shift);
            if (piece.some) return true;
        }
        return false;
    }
};

/* Workspace of a call whose slots may be cut: one KVRecord per slot (record 0
 * is the number of slots), then the sums of the pieces, then their (maximum,
 * total).  A workgroup has two pieces of cut slots at most, kv_place. */
struct KVRecord {
    uint32_t pieces, first_piece, row, rem, columns, unused[3];    /* row: of the call */
};
__device__ __forceinline__ KVRecord *kv_records(const KVAttention &a) { return reinterpret_cast<KVRecord *>(a.partial); }
__device__ __forceinline__ float *kv_partial(const KVAttention &a, uint64_t piece, uint32_t head)
{
    return a.partial + (a.slots + 1) * (sizeof(KVRecord) / 4) + (piece * a.cache.kv_heads + head) * a.columns * a.cache.head_dim;
}
__device__ __forceinline__ float *kv_stats(const KVAttention &a, uint64_t piece, uint32_t head)
{
    return kv_partial(a, 2ull * a.workgroups, 0) + (piece * a.cache.kv_heads + head) * a.columns * 2;
}

/* ---- codes to LDS -------------------------------------------------------------- */

__device__ __forceinline__ uint32_t kv_lds(const void *p)
{
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}
/* 16 (4) bytes per lane to LDS at `to` + 16 (4) lane.  Inline assembly keeps
 * the compiler's wait counts out of it: callers wait.  So is the wait state
 * that a load to LDS needs behind a scalar write of the M0 that it reads. */
__device__ __forceinline__ void kv_copy16(const void *from, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
__device__ __forceinline__ void kv_copy4(const void *from, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void kv_wait()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
/* the wavefront's LDS reads have returned: what they read may be overwritten */
__device__ __forceinline__ void kv_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void kv_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

/* Places in LDS.  A read of 16 bytes by all lanes is served 16 lanes at a time,
 * of each 32 the lanes 0..3, 12..15, 20..27, then the others; the turns below put
 * the 16 pieces that are read together, two columns (g) of eight rows, at places
 * of their own modulo 256 bytes.
 *
 * Codes of a step's 64 tokens, D * 64 bytes of keys and as many of values: key
 * row r = 16 i + n (token 16 (n / 4) + 4 i + n % 4) holds its 16-byte pieces p
 * at p ^ kv_key_turn(n); a value row (channel) its four at p ^ kv_value_turn(n),
 * n the channel's low four bits. */
template <int D>
__device__ __forceinline__ uint32_t kv_key_turn(uint32_t n)
{
    return D == 256 ? n : D == 128 ? n >> 1 : ((n >> 2) + 1) & 3;
}
__device__ __forceinline__ uint32_t kv_value_turn(uint32_t n) { return ((n >> 2) + 1) & 3; }
/* the same of rows of fp16 keys (2 D bytes) and values (128 bytes) */
__device__ __forceinline__ uint32_t kv_wide_value_turn(uint32_t n) { return ((n >> 1) + 2) & 7; }
template <int D>
__device__ __forceinline__ uint32_t kv_wide_turn(uint32_t n)
{
    return D == 64 ? kv_wide_value_turn(n) : n;
}

/* One workgroup per (range of work, key/value head).
 * COLUMNS false: four wavefronts take steps of the tokens in turn, over the same
 * NT tiles of columns, each with its own step's codes in LDS, and are joined at
 * the end.  COLUMNS true: every wavefront has NT column tiles of its own over
 * all steps; a step is decoded once for all of them, through registers, a step
 * ahead, into one of two tiles of fp16, 2 D bytes a key and 128 a channel, whose
 * 16-byte pieces of eight are turned by the row like those of the codes. */
template <int D>
constexpr int kv_ring_bytes() { return 512 * D; }
template <int D, int WAVES>
constexpr int kv_lds_bytes()
{
    constexpr int merge = WAVES * 16 * (D + 4) * 4;
    return kv_ring_bytes<D>() > merge ? kv_ring_bytes<D>() : merge;
}

template <bool E4M3, int D, int NT, bool SPLIT, bool COLUMNS>
__global__ __launch_bounds__(64 * kv_workgroup_waves(D, COLUMNS), kv_waves(D, COLUMNS)) void kv_attention_kernel(KVAttention a)
{
    constexpr int kTile = SPLIT ? 8 : 16, kWaves = kv_workgroup_waves(D, COLUMNS);
    constexpr bool kAccumulators = kv_waves(D, COLUMNS) == 1;  /* more registers than VGPRs: sums in AGPRs */
    constexpr int kChunks = D / 64, kChannels = D / 16;
    constexpr int kPitch = D + 4;
    constexpr int kCopies = D / 16;                                /* copies of 1 KiB of a step's keys or values */
    constexpr int kRuns = D / 64;                                  /* of 16-token groups that a lane copies keys of */
    constexpr uint32_t kColumns = NT * kTile * (COLUMNS ? kWaves : 1);
    constexpr int kTileBytes = 16 * D * 2;                          /* a tile's queries in fp16, as the products take them */
    __shared__ __attribute__((aligned(16))) uint8_t ring[kv_lds_bytes<D, kWaves>()];
    __shared__ float metas[kWaves * 128];                           /* scales: of 16 steps, keys then values, each wavefront's */
    __shared__ __attribute__((aligned(16))) uint8_t queries[COLUMNS ? 16 : NT * kTileBytes];
    __shared__ kv_float4 bounces[kAccumulators ? 256 : 1];
    kv_float4 *bounce = bounces + (kAccumulators ? threadIdx.x : 0);
    __shared__ float merge_m[kWaves * NT * kTile], merge_l[kWaves * NT * kTile], to_exponent[kColumns];

    const uint32_t head = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const uint32_t T = a.cache.page_tokens, low_half = n >= 8 ? 0xffffffffu : 0u, f16 = kv_f16(a);
    uint8_t *mine = ring + (COLUMNS ? 0 : wave * 128 * D);        /* the (first) keys; values 64 D behind */
    float *meta = metas + wave * 128;

    /* LDS places of the lane's reads; COLUMNS: of eight channels, of eight tokens */
    const uint32_t wide_key_at = n * 2 * D + ((2 * g) ^ kv_wide_turn<D>(n)) * 16;
    const uint32_t wide_value_at = 128 * D + n * 128 + ((2 * g) ^ kv_wide_value_turn(n)) * 16;
    const uint32_t value_at = 64 * D + n * 64 + (g ^ kv_value_turn(n)) * 16;
    /* what the lane copies.  Keys: copy d = kRuns i + run is rows 16 i + (64 /
     * D..) of the tile: within a run every i is four tokens further on */
    constexpr int kLanesPerRow = D / 16, kRowsPerCopy = 64 / kLanesPerRow;
    const uint32_t copy_row = lane / kLanesPerRow;                /* + run * kRowsPerCopy = n of the row */
    const uint32_t value_group = (lane & 3) ^ kv_value_turn(lane >> 2);

    KVWalk<kColumns> walk;
    walk.start(a, blockIdx.x);
    if (a.cut && blockIdx.x == 0 && head == 0 && threadIdx.x == 0) kv_records(a)->pieces = walk.total_slots;
    KVSlot s;
    KVPiece piece;
    while (walk.next(a, s, piece)) {
        /* the wavefront's columns, and least and most that they see: columns are in row order */
        const uint32_t first_column = COLUMNS ? wave * NT * kTile : 0;
        int32_t seen[NT], seen_least = 0x7fffffff, seen_most = 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t first = first_column + t * kTile, c = first + (SPLIT ? n & 7 : n);
            seen[t] = c < s.columns ? s.seen_by(a, c) : 0;
            if (first < s.columns) {
                seen_least = min(seen_least, s.seen_by(a, first));
                seen_most = max(seen_most, s.seen_by(a, min(first + kTile, s.columns) - 1));
            }
        }
        constexpr uint32_t kStride = COLUMNS ? 1 : 4;
        uint32_t step = piece.first + (COLUMNS ? 0 : wave);
        const uint32_t end = piece.last, own_end = COLUMNS ? min(end, kv_steps((uint32_t)max(seen_most, 0))) : end;

        /* pages of 16 steps: lane l has that of tokens 16 (l % 4) .. of the
         * step that is l / 4 turns after the first; their scales go to LDS */
        int32_t pages = -1;
        uint32_t turn = 0;
        auto load_pages = [&](uint32_t first) {
            const uint32_t at = first + (lane >> 2) * kStride, token = at * kKVStep + 16 * (lane & 3);
            pages = -1;
            if (at < end && s.sequence >= 0 && token < (uint32_t)s.seen) {
                pages = kv_page(a.cache, s.sequence, token >> a.page_shift);
                /* (anywhere in the loop or before it this costs four rows at 131k tokens 3 us of 68) */
                if (pages < 0) atomicOr(a.cache.status, Q38_KV_BAD_PAGE);
            }
            turn = 0;
            const float *scales = a.cache.scales + kv_block(a.cache, max(pages, 0), 0, head);
            kv_copy4(scales, kv_lds(meta));
            kv_copy4(scales + a.cache.kv_heads, kv_lds(meta + 64));
        };
        auto copy_keys = [&](uint32_t at, uint32_t to) {
#pragma unroll
            for (int run = 0; run < kRuns; ++run) {
                const uint32_t row = run * kRowsPerCopy + copy_row;            /* n */
                const uint32_t chunk = ((lane % kLanesPerRow) ^ kv_key_turn<D>(row)) & (kLanesPerRow - 1);
                const uint32_t token = at * kKVStep + 16 * (row >> 2) + (row & 3);
                const int32_t page = max(__shfl(pages, (int)(4 * turn + (row >> 2))), 0);
                const uint8_t *from = a.cache.data + kv_block(a.cache, page, 0, head) * (T * D) + (token & (T - 1)) * D + chunk * 16;
#pragma unroll 1
                for (int i = 0; i < 4; ++i) kv_copy16(from + 4 * i * D, to + (kRuns * i + run) * 1024);
            }
        };
        /* where the lane's 16 bytes of value copy 0 of a step come from; copy c is 16 channels on */
        auto value_from = [&](uint32_t at) {
            const int32_t page = max(__shfl(pages, (int)(4 * turn + value_group)), 0);
            return a.cache.data + kv_block(a.cache, page, 1, head) * (T * D) + (lane >> 2) * T +
                   ((at * kKVStep + 16 * value_group) & (T - 1));
        };
        auto copy_values = [&](uint32_t at, uint32_t to) {
            const uint8_t *from = value_from(at);
#pragma unroll 4
            for (int c = 0; c < kCopies; ++c) kv_copy16(from + c * 16 * T, to + c * 1024);
        };

        /* COLUMNS: the thread's part of a step, 16 codes at a time: to registers, and from there decoded to LDS */
        constexpr int kPieces = COLUMNS ? D * 4 / (64 * kWaves) : 1;
        using kv_codes16 = uint32_t __attribute__((ext_vector_type(4)));
        kv_codes16 raw_codes[COLUMNS ? 2 * kPieces : 1];
        int32_t value_good = 16;
        bool value_partial = false;
        /* Pieces of 16 codes of a key that the thread takes, of token stage_token + kStageTokens k:
         * 16 lanes write two rows or more, whose turns differ, so their two halves use all banks */
        const uint32_t stage_piece = D == 256 ? (threadIdx.x & 7) + (threadIdx.x >> 1 & 8) : threadIdx.x % (D / 16);
        const uint32_t stage_token = D == 256 ? (threadIdx.x >> 5) * 2 + (threadIdx.x >> 3 & 1) : threadIdx.x / (D / 16);
        const uint32_t stage_group = wave * 64 / D;            /* its 16-token group, the wavefront's */
        constexpr int kStageTokens = 1024 * kWaves / D;
        int32_t value_page = -1;
        /* the page of the thread's values comes from another lane: asked for some time before its use */
        auto find_codes = [&] { value_page = __shfl(pages, (int)(4 * turn + (threadIdx.x & 3))); };
        auto load_codes = [&](uint32_t at) {
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                const uint32_t group = stage_group + k * kStageTokens / 16;
                const int32_t page = max(__builtin_amdgcn_readlane(pages, (int)(4 * turn + group)), 0);
                const uint8_t *keys = a.cache.data + kv_block(a.cache, page, 0, head) * (T * D) + ((at * kKVStep + group * 16) & (T - 1)) * D;
                raw_codes[COLUMNS ? k : 0] =
                    *reinterpret_cast<const kv_codes16 *>(keys + (stage_token + k * kStageTokens - group * 16) * D + stage_piece * 16);
            }
            const uint32_t token = at * kKVStep + 16 * (threadIdx.x & 3);
            value_good = value_page < 0 ? 0 : min(16, max(0, s.seen - (int32_t)token));
            value_partial = E4M3 && __any(value_good < 16);
            const uint8_t *from =
                a.cache.data + kv_block(a.cache, max(value_page, 0), 1, head) * (T * D) + (threadIdx.x >> 2) * T + (token & (T - 1));
#pragma unroll
            for (int k = 0; k < kPieces; ++k) raw_codes[COLUMNS ? kPieces + k : 0] = *reinterpret_cast<const kv_codes16 *>(from + k * 16 * kWaves * T);
        };
        /* half 0 or 1 of the k-th piece, eight codes, to its tile */
        auto write_codes = [&](int k, int part, uint8_t *to) {
            kv_codes16 v = raw_codes[COLUMNS ? k : 0];
            if (k < kPieces) {
                const uint32_t token = stage_token + k * kStageTokens, row = (token >> 4) * 4 + (token & 3);     /* n of the key row */
                to += ((token >> 2 & 3) * 16 + row) * 2 * D + ((2 * stage_piece + part) ^ kv_wide_turn<D>(row)) * 16;
            } else {
                if (E4M3 && value_partial) {
                    /* codes of tokens that no column of the slot sees may be any bytes, NaN among them */
#pragma unroll
                    for (int b = 2 * part; b < 2 * part + 2; ++b) {
                        const int left = value_good - 4 * b;
                        v[b] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
                    }
                }
                const uint32_t channel = (threadIdx.x >> 2) + (k - kPieces) * 16 * kWaves;
                to += 128 * D + channel * 128 + ((2 * (threadIdx.x & 3) + part) ^ kv_wide_value_turn(channel & 15)) * 16;
            }
            *reinterpret_cast<kv_half8 *>(to) = kv_decode8<E4M3>(v[2 * part], v[2 * part + 1]);
        };
        auto write_all = [&](uint8_t *to) {
#pragma unroll
            for (int k = 0; k < 4 * kPieces; ++k) write_codes(k / 2, k % 2, to);
        };

        /* Queries to fp16, scaled to a power of two by the largest of their row: a thread
         * takes eight channels, a row's threads are neighbours.  Lane (n, g) of the i-th
         * of a tile's 1 KiB has what it multiplies in the i-th product. */
        constexpr int kThreads = COLUMNS ? 64 : 64 * kWaves, kEights = D / 8;
        constexpr int kRows = COLUMNS ? kTile : NT * kTile, kEach = (kRows * kEights + kThreads - 1) / kThreads;
        uint32_t raw[kEach][SPLIT ? 8 : 4];
        const uint32_t eight = threadIdx.x % kEights, row_at = (COLUMNS ? lane : threadIdx.x) / kEights;
        auto load_queries = [&](uint32_t first) {
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const uint32_t c = first + k * (kThreads / kEights) + row_at, taken = min(c, s.columns - 1);
                kv_load8<SPLIT>(raw[k], a.query,
                                (s.first_row + s.row + s.row_of(a, taken)) * a.query_row +
                                    (head * a.group + s.head_of(a, taken)) * a.query_head + eight * 8);
            }
        };
        auto convert_queries = [&](uint32_t first, uint8_t *to) {
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const uint32_t at = k * (kThreads / kEights) + row_at, c = first + at;
                uint32_t largest = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    largest = max(largest, __float_as_uint(kv_element8<SPLIT>(raw[k], e, f16)) & 0x7fffffffu);
                /* non-negative floats order as their bits; NaN is above all of them */
                largest = kv_largest<kEights>(largest);
                const uint32_t exponent = max(largest >> 23, 30u);
                /* largest * scale is in 2^13..2^14; columns that are not there are zero */
                const float scale = c < s.columns ? __uint_as_float((267u - exponent) << 23) : 0.0f;
                if (kRows * kEights % kThreads && at >= kRows) break;
                if (eight == 0) to_exponent[c] = a.scale * __uint_as_float((exponent - 13u) << 23);
                kv_half8 high, low;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float v = c < s.columns ? kv_element8<SPLIT>(raw[k], e, f16) * scale : 0.0f;
                    const float w = c < s.columns ? kv_element8<SPLIT>(raw[k], e + 1, f16) * scale : 0.0f;
                    const kv_half2 a2 = kv_round2<false>(v, w, 0), b2 = kv_round2<SPLIT>(v, w, 0xffffffffu);
                    high[e] = a2[0], high[e + 1] = a2[1];
                    low[e] = b2[0], low[e + 1] = b2[1];
                }
                kv_half8 *fragment = reinterpret_cast<kv_half8 *>(to + at / kTile * kTileBytes) +
                                     ((eight >> 3) * 2 + (eight & 1)) * 64 + (eight >> 1 & 3) * 16 + at % kTile;
                fragment[0] = high;
                if (SPLIT) fragment[8] = low;
            }
        };

        /* The outputs' gates are asked for an item ahead, or here where a thread has two items at most */
        constexpr uint32_t kItems = kTile * (D / 4), kItemStep = COLUMNS ? 64 : 256, kEarlyGates = (kItems + 255) / 256;
        constexpr bool kEarly = !COLUMNS && NT == 1 && kEarlyGates <= 2;
        auto gate_of = [&](uint32_t first, uint32_t at) -> kv_float4 {
            const uint32_t of = first + at / (D / 4);
            if (!piece.whole || at >= kItems || of >= s.columns) return {0.0f, 0.0f, 0.0f, 0.0f};
            return kv_gate4(a, s.first_row + s.row + s.row_of(a, of), head * a.group + s.head_of(a, of), at % (D / 4) * 4);
        };
        kv_float4 early_gate[kEarly ? kEarlyGates : 1];

        kv_half8 q[COLUMNS ? NT : 1][2 * kChunks];
        if (COLUMNS) {
            load_pages(step);
            if (step < end) {
                find_codes();
                load_codes(step);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                uint8_t *to = ring + 256 * D + wave * kTileBytes;   /* the second tile */
                load_queries(first_column + t * kTile);
                convert_queries(first_column + t * kTile, to);
                kv_reads_done();
#pragma unroll
                for (int c = 0; c < 2 * kChunks; ++c) q[COLUMNS ? t : 0][c] = reinterpret_cast<const kv_half8 *>(to)[c * 64 + lane];
                kv_reads_done();
            }
            if (step < end) write_all(ring);
            kv_barrier();
        } else {
            load_queries(0);
            if (kEarly)
#pragma unroll
                for (uint32_t e = 0; e < kEarlyGates; ++e) early_gate[e] = gate_of(0, threadIdx.x + e * 256);
            /* here, so that nothing the compiler waits for is behind the copies */
#pragma unroll
            for (int k = 0; k < kEach; ++k)
#pragma unroll
                for (int e = 0; e < (SPLIT ? 8 : 4); ++e) asm volatile("" ::"v"(raw[k][e]));
            load_pages(step);
            if (step < end) {
                copy_keys(step, kv_lds(mine));
                copy_values(step, kv_lds(mine) + 64 * D);
            }
            convert_queries(0, queries);
            kv_barrier();
        }
        float to_u[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) to_u[t] = to_exponent[first_column + t * kTile + (SPLIT ? n & 7 : n)];

        kv_float4 o[NT][kChannels];
        float m[NT], l[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int c = 0; c < kChannels; ++c) o[t][c] = {0.0f, 0.0f, 0.0f, 0.0f};
        }

        auto accumulate = [](kv_float4 &sums, kv_half8 x, kv_half8 y, bool last) {
            if constexpr (kAccumulators) kv_accumulate(sums, x, y, last);
            else sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, sums, 0, 0, 0);
        };

        /* one step's columns: keys and values of `tile` */
        uint32_t tile = 0;
        while (step < end) {
            const bool more = step + kStride < end;
            if (!COLUMNS) kv_wait<kCopies>();                     /* the keys are there */
            const int32_t page = __shfl(pages, (int)(4 * turn + g));
            float key_scale = meta[4 * turn + g], value_scale = meta[64 + 4 * turn + g];
            const bool refresh = turn == 15;
            if (COLUMNS && more) {
                if (refresh) {
                    kv_reads_done();
                    load_pages(step + kStride);
                } else {
                    ++turn;
                }
                find_codes();
                if (step >= own_end) load_codes(step + kStride);
            }
            uint8_t *const next_tile = ring + (tile ^ (256 * D));
            const uint8_t *codes = mine + tile;
            if (!COLUMNS || step < own_end) {
                kv_float4 score[NT][4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < NT; ++t) score[t][i] = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (COLUMNS) {
                    /* 1 KiB fragments in the order (c, i), read ahead; the fences keep the compiler
                     * from reading all of them first, for which there are no registers */
                    constexpr int kAhead = 6, kFragments = 8 * kChunks;
                    kv_half8 fragment[kAhead + 1];
                    auto read = [&](int f) {
                        const int i = f % 4, c = f / 4;
                        return *reinterpret_cast<const kv_half8 *>(codes + (wide_key_at ^ (uint32_t)((8 * (c / 2) + (c & 1)) * 16)) +
                                                                   i * 32 * D);
                    };
#pragma unroll
                    for (int f = 0; f < kAhead; ++f) fragment[f] = read(f);
#pragma unroll
                    for (int f = 0; f < kFragments; ++f) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (f + kAhead < kFragments) fragment[(f + kAhead) % (kAhead + 1)] = read(f + kAhead);
#pragma unroll
                        for (int t = 0; t < NT; ++t)
                            score[t][f % 4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fragment[f % (kAhead + 1)], q[t][f / 4],
                                                                                     score[t][f % 4], 0, 0, 0);
                        if (f == kFragments / 4 && more) load_codes(step + kStride);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    /* queries in LDS: their registers hold the sums */
                    const kv_half8 *mine_q = reinterpret_cast<const kv_half8 *>(queries) + lane;
#pragma unroll
                    for (int j = 0; j < kChunks; ++j) {
                        const uint8_t *keys = codes + n * D + (((uint32_t)(4 * j + g) ^ kv_key_turn<D>(n)) & (D / 16 - 1)) * 16;
                        kv_half8 q0[NT], q1[NT];
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            q0[t] = mine_q[(t * 2 * kChunks + 2 * j) * 64];
                            q1[t] = mine_q[(t * 2 * kChunks + 2 * j + 1) * 64];
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 k = *reinterpret_cast<const uint4 *>(keys + i * 16 * D);
                            const kv_half8 low = kv_decode8<E4M3>(k.x, k.y), high = kv_decode8<E4M3>(k.z, k.w);
#pragma unroll
                            for (int t = 0; t < NT; ++t)
                                score[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(low, q0[t], score[t][i], 0, 0, 0);
#pragma unroll
                            for (int t = 0; t < NT; ++t)
                                score[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, q1[t], score[t][i], 0, 0, 0);
                        }
                    }
                }
                if (!COLUMNS && more) {
                    kv_reads_done();
                    ++turn;
                    if (refresh) load_pages(step + kStride);
                    copy_keys(step + kStride, kv_lds(mine));
                }

                if (page < 0) key_scale = value_scale = 1.0f;
                const uint32_t token = step * kKVStep + 16 * g;
                const uint32_t scale_bits = __float_as_uint(value_scale);
                const float value_log = value_scale == value_scale ? (float)((int)(scale_bits >> 23) - 127) : value_scale;
                const float inverse = __uint_as_float((254u << 23) - scale_bits);
                const bool whole = step * kKVStep + kKVStep <= (uint32_t)max(seen_least, 0) && __all(page >= 0);
                kv_half8 weight[NT][2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float factor = to_u[t] * key_scale;
                    const float base = value_log + kKVWeightExponent - m[t];
                    float u[16], most = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        if (SPLIT) score[t][e / 4][e & 3] += kv_partner(score[t][e / 4][e & 3]);
                        u[e] = fmaf(score[t][e / 4][e & 3], factor, base);
                    }
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (page < 0 || (int32_t)(token + e) >= seen[t]) u[e] = score[t][e / 4][e & 3] = -INFINITY;
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) most = fmaxf(most, u[e]);
                    const bool passed = __any(most > kKVWeightExponent + kKVMaximumSlack);
                    float keep = 1.0f;
                    uint64_t scaled = 0;
                    if (passed) {
                        /* a maximum was passed by that much (m = -inf: the first tokens): sums follow the new one */
                        most = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const bool hidden = score[t][e / 4][e & 3] == -INFINITY;
                            u[e] = hidden ? -INFINITY : fmaf(score[t][e / 4][e & 3], factor, value_log);
                            most = fmaxf(most, u[e]);
                        }
                        most = kv_other_rows(most, true);
                        const float now = fmaxf(m[t], most);
                        const float by = m[t] == now ? 0.0f : m[t] - now;
                        keep = exp2f(by);
                        scaled = __ballot(by != 0.0f && by != -INFINITY);
                        m[t] = now;
                        l[t] = kv_lower(l[t], by);
                        if (!kAccumulators)
#pragma unroll
                            for (int c = 0; c < kChannels; ++c) o[t][c] *= keep;
                        const float offset = kKVWeightExponent - (now == -INFINITY ? 0.0f : now);
#pragma unroll
                        for (int e = 0; e < 16; ++e) u[e] += offset;
                    }
                    if (kAccumulators && scaled)
#pragma unroll
                        for (int c = 0; c < kChannels; ++c) kv_scale(o[t][c], keep, kv_lds(bounce));
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float w = __builtin_amdgcn_exp2f(u[e]), v = __builtin_amdgcn_exp2f(u[e + 1]);
                        sum += w;
                        sum += v;
                        const kv_half2 pair = kv_round2<SPLIT>(w, v, low_half);
                        weight[t][e / 8][e & 7] = pair[0], weight[t][e / 8][(e & 7) + 1] = pair[1];
                    }
                    /* weights of a page whose value scale lies that far below the sums'
                     * largest leave fp32 before they leave the total: theirs is taken
                     * without the scale */
                    if (__any(value_log < m[t] - 64.0f && page >= 0)) {
                        const float back = value_scale == value_scale ? -value_log : 0.0f;
                        sum = 0.0f;
#pragma unroll
                        for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f(u[e] + back);
                        l[t] += sum;
                    } else {
                        l[t] = fmaf(sum, inverse, l[t]);
                    }
                }

                if (!COLUMNS) {
                    if (more) kv_wait<kCopies>();                 /* the values are there; the next keys may not be */
                    else kv_wait<0>();
                }
                if (E4M3 && !COLUMNS && !whole) {
                    /* codes of tokens that no column of the slot sees may be any bytes, NaN among
                     * them: made zero */
                    const int32_t good = page < 0 ? 0 : min(16, max(0, s.seen - (int32_t)token));
                    if (__any(good < 16))
#pragma unroll 1
                        for (int c = 0; c < kChannels; ++c) {
                            uint4 *at = reinterpret_cast<uint4 *>(mine + tile + value_at + c * 1024);
                            uint4 v = *at;
                            uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int b = 0; b < 4; ++b) {
                                const int left = good - 4 * b;
                                word[b] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
                            }
                            *at = make_uint4(word[0], word[1], word[2], word[3]);
                        }
                }
                if constexpr (COLUMNS) {
                    constexpr int kAhead = 6, kFragments = 2 * kChannels;
                    kv_half8 fragment[kAhead + 1];
                    /* four channel tiles' first halves, then their second ones: a product waits for the
                     * one before it on the same sums */
                    auto tile_of = [](int f) { return f / 8 * 4 + f % 4; };
                    auto read = [&](int f) {
                        return *reinterpret_cast<const kv_half8 *>(codes + (wide_value_at ^ (uint32_t)(f / 4 % 2 * 16)) +
                                                                   tile_of(f) * 2048);
                    };
#pragma unroll
                    for (int f = 0; f < kAhead; ++f) fragment[f] = read(f);
#pragma unroll
                    for (int f = 0; f < kFragments; ++f) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (f + kAhead < kFragments) fragment[(f + kAhead) % (kAhead + 1)] = read(f + kAhead);
#pragma unroll
                        for (int t = 0; t < NT; ++t)
                            accumulate(o[t][tile_of(f)], fragment[f % (kAhead + 1)], weight[t][f / 4 % 2], false);
                        /* the next step's codes, in the products' shadow (what is there without one goes unread) */
                        constexpr int kEvery = kFragments / (4 * kPieces);
                        if (f % kEvery == kEvery - 1) write_codes(f / kEvery / 2, f / kEvery % 2, next_tile);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    /* the next step's channels follow those that were read */
                    const uint8_t *from = !COLUMNS && more ? value_from(step + kStride) : nullptr;
                    uint4 next[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) next[c] = *reinterpret_cast<const uint4 *>(codes + value_at + c * 1024);
#pragma unroll
                    for (int c = 0; c < kChannels; c += 2) {
                        __builtin_amdgcn_sched_barrier(0);
                        const uint4 v = next[0], w = next[1];
                        if (c + 2 < kChannels)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                next[e] = *reinterpret_cast<const uint4 *>(codes + value_at + (c + 2 + e) * 1024);
                        /* first halves, then second ones: a product waits for the one before it on the same sums */
                        const kv_half8 v0 = kv_decode8<E4M3>(v.x, v.y), w0 = kv_decode8<E4M3>(w.x, w.y);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            accumulate(o[t][c], v0, weight[t][0], false);
                            accumulate(o[t][c + 1], w0, weight[t][0], false);
                        }
                        const kv_half8 v1 = kv_decode8<E4M3>(v.z, v.w), w1 = kv_decode8<E4M3>(w.z, w.w);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            accumulate(o[t][c], v1, weight[t][1], false);
                            accumulate(o[t][c + 1], w1, weight[t][1], c + 2 == kChannels && t == NT - 1);
                        }
                        if (!COLUMNS && more && c % 4 == 2) {
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                            for (int e = c - 2; e < c + 2; ++e) kv_copy16(from + e * 16 * T, kv_lds(mine) + 64 * D + e * 1024);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (COLUMNS) {
                if (more && step >= own_end) write_all(next_tile);
                kv_barrier();
                tile ^= 256 * D;
            }
            step += kStride;
        }

        kv_wait<0>();                               /* nothing is on its way to LDS */

        const uint32_t index = kv_place(blockIdx.x, piece.first_piece);
        float *partial = kv_partial(a, index, head), *stats = kv_stats(a, index, head);
        if (a.cut && head == 0 && piece.first_piece && threadIdx.x == 0) {
            uint32_t chunk = walk.chunk;
            asm volatile("" : "+v"(chunk));
            kv_records(a)[1 + s.index] = {piece.whole ? 1 : kv_pieces(piece.units, chunk, walk.at, piece.each),
                                          index, s.first_row + s.row, s.rem, s.columns, {0, 0, 0}};
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            l[t] = kv_other_rows(l[t], false);
            if (l[t] != l[t]) m[t] = INFINITY;      /* a NaN outweighs the other parts */
            if (g == 0 && (!SPLIT || n < 8)) {
                merge_m[(wave * NT + t) * kTile + n] = m[t];
                merge_l[(wave * NT + t) * kTile + n] = l[t];
            }
        }
        __syncthreads();                            /* also: every wavefront is done with its codes */
        /* tile by tile through LDS: rows of one column, from there on whole rows */
        float *merge_o = reinterpret_cast<float *>(ring);
        const uint32_t tiles = COLUMNS ? NT : (s.columns + kTile - 1) / kTile;
#pragma unroll 1
        for (uint32_t tile_at = 0; tile_at < tiles; ++tile_at) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (tile_at != t) continue;
#pragma unroll
                for (int c = 0; c < kChannels; ++c)
                    *reinterpret_cast<kv_float4 *>(&merge_o[(wave * 16 + n) * kPitch + c * 16 + 4 * g]) = o[t][c];
            }
            const uint32_t first = COLUMNS ? (wave * NT + tile_at) * kTile : tile_at * kTile;
            uint32_t at = COLUMNS ? lane : threadIdx.x;
            kv_float4 gate = kEarly ? early_gate[0] : gate_of(first, at);
            if (COLUMNS) kv_reads_done();           /* the wavefront's own rows; the writes too */
            else __syncthreads();
            for (; at < kItems; at += kItemStep) {
                const uint32_t c = at / (D / 4), d = at % (D / 4) * 4, of = first + c;
                if (of >= s.columns) break;
                const kv_float4 next_gate = kEarly ? early_gate[1 % kEarlyGates] : gate_of(first, at + kItemStep);
                float top = -INFINITY, total = 0.0f;
                kv_float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
                auto row = [&](uint32_t w) {
                    const float *from = &merge_o[(w * 16 + c) * kPitch + d];
                    const kv_float4 v = *reinterpret_cast<const kv_float4 *>(from);
                    return SPLIT ? v + *reinterpret_cast<const kv_float4 *>(from + 8 * kPitch) : v;
                };
                if (COLUMNS) {
                    top = merge_m[of];
                    total = merge_l[of];
                    sum = row(wave);
                } else {
                    float part_m[4], part_l[4];
                    kv_float4 part[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        part_m[w] = merge_m[w * NT * kTile + of];
                        part_l[w] = merge_l[w * NT * kTile + of];
                        part[w] = row(w);
                        top = fmaxf(top, part_m[w]);
                    }
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        /* (a wavefront without any token has sums of zero) */
                        const float by = part_m[w] == top ? 0.0f : part_m[w] - top;
                        total += kv_lower(part_l[w], by);
                        sum += part[w] * __builtin_amdgcn_exp2f(by);
                    }
                }
                if (piece.whole) {
                    kv_finish4(a, s.first_row + s.row + s.row_of(a, of), head * a.group + s.head_of(a, of), d, sum, total, gate);
                } else {
                    *reinterpret_cast<kv_float4 *>(partial + of * D + d) = sum;
                    if (d == 0) {
                        stats[2 * of] = top;
                        stats[2 * of + 1] = total;
                    }
                }
                gate = next_gate;
            }
            if (!COLUMNS) __syncthreads();
        }
        if (COLUMNS) __syncthreads();               /* the tiles are free for the next piece */
    }
}

template <int D>
bool launch_kv_attention_width(const KVAttention &a, hipStream_t stream);

}  // namespace q38
