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
 * One workgroup per (page touched, head, half): no other writes there.  A
 * thread holds eight times four channels of the page's tokens in registers, as
 * two groups of four tokens, so the rows are read once.  Keys are
 * [token][channel] and go out as they come; values are [channel][token]: four
 * tokens make a dword, and the dwords turn in LDS. */
#include "q38_kernels.h"
#include "q38_device.h"
#include "q38_kv.h"

namespace q38 {

namespace {

constexpr int kMostThreads = 1024, kQuads = 8;

struct KVAppend {
    Q38KVPages cache;     /* data and scales moved to the layer */
    KVRows rows;
    const void *key, *value;
    uint64_t row_stride;
    uint32_t page_shift, dim_shift;
};

/* the sequence whose slots hold `slot` (kv_slot_base of pages), found by the
 * whole wavefront: 64 sequences at a time, one per lane */
struct KVFound {
    int index;                      /* -1: none */
    uint32_t begin, end;            /* its rows */
    int32_t sequence;
};
__device__ __forceinline__ KVFound find_sequence(const KVRows &rows, uint32_t slot, uint32_t T)
{
    const uint32_t lane = threadIdx.x & 63;
    KVFound found{-1, 0, 0, -1};
    for (uint32_t first = 0; first < rows.count; first += 64) {
        const uint32_t i = first + lane;
        uint32_t begin = 0, end = 0;
        int32_t sequence = -1;
        if (i < rows.count) {
            begin = kv_row_start(rows, i);
            end = kv_row_start(rows, i + 1);
            sequence = rows.sequences[i];
        }
        const int before = __popcll(__ballot(i < rows.count && kv_slot_base(begin, i, 1, T, 2) <= slot));
        if (before)
            found = {(int)first + before - 1, (uint32_t)__builtin_amdgcn_readlane((int)begin, before - 1),
                     (uint32_t)__builtin_amdgcn_readlane((int)end, before - 1), __builtin_amdgcn_readlane(sequence, before - 1)};
        if (before < 64) break;
    }
    return found;
}

/* Row offsets that decrease, among those that the thread looks at.  A workgroup's
 * threads look at all of them: 4096 rows of one sequence 9.4 to 9.5 us, a row to
 * each of 512 sequences 31 to 33, of 1024 68 to 74. */
__device__ __forceinline__ bool rows_decrease(const KVRows &rows)
{
    bool bad = false;
    if (rows.row_starts)
        for (uint32_t i = threadIdx.x; i < rows.count; i += blockDim.x) bad |= kv_row_start(rows, i) > kv_row_start(rows, i + 1);
    return bad;
}

/* four elements at any alignment of their own */
template <int TYPE>
struct Raw4 {
    struct __attribute__((packed, aligned(2))) Words {
        uint32_t word[TYPE == kElementF32 ? 4 : 2];
    } bits;
    __device__ __forceinline__ void load(const void *base, uint64_t at)
    {
        bits = *reinterpret_cast<const Words *>(static_cast<const uint8_t *>(base) + at * (TYPE == kElementF32 ? 4 : 2));
    }
    __device__ __forceinline__ float element(int e) const
    {
        if constexpr (TYPE == kElementF32) return __uint_as_float(bits.word[e]);
        const uint32_t half = bits.word[e / 2] >> (e % 2 * 16) & 0xffffu;
        return TYPE == kElementF16 ? f16_to_f32(half) : __uint_as_float(half << 16);
    }
};

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

/* bytes of `word` that are codes before `used`, rounded to a scale 1 / shrink times as large */
template <bool E4M3>
__device__ __forceinline__ uint32_t follow(uint32_t word, uint32_t used, float shrink)
{
    uint32_t out = word;
    for (uint32_t e = 0; e < 4; ++e)
        if (e < used)
            out = (out & ~(0xffu << (8 * e))) | encode<E4M3>(decode<E4M3>(word >> (8 * e) & 0xffu) * shrink) << (8 * e);
    return out;
}

template <bool E4M3, int TYPE>
__global__ __launch_bounds__(kMostThreads) void kv_append_kernel(KVAppend a)
{
    extern __shared__ uint32_t turned[];      /* values: [channel][T / 4 + 1] dwords of four tokens */
    __shared__ uint32_t wave_largest[kMostThreads / 64];
    const uint32_t T = a.cache.page_tokens, D = a.cache.head_dim, threads = blockDim.x;
    const uint32_t slot = blockIdx.x, half = blockIdx.y & 1, head = blockIdx.y >> 1;
    /* the last slot is seldom any sequence's: a workgroup that has time to report bad offsets */
    if (slot == gridDim.x - 1 && blockIdx.y == 0 && rows_decrease(a.rows)) atomicOr(a.cache.status, Q38_KV_BAD_ROWS);
    const KVFound at_rows = find_sequence(a.rows, slot, T);
    const uint32_t begin = at_rows.begin, end = at_rows.end;
    if (at_rows.index < 0 || end <= begin) return;
    const int32_t sequence = at_rows.sequence;
    const uint32_t tokens = kv_tokens(a.cache, sequence);
    /* the page's new tokens: from .. to - 1 */
    const KVPageRows part = kv_page_rows(begin, end, tokens, slot, kv_slot_base(begin, at_rows.index, 1, T, 2), a.page_shift,
                                         a.cache.table_entries);
    if (!part.some) return;
    const uint32_t entry = part.entry, from = part.from, to = part.to;
    const int32_t page = kv_page(a.cache, sequence, entry);
    if (page < 0) {
        if (threadIdx.x == 0) atomicOr(a.cache.status, Q38_KV_BAD_PAGE);
        return;
    }
    const void *source = half ? a.value : a.key;
    /* element of the page's token 0 (which may lie before the rows), channel 0 */
    const uint64_t origin = ((uint64_t)end - tokens + entry * T) * a.row_stride + (uint64_t)head * D;
    const uint64_t block = kv_block(a.cache, page, half, head);
    uint8_t *codes = a.cache.data + block * (T * D);
    const float was = from ? a.cache.scales[block] : 0.0f;

    /* item k of a thread: token 4 (item / quads) + k % 4 of channels 4 (item % quads) .. */
    Raw4<TYPE> raw[kQuads];
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
        const uint32_t item = threadIdx.x + (k / 4) * threads, t = (item >> (a.dim_shift - 2)) * 4 + k % 4;
        /* a token that is not new stands in for none: the nearest that is */
        raw[k].load(source, origin + min(max(t, from), to - 1) * a.row_stride + (item & (D / 4 - 1)) * 4);
    }
    const bool decrease = rows_decrease(a.rows);       /* here: under way with the rows */
    float x[kQuads][4];
    uint32_t largest = 0;
#pragma unroll
    for (int k = 0; k < kQuads; ++k)
        for (int e = 0; e < 4; ++e) {
            x[k][e] = raw[k].element(e);
            largest = max(largest, __float_as_uint(x[k][e]) & 0x7fffffffu);
        }
    for (int by = 1; by < 64; by *= 2) largest = max(largest, (uint32_t)__shfl_xor((int)largest, by));
    if (__any(decrease)) largest = 0xffffffffu;       /* above all values: the call does nothing */
    if ((threadIdx.x & 63) == 0) wave_largest[threadIdx.x >> 6] = largest;
    __syncthreads();                                   /* also: every thread has read the old scale */
    for (uint32_t w = 0; w < threads / 64; ++w) largest = max(largest, wave_largest[w]);
    if (largest == 0xffffffffu) return;

    const bool finite = largest < 0x7f800000u;
    float scale = finite ? __uint_as_float((uint32_t)(kv_scale_exponent(largest, E4M3) + 127) << 23) : NAN;
    if (!(was <= scale) && finite) scale = was;        /* the larger, or an older NaN */
    if (threadIdx.x == 0) a.cache.scales[block] = scale;
    uint32_t *words = reinterpret_cast<uint32_t *>(codes);
    if (from && scale > was) {
        const float shrink = was / scale;
        if (!half) {
            for (uint32_t at = threadIdx.x; at < from * (D / 4); at += threads) words[at] = follow<E4M3>(words[at], 4, shrink);
        } else {
            const uint32_t shift = a.page_shift - 2;
            for (uint32_t at = threadIdx.x; at < D << shift; at += threads) {
                const uint32_t t = (at & (T / 4 - 1)) * 4;
                if (t < from) words[at] = follow<E4M3>(words[at], from - t, shrink);
            }
            __syncthreads();                           /* a dword of old codes may hold new ones too */
        }
    }
    const bool usable = scale == scale;
    const float inverse = usable ? 1.0f / scale : 0.0f;
    uint32_t code[kQuads][4];
#pragma unroll
    for (int k = 0; k < kQuads; ++k)
        for (int e = 0; e < 4; ++e) code[k][e] = usable ? encode<E4M3>(x[k][e] * inverse) : 0u;
    const bool turn = half && to - from >= 4;
    const uint32_t pitch = T / 4 + 1;
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
        const uint32_t item = threadIdx.x + (k / 4) * threads, group = item >> (a.dim_shift - 2), t = group * 4 + k % 4;
        const uint32_t d = (item & (D / 4 - 1)) * 4;
        if (turn) {
            /* of the four tokens, channel k % 4 here: 4 x 4 bytes turn in registers */
            const int b = k & ~3, e = k & 3;
            if (t - e < to) turned[(d + e) * pitch + group] = code[b][e] | code[b + 1][e] << 8 | code[b + 2][e] << 16 | code[b + 3][e] << 24;
        } else if (t >= from && t < to) {
            if (!half) words[(t * D + d) / 4] = code[k][0] | code[k][1] << 8 | code[k][2] << 16 | code[k][3] << 24;
            else
                for (int e = 0; e < 4; ++e) codes[(d + e) * T + t] = (uint8_t)code[k][e];
        }
    }
    if (!turn) return;
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < D << (a.page_shift - 2); at += threads) {
        const uint32_t d = at >> (a.page_shift - 2), group = at & (T / 4 - 1), t = group * 4;
        if (t >= to || t + 4 <= from) continue;
        const uint32_t word = turned[d * pitch + group];
        if (t >= from && t + 4 <= to) words[at] = word;
        else
            for (uint32_t e = 0; e < 4; ++e)
                if (t + e >= from && t + e < to) codes[d * T + t + e] = (uint8_t)(word >> (8 * e));
    }
}

template <bool E4M3, int TYPE>
bool launch_typed(const KVAppend &a, uint32_t slots, hipStream_t stream)
{
    KVAppend call = a;
    void *arguments[] = {&call};
    const uint32_t lds = a.cache.head_dim * (a.cache.page_tokens + 4);
    static_assert(kQuads == 8, "kv_append_threads");
    return hipLaunchKernel(reinterpret_cast<const void *>(kv_append_kernel<E4M3, TYPE>),
                           dim3(slots, 2 * a.cache.kv_heads), dim3(kv_append_threads(a.cache)), arguments, lds, stream) == hipSuccess;
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
    KVAppend a{cache, rows, key, value, row_stride, (uint32_t)__builtin_ctz(cache.page_tokens),
               (uint32_t)__builtin_ctz(cache.head_dim)};
    a.cache.data += (uint64_t)layer * cache.pages * kv_page_bytes(cache);
    a.cache.scales += (uint64_t)layer * cache.pages * 2 * cache.kv_heads;
    const uint32_t slots = (uint32_t)kv_slots(rows.total_rows, rows.count, 1, cache.page_tokens, 2);
    return cache.type == Q38_KV_E4M3 ? launch_kind<true>(a, type, slots, stream)
                                     : launch_kind<false>(a, type, slots, stream);
}

}  // namespace q38
